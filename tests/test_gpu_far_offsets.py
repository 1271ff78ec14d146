"""4-bit rows and products, distributions and verification where places lie beyond 32 bits: rows of more than 4 GiB, more than 2^31 numbers.

A few rows at the front, at the end and at the borders of 2^31 and 2^32 bytes are held against plain 64-bit results, the tolerances being those of the small cases."""
from __future__ import annotations

import pytest
import torch

from divasun_common import assert_close
from test_gpu_mx4 import REL, quantised, values, weight
from test_gpu_token_probs import check
from test_gpu_verify import plain

pytestmark = pytest.mark.gpu


def far(m, k, dtype, seed):
    """Rows made on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(m, k, dtype=dtype, device="cuda").normal_(generator=g)


def some(m, row_bytes):
    """The first rows, the last, and those around every border of 2^31 bytes."""
    rows = {0, 1, m - 1, m - 2, m // 2}
    for border in range(1, m * row_bytes >> 31):
        at = (border << 31) // row_bytes
        rows |= {at - 513, at - 512, at - 1, at, at + 1}
    return sorted(r for r in rows if 0 <= r < m)


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "four"])
def test_products(kind):
    from llama_cu_amd.kernels import ops
    k, n = {"bfloat16": (2048, 40), "float32": (512, 33), "four": (8192, 24)}[kind]
    m = 1_049_601 if kind != "float32" else 1_400_003           # (three planes of bfloat16: 3 KB a row)
    row_bytes = {"bfloat16": 2 * k, "float32": 6 * k, "four": k // 2}[kind]
    assert m * row_bytes > 1 << 32
    w, exact = weight(n, k)
    x = far(m, k, torch.float32 if kind == "float32" else torch.bfloat16, 1)
    rows = some(m, row_bytes)
    mine = x[rows].cpu()
    if kind == "four":
        x = ops.mx4_quantize(x)
        codes, scales = quantised(mine)
        mine = values(codes, scales, k)
        assert torch.equal(ops.mx4_values(ops.Mx4(x.codes[rows], x.scales[rows], k), torch.float32).cpu().double(), mine)
        assert torch.equal(ops.mx4_values(x)[rows].cpu().double(), mine)
    got = ops.gemm_mx4(x, w, out_dtype=torch.float32)
    assert got.shape == (m, n)
    assert_close(got[rows], mine.double() @ exact.T, REL[torch.float32], kind)


def test_distributions():
    from llama_cu_amd import sampling
    rows, vocab = 17_001, 128_256
    assert rows * vocab > 1 << 31
    logits = far(rows, vocab, torch.float32, 2).mul_(3.0)
    kinds = [(0.8, 0.9, vocab), (1.0, 1.0, 50), (0.0, 1.0, vocab), (1.2, 0.95, 200), (1.0, 1.0, vocab)]
    ts, ps, ks = ([kinds[r % 5][i] for r in range(rows)] for i in range(3))
    got = sampling.token_probs(logits, ts, ps, ks)
    at = some(rows, 4 * vocab)
    check(got[at], logits[at].cpu(), [ts[r] for r in at], [ps[r] for r in at], [ks[r] for r in at])


def test_verification():
    from llama_cu_amd import sampling
    requests, most, vocab = 5_700, 2, 128_259
    rows, n = 3 * requests, 2 * requests
    assert rows * vocab > 1 << 31
    probs = torch.softmax(far(rows, vocab, torch.float32, 3).mul_(2.0), 1)
    q = torch.softmax(far(n, vocab, torch.float32, 4).mul_(2.0), 1)
    g = torch.Generator().manual_seed(5)
    number = lambda m: torch.randint(0, 1 << 24, (m,), generator=g).float() / (1 << 24)
    # a draft the target likes best, or any
    best = probs.argmax(1).cpu().view(requests, 3)[:, :2].reshape(-1)
    drafts = torch.where(torch.rand(n, generator=g) < 0.6, best, torch.randint(0, vocab, (n,), generator=g)).int()
    accept, final = number(n), number(requests)
    starts = torch.arange(0, rows + 1, 3, dtype=torch.int32)
    accepted, tokens = sampling.verify_drafts(probs, starts.cuda(), drafts.cuda(), accept.cuda(), final.cuda(), most, q)
    for b in [0, 1, requests // 2, requests - 2, requests - 1]:
        want_n, want, near = plain(probs[3 * b:3 * b + 3].cpu(), [0, 3], drafts[2 * b:2 * b + 2], accept[2 * b:2 * b + 2], final[b:b + 1], most, q[2 * b:2 * b + 2].cpu())
        assert accepted[b].item() == want_n[0]
        assert tokens[b].tolist() == want[0] or near[0] < 1e-12
