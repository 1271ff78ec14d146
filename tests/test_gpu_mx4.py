"""Microscaled 4-bit numbers and the products with weights of them, against 64 bits.

Quantisation has one right answer, number by number.  A product sums exact terms in 32 bits: held against 64 bits to 1e-5 of the largest result in
float32 (k rounding errors of 2^-24 of a partial sum each, their signs as they fall: sqrt(k) 2^-24, 4e-6 at the longest k here), and to half a step
of bfloat16 more where the result is rounded."""
from __future__ import annotations

import pytest
import torch

from divasun_common import assert_close
from test_gpu_divasun import rnd

pytestmark = pytest.mark.gpu

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
REL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8 + 1e-5}


def quantised(x):
    """``(codes [m, 32 * blocks], biased scales [m, blocks])`` in 64 bits; NaN blocks have the scale 255 and codes 0."""
    m, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(m, -1, 32)
    bad = ~torch.isfinite(b).all(2)
    b = torch.where(bad.unsqueeze(2), torch.zeros_like(b), b)
    top = b.abs().amax(2)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, torch.full_like(top, -127).int()).clamp(min=-127)
    y = torch.ldexp(b, -e.unsqueeze(2))
    gap = (y.abs().unsqueeze(-1) - GRID).abs()
    # the nearest; of two as near the one with the even code
    order = gap * 2 + (torch.arange(8) % 2) * 1e-12
    code = torch.where(y.abs() > 6, torch.full_like(y, 7).long(), order.argmin(-1)) + 8 * torch.signbit(b)
    return torch.where(bad.unsqueeze(2), torch.zeros_like(code), code).view(m, -1), torch.where(bad, torch.full_like(e, 255), e + 127)


def packed(codes):
    return (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8)


def values(codes, scales, k):
    v = torch.cat([GRID, -GRID])[codes].view(codes.shape[0], -1, 32) * torch.pow(2.0, (scales.double() - 127)).unsqueeze(2)
    return torch.where((scales == 255).unsqueeze(2), torch.full_like(v, float("nan")), v).view(codes.shape[0], -1)[:, :k]


def make(m, k, dtype, seed=0):
    """Rows with loud numbers, ties, zero blocks and both ends of the scales' range among them."""
    x = rnd(m, k, seed=seed)
    x[:, ::7] *= 20.0
    x[0, :min(k, 16)] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 7.9])[:min(k, 16)]
    if m > 2:
        x[1] = 0.0
        x[2] *= 2.0 ** -126
    if m > 4:
        x[3] *= 1e36
        x[4] *= 2.0 ** -120
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 257), (1, 4096), (130, 512), (9, 1000)])
def test_quantise(m, k, dtype):
    from llama_cu_amd.kernels import ops
    x = make(m, k, dtype, seed=m + k)
    codes, scales = quantised(x)
    wide = torch.full((m, k + 3), 9.0, dtype=dtype)
    wide[:, 1:1 + k] = x
    for got in (ops.mx4_quantize(x.cuda()), ops.mx4_quantize(wide.cuda()[:, 1:1 + k])):
        assert torch.equal(got.scales.cpu().int(), scales.int())
        assert torch.equal(got.codes.cpu(), packed(codes)) and got.shape == (m, k)
        want = values(codes, scales, k)
        assert torch.equal(ops.mx4_values(got, torch.float32).cpu().double(), want)
        assert torch.equal(ops.mx4_values(got).cpu().double(), want.bfloat16().double())
        mine = ops.Mx4(got.codes.clone(), got.scales.clone(), k)
        assert torch.equal(ops.mx4_values(mine, torch.float32).cpu().double(), want)


def test_quantise_rows_in_any_order():
    from llama_cu_amd.kernels import ops
    x = make(40, 96, torch.bfloat16)
    want = ops.mx4_quantize(x.cuda())
    for there in (x.cuda().t().contiguous().t(), x.cuda().repeat_interleave(2, 0)[::2]):
        got = ops.mx4_quantize(there)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    same = ops.mx4_quantize(x[:1].cuda().expand(5, 96))
    assert torch.equal(same.codes, want.codes[:1].expand(5, -1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_block_with_no_number_in_it(dtype):
    from llama_cu_amd.kernels import ops
    x = rnd(4, 128, seed=3).to(dtype)
    x[0, 5], x[1, 40], x[2, 127] = float("nan"), float("inf"), float("-inf")
    q = ops.mx4_quantize(x.cuda())
    bad = torch.zeros(4, 4, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    assert torch.equal(q.scales.cpu() == 255, bad)
    assert torch.equal(torch.isnan(ops.mx4_values(q).cpu()).view(4, 4, 32).all(2), bad) and torch.equal(torch.isnan(ops.mx4_values(q).cpu()).view(4, 4, 32).any(2), bad)
    # and it reaches its own row of a product, as a weight its own feature
    w = ops.pack_mx4(ops.mx4_quantize(rnd(48, 128, seed=4).bfloat16().cuda()))
    for y in (ops.gemm_mx4(q, w), ops.gemm_mx4(x.cuda(), w)):
        assert torch.equal(torch.isfinite(y).all(1).cpu(), torch.tensor([False, False, False, True]))
    as_weight = ops.pack_mx4(q)
    for rows in (rnd(3, 128, seed=5).to(dtype).cuda(), ops.mx4_quantize(rnd(3, 128, seed=5).to(dtype).cuda())):
        y = ops.gemm_mx4(rows, as_weight)
        assert torch.isnan(y[:, :3]).all() and torch.isfinite(y[:, 3]).all()


def test_every_code_at_every_scale():
    from llama_cu_amd.kernels import ops
    codes = torch.arange(256, dtype=torch.uint8).view(-1, 1).repeat(1, 16)
    codes[:, 1::2] = torch.arange(255, -1, -1, dtype=torch.uint8).view(-1, 1)
    scales = torch.arange(256, dtype=torch.uint8).view(-1, 1)
    loose = torch.stack([codes & 15, codes >> 4], 2).view(256, 32).long()
    want = values(loose, scales.int(), 32)
    q = ops.Mx4(codes.cuda(), scales.cuda(), 32)
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.mx4_values(q, dtype).cpu()
        assert torch.equal(torch.nan_to_num(got.double(), nan=-7.0), torch.nan_to_num(want.to(dtype).double(), nan=-7.0))


def weight(n, k, seed=1):
    from llama_cu_amd.kernels import ops
    w = rnd(n, k, seed=seed, std=k ** -0.5)
    w[:, ::11] *= 6.0
    codes, scales = quantised(w.bfloat16())
    return ops.pack_mx4(ops.Mx4(packed(codes).cuda(), scales.to(torch.uint8).cuda(), k)), values(codes, scales, k)


ROWS = [1, 3, 4, 5, 8, 9, 16, 17, 31, 33, 48, 65, 130]
SHAPES = [(16, 32), (48, 128), (40, 384), (130, 1000), (7, 33), (96, 640), (4104, 256), (33, 4096)]


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "four"])
@pytest.mark.parametrize("n,k", SHAPES)
def test_product(n, k, kind):
    from llama_cu_amd.kernels import ops
    w, exact = weight(n, k)
    for m in ROWS:
        x = make(m, k, torch.float32 if kind == "float32" else torch.bfloat16, seed=m)
        if m > 4:
            x[2:5] = rnd(3, k, seed=m + 1).to(x.dtype)          # (the others are then not measured by rows of 1e36)
        if kind == "four":
            rows, mine = ops.mx4_quantize(x.cuda()), values(*quantised(x), k)
        else:
            rows, mine = x.cuda(), x.double()
        want = mine @ exact.T
        for dtype in (torch.bfloat16, torch.float32):
            assert_close(ops.gemm_mx4(rows, w, out_dtype=dtype), want, REL[dtype], f"{m} rows to {dtype}")
        if n % 2 == 0:
            gate, up = want.chunk(2, 1)
            act = gate * torch.sigmoid(gate) * up
            for dtype in (torch.bfloat16, torch.float32):
                # (the gate's error passes through a slope of at most 1.1, the product's two factors add theirs)
                assert_close(ops.gemm_mx4(rows, w, out_dtype=dtype, swiglu=True), act, REL[dtype] + 2e-5, f"swiglu of {m} rows to {dtype}")


@pytest.mark.parametrize("shape", [(0, 1), (1, 1), (2, 1), (2, 3), (0, 2), (1, 5), (2, 100)])
@pytest.mark.parametrize("kind", ["bfloat16", "float32", "four"])
# fewer steps of k than a ring holds, as many, and more; tiles that end within rows and features; gate and up that meet within a tile of 16
@pytest.mark.parametrize("m,n,k", [(1, 48, 32), (127, 130, 128), (130, 258, 640), (257, 600, 1000), (300, 72, 1536), (515, 1030, 384)])
def test_product_in_tiles(m, n, k, kind, shape, monkeypatch):
    from llama_cu_amd.kernels import ops
    monkeypatch.setattr(ops, "mx4_choice", lambda *a: shape)
    w, exact = weight(n, k)
    x = rnd(m, k, seed=m).to(torch.float32 if kind == "float32" else torch.bfloat16)
    x[:, ::7] *= 20.0
    rows, mine = (ops.mx4_quantize(x.cuda()), values(*quantised(x), k)) if kind == "four" else (x.cuda(), x.double())
    want = mine @ exact.T
    gate, up = want.chunk(2, 1)
    act = gate * torch.sigmoid(gate) * up
    for dtype in (torch.bfloat16, torch.float32):
        for swiglu in (False, True):
            cols = n // 2 if swiglu else n
            got = ops.gemm_mx4(rows, w, out_dtype=dtype, swiglu=swiglu)
            assert_close(got, act if swiglu else want, REL[dtype] + 2e-5 * swiglu, f"{dtype} swiglu {swiglu}")
            for shift in (0, 3):
                room = torch.full((m + 2, cols + 11), 7.0, dtype=dtype, device="cuda")
                ops.gemm_mx4(rows, w, out=room[1:1 + m, shift:shift + cols], swiglu=swiglu)
                assert torch.equal(room[1:1 + m, shift:shift + cols], got)
                assert (room[0] == 7).all() and (room[m + 1:] == 7).all() and (room[:, :shift] == 7).all() and (room[:, shift + cols:] == 7).all()


@pytest.mark.parametrize("shape", [(-1, 1), (0, 1), (1, 1), (2, 1), (2, 2)])
@pytest.mark.parametrize("kind", ["bfloat16", "float32", "four"])
def test_rows_and_features_know_nothing_of_each_other(kind, shape, monkeypatch):
    """A row of NaN and a feature of NaN reach their own row and column only; what lies behind the rows' k and behind the last row is not looked at."""
    from llama_cu_amd.kernels import ops
    monkeypatch.setattr(ops, "mx4_choice", lambda *a: shape)
    m, n, k = 200, 144, 128
    wide = rnd(m + 1, 2 * k, seed=1).to(torch.float32 if kind == "float32" else torch.bfloat16)
    wide[:, k:] = float("nan")
    wide[m] = float("nan")
    wide[70, :k] = float("nan")
    source = rnd(n, k, seed=2).bfloat16()
    source[9] = float("inf")
    w = ops.pack_mx4(ops.mx4_quantize(source.cuda()))
    x = wide.cuda()[:m, :k]
    y = ops.gemm_mx4(ops.mx4_quantize(x) if kind == "four" else x, w).float().cpu()
    good = torch.ones(m, n, dtype=torch.bool)
    good[70] = False
    good[:, 9] = False
    assert torch.isfinite(y[good]).all() and torch.isnan(y[70]).all() and torch.isnan(y[:, 9]).all()


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "four"])
def test_where_the_product_goes(kind):
    """Into rows of wider memory, aligned or not, and nowhere else; from rows of wider memory, on any address."""
    from llama_cu_amd.kernels import ops
    m, n, k = 21, 70, 256
    w, exact = weight(n, k)
    wide = rnd(m, 3 * k, seed=7).to(torch.float32 if kind == "float32" else torch.bfloat16)
    wide[:, 2 * k + 5:] = float("nan")
    for at in (0, 8, 5):
        x = wide.cuda()[:, at:at + k]
        want = (values(*quantised(wide[:, at:at + k]), k) if kind == "four" else wide[:, at:at + k].double()) @ exact.T
        rows = ops.mx4_quantize(x) if kind == "four" else x
        for dtype in (torch.bfloat16, torch.float32):
            for shift in (0, 3):
                room = torch.full((m + 2, n + 9), 7.0, dtype=dtype, device="cuda")
                got = ops.gemm_mx4(rows, w, out=room[1:1 + m, shift:shift + n])
                assert got.data_ptr() == room[1:, shift:].data_ptr()
                assert_close(got, want, REL[dtype], f"{dtype} at {at}, {shift}")
                assert (room[0] == 7).all() and (room[m + 1:] == 7).all() and (room[:, :shift] == 7).all() and (room[:, shift + n:] == 7).all()


def test_rows_in_4_bits_of_other_memory():
    from llama_cu_amd.kernels import ops
    m, n, k = 19, 48, 224
    w, exact = weight(n, k)
    x = make(m, k, torch.bfloat16)
    x[2:5] = rnd(3, k).bfloat16()
    q = ops.mx4_quantize(x.cuda())
    codes, scales = torch.full((m, 16 * 7 + 5), 0xff, dtype=torch.uint8, device="cuda"), torch.full((m, 9), 0xff, dtype=torch.uint8, device="cuda")
    codes[:, 3:3 + 16 * 7] = q.codes
    scales[:, 1:8] = q.scales
    other = ops.Mx4(codes[:, 3:3 + 16 * 7], scales[:, 1:8], k)
    assert torch.equal(ops.gemm_mx4(other, w), ops.gemm_mx4(q, w))
    assert torch.equal(ops.mx4_values(other), ops.mx4_values(q))
    again = ops.pack_mx4(other)
    there = ops.pack_mx4(q)
    assert torch.equal(again.codes, there.codes) and torch.equal(again.scales, there.scales)


def test_rows_in_4_bits_that_were_changed():
    """What the scales are when the product is called counts, however many rows there are."""
    from llama_cu_amd.kernels import ops
    n, k = 64, 288
    w, exact = weight(n, k)
    for m in (4, 40, 200):
        q = ops.mx4_quantize(rnd(m, k, seed=m).bfloat16().cuda())
        before = ops.gemm_mx4(q, w, out_dtype=torch.float32)
        q.scales.add_(1)
        assert torch.equal(ops.gemm_mx4(q, w, out_dtype=torch.float32), 2 * before)
        q.scales[m // 2] = 255
        after = ops.gemm_mx4(q, w, out_dtype=torch.float32)
        assert torch.isnan(after[m // 2]).all() and torch.equal(after[:m // 2], 2 * before[:m // 2]) and torch.equal(after[m // 2 + 1:], 2 * before[m // 2 + 1:])


def test_rows_in_4_bits_that_are_changed_between_replays():
    """A captured product reads the scales that stand there when it is replayed, whether the rows were quantised before the capture, in another one or in its own."""
    from llama_cu_amd.kernels import ops
    n, k, m = 64, 288, 200
    w, _ = weight(n, k)
    x = rnd(m, k, seed=1).bfloat16().cuda()
    q = ops.mx4_quantize(x)
    ops.gemm_mx4(q, w), ops.gemm_mx4(ops.mx4_quantize(x), w)
    torch.cuda.synchronize()
    first, second, third = (torch.cuda.CUDAGraph() for _ in range(3))
    with torch.cuda.graph(first):
        of_eager = ops.gemm_mx4(q, w, out_dtype=torch.float32)
    with torch.cuda.graph(second):
        captured = ops.mx4_quantize(x)
        of_own = ops.gemm_mx4(captured, w, out_dtype=torch.float32)
    with torch.cuda.graph(third):
        of_other = ops.gemm_mx4(captured, w, out_dtype=torch.float32)
    for seed in (2, 3, 4):
        now = ops.mx4_quantize(rnd(m, k, seed=seed).bfloat16().cuda())
        q.codes.copy_(now.codes), q.scales.copy_(now.scales)
        first.replay()
        x.copy_(rnd(m, k, seed=seed + 10))
        second.replay()
        captured.scales.add_(1)
        third.replay()
        torch.cuda.synchronize()
        assert torch.equal(of_eager, ops.gemm_mx4(now, w, out_dtype=torch.float32))
        assert torch.equal(of_own, ops.gemm_mx4(ops.mx4_quantize(x), w, out_dtype=torch.float32))
        assert torch.equal(of_other, 2 * of_own) and torch.equal(ops.gemm_mx4(captured, w, out_dtype=torch.float32), of_other)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_in_inference_mode(m):
    from llama_cu_amd.kernels import ops
    w, _ = weight(64, 288)
    x = rnd(m, 288).bfloat16().cuda()
    want = ops.gemm_mx4(ops.mx4_quantize(x), w, out_dtype=torch.float32)
    outside = ops.mx4_quantize(x)
    with torch.inference_mode():
        inside = ops.mx4_quantize(x)
        for q in (inside, outside):
            assert torch.equal(ops.gemm_mx4(q, w, out_dtype=torch.float32), want)
            q.scales.add_(1)
            assert torch.equal(ops.gemm_mx4(q, w, out_dtype=torch.float32), 2 * want)
    assert torch.equal(ops.gemm_mx4(outside, w, out_dtype=torch.float32), 2 * want)


@pytest.mark.parametrize("m", [1, 3, 40, 200])
@pytest.mark.parametrize("k", [70, 257, 300])
def test_whatever_lies_behind_k(m, k):
    """Codes behind the last number, which a file may hold anything in, are not numbers of a row."""
    from llama_cu_amd.kernels import ops
    blocks = -(-k // 32)

    def filled(q):
        codes = q.codes.clone()
        codes[:, (k + 1) // 2:] = 0x77
        if k % 2:
            codes[:, k // 2] |= 0x70
        return ops.Mx4(codes, q.scales.clone(), k)

    source, rows = ops.mx4_quantize(rnd(48, k, seed=1).bfloat16().cuda()), ops.mx4_quantize(rnd(m, k, seed=2).bfloat16().cuda())
    assert source.codes.shape == (48, 16 * blocks)
    want = ops.gemm_mx4(rows, ops.pack_mx4(source))
    assert torch.equal(ops.gemm_mx4(filled(rows), ops.pack_mx4(filled(source))), want)
    assert torch.equal(ops.mx4_values(filled(rows)), ops.mx4_values(rows))


def test_copies_of_rows_in_4_bits():
    import copy
    from llama_cu_amd.kernels import ops
    w, _ = weight(64, 300)
    q = ops.mx4_quantize(rnd(40, 300).bfloat16().cuda())
    want = ops.gemm_mx4(q, w)
    for other in (copy.copy(q), copy.deepcopy(q), ops.Mx4(q.codes.cpu().cuda(), q.scales.cpu().cuda(), 300)):
        assert torch.equal(ops.gemm_mx4(other, w), want)


def test_infinities_of_32_bit_rows():
    from llama_cu_amd.kernels import ops
    w, exact = weight(32, 128)
    x = rnd(4, 128, seed=2)
    x[0, 3], x[1, 4], x[2, 5] = float("inf"), float("-inf"), 3.3e38
    y = ops.gemm_mx4(x.cuda(), w).cpu()
    want = x.double() @ exact.T
    some = exact[:, 3] != 0
    assert torch.equal(y[0, some].double(), want[0, some]) and torch.equal(y[1, exact[:, 4] != 0].double(), want[1, exact[:, 4] != 0])
    assert torch.isnan(y[0, ~some]).all()
    finite = want[2].abs() < 3.4e38
    assert_close(y[2, finite], want[2, finite], 1e-5)


def test_empty_and_captured():
    from llama_cu_amd.kernels import ops
    w, exact = weight(64, 256)
    assert ops.gemm_mx4(torch.empty(0, 256, dtype=torch.bfloat16, device="cuda"), w).shape == (0, 64)
    assert ops.gemm_mx4(ops.mx4_quantize(torch.empty(0, 256, device="cuda")), w, swiglu=True).shape == (0, 32)
    assert ops.mx4_values(ops.mx4_quantize(torch.empty(3, 0, device="cuda"))).shape == (3, 0)
    x = torch.empty(5, 256, device="cuda")
    x.copy_(rnd(5, 256, seed=1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            ops.gemm_mx4(x, w), ops.gemm_mx4(ops.mx4_quantize(x), w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        full, four = ops.gemm_mx4(x, w), ops.gemm_mx4(ops.mx4_quantize(x), w)
    for seed in (2, 3, 4):
        x.copy_(rnd(5, 256, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(full, ops.gemm_mx4(x, w)) and torch.equal(four, ops.gemm_mx4(ops.mx4_quantize(x), w))
        assert_close(full, rnd(5, 256, seed=seed).double() @ exact.T, 1e-5)


def test_two_streams_at_once():
    from llama_cu_amd.kernels import ops
    w, exact = weight(512, 512)
    xs = [rnd(24, 512, seed=s).cuda() for s in range(2)]
    want = [ops.gemm_mx4(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.gemm_mx4(xs[i], w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_rows_in_4_bits_on_another_stream():
    """Rows that another stream made: what their maker keeps beside the codes and scales is not read, for nobody can tell its allocator of that use."""
    from llama_cu_amd.kernels import ops
    n, k, m = 64, 288, 200
    w, _ = weight(n, k)
    q = ops.mx4_quantize(rnd(m, k, seed=1).bfloat16().cuda())
    want = ops.gemm_mx4(q, w, out_dtype=torch.float32)
    blocks = q.scales.shape[1]
    whole = ops._mx4_whole(q, blocks)
    assert ops._mx4_by_pair(whole, blocks, ops.raw_stream()) is q._by_pair
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = ops._mx4_by_pair(whole, blocks, ops.raw_stream())
        got = ops.gemm_mx4(q, w, out_dtype=torch.float32)
    torch.cuda.current_stream().wait_stream(side)
    assert there.data_ptr() != q._by_pair.data_ptr() and torch.equal(there, q._by_pair) and torch.equal(got, want)
