"""The distribution that temperature, top_p and top_k leave of a row of logits, against 64 bits.

A share is a weight exp(-d) over a sum of weights.  In 32 bits the distance d <= 104 carries a rounding of the difference and one of the product with
1 / T, itself rounded, d * 1.5 * 2^-23 at most together, so a weight is off by d * 1.8e-7 relative and the exponential's own last places; weights fall
with d, and d exp(-d) <= 0.37, so against the row's largest share everything is within 2e-6, and each share that is kept whole within
(d + 8) * 4e-7 of itself.  The entry at the cut holds the rest of a sum: off by the errors of all weights above it, 2e-6 of the whole at most."""
from __future__ import annotations

import pytest
import torch

from llama_cu_amd.kernels.ops import KernelError
from test_gpu_divasun import rnd

pytestmark = pytest.mark.gpu

CAP = 8192              # entries that the kernel gathers of a row


def exact(row, t, p, k):
    """``(shares, entries kept, place of the entry at the cut or -1)``."""
    v = row.numel()
    out = torch.zeros(v, dtype=torch.float64)
    l = torch.where(torch.isnan(row), torch.full_like(row, -float("inf")), row)
    order = torch.sort(l, descending=True, stable=True)[1]
    best = l[order[0]]
    if best == -float("inf"):
        return out, 0, -1
    if t == 0 or k == 1:
        out[order[0]] = 1.0
        return out, 1, -1
    s = l[order].double()
    d = torch.where(s == s[0], torch.zeros_like(s), (s - s[0]) / torch.tensor(t, dtype=torch.float32).double())
    w = torch.exp(d)
    c = torch.cumsum(w, 0)
    limit = c[min(k, v) - 1]
    if p < 1:
        limit = torch.minimum(limit, torch.tensor(p, dtype=torch.float32).double() * c[-1])
    # (a weight that is kept whole as it is: the difference of two sums has not its digits)
    share = torch.where(c <= limit, w, (limit - (c - w)).clamp(min=0)) / limit
    out[order] = share
    kept = int((share > 0).sum())
    return out, kept, int(order[kept - 1]) if p < 1 else -1


def check(got, logits, ts, ps, ks, what=""):
    got = got.cpu().double()
    assert torch.isfinite(got).all() and (got >= 0).all()
    for r in range(logits.shape[0]):
        want, kept, edge = exact(logits[r], ts[r], ps[r], ks[r])
        name = f"{what} row {r}: T {ts[r]} top_p {ps[r]} top_k {ks[r]}"
        diff = (got[r] - want).abs()
        assert diff.max() <= 4e-6, f"{name}: off by {diff.max():.2e}"
        if kept:
            assert abs(got[r].sum() - 1) < 2e-5, name
        # entry by entry, but for those next to the cut: equal ones that one side keeps and the other does not lie there
        whole = want > 0
        if edge >= 0:
            whole &= logits[r] > logits[r][edge]
            low = logits[r] < logits[r][edge]
            if ts[r] > 0 and kept > 1:
                at_edge = want[whole].sum()
                # (the cut may fall on the neighbouring entry where it lies within the sums' error of a border)
                if 1 - at_edge > 4e-6 and want[edge] > 4e-6 and (want[edge] < want[whole].min() - 4e-6 if whole.any() else True):
                    assert (got[r][low] == 0).all(), name
        else:
            assert (got[r][want == 0] <= 1e-30).all(), name
        if whole.any() and ts[r] > 0:
            far = -torch.log(want[whole] / want.max())
            assert ((got[r][whole] / want[whole] - 1).abs() <= (far + 8) * 4e-7 + 2e-6).all(), name


def run(logits, ts, ps, ks):
    from llama_cu_amd import sampling
    return sampling.token_probs(logits.cuda(), ts, ps, ks)


OPTIONS = [(1.0, 1.0, 10 ** 9), (0.7, 0.9, 10 ** 9), (1.0, 1.0, 40), (1.3, 0.95, 100), (0.0, 0.5, 7), (2.0, 0.3, 1), (0.01, 0.99, 5), (50.0, 0.5, 10 ** 9),
           (1.0, 1e-6, 10 ** 9), (1.0, 1 - 2.0 ** -20, 3), (0.8, 0.999, 2), (1e-30, 0.9, 20)]


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 257, 1000, 1025, 4096, 4097, 8192, 8193, 32003])
def test_options(vocab):
    n = len(OPTIONS)
    logits = rnd(n, vocab, seed=vocab, std=3.0)
    ts, ps, ks = ([o[i] for o in OPTIONS] for i in range(3))
    check(run(logits, ts, ps, ks), logits, ts, ps, ks, f"vocabulary {vocab}")
    # more rows than a launch holds the options of
    many = run(logits.repeat(6, 1), ts * 6, ps * 6, ks * 6)
    assert torch.equal(many, run(logits, ts, ps, ks).repeat(6, 1)) or vocab > 8192          # (a long row's sums go by its parts, which are fewer of many rows)
    check(many, logits.repeat(6, 1), ts * 6, ps * 6, ks * 6, "many")
    # each alone: in more parts a row, and rows without a cut on their own
    for i in range(n):
        check(run(logits[i:i + 1], ts[i:i + 1], ps[i:i + 1], ks[i:i + 1]), logits[i:i + 1], ts[i:i + 1], ps[i:i + 1], ks[i:i + 1], "alone")


@pytest.mark.parametrize("vocab", [20001, 128256])
def test_rows_that_keep_more_than_is_gathered(vocab):
    """A flat distribution, of which tens of thousands of entries are kept: only those near the cut are gathered."""
    logits = rnd(5, vocab, seed=1, std=1.0)
    ts, ps, ks = [1.0, 1.0, 0.9, 1.0, 5.0], [0.9, 1.0, 0.97, 0.9999, 0.6], [10 ** 9, 15000, 18000, 10 ** 9, 10 ** 9]
    check(run(logits, ts, ps, ks), logits, ts, ps, ks)


@pytest.mark.parametrize("vocab", [300, 30000])
def test_equal_logits(vocab):
    """Equal logits are kept in the order of their indices; as many as are not gathered are found by searching the row."""
    same = torch.zeros(6, vocab)
    coarse = (rnd(6, vocab, seed=2, std=2.0) * 2).round() / 2
    ts, ps, ks = [1.0, 1.0, 0.5, 1.0, 1.0, 0.0], [0.5, 1.0, 0.25, 1.0, 0.9, 1.0], [10 ** 9, 77, vocab // 2, vocab - 1, vocab // 3, 5]
    for logits in (same, coarse):
        got = run(logits, ts, ps, ks).cpu()
        for r in range(6):
            want, kept, edge = exact(logits[r], ts[r], ps[r], ks[r])
            assert (got[r].double() - want).abs().max() <= 4e-6
            l = logits[r]
            if ps[r] == 1.0 and ts[r] > 0:            # a count: exactly which
                assert torch.equal(got[r] > 0, want > 0)
            # of equal logits the first ones: no entry is kept behind one that is not
            for value in l.unique():
                kept_here = got[r][l == value] > 0
                assert torch.equal(kept_here, kept_here.sort(descending=True, stable=True)[0])


@pytest.mark.parametrize("vocab", [20000, 20001])
@pytest.mark.parametrize("times", [1, 14])
def test_rows_of_every_kind_together(vocab, times):
    """A row whose kept entries are gathered, one of which only those near the cut are, one that is searched, one without a cut, a greedy and an empty one: beside each other, in
    few rows (whose last launch does more) and in many."""
    logits = rnd(6, vocab, seed=vocab, std=3.0)
    logits[1] /= 3
    logits[2] = 0
    logits[5] = -float("inf")
    ts, ps, ks = [0.8, 1.0, 1.0, 1.2, 0.0, 1.0], [0.95, 0.97, 0.6, 1.0, 1.0, 0.9], [10 ** 9, 15000, 10 ** 9, 10 ** 9, 3, 50]
    got = run(logits.repeat(times, 1), ts * times, ps * times, ks * times).cpu()
    assert torch.equal(got, got[:6].repeat(times, 1))
    check(got[:5], logits[:5], ts[:5], ps[:5], ks[:5])
    assert (got[5] == 0).all()
    want, _, _ = exact(logits[2], 1.0, 0.6, 10 ** 9)
    assert (got[2].double() - want).abs().max() <= 4e-6 and torch.equal(got[2] > 0, want > 0)


@pytest.mark.parametrize("vocab", [300, 6000, 30000])
@pytest.mark.parametrize("apart", [1, 3, 40])
def test_logits_a_few_steps_apart_at_the_cut(vocab, apart):
    """Logits whose last places alone tell them apart, the cut at each of them in turn, and a smallest one that makes the keys differ in any number of bits."""
    near = 1.0 + torch.arange(60).flip(0) * apart * 2.0 ** -23
    rows, ts, ps, ks = [], [], [], []
    for i in range(60):
        row = torch.full((vocab,), -float("inf"))
        at = torch.randperm(vocab, generator=torch.Generator().manual_seed(i))
        row[at[:60]] = near
        row[at[60:160]] = near[-1] - 2.0 ** (i % 24 - 22) * (1 + torch.arange(100) / 100)
        rows.append(row)
        ts.append(1.0)
        ps.append(1.0 if i % 3 else 0.5)
        ks.append(i + 1 if i % 3 else vocab)
    logits = torch.stack(rows)
    got = run(logits, ts, ps, ks)
    cut = [i for i in range(60) if i % 3 == 0]
    check(got[cut], logits[cut], [1.0] * 20, [0.5] * 20, [vocab] * 20, f"{apart} steps apart")
    for i in range(60):
        if i % 3:                       # as many entries as were asked for, and the first of them (`check` would take the oracle's 1e-17 behind them for an entry)
            kept = logits[i] >= near[i]
            assert int(kept.sum()) == i + 1 and torch.equal((got[i] > 0).cpu(), kept)
            want = torch.softmax(logits[i][kept].double(), 0)
            assert ((got[i].cpu()[kept] / want - 1).abs() <= 5.2e-6).all()


@pytest.mark.parametrize("vocab", [5, 300, 6000, 30000])
def test_a_top_p_of_nearly_nothing(vocab):
    """The first entry has all, however small the part of the sum is that is asked for."""
    logits = rnd(4, vocab, seed=vocab)
    logits[1] = 0.0
    for p in (1e-12, 1e-14, 1e-20, 1e-38):
        for k in (vocab, 3):
            got = run(logits, [1.0] * 4, [p] * 4, [k] * 4).cpu()
            assert torch.equal(got, torch.nn.functional.one_hot(logits.argmax(1), vocab).float()), (p, k)


def test_masked_logits():
    inf, low = float("inf"), torch.finfo(torch.float32).min
    v = 5000
    logits = rnd(10, v, seed=4, std=2.0)
    logits[0, 10:] = -inf
    logits[1] = -inf
    logits[2, :-1] = -inf
    logits[3, ::2] = low
    logits[4, 7] = float("nan")
    logits[5, 100], logits[5, 200] = inf, inf
    logits[6] = float("nan")
    logits[7] = low
    logits[8, 1:] = low
    logits[9, ::3] = float("nan")
    for t, p, k in ((1.0, 1.0, 10 ** 9), (0.9, 0.9, 10 ** 9), (1.0, 1.0, 50), (1.0, 0.8, 5), (0.0, 1.0, 10 ** 9), (1.0, 1.0, 4999)):
        ts, ps, ks = [t] * 10, [p] * 10, [k] * 10
        check(run(logits, ts, ps, ks), logits, ts, ps, ks)
    assert (run(logits, [1.0] * 10, [1.0] * 10, [9] * 10)[1] == 0).all()
    # whatever the temperature, -inf has no share
    for t in (1e-38, 1e38, 3.4e38, 1e300):
        got = run(logits[:1], [t], [1.0], [v])
        assert (got[0, 10:] == 0).all() and abs(float(got.sum()) - 1) < 1e-5


def test_where_it_reads_and_writes():
    from llama_cu_amd import sampling
    v = 1000
    wide = rnd(6, v + 25, seed=3, std=2.0)
    opts = ([0.8] * 6, [0.9, 1.0] * 3, [40, 10 ** 9, 10 ** 9] * 2)
    for at in (0, 1, 4):
        logits = wide[:, at:at + v]
        there = wide.cuda()[:, at:at + v]
        room = torch.full((8, v), 7.0, device="cuda")
        got = sampling.token_probs(there, *opts, out=room[1:7])
        assert got.data_ptr() == room[1:7].data_ptr() and (room[0] == 7).all() and (room[7] == 7).all()
        check(got, logits, *opts)
        as_tensors = [torch.tensor(o).cuda() for o in opts[:2]] + [torch.tensor([min(k, v) for k in opts[2]], dtype=torch.int32).cuda()]
        assert torch.equal(sampling.token_probs(there, *as_tensors), got)
    assert sampling.token_probs(there[:0], [], [], []).shape == (0, v)
    # numbers that nobody looked at: the largest logit
    odd = sampling.token_probs(there, torch.tensor([-1.0, float("nan"), 0.0, 1.0, 1.0, 1.0]).cuda(), torch.tensor([1.0, 1.0, 1.0, 0.0, -2.0, 1.0]).cuda(),
                               torch.tensor([v, v, v, v, v, -3], dtype=torch.int32).cuda())
    assert torch.equal(odd.argmax(1), there.argmax(1)) and (odd.max(1)[0] == 1).all() and (odd.sum(1) == 1).all()


def test_it_is_what_sample_rows_draws_from():
    """A draw with the number u is the first entry, in descending order of the logits, at which the shares' sum reaches u."""
    from llama_cu_amd import sampling
    rows, v = 16, 700
    logits = rnd(rows, v, seed=6, std=3.0)
    ts, ps, ks = [0.5 + 0.1 * i for i in range(rows)], [0.6 + 0.025 * i for i in range(rows)], [3 + 20 * i for i in range(rows)]
    probs = run(logits, ts, ps, ks).cpu().double()
    for j in range(40):
        u = (j + 0.5) / 40
        got = sampling.sample_rows(logits.cuda(), ts, ps, ks, [u] * rows).tolist()
        for r in range(rows):
            order = torch.sort(logits[r], descending=True, stable=True)[1]
            reach = torch.cumsum(probs[r][order], 0)
            i = int((order == got[r]).nonzero())
            assert reach[i] >= u - 1e-5 and (i == 0 or reach[i - 1] <= u + 1e-5)


@pytest.mark.parametrize("v", [900, 9000, 40000])
def test_captured(v):
    from llama_cu_amd import sampling
    rows = 4
    options = [torch.tensor([0.7, 1.0, 0.0, 1.3]).cuda(), torch.tensor([0.9, 1.0, 1.0, 1.0]).cuda(), torch.tensor([v, v, v, 30], dtype=torch.int32).cuda()]
    logits = rnd(rows, v, seed=1, std=3.0).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sampling.token_probs(logits, *options)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sampling.token_probs(logits, *options)
        again = sampling.token_probs(logits, [0.7, 1.0, 0.0, 1.3], [0.9, 1.0, 1.0, 1.0], [v, v, v, 30])
        with pytest.raises(KernelError, match="as tensors"):
            sampling.token_probs(logits, options[0], [1.0] * rows, [v] * rows)
        with pytest.raises(KernelError, match="as tensors"):
            sampling.token_probs(logits[:1].expand(65, v).contiguous(), [1.0] * 65, [1.0] * 65, [v] * 65)
    for seed in (2, 3, 4, 5):
        logits.copy_(rnd(rows, v, seed=seed, std=3.0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, sampling.token_probs(logits, *options)) and torch.equal(again, got)
