"""Verification of drafted tokens: token for token what the definition gives in 64 bits, and the target's distribution in the long run."""
from __future__ import annotations

import pytest
import torch

from test_gpu_divasun import rnd

pytestmark = pytest.mark.gpu


def clean(t):
    return torch.where((t > 0) & torch.isfinite(t), t, torch.zeros_like(t)).double()


def plain(probs, starts, drafts, accept, final, most, draft_probs=None):
    """``(accepted, tokens, distance of the drawn number from the nearest border)``, request by request."""
    accepted, tokens, near = [], [], []
    vocab = probs.shape[1]
    for b in range(len(starts) - 1):
        row, count = starts[b], starts[b + 1] - starts[b] - 1
        d, taken = row - b, 0
        while taken < count:
            t = int(drafts[d + taken])
            if not 0 <= t < vocab:
                break
            q = 1.0 if draft_probs is None else float(clean(draft_probs[d + taken, t]))
            if not float(accept[d + taken]) * q < float(clean(probs[row + taken, t])):
                break
            taken += 1
        left = clean(probs[row + taken])
        if taken < count:
            if draft_probs is None:
                rest = left.clone()
                if 0 <= drafts[d + taken] < vocab:
                    rest[drafts[d + taken]] = 0
            else:
                rest = (left - clean(draft_probs[d + taken])).clamp(min=0)
            if rest.sum() > 0:
                left = rest
        c = torch.cumsum(left, 0)
        goal = float(final[b]) * float(c[-1])
        if c[-1] > 0:
            token = int((c > goal).nonzero()[0]) if bool((c > goal).any()) else int((left > 0).nonzero()[-1])
            near.append(float((c - goal).abs().min() / c[-1]))
        else:
            token = -1
            near.append(1.0)
        accepted.append(taken)
        tokens.append(drafts[d:d + taken].tolist() + [token] + [-1] * (most - taken))
    return accepted, tokens, near


def agree(probs, starts, drafts, accept, final, most, draft_probs=None):
    from llama_cu_amd import sampling
    got = sampling.verify_drafts(probs.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), drafts.cuda(), accept.cuda(), final.cuda(), most,
                                 None if draft_probs is None else draft_probs.cuda())
    accepted, tokens, near = plain(probs, starts, drafts, accept, final, most, draft_probs)
    assert got[0].tolist() == accepted
    for b, (have, want) in enumerate(zip(got[1].tolist(), tokens)):
        # 64-bit sums in another order: a border nearer than their error may fall either way
        assert have == want or near[b] < 1e-12, (b, have, want, near[b])
    return accepted


def case(requests, most, vocab, seed, ragged=True, std=2.0, apart=0.7):
    g = torch.Generator().manual_seed(seed)
    counts = torch.randint(0, most + 1, (requests,), generator=g).tolist() if ragged else [most] * requests
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c + 1)
    n = sum(counts)
    logits = torch.randn(n + requests, vocab, generator=g) * std
    of = [starts[b] + i for b in range(requests) for i in range(counts[b])]
    probs = torch.softmax(logits, 1)
    q = torch.softmax(logits[of] + apart * torch.randn(n, vocab, generator=g), 1)
    drafts = torch.multinomial(q, 1, generator=g).view(-1).int() if n else torch.zeros(0, dtype=torch.int32)
    number = lambda m: torch.randint(0, 1 << 24, (m,), generator=g).float() / (1 << 24)
    return probs, starts, drafts, number(n), number(requests), q


@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("requests,most,vocab", [(1, 1, 2), (1, 4, 1), (3, 0, 50), (1, 5, 257), (9, 3, 1000), (17, 7, 4099), (40, 8, 131), (2, 4, 128259), (300, 2, 67), (5, 3, 1024), (5, 3, 1025), (4, 3, 8192), (4, 3, 8193), (6, 4, 20000), (2, 2, 300001)])
def test_token_for_token(requests, most, vocab, lookup):
    for seed in range(3):
        probs, starts, drafts, accept, final, q = case(requests, most, vocab, seed, ragged=seed > 0)
        agree(probs, starts, drafts, accept, final, most + (seed == 2), None if lookup else q)


def test_all_kinds_of_endings():
    probs, starts, drafts, accept, final, q = case(60, 6, 500, 5)
    taken = agree(probs, starts, drafts, accept, final, 6, q)
    counts = [starts[b + 1] - starts[b] - 1 for b in range(60)]
    assert any(t == c and c > 0 for t, c in zip(taken, counts)) and any(t == 0 and c > 0 for t, c in zip(taken, counts)) and any(0 < t < c for t, c in zip(taken, counts))
    # the same distribution on both sides: every draft stands
    of = [starts[b] + i for b in range(60) for i in range(counts[b])]
    assert agree(probs, starts, drafts, accept, final, 6, probs[of]) == counts
    # numbers at the ends of their range
    for u in (0.0, 1 - 2.0 ** -24):
        agree(probs, starts, drafts, torch.full_like(accept, u), torch.full_like(final, u), 6, q)
        agree(probs, starts, drafts, torch.full_like(accept, u), torch.full_like(final, u), 6)


@pytest.mark.parametrize("v", [300, 10000])
def test_greedy_rows(v):
    """One-hot distributions: a draft stands where it is the target's token, and that token comes out."""
    n = 5
    want = torch.randint(0, v, (n + 1,), generator=torch.Generator().manual_seed(1))
    probs = torch.nn.functional.one_hot(want, v).float()
    drafts = want[:n].int().clone()
    for wrong in range(n + 1):
        d = drafts.clone()
        if wrong < n:
            d[wrong] = (d[wrong] + 1) % v
        for q in (None, torch.nn.functional.one_hot(d.long(), v).float()):
            assert agree(probs, [0, n + 1], d, torch.full((n,), 0.9), torch.tensor([0.4]), n, q) == [wrong]
            from llama_cu_amd import sampling
            got = sampling.verify_drafts(probs.cuda(), torch.tensor([0, n + 1], dtype=torch.int32).cuda(), d.cuda(), torch.full((n,), 0.9).cuda(), torch.tensor([0.4]).cuda(), n,
                                         None if q is None else q.cuda())
            assert got[1][0].tolist() == want[:wrong + 1].tolist() + [-1] * (n - wrong)


@pytest.mark.parametrize("v", [100, 9000])
def test_rows_that_leave_nothing(v):
    probs, starts, drafts, accept, final, q = case(6, 3, v, 9, ragged=False)
    probs[starts[1]] = 0.0                              # a row without any probability
    probs[starts[2]] = q[3 * 2] * 0.5                   # less than the draft's everywhere: nothing is left but the target's own
    accept[3 * 2] = 0.99
    probs[starts[3], ::3] = float("nan")
    probs[starts[3], 1::3] = -1.0
    q[3 * 4, ::2] = float("inf")
    q[3 * 4 + 1] = float("nan")
    drafts[3 * 5] = v + 3
    taken = agree(probs, starts, drafts, accept, final, 3, q)
    assert taken[1] == 0 and taken[2] == 0 and taken[5] == 0
    drafts[3 * 5] = -1
    agree(probs, starts, drafts, accept, final, 3)
    lone = torch.zeros(2, v)
    lone[0, 7] = 1.0                                    # the certain draft holds all there is and is refused all the same: its own row again
    agree(lone, [0, 2], torch.tensor([7], dtype=torch.int32), torch.tensor([1.0]), torch.tensor([0.5]), 1)


@pytest.mark.parametrize("v", [64, 9000])
def test_starts_that_make_no_sense(v):
    from llama_cu_amd import sampling
    probs, starts, drafts, accept, final, q = case(4, 3, v, 2, ragged=False)
    for bad in ([0, 4, 3, 12, 16], [0, -5, 8, 12, 16], [0, 4, 8, 12, 400], [2 ** 31 - 1, 4, 8, -2 ** 31, 16], [0, 16, 16, 16, 16], [1, 5, 9, 13, 17]):
        a, t = sampling.verify_drafts(probs.cuda(), torch.tensor(bad, dtype=torch.int64).int().cuda(), drafts.cuda(), accept.cuda(), final.cuda(), 3, q.cuda())
        good = sampling.verify_drafts(probs.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), drafts.cuda(), accept.cuda(), final.cuda(), 3, q.cuda())
        for b in range(4):
            count, row = bad[b + 1] - bad[b] - 1, bad[b]
            if row < 0 or count < 0 or count > 3 or row + count >= 16 or row - b < 0 or row - b + count > 12:
                assert int(a[b]) == 0 and t[b].tolist() == [-1] * 4
            elif bad[b:b + 2] == starts[b:b + 2]:
                assert int(a[b]) == int(good[0][b]) and torch.equal(t[b], good[1][b])


def test_tokens_are_distributed_as_the_targets():
    """First tokens of 40,000 requests with the same target and draft distributions: their frequencies are the target's, chi squared over 12 tokens
    within its 1 - 1e-9 quantile (11 degrees of freedom: 66)."""
    from llama_cu_amd import sampling
    n, v = 40000, 12
    g = torch.Generator().manual_seed(3)
    p, q = torch.softmax(torch.randn(v, generator=g), 0), torch.softmax(torch.randn(v, generator=g), 0)
    probs = p.repeat(2 * n, 1)
    drafts = torch.multinomial(q, n, replacement=True, generator=g).int()
    number = lambda m: torch.randint(0, 1 << 24, (m,), generator=g).float() / (1 << 24)
    a, t = sampling.verify_drafts(probs.cuda(), (torch.arange(n + 1) * 2).int().cuda(), drafts.cuda(), number(n).cuda(), number(n).cuda(), 1, q.repeat(n, 1).cuda())
    for tokens in (t[:, 0], t[a == 1, 1]):
        seen = torch.bincount(tokens.cpu().long(), minlength=v).double()
        want = p.double() * tokens.numel()
        assert float(((seen - want) ** 2 / want).sum()) < 66


def test_strides_and_capture():
    from llama_cu_amd import sampling
    probs, starts, drafts, accept, final, q = case(7, 4, 900, 4)
    wide_p, wide_q = torch.full((probs.shape[0], 1003), 9.0), torch.full((q.shape[0], 1001), 9.0)
    wide_p[:, 3:903], wide_q[:, 1:901] = probs, q
    put = lambda: (wide_p.cuda()[:, 3:903], torch.tensor(starts, dtype=torch.int32).cuda(), drafts.cuda(), accept.cuda(), final.cuda())
    args = put()
    qs = wide_q.cuda()[:, 1:901]
    want = sampling.verify_drafts(probs.cuda(), *args[1:], 4, q.cuda())
    got = sampling.verify_drafts(*args, 4, qs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sampling.verify_drafts(*args, 4, qs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sampling.verify_drafts(*args, 4, qs)
    for seed in range(4):
        fresh = case(7, 4, 900, 4)[4].roll(seed)
        args[4].copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want = sampling.verify_drafts(*args, 4, qs)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("v", [700, 9000, 40000])
def test_two_graphs_and_two_streams(v):
    """Distributions and their verification: two graphs replayed in turn and at once on two streams, with calls of the program's own between them."""
    from llama_cu_amd.sampling import token_probs, verify_drafts
    requests, most = 30, 4
    rows, n = requests * (most + 1), requests * most            # (more than 64 rows: options go through pinned memory outside a graph)
    starts = torch.arange(0, rows + 1, most + 1, dtype=torch.int32).cuda()
    opts = ([0.6 + 0.01 * (r % 70) for r in range(rows)], [0.8 + 0.001 * (r % 200) for r in range(rows)], [v if r % 3 else 1 + r for r in range(rows)])
    there = [torch.tensor(opts[0]).cuda(), torch.tensor(opts[1]).cuda(), torch.tensor(opts[2], dtype=torch.int32).cuda()]

    def fill(state, seed):
        g = torch.Generator().manual_seed(seed)
        state["logits"].copy_(torch.randn(rows, v, generator=g) * 2.5)
        state["drafts"].copy_(torch.randint(0, v, (n,), generator=g, dtype=torch.int32))
        # some drafts that the target likes
        best = state["logits"].argmax(1).view(requests, most + 1)[:, :most].reshape(-1).int()
        state["drafts"][::2] = best[::2]
        for name in ("accept", "final"):
            state[name].copy_(torch.randint(0, 1 << 24, state[name].shape, generator=g).float() / (1 << 24))

    def make():
        return dict(logits=torch.empty(rows, v, device="cuda"), drafts=torch.empty(n, dtype=torch.int32, device="cuda"), accept=torch.empty(n, device="cuda"), final=torch.empty(requests, device="cuda"))

    def work(s, options):
        probs = token_probs(s["logits"], *options)
        return (probs,) + verify_drafts(probs, starts, s["drafts"], s["accept"], s["final"], most)

    states, graphs, outs = [make(), make()], [], []
    for i, s in enumerate(states):
        fill(s, i)
        work(s, there)
    torch.cuda.synchronize()
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(s, there))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for i, s in enumerate(states):
            fill(s, 10 * turn + i)
        torch.cuda.synchronize()
        if turn % 2:
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        else:
            graphs[1].replay()
            graphs[0].replay()
        eager = []
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                eager.append([work(s, opts) for _ in range(3)])
        torch.cuda.synchronize()
        for s, out, calls in zip(states, outs, eager):
            want = work(s, there)
            for got in [out] + calls:
                assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        assert int(outs[0][1].sum()) > 0
