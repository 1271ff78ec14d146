"""Products with weights held in 4 bits, and drafts verified against a target: cases, plain forms and 64-bit results.

The two belong to one way of serving.  A copy of a model's matrices in microscaled 4-bit numbers (a block of 32 along k shares a
power of two) drafts tokens out of a quarter of the bytes; the full model then judges all drafts of a request in one step, and the
verification keeps the full model's distribution exactly.  The operators:

``quantise``  rows -> 4-bit codes and scales, read back as the values they stand for (``ops.mx4_quantize``, ``ops.mx4_values``)
``product``   rows in the compute type times a 4-bit weight, SwiGLU in the epilogue if asked for (``ops.gemm_mx4``)
``product4``  rows quantised on the way, 4 bits times 4 bits (``ops.mx4_quantize``, ``ops.gemm_mx4``)
``probs``     the distribution that a row's temperature, top_p and top_k leave of its logits (``sampling.token_probs``)
``verify``    which of a request's drafted tokens stand, and the token after them (``sampling.verify_drafts``)

A case holds plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass, ``exact`` computes the same in 64 bits.
"""
import math

import torch

own = False                                     # whether ``run`` calls the framework's operators or computes their plain forms

BLOCK = 32                                      # numbers along k that share a scale
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # what the three low bits of a code stand for; the fourth is the sign
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # a decoding step's row of the 8B shape on its way into a 4-bit product: latency
        dict(name="quantise one token's row", op="quantise", rows=1, k=4096, type="bfloat16"),
        # a layer's gate and up matrix when a model is loaded
        dict(name="quantise a gate and up matrix", op="quantise", rows=28672, k=4096, type="bfloat16"),
        # a single request drafts: the q, k, v product
        dict(name="one token, q k v", op="product", rows=1, n=6144, k=4096, type="bfloat16", out="bfloat16", swiglu=False),
        # eight requests draft: gate and up with the activation
        dict(name="eight tokens, gate and up", op="product", rows=8, n=28672, k=4096, type="bfloat16", out="bfloat16", swiglu=True),
        # an odd batch of a model that computes in 32 bits, its features no whole tiles
        dict(name="37 tokens in 32 bits", op="product", rows=37, n=4104, k=11008, type="float32", out="float32", swiglu=False),
        # a prompt's portion
        dict(name="a prompt, gate and up", op="product", rows=2048, n=28672, k=4096, type="bfloat16", out="bfloat16", swiglu=True),
        # a batch of 64, rows in 4 bits too: the down projection
        dict(name="64 tokens, 4 bits by 4", op="product4", rows=64, n=4096, k=14336, type="bfloat16", out="bfloat16"),
        # a long prompt through a 70B down projection
        dict(name="a long prompt, 4 bits by 4", op="product4", rows=4096, n=8192, k=28672, type="bfloat16", out="bfloat16"),
        # the target's rows of one request with four drafts
        dict(name="one request's distributions", op="probs", rows=5, vocab=128256, cut="mixed"),
        # a served batch: 64 requests with four drafts each, every one with its own options
        dict(name="a batch's distributions", op="probs", rows=320, vocab=128256, cut="mixed"),
        # one request, four drafts
        dict(name="one request's drafts", op="verify", requests=1, drafts=4, vocab=128256, ragged=False, lookup=False),
        # a batch whose requests bring zero to seven drafts, odd vocabulary
        dict(name="a batch's drafts", op="verify", requests=61, drafts=7, vocab=128259, ragged=True, lookup=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _whole(rng, v, steps):
    """``v`` as it is, or rounded to one of ``steps``."""
    s = rng.choice(steps)
    return max(s, v // s * s)


def draw(rng):
    """One more case out of the ranges that the listed ones stand for."""
    op = rng.choice(["quantise", "product", "product", "product4", "probs", "verify"])
    if op == "quantise":
        return dict(op=op, rows=_log(rng, 1, 28672), k=_whole(rng, _log(rng, 1, 8192), (1, 8, 32, 128)), type=rng.choice(sorted(TYPES)))
    if op in ("product", "product4"):
        kind = rng.choice(sorted(TYPES))
        # most layers' features come in whole tiles, some do not; 4-bit blocks may end behind k
        n, k = _whole(rng, _log(rng, 16, 28672), (1, 16, 16, 64)), _whole(rng, _log(rng, 32, 14336), (1, 32, 128, 128))
        rows = _log(rng, 1, max(1, min(2048, (1 << 37) // (n * k))))
        if op == "product4":
            return dict(op=op, rows=rows, n=n, k=k, type=kind, out=rng.choice(sorted(TYPES)))
        swiglu = rng.random() < 0.3
        if swiglu:
            n += n % 2
        return dict(op=op, rows=rows, n=n, k=k, type=kind, out=kind if swiglu else rng.choice(sorted(TYPES)), swiglu=swiglu)
    vocab = _whole(rng, _log(rng, 257, 131072), (1, 1, 32))
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, 320), vocab=vocab, cut=rng.choice(["none", "top_p", "top_k", "mixed", "mixed"]))
    drafts = rng.randint(1, 8)
    return dict(op=op, requests=_log(rng, 1, 64), drafts=drafts, vocab=vocab, ragged=rng.random() < 0.6, lookup=rng.random() < 0.3)


# ------------------------------------------------------------------ 4-bit numbers


def _blocks(x):
    """Rows as blocks of 32 in 64 bits, the last one filled up with zeros."""
    rows, k = x.shape
    full = torch.zeros(rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :k] = x
    return full.view(rows, -1, BLOCK)


def _quantise(x):
    """``(magnitude codes with the sign in bit 3, exponents)``: a block's scale is the power of two two below its largest
    number's, a number goes to the nearest of the grid (ties to the even code) and beyond 6 to 6."""
    b = _blocks(x)
    most = b.abs().amax(2)
    exponent = torch.where(most > 0, torch.frexp(most)[1] - 3, torch.full_like(most, -127).int()).clamp_(min=-127)
    y = torch.ldexp(b, -exponent.unsqueeze(2))
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    near = (torch.round(y.abs() / step) * step).clamp_(max=6.0)
    code = torch.searchsorted(torch.tensor(GRID, dtype=torch.float64, device=x.device), near)
    return (code + 8 * torch.signbit(b)).to(torch.uint8), exponent


def _pack(code):
    """Two codes a byte, the first in the low half."""
    rows = code.shape[0]
    flat = code.reshape(rows, -1)
    return (flat[:, 0::2] | (flat[:, 1::2] << 4)).contiguous()


def _values(codes, scales, k, dtype=torch.float32):
    """What packed codes and biased scales stand for."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=dtype, device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], dim=2).view(codes.shape[0], -1)
    scale = torch.ldexp(torch.ones((), dtype=dtype, device=codes.device), scales.to(torch.int32) - 127)
    return (grid[both.int()].view(codes.shape[0], -1, BLOCK) * scale.unsqueeze(2)).view(codes.shape[0], -1)[:, :k]


def _plain_rows4(x):
    code, exponent = _quantise(x)
    return _values(_pack(code), (exponent + 127).to(torch.uint8), x.shape[1])


# ------------------------------------------------------------------ the inputs


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _uniform(gen, n):
    """Numbers in [0, 1) with 24 random bits, as the sampler draws them."""
    return torch.randint(0, 1 << 24, (n,), device="cuda", generator=gen).float() / float(1 << 24)


def _rows(gen, case):
    """Activations: some channels are larger than the others, as a model's are."""
    x = _normal(gen, case["rows"], case["k"])
    loud = torch.rand(case["k"], device="cuda", generator=gen) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(TYPES[case["type"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "quantise":
        return dict(case=case, x=_rows(gen, case))
    if op in ("product", "product4"):
        x = _rows(gen, case)
        weight = (_normal(gen, case["n"], case["k"]) * 0.02).to(torch.bfloat16)
        parts = [_quantise(p) for p in weight.split(2048)]
        codes = torch.cat([_pack(c) for c, _ in parts])
        scales = torch.cat([(e + 127).to(torch.uint8) for _, e in parts])
        state = dict(case=case, x=x, codes=codes, scales=scales)
        if own:                                 # a program lays a weight out once, when it loads it
            from llama_cu_amd.kernels import ops
            state["weight"] = ops.pack_mx4(ops.Mx4(codes, scales, case["k"]))
        return state
    if op == "probs":
        rows, vocab, cut = case["rows"], case["vocab"], case["cut"]
        pick = torch.Generator().manual_seed(seed)
        number = lambda lo, hi: [lo + (hi - lo) * v for v in torch.rand(rows, generator=pick, dtype=torch.float64).tolist()]
        # a model's logits: the head's product rounds nothing, a few tokens stand out
        logits = _normal(gen, rows, vocab) * 2.5
        top = torch.randint(0, vocab, (rows, 40), device="cuda", generator=gen)
        logits.scatter_add_(1, top, torch.rand(rows, 40, device="cuda", generator=gen) * 12.0)
        temperature, top_p = number(0.5, 1.2), [1.0] * rows
        top_k = [vocab] * rows
        if cut in ("top_p", "mixed"):
            top_p = number(0.7, 0.99)
        if cut in ("top_k", "mixed"):
            top_k = [1 + int(v) for v in number(0, min(200, vocab - 1))]
        if cut == "mixed":                      # some rows without a cut, some greedy, some with one only
            for i in range(rows):
                if i % 5 == 1:
                    top_k[i] = vocab
                elif i % 5 == 2:
                    top_p[i] = 1.0
                elif i % 5 == 3:
                    temperature[i] = 0.0
                elif i % 10 == 4:
                    top_p[i], top_k[i] = 1.0, vocab
        as_floats = lambda v: torch.tensor(v, dtype=torch.float32).tolist()     # what 32 bits hold of them
        return dict(case=case, logits=logits, temperature=as_floats(temperature), top_p=as_floats(top_p), top_k=top_k)
    # verify
    requests, vocab, most = case["requests"], case["vocab"], case["drafts"]
    pick = torch.Generator().manual_seed(seed)
    counts = torch.randint(0, most + 1, (requests,), generator=pick).tolist() if case["ragged"] else [most] * requests
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c + 1)
    drafted = sum(counts)
    rows = starts[-1]
    of_draft = torch.tensor([starts[b] + i for b in range(requests) for i in range(counts[b])], dtype=torch.int64, device="cuda")
    logits = _normal(gen, rows, vocab) * 3.0
    probs = torch.softmax(logits, dim=1)
    # the draft's model agrees with the target's mostly
    drafting = torch.softmax(logits[of_draft] + 0.5 * _normal(gen, drafted, vocab), dim=1)
    drafts = torch.zeros(drafted, dtype=torch.int32, device="cuda")
    if drafted:
        reach = torch.cumsum(drafting.double(), 1)
        u = torch.rand(drafted, 1, device="cuda", generator=gen, dtype=torch.float64)
        drafts = torch.searchsorted(reach, u * reach[:, -1:]).clamp_(max=vocab - 1).view(-1).int()
    return dict(case=case, probs=probs, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), drafts=drafts,
                accept=_uniform(gen, drafted), final=_uniform(gen, requests), draft_probs=None if case["lookup"] else drafting)


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    return (_run_own if own else _run_plain)(state, op)


def _run_own(s, op):
    from llama_cu_amd import sampling
    from llama_cu_amd.kernels import ops
    case = s["case"]
    if op == "quantise":
        q = ops.mx4_quantize(s["x"])
        return ops.mx4_values(q, TYPES[case["type"]]), q.scales
    if op == "product":
        return ops.gemm_mx4(s["x"], s["weight"], out_dtype=TYPES[case["out"]], swiglu=case["swiglu"])
    if op == "product4":
        return ops.gemm_mx4(ops.mx4_quantize(s["x"]), s["weight"], out_dtype=TYPES[case["out"]])
    if op == "probs":
        return sampling.token_probs(s["logits"], s["temperature"], s["top_p"], s["top_k"])
    return sampling.verify_drafts(s["probs"], s["starts"], s["drafts"], s["accept"], s["final"], case["drafts"], draft_probs=s["draft_probs"])


def _run_plain(s, op):
    case = s["case"]
    if op == "quantise":
        code, exponent = _quantise(s["x"])
        scales = (exponent + 127).to(torch.uint8)
        return _values(_pack(code), scales, case["k"]).to(TYPES[case["type"]]), scales
    if op in ("product", "product4"):
        x = _plain_rows4(s["x"]) if op == "product4" else s["x"].float()
        y = x @ _values(s["codes"], s["scales"], case["k"]).t()
        if op == "product" and case["swiglu"]:
            half = case["n"] // 2
            gate, up = y[:, :half], y[:, half:]
            y = gate / (1 + torch.exp(-gate)) * up
        return y.to(TYPES[case["out"]])
    if op == "probs":
        return _plain_probs(s)
    return _plain_verify(s)


def _plain_probs(s):
    logits = s["logits"]
    column = lambda v, t: torch.tensor(v, dtype=t, device=logits.device).unsqueeze(1)
    temperature, top_p, top_k = column(s["temperature"], torch.float32), column(s["top_p"], torch.float64), column(s["top_k"], torch.int64)
    ordered, index = torch.sort(logits, dim=1, descending=True, stable=True)
    # arg-max is a cut after the first entry
    top_k = torch.where(temperature > 0, top_k, torch.ones_like(top_k))
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(temperature > 0, temperature, torch.ones_like(temperature))).double()
    reach = torch.cumsum(weight, 1)
    limit = torch.minimum(top_p * reach[:, -1:], torch.gather(reach, 1, top_k.clamp(max=logits.shape[1]) - 1))
    before = torch.cat([torch.zeros_like(limit), reach[:, :-1]], dim=1)
    share = (torch.minimum(reach, limit) - torch.minimum(before, limit)) / limit
    return torch.zeros_like(logits).scatter_(1, index, share.float())


def _plain_verify(s):
    probs, starts, drafts, drafting = s["probs"], s["starts"].long(), s["drafts"].long(), s["draft_probs"]
    requests, most, dev = starts.numel() - 1, s["case"]["drafts"], probs.device
    counts = starts[1:] - starts[:-1] - 1
    first = starts[:-1] - torch.arange(requests, device=dev)             # a request's first draft
    i = torch.arange(most, device=dev).unsqueeze(0)
    there = i < counts.unsqueeze(1)
    at = torch.where(there, first.unsqueeze(1) + i, torch.zeros_like(i))
    tokens = torch.full((requests, most + 1), -1, dtype=torch.int64, device=dev)
    stands = torch.zeros(requests, most, dtype=torch.bool, device=dev)
    if drafts.numel():
        token = drafts[at]
        p = probs[torch.where(there, starts[:-1].unsqueeze(1) + i, torch.zeros_like(i)), token].double()
        q = torch.ones_like(p) if drafting is None else drafting[at, token].double()
        stands = there & (s["accept"][at].double() * q < p)
        tokens[:, :most] = torch.where(there, token, tokens[:, :most])
    accepted = torch.cumprod(stands.long(), 1).sum(1)
    tokens[:, :most] = torch.where(i < accepted.unsqueeze(1), tokens[:, :most], torch.full_like(tokens[:, :most], -1))
    left = probs[starts[:-1] + accepted].double()
    refused = accepted < counts
    if drafts.numel():
        place = torch.where(refused, first + accepted, torch.zeros_like(first))
        if drafting is None:
            off = torch.zeros_like(left).scatter_(1, drafts[place].unsqueeze(1), 1.0)
        else:
            off = drafting[place].double()
        rest = torch.where(refused.unsqueeze(1), (left - off).clamp_(min=0), left)
        left = torch.where(rest.sum(1, keepdim=True) > 0, rest, left)
    reach = torch.cumsum(left, 1)
    last = torch.searchsorted(reach, s["final"].double().unsqueeze(1) * reach[:, -1:], right=True)
    tokens.scatter_(1, accepted.unsqueeze(1), last.clamp_(max=probs.shape[1] - 1))
    return accepted.int(), tokens.int()


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op = case["op"]
    size = lambda name: 2 if case[name] == "bfloat16" else 4
    if op == "quantise":
        numbers, blocks = case["rows"] * case["k"], case["rows"] * -(-case["k"] // BLOCK)
        return {"bytes": numbers * 2 * size("type") + blocks, "flops": 0}
    if op in ("product", "product4"):
        m, n, k = case["rows"], case["n"], case["k"]
        out = n // 2 if op == "product" and case["swiglu"] else n
        return {"bytes": m * k * size("type") + n * -(-k // BLOCK) * (BLOCK // 2 + 1) + m * out * size("out"), "flops": 2 * m * n * k}
    if op == "probs":
        return {"bytes": case["rows"] * case["vocab"] * 8, "flops": 4 * case["rows"] * case["vocab"]}
    # a draft is judged by one number of each row; the token behind them takes the whole of one row, and of the draft's
    return {"bytes": case["requests"] * case["vocab"] * (4 if case["lookup"] else 8), "flops": 3 * case["requests"] * case["vocab"]}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_values(x):
    """The 4-bit numbers next to ``x``, by comparing with the points midway between two of the grid: ``(values, biased scales)``."""
    rows, k = x.shape
    wide = torch.nn.functional.pad(x.double(), (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    top = wide.abs().max(dim=2).values
    # the power of two not above the largest number: a 64-bit number's own exponent field
    power = ((top.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), power.double()).unsqueeze(2)
    size = wide.abs() / unit
    out = torch.zeros_like(size)
    # a tie goes up where the number above has an even code
    for low, high, up in ((0.0, 0.5, False), (0.5, 1.0, True), (1.0, 1.5, False), (1.5, 2.0, True), (2.0, 3.0, False), (3.0, 4.0, True), (4.0, 6.0, False)):
        middle = (low + high) / 2
        out = torch.where((size >= middle) if up else (size > middle), torch.full_like(out, high), out)
    return (torch.copysign(out, wide) * unit).reshape(rows, -1)[:, :k], (power + 127).to(torch.uint8)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantise":
        return _exact_values(s["x"])
    if op in ("product", "product4"):
        x = _exact_values(s["x"])[0] if op == "product4" else s["x"].double()
        halves = []
        n = case["n"]
        for lo in range(0, n, 4096):
            w = _values(s["codes"][lo:lo + 4096], s["scales"][lo:lo + 4096], case["k"], torch.float64)
            halves.append(torch.matmul(x, w.t()))
        y = torch.cat(halves, dim=1)
        if op == "product" and case["swiglu"]:
            gate, up = y.split(n // 2, dim=1)
            y = gate * torch.sigmoid(gate) * up
        return y
    if op == "probs":
        out = torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device="cuda")
        for r in range(case["rows"]):
            row = s["logits"][r].double()
            order = torch.argsort(row, descending=True, stable=True)
            if s["temperature"][r] == 0:
                out[r] = 0
                out[r, order[0]] = 1
                continue
            w = torch.softmax(row[order] / s["temperature"][r], dim=0)
            kept = w[:s["top_k"][r]]
            limit = min(float(kept.sum()), s["top_p"][r])
            reach = kept.cumsum(0)
            mine = (limit - (reach - kept)).clamp(min=0).minimum(kept)
            out[r] = 0
            out[r, order[:s["top_k"][r]]] = mine / limit
        return out
    accepted, tokens = [], []
    starts = s["starts"].tolist()
    drafts, accept, final = s["drafts"].tolist(), s["accept"].tolist(), s["final"].tolist()
    for b in range(case["requests"]):
        count, row, d = starts[b + 1] - starts[b] - 1, starts[b], starts[b] - b
        taken = 0
        while taken < count:
            t = drafts[d + taken]
            q = 1.0 if case["lookup"] else float(s["draft_probs"][d + taken, t])
            if not accept[d + taken] * q < float(s["probs"][row + taken, t]):
                break
            taken += 1
        p = s["probs"][row + taken].double()
        if taken < count:
            rest = p.clone()
            if case["lookup"]:
                rest[drafts[d + taken]] = 0
            else:
                rest = torch.relu(p - s["draft_probs"][d + taken].double())
            p = rest if float(rest.sum()) > 0 else p
        reach = p.cumsum(0)
        token = int((reach <= final[b] * float(reach[-1])).sum())
        accepted.append(taken)
        tokens.append((drafts[d:d + taken] + [min(token, case["vocab"] - 1)] + [-1] * case["drafts"])[:case["drafts"] + 1])
    return (torch.tensor(accepted, dtype=torch.int32, device="cuda"), torch.tensor(tokens, dtype=torch.int32, device="cuda"))
