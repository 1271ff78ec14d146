"""4-bit weights in a model, and drafts from a 4-bit copy verified against the full one."""
from __future__ import annotations

import pytest
import torch

import common
from divasun_common import assert_close
from test_gpu_divasun import rnd

pytestmark = pytest.mark.gpu

DATA = dict(architectures=["LlamaForCausalLM"], num_hidden_layers=2, hidden_size=96, num_attention_heads=6, num_key_value_heads=2, head_dim=16, intermediate_size=168, vocab_size=320,
            max_position_embeddings=512, rope_theta=10000.0, rms_norm_eps=1e-5)


def model(std=0.2):
    from llama_cu_amd.config import LlamaConfig
    from llama_cu_amd.models.llama import llama_spec
    from llama_cu_amd.parts import DecoderModel
    from llama_cu_amd.weights import random_tensors
    spec = llama_spec(LlamaConfig.from_dict(DATA))
    return spec, random_tensors(DecoderModel(spec).tensors(), 5, dtype=torch.float32, std=std, device="cpu")


def rounded(tensors):
    """The matrices of attention and feed-forward as the 4-bit numbers they become."""
    from llama_cu_amd.kernels import ops
    hit = lambda name: any(part in name for part in ("self_attn.", "mlp.")) and name.endswith("proj.weight")
    assert sum(hit(n) for n in tensors) == 14
    return {n: ops.mx4_values(ops.mx4_quantize(t.cuda()), torch.float32).cpu() if hit(n) else t for n, t in tensors.items()}


def runner(spec, tensors, dtype, weights, **kw):
    from llama_cu_amd.engine.runner import ModelRunner
    dt = torch.float32 if dtype == "float32" else torch.bfloat16
    mine = {n: (t.to(dt) if t.dim() == 2 else t).cuda() for n, t in tensors.items()}
    return ModelRunner(spec, mine, dtype, max_tokens=2048, max_seqs=8, weights=weights, **kw)


def test_a_model_computes_with_the_rounded_matrices():
    """The 32-bit engine with 4-bit matrices generates what the same engine generates with the numbers that they stand for: the rows are multiplied in
    full, so only the sums' order differs."""
    from llama_cu_amd.engine.engine import Engine
    spec, tensors = model()
    prompts = list(common.random_requests(320, [1, 7, 40, 150], seed=3).values())
    tokens = []
    for source, weights in ((tensors, "mx4"), (rounded(tensors), "file")):
        r = runner(spec, source, "float32", weights)
        engine = Engine(r)
        tokens.append(engine.generate(prompts, max_steps=12, ignore_eos=True))
        r.cache.check()
    assert tokens[0] == tokens[1]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_engine_option(dtype):
    """Through the engine's own entry point: prompts in portions beside single tokens, with and without captured graphs, give the same tokens."""
    from llama_cu_amd.engine.engine import Engine
    from llama_cu_amd.config import LlamaConfig
    cfg = LlamaConfig.from_dict(DATA)
    prompts = list(common.random_requests(320, [3, 30, 100], seed=4).values())
    out = []
    for graphs in (True, False):
        engine = Engine.from_config(cfg, 7, dtype=dtype, std=0.2, page_size=16, max_tokens=1024, max_seqs=4, prefill_chunk=48, weights="mx4", use_graphs=graphs)
        out.append(engine.generate(prompts, max_steps=10, ignore_eos=True))
        engine.runner.cache.check()
    assert out[0] == out[1] and all(len(o) == 10 for o in out[0])


def test_linear_takes_it():
    from llama_cu_amd.kernels import ops
    from llama_cu_amd.parts.base import BuildContext
    from llama_cu_amd.parts.linear import Weight, finish, linear, project
    w = rnd(80, 160, seed=1).bfloat16().cuda()
    build = BuildContext(torch.bfloat16, torch.device("cuda"), 64, 16, weights="mx4")
    four, full = Weight(w, build, four_bits=True), Weight(w, build)
    assert four.four_bits and isinstance(four.plain, ops.PackedMx4) and not full.four_bits and tuple(four.shape) == (80, 160)
    exact = ops.mx4_values(ops.mx4_quantize(w), torch.float32).double().cpu()
    for m in (1, 8, 40, 300):
        x = rnd(m, 160, seed=m).bfloat16().cuda()
        want = x.double().cpu() @ exact.T
        assert_close(linear(x, four, out_dtype=torch.float32), want, 1e-5)
        assert_close(linear(x.float(), four), want, 1e-5)
        assert_close(project(x, four, torch.bfloat16), want, 2.0 ** -8 + 1e-5)
        assert_close(finish(x, four, torch.bfloat16, planes_ok=True), want, 2.0 ** -8 + 1e-5)
        total = torch.ones(m, 80, device="cuda")
        assert_close(linear(x, four, out=total, accumulate=True), want + 1, 1e-5)


def test_drafts_from_a_4_bit_copy():
    """One round of speculation by hand, and its pieces against 64 bits: hidden states -> the 4-bit output matrix's logits -> their distributions -> drafts
    drawn from them; the full matrix's logits -> Sampler.verify.  Then in the long run: the tokens that come out are distributed as the full model's
    (chi squared of 3,000 first tokens over 16 of them within its 1 - 1e-9 quantile, 15 degrees of freedom: 75)."""
    from llama_cu_amd.kernels import ops
    from llama_cu_amd.parts.linear import linear
    from llama_cu_amd.sampling import Sampler, SamplingParams, sample_rows, verify_drafts
    from llama_cu_amd.sampling.sampler import FINAL, JUDGE, uniform
    from test_gpu_verify import plain
    vocab, width, requests, each = 500, 256, 24, 3
    w = (rnd(vocab, width, seed=1) * 0.15).bfloat16().cuda()
    four = ops.pack_mx4(ops.mx4_quantize(w))
    hidden = rnd(requests * (each + 1), width, seed=2).bfloat16().cuda()
    params = [SamplingParams(temperature=0.6 + 0.05 * i, top_p=0.9 if i % 3 else 1.0, top_k=50 if i % 2 else 10 ** 6, seed=9) if i % 5 else SamplingParams() for i in range(requests)]
    sampler = Sampler()
    of = [i * (each + 1) + j for i in range(requests) for j in range(each)]
    drafting = sampler.probs(ops.gemm_mx4(hidden[of], four, out_dtype=torch.float32), [params[i] for i in range(requests) for _ in range(each)])
    drafts = [int(torch.multinomial(drafting[i * each + j].cpu(), 1, generator=torch.Generator().manual_seed(i * 7 + j))) for i in range(requests) for j in range(each)]
    drafts = [drafts[i * each:(i + 1) * each] for i in range(requests)]
    logits = linear(hidden, w, out_dtype=torch.float32)
    keys = [(i, 100 + i) for i in range(requests)]
    got = sampler.verify(logits, drafts, params, keys, drafting)
    probs = sampler.probs(logits, [p for p in params for _ in range(each + 1)])
    starts = [i * (each + 1) for i in range(requests + 1)]
    judge = torch.tensor([uniform(p.seed, k[0], k[1] + j, JUDGE) for p, k in zip(params, keys) for j in range(each)])
    final = torch.tensor([uniform(p.seed, k[0], k[1], FINAL) for p, k in zip(params, keys)])
    accepted, tokens, _ = plain(probs.cpu(), starts, torch.tensor(drafts).view(-1), judge, final, each, drafting.cpu())
    assert got == [t[:a + 1] for a, t in zip(accepted, tokens)]
    assert sum(accepted) > requests // 2 and any(a < each for a in accepted)                 # (some of both)
    greedy = [i for i in range(requests) if params[i].is_argmax]
    for i in greedy:
        best = logits[i * (each + 1):(i + 1) * (each + 1)].argmax(1).tolist()
        assert got[i] == best[:len(got[i])]
    # the long run: the same row again and again, drafts drawn on the device, numbers of their own
    n = 3000
    row, p = logits[1:2], [SamplingParams(temperature=0.7, top_k=16)]
    target, draft = sampler.probs(row, p), sampler.probs(ops.gemm_mx4(hidden[1:2], four, out_dtype=torch.float32), p)
    u = torch.Generator().manual_seed(5)
    number = lambda m: torch.randint(0, 1 << 24, (m,), generator=u).float() / (1 << 24)
    drawn = sample_rows(ops.gemm_mx4(hidden[1:2], four, out_dtype=torch.float32).expand(n, vocab).contiguous(), [0.7] * n, [1.0] * n, [16] * n, number(n).tolist())
    a, t = verify_drafts(target.expand(2 * n, vocab).contiguous(), (torch.arange(n + 1) * 2).int().cuda(), drawn, number(n).cuda(), number(n).cuda(), 1, draft.expand(n, vocab).contiguous())
    want = target[0].double().cpu()
    seen = torch.bincount(t[:, 0].cpu().long(), minlength=vocab).double()
    kept = want > 0
    assert int(kept.sum()) == 16 and seen[~kept].sum() == 0
    assert float(((seen - n * want)[kept] ** 2 / (n * want)[kept]).sum()) < 75
    assert 0 < int(a.sum()) < n


def test_verify_refusals():
    from llama_cu_amd.kernels.ops import KernelError
    from llama_cu_amd.sampling import Sampler, SamplingParams
    s, p = Sampler(), SamplingParams(temperature=1.0)
    logits = rnd(3, 50).cuda()
    assert s.verify(logits[:0], [], [], []) == []
    for args in (([[1, 2]], [p, p], [(0, 0)]), ([[1]], [p], [(0, 0)]), ([[1, 2], []], [p] * 2, [(0, 0)] * 2)):
        with pytest.raises(KernelError, match="verify"):
            s.verify(logits, *args)
    with pytest.raises(KernelError, match="probs"):
        s.probs(logits, [p])
    assert [len(t) for t in s.verify(logits, [[], [], []], [p] * 3, [(i, 0) for i in range(3)])] == [1, 1, 1]


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("family", ["divasun", "lozezen", "ralepel", "mufotar", "gefudra", "lapunex"])
def test_other_designs_compute_with_the_rounded_matrices(family, name, monkeypatch):
    """As the Llama model above, by logits: a prompt as a whole, and then two requests' tokens one by one."""
    import importlib
    from llama_cu_amd.engine.runner import ModelRunner
    from llama_cu_amd.kernels import ops
    from llama_cu_amd.parts import ffn, linear
    C, T = importlib.import_module(f"{family}_common"), importlib.import_module(f"test_gpu_{family}")
    cfg = getattr(C, f"CFG_{name}")
    args = (cfg, getattr(C, f"RANKS_{name}"), 5) if family == "divasun" else (cfg, 5)
    folder = C.make_folder(cfg, C.random_weights(*args))
    a, b = C.tokens_of(cfg["vocab"], 60, 1), C.tokens_of(cfg["vocab"], 9, 2)

    def logits(**kw):
        r = ModelRunner.from_folder(folder, dtype="float32", page_size=16, max_tokens=1024, max_seqs=4, max_batch_tokens=1024, **kw)
        held = sum(isinstance(v, ops.PackedMx4) for v in seen)
        out = [r.step([0], [a[:50]], [list(range(50))]).clone(), r.step([1, 0], [b[:8], a[50:51]], [list(range(8)), [0]]).clone()]
        for i in range(51, 54):
            out.append(r.step([0], [a[i:i + 1]], [[0]]).clone())
        r.end(0); r.end(1)
        r.cache.check()
        return torch.cat(out).double().cpu(), held

    seen, plain = [], linear.Weight.__init__

    def watched(self, tensor, build=None, packed_from=None, halves=False, four_bits=False):
        if watched.round and (four_bits or halves):                  # (gate and up, which the feed-forward alone says are halves)
            tensor = ops.mx4_values(ops.mx4_quantize(tensor), torch.float32).to(tensor.dtype)
            packed_from = None
        plain(self, tensor, build, packed_from, halves, four_bits)
        seen.append(self.plain)
    monkeypatch.setattr(linear.Weight, "__init__", watched)
    watched.round = False
    got, held = logits(weights="mx4")
    watched.round = True
    want, _ = logits()
    assert_close(got, want, T.REL["float32"], f"{family} {name}: {held} matrices in 4 bits")
