"""A round of speculation with the engine's own steps: the copy with 4-bit matrices drafts token by token, the model with its file's judges all drafts of every request in one step."""
from __future__ import annotations

import pytest
import torch

import common
from test_gpu_mx4_model import model, runner
from test_gpu_verify import plain

pytestmark = pytest.mark.gpu

PROMPTS, EACH = [3, 40, 17, 150], 4


def drafted(r, prompts, params, sampler):
    """``EACH`` tokens for every request, drawn by the engine's own sampler, and the distributions they were drawn from (request by request)."""
    ids = list(range(len(prompts)))
    drafts, probs = [[] for _ in ids], [[] for _ in ids]
    logits = r.step(ids, prompts)
    for j in range(EACH):
        dist = sampler.probs(logits, params)
        for i, t in enumerate(sampler.sample(logits, params, [(i, len(prompts[i]) + j) for i in ids])):
            drafts[i].append(t)
            probs[i].append(dist[i])
        if j + 1 < EACH:
            logits = r.step(ids, [[d[-1]] for d in drafts])
    for i in ids:
        r.end(i)
    return drafts, torch.stack([p for of in probs for p in of])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_round(dtype):
    from llama_cu_amd.sampling import Sampler, SamplingParams
    from llama_cu_amd.sampling.sampler import FINAL, JUDGE, uniform
    spec, tensors = model()
    prompts = list(common.random_requests(320, PROMPTS, seed=11).values())
    params = [SamplingParams(), SamplingParams(temperature=0.8, top_p=0.9, seed=3), SamplingParams(temperature=1.2, top_k=40, seed=4), SamplingParams()]
    sampler, ids = Sampler(), list(range(len(prompts)))
    copy, full = runner(spec, tensors, dtype, "mx4"), runner(spec, tensors, dtype, "file")
    drafts, of_drafts = drafted(copy, prompts, params, sampler)
    # one step: the prompt and all drafts in, the rows behind the prompt's last token and behind every draft out
    logits = full.step(ids, [p + d for p, d in zip(prompts, drafts)], [[len(p) - 1 + j for j in range(EACH + 1)] for p in prompts]).clone()
    assert logits.shape == (len(ids) * (EACH + 1), 320)
    keys = [(i, len(p)) for i, p in enumerate(prompts)]
    got = sampler.verify(logits, drafts, params, keys, of_drafts)
    # the pieces by themselves, in 64 bits
    probs = sampler.probs(logits, [p for p in params for _ in range(EACH + 1)]).cpu()
    judge = torch.tensor([uniform(p.seed, k[0], k[1] + j, JUDGE) for p, k in zip(params, keys) for j in range(EACH)])
    final = torch.tensor([uniform(p.seed, k[0], k[1], FINAL) for p, k in zip(params, keys)])
    accepted, tokens, near = plain(probs, [i * (EACH + 1) for i in range(len(ids) + 1)], torch.tensor(drafts).view(-1), judge, final, EACH, of_drafts.cpu())
    assert min(near) > 1e-9 and got == [t[:a + 1] for a, t in zip(accepted, tokens)]
    # greedy requests: what the model generates by itself, as far as it goes
    for i in (0, 3):
        rows = logits[i * (EACH + 1):(i + 1) * (EACH + 1)]
        best = rows.argmax(1).tolist()
        stand = next((j for j in range(EACH) if drafts[i][j] != best[j]), EACH)
        assert got[i] == best[:stand + 1]
    for r in (copy, full):
        for i in ids:
            r.end(i)
        r.cache.check()


def test_greedy_speculation_generates_what_greedy_decoding_does():
    """Round after round, in 32 bits: the tokens are those that the model generates one at a time.  (The logits of a step of several rows and of a single row differ in their sums' order, by
    1e-5 of the largest; the test's own tokens are asked to lie further from a tie than that.)"""
    from llama_cu_amd.sampling import Sampler, SamplingParams
    spec, tensors = model()
    sampler, params, wanted = Sampler(), [SamplingParams()] * len(PROMPTS), 12
    prompts = list(common.random_requests(320, PROMPTS, seed=12).values())
    ids = list(range(len(prompts)))
    full, copy = runner(spec, tensors, "float32", "file"), runner(spec, tensors, "float32", "mx4")
    plainly, logits = [[] for _ in ids], full.step(ids, prompts)
    for _ in range(wanted):
        top = logits.topk(2, 1).values
        assert float(((top[:, 0] - top[:, 1]) / logits.abs().amax(1)).min()) > 2e-5
        for i, t in enumerate(logits.argmax(1).tolist()):
            plainly[i].append(t)
        logits = full.step(ids, [[p[-1]] for p in plainly])
    for i in ids:
        full.end(i)
    texts, rounds = [list(p) for p in prompts], 0
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < wanted:
        drafts, of_drafts = drafted(copy, texts, params, sampler)
        logits = full.step(ids, [t + d for t, d in zip(texts, drafts)], [[len(t) - 1 + j for j in range(EACH + 1)] for t in texts]).clone()
        for i in ids:
            full.end(i)
        for t, new in zip(texts, sampler.verify(logits, drafts, params, [(i, len(t)) for i, t in enumerate(texts)], of_drafts)):
            t += new
        rounds += 1
    assert rounds <= wanted
    for t, p, want in zip(texts, prompts, plainly):
        assert t[len(p):len(p) + wanted] == want
