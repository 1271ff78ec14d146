"""What token_probs and verify_drafts refuse, before anything is launched."""
from __future__ import annotations

import pytest
import torch

from llama_cu_amd.kernels.ops import KernelError
from llama_cu_amd.sampling import token_probs, verify_drafts


def refused(what, f, *args, **kw):
    with pytest.raises(KernelError, match=what):
        f(*args, **kw)


def test_token_probs():
    x = torch.zeros(2, 8)
    fine = ([1.0, 1.0], [1.0, 1.0], [8, 8])
    refused("on the GPU", token_probs, x, *fine)
    refused("must be float32", token_probs, x.double(), *fine)
    refused("must be float32", token_probs, x[0], *fine)
    refused("contiguous rows", token_probs, torch.zeros(2, 16)[:, ::2], *fine)
    refused("vocabulary of 0", token_probs, x[:, :0], *fine)
    refused("vocabulary of", token_probs, torch.zeros(1).expand(1, (1 << 19) + 1).contiguous(), [1.0], [1.0], [1])
    for t in ([1.0], [1.0, -1.0], [1.0, float("nan")], [1.0, float("inf")]):
        refused("temperature must be 2 numbers >= 0", token_probs, x, t, fine[1], fine[2])
    for p in ([1.0], [1.0, 0.0], [1.0, float("nan")]):
        refused("top_p must be 2 numbers > 0", token_probs, x, fine[0], p, fine[2])
    for k in ([1], [0, 8], [8, -1], [8, float("nan")], [float("nan"), 8]):
        refused("top_k must be 2 numbers >= 1", token_probs, x, fine[0], fine[1], k)
    for out in (torch.zeros(2, 9), torch.zeros(2, 8).double(), torch.zeros(2, 16)[:, :8], torch.zeros(1, 8)):
        refused("out: must be contiguous float32", token_probs, x, *fine, out=out)


def test_verify_drafts():
    def call(probs=torch.zeros(5, 8), starts=torch.tensor([0, 3, 5], dtype=torch.int32), drafts=torch.zeros(3, dtype=torch.int32), accept=torch.zeros(3),
             final=torch.zeros(2), most=2, draft_probs=torch.zeros(3, 8)):
        return verify_drafts(probs, starts, drafts, accept, final, most, draft_probs)
    refused("on the GPU", call)
    refused("on the GPU", call, draft_probs=None)
    for bad in (torch.zeros(5, 8).double(), torch.zeros(40), torch.zeros(5, 16)[:, ::2], torch.zeros(1, 8).expand(5, 8)):
        refused("probs must be float32", call, probs=bad)
    for bad in (torch.zeros(3), torch.zeros(0, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2]):
        refused("starts must be", call, starts=bad)
    for bad in (torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int64), torch.zeros(6, dtype=torch.int32)[::2]):
        refused("drafts must be contiguous int32", call, drafts=bad)
    for bad in (torch.zeros(2), torch.zeros(3).double()):
        refused("accept must be", call, accept=bad)
    for bad in (torch.zeros(3), torch.zeros(2).double()):
        refused("final must be", call, final=bad)
    for bad in (torch.zeros(3, 9), torch.zeros(2, 8), torch.zeros(3, 8).double()):
        refused("draft_probs must be float32", call, draft_probs=bad)
    for most in (-1, 1025):
        refused("max_drafts", call, most=most)
    refused("drafts must be", call, probs=torch.zeros(1, 8))
    refused("vocabulary of 0", call, probs=torch.zeros(5, 0), draft_probs=torch.zeros(3, 0))


def test_a_distribution_does_not_go_over_its_logits():
    logits = torch.zeros(4, 40)
    for out in (logits, logits.view(-1)[20:100].view(2, 40)):
        with pytest.raises(KernelError, match="over an operand"):
            token_probs(logits[:out.shape[0]], [1.0] * len(out), [0.9] * len(out), [5] * len(out), out=out)
