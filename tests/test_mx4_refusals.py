"""What the 4-bit numbers' and products' entry points refuse, before anything is launched."""
from __future__ import annotations

import pytest
import torch

from llama_cu_amd.kernels import ops
from llama_cu_amd.kernels.ops import KernelError


def four(m=4, k=64):
    return ops.Mx4(torch.zeros(m, -(-k // 32) * 16, dtype=torch.uint8), torch.zeros(m, -(-k // 32), dtype=torch.uint8), k)


def weight(n=32, k=64):
    size = -(-n // 16) * -(-k // 256) * 2048
    return ops.PackedMx4(torch.zeros(size, dtype=torch.uint8), torch.zeros(size // 16, dtype=torch.uint8), n, k)


def refused(what, f, *args, **kw):
    with pytest.raises(KernelError, match=what):
        f(*args, **kw)


def test_types_and_shapes():
    refused("not supported", ops.mx4_quantize, torch.zeros(2, 32, dtype=torch.float16))
    refused("need rows", ops.mx4_quantize, torch.zeros(2, 2, 32))
    refused("on the GPU", ops.mx4_quantize, torch.zeros(2, 32))
    refused("need an Mx4", ops.mx4_values, torch.zeros(2, 32))
    refused("not supported", ops.mx4_values, four(), torch.float16)
    refused("on the GPU", ops.mx4_values, four())
    for bad in (ops.Mx4(four().codes, four().scales, 65), ops.Mx4(four().codes.int(), four().scales, 64), ops.Mx4(four().codes, four().scales[:3], 64),
                ops.Mx4(four().codes[:, :31], four().scales, 64), ops.Mx4(four(4, 64).codes, four(4, 32).scales, 64)):
        refused("are not those of rows", ops.mx4_values, bad)
        refused("are not those of rows", ops.pack_mx4, bad)
    refused("contiguous and apart", ops.mx4_values, ops.Mx4(torch.zeros(1, 32, dtype=torch.uint8).expand(4, 32), four().scales, 64))
    refused("contiguous and apart", ops.mx4_values, ops.Mx4(torch.zeros(4, 64, dtype=torch.uint8)[:, ::2], four().scales, 64))
    refused("nothing to multiply", ops.pack_mx4, four(0, 64))
    refused("nothing to multiply", ops.pack_mx4, four(4, 0))


def test_products():
    x = torch.zeros(3, 64)
    refused("must be a PackedMx4", ops.gemm_mx4, x, four())
    refused("not supported", ops.gemm_mx4, x.half(), weight())
    refused("need rows", ops.gemm_mx4, x[0], weight())
    refused("with a weight of", ops.gemm_mx4, x, weight(32, 96))
    refused("with a weight of", ops.gemm_mx4, four(3, 96), weight())
    refused("as many gate as up", ops.gemm_mx4, x, weight(33), swiglu=True)
    refused("not supported", ops.gemm_mx4, x, weight(), out_dtype=torch.float16)
    refused("not supported", ops.gemm_mx4, x, weight(), out=torch.zeros(3, 32), out_dtype=torch.bfloat16)
    refused("on the GPU", ops.gemm_mx4, x, weight())
    refused("on the GPU", ops.gemm_mx4, four(3), weight())


def test_what_is_fixed():
    """Rows' tensors are not replaced, and a packed weight has the bytes that its sizes ask for: the kernels read all of them."""
    q = four()
    for name in ("codes", "scales", "k"):
        with pytest.raises(AttributeError):
            setattr(q, name, getattr(q, name))
    w = weight(40, 300)
    for codes, scales, n, k in ((w.codes[:-1], w.scales, 40, 300), (w.codes, w.scales[1:], 40, 300), (w.codes, w.scales, 49, 300), (w.codes, w.scales, 40, 513), (w.codes.int(), w.scales, 40, 300),
                                (w.codes.view(2, -1), w.scales, 40, 300), (w.codes[:0], w.scales[:0], 0, 300)):
        refused("bytes of codes", ops.PackedMx4, codes, scales, n, k)


def test_copies_hold_what_they_were():
    import copy
    import pickle
    q = four(3, 40)
    for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert torch.equal(other.codes, q.codes) and torch.equal(other.scales, q.scales) and other.shape == q.shape


@pytest.mark.gpu
def test_outputs():
    w = ops.pack_mx4(ops.Mx4(four(32).codes.cuda(), four(32).scales.cuda(), 64))
    x = torch.zeros(3, 64).cuda()
    for out in (torch.zeros(3, 31), torch.zeros(4, 32), torch.zeros(3, 64)[:, ::2], torch.zeros(1, 32).expand(3, 32)):
        there = out.cuda() if out.is_contiguous() else torch.empty_strided(out.shape, out.stride(), device="cuda")
        refused("contiguous rows apart", ops.gemm_mx4, x, w, out=there)
    refused("contiguous rows apart", ops.gemm_mx4, x, w, out=torch.zeros(3, 32).cuda(), swiglu=True)
    refused("on the GPU", ops.gemm_mx4, x, w, out=torch.zeros(3, 32))
    wide = torch.zeros(3, 128).cuda()
    refused("over an operand", ops.gemm_mx4, wide[:, :64], w, out=wide[:, 32:64])
    refused("over an operand", ops.gemm_mx4, wide[:, :64], w, out=wide[:, 96:])       # between the rows: refused too
    assert ops.gemm_mx4(wide[:1, :64], w, out=wide[:1, 96:]).shape == (1, 32)
