"""Which operands a result lies over (``ops.apart``): rows and vectors, from the first byte of each to its last."""
from __future__ import annotations

import pytest
import torch

from llama_cu_amd.kernels import ops
from llama_cu_amd.kernels.ops import KernelError

memory = torch.zeros(1000)


def rows(at, m, k, stride=None):
    return memory.as_strided((m, k), (k if stride is None else stride, 1), at)


def vector(at, n):
    return memory[at:at + n]


@pytest.mark.parametrize("out,read", [
    (rows(100, 4, 10), rows(60, 4, 10)), (rows(100, 4, 10), rows(140, 4, 10)), (rows(100, 4, 10), vector(140, 7)), (rows(100, 4, 10), vector(93, 7)),
    (rows(107, 4, 10), vector(100, 7)), (rows(100, 1, 10), vector(99, 1)), (rows(100, 1, 10), vector(110, 1)), (rows(100, 4, 10), rows(0, 5, 10, 22)),
    (rows(100, 4, 10), vector(120, 0)), (rows(100, 4, 10), rows(120, 0, 10)), (rows(100, 4, 10), rows(120, 4, 0)), (rows(100, 4, 10), None),
    (rows(100, 1, 10, 900), rows(110, 1, 10, 900)), (vector(100, 9), vector(109, 9)), (vector(109, 9), vector(100, 9))])
def test_beside_each_other(out, read):
    ops.apart("this", out, read)


@pytest.mark.parametrize("out,read", [
    (rows(100, 4, 10), rows(61, 4, 10)), (rows(100, 4, 10), rows(139, 4, 10)), (rows(100, 4, 10), vector(139, 7)), (rows(100, 4, 10), vector(94, 7)),
    (rows(106, 4, 10), vector(100, 7)), (rows(100, 4, 10), vector(115, 1)), (rows(100, 4, 10), rows(0, 5, 10, 23)), (rows(100, 3, 10, 20), vector(112, 5)),
    (vector(100, 9), vector(108, 9)), (vector(108, 9), vector(100, 9)), (rows(100, 4, 10), rows(100, 4, 10))])
def test_over_each_other(out, read):
    with pytest.raises(KernelError, match="this: out lies over an operand"):
        ops.apart("this", out, None, read)
