"""What ``gemm_mx4`` asks of the libraries, without a GPU: tensors that have sizes and no memory, and a recorder in the libraries' place."""
from __future__ import annotations

import pytest
import torch

from llama_cu_amd.kernels import ops

ENTRY = {"lcu_mx4_tiles": "x ldx kind xs lds codes scales pairs y ldy m n k epilogue shape slices planes stream",
         "lcu_mx4_stream": "x ldx kind xs lds codes scales pairs y ldy m n k epilogue stream",
         "lcu_mx4_by_pair": "scales lds rows pairs out stream",
         "lcu_mx4_rows": "x ldx type rows k out stream"}


@pytest.fixture
def calls(monkeypatch):
    """The calls of the libraries' entry points, in their order: ``(entry, {argument: value})``."""
    made = []

    def bind(library, name, arguments):
        def entry(*args):
            if name == "lcu_capture_id":
                return 0
            names = ENTRY[name].split()
            assert len(args) == len(names) == len(arguments) + 1
            made.append((name, dict(zip(names, args))))
            return 0
        return entry
    monkeypatch.setattr(ops, "bind", bind)
    monkeypatch.setattr(ops, "here", lambda *a: None)
    monkeypatch.setattr(ops, "raw_stream", lambda: 0)
    return made


def weight(n, k):
    size = -(-n // 16) * -(-k // 256) * 2048
    return ops.PackedMx4(torch.empty(size, dtype=torch.uint8, device="meta"), torch.empty(size // 16, dtype=torch.uint8, device="meta"), n, k)


def rows(kind, m, k):
    if kind == "four":
        blocks = -(-k // 32)
        return ops.Mx4(torch.empty(m, 16 * blocks, dtype=torch.uint8, device="meta"), torch.empty(m, blocks, dtype=torch.uint8, device="meta"), k)
    return torch.empty(m, k, dtype=torch.float32 if kind == "float32" else torch.bfloat16, device="meta")


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "four"])
@pytest.mark.parametrize("shape", [(-1, 1), (0, 1), (1, 3), (2, 2)])
def test_the_choice_is_what_is_called(kind, shape, calls, monkeypatch):
    """``mx4_choice`` chooses: whoever replaces it, as the tests of single kernels do, replaces the kernel."""
    monkeypatch.setattr(ops, "mx4_choice", lambda *a: shape)
    ops.gemm_mx4(rows(kind, 48, 1024), weight(256, 1024))
    name, args = calls[-1]
    assert name == ("lcu_mx4_stream" if shape[0] < 0 else "lcu_mx4_tiles")
    assert shape[0] < 0 or (args["shape"], args["slices"]) == shape
