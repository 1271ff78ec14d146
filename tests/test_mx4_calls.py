"""What ``gemm_mx4`` asks of the libraries, without a GPU: tensors that have sizes and no memory, and a recorder in the libraries' place."""
from __future__ import annotations

import pytest
import torch

from llama_cu_amd.kernels import ops

ENTRY = {"lcu_mx4_tiles": "x ldx kind xs lds codes scales pairs y ldy m n k epilogue shape slices planes stream",
         "lcu_mx4_stream": "x ldx kind xs lds codes scales pairs y ldy m n k epilogue stream",
         "lcu_mx4_by_pair": "scales lds rows pairs out stream",
         "lcu_mx4_rows": "x ldx type rows k out stream",
         "lcu_mx4_quantize": "x ldx type rows k codes scales by_pair stream",
         "lcu_mx4_values": "codes ldc scales lds rows k y ldy type stream"}


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


def allowed(name, a):
    """What the library asks of sizes (``lcu_mx4_tiles``, ``lcu_mx4_stream``, ``lcu_mx4_by_pair``)."""
    if name == "lcu_mx4_by_pair":
        return a["lds"] >= 8 * a["pairs"] and a["rows"] > 0
    macros = -(-a["k"] // 128)
    if name == "lcu_mx4_stream":
        return -(-a["m"] // 16) <= 65535 and a["ldx"] < 1 << 24
    row_bytes = a["ldx"] * (1 if a["kind"] == 4 else 2)
    return ((a["m"] + 512) * row_bytes < 1 << 32 and (-(-a["n"] // 16) * 16 + 512) * a["pairs"] * 128 < 1 << 32
            and (a["kind"] != 4 or (a["lds"] >= 8 * a["m"] and (macros + 1) // 2 * a["lds"] + 4096 < 1 << 32)))


def pieces(calls, name, m, row_bytes, out_bytes):
    """The rows of the products' calls: all of them, one after the other, each where it belongs."""
    at = 0
    for entry, a in calls:
        assert allowed(entry, a), (entry, a)
        if entry == name:
            assert (a["x"], a["y"]) == (at * row_bytes, at * out_bytes)
            at += a["m"]
    assert at == m


@pytest.mark.parametrize("m,k", [(4_700_000, 28672), (4_900_000, 28672), (30_000_000, 4096), (40_000_001, 4096), (600_000_000, 256)])
def test_any_number_of_rows_in_4_bits(m, k, calls):
    """The scales of all rows are more than 32 bits say from some number of rows on: each piece of the rows then has its own laid out."""
    w = weight(32, k)
    ops.gemm_mx4(rows("four", m, k), w)
    assert {name for name, _ in calls} == {"lcu_mx4_tiles", "lcu_mx4_by_pair"}
    pieces(calls, "lcu_mx4_tiles", m, k // 2, 2 * 32)
    laid = [a for name, a in calls if name == "lcu_mx4_by_pair"]
    together = k // 256 * 8 * m + 4096 < 1 << 32
    assert sum(a["rows"] for a in laid) == m and (len(laid) == 1) == together
    of = 0
    for name, a in calls:
        if name == "lcu_mx4_by_pair":
            assert together or a["scales"] == of * k // 32
            rows_of = a["rows"]
        else:
            assert a["xs"] == (8 * of if together else 0) and a["lds"] == 8 * (m if together else a["m"]) and (together or rows_of == a["m"])
            of += a["m"]


@pytest.mark.parametrize("kind", ["bfloat16", "four"])
def test_any_number_of_rows_of_a_large_weight(kind, calls):
    """A weight of more than 4 GiB is streamed, whatever the rows, so many of them at a time as a launch takes."""
    n, k, m = 300_000, 28672, 2_500_001
    ops.gemm_mx4(rows(kind, m, k), weight(n, k))
    assert {name for name, _ in calls} == {"lcu_mx4_stream"}
    pieces(calls, "lcu_mx4_stream", m, k // 2 if kind == "four" else 2 * k, 2 * n)
    at = 0
    for _, a in calls:
        assert a["xs"] == (at * k // 32 if kind == "four" else None)
        at += a["m"]


def covered(calls, name, m, most, **bytes_of):
    """The rows of the calls of ``name``: all of them, one after the other, at most ``most`` at a time, each at the bytes a row that are said for its arguments."""
    at = 0
    for entry, a in calls:
        if entry == name:
            assert 0 < a["rows"] <= most and {what: a[what] for what in bytes_of} == {what: at * size for what, size in bytes_of.items()}
            at += a["rows"]
    assert at == m


@pytest.mark.parametrize("m,k", [(1, 1), (16, 4096), (4_194_303, 4096), (4_194_304, 4096), (10_000_001, 4096), (70_000_000, 1000), (3, 1_000_000_000), (20, 1_000_000_000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_conversions_of_any_number_of_rows(m, k, dtype, calls):
    """A launch counts its units of 8 numbers in 31 bits: more of them go in pieces of the rows."""
    size = torch.empty(0, dtype=dtype).element_size()
    x = torch.empty(m, k, dtype=dtype, device="meta")
    whole = -(-k // 256) * 256
    q = ops.mx4_quantize(x)
    assert q.shape == (m, k) and q.codes.shape == (m, -(-k // 32) * 16)
    covered(calls, "lcu_mx4_quantize", m, ((1 << 31) - 1) * 8 // whole, x=k * size, codes=whole // 2, scales=whole // 32)
    calls.clear()
    ops.mx4_values(q, dtype)
    covered(calls, "lcu_mx4_values", m, ((1 << 31) - 1) // -(-k // 8), codes=whole // 2, scales=whole // 32, y=k * size)
    calls.clear()
    if k < 1 << 20 and (dtype == torch.float32 or k % 128):
        planes = 3 if dtype == torch.float32 else 1
        out, kind = ops._mx4_rows(x, k)
        assert out.shape == (m, planes * whole) and kind == planes
        covered(calls, "lcu_mx4_rows", m, ((1 << 31) - 1) * 8 // whole, x=k * size, out=planes * whole * 2)


def test_the_second_copy_of_scales_is_of_all_rows(calls):
    """The scales as the products in tiles read them are written by one launch or not at all."""
    assert ops.mx4_quantize(torch.empty(4_194_303, 4096, dtype=torch.bfloat16, device="meta"))._by_pair is not None
    assert ops.mx4_quantize(torch.empty(4_194_304, 4096, dtype=torch.bfloat16, device="meta"))._by_pair is None


def test_lengths_that_no_kernel_counts(calls):
    """Counts along k, and of features, go to the libraries as 32-bit numbers: longer ones would arrive as others."""
    def refused(f, *args):
        with pytest.raises(ops.KernelError, match="less than 2\\^30"):
            f(*args)
    empty = lambda *shape: torch.empty(*shape, dtype=torch.uint8, device="meta")
    longest = (1 << 30) - 1
    for k in (1 << 30, (1 << 31) + 5, (1 << 32) + 256):
        q = ops.Mx4(empty(1, -(-k // 32) * 16), empty(1, -(-k // 32)), k)
        refused(ops.mx4_quantize, torch.empty(1, k, dtype=torch.bfloat16, device="meta"))
        refused(ops.mx4_values, q)
        refused(ops.pack_mx4, q)
        refused(weight, 16, k)
        refused(weight, k, 16)
    ops.mx4_values(ops.mx4_quantize(torch.empty(1, longest, dtype=torch.bfloat16, device="meta")))
    assert all(a["k"] == longest for _, a in calls) and len(calls) == 2
    assert weight(16, longest).k == longest and weight(longest, 16).n == longest


@pytest.mark.parametrize("weights", ["MX4", "4bit", "", None])
def test_how_matrices_are_held(weights):
    """A word that is none of the ways is refused wherever it comes in, not taken for the file's."""
    from llama_cu_amd.engine.config import EngineConfig
    from llama_cu_amd.parts.base import BuildContext
    for make in (lambda w: BuildContext(torch.bfloat16, torch.device("cpu"), 64, 16, weights=w), lambda w: EngineConfig(weights=w)):
        assert make("file").weights == "file" and make("mx4").weights == "mx4"
        with pytest.raises(ValueError, match="neither file nor mx4"):
            make(weights)
