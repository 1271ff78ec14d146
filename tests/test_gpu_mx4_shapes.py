"""Every shape of the 4-bit products in tiles, forced, and seen to be the one that the library is asked for.

Against 64 bits with the tolerances of ``test_gpu_mx4``: exact terms summed in 32 bits, 1e-5 of the largest result, half a step of bfloat16 (2^-8) more where it is rounded; SwiGLU 2e-5
more (the gate's error passes through a slope of at most 1.1, the product's two factors add theirs)."""
from __future__ import annotations

import pytest
import torch

from divasun_common import assert_close
from test_gpu_divasun import rnd
from test_gpu_mx4 import REL, quantised, values, weight

pytestmark = pytest.mark.gpu

SHAPES = {"bfloat16": 5, "float32": 3, "four": 4}
EVERY = [(kind, shape) for kind, n in SHAPES.items() for shape in range(n)]


@pytest.fixture
def force(monkeypatch):
    """``force(shape, slices)``, and what the library was asked for since: ``[(shape, slices)]``."""
    from llama_cu_amd.kernels import ops
    asked, bind = [], ops.bind

    def watched(library, name, arguments):
        f = bind(library, name, arguments)
        if name != "lcu_mx4_tiles":
            return f

        def call(*args):
            asked.append(args[14:16])
            return f(*args)
        return call
    monkeypatch.setattr(ops, "bind", watched)

    def to(shape, slices):
        asked.clear()
        monkeypatch.setattr(ops, "mx4_choice", lambda *a: (shape, slices))
        return asked
    return to


def operands(kind, m, k, seed=None):
    from llama_cu_amd.kernels import ops
    x = rnd(m, k, seed=m if seed is None else seed).to(torch.float32 if kind == "float32" else torch.bfloat16)
    x[:, ::7] *= 20.0
    return (ops.mx4_quantize(x.cuda()), values(*quantised(x), k)) if kind == "four" else (x.cuda(), x.double())


def steps_of(kind, k):
    return -(-k // 256) if kind == "four" else 2 * -(-k // 128)


def test_all_shapes_are_here():
    from llama_cu_amd.kernels import ops
    assert {"bfloat16": len(ops._MX4_TILES[1]), "float32": len(ops._MX4_TILES[3]), "four": len(ops._MX4_TILES[4])} == SHAPES


@pytest.mark.parametrize("kind,shape", EVERY)
@pytest.mark.parametrize("slices", [1, 3, 100])
# one row, fewer steps of k than a ring holds; tiles that end within rows and features; a gate and its up in one tile of 16, and in tiles apart; several tiles each way
@pytest.mark.parametrize("m,n,k", [(1, 48, 32), (33, 514, 256), (127, 130, 128), (130, 258, 640), (257, 600, 1000), (300, 72, 1536), (515, 1030, 384)])
def test_products(m, n, k, kind, shape, slices, force):
    from llama_cu_amd.kernels import ops
    w, exact = weight(n, k)
    rows, mine = operands(kind, m, k)
    want = mine @ exact.T
    gate, up = want.chunk(2, 1)
    act = gate * torch.sigmoid(gate) * up
    asked = force(shape, slices)
    for dtype in (torch.bfloat16, torch.float32):
        for swiglu in (False, True):
            cols = n // 2 if swiglu else n
            got = ops.gemm_mx4(rows, w, out_dtype=dtype, swiglu=swiglu)
            assert_close(got, act if swiglu else want, REL[dtype] + 2e-5 * swiglu, f"{dtype} swiglu {swiglu}")
            for shift in (0, 3):
                room = torch.full((m + 2, cols + 11), 7.0, dtype=dtype, device="cuda")
                ops.gemm_mx4(rows, w, out=room[1:1 + m, shift:shift + cols], swiglu=swiglu)
                assert torch.equal(room[1:1 + m, shift:shift + cols], got)
                assert (room[0] == 7).all() and (room[m + 1:] == 7).all() and (room[:, :shift] == 7).all() and (room[:, shift + cols:] == 7).all()
    assert asked == [(shape, min(slices, steps_of(kind, k)))] * 12


@pytest.mark.parametrize("kind,shape", EVERY)
def test_rows_and_features_know_nothing_of_each_other(kind, shape, force):
    """A row of NaN and a feature of NaN reach their own row and column only; what lies behind the rows' k and behind the last row is not looked at."""
    from llama_cu_amd.kernels import ops
    m, n, k = 300, 288, 256
    wide = rnd(m + 1, 2 * k, seed=1).to(torch.float32 if kind == "float32" else torch.bfloat16)
    wide[:, k:] = float("nan")
    wide[m] = float("nan")
    wide[70, :k] = float("nan")
    source = rnd(n, k, seed=2).bfloat16()
    source[9] = float("inf")
    w = ops.pack_mx4(ops.mx4_quantize(source.cuda()))
    x = wide.cuda()[:m, :k]
    rows = ops.mx4_quantize(x) if kind == "four" else x
    good = torch.ones(m, n, dtype=torch.bool)
    good[70] = False
    good[:, 9] = False
    for slices in (1, 2):
        asked = force(shape, slices)
        y = ops.gemm_mx4(rows, w).float().cpu()
        assert len(asked) == 1
        steps = steps_of(kind, k)
        assert asked[0] == (shape, min(slices, steps))
        assert torch.isfinite(y[good]).all() and torch.isnan(y[70]).all() and torch.isnan(y[:, 9]).all()


@pytest.mark.parametrize("kind,shape", EVERY)
@pytest.mark.parametrize("slices", [1, 2])
def test_long_sums_again_and_again(kind, shape, slices, force):
    """Rings that go round many times: the same bits from call to call, with other products between, and 64 bits' numbers.  (4e-6 of the largest result at this k, as at the longest of the
    small cases: sqrt(k) 2^-24.)"""
    from llama_cu_amd.kernels import ops
    m, n, k = 290, 560, 5000
    w, exact = weight(n, k)
    rows, mine = operands(kind, m, k)
    other, _ = operands(kind, 64, k, seed=5)
    asked = force(shape, slices)
    first = ops.gemm_mx4(rows, w, out_dtype=torch.float32)
    assert_close(first, mine @ exact.T, REL[torch.float32], f"{kind} {shape}")
    again = []
    for _ in range(6):
        ops.gemm_mx4(other, w, out_dtype=torch.float32)
        again.append(ops.gemm_mx4(rows, w, out_dtype=torch.float32))
    assert all(torch.equal(y, first) for y in again)
    assert asked == [(shape, slices)] * 13


@pytest.mark.parametrize("kind", list(SHAPES))
# two tiles of features a workgroup (more than 8,192 features) and one; more workgroups than the card holds at once, which have four waves; features that end within a tile, and within four
@pytest.mark.parametrize("n,k", [(8210, 300), (70001, 160), (1036, 1030)])
def test_the_kernel_that_streams_the_weight(n, k, kind, force):
    """Every number of rows that it tells apart, the most that the choice gives it (64), and more."""
    from llama_cu_amd.kernels import ops
    w, exact = weight(n, k)
    all_rows, all_mine = operands(kind, 100, k)
    want = all_mine @ exact.T
    asked = force(-1, 1)
    for m in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64, 100):
        rows = ops.Mx4(all_rows.codes[:m], all_rows.scales[:m], k) if kind == "four" else all_rows[:m]
        for dtype in (torch.bfloat16, torch.float32):
            assert_close(ops.gemm_mx4(rows, w, out_dtype=dtype), want[:m], REL[dtype], f"{m} rows to {dtype}")
            if n % 2 == 0:
                gate, up = want[:m].chunk(2, 1)
                assert_close(ops.gemm_mx4(rows, w, out_dtype=dtype, swiglu=True), gate * torch.sigmoid(gate) * up, REL[dtype] + 2e-5, f"swiglu of {m} rows to {dtype}")
    assert asked == []


@pytest.mark.parametrize("kind", list(SHAPES))
@pytest.mark.parametrize("m", [1500, 17001])
def test_rows_in_pieces(m, kind, force, monkeypatch):
    """Rows beyond what one call takes, with a small limit in the place of the 4 GiB: the same bits in pieces as at once.  In 4 bits with the scales of all rows laid out together, and (17,001
    rows) for each piece by itself."""
    from llama_cu_amd.kernels import ops
    n, k = 40, 512
    w, exact = weight(n, k)
    rows, mine = operands(kind, m, k)
    row_bytes = {"bfloat16": 2, "float32": 6, "four": 0.5}[kind] * k
    mine = mine @ exact.T
    for slices in (1, 2):
        asked = force(2, slices)
        want = ops.gemm_mx4(rows, w, out_dtype=torch.float32)
        assert_close(want, mine, REL[torch.float32], f"{kind} {slices}")
        assert len(asked) == 1
        with monkeypatch.context() as limit:
            limit.setattr(ops, "_MX4_PLACES", int(row_bytes) * (512 + 513) + 1)
            room = torch.full((m + 2, n + 5), 7.0, device="cuda")
            got = ops.gemm_mx4(rows, w, out=room[1:1 + m, 3:3 + n])
        assert len(asked) == 1 + -(-m // 513)
        assert torch.equal(got, want) and (room[0] == 7).all() and (room[m + 1:] == 7).all() and (room[:, :3] == 7).all() and (room[:, 3 + n:] == 7).all()


@pytest.mark.parametrize("kind", list(SHAPES))
def test_rows_in_pieces_past_a_streamed_weight(kind, force, monkeypatch):
    from llama_cu_amd.kernels import ops
    m, n, k = 201, 72, 512
    w, exact = weight(n, k)
    rows, mine = operands(kind, m, k)
    asked = force(-1, 1)
    monkeypatch.setattr(ops, "_MX4_STREAM_ROWS", 64)
    room = torch.full((m + 2, n + 5), 7.0, device="cuda")
    got = ops.gemm_mx4(rows, w, out=room[1:1 + m, 3:3 + n])
    assert_close(got, mine @ exact.T, REL[torch.float32], kind)
    assert asked == [] and (room[0] == 7).all() and (room[m + 1:] == 7).all() and (room[:, :3] == 7).all() and (room[:, 3 + n:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(41, 300), (7, 1024), (200, 40)])
def test_conversions_in_pieces(m, k, dtype, monkeypatch):
    """Rows beyond what one launch takes, with a small limit in the place of 2^31 units: the same bits in pieces as at once."""
    from llama_cu_amd.kernels import ops
    wide = rnd(m, k + 8, seed=m).to(dtype).cuda()
    x = wide[:, 3:3 + k]
    want = ops.mx4_quantize(x)
    values_of, w = ops.mx4_values(want, dtype), weight(40, k)[0]
    laid_out = ops._mx4_rows(x, k)
    product, of_four = ops.gemm_mx4(x, w), ops.gemm_mx4(want, w)
    monkeypatch.setattr(ops, "_MX4_UNITS", 3 * 32 * -(-k // 256) + 5)
    got = ops.mx4_quantize(x)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales) and got._by_pair is None
    assert torch.equal(ops.mx4_values(want, dtype), values_of)
    again = ops._mx4_rows(x, k)
    assert again[1] == laid_out[1] and torch.equal(again[0], laid_out[0])
    assert torch.equal(ops.gemm_mx4(x, w), product) and torch.equal(ops.gemm_mx4(got, w), of_four)
