"""The 4-bit products' libraries under the check of ``test_matrix_waits``: no kernel reads what a matrix instruction makes before it is there.

Their matrix instructions stand in one header, ``mx4/matrix.h``; the scaled ones' waits are what the compiler leaves behind them where no branch lies
between (4 and 8 passes with 4-bit operands on both sides, as the bfloat16 ones')."""
from __future__ import annotations

import os
import subprocess

import pytest

import test_matrix_waits as waits
from llama_cu_amd.kernels import build

SCALED = {"v_mfma_scale_f32_16x16x128_f8f6f4": 8, "v_mfma_scale_f32_32x32x64_f8f6f4": 12}
LIBRARIES = ["mx4_stream", "mx4_tiles"]


def test_every_library_with_these_instructions_is_looked_at():
    header = os.path.join(os.path.dirname(build._sources("mx4")[0]), "mx4", "matrix.h")
    assert sorted(n for n in build.KERNEL_LIBRARIES if header in build._headers(n)) == sorted(LIBRARIES)


@pytest.mark.parametrize("name", LIBRARIES)
def test_results_of_matrix_instructions(name, tmp_path, monkeypatch):
    if not os.path.isfile(waits.OBJDUMP):
        pytest.skip("no llvm-objdump")
    for op, states in SCALED.items():
        monkeypatch.setitem(waits.WAITS, op, states)
    copy = tmp_path / "library.so"
    copy.write_bytes(open(build.build(name), "rb").read())
    subprocess.run([waits.OBJDUMP, "--offloading", copy.name], cwd=tmp_path, check=True, capture_output=True)
    device = [p for p in tmp_path.iterdir() if p.name.endswith("gfx950")]
    assert len(device) == 1
    listing = subprocess.run([waits.OBJDUMP, "-d", "--no-show-raw-insn", str(device[0])], check=True, capture_output=True, text=True).stdout
    count = 0
    for fn, rows in waits.functions(listing).items():
        faults = waits.too_early(rows)
        assert not faults, (fn, faults[:4])
        count += sum("mfma" in r[0] for r in rows)
    assert count > 0
