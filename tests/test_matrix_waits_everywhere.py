"""Every library whose sources name a matrix instruction, in whatever folder and through whatever header, is under the check of ``test_matrix_waits``: by the list there, which is that of
the sources in ``csrc/kernels`` itself, or by the list of ``test_matrix_waits_mx4``."""
from __future__ import annotations

import os

import pytest

import test_load_order
import test_matrix_waits
import test_matrix_waits_mx4

from llama_cu_amd.kernels import build

CHECKED = test_matrix_waits.LIBRARIES + test_matrix_waits_mx4.LIBRARIES


def naming():
    return [n for n in build.KERNEL_LIBRARIES if any("_mfma_" in open(p).read() for p in build._sources(n) + build._headers(n))]


def test_every_library_that_names_one_is_checked_once():
    assert sorted(naming()) == sorted(CHECKED)


def test_headers_of_every_folder_are_followed():
    """The headers that are read for it are all that the kernels' folder holds, but for those that no kernel includes."""
    root = os.path.dirname(build._sources("moe")[0])
    there = {os.path.join(d, f) for d, _, files in os.walk(root) for f in files if f.endswith((".h", ".hip"))}
    read = {p for n in build.KERNEL_LIBRARIES for p in build._sources(n) + build._headers(n)}
    assert there <= read, sorted(there - read)


@pytest.mark.parametrize("name", [n for n in build.KERNEL_LIBRARIES if n not in CHECKED])
def test_no_other_library_has_one(name, tmp_path):
    assert not any("mfma" in op for rows in test_load_order.kernels(name, tmp_path).values() for op, _, _ in rows)
