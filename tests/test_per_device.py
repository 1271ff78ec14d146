"""Numbers that each device has one of (``csrc/shared/per_device.h``), compiled for the host; and that the kernel which streams 4-bit weights keeps what a device holds at once so."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from llama_cu_amd.kernels import build

PROGRAM = """
#include "per_device.h"
#include <cstdio>
int main() {
    static LcuPerDevice held;
    int asked = 0;
    long long answer = 0;
    auto ask = [&](int device) { ++asked; return answer ? answer + device : 0; };
    auto show = [&](int device) { const long long n = held.get(device, ask, -7); printf("%lld/%d ", n, asked); };
    show(0); show(0);                       // no answer: asked again
    answer = 512; show(0); show(0);         // kept
    show(1); show(1);                       // another device: asked for itself
    answer = 99; show(0); show(1); show(63);
    show(64); show(-1);                     // no such device
}
"""


def test_each_device_is_asked_until_it_answers(tmp_path):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no g++")
    (tmp_path / "program.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-I", build._SHARED_DIR, str(tmp_path / "program.cpp"), "-o", str(tmp_path / "program")], check=True)
    out = subprocess.run([str(tmp_path / "program")], check=True, capture_output=True, text=True).stdout.split()
    assert out == ["-7/1", "-7/2", "512/3", "512/3", "513/4", "513/4", "512/4", "513/4", "162/5", "-7/5", "-7/5"]


def test_what_a_device_holds_is_kept_for_each():
    source = open(build._sources("mx4_stream")[0]).read()
    assert os.path.join(build._SHARED_DIR, "per_device.h") in build._headers("mx4_stream")
    assert re.findall(r"static (?:const )?(\w[\w ]*?) held\b", source) == ["LcuPerDevice"]
