"""What launchers remember about a kernel (host C++): for each device by itself, and only what succeeded."""
import os
import shutil
import subprocess

import pytest

from logssms_b200.ops import build

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "lb200/per_device.h"
int main() {
    lb200::SharedLimits limits;
    int calls = 0, answer = 0;
    auto set = [&](size_t) { ++calls; return answer; };
    auto ask = [&](int device, size_t bytes) { const int before = calls, rc = limits.raise(device, bytes, set); std::printf("%d/%d ", rc, calls - before); };
    ask(0, 40 << 10);                 // nothing to raise
    ask(0, 100 << 10); ask(0, 100 << 10); ask(0, 90 << 10); ask(0, 120 << 10);
    ask(1, 100 << 10); ask(1, 100 << 10); ask(0, 120 << 10);
    answer = 7; ask(2, 300 << 10); ask(2, 300 << 10);
    answer = 0; ask(2, 60 << 10); ask(2, 60 << 10);
    ask(64, 100 << 10); ask(64, 100 << 10); ask(-1, 100 << 10);
    std::printf("\n");
    lb200::AskedOnce asked;
    int times = 0;
    for (int device : {0, 1, 0, 1, 63, 64, 64, -1}) std::printf("%d ", asked.get(device, [&] { ++times; return device == 1 ? 0 : 15 + device; }));
    std::printf("%d\n", times);
}
"""


def test_each_device_by_itself(tmp_path):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "p.cpp").write_text(PROGRAM)
    exe = os.path.join(tmp_path, "p")
    subprocess.run([compiler, "-std=c++17", "-I", build.INCLUDE, "-o", exe, str(tmp_path / "p.cpp")], check=True)
    limits, asked = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines()
    assert limits.split() == ["0/0", "0/1", "0/0", "0/0", "0/1", "0/1", "0/0", "0/0", "7/1", "7/1", "0/1", "0/0", "0/1", "0/1", "0/1"]
    assert asked.split() == ["15", "0", "15", "0", "78", "79", "79", "14", "6"]


def test_the_8_bit_launchers_remember_by_device():
    """No launcher of these operators keeps a plain static beside its kernel: a limit raised on one device would count on the next."""
    for name in ("fp8_linear", "fp8_rows"):
        with open(build.source_path(name)) as f:
            source = f.read()
        assert "static SharedLimits" in source and "static size_t" not in source
