"""Settings that a launcher makes once for its kernel: each kernel, each device by itself, and only what succeeded is remembered."""
import os
import re
import shutil
import subprocess

import pytest

from logssms_b200.ops import build

PROGRAM = r"""
#include <cstdio>
#include "lb200/per_device.h"
int main() {
    lb200::DoneOnce once, other;
    int calls = 0, answer = 0;
    auto run = [&](lb200::DoneOnce& o, int device) { const int before = calls, rc = o.run(device, [&] { ++calls; return answer; }); std::printf("%d/%d ", rc, calls - before); };
    run(once, 0); run(once, 0); run(once, 1); run(once, 1);
    run(other, 0); run(other, 0);                     // another kernel's
    answer = 7; run(once, 2); run(once, 2);
    answer = 0; run(once, 2); run(once, 2);
    run(once, 64); run(once, 64); run(once, -1);
    std::printf("\n");
}
"""


def test_only_success_is_remembered(tmp_path):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "p.cpp").write_text(PROGRAM)
    exe = os.path.join(tmp_path, "p")
    subprocess.run([compiler, "-std=c++17", "-I", build.INCLUDE, "-o", exe, str(tmp_path / "p.cpp")], check=True)
    got = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()
    assert got == ["0/1", "0/0", "0/1", "0/0", "0/1", "0/0", "7/1", "7/1", "0/1", "0/0", "0/1", "0/1", "0/1"]


def test_every_kernel_of_shared_attention_has_its_own():
    """The helper keeps nothing by a kernel's type, which all instantiations share: each launcher, itself a template of what its kernel
    is a template of, hands over a static of its own."""
    def text(name):
        with open(os.path.join(build.INCLUDE, "lb200", name)) as f:
            return f.read()

    helper = re.search(r"inline int whole_carveout\((.*?)\n}", text("attention_shared.h"), re.S).group(1)
    assert "DoneOnce&" in helper and "static" not in helper
    for name, parameters in (("attention_shared_tc.cuh", "int HD, bool TWO"), ("attention_shared_own.cuh", "int HD")):
        launcher = re.search(r"template <%s>\ninline int launch_\w+\((.*?)\n}" % parameters, text(name), re.S).group(1)
        assert "static DoneOnce carveout;" in launcher and ", carveout)" in launcher
