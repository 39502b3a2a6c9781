"""A launch that CUDA refuses (a grid beyond its limits: nothing runs) is that call's error, and no later call's."""
import ctypes
import os
import re

import pytest
import torch

from logssms_b200.ops import build

TOO_LARGE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "toy_kernels", "too_large_grid.cu")


@pytest.mark.gpu
def test_a_refused_launch_leaves_nothing_behind():
    lib = build.load(TOO_LARGE)
    lib.lb_too_large_grid.argtypes = [ctypes.c_int, ctypes.c_void_p]
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.lb_too_large_grid(1, stream) == 0 and lib.lb_left_behind() == 0
    assert lib.lb_too_large_grid(1 << 17, stream) != 0
    assert lib.lb_left_behind() == 0 and lib.lb_too_large_grid(1, stream) == 0
    torch.cuda.synchronize()


def test_every_launcher_takes_its_error_back():
    for root, _, files in os.walk(build.CSRC):
        for name in files:
            if name.endswith((".cu", ".cuh")):
                with open(os.path.join(root, name)) as f:
                    text = f.read()
                assert len(re.findall(r"cudaLaunchKernelEx\(", text)) == len(re.findall(r"launched\(cudaLaunchKernelEx\(", text)), name
