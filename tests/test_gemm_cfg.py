"""Which instances of the GEMM template there may be: what the kernel does not handle does not compile."""
import os
import subprocess

import pytest

from thunderkittens_b200 import build

ALLOWED = ["KIND_INT8, 1, 64", "KIND_INT8, 1, 128", "KIND_INT8, 2, 128", "KIND_INT8, 1, 256", "KIND_INT8, 2, 256", "KIND_NVFP4, 2, 256", "KIND_MXFP8, 1, 128",
           "KIND_BF16, 2, 256, 2", "KIND_FP8, 2, 256, 2"]
REFUSED = ["KIND_INT8, 2, 64",            # a CTA pair's producer would load one of the two blocks of K that its barriers wait for
           "KIND_INT8, 1, 64, 2", "KIND_BF16, 1, 64", "KIND_INT8, 2, 256, 2", "KIND_BF16, 1, 256, 2", "KIND_INT8, 1, 96"]


def _compiles(args):
    code = f'#include "gemm_cfg.h"\nusing namespace tkb;\ntemplate struct tkb::GemmCfg<{args}>;\n'
    r = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-I", build.CSRC, "-I", os.path.join(build.CUDA_HOME, "include"), "-x", "c++", "-"],
                       input=code, capture_output=True, text=True)
    return r.returncode == 0, r.stderr


@pytest.mark.parametrize("args", ALLOWED)
def test_instances_that_the_kernel_has(args):
    ok, text = _compiles(args)
    assert ok, text


@pytest.mark.parametrize("args", REFUSED)
def test_instances_that_the_kernel_cannot_run(args):
    ok, text = _compiles(args)
    assert not ok and "static assertion" in text, text
