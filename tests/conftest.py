import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100a) GPU; run with -m gpu")


@pytest.fixture(scope="session")
def lib():
    """The product library, built in-tree if needed (nvcc cross-compiles without a GPU)."""
    from thunderkittens_b200 import build, _lib
    if not (os.path.exists(_lib.LIB_PATH) and os.path.exists(build.TORCH_OPS)):
        build.build()
    return _lib.lib()


@pytest.fixture(scope="session")
def cuda():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if torch.cuda.get_device_capability(0)[0] != 10:
        pytest.skip("not an sm_100 device")
    return torch.device("cuda:0")
