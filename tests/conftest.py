import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a) and the built extension")
    config.addinivalue_line("markers", "multigpu: needs 2+ CUDA GPUs")
    config.addinivalue_line("markers", "slow: long-running test")


def pytest_collection_modifyitems(config, items):
    import torch

    has_gpu = torch.cuda.is_available()
    n_gpu = torch.cuda.device_count() if has_gpu else 0
    for item in items:
        if "gpu" in item.keywords and not has_gpu:
            item.add_marker(pytest.mark.skip(reason="no CUDA GPU"))
        if "multigpu" in item.keywords and n_gpu < 2:
            item.add_marker(pytest.mark.skip(reason="needs 2+ GPUs"))


@pytest.fixture(autouse=True)
def no_wait_ran_out(request):
    """After a GPU test of the 8-bit paged cache: no bounded wait inside its kernels ran out."""
    yield
    if "gpu" in request.keywords and request.module.__name__.startswith("test_paged8"):
        import torch

        from verl_omni_b200.ops import paged8

        if torch.cuda.is_available():
            paged8.raise_on_timeout("cuda")
