from __future__ import annotations

import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line(
        "markers", "gpu: needs a HIP device (MI355X) and the built libcowsdm.so")


@pytest.fixture(scope="session")
def device():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("GPU test requested but no HIP device is visible")
    return torch.device("cuda:0")


@pytest.fixture(scope="module", autouse=True)
def cleared_memory():
    """GPU tests of a module start on memory without the NaN that other modules
    leave: some compare whole buffers, places that nothing has written too, and
    a NaN there differs from its own copy."""

    import torch

    if torch.cuda.is_available():
        torch.cuda.empty_cache()
        taken = []
        # what the allocator holds free in segments that are in use
        for size in [1 << n for n in range(24, 20, -1)] + [(1 << 20) + 512] + [
                1 << n for n in range(20, 8, -1)]:
            while True:
                held = torch.cuda.memory_reserved()
                part = torch.zeros(size, dtype=torch.uint8, device="cuda")
                if torch.cuda.memory_reserved() > held:
                    break
                taken.append(part)
            del part
            torch.cuda.empty_cache()
        taken.clear()
        torch.cuda.empty_cache()
    yield
