import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200); runs through the C ABI")


# Tests that cannot pass without oracle/_ref, which build() makes from the
# reference's sources where it finds them.
NEED_REFERENCE_BUILD = ("test_gpu_gemm.py::test_gemm_8192_full_matrix_vs_reference_kernel",
                        "test_gpu_reference_capi.py::test_reference_capi_test_passes")


def pytest_collection_modifyitems(items):
    """Where oracle/_ref is missing they run last and fail there, so that a run
    that stops at its first failure has run everything else first."""
    if not (ROOT / "oracle" / "_ref" / "libref_kernels.so").exists():
        items.sort(key=lambda item: any(name in item.nodeid for name in NEED_REFERENCE_BUILD))


def gpu_available() -> bool:
    try:
        import torch

        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.fixture(scope="session")
def session():
    from fercuda_b200 import capi

    s = capi.Session(0, pool_bytes=4 << 30)
    yield s
    s.close()
