import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP path)")
    try:
        # before any test file loads the library: torch brings a HIP runtime of its own,
        # and a process that has loaded another one first gives torch no device
        import torch  # noqa: F401
    except ImportError:
        pass


def gpu_available() -> bool:
    try:
        import torch  # plumbing only: device presence
        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.fixture(scope="session")
def hip():
    """The built extension; GPU tests fail loudly when it is missing."""
    import sili__new_amd
    return sili__new_amd
