import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a ROCm GPU (run on the MI355X box)")


# Cases whose expectation is not what the operator promises.  They run as they are, and are expected to fail.
HOLD_A_WRONG_VALUE = {
    "test_gpu_paged_cache.py": ({f"test_every_code_in_fp16[{e}]" for e in (22, 23, 24, 25, 40, 119)},
                                "expects the largest code of the block within fp16 (57344, 49152, 32768, 0) where the cache holds more "
                                "than 65504; documented is 61440, which test_gpu_paged_fp16_range.py checks"),
}


def pytest_collection_modifyitems(items):
    for item in items:
        names, reason = HOLD_A_WRONG_VALUE.get(os.path.basename(str(item.path)), ((), ""))
        if item.name in names:
            item.add_marker(pytest.mark.xfail(reason=reason, strict=True))


@pytest.fixture(scope="session")
def gpu():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")
    return torch.device("cuda:0")
