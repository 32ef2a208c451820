import functools
import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU and the built HIP library")


@functools.lru_cache(maxsize=None)
def _calls_entries(path) -> bool:
    return "_lib.call(" in Path(path).read_text()


def pytest_collection_modifyitems(config, items):
    """GPU tests need a device.  Host tests that hand the C entries made-up addresses
    need one to be absent: a call that is not refused would run on them."""
    import torch
    there = torch.cuda.is_available()
    skip = pytest.mark.skip(reason="made-up addresses: runs where no GPU is visible" if there
                            else "no GPU in this environment")
    for item in items:
        gpu = "gpu" in item.keywords
        if _calls_entries(item.path) and not gpu if there else gpu:
            item.add_marker(skip)


@pytest.fixture(scope="session")
def oracle_codec():
    from oracle import codec
    codec.build()
    return codec


@pytest.fixture(scope="session")
def dev():
    import torch
    torch.backends.cuda.matmul.allow_tf32 = False
    return torch.device("cuda:0")
