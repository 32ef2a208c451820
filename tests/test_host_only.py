"""Tests that hand made-up addresses to the C entries are kept from a device."""
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from tests import conftest

HERE = Path(__file__).parent


def _skipped(monkeypatch, there, name, gpu):
    marks = []
    item = SimpleNamespace(path=HERE / name, keywords={"gpu": None} if gpu else {},
                           add_marker=marks.append)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: there)
    conftest.pytest_collection_modifyitems(None, [item])
    return bool(marks)


@pytest.mark.parametrize("name", [
    "test_abi.py", "test_balance.py", "test_embedding.py", "test_embedding_limits.py",
    "test_launch_limits.py", "test_logprobs.py", "test_muon.py", "test_packed.py",
    "test_residual_norms.py"])
def test_made_up_addresses_stay_on_the_host(monkeypatch, name):
    assert _skipped(monkeypatch, True, name, gpu=False)
    assert not _skipped(monkeypatch, False, name, gpu=False)


def test_others_run_as_they_did(monkeypatch):
    assert not _skipped(monkeypatch, True, "test_gpu_moe.py", gpu=True)
    assert _skipped(monkeypatch, False, "test_gpu_moe.py", gpu=True)
    assert not _skipped(monkeypatch, True, "test_archive.py", gpu=False)
    assert not _skipped(monkeypatch, False, "test_archive.py", gpu=False)
