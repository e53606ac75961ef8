"""The extension module behind the paged operators' Python functions: which file is loaded, without a GPU."""

import sysconfig

import pytest
import torch

from ipe_b200 import _native as nat
from ipe_b200 import build


@pytest.fixture
def unloaded(monkeypatch):
    monkeypatch.setattr(nat, "_calls", None)


def test_a_module_of_another_torch_is_stale_and_not_loaded(unloaded, monkeypatch, tmp_path):
    here = nat.paged_calls_path()
    assert here.exists() and torch.__version__ in here.name and sysconfig.get_config_var("SOABI") in here.name
    assert build.build_calls() == here
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    other = nat.paged_calls_path()
    assert other != here and not other.exists()
    assert build._stale(other, [])
    assert nat._calls is None


def test_the_module_of_this_torch_is_loaded(unloaded):
    assert nat.paged_calls().__spec__.origin == str(nat.paged_calls_path())
