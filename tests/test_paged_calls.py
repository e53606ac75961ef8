"""The extension module behind the paged operators' Python functions: which file is loaded, without a GPU."""

import contextlib
import sysconfig

import pytest
import torch

from ipe_b200 import _native as nat
from ipe_b200 import build, ops


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


@pytest.mark.parametrize("content", [None, b"", b"no module"])
def test_without_a_module_the_operators_are_there(unloaded, monkeypatch, tmp_path, content):
    path = tmp_path / "_paged_calls.so"
    if content is not None:
        path.write_bytes(content)
    monkeypatch.setattr(nat, "paged_calls_path", lambda: path)
    with pytest.warns(RuntimeWarning, match="_paged_calls"):
        calls = nat.paged_calls()
    assert all(getattr(calls, name)() is None for name in nat.PAGED_CALLS)
    cpu = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):  # the checks of the Python functions are reached
        ops.paged_decode_attention(cpu, cpu, cpu, cpu, cpu, cpu)


@pytest.mark.parametrize("missing", ["g++", "Python.h"])
def test_the_library_is_built_where_the_module_cannot_be(monkeypatch, tmp_path, missing):
    find, paths = build.shutil.which, build.sysconfig.get_paths
    monkeypatch.setattr(nat, "paged_calls_path", lambda: tmp_path / "_paged_calls.so")
    if missing == "g++":
        monkeypatch.setattr(build.shutil, "which", lambda name: None if name == "g++" else find(name))
    else:
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {**paths(), "include": str(tmp_path)})
    with pytest.warns(RuntimeWarning, match=r"g\+\+" if missing == "g++" else "Python.h"):
        assert build.build() == build.LIBRARY
    assert not (tmp_path / "_paged_calls.so").exists()


@pytest.mark.gpu
def test_without_a_module_the_results_are_the_same(unloaded, monkeypatch, tmp_path):
    from test_gpu_paged import Batch, decode, normal, prefill, shared

    b = Batch([1] * 3, [99, 40, 300], 16, 2, seed=1, prefix=2).fill(10)
    q = normal((3, 4, 128), 2)
    whole = b.page_table.clone()
    whole[:, :2] = b.prefix_pages
    qkv, w = normal((3, 8 * 128), 3), torch.ones(128, dtype=torch.bfloat16, device="cuda")
    cos, sin = normal((400, 128), 4), normal((400, 128), 5)

    def outputs():
        k, v, q_out = b.k.clone(), b.v.clone(), torch.zeros_like(q)
        ops.paged_qk_norm_rope_append(qkv, w, w, cos, sin, b.cu, b.lengths, whole, 1e-6, q_out, k, v)
        outs = [shared(b, q)]
        b.page_table, table = whole, b.page_table
        outs += [decode(b, q), prefill(b, q), q_out, k.nan_to_num(), v.nan_to_num()]
        b.page_table = table
        return outs

    with_module = outputs()
    monkeypatch.setattr(nat, "_calls", None)
    monkeypatch.setattr(nat, "paged_calls_path", lambda: tmp_path / "_paged_calls.so")
    with pytest.warns(RuntimeWarning, match="_paged_calls"):
        without = outputs()
    assert all(torch.equal(x, y) for x, y in zip(with_module, without))
    assert nat.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("module", [True, False])
def test_a_workspace_that_does_not_fit_is_out_of_memory(unloaded, monkeypatch, tmp_path, module):
    if not module:
        monkeypatch.setattr(nat, "paged_calls_path", lambda: tmp_path / "_paged_calls.so")
    from test_gpu_paged import DEV

    pages = torch.zeros(1, 8, 16, 128, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(64, 64, 128, dtype=torch.bfloat16, device=DEV)
    table, lengths = torch.zeros(64, 100, dtype=torch.int32, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    prefix, out = torch.zeros(100, dtype=torch.int32, device=DEV), torch.ones(64, 64 * 128, dtype=torch.bfloat16, device=DEV)
    need, held = nat.load().ipe_shared_prefix_attention_workspace(64, 64, 8, 16, 100), []
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(1e-6)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            while True:  # what the allocator has left over in blocks that it cannot give back
                held.append(torch.empty(need, dtype=torch.uint8, device=DEV))
        with pytest.warns(RuntimeWarning) if not module else contextlib.nullcontext(), pytest.raises(torch.OutOfMemoryError):
            ops.shared_prefix_attention(q, pages, pages, prefix, table, lengths, out)
    finally:
        held.clear()
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert (out == 1).all()
    ops.shared_prefix_attention(q, pages, pages, prefix, table, lengths, out)
    assert (out == 0).all()
