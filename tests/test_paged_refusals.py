"""What the paged-cache operators refuse on the host, without a GPU: the C entry points reject bad sizes and pointers
before any device call, and the Python functions reject wrong devices, types, shapes and strides."""

import pytest
import torch

from ipe_b200 import _native as nat
from ipe_b200 import ops

GOOD = {
    "ipe_paged_qk_norm_rope_append": dict(qkv=16, tokens=4, q_heads=16, kv_heads=8, q_norm=16, k_norm=16, cos=16, sin=16,
                                          table_dtype=0, table_rows=64, cu_tokens=16, lengths=16, page_table=16, sequences=2,
                                          max_pages=4, q_out=16, k_pages=16, v_pages=16, num_pages=9, page_size=16, eps=1e-6,
                                          stream=None),
    "ipe_paged_decode_attention": dict(q=16, k_pages=16, v_pages=16, page_table=16, lengths=16, out=16, sequences=2,
                                       q_heads=16, kv_heads=8, num_pages=9, page_size=16, max_pages=4, workspace=256,
                                       workspace_bytes=1 << 30, stream=None),
    "ipe_paged_prefill_attention": dict(q=16, k_pages=16, v_pages=16, page_table=16, cu_tokens=16, lengths=16, out=16,
                                        tokens=5, sequences=2, q_heads=16, kv_heads=8, num_pages=9, page_size=16,
                                        max_pages=4, workspace=256, workspace_bytes=1 << 30, stream=None),
    "ipe_shared_prefix_attention": dict(q=16, k_pages=16, v_pages=16, prefix_pages=16, prefix_count=2, page_table=16,
                                        lengths=16, out=16, sequences=2, q_heads=16, kv_heads=8, num_pages=9, page_size=16,
                                        max_pages=4, workspace=256, workspace_bytes=1 << 30, stream=None),
}

BAD = [
    ("ipe_paged_qk_norm_rope_append", dict(q_heads=15)),
    ("ipe_paged_qk_norm_rope_append", dict(q_heads=72)),
    ("ipe_paged_qk_norm_rope_append", dict(kv_heads=0)),
    ("ipe_paged_qk_norm_rope_append", dict(page_size=24)),
    ("ipe_paged_qk_norm_rope_append", dict(page_size=256)),
    ("ipe_paged_qk_norm_rope_append", dict(num_pages=0)),
    ("ipe_paged_qk_norm_rope_append", dict(num_pages=2 ** 24)),
    ("ipe_paged_qk_norm_rope_append", dict(max_pages=0)),
    ("ipe_paged_qk_norm_rope_append", dict(max_pages=2 ** 27)),
    ("ipe_paged_qk_norm_rope_append", dict(tokens=-1)),
    ("ipe_paged_qk_norm_rope_append", dict(tokens=2 ** 31)),
    ("ipe_paged_qk_norm_rope_append", dict(sequences=-1)),
    ("ipe_paged_qk_norm_rope_append", dict(table_dtype=2)),
    ("ipe_paged_qk_norm_rope_append", dict(table_rows=0)),
] + [("ipe_paged_qk_norm_rope_append", {p: v}) for p in
     ("qkv", "q_norm", "k_norm", "cos", "sin", "cu_tokens", "lengths", "page_table", "q_out", "k_pages", "v_pages")
     for v in (None, 18)] + [
    (name, change)
    for name in ("ipe_paged_decode_attention", "ipe_paged_prefill_attention", "ipe_shared_prefix_attention")
    for change in [dict(q_heads=15), dict(q_heads=72), dict(q_heads=0), dict(kv_heads=0), dict(page_size=8), dict(page_size=48),
                   dict(num_pages=0), dict(num_pages=2 ** 25), dict(max_pages=0), dict(max_pages=2 ** 24),
                   dict(sequences=-1), dict(sequences=2 ** 25), dict(workspace=None), dict(workspace=16),
                   dict(workspace_bytes=64)] +
                  [{p: v} for p in ("q", "k_pages", "v_pages", "page_table", "lengths", "out") for v in (None, 18)]] + [
    ("ipe_paged_prefill_attention", dict(tokens=-1)),
    ("ipe_paged_prefill_attention", dict(tokens=2 ** 28)),
    ("ipe_paged_prefill_attention", dict(cu_tokens=None)),
    ("ipe_paged_prefill_attention", dict(cu_tokens=17)),
    ("ipe_shared_prefix_attention", dict(prefix_count=-1)),
    ("ipe_shared_prefix_attention", dict(prefix_count=5)),
    ("ipe_shared_prefix_attention", dict(prefix_pages=None)),
    ("ipe_shared_prefix_attention", dict(prefix_pages=18)),
    ("ipe_shared_prefix_attention", dict(sequences=2 ** 22, prefix_count=2 ** 11, max_pages=2 ** 11)),
    # units of 64 keys past 32 bits
    ("ipe_paged_decode_attention", dict(sequences=2 ** 20, max_pages=2 ** 20)),
]


@pytest.mark.parametrize(("name", "change"), BAD)
def test_the_entry_points_refuse(name, change):
    args = {**GOOD[name], **change}
    assert getattr(nat.load(), name)(*args.values()) in (1, 2)
    assert nat.load().ipe_last_error().decode().startswith(name)


def test_nothing_to_do_is_no_error():
    for name, change in [("ipe_paged_qk_norm_rope_append", dict(tokens=0, qkv=None, q_out=None)),
                         ("ipe_paged_qk_norm_rope_append", dict(sequences=0, page_table=None)),
                         ("ipe_paged_decode_attention", dict(sequences=0, q=None, out=None, page_table=None, workspace=None)),
                         ("ipe_paged_prefill_attention", dict(tokens=0, q=None, out=None, workspace=None)),
                         ("ipe_shared_prefix_attention", dict(sequences=0, q=None, out=None, lengths=None))]:
        assert getattr(nat.load(), name)(*{**GOOD[name], **change}.values()) == 0


def test_the_workspaces_sizes():
    """Nothing for sizes that make no call; what splits work needs room, and more where there are more parts."""
    lib = nat.load()
    assert lib.ipe_paged_decode_attention_workspace(0, 16, 8) == 0
    assert lib.ipe_paged_decode_attention_workspace(4, 40, 8) > lib.ipe_paged_decode_attention_workspace(4, 16, 8) > 0
    assert lib.ipe_paged_prefill_attention_workspace(0, 1, 16, 8) == 0
    assert lib.ipe_paged_prefill_attention_workspace(100, 1, 16, 8) > 0
    assert lib.ipe_paged_prefill_attention_workspace(100000, 1, 16, 8) == 0  # whole blocks: no parts
    assert lib.ipe_shared_prefix_attention_workspace(4, 16, 8, 16, 9) > lib.ipe_paged_decode_attention_workspace(4, 16, 8)


def test_no_workspace_for_pages_of_no_size():
    for page_size in (0, 129, 2 ** 31 - 1):
        assert nat.load().ipe_shared_prefix_attention_workspace(4, 16, 8, page_size, 9) == 0


@pytest.mark.parametrize(("q_heads", "kv_heads"), [(4096, 1), (9, 1), (15, 8), (8, 16), (0, 1), (16, 0), (-16, 8), (16, -8)])
def test_no_workspace_for_heads_that_are_refused(q_heads, kv_heads):
    lib = nat.load()
    assert lib.ipe_paged_decode_attention_workspace(64, q_heads, kv_heads) == 0
    assert lib.ipe_paged_prefill_attention_workspace(64, 2, q_heads, kv_heads) == 0
    assert lib.ipe_shared_prefix_attention_workspace(64, q_heads, kv_heads, 16, 4) == 0


@pytest.mark.parametrize(("page_size", "prefix_count"), [(24, 4), (1, 4), (8, 4), (128, 2 ** 20 + 1), (16, 2 ** 31 - 1), (64, -1)])
def test_no_workspace_for_prefixes_that_are_refused(page_size, prefix_count):
    assert nat.load().ipe_shared_prefix_attention_workspace(64, 16, 8, page_size, prefix_count) == 0


def test_the_extension_module_leaves_other_calls_to_the_checks():
    x = torch.zeros(2, 2)
    calls = nat.paged_calls()
    for name, n in (("paged_qk_norm_rope_append", 12), ("paged_decode_attention", 6), ("paged_prefill_attention", 7),
                    ("shared_prefix_attention", 7)):
        assert getattr(calls, name)(*[x] * n) is None
        assert getattr(calls, name)(*[None] * n) is None
        assert getattr(calls, name)(*["pages"] * n) is None
        with pytest.raises(TypeError, match=str(n)):
            getattr(calls, name)(*[x] * (n - 1))


def test_cpu_tensors_are_refused():
    pages, table, one = torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, out, cu = torch.zeros(1, 4, 128, dtype=torch.bfloat16), torch.zeros(1, 512, dtype=torch.bfloat16), torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode_attention(q, pages, pages, table, one, out)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_prefill_attention(q, pages, pages, table, cu, one, out)
    with pytest.raises(ValueError, match="CUDA"):
        ops.shared_prefix_attention(q, pages, pages, one, table, one, out)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_qk_norm_rope_append(q, q, q, q, q, cu, one, table, 1e-6, q, pages, pages)


def test_the_operators_are_registered():
    for name in ("paged_qk_norm_rope_append", "paged_decode_attention", "paged_prefill_attention", "shared_prefix_attention"):
        assert hasattr(torch.ops.ipe_b200, name)
