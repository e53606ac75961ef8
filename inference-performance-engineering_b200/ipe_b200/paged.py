"""Operators over a paged K/V cache, for batches of sequences of different lengths.

The cache is two bf16 tensors of pages, keys and values apart, [pages, KV heads, page size, 128] with
a page size of 16, 32, 64 or 128. Position p of sequence s is row p % page size of page
page_table[s, p // page size]; entries of page_table past a sequence's last page are never read. A
batch of new tokens is ragged: sequence s brings rows cu_tokens[s] .. cu_tokens[s + 1] - 1, which are
the last of its lengths[s] positions. Rows behind the last sequence (a buffer of fixed size) are left
as they are, in the outputs too. A decode step brings one row per sequence.

page_table [S, pages per sequence], cu_tokens [S + 1], lengths [S] and prefix_pages are int32 tensors
on the device: a call reads none of them on the host, allocates at most a workspace, never
synchronises, and replays from a CUDA graph with other values in them. What only the device can see it
checks there (`ipe_b200._native.device_error`): a length that is negative, too long for its row of the
page table or less than the sequence's new tokens sets device error 2, a page outside the cache device
error 5. Keys without a place are not appended and such a sequence's output rows hold no meaning; the other
sequences are served, and nothing outside the tensors is touched. Offsets that are not ascending rows set device error 2
in paged_prefill_attention, which serves the sequences before the first such one.

Scores, weighted sums of values and their sums of weights are fp32; sums that pass its range are infinite.
Every function runs on the current stream of its tensors' device. Outputs must not overlap inputs.

  paged_qk_norm_rope_append   q/k norm, rotation and the append (src/ipe/forward.py:101-109)
  paged_decode_attention      one new token per sequence (src/ipe/ops.py:78-101, decode)
  paged_prefill_attention     prompts, or pieces of prompts on a context (src/ipe/ops.py:78-101, causal)
  shared_prefix_attention     a decode step of sequences that begin with the same pages
"""

from __future__ import annotations

import functools

import torch

from ipe_b200 import _native as nat

# An ordinary call is checked and launched by csrc/paged_calls.cpp: the kernels of a small step take a few
# microseconds, the same work here takes the host 10 to 13. A call that it does not take (None) comes here, where the
# checks say what is wrong with it; what passes them, a call on another device than the current one or of
# subclasses of Tensor, is launched from here. What follows from the tensors' shapes alone (their agreement, the
# sizes the kernels get, the workspace) is worked out once per set of shapes.


def _check(name: str, dtype: torch.dtype, labels: tuple[str, ...], tensors: tuple[torch.Tensor, ...], device: int) -> None:
    """Every tensor is contiguous, on CUDA device `device` and of `dtype`."""
    for t in tensors:
        if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == device and t.is_contiguous()):
            break
    else:
        return
    for label, t in zip(labels, tensors):
        if not isinstance(t, torch.Tensor) or t.get_device() != device:
            raise ValueError(f"{name}: {label} must be a CUDA tensor, on the device of the others")
        if t.dtype is not dtype:
            raise ValueError(f"{name}: {label} must be {dtype}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: {label} must be contiguous")


def _device(name: str, pages: torch.Tensor) -> int:
    if not isinstance(pages, torch.Tensor) or not pages.is_cuda:
        raise ValueError(f"{name}: expected CUDA tensors")
    return pages.get_device()


def _cache_sizes(name, k_pages, v_pages, page_table, lengths):
    """(pages, KV heads, page size, sequences, pages per sequence) from the shapes."""
    if len(k_pages) != 4 or k_pages[3] != 128 or v_pages != k_pages:
        raise ValueError(f"{name}: k_pages and v_pages must share a shape [pages, KV heads, page size, 128]")
    if len(page_table) != 2 or lengths != page_table[:1]:
        raise ValueError(f"{name}: page_table must be [sequences, pages per sequence] and lengths [sequences]")
    return k_pages[0], k_pages[1], k_pages[2], page_table[0], page_table[1]


@functools.lru_cache(maxsize=4096)
def _append_sizes(name, qkv, q_norm, k_norm, cos, sin, cu_tokens, lengths, page_table, q_out, k_pages, v_pages):
    sizes = _cache_sizes(name, k_pages, v_pages, page_table, lengths)
    if len(q_out) != 3 or q_out[2] != 128 or qkv != (q_out[0], (q_out[1] + 2 * sizes[1]) * 128):
        raise ValueError(f"{name}: qkv must be [rows, (query heads + 2 * KV heads) * 128] and q_out [rows, query heads, 128]")
    if q_norm != (128,) or k_norm != (128,) or len(cos) != 2 or cos[1] != 128 or sin != cos:
        raise ValueError(f"{name}: q_norm and k_norm must be [128], cos and sin [positions, 128]")
    if cu_tokens != (sizes[3] + 1,):
        raise ValueError(f"{name}: cu_tokens must be [sequences + 1]")
    return sizes


@functools.lru_cache(maxsize=4096)
def _attention_sizes(name, device, q, k_pages, v_pages, page_table, lengths, out, cu_tokens=None, prefix_pages=None):
    """The cache's sizes, the query heads and the workspace's bytes on CUDA device `device`."""
    sizes = pages, kv_heads, page_size, sequences, width = _cache_sizes(name, k_pages, v_pages, page_table, lengths)
    rows = sequences if cu_tokens is None else "rows"
    if len(q) != 3 or q[2] != 128 or (cu_tokens is None and q[0] != sequences):
        raise ValueError(f"{name}: q must be [{rows}, query heads, 128]")
    if out != (q[0], q[1] * 128):
        raise ValueError(f"{name}: out must be [rows, query heads * 128]")
    if cu_tokens is not None and cu_tokens != (sequences + 1,):
        raise ValueError(f"{name}: cu_tokens must be [sequences + 1]")
    if prefix_pages is not None and (len(prefix_pages) != 1 or prefix_pages[0] > width):
        raise ValueError(f"{name}: prefix_pages must be [prefix pages], no more than the {width} pages per sequence")
    lib = nat.load()
    if cu_tokens is not None:
        workspace = lib.ipe_paged_prefill_attention_workspace(q[0], sequences, q[1], kv_heads)
    elif prefix_pages is not None:
        workspace = lib.ipe_shared_prefix_attention_workspace(sequences, q[1], kv_heads, page_size, prefix_pages[0])
    else:
        workspace = lib.ipe_paged_decode_attention_workspace(sequences, q[1], kv_heads)
    return (*sizes, q[1], int(workspace))


def _launched(status: int | None, name: str) -> bool:
    """Whether the extension module took the call; an entry point's refusal is raised."""
    if status:
        nat.check(status, "ipe_" + name)
    return status is not None


def _elsewhere(device, function, *args):
    """The call under its tensors' device, to which its launches, workspace and stream belong."""
    with torch.cuda.device(device):
        return function(*args)


def paged_qk_norm_rope_append(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, cos: torch.Tensor,
                              sin: torch.Tensor, cu_tokens: torch.Tensor, lengths: torch.Tensor,
                              page_table: torch.Tensor, eps: float, q_out: torch.Tensor, k_pages: torch.Tensor,
                              v_pages: torch.Tensor) -> torch.Tensor:
    """q/k RMSNorm per head, split-half rotation at every token's own position, and the append of K and V.

    qkv [rows, (Hq + 2 Hkv) * 128] (q | k | v per token), q_norm / k_norm [128], cos / sin [positions, 128]
    bf16 or fp32, q_out [rows, Hq, 128]. Computed in fp32 and rounded to bf16 once. A position past the tables
    sets device error 2, and its row is skipped. Sequences may share pages that they read, not one that they append to.
    """
    name = "paged_qk_norm_rope_append"
    if _launched(nat.paged_calls().paged_qk_norm_rope_append(qkv, q_norm, k_norm, cos, sin, cu_tokens, lengths, page_table, eps, q_out, k_pages,
            v_pages), name):
        return q_out
    device = _device(name, k_pages)
    if device != torch._C._cuda_getDevice():
        return _elsewhere(device, paged_qk_norm_rope_append, qkv, q_norm, k_norm, cos, sin, cu_tokens, lengths, page_table, eps,
                          q_out, k_pages, v_pages)
    table = torch.float32 if getattr(cos, "dtype", None) is torch.float32 else torch.bfloat16
    _check(name, torch.bfloat16, ("k_pages", "v_pages", "qkv", "q_norm", "k_norm", "q_out"),
           (k_pages, v_pages, qkv, q_norm, k_norm, q_out), device)
    _check(name, table, ("cos", "sin"), (cos, sin), device)
    _check(name, torch.int32, ("cu_tokens", "lengths", "page_table"), (cu_tokens, lengths, page_table), device)
    rows = q_out.shape
    pages, kv_heads, page_size, sequences, width = _append_sizes(
        name, qkv.shape, q_norm.shape, k_norm.shape, cos.shape, sin.shape, cu_tokens.shape, lengths.shape,
        page_table.shape, rows, k_pages.shape, v_pages.shape)
    status = nat.load().ipe_paged_qk_norm_rope_append(qkv.data_ptr(), rows[0], rows[1], kv_heads, q_norm.data_ptr(),
             k_norm.data_ptr(), cos.data_ptr(), sin.data_ptr(), 1 if table is torch.float32 else 0, cos.shape[0],
             cu_tokens.data_ptr(), lengths.data_ptr(), page_table.data_ptr(), sequences, width, q_out.data_ptr(),
             k_pages.data_ptr(), v_pages.data_ptr(), pages, page_size, eps, torch._C._cuda_getCurrentRawStream(device))
    if status:
        nat.check(status, "ipe_paged_qk_norm_rope_append")
    return q_out


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lengths: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """out [S, Hq * 128] = softmax(q k^T / sqrt(128)) v over keys 0 .. lengths[s] - 1 of every sequence, one query
    token q [S, Hq, 128] each, 1 to 8 query heads per KV head. A sequence of length 0 gives zeros. An infinite value that
    a row sees gives infinity, however small its weight (NaN beside one of the other sign, or where its score is -infinity)."""
    name = "paged_decode_attention"
    if _launched(nat.paged_calls().paged_decode_attention(q, k_pages, v_pages, page_table, lengths, out), name):
        return out
    device = _device(name, k_pages)
    if device != torch._C._cuda_getDevice():
        return _elsewhere(device, paged_decode_attention, q, k_pages, v_pages, page_table, lengths, out)
    _check(name, torch.bfloat16, ("k_pages", "v_pages", "q", "out"), (k_pages, v_pages, q, out), device)
    _check(name, torch.int32, ("page_table", "lengths"), (page_table, lengths), device)
    pages, kv_heads, page_size, sequences, width, q_heads, need = _attention_sizes(
        name, device, q.shape, k_pages.shape, v_pages.shape, page_table.shape, lengths.shape, out.shape)
    workspace = k_pages.new_empty(need, dtype=torch.uint8)  # the call's own: other streams and graphs have others
    status = nat.load().ipe_paged_decode_attention(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(),
             lengths.data_ptr(), out.data_ptr(), sequences, q_heads, kv_heads, pages, page_size, width,
             workspace.data_ptr(), need, torch._C._cuda_getCurrentRawStream(device))
    if status:
        nat.check(status, "ipe_paged_decode_attention")
    return out


def paged_prefill_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                            cu_tokens: torch.Tensor, lengths: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """Causal attention of ragged new tokens q [rows, Hq, 128] over their sequences' pages: token i of the n that
    sequence s brings sees keys 0 .. lengths[s] - n + i. out [rows, Hq * 128]; 1 to 8 query heads per KV head. Infinite
    values as in paged_decode_attention; rows that see values that are not finite take longer, behind all the others."""
    name = "paged_prefill_attention"
    if _launched(nat.paged_calls().paged_prefill_attention(q, k_pages, v_pages, page_table, cu_tokens, lengths, out), name):
        return out
    device = _device(name, k_pages)
    if device != torch._C._cuda_getDevice():
        return _elsewhere(device, paged_prefill_attention, q, k_pages, v_pages, page_table, cu_tokens, lengths, out)
    _check(name, torch.bfloat16, ("k_pages", "v_pages", "q", "out"), (k_pages, v_pages, q, out), device)
    _check(name, torch.int32, ("page_table", "cu_tokens", "lengths"), (page_table, cu_tokens, lengths), device)
    rows = q.shape
    pages, kv_heads, page_size, sequences, width, q_heads, need = _attention_sizes(
        name, device, rows, k_pages.shape, v_pages.shape, page_table.shape, lengths.shape, out.shape, cu_tokens.shape)
    workspace = k_pages.new_empty(need, dtype=torch.uint8)
    status = nat.load().ipe_paged_prefill_attention(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(),
             cu_tokens.data_ptr(), lengths.data_ptr(), out.data_ptr(), rows[0], sequences, q_heads, kv_heads, pages,
             page_size, width, workspace.data_ptr(), need, torch._C._cuda_getCurrentRawStream(device))
    if status:
        nat.check(status, "ipe_paged_prefill_attention")
    return out


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, prefix_pages: torch.Tensor,
                            page_table: torch.Tensor, lengths: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """paged_decode_attention of sequences that begin with the same pages: position p < prefix_pages.numel() * page
    size of every sequence is in prefix_pages, whose keys are read once for the batch; page_table [S, pages per
    sequence] is read for the positions behind it alone (its first prefix_pages.numel() columns may hold anything).
    lengths [S] count the prefix; a sequence that ends inside the prefix sees its own lengths[s] keys of it."""
    name = "shared_prefix_attention"
    if _launched(nat.paged_calls().shared_prefix_attention(q, k_pages, v_pages, prefix_pages, page_table, lengths, out), name):
        return out
    device = _device(name, k_pages)
    if device != torch._C._cuda_getDevice():
        return _elsewhere(device, shared_prefix_attention, q, k_pages, v_pages, prefix_pages, page_table, lengths, out)
    _check(name, torch.bfloat16, ("k_pages", "v_pages", "q", "out"), (k_pages, v_pages, q, out), device)
    _check(name, torch.int32, ("prefix_pages", "page_table", "lengths"), (prefix_pages, page_table, lengths), device)
    prefix = prefix_pages.shape
    pages, kv_heads, page_size, sequences, width, q_heads, need = _attention_sizes(
        name, device, q.shape, k_pages.shape, v_pages.shape, page_table.shape, lengths.shape, out.shape, None, prefix)
    workspace = k_pages.new_empty(need, dtype=torch.uint8)
    status = nat.load().ipe_shared_prefix_attention(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
             prefix_pages.data_ptr(), prefix[0], page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(), sequences,
             q_heads, kv_heads, pages, page_size, width, workspace.data_ptr(), need,
             torch._C._cuda_getCurrentRawStream(device))
    if status:
        nat.check(status, "ipe_shared_prefix_attention")
    return out
