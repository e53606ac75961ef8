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
sequences are served, and nothing outside the tensors is touched.

Every function runs on the current stream of its tensors' device. Outputs must not overlap inputs.

  paged_qk_norm_rope_append   q/k norm, rotation and the append (src/ipe/forward.py:101-109)
  paged_decode_attention      one new token per sequence (src/ipe/ops.py:78-101, decode)
  paged_prefill_attention     prompts, or pieces of prompts on a context (src/ipe/ops.py:78-101, causal)
  shared_prefix_attention     a decode step of sequences that begin with the same pages
"""

from __future__ import annotations

import contextlib
import functools

import torch

from ipe_b200 import _native as nat

_SAME_DEVICE = contextlib.nullcontext()


def _device(name: str, pages: torch.Tensor) -> int:
    if not isinstance(pages, torch.Tensor) or not pages.is_cuda:
        raise ValueError(f"{name}: expected CUDA tensors")
    return pages.get_device()


def _check(name: str, device: int, dtype: torch.dtype, **tensors: torch.Tensor) -> None:
    """Every tensor is contiguous, on CUDA device `device` and of `dtype`."""
    for label, t in tensors.items():
        if not isinstance(t, torch.Tensor) or t.get_device() != device:
            raise ValueError(f"{name}: {label} must be a CUDA tensor, on the device of the others")
        if t.dtype is not dtype:
            raise ValueError(f"{name}: {label} must be {dtype}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: {label} must be contiguous")


def _cache(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
           lengths: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(pages, KV heads, page size, sequences, pages per sequence)."""
    if k_pages.dim() != 4 or k_pages.shape[3] != 128 or v_pages.shape != k_pages.shape:
        raise ValueError(f"{name}: k_pages and v_pages must share a shape [pages, KV heads, page size, 128]")
    if page_table.dim() != 2 or lengths.shape != page_table.shape[:1]:
        raise ValueError(f"{name}: page_table must be [sequences, pages per sequence] and lengths [sequences]")
    pages, kv_heads, page_size, _ = k_pages.shape
    return pages, kv_heads, page_size, page_table.shape[0], page_table.shape[1]


def _heads(name: str, q: torch.Tensor, out: torch.Tensor, rows: int | None = None) -> int:
    if q.dim() != 3 or q.shape[2] != 128 or (rows is not None and q.shape[0] != rows):
        raise ValueError(f"{name}: q must be [{'rows' if rows is None else rows}, query heads, 128]")
    if out.shape != (q.shape[0], q.shape[1] * 128):
        raise ValueError(f"{name}: out must be [rows, query heads * 128]")
    return q.shape[1]


def _on(device: int):
    """The guard under which a call's stream, workspace and launches belong to `device`."""
    return _SAME_DEVICE if device == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(entry: str, device: int, *sizes: int) -> int:
    return int(getattr(nat.load(), entry)(*sizes))


def _workspace(device: int, entry: str, *sizes: int) -> torch.Tensor:
    """The call's own scratch, from torch's allocator: calls on other streams, and captured ones, have others."""
    return torch.empty(_workspace_bytes(entry, device, *sizes), dtype=torch.uint8, device=device)


def paged_qk_norm_rope_append(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, cos: torch.Tensor,
                              sin: torch.Tensor, cu_tokens: torch.Tensor, lengths: torch.Tensor,
                              page_table: torch.Tensor, eps: float, q_out: torch.Tensor, k_pages: torch.Tensor,
                              v_pages: torch.Tensor) -> torch.Tensor:
    """q/k RMSNorm per head, split-half rotation at every token's own position, and the append of K and V.

    qkv [rows, (Hq + 2 Hkv) * 128] (q | k | v per token), q_norm / k_norm [128], cos / sin [positions, 128]
    bf16 or fp32, q_out [rows, Hq, 128]. Computed in fp32 and rounded to bf16 once. A position past the tables
    sets device error 2, and its row is skipped.
    """
    name = "paged_qk_norm_rope_append"
    device = _device(name, k_pages)
    table = torch.float32 if getattr(cos, "dtype", None) is torch.float32 else torch.bfloat16
    _check(name, device, torch.bfloat16, k_pages=k_pages, v_pages=v_pages, qkv=qkv, q_norm=q_norm, k_norm=k_norm, q_out=q_out)
    _check(name, device, table, cos=cos, sin=sin)
    _check(name, device, torch.int32, cu_tokens=cu_tokens, lengths=lengths, page_table=page_table)
    pages, kv_heads, page_size, sequences, width = _cache(name, k_pages, v_pages, page_table, lengths)
    if q_out.dim() != 3 or q_out.shape[2] != 128 or qkv.shape != (q_out.shape[0], (q_out.shape[1] + 2 * kv_heads) * 128):
        raise ValueError(f"{name}: qkv must be [rows, (query heads + 2 * KV heads) * 128] and q_out [rows, query heads, 128]")
    if q_norm.shape != (128,) or k_norm.shape != (128,) or cos.dim() != 2 or cos.shape[1] != 128 or sin.shape != cos.shape:
        raise ValueError(f"{name}: q_norm and k_norm must be [128], cos and sin [positions, 128]")
    if cu_tokens.shape != (sequences + 1,):
        raise ValueError(f"{name}: cu_tokens must be [sequences + 1]")
    with _on(device):
        nat.call("ipe_paged_qk_norm_rope_append", qkv.data_ptr(), q_out.shape[0], q_out.shape[1], kv_heads,
                 q_norm.data_ptr(), k_norm.data_ptr(), cos.data_ptr(), sin.data_ptr(), int(table is torch.float32),
                 cos.shape[0], cu_tokens.data_ptr(), lengths.data_ptr(), page_table.data_ptr(), sequences, width,
                 q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), pages, page_size, float(eps), _stream(device))
    return q_out


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lengths: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """out [S, Hq * 128] = softmax(q k^T / sqrt(128)) v over keys 0 .. lengths[s] - 1 of every sequence, one query
    token q [S, Hq, 128] each, 1 to 8 query heads per KV head. A sequence of length 0 gives zeros."""
    name = "paged_decode_attention"
    device = _device(name, k_pages)
    _check(name, device, torch.bfloat16, k_pages=k_pages, v_pages=v_pages, q=q, out=out)
    _check(name, device, torch.int32, page_table=page_table, lengths=lengths)
    pages, kv_heads, page_size, sequences, width = _cache(name, k_pages, v_pages, page_table, lengths)
    q_heads = _heads(name, q, out, sequences)
    with _on(device):
        ws = _workspace(device, "ipe_paged_decode_attention_workspace", sequences, q_heads, kv_heads)
        nat.call("ipe_paged_decode_attention", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                 page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(), sequences, q_heads, kv_heads, pages,
                 page_size, width, ws.data_ptr(), ws.numel(), _stream(device))
    return out


def paged_prefill_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                            cu_tokens: torch.Tensor, lengths: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """Causal attention of ragged new tokens q [rows, Hq, 128] over their sequences' pages: token i of the n that
    sequence s brings sees keys 0 .. lengths[s] - n + i. out [rows, Hq * 128]; 1 to 8 query heads per KV head."""
    name = "paged_prefill_attention"
    device = _device(name, k_pages)
    _check(name, device, torch.bfloat16, k_pages=k_pages, v_pages=v_pages, q=q, out=out)
    _check(name, device, torch.int32, page_table=page_table, cu_tokens=cu_tokens, lengths=lengths)
    pages, kv_heads, page_size, sequences, width = _cache(name, k_pages, v_pages, page_table, lengths)
    q_heads = _heads(name, q, out)
    if cu_tokens.shape != (sequences + 1,):
        raise ValueError(f"{name}: cu_tokens must be [sequences + 1]")
    with _on(device):
        ws = _workspace(device, "ipe_paged_prefill_attention_workspace", q.shape[0], sequences, q_heads, kv_heads)
        nat.call("ipe_paged_prefill_attention", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                 page_table.data_ptr(), cu_tokens.data_ptr(), lengths.data_ptr(), out.data_ptr(), q.shape[0], sequences,
                 q_heads, kv_heads, pages, page_size, width, ws.data_ptr(), ws.numel(), _stream(device))
    return out


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, prefix_pages: torch.Tensor,
                            page_table: torch.Tensor, lengths: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """paged_decode_attention of sequences that begin with the same pages: position p < prefix_pages.numel() * page
    size of every sequence is in prefix_pages, whose keys are read once for the batch; page_table [S, pages per
    sequence] is read for the positions behind it alone (its first prefix_pages.numel() columns may hold anything).
    lengths [S] count the prefix; a sequence that ends inside the prefix sees its own lengths[s] keys of it."""
    name = "shared_prefix_attention"
    device = _device(name, k_pages)
    _check(name, device, torch.bfloat16, k_pages=k_pages, v_pages=v_pages, q=q, out=out)
    _check(name, device, torch.int32, prefix_pages=prefix_pages, page_table=page_table, lengths=lengths)
    pages, kv_heads, page_size, sequences, width = _cache(name, k_pages, v_pages, page_table, lengths)
    q_heads = _heads(name, q, out, sequences)
    if prefix_pages.dim() != 1 or prefix_pages.shape[0] > width:
        raise ValueError(f"{name}: prefix_pages must be [prefix pages], no more than the {width} pages per sequence")
    with _on(device):
        ws = _workspace(device, "ipe_shared_prefix_attention_workspace", sequences, q_heads, kv_heads, page_size,
                        prefix_pages.shape[0])
        nat.call("ipe_shared_prefix_attention", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                 prefix_pages.data_ptr(), prefix_pages.shape[0], page_table.data_ptr(), lengths.data_ptr(),
                 out.data_ptr(), sequences, q_heads, kv_heads, pages, page_size, width, ws.data_ptr(), ws.numel(),
                 _stream(device))
    return out
