"""Dense MLA attention of every request's newest tokens over its whole paged cache: what a layer runs that has no
indexer, a context too short for one, or drafted tokens that are verified together.  The caches are those of
`sparse_attention`, addressed by the indexer's block table (the reference has no counterpart; its attention reads a
list of slots: archive/dsa_sparse_attention_h16_ckv512_kpe64_topk2048_ps64/solution/triton/sparse_baseline.py:12-45,
whose softmax, base-2 LSE and rounding are kept here).

All tensors must be CUDA tensors on one device; there is no CPU path.  With `new_token_weights` the call also adds
up how much attention every cached token received, which `cache_evict` chooses by.
"""
from __future__ import annotations

import torch

from . import _lib, workspace

CKV = 512
KPE = 64
PAGE = 64
MAX_HEADS = 128


def check_tables(what, seq_lens, block_table, device):
    """Checks shared by the operators that walk a block table; returns (batch, max_pages)."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"{what}: block_table must be [B,max_pages] int32")
    batch, max_pages = block_table.shape
    if seq_lens.shape != (batch,) or seq_lens.dtype != torch.int32 or not seq_lens.is_contiguous():
        raise ValueError(f"{what}: seq_lens must be a contiguous [B] int32 tensor")
    if max_pages > 1 and block_table.stride(1) != 1:
        raise ValueError(f"{what}: block_table rows must be dense (stride(1) == 1)")
    if seq_lens.device != device or block_table.device != device:
        raise RuntimeError(f"{what}: seq_lens and block_table must be on {device}")
    return batch, max_pages


def check_caches(what, ckv_cache, kpe_cache, device):
    """The two paged caches, [P,64,512] and [P,64,64] bf16; returns P."""
    if ckv_cache.dim() != 3 or ckv_cache.shape[1:] != (PAGE, CKV) or ckv_cache.dtype != torch.bfloat16 \
            or not ckv_cache.is_contiguous():
        raise ValueError(f"{what}: ckv_cache must be a contiguous [P,64,512] bf16 tensor")
    pages = ckv_cache.shape[0]
    if kpe_cache.shape != (pages, PAGE, KPE) or kpe_cache.dtype != torch.bfloat16 or not kpe_cache.is_contiguous():
        raise ValueError(f"{what}: kpe_cache must be a contiguous [P,64,64] bf16 tensor with as many pages as ckv_cache")
    if ckv_cache.device != device or kpe_cache.device != device:
        raise RuntimeError(f"{what}: the caches must be on {device}")
    return pages


def _check_weights(name, t, batch, width, device):
    if t.dim() != 2 or t.shape[0] != batch or t.shape[1] < width or t.dtype != torch.float32 \
            or (t.shape[1] > 1 and t.stride(1) != 1) or (batch > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"paged attention: {name} must be [B,>= 64*max_pages] float32 with dense rows of their own")
    if t.device != device:
        raise RuntimeError(f"paged attention: {name} must be on {device}")


def kernel(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output, lse, token_weights=None,
           new_token_weights=None):
    """Write the attention output and the base-2 LSE in place; enqueued on the current stream, returns None.

    q_nope [B*n,heads,512] / q_pe [B*n,heads,64] bf16: the n newest tokens of every request, oldest first (1 to 128
    heads).  `seq_lens` counts the cached tokens of each request, the new ones among them: token i of n sees the
    positions below seq_len - n + 1 + i, and one that sees none gets output 0 and lse -inf.  Cache rows at or
    behind seq_len may hold anything, those in front of it must be finite.

    `new_token_weights` [B,>= 64*max_pages] float32 receives, for every position below seq_len, `token_weights` (same
    shape; None = zeros; may be the same tensor) plus the softmax weight the position got from all query rows of
    its request; other entries stay as they were."""
    if not q_nope.is_cuda:
        raise RuntimeError("paged attention: CUDA tensors required (this operator has no CPU path)")
    dev = q_nope.device
    batch, max_pages = check_tables("paged attention", seq_lens, block_table, dev)
    pages = check_caches("paged attention", ckv_cache, kpe_cache, dev)
    if q_nope.dim() != 3 or q_nope.shape[2] != CKV or q_nope.dtype != torch.bfloat16:
        raise ValueError("paged attention: q_nope must be [B*n,heads,512] bf16")
    rows, heads, _ = q_nope.shape
    if not 1 <= heads <= MAX_HEADS:
        raise ValueError(f"paged attention: 1 to {MAX_HEADS} heads, got {heads}")
    if q_pe.shape != (rows, heads, KPE) or q_pe.dtype != torch.bfloat16:
        raise ValueError("paged attention: q_pe must be [B*n,heads,64] bf16")
    if output.shape != q_nope.shape or output.dtype != torch.bfloat16 or lse.shape != (rows, heads) \
            or lse.dtype != torch.float32:
        raise ValueError("paged attention: output must be [B*n,heads,512] bf16 and lse [B*n,heads] float32")
    if not (q_nope.is_contiguous() and q_pe.is_contiguous() and output.is_contiguous() and lse.is_contiguous()):
        raise ValueError("paged attention: q_nope, q_pe, output and lse must be contiguous")
    if q_pe.device != dev or output.device != dev or lse.device != dev:
        raise RuntimeError(f"paged attention: all tensors must be on {dev}")
    if rows == 0:
        return None
    if batch == 0 or rows % batch:
        raise ValueError(f"paged attention: {rows} query tokens are no multiple of the {batch} requests")
    old = new = old_stride = new_stride = 0
    if new_token_weights is not None:
        _check_weights("new_token_weights", new_token_weights, batch, max_pages * PAGE, dev)
        new, new_stride = new_token_weights.data_ptr(), max(new_token_weights.stride(0), new_token_weights.shape[1])
    if token_weights is not None:
        if new_token_weights is None:
            raise ValueError("paged attention: token_weights without new_token_weights")
        _check_weights("token_weights", token_weights, batch, max_pages * PAGE, dev)
        old, old_stride = token_weights.data_ptr(), max(token_weights.stride(0), token_weights.shape[1])
        if old != new and workspace.overlap(token_weights, new_token_weights) or old == new and old_stride != new_stride:
            raise ValueError("paged attention: token_weights and new_token_weights overlap without being one tensor")
    if max_pages == 0:
        output.zero_()
        lse.fill_(float("-inf"))
        return None
    lib = _lib.load()
    tokens = rows // batch
    with workspace.device_guard(dev):
        need = lib.dsa_paged_attn_workspace_bytes(batch, tokens, heads, max_pages, new_token_weights is not None)
        # a buffer of the call's own: torch's allocator orders it by stream and by graph
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        rc = lib.dsa_paged_attn(
            q_nope.data_ptr(), q_pe.data_ptr(), ckv_cache.data_ptr(), kpe_cache.data_ptr(), seq_lens.data_ptr(),
            block_table.data_ptr(), block_table.stride(0), float(sm_scale), output.data_ptr(), lse.data_ptr(), old,
            old_stride, new, new_stride, batch, tokens, heads, pages, max_pages, scratch.data_ptr(), need,
            workspace.status_word(dev).data_ptr(), workspace.stream_handle(dev))
    _lib.check(rc, "dsa_paged_attn")
    return None


def run(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output=None, lse=None, token_weights=None,
        new_token_weights=None):
    """Value-returning form: allocates the outputs that are not passed; returns (output, lse)."""
    if output is None:
        output = torch.empty_like(q_nope, memory_format=torch.contiguous_format)
    if lse is None:
        lse = torch.empty(q_nope.shape[:2], dtype=torch.float32, device=q_nope.device)
    kernel(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output, lse, token_weights,
           new_token_weights)
    return output, lse
