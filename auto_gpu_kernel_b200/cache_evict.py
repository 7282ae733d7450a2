"""Eviction from the paged caches by accumulated attention weight: every request is cut down to a budget of tokens,
the heaviest ones by the weights that `paged_attention` adds up, and the kept tokens move, in order, to new pages of
the same caches (the reference has no counterpart).  Old pages are only read, so pages that requests share stay
whole; the caller frees the ones that nobody needs any more.

All tensors must be CUDA tensors on one device; there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib, workspace
from .paged_attention import PAGE, check_caches, check_tables


def _rows(name, t, batch, width, dtype, device):
    if t.dim() != 2 or t.shape[0] != batch or t.shape[1] < width or t.dtype != dtype \
            or (t.shape[1] > 1 and t.stride(1) != 1) or (batch > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"cache eviction: {name} must be [{batch},>= {width}] {dtype} with dense rows of their own")
    if t.device != device:
        raise RuntimeError(f"cache eviction: {name} must be on {device}")
    return t.data_ptr(), max(t.stride(0), t.shape[1])


def kernel(token_weights, seq_lens, block_table, new_block_table, budget, ckv_cache, kpe_cache, k_index_cache_fp8,
           new_seq_lens, new_token_weights, kept_positions, keep_first=0, keep_last=0):
    """Move the kept tokens and write `new_seq_lens` [B] int32, `new_token_weights` [B,>= budget] float32 and
    `kept_positions` [B,>= budget] int32 in place; enqueued on the current stream, returns None.

    A request of at most `budget` tokens keeps them all; a longer one keeps its first `keep_first` positions, its last
    `keep_last`, and of the others the heaviest by `token_weights` [B,>= 64*max_pages] (equal weights: the lower
    position; -inf and NaN last).  Token j of request b moves to position j of the pages new_block_table[b] with its
    ckv and kpe rows and, unless `k_index_cache_fp8` is None, its index key.  Columns up to `budget` behind the last
    kept token become 0 and -1.

    A page of new_block_table must not be one that a request of this call still reads from, unless every kept
    token on it keeps its place (a request within the budget may pass its old row: nothing moves then), and must
    not stand in it twice: such moves race."""
    if not token_weights.is_cuda:
        raise RuntimeError("cache eviction: CUDA tensors required (this operator has no CPU path)")
    dev = token_weights.device
    budget = int(budget)
    if budget < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget:
        raise ValueError("cache eviction: budget >= 1 and 0 <= keep_first + keep_last <= budget")
    batch, max_pages = check_tables("cache eviction", seq_lens, block_table, dev)
    pages = check_caches("cache eviction", ckv_cache, kpe_cache, dev)
    new_batch, new_pages = check_tables("cache eviction (new_block_table)", seq_lens, new_block_table, dev)
    if new_pages * PAGE < min(budget, max_pages * PAGE):
        raise ValueError(f"cache eviction: new_block_table has room for {new_pages * PAGE} tokens of a budget of {budget}")
    index = 0
    if k_index_cache_fp8 is not None:
        if k_index_cache_fp8.shape != (pages, PAGE, 1, 132) or k_index_cache_fp8.element_size() != 1 \
                or not k_index_cache_fp8.is_contiguous():
            raise ValueError("cache eviction: k_index_cache_fp8 must be a contiguous [P,64,1,132] int8 tensor with as many "
                             "pages as ckv_cache")
        if k_index_cache_fp8.device != dev:
            raise RuntimeError(f"cache eviction: k_index_cache_fp8 must be on {dev}")
        index = k_index_cache_fp8.data_ptr()
    if new_seq_lens.shape != (batch,) or new_seq_lens.dtype != torch.int32 or not new_seq_lens.is_contiguous() \
            or new_seq_lens.device != dev:
        raise ValueError(f"cache eviction: new_seq_lens must be a contiguous [B] int32 tensor on {dev}")
    w, w_stride = _rows("token_weights", token_weights, batch, max_pages * PAGE, torch.float32, dev)
    nw, nw_stride = _rows("new_token_weights", new_token_weights, batch, budget, torch.float32, dev)
    kept, kept_stride = _rows("kept_positions", kept_positions, batch, budget, torch.int32, dev)
    if workspace.overlap(token_weights, new_token_weights) or workspace.overlap(seq_lens, new_seq_lens):
        raise ValueError("cache eviction: the outputs must not overlap the inputs")
    if batch == 0:
        return None
    if max_pages == 0:
        new_seq_lens.zero_()
        new_token_weights[:, :budget].zero_()
        kept_positions[:, :budget].fill_(-1)
        return None
    lib = _lib.load()
    with workspace.device_guard(dev):
        rc = lib.dsa_cache_evict(
            w, w_stride, seq_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), new_block_table.data_ptr(),
            new_block_table.stride(0), ckv_cache.data_ptr(), kpe_cache.data_ptr(), index, new_seq_lens.data_ptr(), nw,
            nw_stride, kept, kept_stride, batch, max_pages, new_pages, pages, budget, int(keep_first), int(keep_last),
            workspace.status_word(dev).data_ptr(), workspace.stream_handle(dev))
    _lib.check(rc, "dsa_cache_evict")
    return None


def run(token_weights, seq_lens, block_table, new_block_table, budget, ckv_cache, kpe_cache, k_index_cache_fp8=None,
        keep_first=0, keep_last=0, new_seq_lens=None, new_token_weights=None, kept_positions=None):
    """Value-returning form: allocates the outputs that are not passed; returns (new_seq_lens, new_token_weights,
    kept_positions)."""
    batch, dev = seq_lens.shape[0], seq_lens.device
    if new_seq_lens is None:
        new_seq_lens = torch.empty(batch, dtype=torch.int32, device=dev)
    if new_token_weights is None:
        new_token_weights = torch.empty(batch, budget, dtype=torch.float32, device=dev)
    if kept_positions is None:
        kept_positions = torch.empty(batch, budget, dtype=torch.int32, device=dev)
    kernel(token_weights, seq_lens, block_table, new_block_table, budget, ckv_cache, kpe_cache, k_index_cache_fp8,
           new_seq_lens, new_token_weights, kept_positions, keep_first, keep_last)
    return new_seq_lens, new_token_weights, kept_positions
