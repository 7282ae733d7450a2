"""Eviction from the paged caches by accumulated attention weight: every request is cut down to a budget of tokens,
the heaviest ones by the weights that `paged_attention` adds up, and the kept tokens move, in order, to new pages of
the same caches (the reference has no counterpart).  Old pages are only read, so pages that requests share stay
whole; the caller frees the ones that nobody needs any more.

All tensors must be CUDA tensors on one device; there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib, workspace
from .paged_attention import PAGE, caches_ok, refuse_caches, refuse_tables, rows_of, tables_ok

MAX_BUDGET = 1 << 30


def _evict(token_weights, seq_lens, block_table, new_block_table, budget, ckv_cache, kpe_cache, k_index_cache_fp8,
           new_seq_lens, new_token_weights, kept_positions, keep_first, keep_last):
    what = "cache eviction"
    if not token_weights.is_cuda:
        raise RuntimeError(f"{what}: CUDA tensors required (this operator has no CPU path)")
    index = token_weights.get_device()
    budget = int(budget)
    if not 1 <= budget <= MAX_BUDGET or keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget:
        raise ValueError(f"{what}: 1 <= budget <= 2^30 and 0 <= keep_first + keep_last <= budget")
    if not tables_ok(seq_lens, block_table, index):
        refuse_tables(what, seq_lens, block_table, index)
    if not tables_ok(seq_lens, new_block_table, index):
        refuse_tables(f"{what} (new_block_table)", seq_lens, new_block_table, index)
    if not caches_ok(ckv_cache, kpe_cache, index):
        refuse_caches(what, ckv_cache, kpe_cache, index)
    batch, max_pages = block_table.shape
    pages, new_pages = ckv_cache.shape[0], new_block_table.shape[1]
    if new_pages * PAGE < min(budget, max_pages * PAGE):
        raise ValueError(f"{what}: new_block_table has room for {new_pages * PAGE} tokens of a budget of {budget}")
    keys = 0
    if k_index_cache_fp8 is not None:
        if k_index_cache_fp8.shape != (pages, PAGE, 1, 132) or k_index_cache_fp8.element_size() != 1 \
                or not k_index_cache_fp8.is_contiguous():
            raise ValueError(f"{what}: k_index_cache_fp8 must be a contiguous [P,64,1,132] int8 tensor with as many pages "
                             "as ckv_cache")
        if k_index_cache_fp8.get_device() != index:
            raise RuntimeError(f"{what}: k_index_cache_fp8 must be on cuda:{index}")
        keys = k_index_cache_fp8.data_ptr()
    w, w_stride = rows_of(what, "token_weights", token_weights, batch, max_pages * PAGE, torch.float32, index)
    if new_seq_lens is None:
        new_seq_lens = seq_lens.new_empty((batch,))
    elif new_seq_lens.dim() != 1 or new_seq_lens.shape[0] != batch or new_seq_lens.dtype is not torch.int32 \
            or not new_seq_lens.is_contiguous() or new_seq_lens.get_device() != index:
        raise ValueError(f"{what}: new_seq_lens must be a contiguous [B] int32 tensor on cuda:{index}")
    if new_token_weights is None:
        new_token_weights = token_weights.new_empty((batch, budget))
        nw, nw_stride = new_token_weights.data_ptr(), budget
    else:
        nw, nw_stride = rows_of(what, "new_token_weights", new_token_weights, batch, budget, torch.float32, index)
    if kept_positions is None:
        kept_positions = seq_lens.new_empty((batch, budget))
        kept, kept_stride = kept_positions.data_ptr(), budget
    else:
        kept, kept_stride = rows_of(what, "kept_positions", kept_positions, batch, budget, torch.int32, index)
    if batch == 0:
        return new_seq_lens, new_token_weights, kept_positions
    if max_pages == 0:
        new_seq_lens.zero_()
        new_token_weights[:, :budget].zero_()
        kept_positions[:, :budget].fill_(-1)
        return new_seq_lens, new_token_weights, kept_positions
    lib = _lib.load()
    rc = workspace.call_on(
        index, lib.dsa_cache_evict, w, w_stride, seq_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0),
        new_block_table.data_ptr(), new_block_table.stride(0), ckv_cache.data_ptr(), kpe_cache.data_ptr(), keys,
        new_seq_lens.data_ptr(), nw, nw_stride, kept, kept_stride, batch, max_pages, new_pages, pages, budget,
        int(keep_first), int(keep_last))
    if rc:
        _lib.check(rc, "dsa_cache_evict")
    return new_seq_lens, new_token_weights, kept_positions


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
    not stand in it twice: such moves race.  Outputs that share memory with an input, a cache or one another are
    refused."""
    if new_seq_lens is None or new_token_weights is None or kept_positions is None:
        raise ValueError("cache eviction: kernel() needs its three outputs")
    _evict(token_weights, seq_lens, block_table, new_block_table, budget, ckv_cache, kpe_cache, k_index_cache_fp8, new_seq_lens,
           new_token_weights, kept_positions, keep_first, keep_last)


def run(token_weights, seq_lens, block_table, new_block_table, budget, ckv_cache, kpe_cache, k_index_cache_fp8=None,
        keep_first=0, keep_last=0, new_seq_lens=None, new_token_weights=None, kept_positions=None):
    """Value-returning form: allocates the outputs that are not passed; returns (new_seq_lens, new_token_weights,
    kept_positions)."""
    return _evict(token_weights, seq_lens, block_table, new_block_table, budget, ckv_cache, kpe_cache, k_index_cache_fp8,
                  new_seq_lens, new_token_weights, kept_positions, keep_first, keep_last)
