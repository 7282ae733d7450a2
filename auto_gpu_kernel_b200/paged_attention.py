"""Dense MLA attention of every request's newest tokens over its whole paged cache: what a layer runs that has no
indexer, a context too short for one, or drafted tokens that are verified together.  The caches are those of
`sparse_attention`, addressed by the indexer's block table (the reference has no counterpart; its attention reads a
list of slots: archive/dsa_sparse_attention_h16_ckv512_kpe64_topk2048_ps64/solution/triton/sparse_baseline.py:12-45,
whose softmax, base-2 LSE and rounding are kept here).

All tensors must be CUDA tensors on one device; there is no CPU path.  With `new_token_weights` the call also adds
up how much attention every cached token received, which `cache_evict` chooses by.
"""
from __future__ import annotations

import functools

import torch

from . import _lib, workspace

CKV = 512
KPE = 64
PAGE = 64
MAX_HEADS = 128


def tables_ok(seq_lens, block_table, index):
    """seq_lens [B] and block_table [B,max_pages], int32 on the device of this index, as every operator here takes them."""
    return (block_table.dim() == 2 and block_table.dtype is torch.int32 and seq_lens.dtype is torch.int32
            and seq_lens.dim() == 1 and seq_lens.shape[0] == block_table.shape[0] and seq_lens.is_contiguous()
            and (block_table.stride(1) == 1 or block_table.shape[1] <= 1)
            and seq_lens.get_device() == index and block_table.get_device() == index)


def refuse_tables(what, seq_lens, block_table, index):
    """Say what `tables_ok` found wrong."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"{what}: block_table must be [B,max_pages] int32")
    if seq_lens.shape != block_table.shape[:1] or seq_lens.dtype != torch.int32 or not seq_lens.is_contiguous():
        raise ValueError(f"{what}: seq_lens must be a contiguous [B] int32 tensor")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError(f"{what}: block_table rows must be dense (stride(1) == 1)")
    raise RuntimeError(f"{what}: seq_lens and block_table must be on cuda:{index}")


def caches_ok(ckv_cache, kpe_cache, index):
    """The two paged caches, contiguous [P,64,512] and [P,64,64] bf16."""
    c, k = ckv_cache.shape, kpe_cache.shape
    return (len(c) == 3 and c[1] == PAGE and c[2] == CKV and len(k) == 3 and k[0] == c[0] and k[1] == PAGE and k[2] == KPE
            and ckv_cache.dtype is torch.bfloat16 and kpe_cache.dtype is torch.bfloat16 and ckv_cache.is_contiguous()
            and kpe_cache.is_contiguous() and ckv_cache.get_device() == index and kpe_cache.get_device() == index)


def refuse_caches(what, ckv_cache, kpe_cache, index):
    """Say what `caches_ok` found wrong."""
    if ckv_cache.dim() != 3 or ckv_cache.shape[1:] != (PAGE, CKV) or ckv_cache.dtype != torch.bfloat16 \
            or not ckv_cache.is_contiguous():
        raise ValueError(f"{what}: ckv_cache must be a contiguous [P,64,512] bf16 tensor")
    if kpe_cache.shape != (ckv_cache.shape[0], PAGE, KPE) or kpe_cache.dtype != torch.bfloat16 \
            or not kpe_cache.is_contiguous():
        raise ValueError(f"{what}: kpe_cache must be a contiguous [P,64,64] bf16 tensor with as many pages as ckv_cache")
    raise RuntimeError(f"{what}: the caches must be on cuda:{index}")


def rows_of(what, name, t, batch, width, dtype, index):
    """(address, row stride) of a [batch,>= width] tensor with dense rows of their own."""
    if t.dim() != 2 or t.dtype is not dtype or t.shape[0] != batch or t.shape[1] < width \
            or (t.stride(1) != 1 and t.shape[1] > 1) or (batch > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{what}: {name} must be [{batch},>= {width}] {dtype} with dense rows of their own")
    if t.get_device() != index:
        raise RuntimeError(f"{what}: {name} must be on cuda:{index}")
    return t.data_ptr(), max(t.stride(0), t.shape[1])


def _refuse(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table):
    what = "paged attention"
    if not q_nope.is_cuda:
        raise RuntimeError(f"{what}: CUDA tensors required (this operator has no CPU path)")
    index = q_nope.get_device()
    if not tables_ok(seq_lens, block_table, index):
        refuse_tables(what, seq_lens, block_table, index)
    if not caches_ok(ckv_cache, kpe_cache, index):
        refuse_caches(what, ckv_cache, kpe_cache, index)
    if q_nope.dim() != 3 or q_nope.shape[2] != CKV or q_nope.dtype != torch.bfloat16:
        raise ValueError(f"{what}: q_nope must be [B*n,heads,512] bf16")
    rows, heads, _ = q_nope.shape
    if not 1 <= heads <= MAX_HEADS:
        raise ValueError(f"{what}: 1 to {MAX_HEADS} heads, got {heads}")
    if q_pe.shape != (rows, heads, KPE) or q_pe.dtype != torch.bfloat16:
        raise ValueError(f"{what}: q_pe must be [B*n,heads,64] bf16")
    if not (q_nope.is_contiguous() and q_pe.is_contiguous()):
        raise ValueError(f"{what}: q_nope and q_pe must be contiguous")
    raise RuntimeError(f"{what}: q_pe must be on cuda:{index}")


def _check_output(name, t, shape, dtype, index):
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        raise ValueError(f"paged attention: {name} must be a contiguous {list(shape)} {dtype} tensor")
    if t.get_device() != index:
        raise RuntimeError(f"paged attention: {name} must be on cuda:{index}")


@functools.lru_cache(maxsize=512)
def _workspace_bytes(index, batch, tokens, heads, max_pages, with_weights):
    with torch.cuda.device(index):
        return _lib.load().dsa_paged_attn_workspace_bytes(batch, tokens, heads, max_pages, with_weights)


def _attend(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output, lse, token_weights,
            new_token_weights):
    shape, index = q_nope.shape, q_nope.get_device()
    bf16 = torch.bfloat16
    if not (index >= 0 and len(shape) == 3 and shape[2] == CKV and 1 <= shape[1] <= MAX_HEADS
            and q_pe.shape == (shape[0], shape[1], KPE) and q_nope.dtype is bf16 and q_pe.dtype is bf16
            and q_nope.is_contiguous() and q_pe.is_contiguous() and q_pe.get_device() == index
            and tables_ok(seq_lens, block_table, index) and caches_ok(ckv_cache, kpe_cache, index)):
        _refuse(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table)
    if output is None:
        output = q_nope.new_empty((shape[0], shape[1], CKV))
    else:
        _check_output("output", output, shape, bf16, index)
    if lse is None:
        lse = q_nope.new_empty((shape[0], shape[1]), dtype=torch.float32)
    else:
        _check_output("lse", lse, shape[:2], torch.float32, index)
    rows, heads, _ = shape
    batch, max_pages = block_table.shape
    if rows == 0:
        if batch and new_token_weights is not None:
            raise ValueError(f"paged attention: no query tokens whose weights {batch} requests could receive")
        return output, lse
    if batch == 0 or rows % batch:
        raise ValueError(f"paged attention: {rows} query tokens are no multiple of the {batch} requests")
    old = new = old_stride = new_stride = 0
    if new_token_weights is not None:
        new, new_stride = rows_of("paged attention", "new_token_weights", new_token_weights, batch, max_pages * PAGE,
                                  torch.float32, index)
    if token_weights is not None:
        if new_token_weights is None:
            raise ValueError("paged attention: token_weights without new_token_weights")
        old, old_stride = rows_of("paged attention", "token_weights", token_weights, batch, max_pages * PAGE, torch.float32,
                                  index)
    if max_pages == 0:
        output.zero_()
        lse.fill_(float("-inf"))
        return output, lse
    lib = _lib.load()
    tokens = rows // batch
    need = _workspace_bytes(index, batch, tokens, heads, max_pages, 1 if new else 0)
    # a buffer of the call's own: torch's allocator orders it by stream and by graph
    scratch = torch.empty(need, dtype=torch.uint8, device=q_nope.device)
    rc = workspace.call_on(
        index, lib.dsa_paged_attn, q_nope.data_ptr(), q_pe.data_ptr(), ckv_cache.data_ptr(), kpe_cache.data_ptr(),
        seq_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), float(sm_scale), output.data_ptr(), lse.data_ptr(), old,
        old_stride, new, new_stride, batch, tokens, heads, ckv_cache.shape[0], max_pages, scratch.data_ptr(), need)
    if rc:
        _lib.check(rc, "dsa_paged_attn")
    return output, lse


def kernel(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output, lse, token_weights=None,
           new_token_weights=None):
    """Write the attention output and the base-2 LSE in place; enqueued on the current stream, returns None.

    q_nope [B*n,heads,512] / q_pe [B*n,heads,64] bf16: the n newest tokens of every request, oldest first (1 to 128
    heads).  `seq_lens` counts the cached tokens of each request, the new ones among them: token i of n sees the
    positions below seq_len - n + 1 + i, and one that sees none gets output 0 and lse -inf.  Cache rows at or
    behind seq_len may hold anything, those in front of it must be finite.  Outputs that share memory
    with an input or with one another are refused.  Logits, sums, lse and accumulated weights are fp32; the softmax weights
    are rounded to bf16 for their product with the bf16 cache, an error of the size of the output's own rounding.

    `new_token_weights` [B,>= 64*max_pages] float32 receives, for every position below seq_len, `token_weights` (same
    shape; None = zeros; may be the same tensor) plus the softmax weight the position got from all query rows of
    its request; other entries stay as they were.  The call's scratch then holds the logits, 256 bytes per query row
    and page of the table, so a table much wider than its lengths costs memory (calls on a few requests at a time hold
    less at once)."""
    if output is None or lse is None:
        raise ValueError("paged attention: kernel() needs output and lse")
    _attend(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output, lse, token_weights, new_token_weights)


def run(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output=None, lse=None, token_weights=None,
        new_token_weights=None):
    """Value-returning form: allocates the outputs that are not passed; returns (output, lse)."""
    return _attend(q_nope, q_pe, ckv_cache, kpe_cache, seq_lens, block_table, sm_scale, output, lse, token_weights,
                   new_token_weights)
