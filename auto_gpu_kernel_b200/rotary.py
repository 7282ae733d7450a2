"""Rotary positions with several axes (time, height, width ..) on the queries and the new keys of a step, and the
append of the keys: the step in front of both attentions, whose inputs arrive rotated (the reference has no
counterpart; the cache rows are those of `cache_write.append_kv`).

CUDA tensors only; enqueued on the current stream.
"""
from __future__ import annotations

import functools

import torch

from . import _lib, workspace

PAIRS = 32


def sections(*counts):
    """Axis of every pair when the axes take consecutive runs of pairs: sections(16, 8, 8) gives the first 16 pairs to
    axis 0, the next 8 to axis 1 and the last 8 to axis 2."""
    if sum(counts) != PAIRS or min(counts, default=0) < 0:
        raise ValueError(f"rotary: sections must add up to {PAIRS} pairs, got {counts}")
    return [axis for axis, n in enumerate(counts) for _ in range(n)]


def _axis_bytes(pair_axes):
    """A byte per pair, from any sequence of whole numbers (by way of a list: bytes() of an array would be its buffer, of a
    number as many zeros)."""
    try:
        return bytes(list(pair_axes))
    except TypeError:
        raise ValueError(f"rotary: pair_axes must be {PAIRS} axis numbers") from None


@functools.lru_cache(maxsize=64)
def _pack(pair_axes, axes):
    """The axes (a byte per pair) in two bits each."""
    if len(pair_axes) != PAIRS:
        raise ValueError(f"rotary: pair_axes must have {PAIRS} entries")
    packed = 0
    for i, axis in enumerate(pair_axes):
        if axis >= axes:
            raise ValueError(f"rotary: pair {i} asks for axis {axis} of {axes}")
        packed |= axis << (2 * i)
    return packed


def _refuse(q_pe, ckv, kpe, positions, inv_freq, slots, ckv_cache, kpe_cache):
    if not q_pe.is_cuda:
        raise RuntimeError("rotary: CUDA tensors required (no CPU path)")
    bf16, i32 = torch.bfloat16, torch.int32
    if q_pe.dim() != 3 or q_pe.shape[2] != 64 or q_pe.dtype is not bf16 or q_pe.stride(2) != 1:
        raise ValueError("rotary: q_pe must be [n,heads,64] bf16 with dense rows")
    n, heads, _ = q_pe.shape
    if not 1 <= heads <= 128:
        raise ValueError(f"rotary: 1 to 128 heads, got {heads}")
    if ckv.shape != (n, 512) or kpe.shape != (n, 64) or ckv.dtype is not bf16 or kpe.dtype is not bf16 \
            or ckv.stride(1) != 1 or kpe.stride(1) != 1:
        raise ValueError("rotary: ckv must be [n,512] and kpe [n,64], bf16 with dense rows")
    if positions.dim() != 2 or not 1 <= positions.shape[0] <= 4 or positions.shape[1] != n \
            or positions.dtype is not i32 or (n > 1 and positions.stride(1) != 1):
        raise ValueError("rotary: positions must be [axes,n] int32 with one to four axes and dense rows")
    if inv_freq.shape != (PAIRS,) or inv_freq.dtype is not torch.float32 or not inv_freq.is_contiguous():
        raise ValueError("rotary: inv_freq must be a contiguous [32] float32 tensor")
    if slots.shape != (n,) or slots.dtype is not i32 or not slots.is_contiguous():
        raise ValueError("rotary: slots must be a contiguous [n] int32 tensor")
    if ckv_cache.shape[-1] != 512 or kpe_cache.shape[-1] != 64 or not ckv_cache.is_contiguous() \
            or not kpe_cache.is_contiguous() or ckv_cache.dtype is not bf16 or kpe_cache.dtype is not bf16:
        raise ValueError("rotary: caches must be contiguous bf16 [...,512] / [...,64]")
    if ckv_cache.numel() != 8 * kpe_cache.numel():
        raise ValueError("rotary: ckv_cache and kpe_cache hold different numbers of slots")
    raise RuntimeError(f"rotary: all tensors must be on {q_pe.device}")


def append(q_pe, ckv, kpe, positions, inv_freq, pair_axes, slots, ckv_cache, kpe_cache, q_out=None, interleaved=False):
    """Rotate `q_pe` [n,heads,64] (bf16, strided token and head rows allowed, 1 to 128 heads) into `q_out` (contiguous;
    allocated when None; may be q_pe itself where that is contiguous) and return it; rotate `kpe` [n,64] and store it
    with `ckv` [n,512] at global slot `slots[t]` of the paged caches [P,64,512] / [P,64,64] (-1 skips the token's
    cache rows; two equal slots race).  `q_out` over any other argument and caches over one another are refused; `ckv`
    and `kpe` may be rows of the caches that no slot of the call names.

    Pair i of token t turns by positions[pair_axes[i], t] * inv_freq[i]: `positions` [axes,n] int32 with one to four axes
    (rows may be expanded),
    `inv_freq` [32] float32, `pair_axes` 32 axis numbers (see `sections`).  A pair is (2i, 2i+1) when `interleaved`,
    else (i, i+32)."""
    index, bf16 = q_pe.get_device(), torch.bfloat16
    shape = q_pe.shape
    n = shape[0] if len(shape) == 3 else -1
    if not (index >= 0 and len(shape) == 3 and shape[2] == 64 and 1 <= shape[1] <= 128 and q_pe.dtype is bf16
            and q_pe.stride(2) == 1 and ckv.shape == (n, 512) and kpe.shape == (n, 64) and ckv.dtype is bf16
            and kpe.dtype is bf16 and ckv.stride(1) == 1 and kpe.stride(1) == 1
            and positions.dim() == 2 and 1 <= positions.shape[0] <= 4 and positions.shape[1] == n
            and positions.dtype is torch.int32 and (positions.stride(1) == 1 or n <= 1)
            and inv_freq.shape == (PAIRS,) and inv_freq.dtype is torch.float32 and inv_freq.is_contiguous()
            and slots.shape == (n,) and slots.dtype is torch.int32 and slots.is_contiguous()
            and ckv_cache.shape[-1] == 512 and kpe_cache.shape[-1] == 64 and ckv_cache.dtype is bf16 and kpe_cache.dtype is bf16
            and ckv_cache.is_contiguous() and kpe_cache.is_contiguous() and ckv_cache.numel() == 8 * kpe_cache.numel()
            and ckv.get_device() == kpe.get_device() == positions.get_device() == inv_freq.get_device() == slots.get_device()
            == ckv_cache.get_device() == kpe_cache.get_device() == index):
        _refuse(q_pe, ckv, kpe, positions, inv_freq, slots, ckv_cache, kpe_cache)
    heads, axes, num_slots = shape[1], positions.shape[0], ckv_cache.numel() // 512
    packed = _pack(_axis_bytes(pair_axes), axes)
    if q_out is None:
        q_out = q_pe.new_empty((n, heads, 64))
    elif q_out.shape != shape or q_out.dtype is not bf16 or not q_out.is_contiguous():
        raise ValueError("rotary: q_out must be a contiguous [n,heads,64] bf16 tensor")
    elif q_out.get_device() != index:
        raise RuntimeError(f"rotary: all tensors must be on cuda:{index}")
    if n == 0:
        return q_out
    # the stride of an axis of one entry says nothing
    one = n == 1
    lib = _lib.load()
    rc = workspace.call_on(
        index, lib.dsa_rotary_append, q_pe.data_ptr(), heads * 64 if one else q_pe.stride(0),
        64 if heads == 1 else q_pe.stride(1), ckv.data_ptr(), 512 if one else ckv.stride(0), kpe.data_ptr(),
        64 if one else kpe.stride(0), positions.data_ptr(), n if axes == 1 else positions.stride(0), axes,
        inv_freq.data_ptr(), packed, 1 if interleaved else 0, slots.data_ptr(), q_out.data_ptr(), ckv_cache.data_ptr(),
        kpe_cache.data_ptr(), n, heads, num_slots)
    if rc:
        _lib.check(rc, "dsa_rotary_append")
    return q_out
