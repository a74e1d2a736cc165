"""Torch-tensor front end of the C-ABI kernels.

Each function validates shapes on the host, passes raw device pointers and the
current CUDA stream to libmlxz_b200.so, and returns without synchronising.
Kernels report out-of-range block ids, slots and context lengths through a
per-device int32 error word instead of trapping; ``check_device_errors`` reads
and clears it (``MLXZ_B200_DEBUG=1`` makes every call check it).
"""
from __future__ import annotations

import ctypes
import math
import os
from collections import OrderedDict
from typing import NamedTuple

import torch

from . import _native as nat

_DTYPES = {torch.float16: nat.MZ_DTYPE_F16, torch.bfloat16: nat.MZ_DTYPE_BF16,
           torch.float32: nat.MZ_DTYPE_F32}
_DEBUG = os.environ.get("MLXZ_B200_DEBUG", "0") not in ("", "0")

_F32_TINY = torch.finfo(torch.float32).tiny

_err_words: dict[int, torch.Tensor] = {}
# Decode workspaces handed out when the caller passes none, one per exact
# problem layout.  The kernels need the arrival counters and scheduler words at
# the front of a workspace to be zero at launch (each launch leaves them zero),
# and where those words sit depends on the problem sizes: a workspace last used
# with other sizes may hold partials there.  So a workspace is never shared
# between layouts.  A few layouts are kept, least recently used dropped first.
_WS_KEEP = 16
_workspaces: "OrderedDict[tuple, torch.Tensor]" = OrderedDict()
_qworkspaces: "OrderedDict[tuple, torch.Tensor]" = OrderedDict()


def _layout_workspace(cache, key: tuple, need: int, device: int, shared: bool) -> torch.Tensor:
    if not shared:
        if torch.cuda.is_current_stream_capturing():
            # its clearing runs with every replay: the counters at the front alone
            ws = torch.empty(max(need, 256), dtype=torch.uint8, device=f"cuda:{device}")
            ws[:4 * (key[1] * key[2] + 2)].zero_()
            return ws
        return torch.zeros(max(need, 256), dtype=torch.uint8, device=f"cuda:{device}")
    ws = cache.get(key)
    if ws is None:
        ws = torch.zeros(max(need, 256), dtype=torch.uint8, device=f"cuda:{device}")
        cache[key] = ws
        while len(cache) > _WS_KEEP:
            cache.popitem(last=False)
    else:
        cache.move_to_end(key)
    return ws


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPES[dt]
    except KeyError:
        raise ValueError(f"unsupported dtype {dt}") from None


def _dev_index(t: torch.Tensor) -> int:
    if t.device.type != "cuda":
        raise ValueError(f"expected a CUDA tensor, got one on {t.device}")
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def _stream(device: int) -> int:
    # the raw handle, without building a torch.cuda.Stream (2 us a call)
    return torch._C._cuda_getCurrentRawStream(device)


def error_word(device: int) -> torch.Tensor:
    """The int32 device error word kernels on `device` report into."""
    w = _err_words.get(device)
    if w is None:
        w = torch.zeros(1, dtype=torch.int32, device=f"cuda:{device}")
        _err_words[device] = w
    return w


def check_device_errors(device: int | None = None, clear: bool = True) -> int:
    """Synchronise with `device`'s error word; raise DeviceError if a bit is set."""
    device = torch.cuda.current_device() if device is None else device
    w = _err_words.get(device)
    if w is None:
        return 0
    bits = int(w.item())
    if bits and clear:
        w.zero_()
    if bits:
        raise nat.DeviceError(bits)
    return 0


def _after(device: int) -> None:
    if _DEBUG:
        check_device_errors(device)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _at(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _call(device: int, name: str, *args) -> None:
    """nat.call_packed with the error word and the current stream behind ``args``, and
    ``device`` current: a launch goes to the current device, which need not be
    the tensors' own."""
    err = error_word(device).data_ptr()
    if torch._C._cuda_getDevice() == device:
        nat.call_packed(name, *args, err, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            nat.call_packed(name, *args, err, _stream(device))
    if _DEBUG:
        check_device_errors(device)


def _i32_on(t: torch.Tensor, dev: int) -> bool:
    return t.dtype is torch.int32 and t.get_device() == dev and t.is_contiguous()


def _check_pools(k_pool: torch.Tensor, v_pool: torch.Tensor) -> tuple[int, int, int, int]:
    shape = k_pool.shape
    if shape != v_pool.shape or k_pool.dtype is not v_pool.dtype:
        raise ValueError("k_pool and v_pool must have the same shape and dtype")
    if len(shape) != 4 or not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise ValueError("pools must be contiguous [n_blocks, n_kv_heads, block_size, head_dim]")
    if k_pool.get_device() != v_pool.get_device():
        raise ValueError("pools must be on the same device")
    n, h, bs, d = shape
    return n, h, bs, d


def _as_i32(t: torch.Tensor, device: torch.device, name: str) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on {device}")
    return t


# ---------------------------------------------------------------------------
# Append / gather
# ---------------------------------------------------------------------------

def kv_append(k_pool: torch.Tensor, v_pool: torch.Tensor, keys: torch.Tensor,
              values: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Write keys/values ``(1, H, n, D)`` (or ``(H, n, D)``) to pool slots.

    slot_mapping: int64 ``[n]`` on the pools' device; a negative slot skips.
    """
    n_blocks, H, bs, D = _check_pools(k_pool, v_pool)
    if keys.shape != values.shape or keys.dtype != k_pool.dtype or values.dtype != k_pool.dtype:
        raise ValueError("keys/values must match each other and the pool dtype")
    kk, vv = keys, values
    if kk.dim() == 4:
        if kk.shape[0] != 1:
            raise ValueError("keys must have batch size 1: (1, H, n, D)")
        kk, vv = kk[0], vv[0]
    if kk.dim() != 3 or kk.shape[0] != H or kk.shape[2] != D:
        raise ValueError(f"keys must be (1, {H}, n, {D}), got {tuple(keys.shape)}")
    if kk.stride(2) != 1 or vv.stride(2) != 1 or kk.stride() != vv.stride():
        kk, vv = kk.contiguous(), vv.contiguous()
    n = kk.shape[1]
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != n or \
            slot_mapping.device != k_pool.device:
        raise ValueError("slot_mapping must be int64 [n] on the pool device")
    if n == 0:
        return
    dev = _dev_index(k_pool)
    nat.call("mz_kv_append", k_pool.data_ptr(), v_pool.data_ptr(), kk.data_ptr(), vv.data_ptr(),
             kk.stride(1), kk.stride(0), slot_mapping.data_ptr(), n, H, D, bs, n_blocks,
             dtype_code(k_pool.dtype), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def kv_append_paged(k_pool: torch.Tensor, v_pool: torch.Tensor, keys: torch.Tensor,
                    values: torch.Tensor, block_tables: torch.Tensor,
                    positions: torch.Tensor) -> None:
    """Decode-step append: keys/values ``[B, H, D]`` (or ``[B, H, 1, D]``), one
    token per sequence at ``positions[b]`` through ``block_tables[b]``."""
    n_blocks, H, bs, D = _check_pools(k_pool, v_pool)
    kk, vv = keys, values
    if kk.dim() == 4:
        kk, vv = kk[:, :, 0, :], vv[:, :, 0, :]
    if kk.dim() != 3 or kk.shape[1:] != (H, D) or kk.shape != vv.shape:
        raise ValueError(f"keys must be [B, {H}, D={D}], got {tuple(keys.shape)}")
    if kk.dtype != k_pool.dtype or vv.dtype != k_pool.dtype:
        raise ValueError("keys/values dtype must match the pool")
    if kk.stride(2) != 1 or vv.stride(2) != 1 or kk.stride() != vv.stride():
        kk, vv = kk.contiguous(), vv.contiguous()
    B = kk.shape[0]
    _as_i32(block_tables, k_pool.device, "block_tables")
    _as_i32(positions, k_pool.device, "positions")
    if block_tables.dim() != 2 or block_tables.shape[0] < B or positions.numel() < B:
        raise ValueError("block_tables must be [>=B, max_blocks] and positions [>=B]")
    if B == 0:
        return
    dev = _dev_index(k_pool)
    nat.call("mz_kv_append_paged", k_pool.data_ptr(), v_pool.data_ptr(), kk.data_ptr(),
             vv.data_ptr(), kk.stride(0), kk.stride(1), block_tables.data_ptr(),
             block_tables.shape[1], positions.data_ptr(), B, H, D, bs, n_blocks,
             dtype_code(k_pool.dtype), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def kv_gather(k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
              ctx_lens: torch.Tensor, ctx_lens_host: list[int]) -> tuple[torch.Tensor, torch.Tensor]:
    """Gather each sequence's KV into contiguous ``[H, ctx_b, D]`` pieces.

    Returns (K, V) as flat tensors ``[sum_b H*ctx_b*D]`` viewed per sequence by
    the caller; with one sequence they are shaped ``(1, H, T, D)``.
    """
    n_blocks, H, bs, D = _check_pools(k_pool, v_pool)
    _as_i32(block_tables, k_pool.device, "block_tables")
    _as_i32(ctx_lens, k_pool.device, "ctx_lens")
    B = len(ctx_lens_host)
    offs = [0] * B
    tot = 0
    for i, c in enumerate(ctx_lens_host):
        offs[i] = tot
        tot += c
    out_k = torch.empty(tot * H * D, dtype=k_pool.dtype, device=k_pool.device)
    out_v = torch.empty_like(out_k)
    if B == 1:
        out_k = out_k.view(1, H, tot, D)
        out_v = out_v.view(1, H, tot, D)
    if B == 0 or tot == 0:
        return out_k, out_v
    off_t = torch.tensor(offs, dtype=torch.int64).to(k_pool.device, non_blocking=True)
    dev = _dev_index(k_pool)
    nat.call("mz_kv_gather", out_k.data_ptr(), out_v.data_ptr(), k_pool.data_ptr(),
             v_pool.data_ptr(), block_tables.data_ptr(), block_tables.shape[1],
             ctx_lens.data_ptr(), off_t.data_ptr(), B, max(ctx_lens_host), H, D, bs, n_blocks,
             dtype_code(k_pool.dtype), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)
    return out_k, out_v


# ---------------------------------------------------------------------------
# Step metadata
# ---------------------------------------------------------------------------

class PagedPlan(NamedTuple):
    """What ``paged_plan`` builds for one step of B sequences and n_rows rows."""

    q_start: torch.Tensor    # int32 [B], first row of each sequence
    positions: torch.Tensor  # int32 [n_rows], position of each row's token
    slots: torch.Tensor      # int64 [n_rows], its pool slot (-1 behind the last sequence)
    lengths: torch.Tensor    # int32 [B], cached tokens with the new ones
    held: torch.Tensor       # int32 [B], blocks in each table
    n_new: torch.Tensor      # int32 [1], new blocks needed


def paged_plan(block_tables: torch.Tensor, ctx_lens: torch.Tensor, q_lens: torch.Tensor,
               n_rows: int, block_size: int, n_blocks: int, new_ids: torch.Tensor | None = None,
               held: torch.Tensor | None = None) -> PagedPlan:
    """Block tables, slot map and positions of a step, from the sequences'
    lengths, in one launch (mz_paged_plan).

    Sequence b has ``ctx_lens[b]`` cached tokens in ``held[b]`` blocks (default
    ``ceil(ctx / block_size)``) of ``block_tables[b]`` and gets ``q_lens[b]``
    new ones.  Blocks that it lacks are taken from ``new_ids`` in order,
    sequence by sequence (``BlockManager.allocate``'s order), and written into
    ``block_tables`` in place.  ``n_rows`` >= ``sum(q_lens)``; rows behind the
    last sequence get slot -1 (skipped by the appends) and position 0.
    ``n_blocks``: blocks of the pools (bounds the ids)."""
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be [B, max_blocks]")
    dev = block_tables.get_device()
    B, width = block_tables.shape
    if not _i32_on(block_tables, dev):
        _as_i32(block_tables, block_tables.device, "block_tables")
    for t, name in ((ctx_lens, "ctx_lens"), (q_lens, "q_lens"), (held, "held")):
        if t is not None and not (_i32_on(t, dev) and t.numel() == B):
            _as_i32(t, block_tables.device, name)
            raise ValueError(f"{name} must hold one entry per sequence ({B})")
    if new_ids is not None and not _i32_on(new_ids, dev):
        _as_i32(new_ids, block_tables.device, "new_ids")
    if width == 0 and B:
        raise ValueError("block_tables must be [B, max_blocks] with max_blocks > 0")
    if not 0 <= n_rows < 1 << 31 or not 1 <= block_size < 1 << 31 or n_blocks < 1:
        raise ValueError("n_rows must be >= 0, block_size and n_blocks >= 1, the first two "
                         "below 2^31")
    dev = _dev_index(block_tables)
    positions, q_start, lengths, held_out, n_new = block_tables.new_empty(
        n_rows + 3 * B + 1).split_with_sizes((n_rows, B, B, B, 1))
    slots = block_tables.new_empty(n_rows, dtype=torch.int64)
    _call(dev, "mz_paged_plan", block_tables.data_ptr(), max(width, 1), ctx_lens.data_ptr(),
          q_lens.data_ptr(), _at(held), _at(new_ids), 0 if new_ids is None else new_ids.numel(),
          B, n_rows, block_size, n_blocks, q_start.data_ptr(), positions.data_ptr(),
          slots.data_ptr(), lengths.data_ptr(), held_out.data_ptr(), n_new.data_ptr())
    return PagedPlan(q_start, positions, slots, lengths, held_out, n_new)


# ---------------------------------------------------------------------------
# Query / key norm, rotation and append
# ---------------------------------------------------------------------------

def _rope_args(q, positions, inv_freq, q_weight, k_weight, eps, weight_offset, interleaved,
               freq_axes):
    """Checks shared by the norm-and-rotation calls; the arguments of
    mz_qk_norm_rope from ``positions`` to ``norm``."""
    T, _, D = q.shape
    dev = q.get_device()
    if not _i32_on(positions, dev):
        _as_i32(positions, q.device, "positions")
    axes = positions.shape
    n_axes = 1 if len(axes) == 1 else axes[0]
    if len(axes) not in (1, 2) or axes[-1] != T:
        raise ValueError(f"positions must be int32 [{T}] or [axes, {T}]")
    if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or \
            inv_freq.get_device() != dev or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must be a contiguous 1-D float32 tensor on {q.device}")
    half = inv_freq.numel()
    if freq_axes is not None:
        if not _i32_on(freq_axes, dev):
            _as_i32(freq_axes, q.device, "freq_axes")
        if freq_axes.numel() != half:
            raise ValueError("freq_axes must name one position axis per frequency")
    elif n_axes > 1 and half:
        raise ValueError("several position axes need freq_axes")
    w_dtype = None
    for x in (q_weight, k_weight):
        if x is None:
            continue
        if eps is None:
            raise ValueError("norm weights need eps")
        if w_dtype is None:
            w_dtype = x.dtype
        if x.dtype is not w_dtype or x.shape != (D,) or x.get_device() != dev or \
                not x.is_contiguous():
            raise ValueError(f"norm weights must be contiguous [{D}] of one dtype on {q.device}")
    return (positions.data_ptr(), T, n_axes, inv_freq.data_ptr(), _at(freq_axes), 2 * half,
            1 if interleaved else 0, _at(q_weight), _at(k_weight),
            0 if w_dtype is None else dtype_code(w_dtype), weight_offset,
            0.0 if eps is None else eps, 0 if eps is None else 1)


def _heads(t: torch.Tensor, name: str, T: int, n_heads: int, like: torch.Tensor,
           dtype: torch.dtype, dev: int) -> tuple[int, int, int]:
    """(pointer, token stride, head stride) of a tensor ``[T, n_heads, D]`` of
    the last dimension, dtype and device of ``like``."""
    if t.shape == (T, n_heads, like.shape[-1]) and t.dtype is dtype and t.get_device() == dev:
        ts, hs, one = t.stride()
        if one == 1:
            return t.data_ptr(), ts, hs
    raise ValueError(f"{name} must be [{T}, {n_heads} heads, {like.shape[-1]}] of {dtype} on "
                     f"{like.device} with unit last stride")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                 inv_freq: torch.Tensor, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float | None = None,
                 weight_offset: float = 0.0, interleaved: bool = False,
                 freq_axes: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each head of q ``[T, Hq, D]`` and k ``[T, Hkv, D]`` and their
    rotation by position, in one pass (mz_qk_norm_rope).

    positions: int32 ``[T]``, or ``[axes, T]`` with ``freq_axes`` int32
    ``[len(inv_freq)]`` naming the axis of every frequency (time, height and
    width of image or video tokens, say).  The first ``2 * len(inv_freq)``
    dimensions rotate by ``position * inv_freq[i]`` (float32), as pairs
    ``(i, i + len(inv_freq))`` or, ``interleaved``, ``(2i, 2i + 1)``.  The norm
    runs if ``eps`` is given, times ``weight + weight_offset`` where a weight
    is.  ``q_out`` / ``k_out`` may be q / k themselves."""
    if q.dim() != 3:
        raise ValueError("q must be [T, heads, D] with unit last stride")
    T, Hq, D = q.shape
    Hkv = k.shape[1] if k.dim() == 3 else 0
    of = q, q.dtype, q.get_device()
    q_at, k_at = _heads(q, "q", T, Hq, *of), _heads(k, "k", T, Hkv, *of)
    args = _rope_args(q, positions, inv_freq, q_weight, k_weight, eps, weight_offset, interleaved,
                      freq_axes)
    if q_out is None:
        q_out = q.new_empty(q.shape)
    if k_out is None:
        k_out = k.new_empty(k.shape)
    qo_at, ko_at = _heads(q_out, "q_out", T, Hq, *of), _heads(k_out, "k_out", T, Hkv, *of)
    _call(_dev_index(q), "mz_qk_norm_rope", *qo_at, *ko_at, *q_at, *k_at,
          0, 0, 0, 0, 0, 0, 0, 0, *args, T, Hq, Hkv, D, dtype_code(q.dtype))
    return q_out, k_out


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        positions: torch.Tensor, inv_freq: torch.Tensor, k_pool: torch.Tensor,
                        v_pool: torch.Tensor, slot_mapping: torch.Tensor,
                        q_weight: torch.Tensor | None = None,
                        k_weight: torch.Tensor | None = None, eps: float | None = None,
                        weight_offset: float = 0.0, interleaved: bool = False,
                        freq_axes: torch.Tensor | None = None,
                        q_out: torch.Tensor | None = None) -> torch.Tensor:
    """``qk_norm_rope`` and ``kv_append`` in one pass: the queries go to the
    returned tensor (or ``q_out``, which may be q), the keys and v ``[T, Hkv, D]``
    to their slots of the pools.  slot_mapping: int64 ``[T]``, distinct; a
    negative slot skips the write."""
    n_blocks, H, bs, D = _check_pools(k_pool, v_pool)
    if q.dim() != 3 or q.shape[2] != D or q.dtype is not k_pool.dtype or \
            q.get_device() != k_pool.get_device():
        raise ValueError(f"q must be [T, heads, {D}] of the pools' dtype and device")
    T, Hq, _ = q.shape
    of = q, q.dtype, q.get_device()
    q_at, k_at, v_at = _heads(q, "q", T, Hq, *of), _heads(k, "k", T, H, *of), _heads(v, "v", T, H, *of)
    if slot_mapping.dtype is not torch.int64 or slot_mapping.numel() != T or \
            slot_mapping.get_device() != q.get_device() or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be a contiguous int64 [T] on the pool device")
    args = _rope_args(q, positions, inv_freq, q_weight, k_weight, eps, weight_offset, interleaved,
                      freq_axes)
    if q_out is None:
        q_out = q.new_empty(q.shape)
    qo_at = _heads(q_out, "q_out", T, Hq, *of)
    _call(_dev_index(q), "mz_qk_norm_rope", *qo_at, 0, 0, 0, *q_at, *k_at,
          *v_at, k_pool.data_ptr(), v_pool.data_ptr(), slot_mapping.data_ptr(), bs, n_blocks,
          *args, T, Hq, H, D, dtype_code(q.dtype))
    return q_out


# ---------------------------------------------------------------------------
# Decode attention
# ---------------------------------------------------------------------------

def decode_workspace(n_seqs: int, n_kv_heads: int, rows: int, head_dim: int, device: int,
                     num_warps: int = 0, shared: bool = True, batch_invariant: bool = False,
                     max_blocks: int = 0, block_size: int = 16,
                     stream: int | None = None) -> torch.Tensor:
    """A zero-initialised decode workspace for exactly these sizes: the one
    kept for this layout (``shared``; with ``stream``, a stream's raw handle,
    for this layout on that stream), or a new one the caller owns.  A
    batch-invariant launch needs room for the pieces of tables ``max_blocks``
    wide (of ``block_size``-token blocks)."""
    key = (device, n_seqs, n_kv_heads, rows, head_dim, num_warps,
           (max_blocks, block_size) if batch_invariant else None, stream)
    if shared and key in _workspaces:
        _workspaces.move_to_end(key)
        return _workspaces[key]
    size = ctypes.c_size_t(0)
    if batch_invariant:
        if max_blocks <= 0:
            raise ValueError("a batch-invariant workspace needs max_blocks")
        nat.call("mz_paged_decode_workspace_size_ex", n_seqs, n_kv_heads, rows, head_dim,
                 num_warps, max_blocks, block_size, nat.MZ_DECODE_BATCH_INVARIANT, device,
                 ctypes.byref(size))
    else:
        nat.call("mz_paged_decode_workspace_size", n_seqs, n_kv_heads, rows, head_dim,
                 num_warps, device, ctypes.byref(size))
    return _layout_workspace(_workspaces, key, int(size.value), device, shared)


def _score_mod(q: torch.Tensor, n_heads: int, softcap: float,
               alibi_slopes: torch.Tensor | None, window: int, sink_tokens: int,
               prefix_lens: torch.Tensor | None, first_keys: torch.Tensor | None, n_seqs: int,
               n_first: int) -> "nat.ScoreMod | None":
    """The checked mz_score_mod of an attention call; None where nothing of it
    is in use (the sink tokens alone change nothing)."""
    if softcap < 0 or not math.isfinite(softcap):
        raise ValueError("softcap must be finite and not negative (0: none)")
    if 0 < softcap < _F32_TINY:  # as a float32 it could become 0, which is none
        raise ValueError(f"softcap must be 0 (none) or at least {_F32_TINY}")
    if window < 0 or sink_tokens < 0:
        raise ValueError("window and sink_tokens must not be negative")
    if not (softcap or window) and alibi_slopes is None and prefix_lens is None and \
            first_keys is None:
        return None
    dev = q.get_device()
    if alibi_slopes is not None and (
            alibi_slopes.dtype is not torch.float32 or alibi_slopes.shape != (n_heads,) or
            alibi_slopes.get_device() != dev or not alibi_slopes.is_contiguous()):
        raise ValueError(f"alibi_slopes must be a contiguous float32 [{n_heads}] on {q.device}")
    for t, name, n in ((prefix_lens, "prefix_lens", n_seqs), (first_keys, "first_keys", n_first)):
        if t is not None and not (_i32_on(t, dev) and t.numel() == n):
            _as_i32(t, q.device, name)
            raise ValueError(f"{name} must hold {n} entries")
    big = (1 << 31) - 1
    return nat.ScoreMod(min(softcap, 1e38), min(window, big), min(sink_tokens, big), _ptr(alibi_slopes),
                        _ptr(prefix_lens), _ptr(first_keys))


def _mod_device(k_pool: torch.Tensor, **tensors: torch.Tensor | None) -> None:
    """A modified-score call's tensors are all on the pools' device."""
    dev = k_pool.get_device()
    for name, t in tensors.items():
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name} must be on the pools' device")


def _mod_workspace(n_seqs: int, n_kv_heads: int, rows: int, head_dim: int, device: int,
                   num_warps: int, **kw) -> torch.Tensor:
    """The workspace of a modified-score call that was given none: one per
    layout and stream, so that calls on two streams do not meet in it, and a
    new one inside a capture (its clearing is captured with it), so that no
    two graphs do."""
    if torch.cuda.is_current_stream_capturing():
        return decode_workspace(n_seqs, n_kv_heads, rows, head_dim, device, num_warps,
                                shared=False, **kw)
    return decode_workspace(n_seqs, n_kv_heads, rows, head_dim, device, num_warps,
                            stream=_stream(device), **kw)


def reset_workspaces() -> None:
    """Zero every cached workspace (needed after a call that reported an error)."""
    for ws in list(_workspaces.values()) + list(_qworkspaces.values()):
        ws.zero_()


def paged_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 block_tables: torch.Tensor, ctx_lens: torch.Tensor, scale: float | None = None,
                 out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                 num_warps: int = 0, workspace: torch.Tensor | None = None, causal: bool = False,
                 softcap: float = 0.0, alibi_slopes: torch.Tensor | None = None, window: int = 0,
                 sink_tokens: int = 0, prefix_lens: torch.Tensor | None = None,
                 first_keys: torch.Tensor | None = None) -> torch.Tensor:
    """Fused GQA paged decode attention.

    q: ``[B, Hq, D]`` (one query token per sequence) or ``[B, n_q, Hq, D]``.
    Returns ``out`` with q's shape, dtype ``out_dtype`` (default q.dtype).

    ``causal``: the n_q tokens are the sequence's last ones (drafted tokens,
    say) and each sees the keys up to its own; without it all see every key.
    Modified scores and masks (mz_score_mod; several tokens then need
    ``causal``): ``softcap`` caps the scaled scores by ``softcap * tanh(x /
    softcap)``; ``alibi_slopes`` float32 ``[Hq]`` subtracts ``slope * distance``;
    a token sees the last ``window`` keys (0: all), not those before
    ``first_keys[b]`` (its document's start), and in any case the first
    ``sink_tokens`` (the sequence's, not its documents') and the first
    ``prefix_lens[b]``.  A token that sees no key gets zeros; blocks behind those
    first ones and below the lowest key that window and ``first_keys`` leave to
    the sequence's tokens need no valid table entry.
    """
    n_blocks, Hkv, bs, D = _check_pools(k_pool, v_pool)
    if q.dtype != k_pool.dtype:
        raise ValueError("q dtype must match the pools")
    if q.dim() == 3:
        B, Hq, Dq = q.shape
        nq = 1
        q_sb, q_st, q_sh = q.stride(0), 0, q.stride(1)
    elif q.dim() == 4:
        B, nq, Hq, Dq = q.shape
        q_sb, q_st, q_sh = q.stride(0), q.stride(1), q.stride(2)
    else:
        raise ValueError("q must be [B, Hq, D] or [B, n_q, Hq, D]")
    if Dq != D or q.stride(-1) != 1:
        raise ValueError(f"q head_dim must be {D} with unit stride")
    if Hq % Hkv:
        raise ValueError(f"n_heads {Hq} is not a multiple of n_kv_heads {Hkv}")
    dev = k_pool.get_device()
    if not (_i32_on(block_tables, dev) and _i32_on(ctx_lens, dev)):
        _as_i32(block_tables, k_pool.device, "block_tables")
        _as_i32(ctx_lens, k_pool.device, "ctx_lens")
    if block_tables.dim() != 2 or block_tables.shape[0] < B or ctx_lens.numel() < B:
        raise ValueError("block_tables must be [>=B, max_blocks] and ctx_lens [>=B]")
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = q.new_empty(q.shape, dtype=out_dtype)
    if out.shape != q.shape or out.dtype != out_dtype or out.stride(-1) != 1:
        raise ValueError("out must match q's shape with unit last stride")
    if q.dim() == 3:
        o_sb, o_st, o_sh = out.stride(0), 0, out.stride(1)
    else:
        o_sb, o_st, o_sh = out.stride(0), out.stride(1), out.stride(2)
    if scale is None:
        scale = D ** -0.5
    mod = _score_mod(q, Hq, softcap, alibi_slopes, window, sink_tokens, prefix_lens,
                     first_keys, B, B)
    if mod is not None and nq > 1 and not causal:
        raise ValueError("modified scores of several query tokens need causal=True")
    if mod is None and causal and nq > 1:
        mod = nat.ScoreMod()
    if mod is not None:
        _mod_device(k_pool, q=q, out=out, workspace=workspace)
    if B == 0:
        return out
    dev = _dev_index(q)
    rows = nq * (Hq // Hkv)
    if workspace is None:
        workspace = (decode_workspace if mod is None else _mod_workspace)(B, Hkv, rows, D, dev,
                                                                          num_warps)
    if mod is not None:
        _call(dev, "mz_paged_decode_mod", out.data_ptr(), dtype_code(out_dtype), o_sb, o_st, o_sh,
              q.data_ptr(), q_sb, q_st, q_sh, nq, k_pool.data_ptr(), v_pool.data_ptr(),
              block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), B, Hq, Hkv, D,
              bs, n_blocks, float(scale), ctypes.addressof(mod), dtype_code(q.dtype), num_warps,
              workspace.data_ptr(), workspace.numel())
        return out
    nat.call("mz_paged_decode", out.data_ptr(), dtype_code(out_dtype), o_sb, o_st, o_sh,
             q.data_ptr(), q_sb, q_st, q_sh, nq, k_pool.data_ptr(), v_pool.data_ptr(),
             block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), B, Hq, Hkv,
             D, bs, n_blocks, float(scale), dtype_code(q.dtype), num_warps,
             workspace.data_ptr(), workspace.numel(), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)
    return out


def paged_append_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                        k_new: torch.Tensor, v_new: torch.Tensor, block_tables: torch.Tensor,
                        ctx_lens: torch.Tensor, scale: float | None = None,
                        out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                        num_warps: int = 0, workspace: torch.Tensor | None = None,
                        overlap_previous: bool = False, batch_invariant: bool = False,
                        softcap: float = 0.0, alibi_slopes: torch.Tensor | None = None,
                        window: int = 0, sink_tokens: int = 0,
                        prefix_lens: torch.Tensor | None = None,
                        first_keys: torch.Tensor | None = None) -> torch.Tensor:
    """Fused decode step for one layer: write ``k_new/v_new [B, Hkv, D]`` at
    position ``ctx_lens[b] - 1`` of each sequence, then attend ``q [B, Hq, D]``
    over the first ``ctx_lens[b]`` tokens (one launch).  ``overlap_previous``:
    the launch may start while the kernel ahead of it on the stream runs
    (MZ_LAUNCH_OVERLAP_PREVIOUS) -- only when that kernel writes none of the
    pools, ``block_tables``, ``ctx_lens``, ``alibi_slopes``, ``prefix_lens`` or
    ``first_keys``.  ``batch_invariant``: each
    sequence's output bytes are independent of the rest of the batch
    (MZ_DECODE_BATCH_INVARIANT).  Modified scores and masks as in
    ``paged_decode``."""
    n_blocks, Hkv, bs, D = _check_pools(k_pool, v_pool)
    if q.dim() != 3 or q.shape[2] != D or q.stride(-1) != 1 or q.dtype != k_pool.dtype:
        raise ValueError(f"q must be [B, Hq, {D}] of the pool dtype with unit last stride")
    B, Hq, _ = q.shape
    if k_new.shape != (B, Hkv, D) or v_new.shape != (B, Hkv, D):
        raise ValueError(f"k_new/v_new must be [{B}, {Hkv}, {D}]")
    if k_new.dtype != k_pool.dtype or v_new.dtype != k_pool.dtype:
        raise ValueError("k_new/v_new dtype must match the pools")
    if k_new.stride() != v_new.stride() or k_new.stride(2) != 1:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    dev = k_pool.get_device()
    if not (_i32_on(block_tables, dev) and _i32_on(ctx_lens, dev)):
        _as_i32(block_tables, k_pool.device, "block_tables")
        _as_i32(ctx_lens, k_pool.device, "ctx_lens")
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = q.new_empty(q.shape, dtype=out_dtype)
    if out.shape != q.shape or out.dtype != out_dtype or out.stride(-1) != 1:
        raise ValueError("out must match q's shape with unit last stride")
    if scale is None:
        scale = D ** -0.5
    mod = _score_mod(q, Hq, softcap, alibi_slopes, window, sink_tokens, prefix_lens,
                     first_keys, B, B)
    if mod is not None:
        _mod_device(k_pool, q=q, k_new=k_new, v_new=v_new, out=out, workspace=workspace)
    if B == 0:
        return out
    dev = _dev_index(q)
    if workspace is None:
        workspace = (decode_workspace if mod is None else _mod_workspace)(
            B, Hkv, Hq // Hkv, D, dev, num_warps, batch_invariant=batch_invariant,
            max_blocks=block_tables.shape[1], block_size=bs)
    if mod is not None:
        _call(dev, "mz_paged_append_decode_mod", out.data_ptr(), dtype_code(out_dtype),
              out.stride(0), out.stride(1), q.data_ptr(), q.stride(0), q.stride(1),
              k_pool.data_ptr(), v_pool.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
              k_new.stride(0), k_new.stride(1), block_tables.data_ptr(), block_tables.shape[1],
              ctx_lens.data_ptr(), B, Hq, Hkv, D, bs, n_blocks, float(scale), ctypes.addressof(mod),
              dtype_code(q.dtype), num_warps,
              (nat.MZ_LAUNCH_OVERLAP_PREVIOUS if overlap_previous else 0)
              | (nat.MZ_DECODE_BATCH_INVARIANT if batch_invariant else 0),
              workspace.data_ptr(), workspace.numel())
        return out
    nat.call("mz_paged_append_decode_ex", out.data_ptr(), dtype_code(out_dtype), out.stride(0),
             out.stride(1), q.data_ptr(), q.stride(0), q.stride(1), k_pool.data_ptr(),
             v_pool.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0),
             k_new.stride(1), block_tables.data_ptr(), block_tables.shape[1],
             ctx_lens.data_ptr(), B, Hq, Hkv, D, bs, n_blocks, float(scale),
             dtype_code(q.dtype), num_warps,
             (nat.MZ_LAUNCH_OVERLAP_PREVIOUS if overlap_previous else 0)
             | (nat.MZ_DECODE_BATCH_INVARIANT if batch_invariant else 0),
             workspace.data_ptr(), workspace.numel(), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)
    return out


def paged_prefill(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                  block_tables: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor,
                  ctx_lens: torch.Tensor, max_q_len: int, scale: float | None = None,
                  out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                  softcap: float = 0.0, alibi_slopes: torch.Tensor | None = None,
                  window: int = 0, sink_tokens: int = 0,
                  prefix_lens: torch.Tensor | None = None,
                  first_keys: torch.Tensor | None = None) -> torch.Tensor:
    """Chunked prefill attention (mz_paged_prefill): ``q [T, Hq, D]`` holds
    sequence b's ``q_len[b]`` query tokens at rows ``q_start[b]...``; they sit
    at the last ``q_len[b]`` of the sequence's ``ctx_lens[b]`` positions (their
    K/V already appended) and attend causally.  Modified scores and masks as in
    ``paged_decode``, with ``first_keys`` int32 ``[T]``, one per row of q."""
    n_blocks, Hkv, bs, D = _check_pools(k_pool, v_pool)
    if q.dim() != 3 or q.shape[2] != D or q.stride(-1) != 1 or q.dtype != k_pool.dtype:
        raise ValueError(f"q must be [T, Hq, {D}] of the pool dtype with unit last stride")
    T, Hq, _ = q.shape
    B = block_tables.shape[0]
    for t, name in ((q_start, "q_start"), (q_len, "q_len"), (ctx_lens, "ctx_lens")):
        _as_i32(t, k_pool.device, name)
        if t.numel() != B:
            raise ValueError(f"{name} must hold one entry per sequence ({B})")
    _as_i32(block_tables, k_pool.device, "block_tables")
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = q.new_empty(q.shape, dtype=out_dtype)
    if out.shape != q.shape or out.dtype != out_dtype or out.stride(-1) != 1:
        raise ValueError("out must match q's shape with unit last stride")
    if scale is None:
        scale = D ** -0.5
    mod = _score_mod(q, Hq, softcap, alibi_slopes, window, sink_tokens, prefix_lens,
                     first_keys, B, T)
    if mod is not None:
        _mod_device(k_pool, q=q, out=out)
    if B == 0 or T == 0 or max_q_len == 0:
        return out
    dev = _dev_index(q)
    if mod is not None:
        _call(dev, "mz_paged_prefill_mod", out.data_ptr(), dtype_code(out_dtype), out.stride(0),
              out.stride(1), q.data_ptr(), q.stride(0), q.stride(1), T, q_start.data_ptr(),
              q_len.data_ptr(), int(max_q_len), k_pool.data_ptr(), v_pool.data_ptr(),
              block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), B, Hq, Hkv, D,
              bs, n_blocks, float(scale), ctypes.addressof(mod), dtype_code(q.dtype))
        return out
    nat.call("mz_paged_prefill", out.data_ptr(), dtype_code(out_dtype), out.stride(0),
             out.stride(1), q.data_ptr(), q.stride(0), q.stride(1), T, q_start.data_ptr(),
             q_len.data_ptr(), int(max_q_len), k_pool.data_ptr(), v_pool.data_ptr(),
             block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), B, Hq, Hkv,
             D, bs, n_blocks, float(scale), dtype_code(q.dtype), error_word(dev).data_ptr(),
             _stream(dev))
    _after(dev)
    return out


def paged_append_decode_allgather(peers: "nat.PeerOutputs", q: torch.Tensor,
                                  k_pool: torch.Tensor, v_pool: torch.Tensor,
                                  k_new: torch.Tensor, v_new: torch.Tensor,
                                  block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                                  out_seq_stride: int, out_head_stride: int,
                                  out_dtype: torch.dtype, scale: float | None = None,
                                  num_warps: int = 0,
                                  workspace: torch.Tensor | None = None,
                                  overlap_previous: bool = False,
                                  wait_previous: bool = False) -> None:
    """paged_append_decode whose output rows go to every rank's gathered
    buffer (``peers.out[r]``: this rank's head block there) and whose last
    warp signals the peers (mz_paged_append_decode_allgather); follow it with
    ``peer_wait``, or with a next launch made with ``wait_previous``, before
    reading the gathered buffer.  ``wait_previous`` (MZ_LAUNCH_WAIT_PREVIOUS):
    the launch first waits, on the device and bounded, for the peers' rows of
    this rank's previous launch."""
    n_blocks, Hkv, bs, D = _check_pools(k_pool, v_pool)
    if q.dim() != 3 or q.shape[2] != D or q.stride(-1) != 1 or q.dtype != k_pool.dtype:
        raise ValueError(f"q must be [B, Hq, {D}] of the pool dtype with unit last stride")
    B, Hq, _ = q.shape
    if B == 0:
        raise ValueError("an all-gather launch needs at least one sequence")
    if k_new.shape != (B, Hkv, D) or v_new.shape != (B, Hkv, D):
        raise ValueError(f"k_new/v_new must be [{B}, {Hkv}, {D}]")
    if k_new.dtype != k_pool.dtype or v_new.dtype != k_pool.dtype:
        raise ValueError("k_new/v_new dtype must match the pools")
    if k_new.stride() != v_new.stride() or k_new.stride(2) != 1:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    _as_i32(block_tables, k_pool.device, "block_tables")
    _as_i32(ctx_lens, k_pool.device, "ctx_lens")
    if scale is None:
        scale = D ** -0.5
    dev = _dev_index(q)
    if workspace is None:
        workspace = decode_workspace(B, Hkv, Hq // Hkv, D, dev, num_warps)
    nat.call("mz_paged_append_decode_allgather", ctypes.byref(peers), dtype_code(out_dtype),
             out_seq_stride, out_head_stride, q.data_ptr(), q.stride(0), q.stride(1),
             k_pool.data_ptr(), v_pool.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
             k_new.stride(0), k_new.stride(1), block_tables.data_ptr(), block_tables.shape[1],
             ctx_lens.data_ptr(), B, Hq, Hkv, D, bs, n_blocks, float(scale),
             dtype_code(q.dtype), num_warps,
             (nat.MZ_LAUNCH_OVERLAP_PREVIOUS if overlap_previous else 0)
             | (nat.MZ_LAUNCH_WAIT_PREVIOUS if wait_previous else 0),
             workspace.data_ptr(), workspace.numel(), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def peer_wait(signal: torch.Tensor, n_ranks: int, rank: int, epoch: int,
              timeout_s: float = 2.0) -> None:
    """Enqueue the bounded wait for every peer's signal word to reach
    ``epoch`` (mz_peer_wait); a timeout shows up as a device error."""
    if signal.dtype != torch.int32 or signal.numel() < n_ranks or not signal.is_cuda:
        raise ValueError(f"signal must be a CUDA int32 tensor of at least {n_ranks} words")
    dev = _dev_index(signal)
    nat.call("mz_peer_wait", signal.data_ptr(), n_ranks, rank, epoch & 0xFFFFFFFF,
             int(timeout_s * 1e9), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def ipc_export(t: torch.Tensor) -> tuple[bytes, int]:
    """(handle, byte offset) of the device allocation holding ``t``'s data."""
    h = ctypes.create_string_buffer(nat.MZ_IPC_HANDLE_BYTES)
    off = ctypes.c_uint64()
    nat.call("mz_ipc_export", t.data_ptr(), h, ctypes.byref(off))
    return h.raw, int(off.value)


def ipc_open(handle: bytes, offset: int) -> tuple[int, int]:
    """Map a peer's exported allocation on the current device: (base, ptr)."""
    if len(handle) != nat.MZ_IPC_HANDLE_BYTES:
        raise ValueError("bad IPC handle length")
    base, ptr = ctypes.c_void_p(), ctypes.c_void_p()
    nat.call("mz_ipc_open", handle, offset, ctypes.byref(base), ctypes.byref(ptr))
    return int(base.value), int(ptr.value)


def ipc_close(base: int) -> None:
    nat.call("mz_ipc_close", base)


# ---------------------------------------------------------------------------
# Quantised KV
# ---------------------------------------------------------------------------

def _check_qpools(pools) -> tuple[int, int, int, int, int]:
    """(n_blocks, H, bs, D, bits) of a 6-tuple (k_codes, k_scales, k_biases,
    v_codes, v_scales, v_biases): codes int32 [N, H, bs, D*bits/32], scales and
    biases fp16 [N, H, bs, D/64]."""
    if len(pools) != 6:
        raise ValueError("quantised pools: (k_codes, k_scales, k_biases, v_codes, v_scales, v_biases)")
    kc, ks, kb, vc, vs, vb = pools
    for t in pools:
        if not t.is_contiguous() or t.device != kc.device or t.dim() != 4:
            raise ValueError("quantised pools must be contiguous 4-D tensors on one device")
    if kc.dtype != torch.int32 or vc.dtype != torch.int32 or kc.shape != vc.shape:
        raise ValueError("codes must be int32 [N, H, bs, words] (same for K and V)")
    for t in (ks, kb, vs, vb):
        if t.dtype != torch.float16 or t.shape != ks.shape:
            raise ValueError("scales/biases must be fp16 [N, H, bs, D/64]")
    n, h, bs, words = kc.shape
    D = ks.shape[3] * 64
    bits = words * 32 // D
    if bits not in (4, 8) or ks.shape[:3] != kc.shape[:3]:
        raise ValueError("codes/scales shapes do not describe 4- or 8-bit groups of 64")
    return n, h, bs, D, bits


def _qptrs(pools):
    return [t.data_ptr() for t in pools]


def kv_quant_append(pools, keys: torch.Tensor, values: torch.Tensor,
                    slot_mapping: torch.Tensor) -> None:
    """Quantise keys/values ``(1, H, n, D)`` (or ``(H, n, D)``) into pool slots."""
    n_blocks, H, bs, D, bits = _check_qpools(pools)
    kk, vv = (keys[0], values[0]) if keys.dim() == 4 else (keys, values)
    if kk.shape != vv.shape or kk.dim() != 3 or kk.shape[0] != H or kk.shape[2] != D:
        raise ValueError(f"keys must be (1, {H}, n, {D})")
    if kk.stride(2) != 1 or vv.stride(2) != 1 or kk.stride() != vv.stride():
        kk, vv = kk.contiguous(), vv.contiguous()
    n = kk.shape[1]
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != n:
        raise ValueError("slot_mapping must be int64 [n]")
    if n == 0:
        return
    dev = _dev_index(pools[0])
    nat.call("mz_kv_quant_append", *_qptrs(pools), kk.data_ptr(), vv.data_ptr(), kk.stride(1),
             kk.stride(0), slot_mapping.data_ptr(), n, H, D, bs, n_blocks, bits, 64,
             dtype_code(kk.dtype), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def kv_quant_append_paged(pools, keys: torch.Tensor, values: torch.Tensor,
                          block_tables: torch.Tensor, positions: torch.Tensor) -> None:
    """Decode-step quantise-append: keys/values ``[B, H, D]``, one token per
    sequence at ``positions[b]`` through ``block_tables[b]``."""
    n_blocks, H, bs, D, bits = _check_qpools(pools)
    kk, vv = keys, values
    if kk.dim() == 4:
        kk, vv = kk[:, :, 0, :], vv[:, :, 0, :]
    if kk.dim() != 3 or kk.shape[1:] != (H, D) or kk.shape != vv.shape:
        raise ValueError(f"keys must be [B, {H}, {D}]")
    if kk.stride(2) != 1 or vv.stride(2) != 1 or kk.stride() != vv.stride():
        kk, vv = kk.contiguous(), vv.contiguous()
    _as_i32(block_tables, pools[0].device, "block_tables")
    _as_i32(positions, pools[0].device, "positions")
    B = kk.shape[0]
    if B == 0:
        return
    dev = _dev_index(pools[0])
    nat.call("mz_kv_quant_append_paged", *_qptrs(pools), kk.data_ptr(), vv.data_ptr(),
             kk.stride(0), kk.stride(1), block_tables.data_ptr(), block_tables.shape[1],
             positions.data_ptr(), B, H, D, bs, n_blocks, bits, 64, dtype_code(kk.dtype),
             error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def kv_dequant_blocks(pools, block_ids: torch.Tensor, k_out: torch.Tensor,
                      v_out: torch.Tensor) -> None:
    """Dequantise quantised blocks ``block_ids`` (int32 on the pools' device)
    of the 6-tuple ``pools`` into ``k_out`` / ``v_out`` ``[n, H, bs, D]``
    (fp16 or bf16): block ``block_ids[i]`` becomes block ``i``."""
    n_blocks, H, bs, D, bits = _check_qpools(pools)
    _as_i32(block_ids, pools[0].device, "block_ids")
    n = block_ids.numel()
    for t in (k_out, v_out):
        if (t.shape != (n, H, bs, D) or t.dtype not in (torch.float16, torch.bfloat16)
                or not t.is_contiguous() or t.device != pools[0].device):
            raise ValueError(f"outputs must be contiguous fp16/bf16 [{n}, {H}, {bs}, {D}]")
    if k_out.dtype != v_out.dtype:
        raise ValueError("k_out and v_out must have the same dtype")
    if n == 0:
        return
    dev = _dev_index(pools[0])
    nat.call("mz_kv_dequant_blocks", k_out.data_ptr(), v_out.data_ptr(), dtype_code(k_out.dtype),
             *_qptrs(pools), block_ids.data_ptr(), n, H, D, bs, n_blocks, bits,
             error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def decode_q_workspace(n_seqs: int, n_kv_heads: int, rows: int, head_dim: int, bits: int,
                       device: int, num_warps: int = 0, shared: bool = True) -> torch.Tensor:
    """As ``decode_workspace``, for the quantised decode."""
    size = ctypes.c_size_t(0)
    nat.call("mz_paged_decode_q_workspace_size", n_seqs, n_kv_heads, rows, head_dim, bits,
             num_warps, device, ctypes.byref(size))
    key = (device, n_seqs, n_kv_heads, rows, head_dim, bits, num_warps)
    return _layout_workspace(_qworkspaces, key, int(size.value), device, shared)


def paged_decode_q(q: torch.Tensor, pools, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                   scale: float | None = None, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype | None = None, num_warps: int = 0,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention over quantised K/V (dequantisation fused in).
    q: ``[B, Hq, D]`` or ``[B, n_q, Hq, D]`` (bf16/fp16)."""
    n_blocks, Hkv, bs, D, bits = _check_qpools(pools)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("q must be fp16 or bf16")
    if q.dim() == 3:
        B, Hq, Dq = q.shape
        nq, q_sb, q_st, q_sh = 1, q.stride(0), 0, q.stride(1)
    elif q.dim() == 4:
        B, nq, Hq, Dq = q.shape
        q_sb, q_st, q_sh = q.stride(0), q.stride(1), q.stride(2)
    else:
        raise ValueError("q must be [B, Hq, D] or [B, n_q, Hq, D]")
    if Dq != D or q.stride(-1) != 1 or Hq % Hkv:
        raise ValueError("q shape does not match the pools")
    _as_i32(block_tables, q.device, "block_tables")
    _as_i32(ctx_lens, q.device, "ctx_lens")
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
    if q.dim() == 3:
        o_sb, o_st, o_sh = out.stride(0), 0, out.stride(1)
    else:
        o_sb, o_st, o_sh = out.stride(0), out.stride(1), out.stride(2)
    if scale is None:
        scale = D ** -0.5
    if B == 0:
        return out
    dev = _dev_index(q)
    rows = nq * (Hq // Hkv)
    if workspace is None:
        workspace = decode_q_workspace(B, Hkv, rows, D, bits, dev, num_warps)
    nat.call("mz_paged_decode_q", out.data_ptr(), dtype_code(out_dtype), o_sb, o_st, o_sh,
             q.data_ptr(), q_sb, q_st, q_sh, nq, *_qptrs(pools), block_tables.data_ptr(),
             block_tables.shape[1], ctx_lens.data_ptr(), B, Hq, Hkv, D, bs, n_blocks, bits, 64,
             float(scale), dtype_code(q.dtype), num_warps, workspace.data_ptr(),
             workspace.numel(), error_word(dev).data_ptr(), _stream(dev))
    _after(dev)
    return out


# ---------------------------------------------------------------------------
# Block movement
# ---------------------------------------------------------------------------

def _pool_geometry(pools: torch.Tensor) -> tuple[int, int, int]:
    """(n_pools, n_blocks, block_bytes) of a contiguous ``[P, n_blocks, ...]``
    stack of pools (or a single pool ``[n_blocks, ...]``)."""
    if not pools.is_contiguous():
        raise ValueError("pools must be contiguous")
    return pools.shape[0], pools.shape[1], pools[0, 0].numel() * pools.element_size()


def block_copy(pools: torch.Tensor, src_ids: torch.Tensor, dst_ids: torch.Tensor) -> None:
    """Copy block src_ids[i] -> dst_ids[i] in every pool of ``pools``
    (a contiguous ``[P, n_blocks, ...]`` stack)."""
    P, N, bb = _pool_geometry(pools)
    _as_i32(src_ids, pools.device, "src_ids")
    _as_i32(dst_ids, pools.device, "dst_ids")
    if src_ids.numel() != dst_ids.numel():
        raise ValueError("src_ids and dst_ids must have the same length")
    n = src_ids.numel()
    if n == 0:
        return
    dev = _dev_index(pools)
    nat.call("mz_block_copy", pools.data_ptr(), N * bb, P, bb, src_ids.data_ptr(),
             dst_ids.data_ptr(), n, N, error_word(dev).data_ptr(), _stream(dev))
    _after(dev)


def block_pack(pools: torch.Tensor, ids: torch.Tensor, staging: torch.Tensor | None = None
               ) -> torch.Tensor:
    """Gather blocks ``ids`` of every pool into ``staging[n, P, block_bytes]`` (uint8)."""
    P, N, bb = _pool_geometry(pools)
    _as_i32(ids, pools.device, "ids")
    n = ids.numel()
    if staging is None:
        staging = torch.empty((n, P, bb), dtype=torch.uint8, device=pools.device)
    if staging.numel() < n * P * bb or not staging.is_contiguous():
        raise ValueError("staging too small or not contiguous")
    if n:
        dev = _dev_index(pools)
        nat.call("mz_block_pack", staging.data_ptr(), pools.data_ptr(), N * bb, P, bb,
                 ids.data_ptr(), n, N, error_word(dev).data_ptr(), _stream(dev))
        _after(dev)
    return staging


def block_unpack(pools: torch.Tensor, ids: torch.Tensor, staging: torch.Tensor) -> None:
    """Scatter ``staging[n, P, block_bytes]`` into blocks ``ids`` of every pool."""
    P, N, bb = _pool_geometry(pools)
    _as_i32(ids, pools.device, "ids")
    n = ids.numel()
    if staging.numel() < n * P * bb or not staging.is_contiguous() or \
            staging.device != pools.device:
        raise ValueError("staging must be a contiguous device buffer of n*P*block_bytes")
    if n:
        dev = _dev_index(pools)
        nat.call("mz_block_unpack", pools.data_ptr(), N * bb, P, bb, staging.data_ptr(),
                 ids.data_ptr(), n, N, error_word(dev).data_ptr(), _stream(dev))
        _after(dev)


def default_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
