"""The paged key-value cache in 8 bits: writing it, reading it back, and the attention
over it.

Pools, block tables, lengths and packed rows are those of ``paged_kv_append`` and
``paged_attention``; only what a pool holds differs.  ``k_cache`` and ``v_cache``
(n_pages, n_kv_head, page_size, head_dim) hold codes, ``torch.float8_e4m3fn`` or
``torch.int8``, and ``k_scale`` and ``v_scale`` (n_pages, n_kv_head, page_size / block)
uint8 an exponent for each ``block`` consecutive slots of a page and head: a cached value
is code * 2^(byte - 127).  A page holds a whole number of blocks; one of page_size or of
one token is a block as well.

    q = paged_kv_append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, table, lens, q=q, rotary=angles)
    o = paged_attention_8bit(q, k_cache, v_cache, k_scale, v_scale, table, lens)

Half the bytes of a 16-bit cache: twice the tokens in the same memory, and a decode step,
which reads every key once, takes little over half the time.  e4m3 keeps each value to 4
significant bits (relative error up to 2^-4); int8 keeps all of a block to 2^-8 .. 2^-7
of its largest value, which is the finer grid unless a block's values differ much in size.

A pool needs no clearing: a block's exponent starts anew when a step writes its first
slot.  When a step goes on behind rows of the block, the exponent only grows, and the
rows in front are rounded again where it does (e4m3: exactly, above its smallest
numbers; int8: all such steps together move a value by less than one step).
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch

from . import _lib
from .paged import _CODE, _HEAD_DIMS, _check_out, _launch, _ptr, _rows

__all__ = ["paged_kv_append_8bit", "paged_kv_read_8bit", "paged_attention_8bit"]

_CODES8 = {torch.float8_e4m3fn: _lib.CGPT_E4M3, torch.int8: _lib.CGPT_INT8}


def _check_cache8(name: str, dev: int, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  cu: Optional[torch.Tensor], err_flag: Optional[torch.Tensor]):
    """Checks the cache's side of a call as far as the native call cannot; returns the
    code, the caches' sizes and strides, the scales' strides, the block, the table's sizes
    and row stride."""
    try:
        same = (dev == k_cache.get_device() == v_cache.get_device() == k_scale.get_device() == v_scale.get_device()
                == block_table.get_device() == seq_lens.get_device() and (cu is None or cu.get_device() == dev)
                and (err_flag is None or err_flag.get_device() == dev))
    except AttributeError:
        same = False
    if not same or dev < 0:
        raise ValueError(f"{name}: tensors must be torch tensors on one GPU")
    code = _CODES8.get(k_cache.dtype)
    if code is None or v_cache.dtype is not k_cache.dtype:
        raise ValueError(f"{name}: the caches must hold float8_e4m3fn or int8 both, got {k_cache.dtype} and {v_cache.dtype}")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"{name}: k_cache and v_cache must share a shape (n_pages, n_kv_head, page_size, "
                         f"head_dim), got {tuple(shape)} and {tuple(v_cache.shape)}")
    n_pages, heads, page, hd = shape
    if hd not in _HEAD_DIMS:
        raise ValueError(f"{name}: head_dim {hd} is not one of {_HEAD_DIMS}")
    kp, kh, ks, kd = k_cache.stride()
    vp, vh, vs, vd = v_cache.stride()
    if kd != 1 or vd != 1:
        raise ValueError(f"{name}: cache rows must be contiguous")
    if k_scale.dtype is not torch.uint8 or v_scale.dtype is not torch.uint8:
        raise ValueError(f"{name}: k_scale and v_scale must be uint8, got {k_scale.dtype} and {v_scale.dtype}")
    sshape = k_scale.shape
    if (len(sshape) != 3 or v_scale.shape != sshape or sshape[0] != n_pages or sshape[1] != heads or not sshape[2]
            or page % sshape[2]):
        raise ValueError(f"{name}: k_scale and v_scale must be ({n_pages}, {heads}, page_size / block) with blocks that "
                         f"divide a page of {page}, got {tuple(sshape)} and {tuple(v_scale.shape)}")
    if block_table.dtype is not torch.int32 or seq_lens.dtype is not torch.int32:
        raise ValueError(f"{name}: block_table and seq_lens must be int32")
    if block_table.dim() != 2 or seq_lens.dim() != 1:
        raise ValueError(f"{name}: block_table must be (B, pages) and seq_lens (B,), got "
                         f"{tuple(block_table.shape)} and {tuple(seq_lens.shape)}")
    B, cols = block_table.shape
    ts, t1 = block_table.stride()
    if (t1 != 1 and cols > 1) or not seq_lens.is_contiguous() or seq_lens.shape[0] != B:
        raise ValueError(f"{name}: block_table must have contiguous rows and seq_lens be {B} contiguous lengths")
    if cu is not None and (cu.dtype is not torch.int32 or cu.dim() != 1 or cu.shape[0] != B + 1
                           or not cu.is_contiguous()):
        raise ValueError(f"{name}: offsets must be {B + 1} contiguous int32, got {cu.dtype} {tuple(cu.shape)}")
    if err_flag is not None and (err_flag.dtype is not torch.int32 or err_flag.numel() != 1):
        raise ValueError(f"{name}: err_flag must be one int32")
    return (code, n_pages, heads, page, hd, (kp, kh, ks, vp, vh, vs), (*k_scale.stride(), *v_scale.stride()),
            page // sshape[2], B, cols, ts)


def _check_rows8(name: str, what: str, x: torch.Tensor, B: int, hd: int, cu: Optional[torch.Tensor]) -> int:
    """Checks the step's rows; returns their dtype's code."""
    code = _CODE.get(x.dtype)
    if code is None:
        raise ValueError(f"{name}: unsupported dtype {x.dtype} (float32, bfloat16 or float16)")
    if x.dim() != 3 or x.shape[2] != hd:
        raise ValueError(f"{name}: {what} must be (n_tokens, heads, {hd}), got {tuple(x.shape)}")
    if cu is None and x.shape[0] != B:
        raise ValueError(f"{name}: {x.shape[0]} rows for {B} sequences need cu_q")
    return code


def paged_kv_append_8bit(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                         seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                         q: Optional[torch.Tensor] = None, rotary: Optional[torch.Tensor] = None,
                         interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                         err_flag: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the step's keys and values (n_tokens, n_kv_head, head_dim; float32, bfloat16
    or float16) into their pages as 8-bit codes, in place, and the blocks' exponents.

    A block's exponent is the smallest for which the step's values in it fit, or, where
    the step goes on behind rows of the block, the larger of that and the one there.  Codes
    are rounded once, to nearest even.  Infinities become the largest code, a NaN a NaN (in
    int8 0); neither takes part in the exponent, and each sets ``err_flag``.  ``q``,
    ``rotary``, ``interleaved`` and ``q_out`` as in ``paged_kv_append``, the turning in
    float64.  Two sequences of a call must not write to the same block of a page."""
    name = "paged_kv_append_8bit"
    try:
        dev = k.get_device()
    except AttributeError:
        dev = -1
    code, n_pages, hkv, page, hd, cs, ss, block, B, cols, ts = _check_cache8(
        name, dev, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_q, err_flag)
    dt = _check_rows8(name, "k", k, B, hd, cu_q)
    if not isinstance(v, torch.Tensor) or not all(t is None or isinstance(t, torch.Tensor) for t in (q, rotary)):
        raise ValueError(f"{name}: k, v, q and rotary must be torch tensors")
    n, vec = k.shape[0], 8 if dt else 4
    if v.shape != k.shape or v.dtype != k.dtype or v.get_device() != dev or k.shape[1] != hkv:
        raise ValueError(f"{name}: k and v must be {k.dtype} (n_tokens, {hkv}, {hd}) rows, got "
                         f"{tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    if k_cache.data_ptr() == v_cache.data_ptr() or k_scale.data_ptr() == v_scale.data_ptr():
        raise ValueError(f"{name}: keys and values are the same memory")
    rot = n_pos = rs = 0
    if rotary is not None:
        if rotary.dim() != 2 or rotary.dtype != torch.float32 or rotary.get_device() != dev:
            raise ValueError(f"{name}: rotary must be a float32 table (n_pos, rot_dim) on {k.device}")
        n_pos, rot = rotary.shape
        rs, r1 = rotary.stride()
        if n_pos < 1 or rot < 2 or rot % 2 or rot > hd or r1 != 1 or rs < rot:
            raise ValueError(f"{name}: rotary must have rows of an even rot_dim of at most {hd} values, got "
                             f"{tuple(rotary.shape)} with strides {rotary.stride()}")
    hq, qr, qs, qh, os_, oh = hkv, None, 0, 0, 0, 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != hd or q.dtype != k.dtype or q.get_device() != dev:
            raise ValueError(f"{name}: q must be {k.dtype} rows ({n}, n_head, {hd}), got {q.dtype} {tuple(q.shape)}")
        hq = q.shape[1]
        if hq == 0 or hq % hkv:
            raise ValueError(f"{name}: n_head {hq} is not a multiple of n_kv_head {hkv}")
        if q_out is None:
            q_out = q.new_empty((n, hq, hd))
        else:
            _check_out(name, q_out, q, vec)
        qr, qs, qh = _rows(q, vec)
        os_, oh, _ = q_out.stride()
    elif q_out is not None:
        raise ValueError(f"{name}: q_out without q")
    kr, ks, kh = _rows(k, vec)
    vr, vs, vh = _rows(v, vec)
    _launch(_lib.load().cgpt_paged_kv_append_8bit, _lib.paged8_args(
        _ptr(qr), kr.data_ptr(), vr.data_ptr(), _ptr(q_out), k_cache.data_ptr(), v_cache.data_ptr(),
        block_table.data_ptr(), seq_lens.data_ptr(), _ptr(cu_q), 0, _ptr(rotary), 0, _ptr(err_flag), 0,
        n, B, hq, hkv, hd, n_pages, page, cols, ts, 0, qs, qh, ks, kh, vs, vh, os_, oh, *cs,
        rot, n_pos, rs, bool(interleaved), dt, 0.0,
        k_scale.data_ptr(), v_scale.data_ptr(), 0, *ss, 0, 0, block, code), dev, name)
    return q_out


def paged_kv_read_8bit(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                       block_table: torch.Tensor, seq_lens: torch.Tensor, cu_rows: torch.Tensor, n_rows: int,
                       dtype: torch.dtype = torch.bfloat16, k_out: Optional[torch.Tensor] = None,
                       v_out: Optional[torch.Tensor] = None,
                       err_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values as ``dtype`` rows (n_rows, n_kv_head, head_dim): rows
    ``cu_rows[b] .. cu_rows[b + 1] - 1`` (int32, B + 1 offsets) are the last of sequence b,
    all of them where the offsets count its length, in order of their positions.

    code * 2^e, exact in float32 and bfloat16 (but for float8 NaN codes, which are NaN),
    rounded in float16.  Rows that the cache does not hold (more rows than the length, or
    a length past the table) are zeros; rows behind ``cu_rows[B]`` are left as they were
    (``k_out`` and ``v_out``) or undefined."""
    name = "paged_kv_read_8bit"
    dev = k_cache.get_device() if isinstance(k_cache, torch.Tensor) else -1
    if cu_rows is None or isinstance(n_rows, bool) or not isinstance(n_rows, int) or n_rows < 0:
        raise ValueError(f"{name}: cu_rows must be offsets and n_rows an int >= 0, got {n_rows!r}")
    code, n_pages, hkv, page, hd, cs, ss, block, B, cols, ts = _check_cache8(
        name, dev, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_rows, err_flag)
    dt = _CODE.get(dtype)
    if dt is None:
        raise ValueError(f"{name}: unsupported dtype {dtype} (float32, bfloat16 or float16)")
    vec = 8 if dt else 4
    outs = []
    for out in (k_out, v_out):
        if out is None:
            out = torch.empty((n_rows, hkv, hd), dtype=dtype, device=k_cache.device)
        elif not isinstance(out, torch.Tensor) or out.shape != (n_rows, hkv, hd) or out.dtype != dtype or out.get_device() != dev:
            raise ValueError(f"{name}: k_out and v_out must be {dtype} tensors of shape {(n_rows, hkv, hd)} on "
                             f"{k_cache.device}")
        else:
            _check_out(name, out, out, vec)
        outs.append(out)
    k_out, v_out = outs
    if n_rows and k_out.data_ptr() == v_out.data_ptr():
        raise ValueError(f"{name}: k_out and v_out are the same memory")
    (os_, oh, _), (vos, voh, _) = k_out.stride(), v_out.stride()
    _launch(_lib.load().cgpt_paged_kv_read_8bit, _lib.paged8_args(
        0, 0, 0, k_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), cu_rows.data_ptr(), 0, 0, 0, _ptr(err_flag), 0,
        n_rows, B, hkv, hkv, hd, n_pages, page, cols, ts, 0, 0, 0, 0, 0, 0, 0, os_, oh, *cs,
        0, 0, 0, 0, dt, 0.0,
        k_scale.data_ptr(), v_scale.data_ptr(), v_out.data_ptr(), *ss, vos, voh, block, code), dev, name)
    return k_out, v_out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes8(n: int, B: int, hq: int, hkv: int, hd: int, page: int, cols: int, dt: int, code: int,
                      device: int) -> int:
    """The C ABI's answer for these sizes (it goes by the device's CU count too)."""
    out = ctypes.c_int64()
    size = dict(n_tokens=n, B=B, Hq=hq, Hkv=hkv, head_dim=hd, page_size=page, max_pages=cols, dtype=dt, code=code)
    args = _lib.paged8_args(*(size.get(f, 0) for f in _lib.PAGED8_FIELDS))
    with torch.cuda.device(device):
        _lib.check(_lib.load().cgpt_paged_attention_8bit_workspace(args, ctypes.byref(out)),
                   "paged_attention_8bit_workspace")
    return out.value


def paged_attention_8bit(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         cu_q: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None, err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attention`` over a cache in 8 bits: causal softmax attention of the step's
    queries (n_tokens, n_head, head_dim; float32, bfloat16 or float16) over their
    sequences' pages; returns the same shape and type.

    Cached values are taken exactly as code * 2^e.  Queries and probabilities enter the
    products with the bits of the queries' type at least, statistics and sums are float32:
    under bfloat16 queries the probabilities are rounded to bfloat16, as in
    ``paged_attention``; float16 and float32 queries keep 16 and 24 bits of them."""
    name = "paged_attention_8bit"
    try:
        dev = q.get_device()
    except AttributeError:
        dev = -1
    code, n_pages, hkv, page, hd, cs, ss, block, B, cols, ts = _check_cache8(
        name, dev, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_q, err_flag)
    dt = _check_rows8(name, "q", q, B, hd, cu_q)
    n, hq, _ = q.shape
    if hq == 0 or hq % hkv:
        raise ValueError(f"{name}: n_head {hq} is not a multiple of n_kv_head {hkv}")
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    elif not 0.0 < scale < math.inf:
        raise ValueError(f"{name}: scale must be positive and finite, got {scale}")
    vec = 8 if dt else 4
    if out is None:
        out = q.new_empty((n, hq, hd))
    else:
        _check_out(name, out, q, vec)
    qr, qs, qh = _rows(q, vec)
    os_, oh, _ = out.stride()
    size = _workspace_bytes8(n, B, hq, hkv, hd, page, cols, dt, code, dev)
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _launch(_lib.load().cgpt_paged_attention_8bit, _lib.paged8_args(
        qr.data_ptr(), 0, 0, out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), _ptr(cu_q), 0, 0, _ptr(ws), _ptr(err_flag), size,
        n, B, hq, hkv, hd, n_pages, page, cols, ts, 0, qs, qh, 0, 0, 0, 0, os_, oh, *cs,
        0, 0, 0, 0, dt, scale,
        k_scale.data_ptr(), v_scale.data_ptr(), 0, *ss, 0, 0, block, code), dev, name)
    return out
