"""A paged key-value cache: writing it, and the attention that reads it.

Keys and values live in pools of pages, ``k_cache`` and ``v_cache`` of shape
(n_pages, n_kv_head, page_size, head_dim).  Row b of ``block_table`` (int32) names
the pages of sequence b in order: its key at position t is in slot t % page_size of
page ``block_table[b, t // page_size]``.  ``seq_lens[b]`` (int32) counts the
sequence's keys with those of the step's tokens, which are its last ones; a row of
length 0 is padding.

The step's tokens are packed rows (n_tokens, heads, head_dim), views into a fused
projection among them: one token a sequence, or, with ``cu_q`` (int32, B + 1
offsets), tokens ``cu_q[b] .. cu_q[b + 1] - 1`` for sequence b.  Rows behind
``cu_q[B]`` are padding: nothing is read for them and their output rows are left as
they were.

    q = paged_kv_append(k, v, k_cache, v_cache, table, lens, q=q, rotary=angles)
    o = paged_attention(q, k_cache, v_cache, table, lens)

``shared_prefix_attention`` is ``paged_attention`` for a batch whose sequences begin
with the same pages (samples of one prompt, users behind one document): those are
read once for all sequences.

Head counts may differ (n_head a multiple of n_kv_head); head_dim is 16, 32, 64 or
128; float32, bfloat16 or float16, one dtype a call; any page size (a table row names
fewer than 2^30 keys, a call holds some 2^26 rows of one head).  The reference
keeps no cache (``cutile_gpt/models/gpt.py:185-229`` runs the whole prefix again for
every token; its attention is ``cutile_gpt/kernels/attention.py:24-175``).

Lengths, tables and offsets stay on the device and are not copied to the host, so a
captured step replays with the values of the moment.  What the host cannot see is
made harmless instead: a page outside the pool is not written, and read as page 0; a
length past the table's pages is cut there; a position past the rotation table takes
its last row.  Each sets ``err_flag`` (one int32) to 1 when it is given.  Two tokens
of one call must not name the same slot.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch

from . import _lib

__all__ = ["rotary_table", "paged_kv_append", "paged_attention", "shared_prefix_attention"]

_HEAD_DIMS = (16, 32, 64, 128)


def rotary_table(n_pos: int, rot_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """Rotation angles of positions 0 .. n_pos - 1 for ``paged_kv_append``:
    (n_pos, rot_dim) float32, row t holding the cosines and then the sines of
    t * base ** (-2 i / rot_dim), i < rot_dim / 2, computed in float64."""
    if n_pos < 1 or rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rotary_table: n_pos >= 1 and an even rot_dim, got {n_pos} and {rot_dim}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
    t = torch.arange(n_pos, dtype=torch.float64, device=device)
    w = t[:, None] * float(base) ** (-i / rot_dim)
    return torch.cat([w.cos(), w.sin()], 1).float()


_CODE = {torch.float32: _lib.CGPT_F32, torch.bfloat16: _lib.CGPT_BF16, torch.float16: _lib.CGPT_F16}


def _rows(t: torch.Tensor, vec: int):
    """(n, heads, hd) rows that 16-byte loads can read, the view itself or a copy, and
    their strides."""
    s0, s1, s2 = t.stride()
    if s2 != 1 or s0 % vec or s1 % vec or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        s0, s1, _ = t.stride()
    return t, s0, s1


def _check_out(name: str, out: torch.Tensor, like: torch.Tensor, vec: int) -> None:
    if (not isinstance(out, torch.Tensor) or out.shape != like.shape or out.dtype != like.dtype
            or out.device != like.device):
        raise ValueError(f"{name}: the output must be a {like.dtype} tensor of shape {tuple(like.shape)} "
                         f"on {like.device}")
    s0, s1, s2 = out.stride()
    n, h, hd = out.shape
    # Apart when the larger stride reaches past what the smaller one places.
    near = hd
    for stride, extent in sorted(((s0, n), (s1, h))):
        if extent > 1:
            near = near + stride * (extent - 1) if stride >= near else math.inf
    if s2 != 1 or s0 % vec or s1 % vec or out.data_ptr() % 16 or near == math.inf:
        raise ValueError(f"{name}: the output's rows must be separate, contiguous and 16-byte aligned")


def _check_cache(name: str, x: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_table: torch.Tensor, seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor],
                 err_flag: Optional[torch.Tensor]):
    """Checks what every entry point takes, as far as the native call cannot (it refuses
    sizes, strides and alignments that the kernels do not take); returns the rows' device
    index, the dtype's code, the elements in 16 bytes, the caches' sizes and strides and
    the table's sizes and row stride."""
    try:
        dev, dt = x.get_device(), x.dtype
        same = (dev == k_cache.get_device() == v_cache.get_device() == block_table.get_device()
                == seq_lens.get_device() and (cu_q is None or cu_q.get_device() == dev)
                and (err_flag is None or err_flag.get_device() == dev))
    except AttributeError:
        same, dev = False, -1
    if not same or dev < 0:
        raise ValueError(f"{name}: tensors must be torch tensors on one GPU")
    code = _CODE.get(dt)
    if code is None:
        raise ValueError(f"{name}: unsupported dtype {dt} (float32, bfloat16 or float16)")
    if k_cache.dtype is not dt or v_cache.dtype is not dt:
        raise ValueError(f"{name}: the caches hold {k_cache.dtype} and {v_cache.dtype}, the rows {dt}")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"{name}: k_cache and v_cache must share a shape (n_pages, n_kv_head, page_size, "
                         f"head_dim), got {tuple(shape)} and {tuple(v_cache.shape)}")
    n_pages, heads, page, hd = shape
    rows = x.shape
    if len(rows) != 3 or rows[2] != hd:
        raise ValueError(f"{name}: the step's rows must be (n_tokens, heads, {hd}), got {tuple(rows)}")
    if hd not in _HEAD_DIMS:
        raise ValueError(f"{name}: head_dim {hd} is not one of {_HEAD_DIMS}")
    kp, kh, ks, kd = k_cache.stride()
    vp, vh, vs, vd = v_cache.stride()
    if kd != 1 or vd != 1:
        raise ValueError(f"{name}: cache rows must be contiguous")
    if block_table.dtype is not torch.int32 or seq_lens.dtype is not torch.int32:
        raise ValueError(f"{name}: block_table and seq_lens must be int32")
    if block_table.dim() != 2 or seq_lens.dim() != 1:
        raise ValueError(f"{name}: block_table must be (B, pages) and seq_lens (B,), got "
                         f"{tuple(block_table.shape)} and {tuple(seq_lens.shape)}")
    B, cols = block_table.shape
    ts, t1 = block_table.stride()
    if (t1 != 1 and cols > 1) or not seq_lens.is_contiguous() or seq_lens.shape[0] != B:
        raise ValueError(f"{name}: block_table must have contiguous rows and seq_lens be {B} contiguous lengths")
    if cu_q is None:
        if rows[0] != B:
            raise ValueError(f"{name}: {rows[0]} rows for {B} sequences need cu_q")
    elif cu_q.dtype is not torch.int32 or cu_q.dim() != 1 or cu_q.shape[0] != B + 1 or not cu_q.is_contiguous():
        raise ValueError(f"{name}: cu_q must be {B + 1} contiguous int32 offsets, got {cu_q.dtype} {tuple(cu_q.shape)}")
    if err_flag is not None and (err_flag.dtype is not torch.int32 or err_flag.numel() != 1):
        raise ValueError(f"{name}: err_flag must be one int32")
    return dev, code, 8 if code else 4, n_pages, heads, page, hd, (kp, kh, ks, vp, vh, vs), B, cols, ts


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _launch(fn, args: bytes, dev: int, name: str) -> None:
    """One native call on the rows' device, on its current stream."""
    if dev == torch._C._cuda_getDevice():
        rc = fn(args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, name)


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                    q: Optional[torch.Tensor] = None, rotary: Optional[torch.Tensor] = None,
                    interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                    err_flag: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the step's keys and values (n_tokens, n_kv_head, head_dim) into their
    pages, in place.

    ``rotary`` (n_pos, rot_dim) float32 (``rotary_table``) turns the first rot_dim
    values of every key, and of the queries ``q`` (n_tokens, n_head, head_dim), by
    their positions on the way: pairs (i, i + rot_dim / 2), or (2 i, 2 i + 1) with
    ``interleaved``, in float32, rounded once.  Returns the turned queries (in
    ``q_out`` when given, which may be ``q`` but shares no memory with ``k`` or
    ``v``), None without ``q``."""
    name = "paged_kv_append"
    dev, code, vec, n_pages, hkv, page, hd, cs, B, cols, ts = _check_cache(
        name, k, k_cache, v_cache, block_table, seq_lens, cu_q, err_flag)
    if not all(t is None or isinstance(t, torch.Tensor) for t in (v, q, rotary)):
        raise ValueError(f"{name}: k, v, q and rotary must be torch tensors")
    n = k.shape[0]
    if v.shape != k.shape or v.dtype != k.dtype or v.get_device() != dev or k.shape[1] != hkv:
        raise ValueError(f"{name}: k and v must be {k.dtype} (n_tokens, {hkv}, {hd}) rows, got "
                         f"{tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    if k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError(f"{name}: k_cache and v_cache are the same memory")
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
    _launch(_lib.load().cgpt_paged_kv_append, _lib.paged_args(
        _ptr(qr), kr.data_ptr(), vr.data_ptr(), _ptr(q_out), k_cache.data_ptr(), v_cache.data_ptr(),
        block_table.data_ptr(), seq_lens.data_ptr(), _ptr(cu_q), 0, _ptr(rotary), 0, _ptr(err_flag), 0,
        n, B, hq, hkv, hd, n_pages, page, cols, ts, 0, qs, qh, ks, kh, vs, vh, os_, oh, *cs,
        rot, n_pos, rs, bool(interleaved), code, 0.0), dev, name)
    return q_out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(n: int, B: int, hq: int, hkv: int, hd: int, page: int, cols: int, prefix: int,
                     code: int, device: int) -> int:
    """The C ABI's answer for these sizes (it goes by the device's CU count too)."""
    out = ctypes.c_int64()
    size = dict(n_tokens=n, B=B, Hq=hq, Hkv=hkv, head_dim=hd, page_size=page, max_pages=cols, prefix_len=prefix,
                dtype=code)
    args = _lib.paged_args(*(size.get(f, 0) for f in _lib.PAGED_FIELDS))
    with torch.cuda.device(device):
        _lib.check(_lib.load().cgpt_paged_attention_workspace(args, ctypes.byref(out)), "paged_attention_workspace")
    return out.value


def _attend(name: str, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
            seq_lens: torch.Tensor, prefix_len: int, prefix_pages: Optional[torch.Tensor],
            cu_q: Optional[torch.Tensor], scale: Optional[float], out: Optional[torch.Tensor],
            err_flag: Optional[torch.Tensor]) -> torch.Tensor:
    dev, code, vec, n_pages, hkv, page, hd, cs, B, cols, ts = _check_cache(
        name, q, k_cache, v_cache, block_table, seq_lens, cu_q, err_flag)
    n, hq, _ = q.shape
    if hq == 0 or hq % hkv:
        raise ValueError(f"{name}: n_head {hq} is not a multiple of n_kv_head {hkv}")
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    elif not 0.0 < scale < math.inf:
        raise ValueError(f"{name}: scale must be positive and finite, got {scale}")
    if out is None:
        out = q.new_empty((n, hq, hd))
    else:
        _check_out(name, out, q, vec)
    qr, qs, qh = _rows(q, vec)
    os_, oh, _ = out.stride()
    size = _workspace_bytes(n, B, hq, hkv, hd, page, cols, prefix_len, code, dev)
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    pages = 0 if not prefix_len else (block_table if prefix_pages is None else prefix_pages).data_ptr()
    _launch(_lib.load().cgpt_paged_attention, _lib.paged_args(
        qr.data_ptr(), 0, 0, out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), _ptr(cu_q), pages, 0, _ptr(ws), _ptr(err_flag), size,
        n, B, hq, hkv, hd, n_pages, page, cols, ts, prefix_len, qs, qh, 0, 0, 0, 0, os_, oh, *cs,
        0, 0, 0, 0, code, scale), dev, name)
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal softmax attention of the step's queries (n_tokens, n_head, head_dim)
    over their sequences' pages; returns the same shape.

    A sequence's m tokens sit at its last m positions and see the keys up to their
    own; a token that sees none (a padding row) gives zeros.  Query head h reads key
    head h // (n_head / n_kv_head).  ``scale`` defaults to 1/sqrt(head_dim).
    Softmax statistics and sums are float32; the probabilities are rounded to the
    dtype before they meet the values, as in ``cutile_causal_attention``."""
    return _attend("paged_attention", q, k_cache, v_cache, block_table, seq_lens, 0, None, cu_q, scale, out,
                   err_flag)


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            block_table: torch.Tensor, seq_lens: torch.Tensor, prefix_len: int,
                            prefix_pages: Optional[torch.Tensor] = None, cu_q: Optional[torch.Tensor] = None,
                            scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                            err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attention`` for sequences whose first ``prefix_len`` keys are the same
    pages, which are read once for the batch.

    The prefix is read from ``prefix_pages`` (int32, at least prefix_len / page_size
    pages), by default the first row of ``block_table``; lengths and positions count
    it, and the rows' own entries for it are not read.  A sequence may be shorter
    than the prefix."""
    name = "shared_prefix_attention"
    if isinstance(prefix_len, bool) or not isinstance(prefix_len, int) or prefix_len < 0:
        raise ValueError(f"{name}: prefix_len must be an int >= 0, got {prefix_len!r}")
    if not all(isinstance(t, torch.Tensor) for t in (q, k_cache, block_table)):
        raise ValueError(f"{name}: tensors must be torch tensors on one GPU")
    if k_cache.dim() == 4 and block_table.dim() == 2:
        page = k_cache.shape[2]
        if prefix_len > page * block_table.shape[1]:
            raise ValueError(f"{name}: prefix_len {prefix_len} exceeds the {block_table.shape[1]} pages of a "
                             f"block_table row")
        if prefix_pages is not None and (
                not isinstance(prefix_pages, torch.Tensor) or prefix_pages.dim() != 1 or prefix_pages.dtype != torch.int32 or prefix_pages.device != q.device
                or not prefix_pages.is_contiguous() or prefix_pages.shape[0] * page < prefix_len):
            raise ValueError(f"{name}: prefix_pages must be a contiguous int32 list of at least "
                             f"{-(-prefix_len // max(page, 1))} pages on {q.device}")
        if block_table.shape[0] == 0 and prefix_pages is None:
            prefix_len = 0
    return _attend(name, q, k_cache, v_cache, block_table, seq_lens, prefix_len, prefix_pages, cu_q, scale, out,
                   err_flag)
