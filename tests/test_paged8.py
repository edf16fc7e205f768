"""The 8-bit paged cache without a GPU: the checks of the C entry points (nothing is
launched) and of the wrappers, and the tests' own oracle."""

import ctypes
import math

import pytest
import torch

import cutilegpt_amd as cg
from cutilegpt_amd import _lib
from paged8_ref import F8, HI, LO, TOP, Problem8, append, exponent, grid, nearest

P = 1 << 20  # a pointer that is never followed
EINVAL, EDTYPE, ESHAPE, ESCRATCH = -1, -2, -3, -4
APPEND, READ, ATTEND = "cgpt_paged_kv_append_8bit", "cgpt_paged_kv_read_8bit", "cgpt_paged_attention_8bit"
FNS = [APPEND, READ, ATTEND]


def fields(**change):
    """Well-formed arguments with no token (nothing to launch), changed."""
    a = dict(q=P, k=P, v=P, out=P, k_cache=P, v_cache=2 * P, block_table=P, seq_lens=P, cu_q=P, prefix_pages=0, rotary=P,
             workspace=0, err_flag=0, workspace_bytes=0, n_tokens=0, B=2, Hq=4, Hkv=2, head_dim=64, n_pages=8, page_size=16,
             max_pages=4, bt_stride=4, prefix_len=0, kc_sp=2048, kc_sh=1024, kc_ss=64, vc_sp=2048, vc_sh=1024, vc_ss=64,
             rot_dim=64, n_pos=64, rot_stride=64, interleaved=0, dtype=_lib.CGPT_BF16, scale=0.125,
             k_scale=3 * P, v_scale=4 * P, v_out=5 * P, ks_sp=8, ks_sh=4, ks_sb=1, vs_sp=8, vs_sh=4, vs_sb=1,
             vo_st=128, vo_sh=64, block=4, code=_lib.CGPT_E4M3)
    a.update({f"{x}_{s}": n for x in ("q", "k", "v", "out") for s, n in (("st", 256), ("sh", 64))})
    assert set(change) <= set(a) and set(a) == set(_lib.PAGED8_FIELDS)
    a.update(change)
    return _lib.paged8_args(*(a[f] for f in _lib.PAGED8_FIELDS))


def call(fn, **change):
    return getattr(_lib.load(), fn)(fields(**change), None)


SIZES = [(dict(n_tokens=-1), EINVAL), (dict(B=-1), EINVAL), (dict(Hq=3), EINVAL), (dict(Hkv=0), EINVAL),
         (dict(page_size=0), EINVAL), (dict(n_pages=0), EINVAL), (dict(max_pages=-1), EINVAL), (dict(bt_stride=-1), EINVAL),
         (dict(k_cache=0), EINVAL), (dict(v_cache=P + 8), EINVAL), (dict(kc_sp=2040), EINVAL), (dict(vc_ss=48), EINVAL),
         (dict(kc_ss=0), EINVAL), (dict(vc_sp=0), EINVAL), (dict(kc_sh=0), EINVAL), (dict(dtype=7), EDTYPE),
         (dict(head_dim=48), ESHAPE), (dict(head_dim=256), ESHAPE), (dict(page_size=1 << 20, max_pages=1 << 11), ESHAPE),
         (dict(n_tokens=1 << 30), ESHAPE), (dict(n_pages=1 << 31), ESHAPE), (dict(code=2), EDTYPE), (dict(code=-1), EDTYPE),
         (dict(block=0), EINVAL), (dict(block=3), EINVAL), (dict(block=32), EINVAL), (dict(k_scale=0), EINVAL),
         (dict(v_scale=0), EINVAL), (dict(ks_sp=0), EINVAL), (dict(vs_sh=0), EINVAL), (dict(ks_sb=0), EINVAL)]


@pytest.mark.parametrize("fn", FNS)
def test_c_entry_points_refuse(fn):
    assert call(fn) == 0
    assert getattr(_lib.load(), fn)(None, None) == EINVAL
    for change, status in SIZES:
        assert call(fn, **change) == status, change
    # With a token the pointers and strides of the rows count too.
    for change in (dict(seq_lens=0), dict(block_table=0), dict(q_st=255), dict(out_sh=4), dict(out_st=8), dict(cu_q=0),
                   dict(q=P + 8), dict(out=P + 2), dict(k_st=-8), dict(vo_st=12), dict(v_out=P + 4)):
        assert call(fn, n_tokens=3, **change) == EINVAL, change


def test_c_append_refuses():
    for change, status in ((dict(q=0), EINVAL), (dict(v_cache=P), EINVAL), (dict(v_scale=3 * P), EINVAL),
                           (dict(rot_dim=3), ESHAPE), (dict(rot_dim=66), ESHAPE), (dict(rot_dim=-2), ESHAPE),
                           (dict(n_pos=0), EINVAL), (dict(rot_stride=62), EINVAL), (dict(rotary=0), EINVAL),
                           (dict(rotary=P + 1), EINVAL),
                           # Rows or exponents that would be written over one another.
                           (dict(kc_sp=1024), EINVAL), (dict(vc_sh=512), EINVAL), (dict(ks_sp=4), EINVAL), (dict(vs_sh=3), EINVAL)):
        assert call(APPEND, **change) == status, change
    for change in (dict(k=0), dict(v=P + 2), dict(out_st=64)):
        assert call(APPEND, n_tokens=3, **change) == EINVAL, change
    assert call(APPEND, rot_dim=0, rotary=0, q=0, out=0) == 0
    # Launches of 2^32 threads and more.
    assert call(APPEND, n_tokens=1 << 20, B=1 << 20, Hq=2048, Hkv=1, head_dim=16) == ESHAPE


def test_c_read_refuses():
    for change in (dict(out=0), dict(v_out=0), dict(out_st=64), dict(vo_st=64)):
        assert call(READ, n_tokens=3, **change) == EINVAL, change


def workspace(**change):
    out = ctypes.c_int64(-1)
    return _lib.load().cgpt_paged_attention_8bit_workspace(fields(**change), ctypes.byref(out)), out.value


def test_c_attention_refuses():
    for change in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e-60),
                   dict(scale=1e60), dict(scale=3e38)):
        assert call(ATTEND, **change) == EINVAL, change
    for change in (dict(q=0), dict(out=0), dict(out_st=64)):
        assert call(ATTEND, n_tokens=3, **change) == EINVAL, change
    # A workspace that is missing, too small or unaligned is refused before any launch.
    long = dict(n_tokens=2, cu_q=0, max_pages=4096, bt_stride=4096)
    status, size = workspace(**long)
    assert status == 0 and size > 64
    assert call(ATTEND, **long) == ESCRATCH
    assert call(ATTEND, **long, workspace=P, workspace_bytes=size - 1) == ESCRATCH
    assert call(ATTEND, **long, workspace=P + 8, workspace_bytes=1 << 40) == EINVAL
    assert call(ATTEND, n_tokens=1 << 20, B=1 << 20, cu_q=0, Hq=1 << 11, Hkv=1) == ESHAPE


def test_workspace_size():
    assert workspace(n_tokens=0) == (0, 0) and workspace(n_tokens=4, B=0) == (0, 0)
    # Short sequences need none, with offsets or without.
    for cu in (0, P):
        assert workspace(n_tokens=8, B=8, cu_q=cu, max_pages=8) == (0, 0)
    assert _lib.load().cgpt_paged_attention_8bit_workspace(None, None) == EINVAL
    for change, status in SIZES:
        if set(change) & {"n_tokens", "B", "Hq", "Hkv", "page_size", "max_pages", "dtype", "head_dim", "code"}:
            assert workspace(**{"n_tokens": 4, **change})[0] == status, change


def test_wrappers_refuse_host_tensors():
    p = Problem8(torch.bfloat16, F8, 64, 16, 16, 2, 2, ctx=[3], new=[1])
    with pytest.raises(ValueError, match="one GPU"):
        cg.paged_kv_append_8bit(p.k, p.v, *p.cache)
    with pytest.raises(ValueError, match="one GPU"):
        cg.paged_attention_8bit(p.q, *p.cache)
    with pytest.raises(ValueError, match="one GPU"):
        cg.paged_kv_read_8bit(*p.cache, p.cu_rows, 4)
    with pytest.raises(ValueError, match="n_rows"):
        cg.paged_kv_read_8bit(*p.cache, p.cu_rows, -1)
    with pytest.raises(ValueError):
        cg.paged_kv_append_8bit(1, p.v, *p.cache)


@pytest.mark.parametrize("code", [F8, torch.int8])
def test_oracle_against_brute_force(code):
    """The oracle's rounding: no code is nearer, ties go to even; its exponent is the smallest."""
    g = torch.Generator().manual_seed(1)
    numbers = grid(code)
    y = torch.randn(2000, generator=g, dtype=torch.float64) * TOP[code] / 3
    y = torch.cat([y, (numbers[1:] + numbers[:-1]) / 2, numbers])
    r = nearest(y, code)
    signed = torch.cat([-numbers.flip(0), numbers])
    best = (y[:, None] - signed).abs().amin(1)
    assert torch.equal((y - r).abs(), best) and bool((r.abs() <= TOP[code]).all())
    mids = (numbers[1:] + numbers[:-1]) / 2
    at = torch.searchsorted(numbers, nearest(mids, code))
    assert bool((at % 2 == 0).all())
    for x in (1e-40, 3.0, 448.0, 449.0, 127.0, 127.5, 1e30, 3.3e38):
        e = exponent(torch.tensor([x, -x / 2], dtype=torch.float64), code)
        fits = x <= TOP[code] * 2.0 ** e
        assert LO <= e <= HI[code] and (fits or e == HI[code]) and (e == LO or x > TOP[code] * 2.0 ** (e - 1))


def test_oracle_append_keeps_and_renews():
    """A block that a step goes on in keeps the larger exponent, one that it begins starts anew."""
    p = Problem8(torch.float32, torch.int8, 16, 4, 4, 1, 1, ctx=[2, 4], new=[1, 1])
    p.k[:] = 1e-6
    out, _ = append(p)
    on, anew = int(p.table[0, 0]), int(p.table[1, 1])
    assert int(out[2][on, 0, 0]) == int(p.k_scale[on, 0, 0])
    assert int(out[2][anew, 0, 0]) == 127 + exponent(p.k[1].double(), torch.int8) < 127 - 20
    assert torch.equal(out[0][on, 0, :2], p.k_cache[on, 0, :2])
