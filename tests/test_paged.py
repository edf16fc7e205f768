"""The paged cache without a GPU: the checks of the C entry points (nothing is launched),
of the wrappers, the rotation table and the tests' own oracle."""

import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import cutilegpt_amd as cg
from cutilegpt_amd import _lib
from paged_ref import Problem, append, attention

P = 1 << 20  # a pointer that is never followed


def call(fn, **change):
    """fn of libcgpt.so on well-formed sizes with no token (nothing to launch), changed."""
    a = dict(q=P, k=P, v=P, out=P, k_cache=P, v_cache=2 * P, block_table=P, seq_lens=P, cu_q=P, prefix_pages=P, rotary=P,
             workspace=0, err_flag=0, workspace_bytes=0, n_tokens=0, B=2, Hq=4, Hkv=2, head_dim=64, n_pages=8, page_size=16,
             max_pages=4, bt_stride=4, prefix_len=16, kc_sp=2048, kc_sh=1024, kc_ss=64, vc_sp=2048, vc_sh=1024, vc_ss=64,
             rot_dim=64, n_pos=64, rot_stride=64, interleaved=0, dtype=_lib.CGPT_BF16, scale=0.125)
    a.update({f"{x}_{s}": n for x in ("q", "k", "v", "out") for s, n in (("st", 256), ("sh", 64))})
    assert set(change) <= set(a) and set(a) == set(_lib.PAGED_FIELDS)
    a.update(change)
    args = _lib.paged_args(*(a[f] for f in _lib.PAGED_FIELDS))
    return getattr(_lib.load(), fn)(args, None)


EINVAL, EDTYPE, ESHAPE, ESCRATCH = -1, -2, -3, -4
SIZES = [(dict(n_tokens=-1), EINVAL), (dict(B=-1), EINVAL), (dict(Hq=3), EINVAL), (dict(Hkv=0), EINVAL),
         (dict(page_size=0), EINVAL), (dict(n_pages=0), EINVAL), (dict(max_pages=-1), EINVAL), (dict(bt_stride=-1), EINVAL),
         (dict(k_cache=0), EINVAL), (dict(v_cache=P + 8), EINVAL), (dict(kc_sp=2047), EINVAL), (dict(vc_ss=32), EINVAL),
         (dict(kc_ss=0), EINVAL), (dict(vc_sp=0), EINVAL), (dict(kc_sh=0), EINVAL), (dict(dtype=7), EDTYPE),
         (dict(head_dim=48), ESHAPE), (dict(head_dim=256), ESHAPE), (dict(page_size=1 << 20, max_pages=1 << 11), ESHAPE),
         (dict(n_tokens=1 << 30), ESHAPE), (dict(n_pages=1 << 31), ESHAPE)]
FNS = ["cgpt_paged_kv_append", "cgpt_paged_attention"]


@pytest.mark.parametrize("fn", FNS)
def test_c_entry_points_refuse(fn):
    assert call(fn) == 0
    assert getattr(_lib.load(), fn)(None, None) == EINVAL
    for change, status in SIZES:
        assert call(fn, **change) == status, change
    # With a token the pointers and strides of the rows count too.
    for change in (dict(seq_lens=0), dict(block_table=0), dict(q_st=255), dict(out_sh=4), dict(out_st=8), dict(cu_q=0),
                   dict(q=P + 8), dict(out=P + 2), dict(k_st=-8)):
        assert call(fn, n_tokens=3, **change) == EINVAL, change


def test_c_append_refuses():
    fn = FNS[0]
    for change, status in ((dict(q=0), EINVAL), (dict(v_cache=P), EINVAL), (dict(rot_dim=3), ESHAPE), (dict(rot_dim=66), ESHAPE),
                           (dict(rot_dim=-2), ESHAPE), (dict(n_pos=0), EINVAL), (dict(rot_stride=62), EINVAL),
                           (dict(rotary=0), EINVAL), (dict(rotary=P + 1), EINVAL)):
        assert call(fn, **change) == status, change
    for change in (dict(k=0), dict(v=P + 2)):
        assert call(fn, n_tokens=3, **change) == EINVAL, change
    assert call(fn, rot_dim=0, rotary=0, q=0, out=0) == 0


def test_c_attention_refuses():
    fn = FNS[1]
    for change in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e-60),
                   dict(scale=1e60), dict(scale=3e38), dict(prefix_len=-1), dict(prefix_len=65)):
        assert call(fn, **change) == EINVAL, change
    for change in (dict(prefix_pages=0), dict(q=0), dict(out=0)):
        assert call(fn, n_tokens=3, **change) == EINVAL, change
    # A workspace that is missing, too small or unaligned is refused before any launch.
    long = dict(n_tokens=2, cu_q=0, prefix_len=0, max_pages=4096, bt_stride=4096)
    assert call(fn, **long) == ESCRATCH
    assert call(fn, **long, workspace=P, workspace_bytes=64) == ESCRATCH
    assert call(fn, **long, workspace=P + 8, workspace_bytes=1 << 40) == EINVAL


def test_workspace_size():
    lib, n = _lib.load(), ctypes.c_int64(-1)
    size = dict(n_tokens=4, B=4, Hq=4, Hkv=2, head_dim=64, page_size=16, max_pages=4096, dtype=_lib.CGPT_BF16)

    def ask(**change):
        args = _lib.paged_args(*({**size, **change}.get(f, 0) for f in _lib.PAGED_FIELDS))
        return lib.cgpt_paged_attention_workspace(args, ctypes.byref(n))

    assert ask() == 0 and n.value > 0
    assert ask(n_tokens=0) == 0 and n.value == 0
    for change, status in ((dict(B=-1), EINVAL), (dict(Hq=3), EINVAL), (dict(prefix_len=-1), EINVAL), (dict(dtype=9), EDTYPE),
                           (dict(head_dim=80), ESHAPE)):
        assert ask(**change) == status, change
    assert lib.cgpt_paged_attention_workspace(None, ctypes.byref(n)) == EINVAL


@pytest.mark.parametrize("dtype", [_lib.CGPT_F32, _lib.CGPT_BF16])
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("group", [1, 4, 17])
def test_workspace_is_what_the_call_needs(dtype, hd, group):
    """The workspace's question holds sizes alone: its answer is enough, and no more than
    enough, for the call with offsets and, at one token a sequence, without.  (Every call is
    refused before a launch: a workspace off its alignment is, once it is large enough.)"""
    lib, n = _lib.load(), ctypes.c_int64(-1)
    seen = set()
    for Hkv in (1, 3, 12, 25):
        for B in (1, 10, 16, 20, 32, 33, 64, 300):
            for tokens in (1, B, B + 1, 2 * B, 4 * B, 9 * B, 16 * B, 17 * B, 70 * B):
                for cols in (1, 64, 128, 144, 400):
                    for prefix in (0, 16, 2048):
                        if prefix > 16 * cols:
                            continue
                        size = dict(n_tokens=tokens, B=B, Hq=group * Hkv, Hkv=Hkv, head_dim=hd, page_size=16, max_pages=cols,
                                    prefix_len=prefix, dtype=dtype)
                        args = _lib.paged_args(*(size.get(f, 0) for f in _lib.PAGED_FIELDS))
                        assert lib.cgpt_paged_attention_workspace(args, ctypes.byref(n)) == 0, size
                        seen.add(n.value > 0)
                        size.update(q_st=size["Hq"] * hd, q_sh=hd, out_st=size["Hq"] * hd, out_sh=hd)
                        size.update({f"{c}_{s}": v for c in ("kc", "vc") for s, v in (("sp", Hkv * 16 * hd), ("sh", 16 * hd), ("ss", hd))})
                        for cu in (P, 0) if tokens == B else (P,):
                            assert call(FNS[1], **size, cu_q=cu, workspace=P + 8, workspace_bytes=n.value) == EINVAL, (size, cu)
                            if n.value:
                                short = dict(workspace=P + 8, workspace_bytes=n.value - 1)
                                assert call(FNS[1], **size, cu_q=cu, **short) == ESCRATCH, (size, cu)
    assert seen == {False, True}


def test_wrappers_refuse_host_tensors():
    p = Problem(torch.float32, 16, 8, 2, 2, ctx=[3], new=[1])
    with pytest.raises(ValueError):
        cg.paged_attention(p.q, p.k_cache, p.v_cache, p.table, p.lens)
    with pytest.raises(ValueError):
        cg.shared_prefix_attention(p.q, p.k_cache, p.v_cache, p.table, p.lens, 8)
    with pytest.raises(ValueError):
        cg.paged_kv_append(p.k, p.v, p.k_cache, p.v_cache, p.table, p.lens)


def test_rotary_table():
    t = cg.rotary_table(70000, 8, base=1000.0, device="cpu")
    assert t.shape == (70000, 8) and t.dtype == torch.float32
    for pos, i in ((0, 0), (1, 3), (69999, 0), (69999, 2)):
        w = pos * 1000.0 ** (-2 * i / 8)
        assert abs(t[pos, i].item() - math.cos(w)) < 1e-7 and abs(t[pos, 4 + i].item() - math.sin(w)) < 1e-7
    for bad in ((0, 8), (4, 3), (4, 0)):
        with pytest.raises(ValueError):
            cg.rotary_table(*bad, device="cpu")


def test_oracle_against_dense_softmax():
    """The oracle's pages against softmax attention of the dense rows it was made from."""
    p = Problem(torch.float32, 16, 8, 4, 2, ctx=[9, 0], new=[4, 11], seed=1)
    kc, vc, _, _, _ = append(p)
    p.k_cache, p.v_cache = kc.float(), vc.float()
    out, bound = attention(p)
    for b in range(2):
        k, v = p.keys(b)
        n, m = p.total[b], p.new[b]
        assert torch.equal(k[n - m:].float(), p.k[int(p.cu[b]):int(p.cu[b + 1])])
        q = p.q[int(p.cu[b]):int(p.cu[b + 1])].double()
        s = torch.einsum("thd,jhd->htj", q, k.repeat_interleave(2, 1)) / 4
        s += torch.full((m, n), -math.inf, dtype=torch.float64).triu(n - m + 1)
        want = torch.einsum("htj,jhd->thd", s.softmax(-1), v.repeat_interleave(2, 1))
        assert (out[int(p.cu[b]):int(p.cu[b + 1])] - want).abs().max() < 1e-12
        assert (bound[int(p.cu[b]):int(p.cu[b + 1])] < 1e-3).all()


HUGE = [dict(n_tokens=1 << 38, B=1 << 38, Hq=1 << 32, Hkv=1 << 32, prefix_len=16, max_pages=4096),
        dict(n_tokens=1 << 62), dict(B=1 << 40),
        dict(Hq=1 << 20, Hkv=1 << 20), dict(page_size=1 << 40, max_pages=1 << 40), dict(max_pages=1 << 40),
        dict(n_tokens=1 << 29, Hq=16, Hkv=16), dict(page_size=1 << 20, max_pages=1 << 11), dict(head_dim=1 << 40)]


def test_workspace_refuses_the_sizes_that_the_call_does():
    """Sizes whose products leave 64 bits among them.  In a process of its own: a division by
    one of those, wrapped to zero, ends the process."""
    code = ("import ctypes, sys; sys.path[:0] = ['.', 'tests']\n"
            "from test_paged import HUGE, _lib\n"
            "lib, n = _lib.load(), ctypes.c_int64(-1)\n"
            "size = dict(n_tokens=4, B=4, Hq=4, Hkv=2, head_dim=64, page_size=16, max_pages=64, dtype=_lib.CGPT_BF16)\n"
            "for change in HUGE:\n"
            "    args = _lib.paged_args(*({**size, **change}.get(f, 0) for f in _lib.PAGED_FIELDS))\n"
            "    status = lib.cgpt_paged_attention_workspace(args, ctypes.byref(n))\n"
            "    assert (status, n.value) == (-3, 0), (change, status, n.value)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert res.returncode == 0, (res.returncode, res.stderr[-500:])
    for change in HUGE:
        assert call(FNS[1], **{**dict(bt_stride=64, max_pages=64, prefix_len=0), **change}) == ESHAPE, change


OVERLAPS = [dict(n_tokens=3, out_st=64, out_sh=64), dict(n_tokens=3, out_st=192, out_sh=64), dict(n_tokens=3, out_st=64, out_sh=128),
            dict(kc_sp=1024, kc_sh=1024), dict(kc_sp=2040), dict(vc_sh=1016), dict(vc_sp=64, vc_sh=504, vc_ss=1024),
            dict(vc_sp=2048, vc_sh=64, vc_ss=64), dict(kc_sp=1 << 62, kc_sh=1 << 62)]
APART = [dict(kc_sp=64, kc_sh=512, kc_ss=1024), dict(vc_sp=1024, vc_sh=64 * 128, vc_ss=64), dict(vc_sp=2048, vc_sh=64, vc_ss=128),
         dict(kc_sp=4096, kc_sh=2048, kc_ss=128), dict(n_pages=1, kc_sp=0), dict(Hq=1, Hkv=1, kc_sh=0, kc_sp=1024),
         dict(page_size=1, max_pages=64, kc_ss=0, prefix_len=0), dict(kc_sp=1 << 60)]


@pytest.mark.parametrize("fn", FNS)
def test_rows_that_overlap_are_refused(fn):
    """Pools that are written and outputs two of whose rows share memory: two blocks would
    write there."""
    for change in OVERLAPS:
        if "out_st" in change or fn == FNS[0]:
            assert call(fn, **{**dict(workspace=P + 8), **change}) == EINVAL, change
    for change in APART:
        assert call(fn, **change) == 0, change


def test_output_rows_that_overlap_are_refused():
    from cutilegpt_amd.paged import _check_out
    like = torch.empty(3, 4, 64)
    for strides in ((64, 64, 1), (192, 64, 1), (64, 128, 1), (0, 64, 1)):
        with pytest.raises(ValueError):
            _check_out("test", torch.empty(2000).as_strided((3, 4, 64), strides), like, 4)
    for strides in ((256, 64, 1), (64, 192, 1), (320, 80, 1)):
        _check_out("test", torch.empty(2000).as_strided((3, 4, 64), strides), like, 4)
    _check_out("test", torch.empty(64).as_strided((1, 1, 64), (0, 0, 1)), like[:1, :1], 4)


def test_wide_tables_of_many_sequences_are_taken():
    """Lengths that a table allows and no batch has: the plan's counts go by them."""
    lib, n = _lib.load(), ctypes.c_int64(-1)
    for dtype in (_lib.CGPT_F32, _lib.CGPT_BF16):
        for size in (dict(B=4096, n_tokens=4096, Hq=32, Hkv=32, page_size=256, max_pages=4096),
                     dict(B=4096, n_tokens=9000, Hq=32, Hkv=32, page_size=256, max_pages=4096),
                     dict(B=4096, n_tokens=4096, Hq=64, Hkv=8, page_size=16, max_pages=(1 << 26) - 1, prefix_len=4096),
                     dict(B=300, n_tokens=300, Hq=8, Hkv=8, page_size=1 << 15, max_pages=(1 << 15) - 1)):
            for hd in (16, 32, 64, 128):
                size.update(head_dim=hd, dtype=dtype)
                args = _lib.paged_args(*(size.get(f, 0) for f in _lib.PAGED_FIELDS))
                assert lib.cgpt_paged_attention_workspace(args, ctypes.byref(n)) == 0 and n.value > 0, size
                a = dict(prefix_len=0, bt_stride=64, kc_sp=1 << 40, kc_sh=1 << 30, kc_ss=hd, vc_sp=1 << 40, vc_sh=1 << 30, vc_ss=hd,
                         q_st=64 * hd, q_sh=hd, out_st=64 * hd, out_sh=hd, workspace=P + 8, workspace_bytes=n.value)
                assert call(FNS[1], **{**a, **size}) == EINVAL, size
                assert call(FNS[1], **{**a, **size, "workspace_bytes": n.value - 1}) == ESCRATCH, size


def test_launches_past_32_bits_are_refused():
    """A launch holds less than 2^32 threads: more is refused before the first one."""
    lib, n = _lib.load(), ctypes.c_int64(-1)
    for dtype in (_lib.CGPT_F32, _lib.CGPT_BF16):
        for size, hds in ((dict(B=1 << 22, n_tokens=1 << 22, Hq=32, Hkv=32, page_size=16, max_pages=4), (16, 64, 128)),
                          (dict(B=1 << 22, n_tokens=1 << 22, Hq=32, Hkv=32, page_size=16, max_pages=400), (16, 64, 128)),
                          (dict(B=1 << 17, n_tokens=1 << 26, Hq=31, Hkv=31, page_size=16, max_pages=400), (16, 64, 128)),
                          (dict(B=1 << 17, n_tokens=1 << 23, Hq=31, Hkv=31, page_size=16, max_pages=400, prefix_len=6400), (16, 64, 128))):
            for hd in hds:
                size.update(head_dim=hd, dtype=dtype)
                args = _lib.paged_args(*(size.get(f, 0) for f in _lib.PAGED_FIELDS))
                assert lib.cgpt_paged_attention_workspace(args, ctypes.byref(n)) == ESHAPE, size
                a = dict(prefix_len=0, bt_stride=400, kc_sp=1 << 40, kc_sh=1 << 30, kc_ss=hd, vc_sp=1 << 40, vc_sh=1 << 30, vc_ss=hd,
                         q_st=64 * hd, q_sh=hd, out_st=64 * hd, out_sh=hd, workspace=P + 8, workspace_bytes=1 << 60)
                assert call(FNS[1], **{**a, **size}) == ESHAPE, size
    # 16 tokens a block at most in fp32 of head_dim 128.
    a = dict(n_tokens=1 << 29, B=1 << 29, Hq=2, Hkv=2, head_dim=128, dtype=_lib.CGPT_F32, kc_sp=4096, kc_sh=2048, kc_ss=128, vc_sp=4096,
             vc_sh=2048, vc_ss=128, out_st=256, out_sh=128)
    assert call(FNS[0], **a) == ESHAPE
