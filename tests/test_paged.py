"""The paged cache without a GPU: the checks of the C entry points (nothing is launched),
of the wrappers, the rotation table and the tests' own oracle."""

import ctypes
import math

import pytest
import torch

import cutilegpt_amd as cg
from cutilegpt_amd import _lib
from paged_ref import Problem, append, attention

P = 1 << 20  # a pointer that is never followed


def call(fn, **change):
    """fn of libcgpt.so on well-formed sizes with no token (nothing to launch), changed."""
    a = dict(q=P, k=P, v=P, q_out=P, k_cache=P, v_cache=2 * P, o=P, table=P, lens=P, cu=P, rotary=P, prefix=P, prefix_len=16,
             n=0, B=2, Hq=4, Hkv=2, hd=64, page=16, n_pages=8, cols=4, stride=4, st=256, sh=64, sp=2048, ch=1024, ss=64,
             rot=64, n_pos=64, rs=64, scale=0.125, dtype=_lib.CGPT_BF16)
    a.update(change)
    g = lambda *names: [a[n] for n in names]
    sizes = g("n", "B", "Hq", "Hkv", "hd", "page", "n_pages", "cols", "stride")
    pools = g("sp", "ch", "ss", "sp", "ch", "ss")
    lib = _lib.load()
    if fn == "append":
        return lib.cgpt_paged_kv_append(*g("q", "k", "v", "q_out", "k_cache", "v_cache", "table", "lens", "cu", "rotary"), *sizes,
                                        *g("st", "sh") * 4, *pools, *g("rot", "n_pos", "rs"), 0, a["dtype"], None, None)
    tail = [*sizes, *g("st", "sh", "st", "sh"), *pools, a["scale"], None, 0, a["dtype"], None, None]
    if fn == "paged":
        return lib.cgpt_paged_attention(*g("q", "k_cache", "v_cache", "o", "table", "lens", "cu"), *tail)
    return lib.cgpt_shared_prefix_attention(*g("q", "k_cache", "v_cache", "o", "table", "lens", "cu", "prefix", "prefix_len"), *tail)


EINVAL, EDTYPE, ESHAPE = -1, -2, -3
SHARED = [(dict(n=-1), EINVAL), (dict(B=-1), EINVAL), (dict(Hq=3), EINVAL), (dict(Hkv=0), EINVAL), (dict(page=0), EINVAL),
          (dict(n_pages=0), EINVAL), (dict(cols=-1), EINVAL), (dict(k_cache=None), EINVAL), (dict(k_cache=P + 8), EINVAL),
          (dict(sp=2047), EINVAL), (dict(ss=32), EINVAL), (dict(ss=0), EINVAL), (dict(sp=0), EINVAL), (dict(ch=0), EINVAL),
          (dict(dtype=7), EDTYPE), (dict(hd=48), ESHAPE), (dict(hd=256), ESHAPE), (dict(page=1 << 20, cols=1 << 11), ESHAPE),
          (dict(n=1 << 30), ESHAPE), (dict(n_pages=1 << 31), ESHAPE)]


@pytest.mark.parametrize("fn", ["append", "paged", "shared"])
def test_c_entry_points_refuse(fn):
    assert call(fn) == 0
    for change, status in SHARED:
        assert call(fn, **change) == status, change
    # With a token the pointers and strides of the rows count too.
    for change in (dict(lens=None), dict(table=None), dict(st=255), dict(cu=None)):
        assert call(fn, n=3, **change) == EINVAL, change


def test_c_append_refuses():
    for change, status in ((dict(q=None), EINVAL), (dict(v_cache=P), EINVAL), (dict(rot=3), ESHAPE), (dict(rot=66), ESHAPE),
                           (dict(rot=-2), ESHAPE), (dict(n_pos=0), EINVAL), (dict(rs=62), EINVAL), (dict(rotary=None), EINVAL)):
        assert call("append", **change) == status, change
    for change in (dict(k=None), dict(v=P + 2)):
        assert call("append", n=3, **change) == EINVAL, change
    assert call("append", rot=0, rotary=None, q=None, q_out=None) == 0


def test_c_attention_refuses():
    for change in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan)):
        assert call("paged", **change) == EINVAL, change
    for change in (dict(prefix_len=-1), dict(prefix_len=65)):
        assert call("shared", **change) == EINVAL, change
    assert call("shared", n=3, prefix=None) == EINVAL
    assert call("paged", n=3, q=None) == EINVAL
    n = ctypes.c_int64(-1)
    lib = _lib.load()
    assert lib.cgpt_paged_attention_workspace(4, 4, 4, 2, 64, 16, 64, 0, _lib.CGPT_BF16, ctypes.byref(n)) == 0
    assert n.value >= 0
    assert lib.cgpt_paged_attention_workspace(4, 4, 4, 2, 64, 16, 64, 0, _lib.CGPT_BF16, None) == EINVAL


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
