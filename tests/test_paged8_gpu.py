"""The 8-bit paged cache on the GPU: every operator against float64 at the sizes, lengths,
layouts and masks where it can go wrong."""

import pytest
import torch

import cutilegpt_amd as cg
from paged8_ref import F8, NAN, Problem8, append, values
from paged_ref import within

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8 = torch.float32, torch.bfloat16, torch.float16, torch.int8


def run_append(p, gpu, rotary=None, interleaved=False, **kw):
    d = p.on(gpu)
    cu = None if p.n == p.B and p.new == [1] * p.B else d.cu
    q = cg.paged_kv_append_8bit(d.k, d.v, *d.cache, cu_q=cu, q=d.q, rotary=None if rotary is None else rotary.to(gpu),
                                interleaved=interleaved, **kw)
    return d, q


def same_bytes(got, want, what):
    got, want = got.cpu().view(torch.uint8), want.view(torch.uint8)
    bad = got != want
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:5].tolist(), want[bad][:5].tolist())


def same_values(got, want):
    """Equal, a NaN for a NaN (codes of either kind are read)."""
    got = got.cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.to(got.dtype).nan_to_num(7.0))


def check_append(p, gpu, rotary=None, interleaved=False):
    want, q = append(p, rotary, interleaved)
    d, got = run_append(p, gpu, rotary, interleaved, q_out=torch.full(p.q.shape, NAN, dtype=p.dtype, device=gpu))
    # Bit by bit, slots of no token, the rest of the pools and untouched exponents too.  (-0 and 0
    # are two codes: both sides keep a value's sign.)
    for x, w, what in zip(d.cache, want, ("k_cache", "v_cache", "k_scale", "v_scale")):
        same_bytes(x, w, what)
    # Queries: rounded once (the 64-bit turn is off by far less).
    u = torch.finfo(p.dtype).eps / 2
    tiny = 2.0 ** -25 if p.dtype == F16 else 2.0 ** -140
    within(got, q, q.abs().nan_to_num() * u * (1 + 2.0 ** -20) + tiny, "q")
    assert torch.isnan(got[int(p.cu[-1]):]).all()
    return d


# --------------------------------------------------------------------------- append

@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,rot,page,block", [(16, 0, 16, 16), (64, 64, 16, 8), (128, 32, 24, 8), (32, 32, 1, 1),
                                               (64, 6, 14, 7), (64, 64, 64, 64), (16, 16, 128, 1)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(gpu, code, dtype, hd, rot, page, block, interleaved):
    p = Problem8(dtype, code, hd, page, block, Hq=6, Hkv=2, ctx=[0, 5, 16, 47, 100], new=[3, 1, 16, 0, 40],
                 seed=hd + rot, pad_rows=2)
    check_append(p, gpu, cg.rotary_table(200, rot, device="cpu") if rot else None, interleaved)


@pytest.mark.parametrize("code", [F8, I8])
def test_append_step(gpu, code):
    """One token a sequence without cu_q, at every place of a block."""
    p = Problem8(BF16, code, 64, 16, 16, Hq=3, Hkv=3, ctx=list(range(40)), new=[1] * 40, seed=3, spread=6)
    check_append(p, gpu)


@pytest.mark.parametrize("code", [F8, I8])
def test_append_long_blocks(gpu, code):
    """Blocks of more rows than a wave takes at once, prompts of many blocks."""
    p = Problem8(F16, code, 128, 256, 256, Hq=2, Hkv=2, ctx=[0, 300], new=[700, 213], seed=4)
    check_append(p, gpu, cg.rotary_table(800, 128, device="cpu"))


@pytest.mark.parametrize("code", [F8, I8])
def test_append_token_by_token(gpu, code):
    """A block filled by single tokens whose sizes grow: its codes are rounded again and
    again.  e4m3 loses nothing by it above its smallest numbers, int8 less than a step."""
    hd, block = 32, 16
    g = torch.Generator().manual_seed(8)
    x = torch.randn(block, 1, hd, generator=g) * torch.logspace(-2, 2, block)[:, None, None]
    p = Problem8(F32, code, hd, block, block, 1, 1, ctx=[0], new=[1], seed=1)
    d = p.on(gpu)
    for t in range(block):
        d.lens.fill_(t + 1)
        cg.paged_kv_append_8bit(x[t:t + 1].to(gpu), -x[t:t + 1].to(gpu), *d.cache)
    page = int(p.table[0, 0])
    got = values(d.k_cache[page].cpu(), d.k_scale[page].cpu(), block)[0]
    step = 2.0 ** (int(d.k_scale[page, 0, 0]) - 127)
    want = x[:, 0].double()
    if code == F8:
        # Half a step of 2^-3 relative, or of the smallest number, 2^-9 units; the second
        # rounding of a value that has become that small adds as much.
        bound = want.abs() * 2.0 ** -4 + 2 * step * 2.0 ** -10
    else:
        # Half a step at every shift: steps at least double, so 1/2 (1 + 1/2 + 1/4 ..) < 1.
        bound = torch.full_like(want, step)
    within(got, want, bound)
    back = values(d.v_cache[page].cpu(), d.v_scale[page].cpu(), block)[0]
    assert torch.equal(back, -got)


@pytest.mark.parametrize("code", [F8, I8])
def test_append_borders(gpu, code):
    """Values next to the largest code, halfway between codes, the smallest of the type,
    zeros of either sign and whole blocks of zeros."""
    hd, n = 128, 40
    p = Problem8(F32, code, hd, 8, 1, 1, 1, ctx=[0], new=[n], seed=2)
    g = torch.arange(127, dtype=torch.uint8).view(F8).float() if code == F8 else torch.arange(128).float()
    top = 448.0 if code == F8 else 127.0
    for i in range(n):
        row = torch.zeros(hd)
        row[:len(g)] = g
        row[1:len(g)] = (g[1:] + g[:-1]) / 2          # ties
        e = (i * 7) % 60 - 30
        row[-1] = top
        up, down = torch.nextafter(row, torch.tensor(torch.inf)), torch.nextafter(row, torch.tensor(-torch.inf))
        row = [row, up, down, -row, -up][i % 5]
        row[3] = -0.0
        p.k[i, 0] = row * 2.0 ** e
        p.v[i, 0] = [0.0, -0.0, 1e-38, 1e-45, 3.4e38, 2.0 ** 127, 1.9921875 * 2.0 ** 127, 2.0 ** -100][i % 8]
        p.v[i, 0, 5] *= 0.99
    check_append(p, gpu)


@pytest.mark.parametrize("code", [F8, I8])
def test_append_not_finite(gpu, code):
    """Infinities take the largest code, a NaN a NaN (int8: 0); the exponent goes by the rest,
    and the flag is set."""
    p = Problem8(BF16, code, 64, 16, 4, 2, 2, ctx=[2, 8], new=[7, 1], seed=5)
    p.k[1, 0, 3], p.k[4, 1, 60], p.k[5, 0, 0] = torch.inf, -torch.inf, NAN
    p.v[7, 1, 9] = NAN
    p.v[3, 0] = torch.inf
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    want, _ = append(p)
    d, _ = run_append(p, gpu, err_flag=flag)
    assert int(flag) == 1
    for x, w in zip(d.cache[:2], want[:2]):
        a, b = x.cpu().double(), w.double()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    for x, w in zip(d.cache[2:], want[2:]):
        same_bytes(x, w, "scale")
    ok = Problem8(BF16, code, 64, 16, 4, 2, 2, ctx=[2, 8], new=[7, 1], seed=5)
    flag.zero_()
    run_append(ok, gpu, err_flag=flag)
    assert int(flag) == 0


def test_append_strided_in_place(gpu):
    """q turned in place, rows out of a fused projection, pools and exponents views of others."""
    B, Hq, Hkv, hd, page, block = 5, 6, 3, 64, 16, 4
    p = Problem8(BF16, F8, hd, page, block, Hq, Hkv, ctx=[7, 15, 16, 31, 100], new=[1] * B, seed=5)
    rotary = cg.rotary_table(128, hd, device="cpu")
    want, q = append(p, rotary)
    fused = torch.cat([p.q, p.k, p.v], 1).reshape(B, -1).to(gpu).view(B, Hq + 2 * Hkv, hd)
    pool = torch.stack([p.k_cache.view(torch.uint8), p.v_cache.view(torch.uint8)], 1).to(gpu)[:, None]
    pool = pool.expand(-1, 3, -1, -1, -1, -1).contiguous()
    # Exponents with the blocks outermost and spare bytes between.
    wide = torch.zeros(page // block, p.n_pages, 2, Hkv, 3, dtype=torch.uint8, device=gpu)
    wide[..., 1] = torch.stack([p.k_scale, p.v_scale], 1).permute(3, 0, 1, 2).to(gpu)
    view = wide[..., 1].permute(1, 2, 3, 0)
    other, spare = pool[:, ::2].clone(), wide[..., ::2].clone()
    qv = fused[:, :Hq]
    out = cg.paged_kv_append_8bit(fused[:, Hq:Hq + Hkv], fused[:, Hq + Hkv:], pool[:, 1, 0].view(F8), pool[:, 1, 1].view(F8),
                                  view[:, 0], view[:, 1], p.table.to(gpu), p.lens.to(gpu), q=qv, rotary=rotary.to(gpu), q_out=qv)
    assert out is qv
    same_bytes(pool[:, 1, 0], want[0], "k")
    same_bytes(pool[:, 1, 1], want[1], "v")
    same_bytes(view[:, 0], want[2], "k_scale")
    same_bytes(view[:, 1], want[3], "v_scale")
    within(fused[:, :Hq], q, q.abs() * 2.0 ** -8 * 1.001, "q")
    assert torch.equal(fused[:, Hq:].cpu(), torch.cat([p.k, p.v], 1))
    assert torch.equal(pool[:, ::2], other) and torch.equal(wide[..., ::2], spare)


def test_append_bad_device_values(gpu):
    """A page outside the pool and a position past the table's pages store nothing and set
    the flag; padding rows of length 0 store nothing and set none."""
    p = Problem8(BF16, F8, 64, 16, 16, 2, 2, ctx=[20, 20, 20, 20, 3], new=[1] * 5, seed=7, spare_cols=0)
    d = p.on(gpu)
    d.table[0, 1], d.table[1, 1] = p.n_pages, -1
    d.lens[2], d.lens[4] = 33, 0
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    one = Problem8(BF16, F8, 64, 16, 16, 2, 2, ctx=[20, 20, 20, 20, 3], new=[1] * 5, seed=7, spare_cols=0)
    want, _ = append(one)
    page = int(p.table[3, 1])
    cg.paged_kv_append_8bit(d.k, d.v, *d.cache, err_flag=flag)
    assert int(flag) == 1
    for x, w, before in zip(d.cache, want, p.cache):
        expect = before.clone()
        expect.view(torch.uint8)[page] = w.view(torch.uint8)[page]
        same_bytes(x, expect, "pools")
    flag.zero_()
    d.lens.zero_()
    cg.paged_kv_append_8bit(d.k, d.v, *d.cache, err_flag=flag)
    assert int(flag) == 0
    # Lengths that no table holds.
    d.lens.fill_(2 ** 31 - 1)
    q = cg.paged_kv_append_8bit(d.k, d.v, *d.cache, q=d.q, rotary=cg.rotary_table(4, 64), err_flag=flag)
    assert int(flag) == 1 and bool(torch.isfinite(q).all())
    d.lens.fill_(-5)
    cg.paged_kv_append_8bit(d.k, d.v, *d.cache, err_flag=flag)
    same_bytes(d.k_scale[page], want[2][page], "k_scale")


# ------------------------------------------------------------------------------ read

@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,page,block", [(16, 16, 16), (64, 10, 5), (128, 24, 8), (32, 1, 1)])
def test_read(gpu, code, dtype, hd, page, block):
    p = Problem8(dtype, code, hd, page, block, 2, 2, ctx=[0, 5, 16, 47, 100], new=[3, 1, 0, 0, 40], seed=hd)
    d = p.on(gpu)
    n = sum(p.total)
    outs = [torch.full((n + 3, 2, hd), NAN, dtype=dtype, device=gpu) for _ in range(2)]
    k, v = cg.paged_kv_read_8bit(*d.cache, d.cu_rows, n + 3, dtype, *outs)
    assert k is outs[0] and v is outs[1]
    for i, x in enumerate((k, v)):
        want = torch.cat([p.keys(b)[i] for b in range(p.B)])
        same_values(x[:n], want)
        assert bool(x[n:].isnan().all())
    # The last rows of every sequence, one of them longer than what the cache holds.
    take = [4, 2, 16, 0, 41]
    cu = torch.tensor([sum(take[:b]) for b in range(6)], dtype=torch.int32, device=gpu)
    k, v = cg.paged_kv_read_8bit(*d.cache, cu, sum(take), dtype)
    for i, x in enumerate((k, v)):
        want = torch.cat([torch.cat([torch.zeros(max(0, m - p.total[b]), 2, hd, dtype=torch.float64),
                                     p.keys(b)[i][max(0, p.total[b] - m):]]) for b, m in enumerate(take)])
        same_values(x, want)


def test_read_every_code(gpu):
    """All 256 codes under exponents from end to end, bytes that no append writes among them."""
    for code in (F8, I8):
        pool = torch.arange(256, dtype=torch.uint8).repeat(32, 1).view(32, 1, 16, 16).contiguous().view(code)
        bytes_ = [0, 1, 26, 27, 28, 60, 100, 118, 119, 120, 127, 128, 150, 200, 245, 246, 247, 248, 249, 254, 255] + [127] * 11
        scale = torch.tensor(bytes_, dtype=torch.uint8).view(32, 1, 1)
        table = torch.arange(32, dtype=torch.int32).view(32, 1)
        lens = torch.full((32,), 16, dtype=torch.int32)
        cu = torch.arange(33, dtype=torch.int32) * 16
        want = values(pool, scale, 16).view(512, 1, 16)
        for dtype in (F32, BF16, F16):
            k, v = cg.paged_kv_read_8bit(*(t.to(gpu) for t in (pool, pool.clone(), scale, scale, table, lens, cu)), 512, dtype)
            same_values(k, want)
            assert torch.equal(k.view(torch.int32 if dtype == F32 else torch.int16), v.view(torch.int32 if dtype == F32 else torch.int16))


def test_read_bad_device_values(gpu):
    p = Problem8(BF16, F8, 64, 16, 16, 2, 2, ctx=[20, 20, 20], new=[0] * 3, seed=7, spare_cols=0)
    d = p.on(gpu)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    cg.paged_kv_read_8bit(*d.cache, d.cu_rows, 60, BF16, err_flag=flag)
    assert int(flag) == 0
    d.lens[1] = 40  # a table row names 32
    k, _ = cg.paged_kv_read_8bit(*d.cache, d.cu_rows, 60, BF16, err_flag=flag)
    assert int(flag) == 1 and bool((k[32:40] == 0).all()) and torch.equal(k[:20].cpu().double(), p.keys(0)[0])
    flag.zero_()
    d.lens[1] = 20
    d.table[2, 0] = p.n_pages + 5
    cg.paged_kv_read_8bit(*d.cache, d.cu_rows, 60, BF16, err_flag=flag)
    assert int(flag) == 1
