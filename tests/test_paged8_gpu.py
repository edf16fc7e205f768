"""The 8-bit paged cache on the GPU: every operator against float64 at the sizes, lengths,
layouts and masks where it can go wrong."""

import pytest
import torch

import cutilegpt_amd as cg
from paged8_ref import F8, NAN, Problem8, append, attention, values
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
@pytest.mark.parametrize("dtype,hd,rot,interleaved", [(BF16, 64, 64, True), (F16, 64, 32, False), (F32, 128, 6, False),
                                                      (BF16, 16, 16, False), (F32, 32, 20, True), (F16, 128, 128, False)])
def test_append_step_turned(gpu, code, dtype, hd, rot, interleaved):
    """Single tokens with every way of turning, more heads than a block's threads have rows."""
    p = Problem8(dtype, code, hd, 12, 4, Hq=30, Hkv=15, ctx=[0, 3, 11, 12, 50], new=[1] * 5, seed=rot, spread=4)
    check_append(p, gpu, cg.rotary_table(64, rot, device="cpu"), interleaved)


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("new", [1, 5])
def test_append_turned_past_the_floats(gpu, code, new):
    """A key that the turning takes past float32 counts as infinite: the largest code, the flag, and
    an exponent that goes by the others."""
    p = Problem8(BF16, code, 64, 16, 1, 1, 1, ctx=[0, 0], new=[new, new], seed=3)
    rotary = torch.full((new, 64), 0.70710678)
    p.k[new - 1, 0, 5], p.k[new - 1, 0, 37] = 3e38, -3e38    # to 4.2e38 and 0
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    d, _ = run_append(p, gpu, rotary, err_flag=flag)
    assert int(flag) == 1
    want, _ = append(p, rotary)
    page, slot = int(p.table[0, 0]), new - 1
    got, top = d.k_cache[page, 0, slot].cpu().double(), 448.0 if code == F8 else 127.0
    assert float(got[5]) == top
    # The rest of the row is there on a scale of its own size.
    e = int(d.k_scale[page, 0, slot]) - 127
    clean = p.k[new - 1, 0].clone()
    clean[5], clean[37] = 0, 0
    assert top * 2.0 ** e >= float(clean.abs().max()) / 2 and top * 2.0 ** e < 1e6
    # Another sequence's rows are as they would be.
    other = int(p.table[1, 0])
    same_bytes(d.k_cache[other], want[0][other], "k")


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


# ------------------------------------------------------------------------- attention
# ``room``: columns of the table past what the lengths need.  A narrow table of short
# sequences runs in one launch, a wide one in shared-out parts and their join.

ROOM = [1, 400]


def run_attention(p, gpu, **kw):
    d = p.on(gpu)
    cu = None if p.n == p.B and p.new == [1] * p.B else d.cu
    return cg.paged_attention_8bit(d.q, *d.cache, cu_q=cu, **kw)


def check_attention(p, gpu, scale=None, **kw):
    want, bound = attention(p, scale)
    got = run_attention(p, gpu, scale=scale, **kw)
    assert got.shape == p.q.shape and got.dtype == p.dtype
    live = int(p.cu[-1])
    within(got[:live], want[:live], bound[:live], "attention")


def problem(dtype, code, hd, page, block, Hq, Hkv, ctx, new, **kw):
    """Keys that are all numbers."""
    return Problem8(dtype, code, hd, page, block, Hq, Hkv, ctx, new, size=40, **kw)


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,Hq,Hkv,page,block", [(16, 4, 2, 16, 16), (32, 3, 3, 8, 8), (64, 12, 12, 16, 16), (64, 8, 1, 24, 8),
                                                  (64, 20, 1, 64, 32), (128, 8, 2, 32, 32), (128, 3, 1, 10, 5), (64, 2, 2, 1, 1)])
def test_single_tokens(gpu, dtype, code, hd, Hq, Hkv, page, block, room):
    p = problem(dtype, code, hd, page, block, Hq, Hkv, ctx=[0, 1, 14, 15, 16, 31, 63, 64, 127, 200, 333], new=[1] * 11,
                seed=hd + page, spare_cols=room)
    check_attention(p, gpu)


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,Hq,Hkv,page,block,new", [
    (64, 4, 2, 16, 16, [3, 1, 0, 8, 2]), (64, 4, 4, 16, 8, [70, 1, 129, 0, 33]), (128, 4, 1, 64, 64, [5, 200, 0, 64, 17]),
    (32, 6, 3, 10, 5, [5, 40, 1, 16, 2]), (16, 2, 1, 16, 16, [90, 3, 65, 1, 0]), (128, 2, 2, 24, 24, [40, 8, 100, 1, 1]),
    (32, 2, 2, 128, 64, [300, 64, 65, 63, 1]), (64, 8, 1, 7, 7, [20, 9, 0, 3, 1])])
def test_ragged_tokens(gpu, dtype, code, hd, Hq, Hkv, page, block, new, room):
    p = problem(dtype, code, hd, page, block, Hq, Hkv, ctx=[0, 17, 40, 100, 250], new=new, seed=sum(new), spare_cols=room,
                pad_rows=3)
    check_attention(p, gpu)


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype,new,hd", [(BF16, 1, 64), (F16, 4, 128), (F32, 2, 64), (BF16, 80, 64), (F16, 40, 32)])
def test_one_long_sequence(gpu, dtype, code, new, hd):
    p = problem(dtype, code, hd, 64, 64, Hq=4, Hkv=2, ctx=[9000], new=[new], seed=new)
    check_attention(p, gpu)


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("new", [1, 5, 40])
def test_rows_without_a_key(gpu, new, room):
    """Sequences shorter than their step: the tokens in front of position 0 give zeros."""
    p = problem(BF16, F8, 64, 16, 16, 4, 2, ctx=[0, 30, 0, 5], new=[new] * 4, seed=new, spare_cols=room)
    for b, n in ((0, 0), (2, max(new - 2, 0))):
        p.lens[b] = n
        p.total[b] = n
    check_attention(p, gpu)


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("hd,new,Hkv", [(64, 1, 2), (64, 6, 2), (128, 3, 1), (64, 70, 2), (16, 30, 1), (32, 150, 2), (128, 90, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_nan_codes_do_not_leak(gpu, dtype, new, Hkv, hd, room):
    """Keys and values that are no numbers count for the rows that see them, and for no
    other."""
    p = problem(dtype, F8, hd, 16, 8, 2 * Hkv, Hkv, ctx=[20, 3, 150], new=[new] * 3, seed=new + hd, spare_cols=room)
    at = {}
    for b in range(3):
        # The last key, and one in the middle of the step, of the first head.
        for pos, which in ((p.total[b] - 1, "k"), (p.total[b] - 1 - new // 2, "v"), (p.total[b] - 1 - new // 3, "v")):
            page, slot = int(p.table[b, pos // 16]), pos % 16
            getattr(p, which + "_cache").view(torch.uint8)[page, 0, slot, 3] = 0x7f if which == "k" else 0xff
            at.setdefault(b, []).append((pos, which))
    G = 2
    clean = problem(dtype, F8, hd, 16, 8, 2 * Hkv, Hkv, ctx=[20, 3, 150], new=[new] * 3, seed=new + hd, spare_cols=room)
    want, bound = attention(clean)
    got = run_attention(p, gpu).cpu()
    for b in range(3):
        for i in range(new):
            t, pos = int(p.cu[b]) + i, p.total[b] - new + i
            rows_nan = any(w == "k" and pos >= a for a, w in at[b])
            d3_nan = rows_nan or any(pos >= a for a, w in at[b])
            first, others = got[t, :G], got[t, G:]
            assert bool(first[:, 3].isnan().all()) == d3_nan and bool(first[:, 3].isnan().any()) == d3_nan, (b, i)
            rest = torch.cat([first[:, :3], first[:, 4:]], 1)
            assert bool(rest.isnan().all()) == rows_nan and bool(rest.isnan().any()) == rows_nan, (b, i)
            if not rows_nan:
                w, e = want[t].clone(), bound[t]
                if d3_nan:
                    w[:G, 3] = NAN
                within(got[t], w, e, f"{b} {i}")
            within(others, want[t, G:], bound[t, G:])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new", [1, 30])
def test_a_query_that_is_not_a_number(gpu, dtype, new):
    """It spoils its own row only."""
    p = problem(dtype, F8, 64, 16, 16, 2, 1, ctx=[40, 10], new=[new, new], seed=3)
    want, bound = attention(p)
    p.q[new, 1, 5] = NAN
    got = run_attention(p, gpu)
    assert bool(got[new, 1].isnan().all())
    want[new, 1] = NAN
    within(got, want, bound)


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("B,new,room", [(130, 1, 1), (300, 1, 40), (70, 3, 1), (90, 20, 1)])
def test_many_sequences(gpu, code, B, new, room):
    g = torch.Generator().manual_seed(B)
    ctx = torch.randint(0, 150, (B,), generator=g).tolist()
    p = problem(BF16, code, 32, 16, 16, 2, 1, ctx=ctx, new=[new] * B, seed=B, spare_cols=room)
    check_attention(p, gpu)


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype,hd,page,block", [(BF16, 64, 16, 16), (F16, 128, 10, 5), (F32, 64, 24, 8), (F32, 128, 16, 16),
                                                 (BF16, 16, 8, 8), (F16, 32, 64, 64)])
def test_tiles_of_128_rows(gpu, code, dtype, hd, page, block):
    """Batches that fill the card with large tiles, most of them not full."""
    g = torch.Generator().manual_seed(hd)
    new = torch.randint(12, 30, (64,), generator=g).tolist()
    new[5], new[9] = 150, 0
    p = problem(dtype, code, hd, page, block, 16, 16, ctx=torch.randint(0, 70, (64,), generator=g).tolist(), new=new, seed=hd)
    check_attention(p, gpu)


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new,room", [(1, 1), (1, 400), (40, 1)])
def test_exponents_far_apart(gpu, code, dtype, new, room):
    """Blocks whose values differ by 2^40, and the ends of the exponents' range."""
    p = problem(dtype, code, 64, 16, 16, 2, 2, ctx=[100, 60], new=[new, new], seed=4, spare_cols=room)
    p.k_scale.fill_(118)
    g = torch.Generator().manual_seed(9)
    p.v_scale.copy_(torch.randint(60, 101, p.v_scale.shape, generator=g, dtype=torch.uint8))
    if dtype != F16:
        p.v_scale += 60
    check_attention(p, gpu)
    # All values of the smallest exponent there is: 2^-100, read from the bytes below too.
    p.v_scale.fill_(0)
    if dtype != F16:
        want, bound = attention(p)
        got = run_attention(p, gpu)
        # (The bound's own floor is of that size: take it without.)
        within(got, want, bound - 2.0 ** -100 + want.abs().amax() * 2.0 ** -20)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new,room", [(1, 1), (3, 400), (60, 1)])
def test_large_scores(gpu, dtype, new, room):
    p = problem(dtype, I8, 64, 16, 16, 4, 2, ctx=[150, 33], new=[new, new], seed=11, spare_cols=room, spread=4)
    check_attention(p, gpu, scale=2.0)


@pytest.mark.parametrize("new", [1, 40])
def test_out_may_be_q(gpu, new):
    p = problem(BF16, F8, 64, 16, 16, 4, 2, ctx=[30, 7], new=[new, new], seed=2)
    d = p.on(gpu)
    got = cg.paged_attention_8bit(d.q, *d.cache, cu_q=d.cu, out=d.q)
    assert got is d.q
    want, bound = attention(p)
    within(got, want, bound)


def test_attention_views(gpu):
    """q out of a fused projection, pools and exponents views of others, out with gaps."""
    p = problem(BF16, I8, 64, 16, 4, 4, 2, ctx=[30, 7, 100], new=[1, 9, 40], seed=2)
    d = p.on(gpu)
    fused = torch.zeros(p.n, 8, 64, dtype=BF16, device=gpu)
    fused[:, :4] = d.q
    pool = torch.stack([d.k_cache, d.v_cache], 2)          # (pages, heads, 2, slots, hd)
    scale = torch.stack([d.k_scale, d.v_scale], -1)        # (pages, heads, blocks, 2)
    out = torch.full((p.n, 6, 64), 7.0, dtype=BF16, device=gpu)
    cg.paged_attention_8bit(fused[:, :4], pool[:, :, 0], pool[:, :, 1], scale[..., 0], scale[..., 1], d.table, d.lens,
                            cu_q=d.cu, out=out[:, 1:5])
    want, bound = attention(p)
    within(out[:, 1:5], want, bound)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 5] == 7).all())


@pytest.mark.parametrize("new", [1, 30])
def test_pool_past_32_bits(gpu, new):
    """Pages and exponents further than 2^32 bytes from the pool's start."""
    p = problem(BF16, F8, 64, 16, 16, 2, 2, ctx=[100], new=[new], seed=1)
    d = p.on(gpu)
    apart = 1 << 30
    big = torch.empty(apart * p.n_pages, dtype=torch.uint8, device=gpu)
    kc = big.as_strided((p.n_pages, 2, 16, 64), (apart, 1024, 64, 1))
    ks = big[4096:].as_strided((p.n_pages, 2, 1), (apart, 1, 1))
    kc.copy_(d.k_cache.view(torch.uint8))
    ks.copy_(d.k_scale)
    got = cg.paged_attention_8bit(d.q, kc.view(F8), d.v_cache, ks, d.v_scale, d.table, d.lens, cu_q=d.cu)
    want, bound = attention(p)
    within(got, want, bound)
    cg.paged_kv_append_8bit(d.k, d.v, kc.view(F8), d.v_cache, ks, d.v_scale, d.table, d.lens, cu_q=d.cu)
    after, _ = append(p)
    same_bytes(kc, after[0], "k_cache")
    same_bytes(ks, after[2], "k_scale")


@pytest.mark.parametrize("new", [1, 40])
def test_attention_bad_device_values(gpu, new):
    """A page outside the pool is read as page 0, a length past the table is cut; each sets the
    flag, and other sequences' rows stay right."""
    p = problem(BF16, F8, 64, 16, 16, 2, 2, ctx=[40, 40, 40], new=[new] * 3, seed=6, spare_cols=0)
    want, bound = attention(p)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    d = p.on(gpu)
    within(cg.paged_attention_8bit(d.q, *d.cache, cu_q=d.cu, err_flag=flag), want, bound)
    assert int(flag) == 0
    d.table[1, 0] = p.n_pages
    got = cg.paged_attention_8bit(d.q, *d.cache, cu_q=d.cu, err_flag=flag)
    assert int(flag) == 1
    for b in (0, 2):
        rows = slice(int(p.cu[b]), int(p.cu[b + 1]))
        within(got[rows], want[rows], bound[rows])
    flag.zero_()
    d = p.on(gpu)
    d.lens[2] = d.table.shape[1] * 16 + 9
    got = cg.paged_attention_8bit(d.q, *d.cache, cu_q=d.cu, err_flag=flag)
    assert int(flag) == 1
    within(got[:2 * new], want[:2 * new], bound[:2 * new])


def test_rows_in_front_of_the_first_sequence(gpu):
    """Offsets that begin past 0: the rows in front are left as they were."""
    p = problem(BF16, F8, 64, 16, 16, 2, 2, ctx=[30, 20], new=[3, 2], seed=6)
    d = p.on(gpu)
    q = torch.cat([d.q[:2], d.q])
    out = torch.full_like(q, 5.0)
    cg.paged_attention_8bit(q, *d.cache, cu_q=d.cu + 2, out=out)
    want, bound = attention(p)
    within(out[2:], want, bound)
    assert bool((out[:2] == 5).all())


def test_empty_calls(gpu):
    p = problem(BF16, F8, 64, 16, 16, 2, 2, ctx=[30], new=[1], seed=6)
    d = p.on(gpu)
    none = d.q[:0]
    cu = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert cg.paged_attention_8bit(none, *d.cache[:4], d.table[:0], d.lens[:0]).shape == (0, 2, 64)
    assert cg.paged_attention_8bit(none, *d.cache[:4], d.table[:0], d.lens[:0], cu_q=cu).shape == (0, 2, 64)
    cg.paged_kv_append_8bit(none, none, *d.cache[:4], d.table[:0], d.lens[:0])
    k, v = cg.paged_kv_read_8bit(*d.cache[:4], d.table[:0], d.lens[:0], cu, 0)
    assert k.shape == v.shape == (0, 2, 64)
    # Tables without a page: nothing to see.
    o = cg.paged_attention_8bit(d.q, *d.cache[:4], d.table[:, :0], torch.zeros_like(d.lens))
    assert bool((o == 0).all())


def test_same_bits_twice_and_on_side_streams(gpu):
    """One answer, whatever the stream and what runs beside it."""
    p = problem(BF16, F8, 64, 16, 16, 4, 2, ctx=[3000, 10, 700], new=[1, 20, 3], seed=8)
    d = p.on(gpu)
    first = cg.paged_attention_8bit(d.q, *d.cache, cu_q=d.cu)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(cg.paged_attention_8bit(d.q, *d.cache, cu_q=d.cu))
    torch.cuda.synchronize()
    for x in got:
        assert torch.equal(x.view(torch.int16), first.view(torch.int16))


def test_captured_steps(gpu):
    """A captured step (append, attention) of single tokens replays with the lengths of the
    moment, as the eager one does bit for bit."""
    B, Hq, Hkv, hd, page = 3, 4, 2, 64, 16
    base = problem(BF16, F8, hd, page, 16, Hq, Hkv, ctx=[5, 14, 40], new=[20] * 3, seed=12)
    rotary = cg.rotary_table(100, hd)
    g = torch.Generator().manual_seed(3)
    steps = [torch.randn(B, Hq + 2 * Hkv, hd, generator=g).to(BF16).to(gpu) for _ in range(18)]

    def fresh():
        d = base.on(gpu)
        d.lens = torch.tensor(base.ctx, dtype=torch.int32, device=gpu)
        return d

    def step(d, x):
        q = cg.paged_kv_append_8bit(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], *d.cache, q=x[:, :Hq], rotary=rotary)
        return cg.paged_attention_8bit(q, *d.cache)

    e, want = fresh(), []
    for x in steps:
        e.lens += 1
        want.append(step(e, x))
    c = fresh()
    x = steps[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(problem(BF16, F8, hd, page, 16, Hq, Hkv, ctx=[5, 14, 40], new=[20] * 3, seed=12).on(gpu), x)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c, x)
    for i, y in enumerate(steps):
        c.lens += 1
        x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want[i].view(torch.int16)), i
    for a, b in zip(c.cache[:4], e.cache[:4]):
        same_bytes(a, b.cpu(), "pools")


def test_written_cache_against_16_bits(gpu):
    """Prompts, then tokens, through the 8-bit cache against the 16-bit one: the answers differ by
    what the codes round.  With one-hot scores (a huge scale) an answer is one cached value."""
    hd, page = 64, 16
    g = torch.Generator().manual_seed(21)
    n, H = 50, 2
    k, v, q = (torch.randn(n, H, hd, generator=g).to(BF16).to(gpu) for _ in range(3))
    table = torch.randperm(8, generator=g).to(torch.int32).view(1, 8).to(gpu)
    lens, cu = torch.tensor([n], dtype=torch.int32, device=gpu), torch.tensor([0, n], dtype=torch.int32, device=gpu)
    for code in (F8, I8):
        pools = [torch.zeros(8, H, page, hd, dtype=torch.uint8, device=gpu).view(code) for _ in range(2)]
        scales = [torch.zeros(8, H, page // 8, dtype=torch.uint8, device=gpu) for _ in range(2)]
        cg.paged_kv_append_8bit(k, v, *pools, *scales, table, lens, cu_q=cu)
        kr, vr = cg.paged_kv_read_8bit(*pools, *scales, table, lens, cu, n)
        # Values within half a step: of 2^-3 relative, or of the block's largest over 64 (a power of
        # two at or above largest / 127).
        for got, want in ((kr, k), (vr, v)):
            want = want.double()
            big = want.reshape(n, H, hd).abs().amax(-1)
            blocks = torch.stack([big[i // 8 * 8:i // 8 * 8 + 8].amax(0) for i in range(n)])[..., None]
            bound = want.abs() / 16 + blocks * 2.0 ** -18 if code == F8 else blocks / 127 + want * 0
            assert bool(((got.double() - want).abs() <= bound).all())
        o8 = cg.paged_attention_8bit(q, *pools, *scales, table, lens, cu_q=cu)
        kc, vc = torch.zeros(8, H, page, hd, dtype=BF16, device=gpu), torch.zeros(8, H, page, hd, dtype=BF16, device=gpu)
        cg.paged_kv_append(kr, vr, kc, vc, table, lens, cu_q=cu)
        o16 = cg.paged_attention(q, kc, vc, table, lens, cu_q=cu)
        # The same values in 16 bits: both round weights and results to bf16.
        assert float((o8.double() - o16.double()).abs().max()) <= 4 * 2.0 ** -8 * float(vr.double().abs().max())


def test_refusals(gpu):
    p = problem(BF16, F8, 64, 16, 8, 4, 2, ctx=[30, 7], new=[1, 1], seed=2)
    d = p.on(gpu)
    kc, vc, ks, vs, table, lens = d.cache

    def refused(match, q=d.q, kc=kc, vc=vc, ks=ks, vs=vs, table=table, lens=lens, **kw):
        with pytest.raises(ValueError, match=match):
            cg.paged_attention_8bit(q, kc, vc, ks, vs, table, lens, **kw)

    refused("float8_e4m3fn or int8", kc=kc.view(I8))
    refused("float8_e4m3fn or int8", kc=kc.to(BF16), vc=vc.to(BF16))
    refused("unsupported dtype", q=d.q.double())
    refused("uint8", ks=ks.to(torch.int32))
    refused("divide a page", ks=ks[..., :1].expand(-1, -1, 3), vs=vs[..., :1].expand(-1, -1, 3))
    refused("page_size / block", ks=ks[:-1], vs=vs[:-1])
    refused("page_size / block", vs=vs[..., :1])
    refused("share a shape", vc=vc[:-1])
    refused("cache rows", kc=kc.transpose(2, 3).contiguous().transpose(2, 3))
    refused("not a multiple", q=d.q[:, :3])
    refused("need cu_q", q=torch.cat([d.q, d.q]))
    refused("int32", table=table.long())
    refused("one GPU", lens=lens.cpu())
    refused("scale must", scale=0.0)
    refused("scale must", scale=float("nan"))
    refused("output", out=torch.empty(2, 4, 64, dtype=F16, device=gpu))
    refused("output's rows", out=torch.empty(2, 1, 64, dtype=BF16, device=gpu).expand(2, 4, 64))
    refused("err_flag", err_flag=torch.zeros(2, dtype=torch.int32, device=gpu))
    refused("offsets", cu_q=torch.zeros(2, dtype=torch.int32, device=gpu))
    with pytest.raises(ValueError, match="invalid argument"):
        off = torch.zeros(kc.numel() + 16, dtype=torch.uint8, device=gpu)[4:4 + kc.numel()].view(kc.shape)
        cg.paged_attention_8bit(d.q, off.view(F8), vc, ks, vs, table, lens)
    with pytest.raises(ValueError, match="same memory"):
        cg.paged_kv_append_8bit(d.k, d.v, kc, kc, ks, vs, table, lens)
    with pytest.raises(ValueError, match="same memory"):
        cg.paged_kv_append_8bit(d.k, d.v, kc, vc, ks, ks, table, lens)
    with pytest.raises(ValueError, match="k and v"):
        cg.paged_kv_append_8bit(d.k, d.v.to(F16), *d.cache)
    with pytest.raises(ValueError, match="invalid argument"):
        cg.paged_kv_append_8bit(d.k, d.v, kc, vc, ks[..., :1].expand(-1, -1, 2), vs, table, lens)
    with pytest.raises(ValueError, match="n_rows"):
        cg.paged_kv_read_8bit(*d.cache, d.cu, 2.0)
    with pytest.raises(ValueError, match="unsupported dtype"):
        cg.paged_kv_read_8bit(*d.cache, d.cu, 2, torch.float64)
    with pytest.raises(ValueError, match="k_out and v_out"):
        cg.paged_kv_read_8bit(*d.cache, d.cu, 2, BF16, k_out=torch.empty(3, 2, 64, dtype=BF16, device=gpu))


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("hd,block", [(64, 16), (64, 8), (128, 8), (16, 16)])
def test_append_sequences_without_tokens(gpu, code, hd, block):
    """A sequence that has no token in the step has nothing read: an unused table entry where its
    last keys would be sets no flag, and nothing is written."""
    p = Problem8(BF16, code, hd, 16, block, 4, 2, ctx=[5, 21, 30, 0, 16], new=[3, 0, 2, 0, 0], seed=hd + block)
    p.table[1], p.table[4] = -7, p.n_pages
    want, _ = append(p)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    d, _ = run_append(p, gpu, err_flag=flag)
    assert int(flag) == 0
    for x, w, what in zip(d.cache, want, ("k_cache", "v_cache", "k_scale", "v_scale")):
        same_bytes(x, w, what)


def test_append_refuses_missing_values(gpu):
    d = Problem8(BF16, F8, 64, 16, 8, 4, 2, ctx=[30], new=[1], seed=2).on(gpu)
    for v in (None, 3):
        with pytest.raises(ValueError, match="torch tensors"):
            cg.paged_kv_append_8bit(d.k, v, *d.cache)


def one_key(dtype, code, score, ctx, new, hd=64, page=16, block=16, B=1, spare_cols=1):
    """Scores 0 but for each sequence's key at ctx - 1, which every token sees: ``score`` in base 2
    with scale score ln 2.  Values 0 but for that key's block, whose exponents are the largest: the key
    itself has the largest code in every other place."""
    p = problem(dtype, code, hd, page, block, 4, 2, ctx=[ctx] * B, new=[new] * B, seed=1, spare_cols=spare_cols)
    p.q.zero_()
    p.q[..., 0] = 1.0
    owned = p.table[:, :-(-p.total[0] // page)].flatten().long()
    for cache in (p.k_cache, p.v_cache):
        cache.view(torch.uint8)[owned] = 0
    p.k_scale.fill_(127)
    p.v_scale.fill_(127)
    at, slot = p.table[:, (ctx - 1) // page].long(), (ctx - 1) % page
    p.k_cache.view(torch.uint8)[at, :, slot, 0] = 0x38 if code == F8 else 1          # 1.0
    p.v_cache.view(torch.uint8)[at, :, slot, ::2] = 0x7e if code == F8 else 127      # 448, 127
    p.v_scale[at, :, slot // block] = 255
    return p, score * 0.6931471805599453


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,new,room,block,hd", [(1, 1, 1, 16, 64), (1, 1, 1, 8, 64), (1, 1, 1, 16, 32), (300, 1, 400, 16, 64),
                                                 (300, 1, 400, 8, 64), (300, 3, 400, 16, 128), (1, 40, 1, 16, 64), (1, 40, 1, 8, 16)])
def test_values_next_to_the_end_of_the_floats(gpu, dtype, code, B, new, room, block, hd):
    """A key whose score comes up to 8 (in base 2) above those in front of it, and values of the
    largest exponent: results next to the largest number of float32, and 0 beside them."""
    for score in (7.9, 1.0, 30.0):
        p, scale = one_key(dtype, code, score, 1220, new, hd, block=block, B=B, spare_cols=room)
        want, bound = attention(p, scale)
        got = run_attention(p, gpu, scale=scale).cpu()
        assert bool((got[..., 1::2] == 0).all()), score
        if dtype == F16:
            assert bool((got[..., ::2] == torch.inf).all()) and float(want[..., ::2].min()) > 1e6, score
        else:
            within(got, want, bound, f"score {score}")


@pytest.mark.parametrize("code", [F8, I8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new,room", [(1, 1), (1, 400), (5, 400), (40, 1)])
def test_scales_far_from_1(gpu, dtype, code, new, room):
    """Scales at which a block's exponent and the scale together leave the floats: blocks of zero keys,
    of the smallest exponent under a tiny scale, of the largest under a large one."""
    p = problem(dtype, code, 64, 16, 16, 4, 2, ctx=[150, 33], new=[new, new], seed=11, spare_cols=room)
    p.k_scale.fill_(27)
    for scale in (1e-16, 1e-30, 1e-43):
        want, bound = attention(p, scale)
        within(run_attention(p, gpu, scale=scale), want, bound, str(scale))
    p.k_scale.fill_(100)
    for b, total in enumerate(p.total):
        for col in range(0, total // 16, 3):
            page = int(p.table[b, col])
            p.k_cache.view(torch.uint8)[page] = 0
            p.k_scale[page] = 255
    for scale in (100.0, 1e4):
        p.q.mul_(0.01)
        want, bound = attention(p, scale)
        within(run_attention(p, gpu, scale=scale), want, bound, str(scale))
