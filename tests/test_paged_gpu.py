"""The paged key-value cache on the GPU: every operator against float64 at the sizes,
lengths, layouts and masks where it can go wrong."""

import math
import random

import pytest
import torch

import cutilegpt_amd as cg
from paged_ref import NAN, Problem, append, attention, within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def run_append(p, gpu, rotary=None, interleaved=False, **kw):
    d = p.on(gpu)
    cu = None if p.n == p.B and p.new == [1] * p.B else d.cu
    q = cg.paged_kv_append(d.k, d.v, d.k_cache, d.v_cache, d.table, d.lens, cu_q=cu, q=d.q,
                           rotary=None if rotary is None else rotary.to(gpu), interleaved=interleaved, **kw)
    return d, q


def run_attention(p, gpu, **kw):
    d = p.on(gpu)
    cu = None if p.n == p.B and p.new == [1] * p.B else d.cu
    if p.prefix:
        return cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, p.prefix, cu_q=cu, **kw)
    return cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, cu_q=cu, **kw)


def check_attention(p, gpu, **kw):
    want, bound = attention(p)
    got = run_attention(p, gpu, **kw)
    assert got.shape == p.q.shape and got.dtype == p.dtype
    live = int(p.cu[-1])
    within(got[:live], want[:live], bound[:live], "attention")


# ------------------------------------------------------------------------------ append

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,rot,page", [(16, 0, 16), (64, 64, 16), (128, 32, 24), (32, 32, 1), (64, 6, 7)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(gpu, dtype, hd, rot, page, interleaved):
    p = Problem(dtype, hd, page, Hq=6, Hkv=2, ctx=[0, 5, 16, 47, 100], new=[3, 1, 16, 0, 40], seed=hd + rot, pad_rows=2)
    rotary = cg.rotary_table(200, rot, device="cpu") if rot else None
    kc, vc, q, kb, qb = append(p, rotary, interleaved)
    d, got = run_append(p, gpu, rotary, interleaved, q_out=torch.full(p.q.shape, NAN, dtype=dtype, device=gpu))
    within(d.k_cache, kc, kb, "k_cache")
    within(d.v_cache, vc, torch.zeros_like(vc), "v_cache")
    within(got, q, qb, "q")
    # Slots of no token keep their contents, rows behind the last sequence theirs.
    untouched = torch.isnan(kc)
    assert torch.isnan(d.k_cache.cpu()[untouched]).all() and torch.isnan(d.v_cache.cpu()[untouched]).all()
    assert torch.isnan(got[int(p.cu[-1]):]).all()


def test_append_step_with_padding_row(gpu):
    """One token a sequence without cu_q; a row of length 0 is stored nowhere."""
    p = Problem(BF16, 64, 16, Hq=4, Hkv=4, ctx=[0, 31, 32, 15], new=[1] * 4, seed=3)
    p.lens[1] = 0
    d = p.on(gpu)
    before = d.k_cache.clone()
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert cg.paged_kv_append(d.k, d.v, d.k_cache, d.v_cache, d.table, d.lens, err_flag=flag) is None
    for b in (0, 2, 3):
        pos = p.total[b] - 1
        page, slot = int(p.table[b, pos // 16]), pos % 16
        assert torch.equal(d.k_cache[page, :, slot].cpu(), p.k[b])
        assert torch.equal(d.v_cache[page, :, slot].cpu(), p.v[b])
        before[page, :, slot] = d.k_cache[page, :, slot]
    assert torch.equal(before.view(torch.int16), d.k_cache.view(torch.int16))
    assert int(flag) == 0


def test_append_in_place_and_strided(gpu):
    """q turned in place, rows out of a fused projection, both pools views of one."""
    B, Hq, Hkv, hd, page = 5, 6, 3, 64, 16
    p = Problem(BF16, hd, page, Hq, Hkv, ctx=[7, 15, 16, 31, 100], new=[1] * B, seed=5)
    rotary = cg.rotary_table(128, hd, device="cpu")
    kc, vc, q, kb, qb = append(p, rotary)
    fused = torch.cat([p.q, p.k, p.v], 1).reshape(B, -1).to(gpu).view(B, Hq + 2 * Hkv, hd)
    pool = torch.stack([p.k_cache, p.v_cache], 1).to(gpu)[:, None].expand(-1, 3, -1, -1, -1, -1).contiguous()
    other = pool[:, ::2].clone()
    qv = fused[:, :Hq]
    out = cg.paged_kv_append(fused[:, Hq:Hq + Hkv], fused[:, Hq + Hkv:], pool[:, 1, 0], pool[:, 1, 1],
                             p.table.to(gpu), p.lens.to(gpu), q=qv, rotary=rotary.to(gpu), q_out=qv)
    assert out is qv
    within(pool[:, 1, 0], kc, kb, "k")
    within(pool[:, 1, 1], vc, torch.zeros_like(vc), "v")
    within(fused[:, :Hq], q, qb, "q")
    assert torch.equal(fused[:, Hq:].cpu(), torch.cat([p.k, p.v], 1))
    assert torch.equal(pool[:, ::2].view(torch.int16), other.view(torch.int16))


def test_append_unaligned_rows(gpu):
    """Keys off the 16-byte rule are copied first."""
    p = Problem(F16, 32, 8, 2, 2, ctx=[3, 9], new=[2, 5], seed=6)
    kc, vc, q, kb, qb = append(p)
    d = p.on(gpu)
    wide = torch.zeros(p.n, 2, 33, dtype=F16, device=gpu)
    wide[:, :, 1:] = d.k
    v_last = d.v.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    cg.paged_kv_append(wide[:, :, 1:], v_last, d.k_cache, d.v_cache, d.table, d.lens, cu_q=d.cu)
    within(d.k_cache, kc, kb)
    within(d.v_cache, vc, torch.zeros_like(vc))


def test_append_bad_device_values(gpu):
    """A page outside the pool and a position past the table's pages store nothing and set
    the flag; a position past the rotation table takes its last row."""
    p = Problem(BF16, 64, 16, 2, 2, ctx=[20, 20, 20, 20], new=[1] * 4, seed=7, spare_cols=0)
    d = p.on(gpu)
    d.table[0, 1], d.table[1, 1] = p.n_pages, -1
    d.lens[2] = 33
    clean = d.k_cache.clone()
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    cg.paged_kv_append(d.k, d.v, d.k_cache, d.v_cache, d.table, d.lens, err_flag=flag)
    assert int(flag) == 1
    page = int(p.table[3, 1])
    assert torch.equal(d.k_cache[page, :, 4].cpu(), p.k[3])
    clean[page, :, 4] = d.k_cache[page, :, 4]
    assert torch.equal(clean.view(torch.int16), d.k_cache.view(torch.int16))
    flag.zero_()
    short = cg.rotary_table(10, 64, device="cpu")
    full = short[torch.arange(40).clamp(max=9)]
    kc, vc, q, kb, qb = append(p, full)
    d, got = run_append(p, gpu, short, err_flag=flag)
    assert int(flag) == 1
    within(d.k_cache, kc, kb)
    within(got, q, qb)


# --------------------------------------------------------------------------- attention

# Tables as short as the sequences, and tables for far longer ones: the kernels are
# chosen by what the lengths may be.
WIDE = pytest.mark.parametrize("room", [0, 5000])


def cols(room, page):
    return 1 + room // page


LENS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300]


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,page", [(3, 3, 16), (8, 2, 10), (16, 1, 64), (18, 1, 16)])
def test_single_tokens(gpu, dtype, hd, Hq, Hkv, page, room):
    """One token a sequence, every length around the tiles, an odd page and one as long as
    a tile, one key head to one, four, sixteen and eighteen query heads."""
    check_attention(Problem(dtype, hd, page, Hq, Hkv, [n - 1 for n in LENS], [1] * len(LENS), seed=hd + Hq,
                            spare_cols=cols(room, page)), gpu)


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,Hq,Hkv,page", [(16, 2, 2, 1), (32, 6, 2, 24), (64, 4, 4, 16), (128, 8, 1, 128), (64, 6, 2, 10)])
@pytest.mark.parametrize("new", [[1, 150, 5, 0, 1, 70], [3, 0, 5, 1, 1, 8], [0, 0, 0, 0, 0, 200]])
def test_ragged_tokens(gpu, dtype, hd, Hq, Hkv, page, new, room):
    """Sequences with no token, one, a few and a long prompt; rows behind the last one are
    left as they were."""
    p = Problem(dtype, hd, page, Hq, Hkv, ctx=[10, 0, 130, 7, 0, 64], new=new, seed=hd, pad_rows=3,
                spare_cols=cols(room, page))
    out = torch.full(p.q.shape, 7.0, dtype=dtype, device=gpu)
    check_attention(p, gpu, out=out)
    assert (out[int(p.cu[-1]):] == 7.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 3])
def test_one_long_sequence(gpu, dtype, new):
    """Few rows against many keys: the work is split along the keys and joined."""
    check_attention(Problem(dtype, 64, 32, 4, 2, ctx=[9001, 40], new=[new, 1], seed=new), gpu)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,Hq,Hkv,page", [(16, 4, 2, 8), (32, 3, 3, 16), (64, 5, 5, 16), (128, 8, 2, 64)])
@pytest.mark.parametrize("prefix", [16, 129, 700])
@WIDE
def test_shared_prefix(gpu, dtype, hd, Hq, Hkv, page, prefix, room):
    prefix = -(-prefix // page) * page
    ctx = [prefix + c for c in (0, 1, 30, 64, 200)]
    check_attention(Problem(dtype, hd, page, Hq, Hkv, ctx, [1] * 5, prefix=prefix, seed=prefix,
                            spare_cols=cols(room, page)), gpu)


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B", [1, 9, 33, 70])
@pytest.mark.parametrize("hd,Hkv", [(64, 2), (128, 1), (32, 4)])
def test_shared_prefix_batches(gpu, dtype, B, hd, Hkv, room):
    """More rows than a tile of the prefix holds; one sequence alone."""
    ctx = [640 + (37 * b) % 50 for b in range(B)]
    check_attention(Problem(dtype, hd, 32, 4, Hkv, ctx, [1] * B, prefix=640, seed=B, spare_cols=cols(room, 32)), gpu)


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("new", [[20, 1, 0, 64], [5, 1, 0, 2], [3, 3, 3, 3]])
def test_shared_prefix_ragged_tokens(gpu, dtype, hd, new, room):
    p = Problem(dtype, hd, 16, 8, 4, ctx=[160, 165, 160, 200], new=new, prefix=160, seed=9, pad_rows=1,
                spare_cols=cols(room, 16))
    check_attention(p, gpu)


@pytest.mark.parametrize("room,copies", [(0, 1), (5000, 1), (5000, 40)])
def test_shared_prefix_inside_a_page_and_short_sequences(gpu, room, copies):
    """The prefix may end inside a page, its pages come as a list of their own; a padding
    row and sequences shorter than the prefix see what they hold."""
    p = Problem(BF16, 64, 16, 4, 4, ctx=[160, 70, 170] * copies, new=[1, 1, 1] * copies, prefix=160, seed=10,
                spare_cols=cols(room, 16))
    assert p.total[1] == 71
    want, bound = attention(p)
    d = p.on(gpu)
    got = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, 153, prefix_pages=d.table[2, :10].clone())
    within(got, want, bound)
    d.lens[0] = 0
    got = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, 160, prefix_pages=d.table[2, :10].clone())
    assert (got[0] == 0).all()
    within(got[1:], want[1:], bound[1:])
    # The rows' own entries for the prefix are not read.
    d.table[:, :10] = -1
    pages = p.table[2, :10].to(gpu)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    again = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, 160, prefix_pages=pages, err_flag=flag)
    assert torch.equal(again, got) and int(flag) == 0


@pytest.mark.parametrize("seed", range(60))
def test_mixed_batches(gpu, seed):
    """Types, heads, pages, lengths (none among them) and prefix ends drawn together, so that
    the kernels meet in combinations that the tests above take one at a time."""
    rng = random.Random(seed)
    B = rng.choice([1, 2, 7, 65, 130])
    Hkv, G = (rng.choice([1, 2, 3, 5, 9]), rng.choice([1, 2, 3, 8, 17])) if B <= 7 else (rng.choice([1, 2]), rng.choice([1, 2]))
    page = rng.choice([1, 8, 10, 16, 24, 32, 64, 100, 128])
    prefix = page * rng.randint(1, max(1, 300 // page)) if rng.random() < 0.6 else 0
    top = rng.choice([1, 1, 5, 40, 130 if B <= 7 else 9])
    new = [rng.randint(0 if rng.random() < 0.2 else 1, top) for _ in range(B)]
    new[0] = max(new[0], 1)
    ctx = [prefix + rng.randint(0, 200) if b == 0 or rng.random() < 0.8 else rng.randint(0, prefix + 20) for b in range(B)]
    p = Problem(rng.choice([F32, BF16, F16]), rng.choice([16, 32, 64, 128]), page, Hkv * G, Hkv, ctx=ctx, new=new,
                prefix=prefix, seed=seed, spare_cols=rng.choice([0, 1, 1 + 300 // page, 1 + 5000 // page]),
                pad_rows=rng.choice([0, 3]))
    want, bound = attention(p)
    d = p.on(gpu)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    end = max(1, prefix - rng.choice([0, 0, rng.randint(0, page)]))
    if prefix:
        got = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, end, cu_q=d.cu, err_flag=flag)
    else:
        got = cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, cu_q=d.cu, err_flag=flag)
    within(got, want, bound)
    assert int(flag) == 0


@pytest.mark.parametrize("most", [80, 100])
def test_tables_that_end_with_the_prefix(gpu, most):
    """Sequences that hold no key past the prefix: nothing is read behind their last page,
    where the row may end or name no page."""
    ctx = [65, 69, 78, 79, most - 1] * 24
    p = Problem(BF16, 64, 16, 4, 4, ctx=ctx, new=[1] * len(ctx), prefix=80, seed=15, spare_cols=0)
    assert p.table.shape[1] == -(-most // 16)
    want, bound = attention(p)
    d = p.on(gpu)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, 80, err_flag=flag)
    within(got, want, bound)
    assert int(flag) == 0


@WIDE
@pytest.mark.parametrize("new", [1, 2, 40])
def test_rows_without_a_key(gpu, new, room):
    """Padding rows (length 0) and tokens in front of position 0 give zeros."""
    p = Problem(BF16, 64, 16, 2, 2, ctx=[5, 5, 5], new=[new] * 3, seed=11, spare_cols=cols(room, 16))
    p.lens[1] = 0
    p.lens[2] = p.total[2] = new // 2
    p.ctx[2] = new // 2 - new
    p.total[1], p.ctx[1] = 0, -new
    check_attention(p, gpu)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new", [1, 12, 90])
@pytest.mark.parametrize("Hkv", [1, 4])
@pytest.mark.parametrize("what", [NAN, float("inf"), -float("inf")])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@WIDE
def test_masked_values_do_not_leak(gpu, dtype, new, Hkv, what, hd, room):
    """What a row may not see has no part in it: keys and values that later tokens of the same
    step brought, whatever they hold."""
    p = Problem(dtype, hd, 16, 4, Hkv, ctx=[0, 21], new=[new, new], seed=12, spare_cols=cols(room, 16))
    poison = max(0, new - 3)
    for b in range(2):
        for pos in range(p.ctx[b] + poison + 1, p.total[b]):
            p.k_cache[int(p.table[b, pos // 16]), :, pos % 16, 5] = what
            p.v_cache[int(p.table[b, pos // 16]), :, pos % 16, 7] = what
    want, bound = attention(p)
    got = run_attention(p, gpu)
    for b in range(2):
        first = int(p.cu[b])
        rows = slice(first, first + poison + 1)
        within(got[rows], want[rows], bound[rows], "rows in front of the poison")


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
def test_value_of_a_seen_key_counts_whatever_it_is(gpu, dtype, new, hd, room):
    p = Problem(dtype, hd, 16, 2, 2, ctx=[40], new=[new], seed=13, spare_cols=cols(room, 16))
    p.v_cache[int(p.table[0, 0]), :, 3, 9] = float("inf")
    p.v_cache[int(p.table[0, 1]), :, 3, 11] = NAN
    got = run_attention(p, gpu).float().cpu()
    assert (got[:, :, 9] == float("inf")).all() and torch.isnan(got[:, :, 11]).all()
    rest = [d for d in range(hd) if d not in (9, 11)]
    want, bound = attention(p)
    within(got[:, :, rest], want[:, :, rest], bound[:, :, rest])


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new,prefix", [([1, 1, 1], 0), ([1, 3, 1], 0), ([20, 40, 30], 0), ([1] * 30, 64), ([8] * 4, 64)])
def test_a_query_that_is_not_a_number(gpu, dtype, new, prefix, room):
    """Its row is NaN, its neighbours' are not."""
    p = Problem(dtype, 64, 16, 4, 2, ctx=[100 + b for b in range(len(new))], new=new, prefix=prefix, seed=31,
                spare_cols=cols(room, 16))
    bad = int(p.cu[1])
    p.q[bad, 2, 5] = NAN
    want, bound = attention(p)
    got = run_attention(p, gpu)
    assert torch.isnan(got[bad, 2]).all()
    got = got.clone()
    got[bad, 2], want[bad, 2], bound[bad, 2] = 0, 0, 0
    within(got, want, bound)


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B", [65, 200, 300])
@pytest.mark.parametrize("new,prefix", [(1, 0), (2, 0), (1, 32), (24, 0)])
def test_many_sequences(gpu, dtype, B, new, prefix, room):
    """More sequences than a wave looks at at once, lengths of zero among them."""
    ctx = [prefix + (b * 37) % 90 for b in range(B)]
    p = Problem(dtype, 64, 16, 2, 1, ctx, [new if b % 5 else 0 for b in range(B)] if new > 1 else [1] * B,
                prefix=prefix, seed=B, spare_cols=cols(room, 16))
    check_attention(p, gpu)


def test_rows_in_front_of_the_first_sequence(gpu):
    """Offsets that do not begin at 0: the rows before the first are padding too."""
    for new, room in (([3, 2], 0), ([3, 2], 5000), ([40, 30], 0)):
        p = Problem(BF16, 64, 16, 4, 2, ctx=[33, 60], new=new, seed=33, spare_cols=cols(room, 16))
        want, bound = attention(p)
        kc, vc, q, kb, qb = append(p)
        d = p.on(gpu)
        shift = 2
        d.cu = d.cu + shift
        rows = lambda t: torch.cat([torch.full_like(t[:shift], 3.0), t])
        out = torch.full_like(rows(d.q), 7.0)
        cg.paged_attention(rows(d.q), d.k_cache, d.v_cache, d.table, d.lens, cu_q=d.cu, out=out)
        assert (out[:shift] == 7.0).all()
        within(out[shift:], want, bound)
        got = cg.paged_kv_append(rows(d.k), rows(d.v), d.k_cache, d.v_cache, d.table, d.lens, cu_q=d.cu, q=rows(d.q),
                                 q_out=torch.full_like(out, 7.0))
        assert (got[:shift] == 7.0).all()
        within(got[shift:], q, qb)
        within(d.k_cache, kc, kb)
        within(d.v_cache, vc, torch.zeros_like(vc))


@WIDE
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new", [[1, 60, 2], [1, 2, 1]])
def test_large_scores(gpu, dtype, new, room):
    """Scores in the hundreds: the running maximum jumps from tile to tile."""
    check_attention(Problem(dtype, 64, 16, 4, 2, ctx=[500, 3, 299], new=new, seed=14, scale=5.0,
                            spare_cols=cols(room, 16)), gpu)


@pytest.mark.parametrize("new,prefix", [(1, 0), (1, 512), (50, 0), (8, 64)])
def test_out_may_be_q(gpu, new, prefix):
    for room in (0, 5000):
        p = Problem(BF16, 64, 16, 4, 2, ctx=[600, 530, 900] * 8, new=[new] * 24, prefix=prefix, seed=34, spare_cols=cols(room, 16))
        d = p.on(gpu)
        want = run_attention(p, gpu)
        call = cg.shared_prefix_attention if prefix else cg.paged_attention
        got = call(d.q, d.k_cache, d.v_cache, d.table, d.lens, *([prefix] if prefix else []),
                   cu_q=None if new == 1 else d.cu, out=d.q)
        assert got is d.q and torch.equal(got, want)


def test_scale_and_out(gpu):
    p = Problem(F32, 32, 16, 4, 2, ctx=[50, 3], new=[1, 1], seed=15)
    want, bound = attention(p, scale=0.7)
    out = torch.empty(2, 9, 4, 32, device=gpu)[:, 5]
    got = run_attention(p, gpu, scale=0.7, out=out)
    assert got is out
    within(out, want, bound)


@pytest.mark.parametrize("new", [1, 40])
def test_pool_past_32_bits(gpu, new):
    """Pages whose offsets pass 2^32 bytes (and 2^31 elements)."""
    p = Problem(BF16, 64, 16, 2, 2, ctx=[100, 37], new=[new, new], seed=16)
    d = p.on(gpu)
    per = 2 * 16 * 64
    far = 2 ** 31 // per + 5
    pool = torch.empty((far + p.n_pages) * 2 * per, dtype=BF16, device=gpu).view(-1, 2, 2, 16, 64)
    pool[far:, 0], pool[far:, 1] = d.k_cache, d.v_cache
    table = torch.where(d.table >= 0, d.table + far, d.table)
    want, bound = attention(p)
    kw = dict(cu_q=d.cu)
    within(cg.paged_attention(d.q, pool[:, 0], pool[:, 1], table, d.lens, **kw), want, bound)
    kc, vc, q, kb, qb = append(p)
    cg.paged_kv_append(d.k, d.v, pool[:, 0], pool[:, 1], table, d.lens, **kw)
    within(pool[far:, 0], kc, kb)
    within(pool[far:, 1], vc, torch.zeros_like(vc))


def test_attention_bad_device_values(gpu):
    """A page outside the pool is read as page 0, a length past the table is cut there; both
    set the flag, and the other sequences do not notice."""
    p = Problem(BF16, 64, 16, 2, 2, ctx=[40, 40, 40], new=[1] * 3, seed=17, spare_cols=0)
    p.k_cache.nan_to_num_(0.0)
    p.v_cache.nan_to_num_(0.0)
    want, bound = attention(p)
    for spoil in ("page", "length", "offsets"):
        d = p.on(gpu)
        d.table, d.lens, d.cu = d.table.clone(), d.lens.clone(), d.cu.clone()
        flag = torch.zeros(1, dtype=torch.int32, device=gpu)
        if spoil == "page":
            d.table[1, 1] = p.n_pages + 3
        elif spoil == "length":
            d.lens[1] = 2 ** 30
        else:
            d.cu[3] = 2 ** 30  # tokens that the rows do not hold
        got = cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, cu_q=d.cu, err_flag=flag)
        if spoil != "offsets":
            assert int(flag) == 1, spoil
            assert torch.isfinite(got).all()
            within(got[::2], want[::2], bound[::2], spoil)
        else:
            within(got[:2], want[:2], bound[:2], spoil)
    zero = p.on(gpu)
    zero.table = zero.table.clone()
    zero.table[1, 1] = 0
    q = Problem.__new__(Problem)
    q.__dict__.update(p.__dict__)
    q.table = zero.table.cpu()
    want, bound = attention(q)
    d = p.on(gpu)
    d.table = d.table.clone()
    d.table[1, 1] = -3
    within(cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens), want, bound)


# -------------------------------------------------------------- streams, graphs, a run

def test_side_stream_and_two_at_once(gpu):
    ps = [Problem(BF16, 64, 16, 4, 4, ctx=[900, 33 + i], new=[1, 1], seed=20 + i) for i in range(2)]
    ds = [p.on(gpu) for p in ps]
    call = lambda d: cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens)
    eager = [call(d) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in ds]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(call(ds[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, eager[i]) for o in outs[i])


def test_same_bits_twice(gpu):
    for p in (Problem(BF16, 64, 16, 4, 4, ctx=[5000, 33], new=[1, 1], seed=22),
              Problem(BF16, 64, 16, 4, 4, ctx=[500, 333], new=[90, 100], seed=23),
              Problem(F32, 64, 16, 4, 4, ctx=[500, 333], new=[1, 1], prefix=320, seed=24)):
        first = run_attention(p, gpu)
        for _ in range(3):
            assert torch.equal(run_attention(p, gpu), first)


def test_captured_steps_replay_with_the_lengths_of_the_moment(gpu):
    """A decode step (append with rotation, attention, the same with a shared prefix) captured
    once and replayed while the lengths grow, two graphs of the same step in turn, against
    eager calls."""
    p = Problem(BF16, 64, 16, 4, 2, ctx=[160, 170, 190], new=[1, 1, 1], prefix=160, seed=25, spare_cols=0)
    # Pages for the tokens to come.
    table = torch.full((3, 16), 0, dtype=torch.int32)
    table[:, :p.table.shape[1]] = p.table
    extra = torch.arange(p.n_pages, p.n_pages + 3 * 16, dtype=torch.int32).view(3, 16)
    for b in range(3):
        n = -(-p.total[b] // 16)
        table[b, n:] = extra[b, n:]
    pad = torch.zeros(3 * 16, *p.k_cache.shape[1:], dtype=BF16)
    pools = [torch.cat([c, pad]).to(gpu) for c in (p.k_cache, p.v_cache)]
    mirror = [c.clone() for c in pools]
    d = p.on(gpu)
    table = table.to(gpu)
    rotary = cg.rotary_table(256, 64, device=gpu)
    lens = d.lens.clone()

    def step(kc, vc, lens):
        q = cg.paged_kv_append(d.k, d.v, kc, vc, table, lens, q=d.q, rotary=rotary)
        return (cg.paged_attention(q, kc, vc, table, lens),
                cg.shared_prefix_attention(q, kc, vc, table, lens, 160))

    step(*mirror, lens)  # loads the kernels
    for m, c in zip(mirror, pools):
        m.copy_(c)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream(gpu)
        side.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                outs.append(step(*pools, lens))
        torch.cuda.current_stream(gpu).wait_stream(side)
        graphs.append(g)
    busy = torch.randn(512, 512, device=gpu)
    for t in range(40):
        d.q.copy_(torch.randn(p.q.shape, generator=p.g).to(BF16))
        d.k.copy_(torch.randn(p.k.shape, generator=p.g).to(BF16))
        graphs[t % 2].replay()
        _ = busy @ busy
        want = step(*mirror, lens)
        torch.cuda.synchronize()
        for a, b in zip(outs[t % 2], want):
            assert torch.equal(a, b), t
        for a, b in zip(pools, mirror):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), t
        lens.add_(1)


def test_decoding_with_pages_is_the_models_forward(gpu):
    """GPT-2 blocks over a paged cache: ragged prompts taken in whole, then token by token,
    give the logits of the model's own forward on each sequence; samples of one prompt read
    it once."""
    cfg = cg.GPTConfig.gpt_nano()
    model = cg.CutileGPT(cfg, dtype=F32, seed=3)
    W, D, H, hd, page = model.weights, cfg.n_embd, cfg.n_head, cfg.head_dim, 16
    g = torch.Generator().manual_seed(4)
    ids = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (37, 5, 60)]
    n_pages, B = 40, len(ids)
    pools = torch.zeros(cfg.n_layer, 2, n_pages, H, page, hd, device=gpu)
    table = torch.randperm(n_pages, generator=g)[:B * 8].view(B, 8).to(gpu, torch.int32)

    def forward(tokens, pos, table, lens, cu, prefix):
        x = cg.cutile_embedding(tokens, W["wte"]) + cg.cutile_embedding(pos, W["wpe"])
        for i in range(cfg.n_layer):
            w = lambda n: W[f"h.{i}.{n}"]
            h = cg.cutile_layer_norm(x, w("ln_1.weight"), w("ln_1.bias"))
            qkv = cg.cutile_linear_bias(h, w("attn.c_attn.weight"), w("attn.c_attn.bias")).view(-1, 3 * H, hd)
            q, k, v = qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:]
            kc, vc = pools[i, 0], pools[i, 1]
            cg.paged_kv_append(k, v, kc, vc, table, lens, cu_q=cu)
            if prefix:
                a = cg.shared_prefix_attention(q, kc, vc, table, lens, prefix, cu_q=cu)
            else:
                a = cg.paged_attention(q, kc, vc, table, lens, cu_q=cu)
            x = x + cg.cutile_linear_bias(a.view(-1, D), w("attn.c_proj.weight"), w("attn.c_proj.bias"))
            h = cg.cutile_layer_norm(x, w("ln_2.weight"), w("ln_2.bias"))
            x = x + cg.cutile_fused_mlp(h, w("mlp.c_fc.weight"), w("mlp.c_fc.bias"), w("mlp.c_proj.weight"),
                                        w("mlp.c_proj.bias"))
        x = cg.cutile_layer_norm(x, W["ln_f.weight"], W["ln_f.bias"])
        return cg.cutile_linear(x, W["lm_head.weight"])

    def same(logits, seqs, last):
        for b, s in enumerate(seqs):
            want = model(s[None].to(gpu))[0][0]
            # Two float32 flows of the same sums: 3 layers, logits of order 1.
            assert (logits[b] - want[-last[b]:]).abs().max() < 1e-4

    lens = torch.tensor([len(s) for s in ids], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 37, 42, 102], dtype=torch.int32, device=gpu)
    pos = torch.cat([torch.arange(len(s)) for s in ids]).to(gpu)
    logits = forward(torch.cat(ids).to(gpu), pos, table, lens, cu, 0)
    same([logits[int(a):int(b)] for a, b in zip(cu, cu[1:])], ids, [len(s) for s in ids])
    for _ in range(3):
        new = torch.randint(0, cfg.vocab_size, (B,), generator=g)
        ids = [torch.cat([s, t[None]]) for s, t in zip(ids, new)]
        lens += 1
        logits = forward(new.to(gpu), lens.long() - 1, table, lens, None, 0)
        same(logits[:, None], ids, [1] * B)
    # Five samples of the third sequence's first 48 tokens: its pages, and pages of their own.
    shared, rows = ids[2][:48], 5
    free = torch.tensor([p for p in range(n_pages) if p not in set(table.flatten().tolist())], dtype=torch.int32)
    table = torch.cat([table[2:, :3].expand(rows, 3), free[:rows].view(rows, 1).to(gpu)], 1)
    seqs, lens = [shared] * rows, torch.full((rows,), 48, dtype=torch.int32, device=gpu)
    for _ in range(2):
        new = torch.randint(0, cfg.vocab_size, (rows,), generator=g)
        seqs = [torch.cat([s, t[None]]) for s, t in zip(seqs, new)]
        lens += 1
        logits = forward(new.to(gpu), lens.long() - 1, table, lens, None, 48)
        same(logits[:, None], seqs, [1] * rows)


def test_matches_the_dense_attention(gpu):
    """One prompt from position 0 is causal attention of the dense tensors."""
    p = Problem(BF16, 64, 16, 4, 4, ctx=[0], new=[200], seed=30)
    d, _ = run_append(p, gpu)
    got = cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, cu_q=d.cu)
    dense = cg.cutile_causal_attention(*(t.transpose(0, 1)[None] for t in (d.q, d.k, d.v)), 4)
    p.k_cache, p.v_cache = d.k_cache.cpu(), d.v_cache.cpu()
    want, bound = attention(p)
    within(got, want, bound)
    within(dense[0].transpose(0, 1), want, bound)


# --------------------------------------------------------------------------- refusals

def test_empty_calls(gpu):
    p = Problem(BF16, 64, 16, 2, 2, ctx=[3], new=[1]).on(gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    q = p.q[:0]
    assert cg.paged_attention(q, p.k_cache, p.v_cache, p.table[:0], none).shape == (0, 2, 64)
    assert cg.shared_prefix_attention(q, p.k_cache, p.v_cache, p.table[:0], none, 16).shape == (0, 2, 64)
    assert cg.paged_kv_append(p.k[:0], p.v[:0], p.k_cache, p.v_cache, p.table[:0], none) is None
    # Sequences without a token, and a table without a page.
    cu = torch.zeros(2, dtype=torch.int32, device=gpu)
    assert cg.paged_attention(q, p.k_cache, p.v_cache, p.table, p.lens, cu_q=cu).shape == (0, 2, 64)
    out = cg.paged_attention(p.q, p.k_cache, p.v_cache, p.table[:, :0], torch.zeros_like(p.lens))
    assert (out == 0).all()


def test_refusals(gpu):
    p = Problem(BF16, 64, 16, 4, 2, ctx=[30, 3], new=[1, 1]).on(gpu)
    args = dict(q=p.q, k_cache=p.k_cache, v_cache=p.v_cache, block_table=p.table, seq_lens=p.lens)

    def refused(fn, base, **change):
        with pytest.raises(ValueError):
            fn(**{**base, **change})

    for change in (dict(q=p.q.cpu()), dict(q=p.q.float()), dict(q=p.q[:, :3]), dict(q=p.q[0]), dict(q=p.q[:1]),
                   dict(q=p.q[..., :32]), dict(k_cache=p.k_cache[:, :, :8]), dict(v_cache=p.v_cache.float()),
                   dict(k_cache=p.k_cache.transpose(2, 3)), dict(k_cache=p.k_cache[0, 0]),
                   dict(block_table=p.table.long()), dict(block_table=p.table[0]), dict(block_table=p.table[:1]),
                   dict(block_table=p.table.repeat(1, 2)[:, ::2]), dict(seq_lens=p.lens.float()),
                   dict(seq_lens=p.lens.repeat(2)[::2]), dict(cu_q=p.cu[:2]), dict(cu_q=p.cu.long()),
                   dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=float("inf")),
                   dict(out=torch.empty_like(p.q).float()), dict(out=torch.empty(2, 4, 65, dtype=BF16, device=gpu)[..., 1:]),
                   dict(out=p.q[:1, :1].expand(2, 4, 64)), dict(err_flag=torch.zeros(2, dtype=torch.int32, device=gpu)),
                   dict(k_cache=p.k_cache[:1].expand_as(p.k_cache), v_cache=p.v_cache)):
        refused(cg.paged_attention, args, **change)
    odd = torch.zeros(3, 2, 16, 48, dtype=BF16, device=gpu)
    refused(cg.paged_attention, args, k_cache=odd, v_cache=odd.clone(), q=p.q[..., :48])
    shared = dict(args, prefix_len=16)
    for change in (dict(prefix_len=-1), dict(prefix_len=1.5), dict(prefix_len=True), dict(prefix_len=10 ** 6),
                   dict(prefix_pages=p.table[0].long()), dict(prefix_pages=p.table[0, :0]),
                   dict(prefix_pages=p.table[:, 0].cpu()), dict(prefix_pages=p.table)):
        refused(cg.shared_prefix_attention, shared, **change)
    args = dict(k=p.k, v=p.v, k_cache=p.k_cache, v_cache=p.v_cache, block_table=p.table, seq_lens=p.lens)
    table = cg.rotary_table(64, 64, device=gpu)
    for change in (dict(k=p.k.cpu()), dict(v=p.v[:1]), dict(v=p.v.float()), dict(k=p.q, v=p.q), dict(v_cache=p.k_cache),
                   dict(q=p.q.float()), dict(q=p.q[:, :3]), dict(q=p.q[:1]), dict(q_out=p.q), dict(q=p.q, q_out=p.k),
                   dict(rotary=table.half()), dict(rotary=table[:, :5]), dict(rotary=table.repeat(1, 2)),
                   dict(rotary=table[:0]), dict(rotary=table.cpu()), dict(rotary=table[0]),
                   dict(rotary=table.t().contiguous().t())):
        refused(cg.paged_kv_append, args, **change)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("new", [1, 20])
def test_many_small_weights_add_up(gpu, dtype, hd, new):
    """One key far above 2^17 others, in as many sequences as leave each to one block: those
    keys have a weight below the smallest float16 each and a few parts in a thousand
    together, which the output keeps."""
    n, gap, B = 2 ** 17, 25.5, 2048
    half = torch.finfo(dtype).eps / 2
    cu = torch.arange(B + 1, dtype=torch.int32, device=gpu) * new
    pages = n // 64
    table = torch.arange(pages, dtype=torch.int32, device=gpu)[None].expand(B, pages)  # the same for all
    lens = torch.full((B,), n, dtype=torch.int32, device=gpu)
    k = torch.zeros(pages, 1, 64, hd, dtype=dtype, device=gpu)
    k[0, 0, 0, 0] = 8.0
    q = torch.zeros(B * new, 1, hd, dtype=dtype, device=gpu)
    q[:, :, 0] = 1.0
    # Scores 0 and, of the first key, gap in base 2; token i of the step sees n - new + 1 + i keys.
    scale = gap * math.log(2.0) / 8.0
    tail = torch.arange(n - new, n, dtype=torch.float64).repeat(B)[:, None, None] * 2.0 ** -gap
    for first, rest in ((1.0, 1.0), (0.0, 1.0), (1.0, -1.0)):
        v = torch.full_like(k, rest)
        v[0, 0, 0] = first
        got = cg.paged_attention(q, k, v, table, lens, cu_q=cu, scale=scale)
        want = ((first + rest * tail) / (1.0 + tail)).expand(B * new, 1, hd)
        # The score in base 2 is off by three roundings of gap in 32 bits, so a weight by
        # 4 gap 2^-24; the sums of positive terms by 2^-24 for each addition that a term goes
        # through, in the numerator and the sum: 16 or fewer within one and at most one for each
        # 16 keys (float32 products are added key by key); the weight by its rounding, half a
        # step, or in float16's smallest numbers 2^-25 beside a largest weight of 2^7 at least;
        # then the result's.
        share = tail / (1.0 + tail)
        adds = n if dtype == F32 else n / 16 + 16
        tol = (share * (half + 4 * gap * 2.0 ** -24) + 2 * adds * 2.0 ** -24 * (want.abs() + share)
               + (n * 2.0 ** -32 if dtype == F16 else 0.0) + half * want.abs())
        within(got, want, tol.expand_as(want), f"first {first}, rest {rest}")


@pytest.mark.parametrize("dtype,hd,Hq,Hkv,B,new,cols", [
    (BF16, 64, 12, 12, 32, 2, 64), (F16, 64, 12, 12, 32, 1, 64), (F32, 64, 12, 12, 32, 4, 64), (BF16, 64, 16, 16, 24, 3, 64),
    (BF16, 64, 24, 24, 16, 8, 64), (F32, 32, 12, 12, 10, 2, 144), (BF16, 16, 48, 12, 16, 5, 144), (BF16, 64, 24, 12, 31, 1, 128)])
@pytest.mark.parametrize("prefix", [0, 16])
def test_guessed_tokens_near_a_full_card(gpu, dtype, hd, Hq, Hkv, B, new, cols, prefix):
    """Offsets (one token each among them) where heads and sequences come to about one and a
    half items a CU, with the tables that one launch serves at most."""
    ctx = [prefix + (b * 29) % 150 for b in range(B)]
    tokens = [1 + (b % new if b else new - 1) for b in range(B)]
    p = Problem(dtype, hd, 16, Hq, Hkv, ctx, tokens, prefix=prefix, seed=B + new)
    p.table = torch.cat([p.table, torch.full((B, cols - p.table.shape[1]), -7, dtype=torch.int32)], 1)
    want, bound = attention(p)
    d = p.on(gpu)
    if prefix:
        got = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, prefix, cu_q=d.cu)
    else:
        got = cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, cu_q=d.cu)
    within(got, want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B", [3, 300])
@pytest.mark.parametrize("keys,prefix", [(0, 0), (160, 0), (160, 160), (1024, 1024)])
def test_lengths_past_the_table_set_the_flag(gpu, dtype, B, keys, prefix):
    """Whatever the table holds: nothing at all, or no key past the prefix."""
    ctx = [max(0, keys - 1)] * B
    p = Problem(dtype, 64, 16, 2, 2, ctx, [1] * B, prefix=prefix, seed=B, spare_cols=0)
    if keys == 0:
        p.table, want, bound = p.table[:, :0], torch.zeros(B, 2, 64, dtype=torch.float64), torch.zeros(1)
    else:
        want, bound = attention(p)
    d = p.on(gpu)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    for past in (0, 5, 2 ** 30):
        d.lens = torch.full_like(d.lens, keys)
        d.lens[B - 1] += past
        flag.zero_()
        if prefix:
            got = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, prefix, err_flag=flag)
        else:
            got = cg.paged_attention(d.q, d.k_cache, d.v_cache, d.table, d.lens, err_flag=flag)
        within(got, want, bound, past)
        assert int(flag) == (1 if past else 0), past


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("prefix", [0, 160])
def test_tables_far_wider_than_the_lengths(gpu, dtype, hd, prefix):
    """270 sequences, 8 heads and columns for 2^28 keys: more units of keys than 32 bits
    count, had the sequences such lengths."""
    B, cols = 270, 2 ** 24
    p = Problem(dtype, hd, 16, 8, 8, ctx=[prefix + (b * 61) % 2900 for b in range(B)], new=[1] * B, prefix=prefix, seed=hd)
    want, bound = attention(p)
    d = p.on(gpu)
    # Rows that run on into the next ones' entries, which no length reaches.
    stride = p.table.shape[1]
    flat = torch.full((B * stride + cols,), -7, dtype=torch.int32, device=gpu)
    flat[:B * stride] = d.table.flatten()
    table = flat.as_strided((B, cols), (stride, 1))
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    if prefix:
        got = cg.shared_prefix_attention(d.q, d.k_cache, d.v_cache, table, d.lens, prefix, err_flag=flag)
    else:
        got = cg.paged_attention(d.q, d.k_cache, d.v_cache, table, d.lens, err_flag=flag)
    within(got, want, bound)
    assert int(flag) == 0
