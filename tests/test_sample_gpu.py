"""sample_tokens on the GPU against the float64 draw: every token has to be the same one."""

import math

import pytest
import torch

import cutilegpt_amd as cg
from sample_ref import draw, kept

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF, NAN = math.inf, math.nan


def check(x, u, T=1.0, k=0, p=1.0, m=0.0, gpu="cuda", per_row=False, view=None):
    """x (B, V) and u (B,) on the CPU; settings numbers or lists of a value a row."""
    B, V = x.shape
    rows = lambda s: s if isinstance(s, (list, tuple)) else [s] * B
    as_tensor = per_row or any(isinstance(s, (list, tuple)) for s in (T, k, p, m))
    if as_tensor:
        t = [torch.tensor(rows(s), dtype=d).to(gpu) for s, d in ((T, F32), (k, torch.int32), (p, F32), (m, F32))]
        Ts, ks, ps, ms = (a.tolist() for a in t)
    else:
        t = [T, k, p, m]
        Ts, ks, ps, ms = rows(T), rows(k), rows(p), rows(m)
    d = x.to(gpu) if view is None else view(x.to(gpu))
    got = cg.sample_tokens(d, u.to(gpu), temperature=t[0], top_k=t[1], top_p=t[2], min_p=t[3])
    assert got.shape == (B,) and got.dtype == torch.int64
    got = got.tolist()
    for b in range(B):
        want, margin = draw(x[b], min(max(float(u[b]), 0.0), 1.0) if u[b] == u[b] else 0.0, Ts[b], ks[b], ps[b], ms[b])
        # Weights are off by 2^-44 of the largest each, borders by as much an entry.
        assert got[b] == want or margin < (V + 64) * 2.0 ** -44, (b, got[b], want, margin)
    return got


def logits(B, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * spread
    x[torch.arange(B), torch.randint(V, (B,), generator=g)] += torch.rand(B, generator=g) * 10
    return x.to(dtype), torch.rand(B, generator=g)


SETTINGS = [dict(), dict(T=0.0), dict(T=0.7, k=40), dict(k=1), dict(T=1.5, p=0.9), dict(m=0.05),
            dict(T=0.8, k=50, p=0.8, m=0.01), dict(T=3.0, k=1000, p=0.99), dict(p=0.0), dict(T=0.05, p=0.5)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 1000, 4095, 4096, 4097, 20011])
def test_vocabularies(gpu, dtype, V):
    for i, s in enumerate(SETTINGS):
        x, u = logits(4, V, dtype, seed=V + i)
        check(x, u, **s)


@pytest.mark.parametrize("dtype,V", [(F32, 50257), (BF16, 50257), (F16, 128000), (F32, 262147)])
def test_large_vocabularies(gpu, dtype, V):
    for i, s in enumerate([dict(), dict(T=0.8, k=40, p=0.95), dict(T=2.0, p=0.99), dict(T=1.0, k=5000, m=1e-4)]):
        x, u = logits(2, V, dtype, seed=i, spread=1.5)
        check(x, u, **s)


def test_many_rows(gpu):
    x, u = logits(300, 700, BF16, seed=1)
    check(x, u, T=0.9, k=30, p=0.9)
    check(x, u)


@pytest.mark.parametrize("V", [300, 5000, 50257])
def test_equal_logits(gpu, V):
    """Equal logits are kept by index."""
    x = torch.zeros(3, V)
    u = torch.tensor([0.0, 0.5, 1 - 2.0 ** -24])
    for s in (dict(), dict(k=3), dict(k=V - 1), dict(p=0.25), dict(p=0.5), dict(k=V // 2, p=0.5), dict(m=1.0), dict(p=1.0 - 2.0 ** -30)):
        check(x, u, **s)
    assert check(x, u, k=10) == [0, 5, 9]
    # A few values, each many times, the largest ones not first.
    g = torch.Generator().manual_seed(V)
    x = torch.randint(0, 4, (3, V), generator=g).float()
    for s in (dict(k=V // 7), dict(p=0.3), dict(p=0.9), dict(k=V // 3, p=0.7), dict(k=V // 2, m=0.2), dict(T=0.01, k=V // 3)):
        check(x, u, **s)


def test_both_zeros_are_equal(gpu):
    x = torch.zeros(2, 40)
    x[0, ::2] = -0.0
    x[1, 1::2] = -0.0
    assert check(x, torch.tensor([0.99, 0.99]), k=4) == [3, 3]


@pytest.mark.parametrize("dtype", [F32, F16])
def test_crowded_logits(gpu, dtype):
    """Thousands of different logits within a hair of each other, near the largest and far
    below it."""
    g = torch.Generator().manual_seed(5)
    V = 9000
    x = torch.empty(4, V).uniform_(2.0, 2.008, generator=g)
    x[1] = 2.0 + torch.randperm(V, generator=g) * 2.0 ** -22
    x[2, 100:] -= 30.0
    x[3] = torch.empty(V).uniform_(-5000.0, 0.0, generator=g)
    u = torch.tensor([0.3, 0.7, 0.2, 0.9])
    for s in (dict(k=1), dict(k=2500), dict(p=0.3), dict(p=0.99), dict(k=4000, p=0.5), dict(k=8999), dict(T=0.01, p=0.6), dict(T=100.0, k=7777, p=0.9)):
        check(x.to(dtype), u, **s)


def test_masked_logits(gpu):
    V = 3000
    x, u = logits(8, V, F32, seed=3)
    low = torch.finfo(F32).min
    x[0] = -INF                      # nothing
    x[1] = -INF
    x[1, 777] = -5.0                 # one token
    x[2, 5:2900] = -INF
    x[3] = low                       # all of the type's lowest value
    x[4, :] = low
    x[4, 9] = 1.0
    x[5, 100], x[5, 7] = INF, INF    # infinities share everything
    x[6, ::3] = NAN                  # skipped
    x[7] = NAN
    for s in (dict(), dict(k=5), dict(p=0.9), dict(T=0.3, k=20, p=0.5, m=0.1), dict(T=0.0), dict(T=INF), dict(T=1e30, k=7)):
        got = check(x, u, **s)
        assert got[0] == -1 and got[7] == -1 and got[1] == 777 and got[4] != -1 and got[5] in (7, 100)
    f16 = x.clone()
    f16[3:5] = f16[3:5].clamp(min=torch.finfo(F16).min)
    check(f16.to(F16), u, T=0.9, k=50, p=0.9)


@pytest.mark.parametrize("T", [1e-30, 1e-6, 1e-3, 50.0, 1e6, 1e38, INF])
def test_temperatures(gpu, T):
    x, u = logits(3, 2500, F32, seed=8)
    for s in (dict(), dict(k=10), dict(p=0.7), dict(k=100, p=0.9, m=0.5)):
        check(x, u, T=T, **s)


def test_random_numbers_at_the_ends(gpu):
    x, _ = logits(7, 500, F32, seed=2)
    x[:, 0], x[:, -1] = -INF, -INF
    u = torch.tensor([0.0, 2.0 ** -149, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, NAN])
    for s in (dict(), dict(k=9), dict(p=0.5), dict(m=0.2)):
        got = check(x, u, **s)
        idx = [kept(x[b], 1.0, s.get("k", 0), s.get("p", 1.0), s.get("m", 0.0))[0] for b in range(7)]
        assert got[0] == min(idx[0]) and got[2] == got[2] and got[3] == max(idx[3]) and got[6] == min(idx[6])


def test_settings_of_rows(gpu):
    B = 12
    x, u = logits(B, 4000, BF16, seed=4)
    check(x, u, T=[0.0, 1.0, 0.5, 2.0] * 3, k=[0, 1, 50, 3999, 4000, 100000, -3, 10, 2, 0, 7, 300],
          p=[1.0, 0.9, 0.5, 0.0, 1.5, 0.99] * 2, m=[0.0, 0.1, 1.0] * 4)
    # What makes no sense counts as the nearest that does.
    d = x.to(gpu)
    one = lambda v, dt=F32: torch.full((B,), v, dtype=dt, device=gpu)
    plain = cg.sample_tokens(d, u.to(gpu))
    for kw in (dict(top_p=one(NAN)), dict(min_p=one(NAN)), dict(top_k=one(-2 ** 31, torch.int32)), dict(min_p=one(-1.0)), dict(top_p=one(INF))):
        assert torch.equal(cg.sample_tokens(d, u.to(gpu), **kw), plain), kw
    greedy = cg.sample_tokens(d, u.to(gpu), temperature=0.0)
    assert torch.equal(greedy, d.float().argmax(-1))
    for kw in (dict(temperature=one(-1.0)), dict(temperature=one(NAN)), dict(min_p=one(7.0), top_k=one(1, torch.int32)),
               dict(top_p=one(-1.0)), dict(top_k=1)):
        assert torch.equal(cg.sample_tokens(d, u.to(gpu), **kw), greedy), kw


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_strided_rows(gpu, dtype):
    """Padded rows of odd strides from odd places, whose padding is never taken; columns apart
    are copied."""
    x, u = logits(5, 777, dtype, seed=6)

    def padded(d, off, ld):
        w = torch.full((5 * ld + off,), 100.0, dtype=dtype, device=d.device)
        v = w.as_strided((5, 777), (ld, 1), off)
        v.copy_(d)
        return v

    for off, ld in ((0, 777), (1, 778), (2, 779), (3, 801), (5, 780), (7, 1024)):
        check(x, u, T=0.9, k=40, p=0.9, view=lambda d: padded(d, off, ld))
        check(x, u, view=lambda d: padded(d, off, ld))
    check(x, u, p=0.8, view=lambda d: d.t().contiguous().t())
    same = x[:1].to(gpu).expand(5, -1)
    got = cg.sample_tokens(same, u.to(gpu), top_p=0.8).tolist()
    assert got == check(x[:1].repeat(5, 1), u, p=0.8)


def test_rows_past_32_bits(gpu):
    V, ld, B = 600, (1 << 30) + 3, 4
    x, u = logits(B, V, BF16, seed=7)
    w = torch.empty(ld * (B - 1) + V, dtype=BF16, device=gpu)
    v = w.as_strided((B, V), (ld, 1))
    v.copy_(x)
    check(x, u, T=0.8, p=0.9, view=lambda d: v)


def test_frequencies(gpu):
    """Evenly spaced numbers hit every token as often as its weight says."""
    n, V = 4096, 50
    g = torch.Generator().manual_seed(1)
    row = torch.randn(V, generator=g)
    u = (torch.arange(n) + 0.5) / n
    got = cg.sample_tokens(row.repeat(n, 1).to(gpu), u.to(gpu), temperature=0.6).cpu()
    share = torch.bincount(got, minlength=V) / n
    assert bool(((share - torch.softmax(row.double() / 0.6, 0)).abs() <= 1.0 / n).all())


def test_out_streams_and_twice(gpu):
    x, u = logits(64, 30000, BF16, seed=9)
    x, u = x.to(gpu), u.to(gpu)
    want = cg.sample_tokens(x, u, top_k=200, top_p=0.9)
    out = torch.empty(64, dtype=torch.int64, device=gpu)
    assert cg.sample_tokens(x, u, top_k=200, top_p=0.9, out=out) is out and torch.equal(out, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(cg.sample_tokens(x, u, top_k=200, top_p=0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) for a in got)
    assert cg.sample_tokens(x[:0], u[:0]).shape == (0,)


def test_captured(gpu):
    """A captured draw replays with the logits, numbers and settings of the moment."""
    B, V = 9, 5000
    x, u = logits(B, V, F32, seed=10)
    x, u = x.to(gpu), u.to(gpu)
    t, k = torch.ones(B, device=gpu), torch.zeros(B, dtype=torch.int32, device=gpu)
    cg.sample_tokens(x, u, temperature=t, top_k=k, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cg.sample_tokens(x, u, temperature=t, top_k=k, top_p=0.9)
    for i in range(4):
        y, v = logits(B, V, F32, seed=20 + i)
        x.copy_(y)
        u.copy_(v)
        t.fill_(0.5 + 0.3 * i)
        k.fill_(10 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cg.sample_tokens(x, u, temperature=t, top_k=k, top_p=0.9)), i


def test_refusals(gpu):
    x, u = torch.zeros(3, 50, device=gpu), torch.zeros(3, device=gpu)

    def refused(match, x=x, u=u, **kw):
        with pytest.raises(ValueError, match=match):
            cg.sample_tokens(x, u, **kw)

    refused("unsupported dtype", x=x.double())
    refused("logits must be", x=x[0])
    refused("logits must be", x=x[:, :0])
    refused("u must", u=u[:2])
    refused("u must", u=u.double())
    refused("u must", u=u.cpu())
    refused("temperature", temperature=-0.5)
    refused("temperature", temperature=NAN)
    refused("temperature", temperature=u[:2])
    refused("top_k", top_k=-1)
    refused("top_k", top_k=2.0)
    refused("top_k", top_k=u)
    refused("top_p", top_p=1.1)
    refused("top_p", top_p=NAN)
    refused("min_p", min_p=-0.1)
    refused("min_p", min_p=torch.zeros(3, dtype=torch.float64, device=gpu))
    refused("out must", out=torch.zeros(3, dtype=torch.int32, device=gpu))
    refused("shape outside", x=torch.zeros(1, (1 << 20) + 1, device=gpu), u=u[:1])


def draws(row, u, T=1.0, k=0, p=1.0, m=0.0):
    """``draw`` of one row for many numbers: (tokens, margins), (tokens that can come)."""
    idx, w = kept(row, T, k, p, m)
    order = sorted((i, a) for i, a in zip(idx, w) if a > 0)
    at, w = torch.tensor([i for i, _ in order]), torch.tensor([a for _, a in order], dtype=torch.float64)
    ends = w.cumsum(0)
    goal = u.double() * ends[-1]
    j = torch.searchsorted(ends, goal, right=True).clamp(max=len(at) - 1)
    return at[j], torch.minimum(goal - (ends[j] - w[j]), ends[j] - goal) / ends[-1], at


def check_row(row, n, gpu, seed, **s):
    """n draws from one row, each the float64 one."""
    u = torch.rand(n, generator=torch.Generator().manual_seed(seed))
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    want, margin, can = draws(row, u, **s)
    T, rest = s.get("T", 1.0), dict(top_k=s.get("k"), top_p=s.get("p"), min_p=s.get("m"))
    got = cg.sample_tokens(row.repeat(n, 1).to(gpu), u.to(gpu), temperature=T, **rest).cpu()
    assert bool(torch.isin(got, can).all()), (s, "tokens without a weight", got[~torch.isin(got, can)][:5].tolist())
    bad = (got != want) & (margin >= (len(row) + 64) * 2.0 ** -44)
    assert not bad.any(), (s, int(bad.sum()), got[bad][:5].tolist(), want[bad][:5].tolist())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [5000, 50257])
@pytest.mark.parametrize("low", [-1e3, -1e4, -65504.0, -1e9, None])
def test_finite_masks(gpu, dtype, V, low):
    """Masked entries are finite (None: the type's lowest value) among thousands that can be drawn,
    with nothing cut, min_p alone, and a top_k that reaches into the masked ones."""
    if dtype == F16 and low == -1e9:
        low = -3e4
    low = torch.finfo(dtype).min if low is None else low
    g = torch.Generator().manual_seed(V)
    for n_masked in (1, 20, V // 2):
        row = torch.randn(V, generator=g) * 2.5
        row[torch.randperm(V, generator=g)[:n_masked]] = low
        row = row.to(dtype)
        for T in (0.1, 0.3, 0.7, 0.8, 1.0, 1.2):
            check_row(row, 48, gpu, n_masked, T=T)
        check_row(row, 48, gpu, 1, T=1.2, m=1e-6)
        check_row(row, 48, gpu, 2, T=0.8, m=1e-12)
        check_row(row, 48, gpu, 3, T=0.8, k=V - n_masked // 2)
        check_row(row, 48, gpu, 4, T=0.7, k=V - n_masked // 2, m=1e-9)
        check_row(row, 48, gpu, 5, T=0.8, p=0.999999)


@pytest.mark.parametrize("T", [1e-7, 1e-8, 1e-9, 1e-10, 1e-20, 1e-38])
@pytest.mark.parametrize("V", [1500, 9000])
def test_temperatures_below_the_logits_steps(gpu, T, V):
    """Thousands of logits a few steps of fp32 apart, at temperatures that make one step the whole
    distribution or more."""
    g = torch.Generator().manual_seed(V)
    row = 10.0 + torch.randint(-30, 1, (V,), generator=g).float() * 2.0 ** -20
    row[::7] = 10.0
    for s in (dict(), dict(k=1000), dict(k=V - 3), dict(p=0.5), dict(p=0.99), dict(m=0.5), dict(m=1e-9), dict(k=1200, p=0.7, m=0.01)):
        check_row(row, 32, gpu, 1, T=T, **s)
