"""float64 restatement of the paged cache's operators on the CPU, one token at a
time, and problems of random pages for their tests."""

import math

import torch

NAN = float("nan")


class Problem:
    """Sequences with ``ctx[b]`` keys in the cache and ``new[b]`` tokens of a step, pages
    in random order, every slot that no sequence owns filled with NaN."""

    def __init__(self, dtype, hd, page, Hq, Hkv, ctx, new, prefix=0, seed=0, spare_cols=1, pad_rows=0,
                 scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dtype, self.hd, self.page, self.Hq, self.Hkv = g, dtype, hd, page, Hq, Hkv
        self.ctx, self.new, self.prefix, self.B = list(ctx), list(new), prefix, len(ctx)
        total = [c + n for c, n in zip(ctx, new)]
        self.total = total
        shared = prefix // page
        need = [max(0, -(-t // page) - shared) for t in total]
        self.n_pages = shared + sum(need) + 2
        cols = max([shared] + [-(-t // page) for t in total]) + spare_cols
        ids = torch.randperm(self.n_pages, generator=g)
        self.table = torch.full((self.B, cols), -7, dtype=torch.int32)  # unused entries name no page
        at = shared
        for b in range(self.B):
            self.table[b, :shared] = ids[:shared]
            self.table[b, shared:shared + need[b]] = ids[at:at + need[b]]
            at += need[b]
        self.lens = torch.tensor(total, dtype=torch.int32)
        self.cu = torch.tensor([sum(new[:b]) for b in range(self.B + 1)], dtype=torch.int32)
        self.n = sum(new) + pad_rows
        rnd = lambda *s: (torch.randn(*s, generator=g) * scale).to(dtype)
        self.q, self.k, self.v = rnd(self.n, Hq, hd), rnd(self.n, Hkv, hd), rnd(self.n, Hkv, hd)
        self.k_cache = torch.full((self.n_pages, Hkv, page, hd), NAN, dtype=dtype)
        self.v_cache = self.k_cache.clone()
        for b in range(self.B):
            pos = torch.arange(total[b])
            where = self.table[b, pos // page].long(), slice(None), pos % page
            self.k_cache[where], self.v_cache[where] = rnd(total[b], Hkv, hd), rnd(total[b], Hkv, hd)

    def on(self, dev):
        """Moved to the device (a shallow copy)."""
        p = Problem.__new__(Problem)
        p.__dict__.update({k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()})
        return p

    def keys(self, b):
        pos = torch.arange(self.total[b])
        where = self.table[b, pos // self.page].long(), slice(None), pos % self.page
        return self.k_cache[where].double(), self.v_cache[where].double()


def attention(p, scale=None):
    """(n, Hq, hd) outputs in float64, zeros for rows without a key, NaN for padding rows,
    and a bound on what rounding may move each by."""
    scale = 1.0 / math.sqrt(p.hd) if scale is None else scale
    out = torch.full((p.n, p.Hq, p.hd), NAN, dtype=torch.float64)
    bound = torch.zeros_like(out)
    u32 = 2.0 ** -24
    u = 0.0 if p.dtype == torch.float32 else torch.finfo(p.dtype).eps / 2
    G = p.Hq // p.Hkv
    for b in range(p.B):
        K, V = p.keys(b) if p.total[b] else (None, None)
        for i in range(p.new[b]):
            t, n = int(p.cu[b]) + i, p.total[b] - p.new[b] + i + 1
            if n <= 0:
                out[t] = 0
                continue
            k = K[:n].repeat_interleave(G, 1).transpose(0, 1)   # (Hq, n, hd)
            v = V[:n].repeat_interleave(G, 1).transpose(0, 1)
            q = p.q[t].double()[:, :, None]
            s = (k @ q)[..., 0] * scale
            w = torch.softmax(s, -1)[:, None]
            o = (w @ v)[:, 0]
            # A score is a sum of hd products (each and every partial sum rounded to 32
            # bits) and a scaling, in base 2; the shift by the maximum, the exponential and
            # the rescaling of a running sum add a few roundings of numbers as large as the
            # scores.  A relative error d of every weight moves the output by at most
            # 2 d sum(w |v|) (numerator and normaliser); the sums over n keys by n u32 each.
            big = (k.abs() @ q.abs())[..., 0].amax(-1) * scale
            d = (p.hd + 16) * u32 * (big + 1)
            mass = (w @ v.abs())[:, 0]
            # The weights are rounded to the dtype before they meet the values, below 2^-14
            # (fp16) by 2^-25 at most; then the result is rounded.
            tiny = 2.0 ** -25 * v.abs().sum(1) if p.dtype == torch.float16 else 0.0
            out[t] = o
            bound[t] = (2 * d[:, None] + 2 * n * u32 + u) * mass + tiny + max(u, u32) * o.abs() + 2 ** -126
    return out, bound


def turn(x, pos, rotary, interleaved):
    """(heads, hd) rows of position ``pos`` turned in float64, and the rounding bound."""
    x = x.double().clone()
    size = x.abs()
    rot = rotary.shape[1]
    h = rot // 2
    c, s = rotary[pos, :h].double(), rotary[pos, h:].double()
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, h), slice(h, rot))
    a, b = x[:, i].clone(), x[:, j].clone()
    size[:, i] = (a * c).abs() + (b * s).abs()
    size[:, j] = (b * c).abs() + (a * s).abs()
    x[:, i], x[:, j] = a * c - b * s, b * c + a * s
    return x, size


def append(p, rotary=None, interleaved=False):
    """(k_cache, v_cache, q, bounds of k_cache and q) in float64 after the step."""
    kc, vc = p.k_cache.double(), p.v_cache.double()
    q = torch.full(p.q.shape, NAN, dtype=torch.float64)
    kb, qb = torch.zeros_like(kc), torch.zeros_like(q)
    # Two products and a sum in 32 bits, then one rounding to the dtype.
    u32, u = 2.0 ** -24, 0.0 if p.dtype == torch.float32 else torch.finfo(p.dtype).eps / 2
    rel = 2 * u32 + u
    for b in range(p.B):
        for i in range(p.new[b]):
            t, pos = int(p.cu[b]) + i, p.total[b] - p.new[b] + i
            if pos < 0:
                continue
            page, slot = int(p.table[b, pos // p.page]), pos % p.page
            kr, ks, qr, qs = p.k[t].double(), 0.0, p.q[t].double(), 0.0
            if rotary is not None:
                (kr, ks), (qr, qs) = turn(p.k[t], pos, rotary, interleaved), turn(p.q[t], pos, rotary, interleaved)
                rot = rotary.shape[1]
                kb[page, :, slot, :rot] = rel * 1.01 * ks[:, :rot] + 2 ** -25 * (p.dtype == torch.float16)
                qb[t, :, :rot] = rel * 1.01 * qs[:, :rot] + 2 ** -25 * (p.dtype == torch.float16)
            kc[page, :, slot], vc[page, :, slot], q[t] = kr, p.v[t].double(), qr
    return kc, vc, q, kb, qb


def within(got, want, bound, what=""):
    """Every value within its bound of the wanted one; NaN where NaN is wanted."""
    got, want = got.detach().cpu().double(), want.double()
    miss = torch.isnan(want)
    err = (got - want).abs()
    bad = ~((err <= bound) | miss)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside their bounds, the worst "
                           f"{(err / bound.clamp(min=1e-300))[bad].max().item():.3g} times it")
