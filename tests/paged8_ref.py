"""float64 restatement of the 8-bit paged cache on the CPU, one block at a time, and
problems of random pages for its tests."""

import math

import torch

NAN = float("nan")
F8 = torch.float8_e4m3fn
TOP = {F8: 448.0, torch.int8: 127.0}
HI = {F8: 119, torch.int8: 121}
LO = -100


def grid(code):
    """The numbers of the codes without a sign, in the codes' order."""
    if code == torch.int8:
        return torch.arange(128, dtype=torch.float64)
    return torch.arange(127, dtype=torch.uint8).view(F8).double()


def nearest(y, code):
    """Values in units of their block on the codes' grid, halves to the even code."""
    g = grid(code)
    mids = (g[1:] + g[:-1]) / 2
    a = y.abs().nan_to_num(0.0, posinf=1e300).contiguous()
    lo, hi = torch.searchsorted(mids, a), torch.searchsorted(mids, a, right=True)
    at = torch.where(lo == hi, lo, torch.where(lo % 2 == 0, lo, hi))
    r = torch.copysign(g[at], y)
    return torch.where(y.isnan(), NAN if code == F8 else 0.0, r)


def exponent(x, code):
    """The smallest exponent for which the finite values of x fit."""
    big = float(x[x.isfinite()].abs().max()) if x.isfinite().any() else 0.0
    e = LO
    while e < HI[code] and big > TOP[code] * 2.0 ** e:
        e += 1
    return e


def values(codes, scale, block):
    """(..., slots, hd) values of codes (..., slots, hd) and bytes (..., blocks)."""
    e = scale.double().clamp(LO + 127, HI[codes.dtype] + 127) - 127
    return codes.double() * torch.pow(torch.tensor(2.0, dtype=torch.float64), e).repeat_interleave(block, -1)[..., None]


class Problem8:
    """Sequences with ``ctx[b]`` keys in the cache and ``new[b]`` tokens of a step; pages in
    random order, slots that no sequence owns full of NaN (int8: of -128), exponents of unused
    blocks of the largest byte.  (e4m3 codes past 448 / ``size`` deviations are NaN.)"""

    def __init__(self, dtype, code, hd, page, block, Hq, Hkv, ctx, new, seed=0, spare_cols=1, pad_rows=0, spread=2,
                 size=100):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dtype, self.code, self.hd, self.page, self.block = g, dtype, code, hd, page, block
        self.Hq, self.Hkv, self.ctx, self.new, self.B = Hq, Hkv, list(ctx), list(new), len(ctx)
        self.total = [c + n for c, n in zip(ctx, new)]
        need = [-(-t // page) for t in self.total]
        self.n_pages = sum(need) + 2
        ids = torch.randperm(self.n_pages, generator=g)
        self.table = torch.full((self.B, max(need + [0]) + spare_cols), -7, dtype=torch.int32)
        for b in range(self.B):
            self.table[b, :need[b]] = ids[sum(need[:b]):sum(need[:b + 1])]
        self.lens = torch.tensor(self.total, dtype=torch.int32)
        self.cu = torch.tensor([sum(new[:b]) for b in range(self.B + 1)], dtype=torch.int32)
        self.cu_rows = torch.tensor([sum(self.total[:b]) for b in range(self.B + 1)], dtype=torch.int32)
        self.n = sum(new) + pad_rows
        # Rows differ in size, so that the blocks' exponents do.
        rnd = lambda n, h: (torch.randn(n, h, hd, generator=g) *
                            2.0 ** torch.randint(-spread, spread + 1, (n, h, 1), generator=g)).to(dtype)
        self.q, self.k, self.v = rnd(self.n, Hq), rnd(self.n, Hkv), rnd(self.n, Hkv)
        shape = (self.n_pages, Hkv, page, hd)
        fill = 0x7f if code == F8 else 0x80
        self.k_cache = torch.full(shape, fill, dtype=torch.uint8).view(code)
        self.v_cache = self.k_cache.clone()
        self.k_scale = torch.full((self.n_pages, Hkv, page // block), 255, dtype=torch.uint8)
        self.v_scale = self.k_scale.clone()
        for b in range(self.B):
            for cache, scale in ((self.k_cache, self.k_scale), (self.v_cache, self.v_scale)):
                x = torch.randn(self.total[b], Hkv, hd, generator=g)
                pos = torch.arange(self.total[b])
                where = self.table[b, pos // page].long(), slice(None), pos % page
                raw = x.mul(size).to(code) if code == F8 else (x * 40).round().clamp(-127, 127).to(code)
                cache.view(torch.uint8)[where] = raw.view(torch.uint8)
                e = torch.randint(127 - 7 - spread, 127 - 7 + spread, (self.total[b] // block + 1, Hkv), generator=g, dtype=torch.uint8)
                scale[self.table[b, pos // page].long(), :, pos % page // block] = e[pos // block]

    def on(self, dev):
        p = Problem8.__new__(Problem8)
        p.__dict__.update({k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()})
        return p

    @property
    def cache(self):
        return self.k_cache, self.v_cache, self.k_scale, self.v_scale, self.table, self.lens

    def keys(self, b):
        """(total, Hkv, hd) keys and values of sequence b in float64."""
        pages = self.table[b, :-(-self.total[b] // self.page)].long()
        out = []
        for cache, scale in ((self.k_cache, self.k_scale), (self.v_cache, self.v_scale)):
            raw = cache.view(torch.uint8)[pages].view(self.code)
            x = values(raw, scale[pages], self.block)
            out.append(x.transpose(1, 2).reshape(-1, self.Hkv, self.hd)[:self.total[b]])
        return out


def turn(x, pos, rotary, interleaved):
    """(heads, hd) rows of position ``pos`` turned in float64."""
    x = x.double().clone()
    rot = rotary.shape[1]
    h = rot // 2
    c, s = rotary[pos, :h].double(), rotary[pos, h:].double()
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, h), slice(h, rot))
    a, b = x[:, i].clone(), x[:, j].clone()
    x[:, i], x[:, j] = a * c - b * s, b * c + a * s
    return x


def append(p, rotary=None, interleaved=False):
    """The pools and exponents after the step, and the turned queries in float64."""
    out = [p.k_cache.clone(), p.v_cache.clone(), p.k_scale.clone(), p.v_scale.clone()]
    q = torch.full(p.q.shape, NAN, dtype=torch.float64)
    bs = p.block
    for b in range(p.B):
        end, t0 = p.total[b], int(p.cu[b]) - (p.total[b] - p.new[b])
        rows = {}
        for pos in range(max(0, end - p.new[b]), end):
            k, qr = p.k[t0 + pos].double(), p.q[t0 + pos].double()
            if rotary is not None:
                k, qr = turn(k, pos, rotary, interleaved), turn(qr, pos, rotary, interleaved)
            q[t0 + pos] = qr
            rows[pos] = (k, p.v[t0 + pos].double())
        for j in sorted({pos // bs for pos in rows}):
            at = [pos for pos in range(j * bs, (j + 1) * bs) if pos in rows]
            page, s0 = int(p.table[b, j * bs // p.page]), j * bs % p.page
            for which in range(2):
                codes, scale = out[which].view(torch.uint8), out[2 + which]
                for h in range(p.Hkv):
                    x = torch.stack([rows[pos][which][h] for pos in at])
                    e = exponent(x, p.code)
                    front = at[0] - j * bs
                    if front:
                        old = min(max(int(scale[page, h, s0 // bs]) - 127, LO), HI[p.code])
                        if e > old:
                            there = codes[page, h, s0:s0 + front].view(p.code).double() * 2.0 ** (old - e)
                            codes[page, h, s0:s0 + front] = nearest(there, p.code).float().to(p.code).view(torch.uint8)
                        e = max(e, old)
                    scale[page, h, s0 // bs] = e + 127
                    codes[page, h, s0 + front:s0 + front + len(at)] = (
                        nearest(x * 2.0 ** -e, p.code).float().to(p.code).view(torch.uint8))
    return out, q


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
            # Cached values are exact in bf16, queries in one (bf16), two (fp16) or three
            # (fp32) bf16 parts, so a score is a sum of up to 3 hd exact products (each partial
            # sum rounded to 32 bits) and a scaling, in base 2; the shift by the maximum, the
            # exponential and the rescaling of a running sum add a few roundings of numbers as
            # large as the scores.  A relative error d of every weight moves the output by at
            # most 2 d sum(w |v|) (numerator and normaliser); the sums over up to 3 n products
            # by 3 n u32 each.
            big = (k.abs() @ q.abs())[..., 0].amax(-1) * scale
            d = (3 * p.hd + 16) * u32 * (big + 1)
            mass = (w @ v.abs())[:, 0]
            # The weights are rounded to the dtype or finer before they meet the values; then
            # the result is rounded.
            out[t] = o
            bound[t] = (2 * d[:, None] + 6 * n * u32 + max(u, u32)) * mass + max(u, u32) * o.abs() + 2 ** -100
            if p.dtype == torch.float16:
                bound[t] += 2.0 ** -25  # half of its smallest step
    return out, bound
