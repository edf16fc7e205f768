"""Performance cases of serving from a cache held in 8 bits, and of choosing the tokens.

A case is a dict of plain values.  ``listed()`` names twelve of them, ``draw(rng)``
gives more of the same ranges, ``prepare`` makes what a serving program holds before
the call, ``run`` is one pass, ``work`` what a pass cannot do without, ``exact`` the
same result in float64.

The kinds of case:

    write    paged_kv_append_8bit, the step's keys and values into their pages as 8-bit
             codes, then paged_kv_read_8bit, the sequences' keys and values back
    attend   paged_attention_8bit: the step's queries against each sequence's pages
    sample   sample_tokens: temperature, top-k, top-p, min-p and given random numbers

A cached value is code * 2^e: the code an e4m3 number or an int8, the exponent e one for
each block of tokens of a page and key head (a byte, e + 127), the smallest for which
the block's largest value fits.  A step that goes on in a block keeps the larger
exponent, the codes there rounded again where it grew.

With ``own`` false ``run`` computes a plain form in elementary torch operations in
32 bits (64 where a rounding border or a long sum is at stake), rounded once at the end.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# The largest code as mantissa * 2^exponent (mantissa in [0.5, 1)), and the exponents a block may have.
_CODES = {"e4m3": dict(top=448.0, mant=0.875, exp=9, hi=119), "int8": dict(top=127.0, mant=127 / 128, exp=7, hi=121)}
_LO = -100


def listed():
    return [
        # The first tokens of eight answers to short prompts enter the cache, heads of the
        # smallest GPT-2: latency.
        dict(name="write_step", kind="write", dtype="bfloat16", cache="e4m3", B=8, q=1, lo=1, hi=60, Hq=12,
             Hkv=12, hd=64, page=16, block=16, rot=0, interleaved=False, order=1),
        # Sixteen ragged prompts entering the cache at once, fully rotated heads, int8.
        dict(name="write_prompts", kind="write", dtype="bfloat16", cache="int8", B=16, q=2048, lo=0, hi=0, Hq=12,
             Hkv=12, hd=64, page=64, block=64, rot=64, interleaved=False, order=2),
        # Chunks of prompts in fp32 on odd pages of three blocks, grouped heads rotated in
        # part, pairs side by side.
        dict(name="write_chunk_fp32", kind="write", dtype="float32", cache="e4m3", B=5, q=300, lo=0, hi=2000, Hq=8,
             Hkv=2, hd=128, page=24, block=8, rot=32, interleaved=True, order=3),
        # One sequence at a prompt, half a context behind it: latency.
        dict(name="attend_single", kind="attend", dtype="bfloat16", cache="e4m3", B=1, q=1, lo=500, hi=500, Hq=12,
             Hkv=12, hd=64, page=16, block=16, order=4),
        # A full decode batch of very different lengths, the heads of the largest GPT-2.
        dict(name="attend_ragged", kind="attend", dtype="bfloat16", cache="int8", B=64, q=1, lo=1, hi=8192, Hq=25,
             Hkv=25, hd=64, page=64, block=64, order=5),
        # Few sequences with very long contexts, four query heads to a key head.
        dict(name="attend_long", kind="attend", dtype="float16", cache="e4m3", B=4, q=1, lo=90000, hi=130000,
             Hq=32, Hkv=8, hd=128, page=128, block=128, order=6),
        # Guessed tokens of seven short sequences checked at once, fp32, odd pages.
        dict(name="attend_verify_fp32", kind="attend", dtype="float32", cache="int8", B=7, q=5, lo=30, hi=700,
             Hq=6, Hkv=3, hd=32, page=10, block=5, order=7),
        # Prompts taken in chunks: long queries, each behind the context it already has.
        dict(name="attend_chunks", kind="attend", dtype="bfloat16", cache="e4m3", B=16, q=2048, lo=0, hi=4096,
             Hq=16, Hkv=16, hd=64, page=32, block=16, order=8),
        # One answer's next token from fp32 logits, the settings a user types: latency.
        dict(name="sample_one", kind="sample", dtype="float32", B=1, V=50257, ld=50257, spread=2.5, masked=0.0,
             rows=False, temperature=0.8, top_k=40, top_p=0.95, min_p=0.0, order=9),
        # A decode batch from the padded LM head in bf16 (many equal logits), every request
        # with settings of its own.
        dict(name="sample_requests", kind="sample", dtype="bfloat16", B=64, V=50257, ld=50304, spread=3.0,
             masked=0.0, rows=True, temperature=1.2, top_k=200, top_p=0.9, min_p=0.05, order=10),
        # A large batch over a large vocabulary, flat distributions, top-p alone.
        dict(name="sample_large", kind="sample", dtype="float32", B=256, V=128000, ld=128000, spread=1.5,
             masked=0.0, rows=False, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, order=11),
        # Answers held to a grammar: nearly all of the vocabulary is masked; nothing cut.
        dict(name="sample_grammar", kind="sample", dtype="float16", B=33, V=32001, ld=32001, spread=2.0,
             masked=0.97, rows=False, temperature=0.7, top_k=0, top_p=1.0, min_p=0.0, order=12),
    ]


# ------------------------------------------------------------------------- drawn cases


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = [work(c) for c in listed()]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    kind = rng.choice(["write", "write", "attend", "attend", "sample", "sample"])
    while True:
        case = _draw_kind(rng, kind)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and _dense_bytes(case) <= 2.0e10:
            return case


def _draw_kind(rng, kind):
    if kind == "sample":
        V = _log_int(rng, 16, 200000)
        return dict(kind=kind, dtype=rng.choice(["float32", "bfloat16", "float16"]), B=_log_int(rng, 1, 256), V=V,
                    ld=V + rng.choice([0, 0, 1, 47]), spread=rng.choice([0.5, 1.5, 3.0, 6.0]),
                    masked=rng.choice([0.0, 0.0, 0.5, 0.99]), rows=rng.choice([False, True]),
                    temperature=rng.choice([0.0, 0.3, 0.8, 1.0, 1.7]), top_k=rng.choice([0, 0, 1, 40, 1000]),
                    top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02, 0.2]),
                    order=rng.randrange(1 << 30))
    group = rng.choice([1, 1, 2, 3, 4, 8])
    kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 20, 25])
    page, block = rng.choice([(1, 1), (8, 8), (10, 5), (16, 16), (16, 1), (24, 8), (32, 16), (32, 32), (64, 64), (64, 32),
                              (100, 25), (128, 128), (128, 16), (256, 256)])
    case = dict(kind=kind, dtype=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]),
                cache=rng.choice(["e4m3", "int8"]), Hkv=kv, Hq=kv * group, hd=rng.choice([16, 32, 64, 64, 128]),
                page=page, block=block, order=rng.randrange(1 << 30))
    if kind == "write":
        rot = rng.choice([0, case["hd"], case["hd"], case["hd"] // 2])
        hi = _log_int(rng, 1, 4096)
        case.update(B=_log_int(rng, 1, 128), q=rng.choice([1, _log_int(rng, 1, 2048)]), lo=rng.randint(0, hi),
                    hi=hi, rot=rot, interleaved=rng.choice([False, True]))
        return case
    # Single tokens, a few guessed ones, or chunks of prompts.
    case["q"] = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
    hi = _log_int(rng, 1, 130000)
    case.update(B=_log_int(rng, 1, 128), lo=rng.randint(0, hi), hi=hi)
    return case


# --------------------------------------------------------------------- lengths and work


def _lengths(case):
    """(tokens of this step, keys with them) of every sequence.  A sequence brings 1 to
    ``q`` tokens behind a context of ``lo`` to ``hi``."""
    rng = random.Random(case["order"])
    new = [rng.randint(max(1, case["q"] // 8), case["q"]) for _ in range(case["B"])]
    return new, [n + rng.randint(case["lo"], case["hi"]) for n in new]


def _dense_bytes(case):
    """What the plain form, or 64 bits, take on the way, roughly."""
    if case["kind"] == "sample":
        return 100 * case["B"] * case["V"]
    new, total = _lengths(case)
    if case["kind"] == "write":
        slots = sum(total) + case["B"] * case["page"]
        return 40 * (sum(new) * (case["Hq"] + 2 * case["Hkv"]) + slots * case["Hkv"]) * case["hd"]
    cells = case["B"] * case["Hkv"] * max(total) * case["hd"]
    return 4 * (4 * cells + 3 * case["B"] * case["Hq"] * max(new) * max(total))


def work(case):
    """Rows, codes, exponents, tables and logits read once, results written once; only the
    pairs that the causal order leaves count."""
    e = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "sample":
        cells = case["B"] * case["V"]
        return {"bytes": cells * e + case["B"] * (4 + 8 + (16 if case["rows"] else 0)), "flops": 4 * cells}
    new, total = _lengths(case)
    Hq, Hkv, hd = case["Hq"], case["Hkv"], case["hd"]
    n, keys = sum(new), sum(total)
    if case["kind"] == "write":
        rot = case["rot"]
        q = Hq if rot else 0
        blocks = sum((t - 1) // case["block"] - (t - m) // case["block"] + 1 for m, t in zip(new, total))
        append = n * (2 * Hkv * hd * (e + 1) + 2 * q * hd * e + rot * 4) + 2 * blocks * Hkv
        read = keys * 2 * Hkv * hd * (1 + e) + 2 * (keys // case["block"]) * Hkv
        tables = 4 * (keys // case["page"] + 4 * case["B"])
        return {"bytes": append + read + tables, "flops": n * (2 * Hkv * hd + 3 * (Hkv + q) * rot) + 2 * keys * Hkv * hd}
    pairs = sum(m * t - m * (m - 1) // 2 for m, t in zip(new, total))
    table = 4 * (keys // case["page"] + 2 * case["B"])
    return {"bytes": 2 * keys * Hkv * hd + 2 * (keys // case["block"]) * Hkv + 2 * n * Hq * hd * e + table,
            "flops": 4 * pairs * Hq * hd}


# ------------------------------------------------------------------------------- inputs


def _pool(g, n_pages, Hkv, page, hd, block, cache):
    """Codes and exponents of pages whose blocks differ in size by their tokens: normal
    values, quantised a few pages at a time."""
    c = _CODES[cache]
    dt = torch.float8_e4m3fn if cache == "e4m3" else torch.int8
    codes = torch.empty(n_pages, Hkv, page, hd, dtype=dt, device="cuda")
    scale = torch.empty(n_pages, Hkv, page // block, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (Hkv * page * hd))
    for i in range(0, n_pages, step):
        m = min(step, n_pages - i)
        x = torch.empty(m, Hkv, page // block, block, hd, device="cuda").normal_(generator=g)
        x *= torch.empty(m, Hkv, page // block, 1, 1, device="cuda").normal_(std=0.5, generator=g).exp_()
        big, ex = torch.frexp(x.abs().amax((-2, -1)))
        ex = ex - c["exp"] + (big > c["mant"]).int()
        x *= torch.exp2(-ex.float())[..., None, None]
        x = x.reshape(m, Hkv, page, hd)
        codes[i:i + m] = x.to(dt) if cache == "e4m3" else x.round_().to(dt)
        scale[i:i + m] = (ex + 127).to(torch.uint8)
    return codes, scale


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    if case["kind"] == "sample":
        return _sample_inputs(case, g, dt, seed)
    new, total = _lengths(case)
    Hq, Hkv, hd, page, block, B = case["Hq"], case["Hkv"], case["hd"], case["page"], case["block"], case["B"]
    cols = -(-max(total) // page)
    cols = -(-cols // 8) * 8
    used = [-(-t // page) for t in total]
    n_pages = sum(used) + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(used[:b]) for b in range(B)], device="cuda")
    table = ids[(first[:, None] + torch.arange(cols, device="cuda")).clamp(max=n_pages - 1)].contiguous()
    heads = Hq + 2 * Hkv
    out = {"qkv": torch.empty(sum(new), heads * hd, device="cuda").normal_(generator=g).to(dt), "table": table,
           "lens": torch.tensor(total, dtype=torch.int32, device="cuda"), "cu": None, "rotary": None}
    out["k_cache"], out["k_scale"] = _pool(g, n_pages, Hkv, page, hd, block, case["cache"])
    out["v_cache"], out["v_scale"] = _pool(g, n_pages, Hkv, page, hd, block, case["cache"])
    if case["q"] > 1:
        at = [sum(new[:b]) for b in range(B + 1)]
        out["cu"] = torch.tensor(at, dtype=torch.int32, device="cuda")
    if case["kind"] == "write":
        at = [sum(total[:b]) for b in range(B + 1)]
        out["cu_rows"] = torch.tensor(at, dtype=torch.int32, device="cuda")
    if case.get("rot"):
        half = torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda")
        pos = torch.arange(max(total), dtype=torch.float64, device="cuda")
        angle = pos[:, None] * 10000.0 ** (-half / case["rot"])
        out["rotary"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    return out


def _sample_inputs(case, g, dt, seed):
    """Logits as a model gives them: a normal bulk, a few likely tokens on top, of another
    sharpness in every row; masked tokens are -inf.  Settings of the rows around the case's."""
    B, V = case["B"], case["V"]
    x = torch.empty(B, case["ld"], device="cuda").normal_(std=case["spread"], generator=g)
    likely = torch.randint(V, (B, 8), generator=g, device="cuda")
    x.scatter_add_(1, likely, torch.rand(B, 8, generator=g, device="cuda") * torch.rand(B, 1, generator=g, device="cuda") * 16)
    if case["masked"]:
        gone = torch.rand(B, case["ld"], generator=g, device="cuda") < case["masked"]
        gone[torch.arange(B, device="cuda"), likely[:, 0]] = False
        x.masked_fill_(gone, float("-inf"))
    out = {"logits": x.to(dt)[:, :V], "u": torch.rand(B, generator=g, device="cuda")}
    if case["rows"]:
        # Requests differ; some take the most likely token, some cut nothing.
        rng = random.Random(case["order"] + seed)
        t = [rng.choice([0.0, 0.5, 1.0, 1.0]) * case["temperature"] for _ in range(B)]
        k = [rng.choice([0, 1, 2]) * case["top_k"] for _ in range(B)]
        p = [rng.choice([1.0, case["top_p"], case["top_p"]]) for _ in range(B)]
        m = [rng.choice([0.0, case["min_p"], case["min_p"]]) for _ in range(B)]
        out.update(temperature=torch.tensor(t, device="cuda"), top_k=torch.tensor(k, dtype=torch.int32, device="cuda"),
                   top_p=torch.tensor(p, device="cuda"), min_p=torch.tensor(m, device="cuda"))
    return out


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["kind"] != "sample":
        # What a scheduler knows on the host: it made the batch.
        new, total = _lengths(case)
        state.update(max_new=max(new), max_len=max(total), n_keys=sum(total))
    return state


def _heads(state):
    """q, k and v of the step's tokens: views (tokens, heads, hd) into the projection."""
    case, x = state["case"], state["qkv"]
    Hq, Hkv, hd = case["Hq"], case["Hkv"], case["hd"]
    x = x.view(x.shape[0], Hq + 2 * Hkv, hd)
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]


# ------------------------------------------------------------------------------- a pass


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    if case["kind"] == "write":
        return _plain_write(state)
    if case["kind"] == "attend":
        return _plain_attention(state)
    return _plain_sample(state)


def _own(case, state):
    import cutilegpt_amd as cg

    if case["kind"] == "sample":
        if case["rows"]:
            t, k, p, m = state["temperature"], state["top_k"], state["top_p"], state["min_p"]
        else:
            t, k, p, m = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
        return cg.sample_tokens(state["logits"], state["u"], temperature=t, top_k=k, top_p=p, min_p=m)
    q, k, v = _heads(state)
    cache = state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"], state["table"], state["lens"]
    if case["kind"] == "attend":
        return cg.paged_attention_8bit(q, *cache, cu_q=state["cu"])
    out = cg.paged_kv_append_8bit(k, v, *cache, cu_q=state["cu"], q=q if case["rot"] else None,
                                  rotary=state["rotary"], interleaved=case["interleaved"])
    kr, vr = cg.paged_kv_read_8bit(*cache, state["cu_rows"], state["n_keys"], dtype=q.dtype)
    return [kr, vr, state["k_scale"], state["v_scale"]] + ([out] if case["rot"] else [])


def _owners(state):
    """Sequence, place in its step and position of every token."""
    n = state["qkv"].shape[0]
    tok = torch.arange(n, device="cuda")
    cu = state["cu"]
    if cu is None:
        seq, start, count = tok, tok, torch.ones_like(tok)
    else:
        seq = torch.searchsorted(cu[1:], tok, right=True)
        start, count = cu[seq], cu[seq + 1] - cu[seq]
    return seq, tok - start, (state["lens"][seq] - count + tok - start).long()


def _rotate(x, angles, rot, interleaved):
    """The first ``rot`` values of every head turned by the token's angles, in 64 bits: a
    code's rounding border is at stake."""
    x = x.double()
    if not rot:
        return x
    angles = angles.double()
    c, s = angles[:, None, :rot // 2], angles[:, None, rot // 2:]
    head = x[..., :rot]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([head, x[..., rot:]], -1)


def _pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exponent(big, cache):
    """The smallest exponent that leaves values of ``big`` within the codes."""
    c = _CODES[cache]
    m, x = torch.frexp(big)
    e = x - c["exp"] + (m > c["mant"]).int()
    return torch.where(big > 0, e, _LO).clamp(_LO, c["hi"])


def _encode(y, cache):
    """64-bit values, already in units of their block, to codes: half to even, once."""
    if cache == "int8":
        return y.round().clamp(-127, 127).to(torch.int8)
    unit = _pow2((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    y = ((y / unit).round() * unit).clamp(-448, 448)
    return y.float().to(torch.float8_e4m3fn).view(torch.int8)


def _decode(codes, cache, to):
    """int8 storage to the numbers it stands for."""
    return (codes.view(torch.float8_e4m3fn).float() if cache == "e4m3" else codes).to(to)


def _store(case, cache, scale, x, page, slot, first):
    """Rows x (n, Hkv, hd) in 64 bits into slots of pages, in place; ``first``: the
    sequences' first rows, which may go on in a block that holds rows already."""
    P, H, S, hd = cache.shape
    blk, kind = case["block"], case["cache"]
    nb = S // blk
    raw = cache.view(torch.int8)
    at = page * nb + slot // blk
    big = torch.zeros(P * nb, H, dtype=torch.float64, device="cuda")
    big.scatter_reduce_(0, at[:, None].expand(-1, H), x.abs().amax(-1), "amax")
    need = _exponent(big, kind)
    written = torch.zeros(P * nb, dtype=torch.bool, device="cuda")
    written[at] = True
    goes_on = torch.zeros_like(written)
    goes_on[at[first]] = slot[first] % blk > 0
    old = scale.transpose(1, 2).reshape(P * nb, H).int() - 127
    new = torch.where(goes_on[:, None], torch.maximum(need, old), need)
    new = torch.where(written[:, None], new, old)
    # Rows that the step found there, where the exponent grew.
    a = at[first]
    blocks = raw.view(P, H, nb, blk, hd)
    held = blocks[a // nb, :, a % nb]
    shrink = _pow2(torch.where(goes_on[a][:, None], old[a] - new[a], 0))[..., None, None]
    blocks[a // nb, :, a % nb] = _encode(_decode(held, kind, torch.float64) * shrink, kind)
    raw[page, :, slot] = _encode(x * _pow2(-new[at])[..., None], kind)
    scale.copy_((new + 127).to(torch.uint8).view(P, nb, H).transpose(1, 2))


def _plain_write(state):
    case = state["case"]
    q, k, v = _heads(state)
    seq, _, pos = _owners(state)
    page = state["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    rot = case["rot"]
    angles = state["rotary"][pos] if rot else None
    first = torch.arange(case["B"], device="cuda") if state["cu"] is None else state["cu"][:-1].long()
    turned = _rotate(k, angles, rot, case["interleaved"])
    _store(case, state["k_cache"], state["k_scale"], turned, page, slot, first)
    _store(case, state["v_cache"], state["v_scale"], v.double(), page, slot, first)
    # Back, all keys of all sequences.
    cu = state["cu_rows"]
    row = torch.arange(state["n_keys"], device="cuda")
    seq = torch.searchsorted(cu[1:], row, right=True)
    pos = row - cu[seq]
    page = state["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]

    def back(cache, scale):
        x = _decode(cache.view(torch.int8)[page, :, slot], case["cache"], torch.float32)
        e = scale[page, :, slot // case["block"]].int() - 127
        return (x * _pow2(e).float()[..., None]).to(q.dtype)

    out = [back(state["k_cache"], state["k_scale"]), back(state["v_cache"], state["v_scale"]), state["k_scale"],
           state["v_scale"]]
    if rot:
        out.append(_rotate(q, angles, rot, case["interleaved"]).to(q.dtype))
    return out


def _plain_attention(state):
    """Padded to the longest sequence: the keys gathered from their pages, scores, a masked
    softmax, the values."""
    case = state["case"]
    q, _, _ = _heads(state)
    B, Hkv, hd, page = case["B"], case["Hkv"], case["hd"], case["page"]
    G, T, L = case["Hq"] // Hkv, state["max_new"], state["max_len"]
    seq, place, pos = _owners(state)

    # (B, Hkv, T * G, hd) queries and their positions, the places behind a sequence empty.
    dense = torch.zeros(B, T, Hkv * G, hd, dtype=torch.float32, device="cuda")
    dense[seq, place] = q.float() / math.sqrt(hd)
    dense = dense.view(B, T, Hkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, hd)
    at = torch.full((B, T), -1, device="cuda")
    at[seq, place] = pos

    keys = torch.arange(L, device="cuda")
    pages, slots = state["table"][:, keys // page].long(), (keys % page).expand(B, L)

    def rows(cache, scale):
        """(B, Hkv, L, hd) values in 32 bits."""
        x = _decode(cache.view(torch.int8)[pages, :, slots], case["cache"], torch.float32)
        x *= _pow2(scale[pages, :, slots // case["block"]].int() - 127).float()[..., None]
        return x.transpose(1, 2).contiguous()

    scores = dense @ rows(state["k_cache"], state["k_scale"]).transpose(2, 3)
    seen = keys <= at[:, :, None]
    scores = scores.view(B, Hkv, T, G, L).masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    scores -= scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = scores.exp_().view(B, Hkv, T * G, L)
    total = p.sum(-1, keepdim=True)
    o = p @ rows(state["v_cache"], state["v_scale"])
    o = o / total.clamp(min=torch.finfo(torch.float32).tiny)
    o = o.view(B, Hkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(B, T, Hkv * G, hd)
    return o[seq, place].to(q.dtype)


def _plain_sample(state):
    """Weights in the order of the logits, the cuts as masks of that order, the draw by the
    running sum in the order of the vocabulary; 64-bit weights, since a sum meets a border."""
    case, x, u = state["case"], state["logits"], state["u"]
    B, V = x.shape
    if case["rows"]:
        t, k, p, m = (state[n][:, None] for n in ("temperature", "top_k", "top_p", "min_p"))
    else:
        t, k, p, m = (torch.tensor([[case[n]]], dtype=torch.float64, device="cuda")
                      for n in ("temperature", "top_k", "top_p", "min_p"))
    srt, order = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = t <= 0
    z = (srt.double() - srt[:, :1].double()) / torch.where(greedy, 1.0, t.double())
    w = z.exp()
    rank = torch.arange(V, device="cuda")
    w = w * (rank < torch.where(greedy, 1, torch.where(k > 0, k, V)))
    cum = w.cumsum(-1)
    w = w * ((cum - w < p.double() * cum[:, -1:]) | (rank == 0)) * (w >= m.double())
    kept = torch.zeros_like(w).scatter_(1, order, w)
    cum = kept.cumsum(-1)
    return (cum <= u.double()[:, None] * cum[:, -1:]).sum(-1)


# -------------------------------------------------------------------------------- exact


def _powers():
    """2^(e - 127) of every byte e."""
    return torch.tensor([math.ldexp(1.0, e - 127) for e in range(256)], dtype=torch.float64, device="cuda")


def _e4m3_numbers():
    """The 127 numbers that an e4m3 code without its sign stands for, in the codes' order."""
    return [m / 512 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if e * 8 + m < 127]


def _nearest(y, numbers):
    """y's size and sign on the grid of ``numbers``; halves go to the even place."""
    mids = (numbers[1:] + numbers[:-1]) / 2
    a = y.abs().contiguous()
    lo, hi = torch.searchsorted(mids, a), torch.searchsorted(mids, a, right=True)
    at = torch.where(lo == hi, lo, torch.where(lo % 2 == 0, lo, hi))
    return numbers[at] * y.sign()


def _exact_write(case, inp):
    new, total = _lengths(case)
    page, blk, hd, c = case["page"], case["block"], case["hd"], _CODES[case["cache"]]
    if sum(m // blk + 2 for m in new) > 3000 or _dense_bytes(case) > 1.0e10:
        return None
    q, k, v = (t.double() for t in _heads({"case": case, **inp}))
    rot, h, n = case["rot"], case["rot"] // 2, 0
    numbers = torch.tensor(_e4m3_numbers() if case["cache"] == "e4m3" else list(range(128)), dtype=torch.float64, device="cuda")
    out = {"k": [], "v": []}
    for b in range(case["B"]):
        rows = slice(n, n + new[b])
        n += new[b]
        start = total[b] - new[b]
        if rot:
            # A pair (x, y) turned by w is (x + iy) e^(iw).
            w = inp["rotary"][start:total[b]].double()
            w = torch.complex(w[:, :h], w[:, h:])[:, None]
            for x in (k, q):
                i, j = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, h), slice(h, rot))
                z = torch.complex(x[rows][..., i], x[rows][..., j]) * w
                x[rows, :, i], x[rows, :, j] = z.real, z.imag
        pages = inp["table"][b, :-(-total[b] // page)].long()
        for name, x in (("k", k), ("v", v)):
            codes = inp[name + "_cache"][pages].double().transpose(0, 1).flatten(1, 2)  # (Hkv, slots, hd)
            power = _powers()[inp[name + "_scale"][pages].long()].transpose(0, 1).flatten(1, 2)  # (Hkv, blocks)
            for j in range(start // blk, (total[b] - 1) // blk + 1):
                a, e = max(start, j * blk), min(total[b], (j + 1) * blk)
                new_rows = x[rows][a - start:e - start].transpose(0, 1)
                e2 = torch.ceil(torch.log2(new_rows.abs().amax((1, 2)) / c["top"])).clamp(_LO, c["hi"])
                s = _powers()[e2.long() + 127]
                if a > j * blk:
                    s = torch.maximum(s, power[:, j])
                    there = slice(j * blk, a)
                    codes[:, there] = _nearest(codes[:, there] * (power[:, j] / s)[:, None, None], numbers)
                power[:, j] = s
                codes[:, a:e] = _nearest(new_rows / s[:, None, None], numbers)
            full = codes * power.repeat_interleave(blk, 1)[..., None]
            out[name].append(full[:, :total[b]].transpose(0, 1))
    return [torch.cat(out["k"]), torch.cat(out["v"]), None, None] + ([q] if rot else [])


def _exact_attention(case, inp):
    new, total = _lengths(case)
    page, blk, hd, Hkv = case["page"], case["block"], case["hd"], case["Hkv"]
    q = _heads({"case": case, **inp})[0].double()
    out, n = torch.zeros_like(q), 0
    for b in range(case["B"]):
        pages = inp["table"][b, :-(-total[b] // page)].long()
        kv = []
        for name in ("k", "v"):
            x = inp[name + "_cache"][pages].float().double().view(-1, Hkv, page // blk, blk, hd)
            x = x * _powers()[inp[name + "_scale"][pages].long()][..., None, None]
            kv.append(x.transpose(0, 1).reshape(Hkv, -1, hd)[:, :total[b]])
        m = new[b]
        ban = torch.ones(m, total[b], dtype=torch.bool, device="cuda").triu_(total[b] - m + 1)
        keys = (kv[0] / math.sqrt(hd)).transpose(1, 2).contiguous()[:, None]
        # A few hundred queries at a time: the scores of long chunks in 64 bits are large.
        for i in range(0, m, 512):
            qi = q[n + i:n + min(i + 512, m)]
            t = qi.shape[0]
            qi = qi.view(t, Hkv, -1, hd).permute(1, 2, 0, 3)
            p = torch.softmax((qi @ keys).masked_fill_(ban[i:i + t], float("-inf")), -1)
            out[n + i:n + i + t] = (p @ kv[1][:, None]).permute(2, 0, 1, 3).reshape(t, -1, hd)
        n += m
    return out


@torch.no_grad()
def exact(case, seed):
    if case["kind"] == "sample":
        return None  # tokens are whole numbers
    inp = _inputs(case, seed)
    return _exact_write(case, inp) if case["kind"] == "write" else _exact_attention(case, inp)
