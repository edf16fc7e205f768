"""Performance cases of serving from a paged key-value cache.

A case is a dict of plain values.  ``listed()`` names twelve of them, ``draw(rng)``
gives more of the same ranges, ``prepare`` makes what a serving program holds before
the call (projections of the step's tokens, page pools, block tables, lengths),
``run`` is one pass through one operator, ``work`` what a pass cannot do without,
``exact`` the same result in float64.

The kinds of case:

    append   paged_kv_append: the step's keys and values into their pages, keys and
             queries rotated on the way where the model has rotary positions
    paged    paged_attention: the step's queries against each sequence's pages
    shared   shared_prefix_attention: the same for a batch whose sequences begin with
             the same pages, which are read once for all

With ``own`` false ``run`` computes a plain form in elementary torch operations in
32 bits, rounded once at the end.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # The cache side of one decode step: a batch of 32, the heads of the largest
        # GPT-2, no rotary positions.  A few hundred kilobytes: launch latency counts.
        dict(name="append_step", kind="append", dtype="bfloat16", B=32, q=1, lo=100, hi=900, Hq=25,
             Hkv=25, hd=64, page=16, rot=0, interleaved=False, order=1),
        # Sixteen ragged prompts entering the cache at once, fully rotated heads.
        dict(name="append_prompts", kind="append", dtype="bfloat16", B=16, q=2048, lo=0, hi=0, Hq=12,
             Hkv=12, hd=64, page=64, rot=64, interleaved=False, order=2),
        # Chunks of prompts in fp32 on odd pages, grouped heads rotated in part, pairs
        # side by side.
        dict(name="append_chunk_fp32", kind="append", dtype="float32", B=5, q=300, lo=0, hi=2000, Hq=8,
             Hkv=2, hd=128, page=24, rot=32, interleaved=True, order=3),
        # One sequence at a prompt, half a context behind it: latency.
        dict(name="paged_single", kind="paged", dtype="bfloat16", B=1, q=1, lo=500, hi=500, Hq=12,
             Hkv=12, hd=64, page=16, order=4),
        # A full decode batch of very different lengths.
        dict(name="paged_ragged", kind="paged", dtype="bfloat16", B=64, q=1, lo=1, hi=8192, Hq=25,
             Hkv=25, hd=64, page=64, order=5),
        # Few sequences with very long contexts, four query heads to a key head.
        dict(name="paged_long", kind="paged", dtype="float16", B=4, q=1, lo=90000, hi=130000, Hq=32,
             Hkv=8, hd=128, page=128, order=6),
        # Guessed tokens of seven short sequences checked at once, fp32, odd pages.
        dict(name="paged_verify_fp32", kind="paged", dtype="float32", B=7, q=5, lo=30, hi=700, Hq=6,
             Hkv=3, hd=32, page=10, order=7),
        # Prompts taken in chunks: long queries, each behind the context it already has.
        dict(name="paged_chunks", kind="paged", dtype="bfloat16", B=16, q=2048, lo=0, hi=4096, Hq=16,
             Hkv=16, hd=64, page=32, order=8),
        # Four short answers to one short prompt in the default dtype.
        dict(name="shared_small_fp32", kind="shared", dtype="float32", B=4, q=1, lo=0, hi=40, prefix=512,
             Hq=12, Hkv=12, hd=64, page=16, order=9),
        # Sixty-four samples drawn from one prompt.
        dict(name="shared_samples", kind="shared", dtype="bfloat16", B=64, q=1, lo=0, hi=512, prefix=4096,
             Hq=25, Hkv=25, hd=64, page=32, order=10),
        # Many users behind one long document, grouped heads.
        dict(name="shared_document", kind="shared", dtype="float16", B=128, q=1, lo=0, hi=1024,
             prefix=32768, Hq=32, Hkv=8, hd=128, page=64, order=11),
        # Candidate answers scored against one prompt: every sequence brings its tokens.
        dict(name="shared_scoring", kind="shared", dtype="bfloat16", B=24, q=64, lo=0, hi=0, prefix=2048,
             Hq=12, Hkv=12, hd=64, page=64, order=12),
    ]


# ------------------------------------------------------------------------- drawn cases


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = [work(c) for c in listed()]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    kind = rng.choice(["append", "paged", "paged", "shared", "shared"])
    while True:
        case = _draw_kind(rng, kind)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and _dense_bytes(case) <= 2.0e10:
            return case


def _draw_kind(rng, kind):
    group = rng.choice([1, 1, 2, 3, 4, 8])
    kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 20, 25])
    case = dict(kind=kind, dtype=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]), Hkv=kv,
                Hq=kv * group, hd=rng.choice([16, 32, 64, 64, 128]),
                page=rng.choice([1, 8, 10, 16, 24, 32, 64, 100, 128, 256]), order=rng.randrange(1 << 30))
    if kind == "append":
        rot = rng.choice([0, case["hd"], case["hd"], case["hd"] // 2])
        hi = _log_int(rng, 1, 4096)
        case.update(B=_log_int(rng, 1, 128), q=rng.choice([1, _log_int(rng, 1, 2048)]), lo=rng.randint(0, hi),
                    hi=hi, rot=rot, interleaved=rng.choice([False, True]))
        return case
    # Single tokens, a few guessed ones, or chunks of prompts.
    case["q"] = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
    case["B"] = _log_int(rng, 1, 128)
    if kind == "paged":
        hi = _log_int(rng, 1, 130000)
        case.update(lo=rng.randint(0, hi), hi=hi)
    else:
        hi = _log_int(rng, 1, 2048)
        prefix = -(-_log_int(rng, 16, 65536) // case["page"]) * case["page"]
        case.update(lo=rng.randint(0, hi), hi=hi, prefix=prefix)
    return case


# --------------------------------------------------------------------- lengths and work


def _lengths(case):
    """(tokens of this step, keys with them) of every sequence.  A sequence brings 1 to
    ``q`` tokens behind a context of ``lo`` to ``hi`` (and the shared prefix)."""
    rng = random.Random(case["order"])
    new = [rng.randint(max(1, case["q"] // 8), case["q"]) for _ in range(case["B"])]
    return new, [n + rng.randint(case["lo"], case["hi"]) + case.get("prefix", 0) for n in new]


def _dense_bytes(case):
    """What the plain form, or 64 bits, take on the way, roughly: whole pools, or padded
    keys, values and scores."""
    new, total = _lengths(case)
    if case["kind"] == "append":
        slots = sum(total) + case["B"] * case["page"]
        return 16 * (sum(new) * (case["Hq"] + 2 * case["Hkv"]) + 2 * slots * case["Hkv"]) * case["hd"]
    own_keys = max(total) - case.get("prefix", 0)
    cells = case["B"] * case["Hkv"] * own_keys * case["hd"]
    return 4 * (3 * cells + 3 * case["B"] * case["Hq"] * max(new) * max(total))


def work(case):
    """Tokens, cached keys and values and tables read once, results written once; the
    shared prefix once for all.  Only the pairs that the causal order leaves count."""
    e = 4 if case["dtype"] == "float32" else 2
    new, total = _lengths(case)
    Hq, Hkv, hd = case["Hq"], case["Hkv"], case["hd"]
    n = sum(new)
    if case["kind"] == "append":
        rot = case["rot"]
        q = Hq if rot else 0
        moved = 2 * n * (2 * Hkv + q) * hd * e + n * rot * 4 + 4 * (n + 2 * case["B"])
        return {"bytes": moved, "flops": max(1, 3 * n * (Hkv + q) * rot)}
    prefix = case.get("prefix", 0)
    keys = prefix + sum(t - prefix for t in total)
    pairs = sum(m * t - m * (m - 1) // 2 for m, t in zip(new, total))
    table = 4 * (keys // case["page"] + 2 * case["B"])
    return {"bytes": 2 * keys * Hkv * hd * e + 2 * n * Hq * hd * e + table, "flops": 4 * pairs * Hq * hd}


# ------------------------------------------------------------------------------- inputs


def _inputs(case, seed):
    """The step's fused projection, the pools (every slot holds something: a pool is used
    again and again), the tables and the lengths."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    new, total = _lengths(case)
    Hq, Hkv, hd, page, B = case["Hq"], case["Hkv"], case["hd"], case["page"], case["B"]
    shared = case.get("prefix", 0) // page
    cols = -(-(max(total)) // page)
    cols = -(-cols // 8) * 8
    used = [-(-t // page) - shared for t in total]
    n_pages = shared + sum(used) + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([shared + sum(used[:b]) for b in range(B)], device="cuda")
    col = torch.arange(cols, device="cuda")
    slot = torch.where(col < shared, col, first[:, None] + col - shared)
    table = ids[slot.clamp(max=n_pages - 1)].contiguous()

    def normal(*shape):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(dt)

    out = {"qkv": normal(sum(new), (Hq + 2 * Hkv) * hd), "k_cache": normal(n_pages, Hkv, page, hd),
           "v_cache": normal(n_pages, Hkv, page, hd), "table": table,
           "lens": torch.tensor(total, dtype=torch.int32, device="cuda"), "cu": None, "rotary": None}
    if case["q"] > 1:
        at = [sum(new[:b]) for b in range(B + 1)]
        out["cu"] = torch.tensor(at, dtype=torch.int32, device="cuda")
    if case.get("rot"):
        half = torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda")
        pos = torch.arange(max(total), dtype=torch.float64, device="cuda")
        angle = pos[:, None] * 10000.0 ** (-half / case["rot"])
        out["rotary"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    return out


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    new, total = _lengths(case)
    # What a scheduler knows on the host: it made the batch.
    state["max_new"], state["max_len"] = max(new), max(total)
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
    q, k, v = _heads(state)
    if not own:
        if case["kind"] == "append":
            return _plain_append(state, q, k, v)
        return _plain_attention(state, q)
    import cutilegpt_amd as cg

    if case["kind"] == "append":
        out = cg.paged_kv_append(k, v, state["k_cache"], state["v_cache"], state["table"], state["lens"],
                                 cu_q=state["cu"], q=q if case["rot"] else None, rotary=state["rotary"],
                                 interleaved=case["interleaved"])
        return [state["k_cache"], state["v_cache"]] + ([out] if case["rot"] else [])
    if case["kind"] == "paged":
        return cg.paged_attention(q, state["k_cache"], state["v_cache"], state["table"], state["lens"],
                                  cu_q=state["cu"])
    return cg.shared_prefix_attention(q, state["k_cache"], state["v_cache"], state["table"], state["lens"],
                                      case["prefix"], cu_q=state["cu"])


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
    return seq, tok - start, state["lens"][seq] - count + tok - start


def _rotate(x, angles, rot, interleaved):
    """The first ``rot`` values of every head turned by the token's angles, in 32 bits."""
    x = x.float()
    if not rot:
        return x
    c, s = angles[:, None, :rot // 2], angles[:, None, rot // 2:]
    head = x[..., :rot]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([head, x[..., rot:]], -1)


def _plain_append(state, q, k, v):
    case = state["case"]
    seq, _, pos = _owners(state)
    page = state["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    rot = case["rot"]
    angles = state["rotary"][pos] if rot else None
    turned = _rotate(k, angles, rot, case["interleaved"]).to(k.dtype)
    state["k_cache"][page, :, slot] = turned
    state["v_cache"][page, :, slot] = v
    out = [state["k_cache"], state["v_cache"]]
    if rot:
        out.append(_rotate(q, angles, rot, case["interleaved"]).to(q.dtype))
    return out


def _plain_attention(state, q):
    """Padded to the longest sequence: the keys gathered from their pages, scores, a masked
    softmax, the values.  A shared prefix is gathered once and multiplied by all queries."""
    case = state["case"]
    B, Hkv, hd, page = case["B"], case["Hkv"], case["hd"], case["page"]
    G, T, L = case["Hq"] // Hkv, state["max_new"], state["max_len"]
    prefix = case.get("prefix", 0)
    seq, place, pos = _owners(state)

    # (B, Hkv, T * G, hd) queries and their positions, the places behind a sequence empty.
    dense = torch.zeros(B, T, Hkv * G, hd, dtype=torch.float32, device="cuda")
    dense[seq, place] = q.float() / math.sqrt(hd)
    dense = dense.view(B, T, Hkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, hd)
    at = torch.full((B, T), -1, device="cuda")
    at[seq, place] = pos.long()

    def rows(cache, table, keys):
        """(.., Hkv, keys, hd) of the positions ``keys`` of every table row, in 32 bits."""
        x = cache[table[..., keys // page].long(), :, keys % page].float()
        return x.transpose(-3, -2).contiguous()

    later = torch.arange(prefix, L, device="cuda")
    scores = dense @ rows(state["k_cache"], state["table"], later).transpose(2, 3)
    if prefix:
        early = torch.arange(prefix, device="cuda")
        flat = dense.transpose(0, 1).reshape(Hkv, B * T * G, hd)
        s = flat @ rows(state["k_cache"], state["table"][0], early).transpose(1, 2)
        s = s.view(Hkv, B, T * G, prefix).transpose(0, 1)
        scores = torch.cat([s, scores], -1)
    keys = torch.arange(L, device="cuda")
    seen = keys <= at[:, :, None]
    scores = scores.view(B, Hkv, T, G, L).masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    scores -= scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = scores.exp_().view(B, Hkv, T * G, L)
    total = p.sum(-1, keepdim=True)
    o = p[..., prefix:] @ rows(state["v_cache"], state["table"], later)
    if prefix:
        flat = p[..., :prefix].transpose(0, 1).reshape(Hkv, B * T * G, prefix)
        e = flat @ rows(state["v_cache"], state["table"][0], early)
        o = o + e.view(Hkv, B, T * G, hd).transpose(0, 1)
    o = o / total.clamp(min=torch.finfo(torch.float32).tiny)
    o = o.view(B, Hkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(B, T, Hkv * G, hd)
    return o[seq, place].to(q.dtype)


# -------------------------------------------------------------------------------- exact


@torch.no_grad()
def exact(case, seed):
    inp = _inputs(case, seed)
    new, total = _lengths(case)
    page, hd, Hkv = case["page"], case["hd"], case["Hkv"]
    q, k, v = (t.double() for t in _heads({"case": case, **inp}))
    if case["kind"] == "append":
        rot, h = case["rot"], case["rot"] // 2
        kc, vc, qo, n = inp["k_cache"].double(), inp["v_cache"].double(), q.clone(), 0
        for b in range(case["B"]):
            for_b = slice(n, n + new[b])
            pos = torch.arange(total[b] - new[b], total[b], device="cuda")
            where = inp["table"][b].long()[pos.div(page, rounding_mode="floor")], slice(None), pos.remainder(page)
            kb, qb = k[for_b].clone(), q[for_b].clone()
            if rot:
                # A pair (x, y) turned by w is (x + iy) e^(iw).
                w = inp["rotary"][pos].double()
                w = torch.complex(w[:, :h], w[:, h:])[:, None]
                for x in (kb, qb):
                    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, h), slice(h, rot))
                    z = torch.complex(x[..., i], x[..., j]) * w
                    x[..., i], x[..., j] = z.real, z.imag
            kc[where], vc[where], qo[for_b] = kb, v[for_b], qb
            n += new[b]
        return [kc, vc] + ([qo] if rot else [])
    out, n = torch.zeros_like(q), 0
    for b in range(case["B"]):
        pages = inp["table"][b, :-(-total[b] // page)].long()
        kb, vb = (inp[c][pages].transpose(0, 1).reshape(Hkv, -1, hd)[:, :total[b]].double() for c in ("k_cache", "v_cache"))
        m = new[b]
        ban = torch.ones(m, total[b], dtype=torch.bool, device="cuda").triu_(total[b] - m + 1)
        # A few hundred queries at a time: the scores of long chunks in 64 bits are large.
        for i in range(0, m, 512):
            qi = q[n + i:n + min(i + 512, m)]
            t = qi.shape[0]
            qi = qi.view(t, Hkv, -1, hd).permute(1, 2, 0, 3)
            s = qi @ (kb / math.sqrt(hd)).transpose(1, 2).contiguous()[:, None]
            p = torch.softmax(s.masked_fill_(ban[i:i + t], float("-inf")), -1)
            out[n + i:n + i + t] = (p @ vb[:, None]).permute(2, 0, 1, 3).reshape(t, -1, hd)
        n += m
    return out
