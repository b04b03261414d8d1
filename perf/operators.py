"""The 4-bit KV cache of a decode step, as cases to be measured: append (quantize
new keys and values into the paged cache), attend (attention of the newest
tokens over it, with or without the running attention weight per slot) and
evict (drop the slots with the least weight).

A case is a dict of plain values.  ``own = False`` computes the operators with
elementary torch operations in 32 bits; ``own = True`` calls dyn_quant.kv_cache.

Cache layout (head_dim D, one unit = 16 tokens of one KV head, D = 128: 2176 bytes):
  units  uint8 [n_pages, kv_heads, page_size / 16, 16 D + 128]
         K: 16 rows of D/2 bytes, column 2j in the low nibble of byte j
         V: 8 token pairs x D/4 quads of columns x (even token, odd token) x 2 bytes
         16 x (K scale, K zero, V scale, V zero) float16
  mass   float32, pos int32 [n_pages, kv_heads, page_size]: accumulated weight, position
  lengths, evicted int32 [seqs]; page_table int32 [seqs, max_pages], -1 where there is no page
``meta`` is one buffer: mass, pos, lengths, evicted one after another.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TOKENS = 16  # tokens of one unit


def _unit(dim):
    """Bytes of one unit."""
    return 16 * dim + 128


def _kv():
    """The framework's operators (imported only where own is true)."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dyn-quant_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from dyn_quant import kv_cache

    return kv_cache


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _append(name, seqs, heads, tokens, lo, hi, dim=128, page=64, ragged=False, values=False):
    return {"name": name, "op": "append", "seqs": seqs, "heads": heads, "tokens": tokens, "min_len": lo,
            "max_len": hi, "dim": dim, "page": page, "ragged": ragged, "values": values}


def _attend(name, seqs, heads, group, lo, hi, tokens=1, dim=128, page=64, ragged=False, mass=False, lse=False):
    return {"name": name, "op": "attend", "seqs": seqs, "heads": heads, "group": group, "tokens": tokens,
            "min_len": lo, "max_len": hi, "dim": dim, "page": page, "ragged": ragged, "mass": mass, "lse": lse}


def _evict(name, seqs, heads, lo, hi, keep, recent, sink, dim=128, page=64):
    return {"name": name, "op": "evict", "seqs": seqs, "heads": heads, "min_len": lo, "max_len": hi, "keep": keep,
            "recent": recent, "sink": sink, "dim": dim, "page": page}


def listed():
    return [
        # one decode step of 16 sequences, 8 KV heads (the 70B layer): launch latency
        _append("append_step", 16, 8, 1, 500, 3500),
        # prompts of up to 2048 tokens, 32 KV heads (the 7B layer), the values as the cache holds them returned
        _append("append_prompts", 4, 32, 2048, 0, 700, ragged=True, values=True),
        # a short chat's step on the 7B layer: the smallest call
        _attend("attend_short", 1, 32, 1, 77, 77),
        # a served batch on the 70B layer, 8 query heads per KV head
        _attend("attend_batch_gqa", 16, 8, 8, 1000, 4100),
        # one long document: the work of 8 KV heads split over its length
        _attend("attend_long", 1, 8, 8, 131071, 131071),
        # a large served batch on the 7B layer: the largest cache
        _attend("attend_batch_mha", 64, 32, 1, 2000, 4096),
        # the step that also accumulates each slot's weight, for eviction
        _attend("attend_mass_gqa", 16, 8, 8, 2000, 4100, mass=True),
        _attend("attend_mass_mha", 8, 32, 1, 500, 2100, mass=True),
        # verifying up to 5 drafted tokens per sequence, heads of 64 columns, small pages
        _attend("attend_draft_d64", 8, 8, 4, 200, 8000, tokens=5, dim=64, page=16, ragged=True, lse=True),
        # a prompt's chunk of 64 tokens over what is cached already
        _attend("attend_chunk", 2, 8, 8, 6000, 8000, tokens=64, mass=True),
        # one slot too many in every head (a step at the cache's bound)
        _evict("evict_step", 16, 8, 2049, 2049, 2048, 256, 4),
        # long prompts cut to a budget, uneven lengths, some below it
        _evict("evict_prompts", 4, 8, 9000, 32768, 16384, 512, 4),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "evict"])
    dim, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128])
    heads = rng.choice([1, 2, 4, 8, 8, 32])
    seqs = _spread(rng, 1, 64)
    room = 64 * 32 * 2900 // (seqs * heads)  # tokens per sequence that keep the cache below the largest listed one
    if op == "append":
        tokens = _spread(rng, 1, max(1, min(2048, 4 * 32 * 1300 // (seqs * heads))))
        lo = rng.randrange(0, 300)
        return {k: v for k, v in _append("", seqs, heads, tokens, lo, lo + _spread(rng, 1, 2000), dim, page,
                                         rng.random() < 0.5, rng.random() < 0.5).items() if k != "name"}
    hi = _spread(rng, 16, max(16, min(131071, room)))
    lo = max(1, int(hi * rng.choice([0.1, 0.5, 1.0])))
    if op == "evict":
        hi = min(hi, 32768)
        lo = min(lo, hi)
        keep = max(1, int(hi * rng.uniform(0.3, 1.0)))
        sink = min(rng.randrange(0, 5), keep)
        return {k: v for k, v in _evict("", seqs, heads, lo, hi, keep, rng.randrange(0, (keep - sink) // 2 + 1), sink,
                                        dim, page).items() if k != "name"}
    group = rng.choice([1, 1, 2, 3, 4, 8])
    tokens = rng.choice([1, 1, 1, 2, 3, 5, _spread(rng, 1, 64)])
    while tokens > 1 and tokens * group * seqs * heads * hi > 512 * 8 * 2 * 7000:
        tokens //= 2
    return {k: v for k, v in _attend("", seqs, heads, group, lo, hi, tokens, dim, page, rng.random() < 0.4,
                                     rng.random() < 0.3, rng.random() < 0.3).items() if k != "name"}


def _lengths(case):
    """Tokens in the cache per sequence: a fixed spread of [min_len, max_len], the longest first."""
    n, lo, hi = case["seqs"], case["min_len"], case["max_len"]
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _counts(case):
    """New tokens (append) or query tokens (attend) per sequence."""
    n, t = case["seqs"], case["tokens"]
    if not case["ragged"]:
        return [t] * n
    return [t - int(t * ((i * 0.7548776662) % 1.0)) for i in range(n)]


def work(case):
    d, h = case["dim"], case["heads"]
    row = d + 8  # codes and scales of one token and KV head
    lens = _lengths(case)
    if case["op"] == "append":
        n = sum(_counts(case)) * h
        return {"bytes": n * (4 * d + row + 8 + (4 * d if case["values"] else 0)), "flops": n * 2 * 4 * d}
    if case["op"] == "attend":
        cnt, g = _counts(case), case["group"]
        keys = sum(lens)
        rows = sum(cnt) * g * h
        pairs = sum(g * h * sum(max(0, n - c + t + 1) for t in range(c)) for n, c in zip(lens, cnt))
        return {"bytes": keys * h * (row + (8 if case["mass"] else 0)) + rows * 4 * d, "flops": 4 * d * pairs}
    moved = sum(max(0, n - case["keep"]) * case["keep"] / n for n in lens) * h
    return {"bytes": sum(lens) * h * 8 + 2 * moved * (row + 8), "flops": sum(lens) * h}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _quantize(v):
    """[..., D] float16 -> codes uint8, scale and zero float16 (dyn_quant.quantize's arithmetic, one group per row)."""
    x = v.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = hi - lo
    step = torch.where(span < 1e-8, torch.ones_like(span), span / torch.full_like(span, 15.0))
    inv = torch.ones_like(step) / step
    codes = ((x - lo) * inv + 0.5).trunc().clamp(0, 15).to(torch.uint8)
    return codes, step.half(), (-lo * inv).half()


def _parts(units, dim):
    """Views of a unit tensor [..., 16 D + 128]: K bytes [..., 16, D/2], V bytes [..., 8, D/4, 2, 2], params [..., 16, 4] float16."""
    head = units.shape[:-1]
    k = units[..., : 8 * dim].unflatten(-1, (TOKENS, dim // 2))
    v = units[..., 8 * dim : 16 * dim].unflatten(-1, (TOKENS // 2, dim // 4, 2, 2))
    p = units.view(torch.float16)[..., 8 * dim :].unflatten(-1, (TOKENS, 4))
    assert k.shape[:-2] == head
    return k, v, p


def _pack(codes):
    """uint8 codes [..., D] -> bytes [..., D/2], column 2j in the low nibble of byte j."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _rows(n, heads, dim, gen, kind, dev):
    """n rows of keys or values [n, heads, dim] float16: keys with a few strong columns, as projections give them."""
    x = torch.randn(n, heads, dim, generator=gen, device=dev)
    if kind == "k":
        cols = torch.rand(heads, dim, generator=gen, device=dev)
        x = x * torch.where(cols < 0.03, 4.0, 1.0)
    return x.half()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s, h, d, page = case["seqs"], case["heads"], case["dim"], case["page"]
    lens = _lengths(case)
    extra = case["tokens"] if case["op"] == "append" else 0
    need = [max(1, -(-(n + extra) // page)) for n in lens]
    max_pages, n_pages = max(need), sum(need) + 2
    per = page // TOKENS
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((s, max_pages), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    table = table.to(dev)
    # pages hold whatever their last owner left, here 0xFF (scales and zeros that are not numbers)
    units = torch.full((n_pages, h, per, _unit(d)), 255, dtype=torch.uint8, device=dev)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    slots = n_pages * h * page
    meta = torch.zeros(2 * slots + 2 * s, dtype=torch.int32, device=dev)
    mass = meta[:slots].view(torch.float32).view(n_pages, h, page)
    pos = meta[slots:2 * slots].view(n_pages, h, page)
    meta[2 * slots:2 * slots + s] = lengths
    if case["op"] != "append":
        for b, n in enumerate(lens):
            if n == 0:
                continue
            pages = table[b, : -(-n // page)].long()
            m = len(pages) * page
            k, v = (_rows(m, h, d, gen, kind, dev) for kind in "kv")
            kc, ks, kz = _quantize(k)
            vc, vs, vz = _quantize(v)
            u = torch.empty(len(pages), h, per, _unit(d), dtype=torch.uint8, device=dev)
            uk, uv, up = _parts(u, d)

            def shaped(x):  # [m, h, c] -> [pages, h, per, 16, c]
                return x.view(len(pages), per, TOKENS, h, -1).permute(0, 3, 1, 2, 4)

            uk.copy_(shaped(_pack(kc)))
            uv.copy_(shaped(_pack(vc)).unflatten(-1, (d // 4, 2)).unflatten(3, (8, 2)).permute(0, 1, 2, 3, 5, 4, 6))
            par = torch.cat([ks, kz, vs, vz], dim=-1)
            par[n:] = float("nan")  # slots behind the last token
            up.copy_(shaped(par))
            units[pages] = u
            pos[pages] = torch.arange(m, dtype=torch.int32, device=dev).view(len(pages), 1, page)
            # a few slots hold most of the weight; the newest hold little, equal weights among them
            w = torch.exp(2.0 * torch.randn(len(pages), h, page, generator=gen, device=dev))
            w = torch.where(torch.rand(w.shape, generator=gen, device=dev) < 0.02, 0.25, w)
            mass[pages] = w / n
    state = {"case": case, "units": units, "meta": meta, "mass": mass, "pos": pos, "table": table,
             "lengths": meta[2 * slots:2 * slots + s], "evicted": meta[2 * slots + s:], "keep": meta.clone()}
    if case["op"] == "append":
        t = case["tokens"]
        state["k"] = _rows(s * t, h, d, gen, "k", dev).view(s, t, h, d)
        state["v"] = _rows(s * t, h, d, gen, "v", dev).view(s, t, h, d)
        state["at"] = lengths
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=dev)
    elif case["op"] == "attend":
        # the queries are a slice of the projections' output, as a layer hands them over
        g, t = case["group"], case["tokens"]
        qkv = torch.randn(s, t, h * g + 2 * h, d, generator=gen, device=dev).half()
        state["q"] = qkv[:, :, : h * g]
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=dev)
    if own:
        state["cache"] = _kv().Int4KVCache(s, n_pages, h, d, page_size=page, max_pages=max_pages, device=dev,
                                           units=units, meta=meta, page_table=table)
    return state


# ---------------------------------------------------------------------------
# The operators in their plain form
# ---------------------------------------------------------------------------
def _slots(state, n):
    """Page and offset of the first n slots of every sequence: [seqs, n] each (page 0 where there is none)."""
    page = state["case"]["page"]
    j = torch.arange(n, device=state["table"].device)
    last = state["table"].shape[1] - 1
    return state["table"][:, (j // page).clamp(max=last)].long().clamp(min=0), (j % page).expand(len(state["table"]), n)


def _plain_append(state):
    case = state["case"]
    s, t, h, d = state["k"].shape
    at, cnt = state["at"].long(), state["counts"].long()
    i = torch.arange(t, device=at.device)
    b = (i[None, :] < cnt[:, None]).nonzero()
    seq, tok = b[:, 0], b[:, 1]
    slot = at[seq] + tok
    pages, off = state["table"][seq, slot // case["page"]].long(), slot % case["page"]
    k, v = state["k"][seq, tok], state["v"][seq, tok]  # [n, h, d]
    kc, ks, kz = _quantize(k)
    vc, vs, vz = _quantize(v)
    uk, uv, up = _parts(state["units"], d)
    unit, row = off // TOKENS, off % TOKENS
    hh = torch.arange(h, device=at.device)
    uk[pages[:, None], hh, unit[:, None], row[:, None]] = _pack(kc)
    uv[pages[:, None], hh, unit[:, None], row[:, None] // 2, :, row[:, None] % 2] = _pack(vc).unflatten(-1, (d // 4, 2))
    up[pages[:, None], hh, unit[:, None], row[:, None]] = torch.cat([ks, kz, vs, vz], dim=-1)
    state["mass"][pages[:, None], hh, off[:, None]] = 0.0
    state["pos"][pages[:, None], hh, off[:, None]] = (state["evicted"][seq].long() + slot).int()[:, None].expand(-1, h)
    state["lengths"].copy_(at + cnt)
    out = [state["units"], state["meta"][state["mass"].numel():], state["mass"]]
    if case["values"]:
        for c, sc, z in ((kc, ks, kz), (vc, vs, vz)):
            full = torch.zeros(s, t, h, d, dtype=torch.float16, device=at.device)
            full[seq, tok] = (sc.float() * (c.float() - z.float())).half()
            out.append(full)
    return out


def _plain_attend(state):
    case = state["case"]
    s, t, hq, d = state["q"].shape
    h, page = case["heads"], case["page"]
    g = hq // h
    lens, cnt = state["lengths"].long(), state["counts"].long()
    n = state["table"].shape[1] * page
    u = state["units"][state["table"].long().clamp(min=0)].transpose(1, 2).reshape(s, h, n // TOKENS, _unit(d))
    uk, uv, up = _parts(u, d)
    p = up.reshape(s, h, n, 4).float()
    there = torch.arange(n, device=lens.device) < lens[:, None]
    kb = uk.reshape(s, h, n, d // 2)
    vb = uv.permute(0, 1, 2, 3, 5, 4, 6).reshape(s, h, n, d // 2)
    keys = torch.stack([kb & 15, kb >> 4], dim=-1).flatten(-2).float()
    keys = p[..., 0:1] * (keys - p[..., 1:2])
    q = state["q"].float().reshape(s, t, h, g, d).transpose(1, 2).reshape(s, h, t * g, d)
    score = torch.matmul(q, keys.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    del keys
    i = torch.arange(t, device=lens.device)
    limit = torch.where(i < cnt[:, None], lens[:, None] - cnt[:, None] + i + 1, 0)  # [s, t] keys that query i sees
    seen = torch.arange(n, device=lens.device) < limit[:, :, None]
    score = score.view(s, h, t, g, n).masked_fill(~seen[:, None, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top.isinf(), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    lse = (torch.log(total) + top).squeeze(-1)
    weight = torch.where(total > 0, weight / total, 0.0)
    del score
    values = torch.stack([vb & 15, vb >> 4], dim=-1).flatten(-2).float()
    values = torch.where(there[:, None, :, None], p[..., 2:3] * (values - p[..., 3:4]), 0.0)
    o = torch.matmul(weight.view(s, h, t * g, n), values)
    out = [o.view(s, h, t, g, d).transpose(1, 2).reshape(s, t, hq, d).half()]
    if case["mass"]:
        pages, off = _slots(state, n)
        b, j = there.nonzero(as_tuple=True)
        hh = torch.arange(h, device=lens.device)
        state["mass"][pages[b, j][:, None], hh, off[b, j][:, None]] += weight.sum((2, 3))[b, :, j]
        out.append(state["mass"])
    if case["lse"]:
        out.append(lse.transpose(1, 2).reshape(s, t, hq))
    return out


def _plain_evict(state):
    case = state["case"]
    h, d, keep = case["heads"], case["dim"], case["keep"]
    lens = state["lengths"].long()
    s, n = len(lens), state["table"].shape[1] * case["page"]
    pages, off = _slots(state, n)
    hh = torch.arange(h, device=lens.device)[None, :, None]
    at = (pages[:, None], hh, off[:, None])
    w, pos = state["mass"][at], state["pos"][at].long()  # [s, h, n]
    there = (torch.arange(n, device=lens.device) < lens[:, None])[:, None]
    newest = (lens + state["evicted"].long())[:, None, None]
    safe = there & ((pos >= newest - case["recent"]) | (pos < case["sink"]))
    w = torch.where(safe, float("inf"), torch.where(there, w, float("-inf")))
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, torch.arange(n, device=lens.device).expand_as(order))
    stays = there & (rank < keep)
    low = torch.arange(n, device=lens.device) < keep
    full = (lens > keep)[:, None, None]
    b, hd, to = (full & low & ~stays).nonzero(as_tuple=True)
    b2, _, src = (full & ~low & stays).nonzero(as_tuple=True)
    unit_to, unit_src = (off[b, to] // TOKENS, off[b, to] % TOKENS), (off[b2, src] // TOKENS, off[b2, src] % TOKENS)
    p_to, p_src = pages[b, to], pages[b2, src]
    uk, uv, up = _parts(state["units"], d)
    for part in (uk, up):
        part[p_to, hd, unit_to[0], unit_to[1]] = part[p_src, hd, unit_src[0], unit_src[1]]
    uv[p_to, hd, unit_to[0], unit_to[1] // 2, :, unit_to[1] % 2] = uv[p_src, hd, unit_src[0], unit_src[1] // 2, :,
                                                                     unit_src[1] % 2]
    for part in (state["mass"], state["pos"]):
        part[p_to, hd, off[b, to]] = part[p_src, hd, off[b2, src]]
    left = lens.clamp(max=keep)
    state["evicted"] += (lens - left).int()
    state["lengths"].copy_(left)
    return [state["units"], state["meta"][state["mass"].numel():], state["mass"]]


def run(state):
    case, op = state["case"], state["case"]["op"]
    if op == "evict":
        state["meta"].copy_(state["keep"])  # the cache as it was before the last pass
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[op](state)
    cache = state["cache"]
    if op == "attend":
        got = cache.attend(state["q"], counts=state["counts"] if case["ragged"] else None, accumulate=case["mass"],
                           return_lse=case["lse"])
        out = [got[0] if case["lse"] else got]
        if case["mass"]:
            out.append(cache.mass)
        return out + [got[1]] if case["lse"] else out
    values = None
    if op == "append":
        values = cache.append(state["k"], state["v"], counts=state["counts"] if case["ragged"] else None,
                              at=state["at"], values=case["values"])
    else:
        cache.evict(case["keep"], recent=case["recent"], sink=case["sink"])
    out = [cache.units, cache.meta[cache.mass.numel():], cache.mass]
    return out + list(values) if values is not None else out


# ---------------------------------------------------------------------------
# The same from the definition, in 64 bits
# ---------------------------------------------------------------------------
def _line64(units, pages, head, dim, n):
    """Keys and values of the first n tokens of one sequence and head, float64 [n, dim]: every byte taken apart by itself."""
    raw = units[pages, head].reshape(-1, _unit(dim))  # [units, bytes]
    par = raw[:, 16 * dim:].contiguous().view(torch.float16).double().view(-1, TOKENS, 4).reshape(-1, 4)[:n]
    c = torch.arange(dim, device=raw.device)
    j = torch.arange(n, device=raw.device)
    shift = 4 * (c % 2)
    kb = raw[(j // TOKENS)[:, None], (j % TOKENS)[:, None] * (dim // 2) + c // 2]
    vb = raw[(j // TOKENS)[:, None], 8 * dim + (j % TOKENS // 2)[:, None] * dim + (c // 4) * 4 + (j % 2)[:, None] * 2
             + (c % 4) // 2]
    k = ((kb.long() >> shift) % 16).double()
    v = ((vb.long() >> shift) % 16).double()
    return par[:, :1] * (k - par[:, 1:2]), par[:, 2:3] * (v - par[:, 3:4])


def _exact_attend(case, state):
    s, t, hq, d = state["q"].shape
    h, page = case["heads"], case["page"]
    g = hq // h
    out = torch.zeros(s, t, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((s, t, hq), float("-inf"), dtype=torch.float64, device="cuda")
    mass = state["mass"].double()
    for b, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        pages = state["table"][b, : -(-n // page)].long()
        for e in range(h):
            k, v = _line64(state["units"], pages, e, d, n)
            q = state["q"][b, :c, e * g:(e + 1) * g].double().transpose(0, 1)  # [g, c, d]
            l = torch.matmul(q, k.T) / math.sqrt(d)
            cut = torch.arange(n, device="cuda") > (n - c + torch.arange(c, device="cuda"))[:, None]
            l = l.masked_fill(cut, float("-inf"))
            z = torch.logsumexp(l, -1)
            p = torch.exp(l - torch.where(z.isinf(), 0.0, z)[..., None])
            out[b, :c, e * g:(e + 1) * g] = torch.matmul(p, v).transpose(0, 1)
            lse[b, :c, e * g:(e + 1) * g] = z.T
            line = mass[pages, e].reshape(-1)
            line[:n] += p.sum((0, 1))
            mass[pages, e] = line.view(-1, page)
    return [out] + ([mass] if case["mass"] else []) + ([lse] if case["lse"] else [])


def _exact_append(case, state):
    if not case["values"]:
        return None
    got = [None, None, None]
    for x in (state["k"], state["v"]):
        y = x.double().cpu().numpy()
        lo, hi = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
        span = hi - lo
        step = np.where(span < 1e-8, 1.0, span / 15.0)
        code = np.clip(np.floor((y - lo) / step + 0.5), 0, 15)
        val = step.astype(np.float16).astype(np.float64) * (code - (-lo / step).astype(np.float16).astype(np.float64))
        for b, c in enumerate(_counts(case)):
            val[b, c:] = 0.0
        got.append(torch.from_numpy(val))
    return got


def _exact_evict(case, state):
    mass, pos = state["mass"].double().cpu().numpy(), state["pos"].cpu().numpy()
    table, page, keep = state["table"].cpu().numpy(), case["page"], case["keep"]
    out = mass.copy()
    for b, n in enumerate(_lengths(case)):
        if n <= keep:
            continue
        j = np.arange(n)
        pg = table[b, j // page]
        for e in range(case["heads"]):
            w, p = mass[pg, e, j % page], pos[pg, e, j % page]
            w = np.where((p >= n - case["recent"]) | (p < case["sink"]), np.inf, w)
            first = np.lexsort((j, -w))[:keep]
            stays = np.zeros(n, bool)
            stays[first] = True
            to, src = np.flatnonzero(~stays[:keep]), keep + np.flatnonzero(stays[keep:])
            out[pg[to], e, to % page] = mass[pg[src], e, src % page]
    return [None, None, torch.from_numpy(out)]


def exact(case, seed):
    if case["op"] == "append" and case["values"] and sum(_counts(case)) * case["heads"] * case["dim"] > 60_000_000:
        return None
    state = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](case, state)
