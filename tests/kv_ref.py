"""The 4-bit KV cache's operators in 64 bits, from their definitions, and the
tolerances of the kernels against them.

Rounding steps are half an ulp: 2^-11 relative in FP16, 2^-24 in FP32.
"""
from __future__ import annotations

import numpy as np
import torch

H16 = 2.0 ** -11


def decode(units, page_table, page_size, b, n):
    """One sequence's codes and parameters: dict of float64 arrays kc, vc [heads, n, D], ks, kz, vs, vz [heads, n]."""
    u = units.cpu().numpy()
    table = page_table.cpu().numpy()
    heads, ub = u.shape[1], u.shape[3]
    d = (ub - 128) // 16
    kc, vc = np.zeros((heads, n, d)), np.zeros((heads, n, d))
    par = np.zeros((heads, n, 4))
    cols = np.arange(d)
    for j in range(n):
        unit = u[table[b, j // page_size], :, j % page_size // 16]  # [heads, ub]
        r = j % 16
        kb = unit[:, r * d // 2:(r + 1) * d // 2]
        kc[:, j] = (kb[:, cols // 2] >> (4 * (cols % 2))) & 15
        words = unit[:, 8 * d + (r // 2) * d:8 * d + (r // 2 + 1) * d]
        vb = words[:, (cols // 4) * 4 + 2 * (r % 2) + (cols % 4) // 2]
        vc[:, j] = (vb >> (4 * (cols % 2))) & 15
        par[:, j] = np.ascontiguousarray(unit[:, 16 * d + 8 * r:16 * d + 8 * r + 8]).view(np.float16)
    return {"kc": kc, "vc": vc, "ks": par[..., 0], "kz": par[..., 1], "vs": par[..., 2], "vz": par[..., 3]}


def attend(q, line, n, scale, count=None):
    """q [T, q_heads, D] (float16 tensor) of one sequence with n slots; `count` of the T queries are real.
    -> dict: out, tol [T, q_heads, D], lse, lse_tol [T, q_heads], mass [heads, n], mass_rel (float64)."""
    q = q.double().cpu().numpy()
    t, hq, d = q.shape
    heads = line["kc"].shape[0]
    g = hq // heads
    count = t if count is None else count
    k = line["ks"][..., None] * (line["kc"] - line["kz"][..., None])
    v = line["vs"][..., None] * (line["vc"] - line["vz"][..., None])
    out, tol = np.zeros((t, hq, d)), np.full((t, hq, d), 2.0 ** -25)
    lse, lse_tol = np.full((t, hq), -np.inf), np.zeros((t, hq))
    mass, mass_err = np.zeros((heads, n)), np.zeros((heads, n))
    for i in range(count):
        seen = min(max(n - count + i + 1, 0), n)
        if seen == 0:
            continue
        for a in range(hq):
            e = a // g
            s = scale * k[e, :seen] @ q[i, a]
            m = s.max()
            w = np.exp(s - m)
            p = w / w.sum()
            out[i, a] = p @ v[e, :seen]
            lse[i, a] = m + np.log(w.sum())
            mass[e, :seen] += p
            # Scores: the products q c are exact; D/16 MMAs and the steps inside each add up FP32 sums
            # (truncated at worst: a full ulp, 2^-23, of at most `terms`), then three FP32 operations.  A weight's
            # relative error is twice the score's (the score and the sum's) plus the exponential's 2^-22 and the
            # subtraction of the maximum from a score of size |s|.
            terms = abs(scale) * line["ks"][e, :seen] * (np.abs(q[i, a]) @ line["kc"][e, :seen].T
                                                         + np.abs(line["kz"][e, :seen]) * np.abs(q[i, a]).sum())
            rel = 2 * (24 * 2.0 ** -23 * terms.max() + 2.0 ** -22 + 2.0 ** -22 * np.abs(s).max()) + 2.0 ** -20
            # Output: p' = p s w is rounded to FP16 once (2^-11 of p s |c - 8| or, in units counted from 15, of
            # p s |c - 7|; below 2^-14 half of 2^-24, with 1 / w <= 2^-6 max s), the sums are FP32 (one truncation
            # per unit), the result is rounded to FP16.  Within an MMA the 16 terms and the sum are cut off 2^-23 below
            # the largest, where a code's subnormal c 2^-24 counts as 2^-14: 17 times 2^-13 of the unit's largest p s.
            sv = line["vs"][e, :seen]
            s8 = (p * sv) @ (np.abs(line["vc"][e, :seen] - 7.5) + 0.5)
            cut = 17 * 2.0 ** -13 * np.pad(p * sv, (0, -seen % 16)).reshape(-1, 16).max(1).sum()
            sz = (p * sv) @ np.abs(line["vz"][e, :seen] - 8)
            sums = (seen / 16 + 64) * 2.0 ** -23
            tol[i, a] = (H16 * (np.abs(out[i, a]) + s8) + 2.0 ** -25 + rel * (p @ np.abs(v[e, :seen]) + s8 + sz)
                         + sums * (s8 + sz) + 8 * seen * sv.max() * 2.0 ** -31 + cut)
            lse_tol[i, a] = rel + 2.0 ** -22 * abs(lse[i, a])
            mass_err[e, :seen] += rel * p
    return {"out": out, "tol": tol, "lse": lse, "lse_tol": lse_tol, "mass": mass, "mass_tol": mass_err}


def check_attend(got, lse, q, cache, scale, counts=None, mass=None, mass0=None):
    """Compare attend()'s outputs of every sequence; mass, mass0: `cache.mass` after and before, per page."""
    lens = cache.lengths.tolist()
    t = q.shape[1]
    for b, n in enumerate(lens):
        c = t if counts is None else counts[b]
        line = decode(cache.units, cache.page_table, cache.page_size, b, n)
        r = attend(q[b], line, n, scale, c)
        err = np.abs(got[b].double().cpu().numpy() - r["out"])
        assert np.isfinite(got[b].float().cpu().numpy()).all(), f"sequence {b}: not finite"
        bad = np.argwhere(err > r["tol"])
        assert len(bad) == 0, (f"sequence {b} (len {n}): {len(bad)} of {err.size} outputs off, first {bad[0]}: "
                               f"{got[b].cpu()[tuple(bad[0])]} for {r['out'][tuple(bad[0])]}, tol {r['tol'][tuple(bad[0])]:.3g}")
        if lse is not None:
            l = lse[b].double().cpu().numpy()
            assert np.array_equal(np.isinf(l), np.isinf(r["lse"])), f"sequence {b}: empty rows"
            f = np.isfinite(r["lse"])
            assert (np.abs(l[f] - r["lse"][f]) <= r["lse_tol"][f]).all(), f"sequence {b}: lse"
        if mass is not None:
            table, size = cache.page_table.cpu().numpy(), cache.page_size
            j = np.arange(n)
            a, z = (x.double().cpu().numpy()[table[b, j // size], :, j % size].T for x in (mass, mass0))
            tol = r["mass_tol"] + 2.0 ** -23 * (z + r["mass"]) + 1e-30
            assert (np.abs(a - z - r["mass"]) <= tol).all(), f"sequence {b}: mass"


def evict(lens, evicted, mass, pos, page_table, page_size, keep, recent, sink):
    """-> per sequence and head: list of (to, from) moves; the new lengths and evicted counts."""
    moves = {}
    table = page_table.cpu().numpy()
    mass, pos = mass.cpu().numpy(), pos.cpu().numpy()
    new_len, new_ev = list(lens), list(evicted)
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        new_len[b], new_ev[b] = keep, evicted[b] + n - keep
        for h in range(mass.shape[1]):
            w = [(float(mass[table[b, j // page_size], h, j % page_size]), int(pos[table[b, j // page_size], h, j % page_size]))
                 for j in range(n)]
            order = sorted(range(n), key=lambda j: (not (w[j][1] >= n + evicted[b] - recent or w[j][1] < sink), -w[j][0], j))
            kept = set(order[:keep])
            to = [j for j in range(keep) if j not in kept]
            src = [j for j in range(keep, n) if j in kept]
            assert len(to) == len(src)
            moves[(b, h)] = list(zip(to, src))
    return moves, new_len, new_ev


def make_cache(lens, heads, dim, page, seed=0, spare=0, mass=False, extra=0, big_pages=None):
    """An Int4KVCache with sequences of these lengths, pages in shuffled order, everything behind them 0xFF."""
    from dyn_quant.kv_cache import Int4KVCache

    gen = torch.Generator().manual_seed(seed)
    need = [max(1, -(-(n + extra) // page)) for n in lens]
    n_pages = sum(need) + spare if big_pages is None else big_pages
    cache = Int4KVCache(len(lens), n_pages, heads, dim, page, max_pages=max(need) + 1)
    cache.units.fill_(255)
    order = torch.randperm(n_pages, generator=gen).tolist() if big_pages is None else \
        [n_pages - 1 - i for i in range(sum(need))]
    at = 0
    for b, m in enumerate(need):
        cache.assign(b, order[at:at + m])
        at += m
    t = max(lens)
    if t:
        k = torch.randn(len(lens), t, heads, dim, generator=gen)
        k[..., ::17] *= 4
        v = torch.randn(len(lens), t, heads, dim, generator=gen) + 0.1
        cache.append(k.half().cuda(), v.half().cuda(), counts=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if mass:
        cache.mass.copy_(torch.rand(cache.mass.shape, generator=gen))
    return cache


def queries(cache, t, group, seed=1, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(cache.n_seqs, t, cache.n_kv_heads * group, cache.head_dim, generator=gen) * scale
    return q.half().cuda()
