"""Plain float64 / sequential forms of the paged KV cache and of the beam search step — TEST
INFRASTRUCTURE ONLY, as the rest of this package: each is the definition in include/kandle_hip.h written
out row by row."""
from __future__ import annotations

import numpy as np


def _sequences(tokens, kv_lens, starts):
    """(sequence, first token, new tokens, cached rows) of each sequence."""
    for b, length in enumerate(kv_lens):
        t0, t1 = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        yield b, int(t0), int(t1) - int(t0), max(0, int(length))


def paged_attention(q, k_pages, v_pages, table, kv_lens, starts=None, scale=None, causal=True, out=None):
    """(o, a, smax): the attention in float64, sum p |v| (what errors of p are multiplied by) and the largest
    scale * sum |q| |k| (what errors of the scores are relative to) of each row.  Rows behind the last
    sequence are those of `out`."""
    q, kp, vp = (np.asarray(x, np.float64) for x in (q, k_pages, v_pages))
    tokens, hq, d = q.shape
    pages, hkv, page, _ = kp.shape
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    o = np.full(q.shape, np.nan) if out is None else np.array(out, np.float64)
    a, smax = np.zeros(q.shape), np.zeros(q.shape[:2])
    for b, t0, n, length in _sequences(tokens, kv_lens, starts):
        rows = np.arange(min(length, table.shape[1] * page))
        ids = table[b, rows // page]
        rows = rows[(ids >= 0) & (ids < pages)]
        ids = table[b, rows // page]
        k, v = kp[ids, :, rows % page], vp[ids, :, rows % page]
        see = rows[None] <= (length - n + np.arange(n))[:, None] if causal else np.ones((n, len(rows)), bool)
        none = ~see.any(1)
        for h in range(hq):
            hk, mine = h // (hq // hkv), q[t0:t0 + n, h]
            p = np.where(see, scale * (mine @ k[:, hk].T), -np.inf)
            p = np.exp(p - np.where(none, 0, p.max(1, initial=-np.inf))[:, None])
            p /= np.where(none, 1, p.sum(1))[:, None]
            o[t0:t0 + n, h] = p @ v[:, hk]
            a[t0:t0 + n, h] = p @ np.abs(v[:, hk])
            smax[t0:t0 + n, h] = abs(scale) * np.where(see, np.abs(mine) @ np.abs(k[:, hk]).T, 0).max(1, initial=0)
    return o, a, smax


def attention_bound(dtype, o, a, smax, d, rows):
    """Elementwise error of paged_attention in `dtype`, by counting roundings (u: half a step).

    Scores: d products summed in fp32, each partial sum within smax: (d + 8) u smax, the 8 for the scaling,
    the subtraction of the maximum and the exponent's argument (log2 units, |s - m| <= 2 smax); p and the
    normaliser both carry it, so twice; exp2 itself and the quotient 8 u.  P V: up to `rows` fp32 additions
    on |p v| <= a, and as many rescalings: 2 (rows + 8) u a.  bfloat16: p rounded once (2^-8 a, and as much
    through the normaliser), the result rounded once."""
    u = 2.0 ** -24
    e = (2 * (d + 8) * u * smax[..., None] + 16 * u + 2 * (rows + 8) * u) * a + u * np.abs(o)
    if dtype == "bfloat16":
        e = e + 2 * 2.0 ** -8 * a + 2.0 ** -8 * (np.abs(o) + e)
    return e + 1e-37


def paged_kv_write(k, v, k_pages, v_pages, table, kv_lens, starts=None, info=None):
    kp, vp = np.array(k_pages), np.array(v_pages)
    if info is not None and (info[1] or info[2]):
        return kp, vp
    pages, _, page, _ = kp.shape
    for b, t0, n, length in _sequences(len(k), kv_lens, starts):
        for j in range(n):
            at = length - n + j
            if 0 <= at < table.shape[1] * page and 0 <= table[b, at // page] < pages:
                kp[table[b, at // page], :, at % page] = k[t0 + j]
                vp[table[b, at // page], :, at % page] = v[t0 + j]
    return kp, vp


def count_refs(table, pages):
    ids = table[(table >= 0) & (table < pages)]
    return np.bincount(ids, minlength=pages).astype(np.int64)


def pages_fork(table, lens, refs, parents):
    new, new_lens, new_refs = np.full_like(table, -1), np.zeros_like(lens), np.array(refs)
    for row in table:
        for p in row[(row >= 0) & (row < len(refs))]:
            new_refs[p] -= 1
    for s, parent in enumerate(parents):
        if 0 <= parent < len(table):
            new[s], new_lens[s] = table[parent], lens[parent]
            for p in table[parent][(table[parent] >= 0) & (table[parent] < len(refs))]:
                new_refs[p] += 1
    return new, new_lens, new_refs


def pages_reserve(table, lens, refs, counts, page):
    """(table, lens, refs, moves, info), one row after the other."""
    t, n, r = np.array(table), np.array(lens), np.array(refs)
    moves, missing, too_long = [], 0, 0
    free = lambda: np.flatnonzero(r <= 0)  # noqa: E731
    for s, grow in enumerate(counts):
        length = max(0, int(n[s]))
        if grow <= 0:
            continue
        if length + grow > t.shape[1] * page:
            too_long += 1
            continue
        for at in range(length // page, -(-(length + int(grow)) // page)):
            inside = at * page < length
            held = inside and 0 <= t[s, at] < len(r)
            if held and r[t[s, at]] <= 1:
                continue
            f = free()
            if len(f) == 0:
                missing += 1
                if held:
                    r[t[s, at]] -= 1
                continue
            if held:
                moves.append((t[s, at], f[0]))
                r[t[s, at]] -= 1
            t[s, at], r[f[0]] = f[0], 1
        n[s] = length + grow
    out = np.full((len(lens), 2), -1, np.int64)
    if missing or too_long:
        return np.array(table), np.array(lens), np.array(refs), out, np.array([0, missing, too_long])
    if moves:
        out[:len(moves)] = moves
    return t, n, r, out, np.array([len(moves), 0, 0])


def pages_compact(table, refs, room):
    t, r = np.array(table), np.array(refs)
    live = np.flatnonzero(r > 0)
    src = live[live >= len(live)]
    dst = [p for p in range(len(live)) if r[p] <= 0]
    moves = np.full((room, 2), -1, np.int64)
    for i, (a, b) in enumerate(zip(src, dst)):
        t[table == a] = b
        r[b], r[a] = r[a], 0
        moves[i] = a, b
    return t, r, moves, np.array([len(src), len(live)])


def pages_copy(pages, moves, count):
    out = np.array(pages)
    for a, b in moves[:count]:
        if 0 <= a < pages.shape[-4] and 0 <= b < pages.shape[-4]:
            out[..., b, :, :, :] = pages[..., a, :, :, :]
    return out


def beam_select(logits, scores, k, finished=None, eos=None):
    """(scores float64, tokens, parents, finished) of each group, best first: the larger score in float64, then the
    lower beam, then (at a finite score) the larger logit, then the lower token."""
    logits = np.asarray(logits, np.float64)
    groups, beams, vocab = logits.shape
    out = [np.zeros((groups, k)), np.zeros((groups, k), np.int64), np.zeros((groups, k), np.int64), np.zeros((groups, k), np.int64)]
    for g in range(groups):
        every = np.full((beams, vocab), -np.inf)
        possible, logit = np.ones((beams, vocab), bool), np.zeros((beams, vocab))
        for b in range(beams):
            base = float(scores[g, b])
            base = -np.inf if np.isnan(base) else base
            if finished is not None and finished[g, b]:
                possible[b] = False
                possible[b, eos], every[b, eos] = True, base
                continue
            x = np.where(np.isnan(logits[g, b]), -np.inf, logits[g, b])
            m = x.max()
            if not np.isfinite(m) or not np.isfinite(base):
                continue
            every[b], logit[b] = x + (base - (m + np.log(np.exp(x - m).sum()))), x
        beam, token = np.divmod(np.arange(beams * vocab), vocab)
        order = np.lexsort((token, -logit.reshape(-1), beam, -every.reshape(-1), ~possible.reshape(-1)))
        for j, i in enumerate(order[:k]):
            out[0][g, j], out[1][g, j], out[2][g, j] = every.reshape(-1)[i], i % vocab, i // vocab
            if finished is not None:
                out[3][g, j] = int(bool(finished[g, i // vocab]) or i % vocab == eos)
    return out[0], out[1], out[2], (out[3] if finished is not None else None)


def attention_spread(q, k_pages, v_pages, table, kv_lens, starts=None, scale=None, causal=True):
    """(sum p^2 v^2, sum p^2) of each row of paged_attention: what independent roundings of p add up to, squared."""
    q, kp, vp = (np.asarray(x, np.float64) for x in (q, k_pages, v_pages))
    pages, hkv, page, d = kp.shape
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    pv, pp = np.zeros(q.shape), np.zeros(q.shape[:2])
    for b, t0, n, length in _sequences(len(q), kv_lens, starts):
        for j in range(n):
            rows = np.arange(max(0, min(length - n + j + 1 if causal else length, table.shape[1] * page)))
            rows = rows[(table[b, rows // page] >= 0) & (table[b, rows // page] < pages)]
            if not len(rows):
                continue
            k, v = (np.repeat(x[table[b, rows // page], :, rows % page], q.shape[1] // hkv, 1) for x in (kp, vp))
            s = scale * np.einsum("hd,khd->kh", q[t0 + j], k)
            p = np.exp(s - s.max(0))
            p /= p.sum(0)
            pv[t0 + j], pp[t0 + j] = np.einsum("kh,khd->hd", p * p, v * v), (p * p).sum(0)
    return pv, pp
