"""Rotary positions, compaction and page selection from their definitions, in numpy
float64 (test infrastructure only).  No counterpart in the reference."""

from __future__ import annotations

import numpy as np

from oracle.attention import decode_one, gather_seq


def turn(x, positions, inv_freq, *, offset=0, interleaved=False, scale=1.0, inverse=False):
    """x (N, H, D) float64 with its rotary pairs turned: as complex numbers times
    scale * exp(+-i p f)."""
    x = np.array(x, np.float64)
    m = len(inv_freq)
    i = np.arange(m)
    first, second = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + m + i)
    # whole turns taken off exactly enough for positions up to 2^40
    a = np.asarray(positions, np.longdouble)[:, None] * np.asarray(inv_freq, np.longdouble)[None, :]
    two_pi = 2 * np.longdouble("3.14159265358979323846264338327950288")
    a = (a - np.rint(a / two_pi) * two_pi).astype(np.float64)
    z = (x[..., first] + 1j * x[..., second]) * (scale * np.exp((-1j if inverse else 1j) * a))[:, None, :]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def turn_tolerance(x, inv_freq, eps, *, offset=0, interleaved=False, scale=1.0):
    """Per element: half a step of the output type, and the 32-bit error of a turned pair.
    cos and sin: the fraction of a turn rounded to 32 bits (2^-25 of a turn: 2 pi 2^-25 =
    3.2 2^-24 of the value's range 1), sincospi's 2 units (2^-23), the product with the
    scale (2^-24): below 7 2^-24; two products, rounded, and their sum below 3 2^-24 of
    |x1| + |x2|.  10 2^-24 (|x1| + |x2|) scale, and eps / 2 of what that gives."""
    x = np.abs(np.array(x, np.float64))
    m = len(inv_freq)
    i = np.arange(m)
    first, second = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + m + i)
    tol = np.zeros(x.shape)
    both = (x[..., first] + x[..., second]) * scale * 10 * 2.0 ** -24
    tol[..., first] = tol[..., second] = both
    return lambda want: tol * (1 + eps) + eps / 2 * np.abs(want) + 2.0 ** -150


def compact(o, seq_ids, keep, *, into_new=False, turn_keys=None):
    """Compaction of ``o`` (``OraclePagedKV``) to kept positions.  ``keep[i]``: (n,) or
    (layers, n).  ``turn_keys(k rows, shift)`` turns copied keys.  In place, or into
    new sequences, whose ids are returned."""
    bs, L = o.block_size, o.num_layers
    plans = []
    for sid, ks in zip(seq_ids, keep):
        s = o._sequences[sid]
        for layer in range(L):
            k = np.asarray(ks if np.ndim(ks) == 1 else ks[layer], np.int64)
            stay = 0
            while stay < len(k) and k[stay] == stay:
                stay += 1
            pages = -(-len(k) // bs)
            lead = pages if stay == len(k) == s.num_tokens[layer] else stay // bs
            old = list(s.page_table[layer])
            new = old[:lead] + [o.allocator.alloc() for _ in range(pages - lead)]
            for j in range(lead * bs, len(k)):
                src, dst = (old[k[j] // bs], k[j] % bs), (new[j // bs], j % bs)
                row = o.k_pools[layer][src]
                if turn_keys is not None and k[j] != j:
                    row = turn_keys(row[None], np.array([j - k[j]]))[0]
                o.k_pools[layer][dst] = row
                o.v_pools[layer][dst] = o.v_pools[layer][src]
            plans.append((sid, layer, lead, old, new, len(k)))
    out = []
    if into_new:
        out = [o.allocate_sequence() for _ in seq_ids]
    names = dict(zip(range(len(seq_ids)), out))
    for n, (sid, layer, lead, old, new, m) in enumerate(plans):
        i = n // L
        s = o._sequences[names[i] if into_new else sid]
        if into_new:
            for b in new[:lead]:
                o.allocator.ref(b)
        else:
            for b in old[lead:]:
                o.allocator.release(b)
        s.page_table[layer] = new
        s.num_tokens[layer] = m
        s.tokens_in_last_block[layer] = m - (len(new) - 1) * bs if m else 0
    return out


def unit_exponent(top):
    """The least e in -50 .. 50 with top <= 127 * 2^e."""
    return next((e for e in range(-50, 50) if top <= 127.0 * 2.0 ** e), 50)


def index_page(k):
    """k (rows, Hkv, D) float64: bounds (Hkv, 2, D) and exponents (Hkv,) of the page index."""
    hkv, d = k.shape[1:]
    bounds, exps = np.zeros((hkv, 2, d), np.int8), np.zeros(hkv, np.int8)
    for h in range(hkv):
        if not np.isfinite(k[:, h]).all():
            exps[h] = 127
            continue
        exps[h] = e = unit_exponent(np.abs(k[:, h]).max())
        bounds[h, 0] = np.clip(np.floor(k[:, h].min(0) / 2.0 ** e), -127, 127)
        bounds[h, 1] = np.clip(np.ceil(k[:, h].max(0) / 2.0 ** e), -127, 127)
    return bounds, exps


def choose_pages(q, bounds, exps, pages, budget, sink, recent):
    """The pages one KV head attends to: q (G, D) float64, bounds (pages, 2, D), exps (pages,)."""
    best = np.full(pages, -np.inf)
    for row in q:
        row = np.where(np.isfinite(row), row, 0.0)
        e = unit_exponent(np.abs(row).max())
        grid = np.clip(np.rint(row / 2.0 ** e), -127, 127) * 2.0 ** e
        products = np.maximum(grid * bounds[:, 0], grid * bounds[:, 1]).sum(1)
        best = np.maximum(best, products * 2.0 ** np.where(exps == 127, 0, exps).astype(float))
    p = np.arange(pages)
    scores = np.where((p < sink) | (p >= pages - recent), np.inf, np.where(exps == 127, 1e300, best))
    order = sorted(range(pages), key=lambda p: (-scores[p], p))
    return sorted(order[:budget])


def sparse_decode(q, k_pool, v_pool, tables, lens, bs, bounds, exps, budget, sink, recent, scale=None):
    """q (N, Hq, D) float64 and one layer's pools and index -> out float64, chosen pages."""
    n, hq, d = q.shape
    hkv = k_pool.shape[2]
    g = hq // hkv
    out, chosen = np.zeros(q.shape), np.full((n, hkv, budget), -1, np.int64)
    for i, (tab, length) in enumerate(zip(tables, lens)):
        pages = -(-length // bs)
        tab = np.asarray(tab[:pages], np.int64)
        k, v = gather_seq(k_pool, tab, length, bs), gather_seq(v_pool, tab, length, bs)
        for h in range(hkv):
            got = choose_pages(q[i, h * g:(h + 1) * g], bounds[tab, h], exps[tab, h], pages, budget, sink, recent)
            chosen[i, h, :len(got)] = got
            at = np.concatenate([np.arange(p * bs, min(length, (p + 1) * bs)) for p in got]) if got else np.zeros(0, int)
            out[i, h * g:(h + 1) * g] = decode_one(q[i, h * g:(h + 1) * g], k[at][:, h:h + 1], v[at][:, h:h + 1], scale)
    return out, chosen
