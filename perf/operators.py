"""The paged cache's newer operators as measured workloads: what a step writes into the cache (rotary
positions), what keeps its pages (fork, free, compaction to kept tokens) and what reads it (attention over
pages that a cheap score selects).

``run`` is one pass through one operator: with ``own`` false in elementary torch operations, with ``own``
true through the package's entry points.  A case's ``kind`` names the operator.
"""

import math
import random

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 16
HEAD, TAIL, PEAK, ALLOCS, WORDS = 0, 1, 2, 5, 16  # the block allocator's control words


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------
def _rotary(name, tokens, heads, kv_heads, head_dim, dtype, *, rotary_dim=None, offset=0, interleaved=False, base=1e6,
            factor=1.0, max_position=4096, append=True, together=False):
    return {"kind": "rotary", "name": name, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "rotary_dim": rotary_dim or head_dim, "offset": offset,
            "interleaved": interleaved, "base": base, "factor": factor, "max_position": max_position,
            "append": append, "together": together}


def _fork(name, layers, parents, children, trees, prefix, suffix):
    return {"kind": "fork", "name": name, "layers": layers, "parents": parents, "children": children,
            "trees": trees, "prefix": prefix, "suffix": suffix}


def _compact(name, layers, seqs, tokens, kept, kv_heads, head_dim, dtype, *, scattered, rotary, per_layer=False):
    return {"kind": "compact", "name": name, "layers": layers, "seqs": seqs, "tokens": tokens, "kept": kept,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "scattered": scattered, "rotary": rotary,
            "per_layer": per_layer}


def _index(name, blocks, kv_heads, head_dim, dtype):
    return {"kind": "index", "name": name, "blocks": blocks, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype}


def _sparse(name, seqs, prefix, suffix, heads, kv_heads, head_dim, dtype, budget, *, sink=1, recent=2):
    return {"kind": "sparse", "name": name, "seqs": seqs, "prefix": prefix, "suffix": suffix, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "budget": budget, "sink": sink,
            "recent": recent}


def listed():
    return [
        # one decode step of a tree of 8 leaves (28-layer model, 16 query and 8 KV heads): latency
        _rotary("rotary step, 8 leaves", 8, 16, 8, 128, "bf16", max_position=512),
        # an odd number of tokens, interleaved pairs in the middle part of an odd head, fp32, no cache
        _rotary("rotary part of the head f32", 1537, 10, 2, 80, "f32", rotary_dim=48, offset=16, interleaved=True,
                base=1e4, max_position=1 << 20, append=False),
        # a long prompt's chunk into the cache, frequencies stretched for long contexts (64 query heads)
        _rotary("rotary prefill 8192", 8192, 64, 8, 128, "bf16", factor=8.0, max_position=131072, together=True),
        # one tree's branch at a step: 2 leaves, 3 children each, 256-token prompt, every layer
        _fork("fork+free 2x3, 28 layers", 28, 2, 3, 1, 256, 200),
        # 64 trees with 2048-token prompts branch at once
        _fork("fork+free 64x3, 32 layers", 32, 64, 3, 64, 2048, 500),
        # window with sinks of a tree's 8 leaves, keys moved to their new positions
        _compact("compact 8 windows", 4, 8, 700, 300, 8, 128, "bf16", scattered=False, rotary=True),
        # long sequences reduced to scattered tokens, another choice for each layer
        _compact("compact 12 long, scattered", 2, 12, 16001, 7003, 8, 128, "bf16", scattered=True, rotary=True,
                 per_layer=True),
        # the pages that a batch of decode steps has just filled
        _index("index 61 pages f16", 61, 8, 64, "f16"),
        # a long prompt's pages
        _index("index 8192 pages", 8192, 8, 128, "bf16"),
        # one sequence, 4k tokens: latency
        _sparse("sparse 1 x 4k", 1, 0, 4093, 16, 8, 128, "bf16", 32),
        # a few sequences of ragged lengths in fp32, small heads, an odd group
        _sparse("sparse 7 ragged f32", 7, 1000, 9000, 10, 2, 64, "f32", 48, sink=2, recent=3),
        # 64 branches of a 32768-token prefix
        _sparse("sparse 64 x 32k tree", 64, 32768, 4096, 32, 8, 128, "bf16", 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    c = _drawn(rng)
    del c["name"]
    return c


def _drawn(rng):
    kind = rng.choice(["rotary", "rotary", "fork", "compact", "index", "sparse", "sparse"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    d = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    if kind == "rotary":
        append = rng.random() < 0.6
        dim = d if append else rng.choice([64, 80, 96, 128, 256])
        part = rng.random() < 0.4
        rd = 2 * rng.randint(4, dim // 2) if part else dim
        offset = rng.randint(0, dim - rd) if part and rng.random() < 0.5 else 0
        return _rotary(None, _log(rng, 1, 8192), kv * rng.choice([1, 2, 4, 5, 8]), kv, dim, dtype, rotary_dim=rd,
                       offset=offset, interleaved=rng.random() < 0.4, base=rng.choice([1e4, 5e5, 1e6]),
                       factor=rng.choice([1.0, 1.0, 4.0, 8.0, 32.0]), max_position=_log(rng, 64, 1 << 20),
                       append=append, together=rng.random() < 0.4)
    if kind == "fork":
        trees = _log(rng, 1, 32)
        return _fork(None, rng.choice([1, 4, 16, 28, 32]), trees * rng.randint(1, 2), rng.randint(1, 3), trees,
                     _log(rng, 1, 2048), _log(rng, 1, 500))
    if kind == "compact":
        tokens = _log(rng, 20, 8000)
        return _compact(None, rng.randint(1, 3), rng.randint(1, 12), tokens, rng.randint(1, tokens), kv, d, dtype,
                        scattered=rng.random() < 0.5, rotary=rng.random() < 0.6, per_layer=rng.random() < 0.4)
    if kind == "index":
        return _index(None, _log(rng, 1, 4096), kv, d, dtype)
    budget = _log(rng, 4, 128)
    return _sparse(None, _log(rng, 1, 64), rng.choice([0, _log(rng, 100, 16000)]), _log(rng, 40, 4000),
                   kv * rng.choice([1, 2, 4, 5, 8, 16] if kv < 8 else [1, 2, 4, 8]), kv, d, dtype, budget, sink=rng.randint(0, 2),
                   recent=rng.randint(1, 2))


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def _frequencies(dim, base, factor, original=8192):
    """Angles per position of the dim / 2 pairs, float64, on the host; with factor > 1 stretched for contexts
    `factor` times longer: pairs that turn often keep their pace, slow ones are interpolated.  And the factor
    that the rotated values are multiplied by."""
    i = np.arange(dim // 2, dtype=np.float64)
    f = base ** (-2.0 * i / dim)
    if factor == 1.0:
        return f, 1.0

    def pair_of(turns):
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair_of(32)), 0), min(math.ceil(pair_of(1)), dim // 2 - 1)
    ramp = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _rand(shape, dtype, g):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _pages(n_tokens):
    return -(-n_tokens // BLOCK)


def _allocator(L, S, M, B, rows, lens, order):
    """Allocator and tables with `rows` (per layer and slot, lists of block ids in use) filled in; free blocks
    in `order`'s order."""
    tables = np.full((L, S, M), -1, np.int32)
    refs = np.zeros(B, np.int32)
    nblocks, ntok, tail = (np.zeros((L, S), np.int32) for _ in range(3))
    for layer in range(L):
        for s, ids in enumerate(rows[layer]):
            tables[layer, s, : len(ids)] = ids
            nblocks[layer, s], ntok[layer, s] = len(ids), lens[s]
            tail[layer, s] = lens[s] - (len(ids) - 1) * BLOCK if lens[s] else 0
    used = tables[tables >= 0]
    np.add.at(refs, used, 1)
    free = order[refs[order] == 0]
    ring = np.zeros(B, np.int32)
    ring[: len(free)] = free
    ctrl = np.zeros(WORDS, np.int64)
    ctrl[TAIL], ctrl[PEAK] = len(free), B - len(free)
    dev = {k: torch.from_numpy(v).cuda() for k, v in dict(tables=tables, refcounts=refs, ring=ring, ctrl=ctrl,
                                                          nblocks=nblocks, ntok=ntok, tail=tail).items()}
    return dev


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _prepare_rotary(c, g, rng):
    n, hq, hkv, d, dt = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"], DT[c["dtype"]]
    qkv = _rand((n, (hq + 2 * hkv) * d), dt, g)  # one projection's output: q, k and v are strided parts of it
    q, k, v = (t.view(n, -1, d) for t in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
    f, scale = _frequencies(c["rotary_dim"], c["base"], c["factor"])
    if c["together"]:  # one sequence's tokens, one after another
        p0 = rng.randrange(max(1, c["max_position"] - n))
        pos = torch.arange(p0, p0 + n, device="cuda")
    else:              # the next token of each of n sequences
        pos = torch.randint(0, c["max_position"], (n,), generator=g, device="cuda")
    s = {"q": q, "k": k, "v": v, "positions": pos, "inv_freq": torch.from_numpy(f).cuda(), "scale": scale}
    if c["append"]:
        blocks = _pages(n) + 64 if c["together"] else n + 64
        shape = (1, blocks, BLOCK, hkv, d)
        s["k_pool"], s["v_pool"] = _rand(shape, dt, g), _rand(shape, dt, g)
        perm = torch.randperm(blocks, generator=g, device="cuda")
        t = torch.arange(n, device="cuda")
        s["slots"] = perm[t // BLOCK] * BLOCK + t % BLOCK if c["together"] else perm[:n] * BLOCK + pos % BLOCK
    return s


def _prepare_fork(c, g, rng):
    L, n, kids, trees = c["layers"], c["parents"], c["children"], c["trees"]
    S = n * (1 + kids)
    per = n // trees
    lens, rows, nid = [c["prefix"] + rng.randint(0, c["suffix"]) for _ in range(n)], [], 0
    shared = c["prefix"] // BLOCK  # whole pages that a tree's leaves share
    M = _pages(c["prefix"] + c["suffix"])
    B = L * (trees * shared + n * (M - shared)) + 40
    order = np.random.RandomState(rng.randrange(1 << 30)).permutation(B).astype(np.int32)
    for _ in range(L):
        row = []
        for t in range(trees):
            pre = order[nid: nid + shared]
            nid += shared
            for i in range(t * per, (t + 1) * per):
                m = _pages(lens[i]) - shared
                row.append(np.concatenate([pre, order[nid: nid + m]]))
                nid += m
        rows.append(row + [[] for _ in range(S - n)])
    s = _allocator(L, S, M, B, rows, lens + [0] * (S - n), order)
    # the tokens themselves are not touched: the smallest rows stand for them
    s["k_pool"] = s["v_pool"] = torch.zeros((L, B, BLOCK, 1, 2), device="cuda")
    s["parents"] = _i32(np.repeat(np.arange(n), kids))
    s["children"] = _i32(np.arange(n, S))
    return s


def _prepare_compact(c, g, rng):
    L, n, hkv, d, dt = c["layers"], c["seqs"], c["kv_heads"], c["head_dim"], DT[c["dtype"]]
    lens = [rng.randint(max(1, c["tokens"] * 9 // 10), c["tokens"]) for _ in range(n)]
    kept = [max(1, min(x, c["kept"] * x // c["tokens"])) for x in lens]
    r = np.random.RandomState(rng.randrange(1 << 30))

    def choice(x, m):
        if c["scattered"]:
            return np.sort(r.permutation(x)[:m])
        sinks = min(4, m)
        return np.concatenate([np.arange(sinks), np.arange(x - (m - sinks), x)])

    keep = np.stack([np.concatenate([choice(x, m) for x, m in zip(lens, kept)])
                     for _ in range(L if c["per_layer"] else 1)]).astype(np.int32)
    M = _pages(c["tokens"])
    B = L * n * (M + _pages(c["kept"])) + 40
    order, nid, rows = r.permutation(B).astype(np.int32), 0, []
    for _ in range(L):
        row = []
        for x in lens:
            row.append(order[nid: nid + _pages(x)])
            nid += _pages(x)
        rows.append(row + [[] for _ in range(n)])
    s = _allocator(L, 2 * n, M, B, rows, lens + [0] * n, order)
    s["k_pool"], s["v_pool"] = (torch.empty((L, B, BLOCK, hkv, d), dtype=dt, device="cuda").normal_(generator=g)
                                for _ in range(2))
    s["src"], s["dst"] = _i32(np.arange(n)), _i32(np.arange(n, 2 * n))
    s["keep"], s["cu"] = _i32(keep), _i32(np.concatenate([[0], np.cumsum(kept)]))
    s["max_keep"] = max(kept)
    f, _ = _frequencies(d, 5e5, 1.0)
    s["inv_freq"] = torch.from_numpy(f).cuda() if c["rotary"] else None
    return s


def _keys(blocks, hkv, d, dt, g):
    """Keys as attention meets them: channels of unequal size, a subject that a page's tokens share."""
    size = torch.randn((hkv, d), generator=g, device="cuda").mul_(0.7).exp_()
    k = torch.empty((blocks, BLOCK, hkv, d), dtype=dt, device="cuda").normal_(generator=g)
    k *= (0.5 * size).to(dt)
    k += (torch.randn((blocks, 1, hkv, d), generator=g, device="cuda") * size).to(dt)
    return k.unsqueeze(0)


def _prepare_index(c, g, rng):
    blocks = c["blocks"]
    pool = blocks + 32
    s = {"k_pool": _keys(pool, c["kv_heads"], c["head_dim"], DT[c["dtype"]], g)}
    s["v_pool"] = s["k_pool"]
    s["blocks"] = torch.randperm(pool, generator=g, device="cuda")[:blocks].to(torch.int32)
    s["tables"] = s["blocks"].view(1, 1, -1)
    s["ntok"] = _i32([[blocks * BLOCK]])
    s["bounds"] = torch.zeros((1, pool, c["kv_heads"], 2, c["head_dim"]), dtype=torch.int8, device="cuda")
    s["exps"] = torch.zeros((1, pool, c["kv_heads"]), dtype=torch.int8, device="cuda")
    return s


def _prepare_sparse(c, g, rng):
    n, hq, hkv, d, dt = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], DT[c["dtype"]]
    lens = [c["prefix"] + rng.randint(max(1, c["suffix"] // 4), c["suffix"]) for _ in range(n)]
    shared = c["prefix"] // BLOCK
    B = shared + sum(_pages(x) - shared for x in lens) + 16
    k_pool = _keys(B, hkv, d, dt, g)
    order = np.random.RandomState(rng.randrange(1 << 30)).permutation(B).astype(np.int32)
    M = (max(_pages(x) for x in lens) + 3) // 4 * 4
    tables, nid = np.full((1, n, M), -1, np.int32), shared
    for i, x in enumerate(lens):
        m = _pages(x) - shared
        tables[0, i, :shared], tables[0, i, shared: shared + m] = order[:shared], order[nid: nid + m]
        nid += m
    s = {"k_pool": k_pool, "v_pool": _rand(tuple(k_pool.shape), dt, g), "tables": torch.from_numpy(tables).cuda(),
         "ntok": _i32([lens]), "slots": _i32(np.arange(n)), "max_len": max(lens)}
    # queries lean towards the subject of a page of their sequence
    at = torch.tensor([tables[0, i, rng.randrange(_pages(x))] for i, x in enumerate(lens)], device="cuda")
    near = k_pool[0][at, 0].float().repeat_interleave(hq // hkv, dim=1)
    near = near / near.square().mean(dim=2, keepdim=True).sqrt()
    s["q"] = (1.2 * near + torch.randn((n, hq, d), generator=g, device="cuda")).to(dt)
    s["bounds"], s["exps"] = _page_index(k_pool[0])
    s["bounds"], s["exps"] = s["bounds"].unsqueeze(0), s["exps"].unsqueeze(0)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = globals()["_prepare_" + case["kind"]](case, g, random.Random(seed))
    s["case"] = case
    if own:  # the handles that a program keeps beside its tensors
        from mentat_b200 import KVCacheView, PageIndex, Rotary
        if "k_pool" in s:
            s["cache"] = KVCacheView(s["k_pool"], s["v_pool"], s.get("tables"), s.get("ntok"),
                                     nblocks=s.get("nblocks"), tail=s.get("tail"), refcounts=s.get("refcounts"),
                                     free_ring=s.get("ring"), ctrl=s.get("ctrl"))
        if "bounds" in s:
            s["index"] = PageIndex(s["cache"], bounds=s["bounds"], exps=s["exps"])
        if s.get("inv_freq") is not None:
            s["rotary"] = Rotary(case["head_dim"], inv_freq=s["inv_freq"], offset=case.get("offset", 0),
                                 interleaved=case.get("interleaved", False), attention_scaling=s.get("scale", 1.0))
    return s


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------
def _rotated(x, positions, inv_freq, scale, offset, interleaved):
    """x (N, H, D) with dims offset .. offset + 2 len(inv_freq) turned by positions * inv_freq, in 32 bits."""
    m = inv_freq.numel()
    a = positions.double().unsqueeze(1) * inv_freq
    cos, sin = (a.cos() * scale).float().unsqueeze(1), (a.sin() * scale).float().unsqueeze(1)
    part = x[..., offset: offset + 2 * m].float()
    u, w = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :m], part[..., m:])
    y, z = u * cos - w * sin, u * sin + w * cos
    turned = torch.stack((y, z), dim=-1).flatten(-2) if interleaved else torch.cat((y, z), dim=-1)
    return torch.cat((x[..., :offset], turned.to(x.dtype), x[..., offset + 2 * m:]), dim=-1)


def _run_rotary(s):
    c = s["case"]
    how = (s["positions"], s["inv_freq"], s["scale"], c["offset"], c["interleaved"])
    q, k = _rotated(s["q"], *how), _rotated(s["k"], *how)
    if not c["append"]:
        return {"q": q, "k": k}
    for pool, rows in ((s["k_pool"], k), (s["v_pool"], s["v"])):
        pool.view(-1, *pool.shape[3:]).index_copy_(0, s["slots"], rows)
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _live(s, slots):
    """Block ids of the slots' pages as (sequence, layer, page), and which of them exist."""
    slots = slots.long()
    ids = s["tables"][:, slots].transpose(0, 1)
    n = s["nblocks"][:, slots].transpose(0, 1)
    return ids, torch.arange(ids.shape[2], device=ids.device) < n.unsqueeze(2)


def _free(s, slots):
    """Every page of the slots released, sequence by sequence, layer by layer, in table order; a page joins the
    free list where its last reference goes."""
    ids, have = _live(s, slots)
    ids = ids[have].long()
    s["refcounts"].index_add_(0, ids, torch.full_like(ids, -1, dtype=torch.int32))
    at = torch.arange(ids.numel(), device=ids.device)
    last = torch.full((s["refcounts"].numel(),), -1, device=ids.device).scatter_reduce_(0, ids, at, "amax")
    gone = ids[(last[ids] == at) & (s["refcounts"][ids] == 0)]
    B = s["ring"].numel()
    s["ring"][(s["ctrl"][TAIL] + torch.arange(gone.numel(), device=ids.device)) % B] = gone.int()
    s["ctrl"][TAIL] += gone.numel()
    for t in ("nblocks", "ntok", "tail"):
        s[t][:, slots.long()] = 0


def _allocator_state(s):
    return {t: s[t] for t in ("tables", "nblocks", "ntok", "tail", "refcounts", "ring", "ctrl")}


def _run_fork(s):
    parents, children = s["parents"].long(), s["children"].long()
    ids, have = _live(s, s["parents"])
    rows = s["tables"][:, children].transpose(0, 1)
    s["tables"][:, children] = torch.where(have, ids, rows).transpose(0, 1)
    for t in ("nblocks", "ntok", "tail"):
        s[t][:, children] = s[t][:, parents]
    ids = ids[have].long()
    s["refcounts"].index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    _free(s, s["children"])
    return _allocator_state(s)


def _run_compact(s):
    c = s["case"]
    L, n = c["layers"], c["seqs"]
    dev = s["keep"].device
    cu = s["cu"].long()
    keep = s["keep"].long().expand(L, -1)
    count = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(n, device=dev), count)
    j = torch.arange(keep.shape[1], device=dev) - cu[seq]
    # full pages at the front whose tokens all stay where they are keep their blocks (a sequence that keeps
    # every token keeps every page)
    moved = torch.where(keep != j, j, count[seq]).to(torch.int64)
    first = torch.full((L, n), 1 << 40, device=dev).scatter_reduce_(1, seq.expand(L, -1), moved, "amin")
    pages = (count + BLOCK - 1) // BLOCK
    whole = (first == count) & (count == s["ntok"][:, s["src"].long()])
    lead = torch.where(whole, pages, first.minimum(count) // BLOCK)
    # fresh blocks, popped sequence by sequence, layer by layer, page by page
    page = torch.arange(s["tables"].shape[2], device=dev)
    mine = page < pages.view(n, 1, 1)
    fresh = mine & (page >= lead.t().unsqueeze(2))
    total = int(fresh.sum())
    src, dst = s["src"].long(), s["dst"].long()
    old = s["tables"][:, src].transpose(0, 1)
    new = torch.where(mine, old, s["tables"][:, dst].transpose(0, 1))
    B = s["ring"].numel()
    new[fresh] = s["ring"][(s["ctrl"][HEAD] + torch.arange(total, device=dev)) % B]
    s["ctrl"][HEAD] += total
    s["ctrl"][ALLOCS] += total
    s["ctrl"][PEAK] = torch.maximum(s["ctrl"][PEAK], B - (s["ctrl"][TAIL] - s["ctrl"][HEAD]))
    s["refcounts"][new[fresh].long()] = 1
    held = new[mine & ~fresh].long()
    s["refcounts"].index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    # the rows of fresh pages: read at the kept position, turned to the new one
    lay = torch.arange(L, device=dev).unsqueeze(1).expand(L, keep.shape[1])
    go = (j // BLOCK).expand(L, -1) >= lead[:, seq]
    lay, at, to, i = lay[go], keep[go], j.expand(L, -1)[go], seq.expand(L, -1)[go]
    from_row = (lay * B + old[i, lay, at // BLOCK]) * BLOCK + at % BLOCK
    to_row = (lay * B + new[i, lay, to // BLOCK]) * BLOCK + to % BLOCK
    for pool, turn in ((s["k_pool"], c["rotary"]), (s["v_pool"], False)):
        rows = pool.view(-1, *pool.shape[3:])
        x = rows[from_row]
        rows[to_row] = _rotated(x, to - at, s["inv_freq"], 1.0, 0, False) if turn else x
    s["tables"][:, dst] = new.transpose(0, 1)
    s["nblocks"][:, dst], s["ntok"][:, dst] = pages.int(), count.int()
    s["tail"][:, dst] = (count - (pages - 1) * BLOCK).int()
    _free(s, s["dst"])
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"], **_allocator_state(s)}


def _exponent(top):
    """The least e with top <= 127 * 2**e, within -50 .. 50."""
    m, e = torch.frexp(top)
    return (e - 7 + (m > 127 / 128).int()).clamp(-50, 50)


def _power(e):
    """2**e exactly, for whole numbers e."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _page_index(k):
    """Bounds of the keys k (pages, 16, H, D) of each page, head and channel: int8 (pages, H, 2, D), lowest
    values rounded down and highest up, times 2**exps."""
    lo, hi = k.amin(dim=1).float(), k.amax(dim=1).float()
    e = _exponent(torch.maximum(lo.abs(), hi.abs()).amax(dim=-1))
    unit = _power(e).unsqueeze(-1)
    b = torch.stack(((lo / unit).floor(), (hi / unit).ceil()), dim=-2)
    return b.clamp(-127, 127).to(torch.int8), e.to(torch.int8)


def _run_index(s):
    b = s["blocks"].long()
    bounds, exps = _page_index(s["k_pool"][0][b])
    s["bounds"][0, b], s["exps"][0, b] = bounds, exps
    values = bounds.float() * _power(exps)[..., None, None]
    return {"low": values[:, :, 0], "high": values[:, :, 1], "exps": exps}


def _run_sparse(s):
    c = s["case"]
    q, n, hkv, k_pool, v_pool = s["q"].float(), c["seqs"], c["kv_heads"], s["k_pool"][0], s["v_pool"][0]
    group, d, budget = c["heads"] // hkv, c["head_dim"], c["budget"]
    lens = s["ntok"][0].long()
    pages = ((lens + BLOCK - 1) // BLOCK).view(n, 1, 1)
    ids = s["tables"][0].long().clamp_min(0)
    P = ids.shape[1]
    # scores: whole numbers times powers of two, exact in 32 bits
    eq = _exponent(q.abs().amax(dim=-1))
    q8 = torch.round(q / _power(eq).unsqueeze(-1)).view(n, hkv, group, d)
    both = torch.cat((q8.clamp_max(0), q8.clamp_min(0)), dim=-1)
    bounds = s["bounds"][0][ids].permute(0, 2, 1, 3, 4).reshape(n, hkv, P, 2 * d).float()
    dots = both @ bounds.transpose(2, 3)
    unit = _power(eq).view(n, hkv, group, 1) * _power(s["exps"][0][ids]).permute(0, 2, 1).unsqueeze(2)
    score = (dots * unit).amax(dim=2)
    at = torch.arange(P, device=q.device)
    score = score.masked_fill((at < c["sink"]) | (at >= pages - c["recent"]), math.inf)
    score = score.masked_fill(at >= pages, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    best = best.masked_fill(best >= pages, P).sort(dim=-1).values
    if best.shape[-1] < budget:
        best = torch.nn.functional.pad(best, (0, budget - best.shape[-1]), value=P)
    # attention over the chosen pages' tokens
    blocks = ids.gather(1, best.clamp_max(P - 1).view(n, -1)).view(n, hkv, budget)
    head = torch.arange(hkv, device=q.device).view(1, hkv, 1)
    k = k_pool[blocks, :, head].reshape(n, hkv, budget * BLOCK, d).float()
    v = v_pool[blocks, :, head].reshape(n, hkv, budget * BLOCK, d).float()
    token = (best.unsqueeze(-1) * BLOCK + torch.arange(BLOCK, device=q.device)).view(n, hkv, 1, -1)
    x = (q.view(n, hkv, group, d) @ k.transpose(2, 3)) / math.sqrt(d)
    x = x.masked_fill((token >= lens.view(n, 1, 1, 1)) | (token >= P * BLOCK), -math.inf)
    p = (x - x.amax(dim=-1, keepdim=True)).exp()
    out = (p @ v) / p.sum(dim=-1, keepdim=True)
    return {"out": out.view(n, c["heads"], d).to(s["q"].dtype),
            "pages": best.masked_fill(best == P, -1).int()}


# ---------------------------------------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------------------------------------
def _own_rotary(s):
    from mentat_b200 import ops
    if not s["case"]["append"]:
        q, k = ops.rotary(s["q"], s["k"], s["positions"], s["rotary"])
        return {"q": q, "k": k}
    q = ops.rotary_append(s["cache"], 0, s["slots"], s["q"], s["k"], s["v"], s["positions"], s["rotary"])
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _own_fork(s):
    from mentat_b200 import ops
    ops.fork_pages(s["cache"], s["parents"], s["children"])
    ops.free_pages(s["cache"], s["children"])
    return _allocator_state(s)


def _own_compact(s):
    from mentat_b200 import ops
    ops.compact_pages(s["cache"], s["src"], s["dst"], s["keep"], s["cu"], s["max_keep"], rotary=s.get("rotary"))
    ops.free_pages(s["cache"], s["dst"])
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"], **_allocator_state(s)}


def _own_index(s):
    from mentat_b200 import ops
    ops.page_index(s["index"], 0, s["blocks"])
    low, high, exps = ops.page_bounds(s["index"], 0, s["blocks"])
    return {"low": low, "high": high, "exps": exps}


def _own_sparse(s):
    from mentat_b200 import ops
    c = s["case"]
    out, pages = ops.sparse_decode(s["index"], 0, s["slots"], s["q"], s["max_len"], c["budget"], sink=c["sink"],
                                   recent=c["recent"], return_pages=True)
    return {"out": out, "pages": pages}


def run(state):
    return globals()[("_own_" if own else "_run_") + state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    size = 4 if c.get("dtype") == "f32" else 2
    if c["kind"] == "rotary":
        row = c["head_dim"] * size
        moved = 2 * c["tokens"] * (c["heads"] + c["kv_heads"] * (2 if c["append"] else 1)) * row
        return {"bytes": moved + 8 * c["tokens"] * (2 if c["append"] else 1),
                "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rotary_dim"]}
    if c["kind"] == "fork":
        # each parent's table once, each child's once; a reference count read and written for each page
        per = _pages(c["prefix"] + c["suffix"] // 2)
        entries = c["layers"] * c["parents"] * per
        pages = c["layers"] * (c["trees"] * (c["prefix"] // BLOCK) + c["parents"] * (per - c["prefix"] // BLOCK))
        return {"bytes": 4 * entries * (1 + c["children"]) + 8 * pages, "flops": entries * c["children"]}
    if c["kind"] == "compact":
        kept = c["seqs"] * max(1, round(c["kept"] * 0.95))
        rows = c["layers"] * kept * c["kv_heads"] * c["head_dim"]
        return {"bytes": 4 * rows * size + 4 * kept * (c["layers"] if c["per_layer"] else 1),
                "flops": 3 * rows if c["rotary"] else 0}
    per_page = c["kv_heads"] * (2 * c["head_dim"] + 1)
    if c["kind"] == "index":
        return {"bytes": c["blocks"] * (BLOCK * c["kv_heads"] * c["head_dim"] * size + per_page
                                        + 8 * c["kv_heads"] * c["head_dim"]),
                "flops": 2 * c["blocks"] * BLOCK * c["kv_heads"] * c["head_dim"]}
    # each page's bounds once; the chosen pages' keys and values once for each sequence
    mean = c["prefix"] + 0.625 * c["suffix"]
    shared = c["prefix"] // BLOCK
    pages = shared + c["seqs"] * (mean / BLOCK - shared)
    tokens = c["seqs"] * min(mean, c["budget"] * BLOCK)
    return {"bytes": int(pages * per_page + 2 * tokens * c["kv_heads"] * c["head_dim"] * size
                         + 2 * c["seqs"] * c["heads"] * c["head_dim"] * size),
            "flops": int(4 * tokens * c["heads"] * c["head_dim"]
                         + 4 * c["seqs"] * mean / BLOCK * c["heads"] * c["head_dim"])}


# ---------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------
def _turned64(x, angle, scale, offset, interleaved):
    """x (N, H, D) in float64: its pairs as complex numbers times scale * exp(i angle) (N, pairs)."""
    x = x.double().clone()
    m = angle.shape[1]
    first = offset + (2 * torch.arange(m, device=x.device) if interleaved else torch.arange(m, device=x.device))
    second = first + (1 if interleaved else m)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(angle, scale), angle).unsqueeze(1)
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rotary(c, s):
    angle = torch.outer(s["positions"].double(), s["inv_freq"])
    q, k = (_turned64(s[t], angle, s["scale"], c["offset"], c["interleaved"]) for t in ("q", "k"))
    if not c["append"]:
        return {"q": q, "k": k}
    pools = {"q": q}
    for name, rows in (("k_pool", k), ("v_pool", s["v"].double())):
        pools[name] = s[name].double()
        pools[name][0, s["slots"] // BLOCK, s["slots"] % BLOCK] = rows
    return pools


def _exact_compact(c, s):
    """The pools; the allocator's whole numbers have no other value than the plain form's."""
    cu, keep = s["cu"].tolist(), s["keep"].cpu().numpy()
    tables, ring = s["tables"].cpu().numpy(), s["ring"].cpu().numpy()
    pools = {"k_pool": s["k_pool"].double(), "v_pool": s["v_pool"].double()}
    head = int(s["ctrl"][HEAD])
    for i in range(c["seqs"]):
        for layer in range(c["layers"]):
            kept = keep[layer if c["per_layer"] else 0, cu[i]: cu[i + 1]]
            stay = 0
            while stay < len(kept) and kept[stay] == stay:
                stay += 1
            if stay == len(kept) == int(s["ntok"][layer, i]):
                continue
            begin = stay // BLOCK * BLOCK
            to = np.arange(begin, len(kept))
            new = ring[(head + np.arange(_pages(len(kept)) - begin // BLOCK)) % len(ring)]
            head += len(new)
            at = torch.from_numpy(kept[begin:].astype(np.int64)).cuda()
            page = torch.from_numpy(tables[layer, i].astype(np.int64)).cuda()[at // BLOCK]
            to = torch.from_numpy(to).cuda()
            target = torch.from_numpy(new.astype(np.int64)).cuda()[to // BLOCK - begin // BLOCK]
            k = s["k_pool"][layer, page, at % BLOCK]
            if c["rotary"]:
                k = _turned64(k, torch.outer((to - at).double(), s["inv_freq"]), 1.0, 0, False)
            pools["k_pool"][layer, target, to % BLOCK] = k.double()
            pools["v_pool"][layer, target, to % BLOCK] = s["v_pool"][layer, page, at % BLOCK].double()
    return {**pools, **{t: None for t in _allocator_state(s)}}


def _exact_index(c, s):
    k = s["k_pool"][0][s["blocks"].long()].double()
    top = k.abs().amax(dim=(1, 3))
    e = torch.full_like(top, -50.0)
    for step in range(-50, 50):  # the least power of two whose 127-fold covers the page's keys
        e = torch.where(top > 127.0 * 2.0 ** step, float(step + 1), e)
    unit = _power64(e).unsqueeze(-1)
    low = -torch.floor(-k.amin(dim=1) / unit)
    return {"low": torch.where(low * unit > k.amin(dim=1), low - 1, low).clamp(-127, 127) * unit,
            "high": (-torch.floor(-k.amax(dim=1) / unit)).clamp(-127, 127) * unit, "exps": e.to(torch.int8)}


def _exact_sparse(c, s):
    group, d, budget = c["heads"] // c["kv_heads"], c["head_dim"], c["budget"]
    out = torch.zeros((c["seqs"], c["heads"], d), dtype=torch.float64, device="cuda")
    chosen = np.full((c["seqs"], c["kv_heads"], budget), -1, np.int32)
    for i in range(c["seqs"]):
        length = int(s["ntok"][0, i])
        pages = _pages(length)
        row = s["tables"][0, i, :pages].long()
        q = s["q"][i].double()
        # queries on the grid of their own power of two, bounds as the numbers that they stand for
        top = q.abs().amax(dim=1, keepdim=True)
        unit = _power64(torch.ceil(torch.log2(top / 127.0)).clamp(-50, 50))
        unit = torch.where(top > 127.0 * unit, 2 * unit, torch.where(top <= 63.5 * unit, unit / 2, unit))
        grid = torch.round(q / unit) * unit
        values = s["bounds"][0][row].double() * _power64(s["exps"][0][row])[..., None, None]
        score = torch.stack([torch.maximum(grid[h] * values[:, h // group, 0], grid[h] * values[:, h // group, 1]).sum(dim=1)
                             for h in range(c["heads"])])
        score = score.view(c["kv_heads"], group, pages).amax(dim=1).cpu().numpy()
        forced = set(range(min(c["sink"], pages))) | set(range(max(0, pages - c["recent"]), pages))
        for h in range(c["kv_heads"]):
            ranked = sorted(range(pages), key=lambda p: (p not in forced, -score[h, p], p))[:budget]
            ranked.sort()
            chosen[i, h, : len(ranked)] = ranked
            at = torch.tensor(ranked, device="cuda")
            k = s["k_pool"][0, row[at], :, h].reshape(-1, d).double()
            v = s["v_pool"][0, row[at], :, h].reshape(-1, d).double()
            token = (at[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten()
            x = (q[h * group: (h + 1) * group] @ k.t()) / math.sqrt(d)
            x[:, token >= length] = -math.inf
            out[i, h * group: (h + 1) * group] = torch.softmax(x, dim=1) @ v
    return {"out": out, "pages": torch.from_numpy(chosen)}


def exact(case, seed):
    if case["kind"] == "fork":
        return None  # whole numbers only
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))
