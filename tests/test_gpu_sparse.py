"""The page index and sparse decode against their definitions (``oracle.cache_ops``): the index and
the chosen pages exactly, the attention over them in 64 bits."""

import math

import numpy as np
import pytest
import torch

from oracle.cache_ops import index_page, sparse_decode
from tests.gpu_util import TORCH_DT

pytestmark = pytest.mark.gpu


def tolerance(dtype, v):
    """Of an output element, from the largest value it averages.  fp32: scores of |s| < 64 carry
    (d / 4 + 8) 2^-24 of sum |q k| <= 64, so a weight's error is below 41 * 64 * 2^-24 < 2^-12.6, which
    two-sided normalisation halves for what does not move together; the bound of 2e-5 (2^-15.6) of the
    other attention tests is kept: |s| here stays near 8.  bf16 / fp16: weights and the result are
    each rounded at most once to the type (half a step each), and the scores add 2^-16."""
    eps = torch.finfo(TORCH_DT[dtype]).eps
    top = float(np.abs(v).max())
    return 2e-5 * top if dtype == "f32" else (eps + 2.0 ** -14) * top


def make(lens, hq, hkv, d, bs, dtype, *, layers=2, shared=0, seed=0, extra=3):
    """One cache of given lengths; the first `shared` pages of all sequences are the same blocks."""
    from mentat_b200 import KVCacheView, PageIndex, ops
    rng = np.random.default_rng(seed)
    pages = [-(-n // bs) for n in lens]
    blocks = shared + sum(max(0, p - shared) for p in pages) + extra
    order = rng.permutation(blocks)
    cap = max(pages + [1]) + 2
    tables = np.full((layers, len(lens) + 1, cap), -7, np.int32)
    nid = shared
    for i, p in enumerate(pages):
        a = min(shared, p)
        tables[:, i, :a] = order[:a]
        tables[:, i, a:p] = order[nid: nid + p - a]
        nid += p - a
    dt = TORCH_DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    size = torch.exp(0.5 * torch.randn((hkv, d), generator=g, device="cuda"))
    k = (torch.randn((layers, blocks, 1, hkv, d), generator=g, device="cuda") * 0.7 +
         torch.randn((layers, blocks, bs, hkv, d), generator=g, device="cuda") * 0.5) * size
    k, v = k.to(dt), torch.randn((layers, blocks, bs, hkv, d), generator=g, device="cuda").to(dt)
    ntok = torch.tensor([list(lens) + [0]] * layers, dtype=torch.int32, device="cuda")
    c = KVCacheView(k, v, torch.from_numpy(tables).cuda(), ntok)
    x = PageIndex(c)
    for layer in range(layers):
        ops.page_index(x, layer, torch.from_numpy(order[:nid].astype(np.int32)).cuda())
    q = torch.randn((len(lens), hq, d), generator=g, device="cuda").to(dt)
    return c, x, q, tables


def run_and_check(c, x, q, tables, lens, budget, sink, recent, dtype, layer=1, scale=None, slots=None):
    from mentat_b200 import ops
    slots = list(range(len(lens))) if slots is None else slots
    out, pages = ops.sparse_decode(x, layer, torch.tensor(slots, dtype=torch.int32, device="cuda"), q, max(lens + [0]),
                                   budget, sink=sink, recent=recent, scale=scale, return_pages=True)
    c.check()
    kp, vp = (t[layer].double().cpu().numpy() for t in (c._tensors["k_pool"], c._tensors["v_pool"]))
    want, chosen = sparse_decode(q.double().cpu().numpy(), kp, vp, [tables[layer, s] for s in slots],
                                 [lens[s] if s < len(lens) else 0 for s in slots], c.block_size,
                                 x.bounds[layer].cpu().numpy(), x.exps[layer].cpu().numpy(), budget, sink, recent, scale)
    np.testing.assert_array_equal(pages.cpu().numpy(), chosen)
    off = np.abs(out.double().cpu().numpy() - want)
    assert np.all(off <= tolerance(dtype, vp)), float(off.max())
    only = ops.sparse_decode(x, layer, torch.tensor(slots, dtype=torch.int32, device="cuda"), q, max(lens + [0]), budget,
                             sink=sink, recent=recent, scale=scale)
    assert torch.equal(only, out)
    return out, pages


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 16), (1, 64, 16), (3, 40, 5), (2, 200, 32)])
def test_page_index(dtype, hkv, d, bs):
    from mentat_b200 import KVCacheView, PageIndex, ops
    g = torch.Generator(device="cuda").manual_seed(0)
    blocks, layer = 23, 1
    k = torch.randn((2, blocks, bs, hkv, d), generator=g, device="cuda")
    k *= torch.exp(4 * torch.randn((2, blocks, 1, 1, 1), generator=g, device="cuda"))
    k[1, 3] = 0
    k[1, 4] = -2.0                      # powers of two, and the borders of one unit
    k[1, 5, 0, 0, 0] = float("nan")
    k[1, 6, bs - 1, hkv - 1, d - 1] = float("inf")
    k[1, 7] = 127.0
    k[1, 8] = 127.5
    k[1, 9] = 0
    k[1, 9, 0, 0, 0] = 6e-8             # fp16's smallest
    k = k.to(TORCH_DT[dtype])
    if dtype != "f16":
        k[1, 10] *= 1e30                # saturates
        k[1, 11] *= 1e-30
    c = KVCacheView(k, k)
    x = PageIndex(c)
    ids = torch.tensor([i for i in range(blocks) if i != 20], dtype=torch.int32, device="cuda")
    ops.page_index(x, layer, torch.cat([ids, ids[:3]]))  # some twice
    low, high, exps = ops.page_bounds(x, layer, ids)
    kk = k[layer].double().cpu().numpy()
    for i, b in enumerate(ids.tolist()):
        bounds, e = index_page(kk[b])
        np.testing.assert_array_equal(x.bounds[layer, b].cpu().numpy(), bounds)
        np.testing.assert_array_equal(x.exps[layer, b].cpu().numpy(), e)
        np.testing.assert_array_equal(exps[i].cpu().numpy(), e)
        fine = e != 127
        unit = 2.0 ** e[fine].astype(float)[:, None]
        np.testing.assert_array_equal(low[i].double().cpu().numpy()[fine], bounds[fine, 0] * unit)
        np.testing.assert_array_equal(high[i].double().cpu().numpy()[fine], bounds[fine, 1] * unit)
        assert torch.isinf(low[i][torch.from_numpy(~fine)]).all()
        if b != 10 and fine.all():
            assert (low[i].double().cpu().numpy() <= kk[b].min(0)).all() and (high[i].double().cpu().numpy() >= kk[b].max(0)).all()
    assert (x.exps[layer, 20] == 127).all() and (x.exps[0] == 127).all()  # not indexed
    c.check()
    ops.page_index(x, layer, torch.tensor([blocks, 0, -1], dtype=torch.int32, device="cuda"))
    with pytest.raises(AssertionError, match="outside the pool"):
        c.check()


CASES = [  # lens, hq, hkv, d, bs, shared, budget, sink, recent
    ([0, 1, 15, 16, 17, 33], 8, 8, 128, 16, 0, 2, 0, 1), ([0, 1, 2, 3, 4, 5, 6, 40], 4, 2, 64, 4, 0, 3, 1, 1),
    ([500, 1, 777, 160], 8, 2, 128, 16, 5, 8, 1, 2), ([1000, 999], 10, 2, 64, 16, 20, 17, 2, 3),
    ([300], 16, 1, 128, 16, 0, 1, 0, 1), ([640, 641], 32, 4, 128, 32, 3, 6, 0, 1), ([200, 90], 3, 1, 64, 5, 2, 9, 1, 1),
    ([4097, 70, 2500], 16, 8, 128, 16, 0, 40, 1, 2), ([350, 20], 7, 7, 64, 24, 0, 5, 0, 2),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][0]}x{len(c[0])}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[6]}")
def test_sparse_decode_matches_definition(case, dtype):
    lens, hq, hkv, d, bs, shared, budget, sink, recent = case
    c, x, q, tables = make(lens, hq, hkv, d, bs, dtype, shared=shared)
    run_and_check(c, x, q, tables, lens, budget, sink, recent, dtype)
    # strided queries, sequences in another order and twice, another scale, a slot without tokens
    wide = torch.cat([q, q], dim=1)[:, :hq]
    slots = [len(lens) - 1, 0, len(lens), 0]
    run_and_check(c, x, wide[[len(lens) - 1, 0, 0, 0]], tables, lens, budget, sink, recent, dtype, layer=0,
                  scale=0.3, slots=slots)


def test_many_pages():
    """Long sequences: selection over thousands of pages, a large budget."""
    lens = [70001, 40000, 64 * 16]
    c, x, q, tables = make(lens, 8, 2, 64, 16, "bf16", layers=1, shared=1000)
    for budget in (64, 1500):
        run_and_check(c, x, q, tables, lens, budget, 1, 2, "bf16", layer=0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_pages_than_one_block_holds(dtype):
    """Pages of one token: 40,000 and 17,000 of them, and a batch beside them without a choice to make."""
    lens = [40000, 30, 17000]
    c, x, q, tables = make(lens, 2, 1, 64, 1, dtype, layers=1, shared=7000)
    run_and_check(c, x, q, tables, lens, 33, 2, 3, dtype, layer=0)
    x.exps.zero_()
    x.bounds.zero_()  # all the same: the lowest
    run_and_check(c, x, q, tables, lens, 33, 2, 3, dtype, layer=0)


def test_batches_of_trees():
    """Batches with a launch of their own for the scores: rows that share all, some or none of their pages,
    rows without a choice, corrupt and empty ones among them, groups that do not divide the columns."""
    rng = np.random.default_rng(5)
    for hq, hkv, d, n in ((24, 8, 64, 41), (10, 2, 128, 90), (16, 1, 64, 160)):
        lens = [int(v) for v in rng.integers(1, 900, n)]
        lens[3], lens[5], lens[n - 1] = 0, 17, 897
        c, x, q, tables = make(lens, hq, hkv, d, 16, "bf16", layers=1, shared=21)
        run_and_check(c, x, q, tables, lens, 8, 1, 2, "bf16", layer=0)


# hq, hkv, d, bs, n, dtype: more heads than CTAs run at once and more than 600 pages, so that scores and choice
# have launches of their own, for groups of 1 to 16 and with and without tensor cores
LONG = [(5, 5, 128, 16, 31, "bf16"), (4, 2, 64, 16, 77, "f16"), (12, 4, 128, 32, 38, "bf16"), (25, 5, 64, 16, 31, "f16"),
        (20, 2, 128, 16, 76, "bf16"), (16, 1, 64, 16, 150, "bf16"), (8, 4, 64, 5, 76, "f32"), (9, 3, 128, 24, 101, "f16")]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(map(str, c)))
def test_large_batches_of_long_sequences(case):
    hq, hkv, d, bs, n, dtype = case
    rng = np.random.default_rng(n)
    lens = [int(v) for v in rng.integers(580 * bs, 640 * bs, n)]
    lens[0] = 640 * bs
    for i in rng.choice(np.arange(1, n), n // 4, replace=False):  # short ones, some without a choice
        lens[i] = int(rng.integers(0, 40 * bs))
    lens[2], lens[n - 1] = 0, 639 * bs + 1
    # a common prefix that ends inside a tile of pages, and its first pages alone
    for shared, budget, sink, recent in ((585, 37, 1, 2), (21, 600, 0, 1)):
        c, x, q, tables = make(lens, hq, hkv, d, bs, dtype, layers=1, shared=shared)
        if budget == 600:  # most of the pages, for sequences in any order and more than once
            some = rng.choice(n, 310 // hkv, replace=True)
            run_and_check(c, x, q[torch.from_numpy(some).cuda()], tables, lens, budget, sink, recent, dtype, layer=0,
                          slots=[int(i) for i in some])
        else:
            run_and_check(c, x, q, tables, lens, budget, sink, recent, dtype, layer=0)


def test_large_batches_record_bad_state():
    """The same with a table entry outside the pool, a bad slot and a row longer than max_len: recorded, not
    read, and the other rows come out as before."""
    from mentat_b200 import ops
    n, lens = 80, [610 * 16] * 80
    c, x, q, tables = make(lens, 4, 2, 64, 16, "bf16", layers=1, shared=600)
    every = torch.arange(n, dtype=torch.int32, device="cuda")
    want = ops.sparse_decode(x, 0, every, q, 610 * 16, 12)
    c.check()
    slots = every.clone()
    slots[7] = n + 5
    got = ops.sparse_decode(x, 0, slots, q, 610 * 16, 12)
    with pytest.raises(ValueError, match="slot"):
        c.check()
    c._tensors["ctrl"].zero_()
    rest = [i for i in range(n) if i != 7]
    assert torch.equal(got[rest], want[rest]) and not got[7].any()
    got = ops.sparse_decode(x, 0, every, q, 610 * 16 - 1, 12)
    with pytest.raises(RuntimeError, match="overflow"):
        c.check()
    c._tensors["ctrl"].zero_()
    assert not got.any()
    for page in (300, 605):                                  # among the shared ones, and a sequence's own
        c._tensors["tables"][0, 11, page] = c.max_blocks
        got = ops.sparse_decode(x, 0, every, q, 610 * 16, 12)
        with pytest.raises(AssertionError):
            c.check()
        c._tensors["ctrl"].zero_()
        rest = [i for i in range(n) if i != 11]
        assert torch.equal(got[rest], want[rest])
        c._tensors["tables"][0, 11, page] = int(tables[0, 11, page])


def test_ties_go_to_the_lowest_page():
    from mentat_b200 import ops
    lens = [2000]
    c, x, q, tables = make(lens, 4, 1, 64, 16, "bf16", layers=1)
    x.bounds.zero_()
    x.exps.zero_()
    _, pages = ops.sparse_decode(x, 0, torch.zeros(1, dtype=torch.int32, device="cuda"), q, 2000, 9, sink=0, recent=2,
                                 return_pages=True)
    assert pages.flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 123, 124]
    run_and_check(c, x, q, tables, lens, 9, 0, 2, "bf16", layer=0)
    run_and_check(c, x, torch.zeros_like(q), tables, lens, 9, 3, 2, "bf16", layer=0)


def test_pages_with_infinities_are_chosen_and_show():
    """A page with a NaN key is attended to, so the output shows it as dense decode does; a query
    element that is not finite counts as 0 in the score."""
    from mentat_b200 import ops
    lens = [800, 800]
    c, x, q, tables = make(lens, 4, 2, 64, 16, "f32", layers=1)
    b = int(tables[0, 0, 30])
    c._tensors["k_pool"][0, b, 3, 1, 5] = float("nan")
    ops.page_index(x, 0, torch.tensor([b], dtype=torch.int32, device="cuda"))
    q[1, 0, 7] = float("inf")
    slots = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    out, pages = ops.sparse_decode(x, 0, slots, q, 800, 4, return_pages=True)
    assert 30 in pages[0, 1].tolist()
    assert torch.isfinite(out[0, :2]).all() and torch.isnan(out[0, 2:]).all()
    assert not torch.isfinite(out[1, 0]).any() and torch.isfinite(out[1, 1:]).all()
    _, chosen = sparse_decode(np.nan_to_num(q.double().cpu().numpy(), posinf=0.0), c._tensors["k_pool"][0].double().cpu().numpy(),
                              c._tensors["v_pool"][0].double().cpu().numpy(), [tables[0, 0], tables[0, 1]], lens, 16,
                              x.bounds[0].cpu().numpy(), x.exps[0].cpu().numpy(), 4, 1, 1)
    np.testing.assert_array_equal(pages.cpu().numpy(), chosen)


def test_sparse_decode_records_bad_state():
    from mentat_b200 import ops
    lens = [500, 300]
    c, x, q, tables = make(lens, 4, 2, 64, 16, "bf16")
    both = torch.tensor([0, 1], dtype=torch.int32, device="cuda")

    def recorded(exc, call):
        call()
        with pytest.raises(exc):
            c.check()
        c._tensors["ctrl"].zero_()
    out = ops.sparse_decode(x, 0, both, q, 499, 8)          # longer than max_len: zeros
    with pytest.raises(RuntimeError, match="overflow"):
        c.check()
    c._tensors["ctrl"].zero_()
    assert not out[0].any() and out[1].any()
    recorded(ValueError, lambda: ops.sparse_decode(x, 0, both + 2, q, 500, 8))
    recorded(ValueError, lambda: ops.sparse_decode(x, 0, both - 2, q, 500, 8))
    c._tensors["tables"][0, 0, 17] = c.max_blocks           # a corrupt table: not read
    recorded(AssertionError, lambda: ops.sparse_decode(x, 0, both, q, 500, 8))
    recorded(AssertionError, lambda: ops.sparse_decode(x, 0, both, q, 500, 40))
    for bad in (dict(budget=2, sink=2, recent=1), dict(budget=2, sink=0, recent=0), dict(budget=2, sink=-1)):
        with pytest.raises(ValueError):
            ops.sparse_decode(x, 0, both, q, 500, **bad)
    with pytest.raises(ValueError):
        ops.sparse_decode(x, 0, both[:1], q, 500, 8)
    with pytest.raises(TypeError):
        ops.sparse_decode(x, 0, both, q.float(), 500, 8)
    assert ops.sparse_decode(x, 0, both[:0], q[:0], 500, 8).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sparse_decode_of_every_page_is_dense_decode(dtype):
    from mentat_b200 import PagedKVCacheManager
    from mentat_b200.attention_backend import attn_decode, attn_decode_sparse
    g = torch.Generator(device="cuda").manual_seed(3)
    m = PagedKVCacheManager(1, 2, 128, max_blocks=200, device="cuda", dtype=TORCH_DT[dtype])
    with pytest.raises(RuntimeError, match="enable_page_index"):
        attn_decode_sparse(torch.zeros((0, 8, 128), device="cuda", dtype=m.dtype), *m.build_packed_kv([], 0)[:2], 8)
    m.enable_page_index()
    a = m.allocate_sequence()
    kv = torch.randn((530, 2, 128), generator=g, device="cuda").to(m.dtype)
    m.append_tokens(a, 0, kv, kv)
    kids = m.fork_sequences([a] * 3)
    q = torch.randn((4, 8, 128), generator=g, device="cuda").to(m.dtype)
    k, v, cu, mx = m.build_packed_kv([a] + kids, 0)
    dense, sparse = attn_decode(q, k, v, None, cu, mx, 4), attn_decode_sparse(q, k, v, 34)
    assert np.abs((dense.double() - sparse.double()).cpu().numpy()).max() <= 2 * tolerance(dtype, kv.double().cpu().numpy())


def test_index_is_kept_by_the_cache():
    """Appends of one and many tokens (plain and rotated), forks, copied tails, trims, compaction,
    recycled blocks: every full page of every sequence is indexed as if anew."""
    from mentat_b200 import PagedKVCacheManager, Rotary
    rng = np.random.default_rng(11)
    g = torch.Generator(device="cuda").manual_seed(4)
    m = PagedKVCacheManager(2, 2, 64, max_blocks=160, block_size=4, device="cuda", dtype=torch.bfloat16, strict=True)
    rot = Rotary(64)

    def rows(n):
        return torch.randn((n, 2, 64), generator=g, device="cuda").bfloat16()

    def check():
        m.check()
        for sid, s in m._sequences.items():
            for layer in range(2):
                full = s.num_tokens[layer] // 4
                tab = m.page_table(sid, layer)[:full]
                for b in tab:
                    bounds, exps = index_page(m.k_pools[layer][b].double().cpu().numpy())
                    np.testing.assert_array_equal(m.page_index.bounds[layer, b].cpu().numpy(), bounds)
                    np.testing.assert_array_equal(m.page_index.exps[layer, b].cpu().numpy(), exps)
    a = m.allocate_sequence()
    for layer in range(2):
        m.append_tokens(a, layer, rows(10), rows(10))
    m.enable_page_index()  # over what is there
    assert m.enable_page_index() is m.page_index
    check()
    b = m.allocate_sequence()
    for layer in range(2):
        m.append_tokens(a, layer, rows(7), rows(7))
        m.append_rotated(b, layer, rows(9), rows(9), rows(9), rot)
    check()
    live = [a, b] + m.fork_sequences([a, a, b])
    for step in range(30):
        for layer in range(2):
            if step % 2:
                m.append_tokens_batched(live, layer, rows(len(live)), rows(len(live)))
            else:
                m.append_rotated_batched(live, layer, rows(len(live)), rows(len(live)), rows(len(live)), rot)
        if step == 9:
            m.compact_sequences(live[:2], [np.arange(3, 20), np.arange(5)], rotary=rot)
            live += m.compact_sequences(live[2:3], [np.r_[0:4, 8:17]], into_new=True)
        if step == 17:
            m.trim_to_window(live[3], 9)
        if step % 8 == 5:
            gone = rng.permutation(live)[:2].tolist()
            m.free_sequences(gone)
            live = [s for s in live if s not in gone]
            live += m.fork_sequences([live[0], live[0]])
        if step % 6 == 5 or step in (9, 17):
            check()
    check()


def test_index_of_a_sequence_twice_in_a_batch():
    """A page that fills in the middle of a batch, under a repeated sequence, holds the bounds of its new keys."""
    from mentat_b200 import PagedKVCacheManager, Rotary
    m = PagedKVCacheManager(1, 2, 64, max_blocks=40, block_size=4, device="cuda", dtype=torch.bfloat16, max_seqs=32)
    g = torch.Generator(device="cuda").manual_seed(3)
    rot = Rotary(64)

    def rows(n):
        return torch.randn((n, 2, 64), generator=g, device="cuda").bfloat16()
    m.enable_page_index()
    for _ in range(2):  # the second time over blocks whose old bounds are in the index
        a, b = m.allocate_sequence(), m.allocate_sequence()
        m.append_tokens(a, 0, rows(2), rows(2))
        m.append_tokens_batched([a, b, a, a, b], 0, rows(5), rows(5))                       # a 5, b 2
        m.append_rotated_batched([b] + [a] * 8 + [b] * 7, 0, rows(16), rows(16), rows(16), rot)  # a 13, b 10
        for s in (a, b):
            st = m._sequences[s]
            for block in m._tables[0, st.slot, : st.num_tokens[0] // 4].tolist():
                bounds, e = index_page(m.k_pools[0][block].double().cpu().numpy())
                np.testing.assert_array_equal(m.page_index.bounds[0, block].cpu().numpy(), bounds)
                np.testing.assert_array_equal(m.page_index.exps[0, block].cpu().numpy(), e)
        m.free_sequences([a, b])
        for s in range(20):  # the ring comes round to the same blocks
            c = m.allocate_sequence()
            m.append_tokens(c, 0, rows(8), rows(8))
            m.free_sequence(c)
    m.check()


def test_captured_and_on_another_stream():
    from mentat_b200 import ops
    lens = [900, 70]
    c, x, q, tables = make(lens, 8, 2, 128, 16, "bf16", layers=1)
    slots = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    want = ops.sparse_decode(x, 0, slots, q, 900, 8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.sparse_decode(x, 0, slots, q, 900, 8)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = ops.sparse_decode(x, 0, slots, q, 900, 8)
    with torch.cuda.graph(g2):
        o2 = ops.sparse_decode(x, 0, slots.flip(0), q, 900, 12)
    c._tensors["ntok"][0, 0] = 850  # replays read the lengths of the time
    q.mul_(0.5)
    for _ in range(2):
        g1.replay()
        g2.replay()
    assert torch.equal(o1, ops.sparse_decode(x, 0, slots, q, 900, 8))
    assert torch.equal(o2, ops.sparse_decode(x, 0, slots.flip(0), q, 900, 12))


def test_steps_of_the_set_together():
    """Decode steps as they are run: rotated appends, forks, sparse attention, a freed branch, compaction,
    against the definitions over the cache's own rows."""
    from mentat_b200 import PagedKVCacheManager, Rotary
    from mentat_b200.attention_backend import attn_decode_sparse
    g = torch.Generator(device="cuda").manual_seed(6)
    m = PagedKVCacheManager(2, 2, 64, max_blocks=400, device="cuda", dtype=torch.bfloat16, strict=True)
    m.enable_page_index()
    rot = Rotary(64, base=5e5, scaling=dict(rope_type="linear", factor=2.0))

    def rows(n, h):
        return torch.randn((n, h, 64), generator=g, device="cuda").bfloat16()
    a = m.allocate_sequence()
    for layer in range(2):
        q = m.append_rotated(a, layer, rows(300, 8), rows(300, 2), rows(300, 2), rot)
        m.prefill_attention(a, layer, q)
    live = m.fork_sequences([a] * 3)
    m.free_sequences([a])
    for step in range(24):
        for layer in range(2):
            q = m.append_rotated_batched(live, layer, rows(len(live), 8), rows(len(live), 2), rows(len(live), 2), rot)
            k, v, _, _ = m.build_packed_kv(live, layer)
            out, pages = attn_decode_sparse(q, k, v, 7, sink=1, recent=2, return_pages=True)
            if step % 6 == 0:
                tabs = [m.page_table(s, layer) for s in live]
                vp = m.v_pools[layer].double().cpu().numpy()
                want, chosen = sparse_decode(q.double().cpu().numpy(), m.k_pools[layer].double().cpu().numpy(), vp, tabs,
                                             k.lens, 16, m.page_index.bounds[layer].cpu().numpy(),
                                             m.page_index.exps[layer].cpu().numpy(), 7, 1, 2)
                np.testing.assert_array_equal(pages.cpu().numpy(), chosen)
                assert np.abs(out.double().cpu().numpy() - want).max() <= tolerance("bf16", vp)
        if step == 7:
            live += m.fork_sequences(live[:1] * 2)
        if step == 11:
            m.free_sequences(live[1:3])
            del live[1:3]
        if step == 15:
            n = m.get_kv_length(live[0])
            m.compact_sequences(live[:1], [np.r_[0:16, n - 100:n]], rotary=rot)
            assert m.get_kv_length(live[0]) == 116
    m.free_sequences(live)
    assert m.get_stats()["blocks_used"] == 0


@pytest.mark.parametrize("mode", ["graphs", "padded", "static", "eager"])
def test_rollout_with_fused_rotary_and_all_pages(mode):
    """The golden fp32 trees again with rotated appends, and with a budget that covers every page."""
    import json
    import os
    from mentat_b200.rollout import TreeRollout
    from tests.golden.cases import ROLLOUT_CASES, rollout_model, rollout_prompts
    golden = json.load(open(os.path.join(os.path.dirname(__file__), "golden", "rollout.json")))
    kw = {"graphs": {}, "padded": dict(graph_bucket=4), "static": dict(cuda_graphs=False, static_decode=True),
          "eager": dict(cuda_graphs=False)}[mode]
    for name, c in sorted(ROLLOUT_CASES.items()):
        model = rollout_model(c, device="cuda")
        for sparse in (dict(), dict(sparse_budget=64, sparse_sink=2)):
            r = TreeRollout(model, eos_token_id=c["eos"], max_active_branches=c["max_active_branches"],
                            branching_factor=c["branching_factor"], max_new_tokens=c["max_new_tokens"], block_size=16,
                            max_blocks=4096, fused_rotary=True, **sparse, **kw)
            for got, want in zip(r.generate_many(rollout_prompts(c)), golden[name]):
                assert [x["token_ids"] for x in got] == [x["token_ids"] for x in want["results"]], name
                np.testing.assert_allclose([x["log_prob"] for x in got], [x["log_prob"] for x in want["results"]],
                                           rtol=1e-4, atol=1e-4)
            assert r.cache.get_stats()["blocks_used"] == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (10, 2, 64), (8, 1, 128), (16, 1, 64), (24, 2, 128)])
def test_weights_keep_more_bits_than_the_element_type(hq, hkv, d, dtype):
    """Off by the rounding of the output and 32-bit sums, not by weights rounded to the element type.

    Keys and queries have one channel, so the scores' products are exact.  A weight: the exponent |s| < 8 after the
    scale, its rounding and the difference from the maximum, 4 roundings of 8 2^-24 ln 2 < 2^-19.4; exp2 and at most 4
    factors between partials, 2^-21 each; 20 tokens' sums 20 2^-24, and as much again in the product unit.  Below
    2^-17.5, in numerator and denominator: 2^-16.5 of sum w |v|.  What two parts of a weight leave: (eps / 2)^2."""
    from mentat_b200 import ops
    lens = [1, 2, 5, 17, 20]
    c, x, q, tables = make(lens, hq, hkv, d, 16, dtype, layers=1)
    k, v = c._tensors["k_pool"], c._tensors["v_pool"]
    k[..., 1:] = 0
    q[..., 1:] = 0
    k.clamp_(-2, 2)
    q.clamp_(-2, 2)
    slots = torch.arange(len(lens), dtype=torch.int32, device="cuda")
    got = ops.sparse_decode(x, 0, slots, q, 20, 4, scale=1.0).double().cpu().numpy()
    c.check()
    half = torch.finfo(c.dtype).eps / 2
    kd, vd, qd = (t.double().cpu().numpy() for t in (k[0], v[0], q))
    for i, n in enumerate(lens):
        rows = tables[0, i][np.arange(n) // 16], np.arange(n) % 16
        for h in range(hq):
            s = kd[rows][:, h // (hq // hkv), 0] * qd[i, h, 0]
            w = np.exp(s - s.max())
            w /= w.sum()
            vals = vd[rows][:, h // (hq // hkv)]
            want, size = w @ vals, w @ np.abs(vals)
            wide = (half * half + 2.0 ** -16.5) * size
            tol = wide + half * (np.abs(want) + wide) + (2.0 ** -25 if dtype == "f16" else 0.0)
            off = np.abs(got[i, h] - want) - tol
            assert off.max() <= 0, (n, h, off.max(), tol[off.argmax()])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq", [8, 16])
def test_infinite_values_show_as_such(hq, dtype):
    """A value of infinity gives infinity in its channel, whatever part of its weight is 0; behind the last token it
    is not seen."""
    from mentat_b200 import ops
    lens = [1, 20]
    c, x, q, tables = make(lens, hq, 1, 64, 16, dtype, layers=1)
    v = c._tensors["v_pool"]
    v[0, int(tables[0, 0, 0]), 0, 0, 3] = float("inf")
    v[0, int(tables[0, 0, 0]), 5, 0, 4] = float("inf")          # no token of the sequence
    v[0, int(tables[0, 1, 1]), 2, 0, 60] = -float("inf")
    slots = torch.arange(2, dtype=torch.int32, device="cuda")
    out = ops.sparse_decode(x, 0, slots, q, 20, 4)
    assert (out[0, :, 3] == float("inf")).all() and (out[1, :, 60] == -float("inf")).all()
    out[0, :, 3] = out[1, :, 60] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("page", [0, 300, 605, 609])
def test_large_batches_choose_unreadable_pages_last(page):
    """A page whose table entry is outside the pool, even one that is always chosen otherwise, has the key that it
    has where one launch does it all: the sequence alone chooses the same pages, and not this one."""
    from mentat_b200 import ops
    n, lens = 80, [610 * 16] * 80  # 610 pages for each of 160 heads: scores and choice have launches of their own
    c, x, q, tables = make(lens, 4, 2, 64, 16, "bf16", layers=1, shared=600)
    c._tensors["tables"][0, 11, page] = c.max_blocks
    every = torch.arange(n, dtype=torch.int32, device="cuda")
    assert x.workspace_bytes(n, 610 * 16, 12) > 0 and x.workspace_bytes(1, 610 * 16, 12) == 0
    _, many = ops.sparse_decode(x, 0, every, q, 610 * 16, 12, return_pages=True)
    with pytest.raises(AssertionError):
        c.check()
    c._tensors["ctrl"].zero_()
    _, one = ops.sparse_decode(x, 0, every[11:12], q[11:12], 610 * 16, 12, return_pages=True)
    assert torch.equal(many[11:12], one)
    assert (one >= 0).all() and not (one == page).any()


def test_large_batches_of_trees():
    """Batches that have launches of their own for the scores and the choice: rows that share all, some or none of
    their pages, rows without a choice and an empty one among them, groups that do not divide the columns."""
    rng = np.random.default_rng(6)
    for hq, hkv, d, n in ((24, 8, 64, 41), (10, 2, 128, 90)):
        lens = [int(v) for v in rng.integers(1, 9900, n)]
        lens[3], lens[5], lens[n - 1] = 0, 17, 9897
        c, x, q, tables = make(lens, hq, hkv, d, 16, "bf16", layers=1, shared=400)
        assert x.workspace_bytes(n, 9897, 8) > 0
        run_and_check(c, x, q, tables, lens, 8, 1, 2, "bf16", layer=0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 40])
def test_bounds_of_the_smallest_keys_keep_their_side(d, dtype):
    """Keys of 2^-133 beside one of 2^40 or 2^57: in units of the page they underflow, and their bounds are still on the
    outer side of them."""
    from mentat_b200 import KVCacheView, PageIndex, ops
    k = torch.zeros((1, 3, 16, 1, d), dtype=TORCH_DT[dtype], device="cuda")
    k[0, 0, 3, 0, 0], k[0, 1, 3, 0, 0] = 2.0 ** 40, -(2.0 ** 57)
    k[0, :, 1, 0, 1], k[0, :, 1, 0, 2], k[0, :, :, 0, 3] = 2.0 ** -133, -(2.0 ** -133), 2.0 ** -133
    x = PageIndex(KVCacheView(k, torch.zeros_like(k)))
    ops.page_index(x, 0, torch.arange(3, dtype=torch.int32, device="cuda"))
    for b in range(3):
        bounds, exps = index_page(k[0, b].double().cpu().numpy())
        np.testing.assert_array_equal(x.bounds[0, b].cpu().numpy(), bounds)
        np.testing.assert_array_equal(x.exps[0, b].cpu().numpy(), exps)
