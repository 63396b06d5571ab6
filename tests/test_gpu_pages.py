"""Batched fork, batched free, compaction and rotated appends of the paged cache against the
single calls' oracle (``oracle.allocator``) and the compaction's definition (``oracle.cache_ops``):
tables, reference counts and the free list's order bit-exact."""

import numpy as np
import pytest
import torch

from oracle.allocator import OraclePagedKV
from oracle.cache_ops import compact, turn, turn_tolerance
from tests.gpu_util import TORCH_DT, round_np

pytestmark = pytest.mark.gpu


def pair(L=2, hkv=2, d=64, pool=300, bs=4, dtype="bf16", seed=0, **kw):
    from mentat_b200 import PagedKVCacheManager
    order = np.random.default_rng(seed).permutation(pool).tolist()
    m = PagedKVCacheManager(L, hkv, d, max_blocks=pool, block_size=bs, device="cuda", dtype=TORCH_DT[dtype],
                            free_order=order, **{"max_seqs": 64, "strict": True, **kw})
    o = OraclePagedKV(L, hkv, d, pool, bs, order=order, elem_bytes=m.dtype_size)
    return m, o


def fill(m, o, sid, n, rng, dtype="bf16"):
    for layer in range(m.num_layers):
        k, v = (round_np(rng.standard_normal((n, m.num_key_value_heads, m.head_dim), dtype=np.float32), dtype)
                for _ in range(2))
        m.append_tokens(sid, layer, *(torch.from_numpy(t).cuda().to(m.dtype) for t in (k, v)))
        o.append_tokens(sid, layer, k, v)


def start(m, o, lens, rng, dtype="bf16"):
    ids = [m.allocate_sequence() for _ in lens]
    assert ids == [o.allocate_sequence() for _ in lens]
    for s, n in zip(ids, lens):
        if n:
            fill(m, o, s, n, rng, dtype)
    return ids


def same(m, o, tol=None):
    """Allocator and tables equal, cached rows equal (or within ``tol(want)``)."""
    snap, want = m.sequence_snapshot(), o.snapshot()
    assert snap == want["seqs"]
    assert m.allocator.refcounts == want["refcounts"]
    assert m.allocator.free_list() == want["free"]
    assert m.allocator.peak_used == want["peak"]
    for sid, s in m._sequences.items():  # the host's mirror
        w = o._sequences[sid]
        assert s.num_tokens == w.num_tokens and s.tokens_in_last_block == w.tokens_in_last_block
        assert s.num_blocks == [len(t) for t in w.page_table]
    ids = sorted(m._sequences)
    for layer in range(m.num_layers):
        pk, pv, _, _ = m.packed_kv_tensors(ids, layer)
        ok, ov, _, _ = o.build_packed_kv(ids, layer)
        np.testing.assert_array_equal(pv.float().cpu().numpy(), ov)
        if tol is None:
            np.testing.assert_array_equal(pk.float().cpu().numpy(), ok)
        else:
            assert np.all(np.abs(pk.double().cpu().numpy() - ok) <= tol(ok))


@pytest.mark.parametrize("seed", range(4))
def test_batched_fork_and_free_are_the_single_calls(seed):
    rng = np.random.default_rng(seed)
    m, o = pair(L=int(rng.integers(1, 4)), pool=2000, seed=seed)
    live = start(m, o, [0, 1, 3, 4, 5, 40], rng)
    for step in range(12):
        parents = rng.choice(live, rng.integers(1, 9)).tolist()  # a parent may have several children
        if len(m._free_slots) < len(parents):
            parents = []
        kids = m.fork_sequences(parents)
        assert kids == [o.fork_sequence(p) for p in parents]
        live += kids
        if step % 3 == 1:
            for layer in range(m.num_layers):
                k = round_np(rng.standard_normal((len(live), 2, 64), dtype=np.float32), "bf16")
                t = torch.from_numpy(k).cuda().bfloat16()
                m.append_tokens_batched(live, layer, t, t)
                o.append_tokens_batched(live, layer, k, k)
        gone = rng.permutation(live)[: rng.integers(0, len(live))].tolist()
        m.free_sequences(gone)
        for s in gone:
            o.free_sequence(s)
        live = [s for s in live if s not in gone] or start(m, o, [7], rng)
        same(m, o)
    m.free_sequences(live)
    for s in live:
        o.free_sequence(s)
    same(m, o)
    assert m.get_stats() == o.get_stats() and m.get_stats()["blocks_used"] == 0


def test_large_batches_of_shared_pages():
    """Many sequences over one prefix, rows of several chunks, more sequences than one launch takes."""
    rng = np.random.default_rng(1)
    m, o = pair(L=3, hkv=1, d=2, pool=8000, bs=2, dtype="f32", max_seqs=1200)
    (root,) = start(m, o, [1403], rng, "f32")
    kids = m.fork_sequences([root] * 1100)
    assert kids == [o.fork_sequence(root) for _ in range(1100)]
    assert m.allocator.refcounts == o.allocator.refcounts
    order = rng.permutation(kids + [root]).tolist()
    last = order.pop()
    m.free_sequences(order)
    for s in order:
        o.free_sequence(s)
    same(m, o)
    m.free_sequences([last])
    o.free_sequence(last)
    same(m, o)


def test_large_compaction_in_place():
    """More table entries than one cluster releases; pages at the front shared by all sequences."""
    rng = np.random.default_rng(11)
    m, o = pair(L=3, hkv=1, d=2, pool=40000, bs=2, dtype="f32")
    (root,) = start(m, o, [463], rng, "f32")
    ids = [root] + m.fork_sequences([root] * 59)
    for _ in range(59):
        o.fork_sequence(root)
    keep = [np.r_[0:100, 100 + np.sort(rng.permutation(363)[: int(rng.integers(0, 363))])] for _ in ids]
    keep[7], keep[8], keep[9] = np.arange(463), np.arange(0), np.arange(462)
    m.compact_sequences(ids, keep)
    compact(o, ids, keep)
    same(m, o)
    m.free_sequences(ids)
    for s in ids:
        o.free_sequence(s)
    same(m, o)


@pytest.mark.parametrize("dtype,hkv,d,bs", [("f32", 8, 128, 32), ("bf16", 1, 64, 24), ("f16", 16, 256, 16), ("f32", 64, 256, 2),
                                            ("bf16", 8, 128, 1), ("bf16", 3, 8, 7), ("f16", 1, 8, 40)])
def test_compaction_of_all_row_sizes(dtype, hkv, d, bs):
    """Rows of 16 bytes to 64 KB (one token to a stage of the copies, or too long for them), with keys turned too."""
    from mentat_b200 import Rotary
    rng = np.random.default_rng(12)
    m, o = pair(L=1, hkv=hkv, d=d, bs=bs, pool=400, dtype=dtype)
    ids = start(m, o, [3, 71, 100], rng, dtype)
    keep = [[2, 0], np.r_[0:2, 30:71], np.sort(rng.permutation(100)[:57])]
    new = m.compact_sequences(ids, keep, into_new=True)
    assert new == compact(o, ids, keep, into_new=True)
    same(m, o)
    rot = Rotary(d)
    f, eps = rot.inv_freq.cpu().numpy(), torch.finfo(m.dtype).eps
    m.compact_sequences(ids, keep, rotary=rot)
    compact(o, ids, keep, turn_keys=lambda k, shift: turn(k, shift, f))
    same(m, o, lambda want: 1.5 * turn_tolerance(want, f, eps)(want) + (2.0 ** -25 if dtype == "f16" else 0))


def test_sizes_are_only_hints():
    from mentat_b200 import ops
    rng = np.random.default_rng(13)
    m, o = pair(L=2, pool=2000, bs=2)
    a, b = ids = start(m, o, [431, 700], rng)
    slots = torch.tensor([m._sequences[s].slot for s in ids], dtype=torch.int32, device="cuda")
    keep = [np.arange(1, 431, 2), np.arange(700)[::-1][:600]]
    flat = torch.from_numpy(np.concatenate(keep)).int().cuda()
    ops.compact_pages(m, slots, None, flat, torch.tensor([0, 215, 815], dtype=torch.int32, device="cuda"), 1, max_blocks=1)
    compact(o, ids, keep)
    for layer in range(2):
        for s in ids:
            st, w = m._sequences[s], o._sequences[s]
            st.num_tokens[layer], st.num_blocks[layer] = w.num_tokens[layer], len(w.page_table[layer])
            st.tokens_in_last_block[layer] = w.tokens_in_last_block[layer]
    same(m, o)
    for hint in (0, 1 << 30):
        (c,) = m.fork_sequences([a])
        assert c == o.fork_sequence(a)
        ops.free_pages(m, torch.tensor([m._sequences[c].slot], dtype=torch.int32, device="cuda"), max_blocks=hint)
        m.free_sequence(c)
        o.free_sequence(c)
        same(m, o)


def test_batched_refusals_change_nothing():
    rng = np.random.default_rng(2)
    m, o = pair(max_seqs=5)
    a, b, c = start(m, o, [9, 4, 0], rng)
    for call in (lambda: m.fork_sequences([a, 99]), lambda: m.free_sequences([a, 99]), lambda: m.free_sequences([a, b, a]),
                 lambda: m.compact_sequences([a, a], [[0], [1]]), lambda: m.compact_sequences([99], [[0]])):
        with pytest.raises(KeyError):
            call()
    with pytest.raises(RuntimeError, match="out of sequence slots"):
        m.fork_sequences([a, a, b])
    with pytest.raises(RuntimeError, match="out of sequence slots"):
        m.compact_sequences([a, a, b], [[0]] * 3, into_new=True)
    for keep in ([9], [-1], [[0], [9]], [[0, 1], [3, -2]]):
        with pytest.raises(IndexError):
            m.compact_sequences([a], [keep])
    with pytest.raises(ValueError):
        m.compact_sequences([a], [[[0], [1], [2]]])
    with pytest.raises(ValueError):
        m.compact_sequences([a, b], [[0]])
    with pytest.raises(TypeError):
        m.compact_sequences([a], [[0.5]])
    for mask in (torch.ones(9, dtype=torch.bool, device="cuda"), torch.zeros(3, device="cuda")):
        with pytest.raises(TypeError):
            m.compact_sequences([a], [mask])
    assert m.get_kv_length(a) == 9
    assert m.fork_sequences([]) == [] and m.free_sequences([]) is None and m.compact_sequences([], []) is None
    same(m, o)


def test_device_refusals_change_nothing():
    """What only the device can see: slots out of range, twice or in use, positions outside, too few
    blocks.  Each is recorded, and nothing has changed."""
    from mentat_b200 import ops
    rng = np.random.default_rng(3)
    m, o = pair(L=1, pool=12, strict=False)
    a, b = start(m, o, [21, 5], rng)  # 6 + 2 of 12 blocks
    i32 = dict(dtype=torch.int32, device="cuda")
    sa, sb = m._sequences[a].slot, m._sequences[b].slot
    free_slot = m._free_slots[-1]

    def ids(*v):
        return torch.tensor(v, **i32)
    cu1, cu2 = ids(0, 3), ids(0, 3, 5)
    bad = [
        (ValueError, lambda: ops.free_pages(m, ids(sa, sb, sa))),
        (ValueError, lambda: ops.free_pages(m, ids(sa, 64))),
        (ValueError, lambda: ops.free_pages(m, ids(-1))),
        (ValueError, lambda: ops.fork_pages(m, ids(sa, sa), ids(free_slot, free_slot))),
        (ValueError, lambda: ops.fork_pages(m, ids(sa, sb), ids(free_slot, sa))),
        (ValueError, lambda: ops.fork_pages(m, ids(64), ids(free_slot))),
        (ValueError, lambda: ops.fork_pages(m, ids(sa), ids(-5))),
        (ValueError, lambda: ops.compact_pages(m, ids(sa, sa), None, ids(0, 1, 2, 3, 4), cu2, 3)),
        (ValueError, lambda: ops.compact_pages(m, ids(sa), ids(sb), ids(0, 1, 2), cu1, 3)),
        (ValueError, lambda: ops.compact_pages(m, ids(sa), ids(sa), ids(0, 1, 2), cu1, 3)),
        (IndexError, lambda: ops.compact_pages(m, ids(sa, sb), None, ids(0, 1, 2, 4, 5), cu2, 3)),
        (IndexError, lambda: ops.compact_pages(m, ids(sa), None, ids(-1, 1, 2), cu1, 3)),
        # lists that leave keep, or end before they begin
        (IndexError, lambda: ops.compact_pages(m, ids(sa), None, ids(0, 1, 2), ids(0, 4), 3)),
        (IndexError, lambda: ops.compact_pages(m, ids(sa, sb), None, ids(0, 1, 2, 0, 1), ids(0, 1 << 30, 5), 3)),
        (IndexError, lambda: ops.compact_pages(m, ids(sa, sb), None, ids(0, 1, 2, 0, 1), ids(-3, 3, 5), 3)),
        (IndexError, lambda: ops.compact_pages(m, ids(sa, sb), ids(free_slot, 50), ids(0, 1, 2, 0, 1), ids(0, 3, 2), 3)),
        (RuntimeError, lambda: ops.compact_pages(m, ids(sa), ids(free_slot), torch.arange(20, 3, -1, **i32), ids(0, 17), 17)),
    ]
    for k, (exc, call) in enumerate(bad):
        call()
        with pytest.raises(exc):
            m.check()
        m.clear_error()
        try:
            same(m, o)
        except AssertionError as e:
            raise AssertionError(f"refusal {k} changed the cache") from e
    # a call after an error that nobody has cleared changes nothing either
    ops.free_pages(m, ids(-1))
    ops.free_pages(m, ids(sa))
    ops.fork_pages(m, ids(sa), ids(free_slot))
    m.clear_error()
    same(m, o)


KEEPS = {
    "all": lambda n, r: np.arange(n), "none": lambda n, r: np.arange(0), "front": lambda n, r: np.arange(n // 2),
    "window": lambda n, r: np.concatenate([np.arange(min(3, n)), np.arange(max(min(3, n), n - 7), n)]),
    "scattered": lambda n, r: np.sort(r.permutation(n)[: (n + 1) // 2]), "reversed": lambda n, r: np.arange(n)[::-1],
    "repeated": lambda n, r: np.repeat(np.arange(n), 2)[: n + 3], "last": lambda n, r: np.arange(n - 1, n),
}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", sorted(KEEPS) + ["mixed"])
@pytest.mark.parametrize("into_new", [False, True], ids=["in place", "new"])
def test_compaction(kind, into_new, dtype):
    rng = np.random.default_rng(4)
    m, o = pair(L=2, pool=400, dtype=dtype)
    ids = start(m, o, [1, 3, 4, 5, 8, 33, 50], rng, dtype)
    ids += m.fork_sequences([ids[5], ids[6]])  # shared pages, one tail full and one partly filled
    for s in (ids[5], ids[6]):
        o.fork_sequence(s)
    lens = [m.get_kv_length(s) for s in ids]
    pick = sorted(KEEPS)
    keep = [KEEPS[pick[i % len(pick)] if kind == "mixed" else kind](n, rng) for i, n in enumerate(lens)]
    if kind == "mixed":  # a choice of its own in each layer
        keep[6] = np.stack([keep[6], np.sort(rng.permutation(lens[6])[: len(keep[6])])])
    as_given = [k if i % 2 else torch.from_numpy(k.copy()) for i, k in enumerate(keep)]
    new = m.compact_sequences(ids, as_given, into_new=into_new)
    assert (new or []) == compact(o, ids, keep, into_new=into_new)
    same(m, o)
    # the cache goes on: every sequence appends (copying shared tails), then all are freed
    every = sorted(m._sequences)
    for layer in range(2):
        k = round_np(rng.standard_normal((len(every), 2, 64), dtype=np.float32), dtype)
        t = torch.from_numpy(k).cuda().to(m.dtype)
        m.append_tokens_batched(every, layer, t, t)
        o.append_tokens_batched(every, layer, k, k)
    same(m, o)
    m.free_sequences(every)
    for s in every:
        o.free_sequence(s)
    same(m, o)


@pytest.mark.parametrize("dtype,d,bs,rd,il", [("bf16", 64, 16, 64, False), ("f32", 128, 4, 64, True), ("f16", 37, 5, 20, False)])
def test_compaction_turns_keys(dtype, d, bs, rd, il):
    from mentat_b200 import Rotary
    rng = np.random.default_rng(6)
    m, o = pair(L=2, d=d, bs=bs, pool=200, dtype=dtype)
    ids = start(m, o, [1, 70, 129], rng, dtype)
    rot = Rotary(d, rotary_dim=rd, interleaved=il, attention_scaling=1.7)  # the factor is not applied again
    f = rot.inv_freq.cpu().numpy()
    keep = [[0], np.r_[0:4, 30:70], np.sort(rng.permutation(129)[:61])]
    m.compact_sequences(ids, keep, rotary=rot)
    compact(o, ids, keep, turn_keys=lambda k, shift: turn(k, shift, f, interleaved=il))
    eps = torch.finfo(m.dtype).eps
    # the tolerance of a turn, from rows of the turned keys (a pair's |x1| + |x2| is at most
    # sqrt(2) times its turned one's); fp16 steps below 2^-14 are 2^-24 wide
    same(m, o, lambda want: 1.5 * turn_tolerance(want, f, eps, interleaved=il)(want) + (2.0 ** -25 if dtype == "f16" else 0))


def test_compaction_of_device_positions_on_another_stream():
    rng = np.random.default_rng(8)
    m, o = pair()
    ids = start(m, o, [40, 17], rng)
    keep = [torch.tensor([1, 2, 39], device="cuda"), torch.tensor([[0, 16], [3, 4]], device="cuda", dtype=torch.int32)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.compact_sequences(ids, keep)
    torch.cuda.current_stream().wait_stream(s)
    compact(o, ids, [k.cpu().numpy() for k in keep])
    same(m, o)


def test_captured_page_operators():
    """Forks, a compaction into new slots, one in place and releases in one graph, replayed: the state that the
    same calls leave one after another."""
    from mentat_b200 import ops
    rng = np.random.default_rng(14)
    m, o = pair(L=2, pool=400)
    a, b = ids = start(m, o, [41, 18], rng)
    i32 = dict(dtype=torch.int32, device="cuda")
    slots = torch.tensor([m._sequences[s].slot for s in ids], **i32)
    kids = torch.tensor(m._free_slots[-4:][::-1], **i32)  # the slots that the next sequences get
    keep = [np.r_[0:4, 9:30], np.r_[5:18]]
    flat = torch.from_numpy(np.concatenate(keep)).to(**i32)
    cu = torch.tensor([0, 25, 38], **i32)

    def step():
        ops.fork_pages(m, slots, kids[:2])
        ops.compact_pages(m, slots, kids[2:], flat, cu, 25)
        ops.free_pages(m, kids[:2])
        ops.free_pages(m, kids[2:])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(3):
        g.replay()
        fork = [o.fork_sequence(s) for s in ids]
        new = compact(o, ids, keep, into_new=True)
        for s in fork + new:
            o.free_sequence(s)
    same(m, o)
    # in place: two graphs over one cache
    g2 = torch.cuda.CUDAGraph()
    back, cu2 = torch.arange(12, -1, -1, **i32), torch.tensor([0, 13], **i32)
    with torch.cuda.graph(g2):
        ops.compact_pages(m, slots[1:], None, back, cu2, 13)
    for graph in (g2, g, g2):
        if graph is g:  # what g keeps of b: its positions 0 .. 12
            flat[25:] = torch.arange(13, **i32)
            keep[1] = np.arange(13)
            g.replay()
            fork = [o.fork_sequence(s) for s in ids]
            for s in fork + compact(o, ids, keep, into_new=True):
                o.free_sequence(s)
        else:
            g2.replay()
            compact(o, [b], [np.arange(13)[::-1]])
        for layer in range(2):
            st, w = m._sequences[b], o._sequences[b]
            st.num_tokens[layer], st.num_blocks[layer] = w.num_tokens[layer], len(w.page_table[layer])
            st.tokens_in_last_block[layer] = w.tokens_in_last_block[layer]
        same(m, o)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,rd,il,bs", [(64, 64, False, 4), (128, 32, True, 16), (38, 10, False, 3)])
def test_rotated_appends(dtype, d, rd, il, bs):
    """append_rotated and append_rotated_batched: append_tokens and append_tokens_batched of turned
    keys, over copied tails, a repeated sequence in a batch, and positions of the caller's."""
    from mentat_b200 import Rotary
    rng = np.random.default_rng(9)
    m, o = pair(L=2, hkv=2, d=d, pool=200, bs=bs, dtype=dtype)
    rot = Rotary(d, rotary_dim=rd, interleaved=il, base=1e4)
    f, eps = rot.inv_freq.cpu().numpy(), torch.finfo(m.dtype).eps
    a = m.allocate_sequence()
    o.allocate_sequence()

    def rows(n, h):
        x = round_np(rng.standard_normal((n, h, d), dtype=np.float32), dtype)
        return x, torch.from_numpy(x).cuda().to(m.dtype)

    def check_q(got, x, pos):
        want = turn(x, pos, f, interleaved=il)
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= turn_tolerance(x, f, eps, interleaved=il)(want))
    for n, first in ((5, 0), (7, 5), (1, 12)):
        for layer in range(2):
            (q, tq), (k, tk), (v, tv) = rows(n, 6), rows(n, 2), rows(n, 2)
            pos = np.arange(first, first + n)
            if layer:
                check_q(m.append_rotated(a, layer, tq, tk, tv, rot), q, pos)
            else:
                assert m.append_rotated(a, layer, None, tk, tv, rot, positions=torch.from_numpy(pos + 900).cuda()) is None
                pos = pos + 900
            o.append_tokens(a, layer, turn(k, pos, f, interleaved=il), v)
    kids = m.fork_sequences([a, a, a])
    assert kids == [o.fork_sequence(a) for _ in range(3)]
    for step in range(bs + 2):
        batch = [a] + kids if step != 3 else [a, kids[1], a, kids[1]]
        for layer in range(2):
            (q, tq), (k, tk), (v, tv) = rows(4, 6), rows(4, 2), rows(4, 2)
            seen, pos = {}, []
            for s in batch:
                seen[s] = seen.get(s, 0) + 1
                pos.append(o._sequences[s].num_tokens[layer] + seen[s] - 1)
            check_q(m.append_rotated_batched(batch, layer, tq, tk, tv, rot), q, pos)
            o.append_tokens_batched(batch, layer, turn(k, pos, f, interleaved=il), v)
    same(m, o, lambda want: 1.5 * turn_tolerance(want, f, eps, interleaved=il)(want))


def test_failed_batches_leave_no_sequence(monkeypatch):
    """A call that fails after its new sequences have slots (another model's rotary, a launch that is refused, too few
    blocks) leaves the host's mirror, the slots and the device as they were, whatever part of it had run."""
    from mentat_b200 import Rotary, ops
    rng = np.random.default_rng(21)
    m, o = pair(L=2, d=64, pool=40, max_seqs=9)
    a, b = start(m, o, [33, 9], rng)  # 24 of 40 blocks
    slots = list(m._free_slots)

    def unchanged(exc, call, **kw):
        with pytest.raises(exc, **kw):
            call()
        m.clear_error()
        assert m._free_slots == slots and sorted(m._sequences) == [a, b]
        same(m, o)
    for new in (False, True):
        unchanged(ValueError, lambda: m.compact_sequences([a], [[1, 2]], rotary=Rotary(128), into_new=new), match="heads of 128")
    # 17 fresh blocks a layer do not fit; nor, in the second call, does what the first one's chunk left
    unchanged(RuntimeError, lambda: m.compact_sequences([a, a], [list(range(32, 0, -1))] * 2, into_new=True), match="out of blocks")

    def refuse_at(name, k):
        real, calls = getattr(ops, name), []

        def call(*args, **kw):
            calls.append(0)
            if len(calls) == k:
                raise RuntimeError("refused on the host")
            return real(*args, **kw)
        monkeypatch.setattr(ops, name, call)
        return real
    monkeypatch.setattr(ops, "MAX_SEQS_PER_PAGES_CALL", 2)
    for k in (1, 2):
        real = refuse_at("fork_pages", k)
        with pytest.raises(RuntimeError, match="refused"):
            m.fork_sequences([a, b, a, b])
        monkeypatch.setattr(ops, "fork_pages", real)
        assert sorted(m._free_slots) == sorted(slots) and sorted(m._sequences) == [a, b]
        same(m, o)  # (forks and their releases leave the free list as it was)
    slots = list(m._free_slots)
    for new in (False, True):
        real = refuse_at("compact_pages", 1)
        unchanged(RuntimeError, lambda: m.compact_sequences([a], [[1, 2]], into_new=new), match="refused")
        monkeypatch.setattr(ops, "compact_pages", real)
    # in place, the second part refused: the first is compacted, on the host too
    real = refuse_at("compact_pages", 2)
    c = m.allocate_sequence()
    assert c > b
    while o.allocate_sequence() < c:  # the ids that failed calls used up
        pass
    for sid in [s for s in o._sequences if s not in (a, b, c)]:
        o.free_sequence(sid)
    with pytest.raises(RuntimeError, match="refused"):
        m.compact_sequences([a, b, c], [[3, 2, 1], [8], []])
    monkeypatch.setattr(ops, "compact_pages", real)
    compact(o, [a, b], [np.array([3, 2, 1]), np.array([8])])
    same(m, o)
    # and what succeeds in several parts
    kids = m.fork_sequences([a, b, a])
    m.free_sequences([kids[2], kids[0], kids[1]])
    same(m, o)


def test_fork_into_a_slot_in_use_changes_nothing():
    """A child that has pages, one that has tokens in one layer alone, among children that are empty: recorded, and no
    table, count or child of the batch has changed."""
    from mentat_b200 import ops
    rng = np.random.default_rng(22)
    m, o = pair(L=3, pool=400, max_seqs=300, strict=False)
    a, b = start(m, o, [45, 7], rng)
    c = m.allocate_sequence()
    assert c == o.allocate_sequence()
    k, v = (round_np(rng.standard_normal((2, 2, 64), dtype=np.float32), "bf16") for _ in range(2))
    m.append_tokens(c, 2, *(torch.from_numpy(t).cuda().to(m.dtype) for t in (k, v)))  # its last layer alone
    o.append_tokens(c, 2, k, v)
    sa, sb, sc = (m._sequences[s].slot for s in (a, b, c))
    empty = m._free_slots[::-1]
    for used in (sb, sc):
        for n, at in ((1, 0), (9, 8), (200, 77)):
            kids = empty[:n]
            kids[at] = used
            ops.fork_pages(m, *(torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([sa] * n, kids)))
            with pytest.raises(ValueError, match=f"slot {used} "):
                m.check()
            m.clear_error()
            assert not m._nblocks[:, empty].any() and not m._ntok[:, empty].any()
            same(m, o)
    # the slots that were empty take the same batch
    n = 200
    ops.fork_pages(m, *(torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([sa] * n, empty[:n])))
    ops.free_pages(m, torch.tensor(empty[:n], dtype=torch.int32, device="cuda"))
    m.check()
    same(m, o)


def test_slots_freed_after_an_error_are_empty_when_it_is_cleared():
    """A free after an error does nothing on the device; clearing the error makes up for it, so the slot can be forked
    into and no page is lost."""
    rng = np.random.default_rng(23)
    m, o = pair(L=2, pool=60, strict=False)
    a, b, c = start(m, o, [21, 9, 13], rng)
    kid = m.fork_sequence(a)
    assert kid == o.fork_sequence(a)
    from mentat_b200 import ops
    ops.free_pages(m, torch.tensor([-1], dtype=torch.int32, device="cuda"))
    m.free_sequence(b)
    m.free_sequences([kid, c])
    with pytest.raises(ValueError):
        m.check()
    m.clear_error()
    m.check()
    for s in (c, kid, b):  # the order in which the free slots were left
        o.free_sequence(s)
    assert m.allocator.refcounts == o.snapshot()["refcounts"]
    assert sorted(m.allocator.free_list()) == sorted(o.snapshot()["free"])
    assert not m._nblocks[:, m._free_slots].any()
    assert sorted(m.fork_sequences([a, a, a])) == sorted(o.fork_sequence(a) for _ in range(3))
    m.check()
    assert m.allocator.refcounts == o.snapshot()["refcounts"]


@pytest.mark.parametrize("together", [1, 600], ids=["one", "many"])  # one cluster's work, and launches of their own
def test_lengths_beyond_the_table_are_recorded(together):
    """Counters of a caller's view that say more than its tables have room for, in the very last row: recorded, and no
    entry behind the table is read.  A fork and a compaction change nothing; a free releases what the table holds."""
    from mentat_b200 import KVCacheView, ops
    L, S, cap, bs, pool = 2, 600, 4, 4, 32
    i32 = dict(dtype=torch.int32, device="cuda")
    kv = torch.randn((L, pool, bs, 1, 64), device="cuda")
    tables = torch.full((L, S, cap), -1, **i32)
    tables[:, S - 1] = torch.arange(2 * cap, **i32).view(L, cap)
    nblocks, ntok, tail = (torch.zeros((L, S), **i32) for _ in range(3))
    nblocks[:, S - 1], ntok[:, S - 1], tail[:, S - 1] = cap, cap * bs, bs
    refs = torch.zeros(pool, **i32)
    refs[: 2 * cap] = 1
    ring = torch.arange(pool, **i32)
    ctrl = torch.zeros(16, dtype=torch.int64, device="cuda")
    ctrl[0], ctrl[1] = 2 * cap, pool  # what follows the blocks in use is free
    c = KVCacheView(kv, kv.clone(), tables, ntok, nblocks=nblocks, tail=tail, refcounts=refs, free_ring=ring, ctrl=ctrl)
    last, other = (torch.tensor([x], **i32) for x in (S - 1, 0))

    def recorded(call, *unchanged):
        before = [t.clone() for t in unchanged]
        call()
        with pytest.raises(RuntimeError, match=f"table overflow .slot {S - 1}"):
            c.check()
        ctrl[3:5] = 0
        for t, w in zip(unchanged, before):
            assert torch.equal(t, w)
    state = (tables, nblocks, ntok, tail, refs, ring, ctrl, kv)
    keep, cu = torch.arange(15, -1, -1, **i32), torch.tensor([0, 16], **i32)  # positions that the table holds
    beyond = torch.stack([keep, keep + 25])                                    # and that the last layer claims to hold
    nblocks[1, S - 1] = cap + 5
    recorded(lambda: ops.fork_pages(c, last, other), *state)
    for dst in (None, other):
        recorded(lambda: ops.compact_pages(c, last, dst, keep, cu, 16), *state)
    nblocks[1, S - 1] = cap
    ntok[1, S - 1] = 50
    recorded(lambda: ops.fork_pages(c, last, other), *state)
    for dst in (None, other):
        for k in (keep, beyond):
            recorded(lambda: ops.compact_pages(c, last, dst, k, cu, 16), *state)
    ntok[1, S - 1] = cap * bs
    nblocks[1, S - 1] = 1 << 30
    recorded(lambda: ops.free_pages(c, torch.arange(S - together, S, **i32)), tables, ring[2 * cap:])
    assert not refs.any() and not nblocks.any() and not ntok.any() and not tail.any()
    assert ctrl[:2].tolist() == [2 * cap, pool + 2 * cap] and ring[: 2 * cap].tolist() == list(range(2 * cap))


def test_rotated_appends_to_no_layer_change_nothing():
    from mentat_b200 import Rotary
    rng = np.random.default_rng(24)
    m, o = pair(L=2)
    a, = start(m, o, [5], rng)
    rot = Rotary(64)
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    for layer in (-1, 2):
        with pytest.raises(ValueError, match="layer"):
            m.append_rotated(a, layer, x, x, x, rot)
        with pytest.raises(ValueError, match="layer"):
            m.append_rotated_batched([a], layer, x, x, x, rot)
    same(m, o)


@pytest.mark.parametrize("capacity", [1001, 20000])  # pages of a table shared out over a few CTAs and over many
def test_forks_of_runs_and_long_tables(capacity):
    """Parents of no page to a thousand, in runs of children around a warp's width, in one batch and by the manager."""
    from mentat_b200 import ops
    rng = np.random.default_rng(25)
    m, o = pair(L=2, hkv=1, d=8, pool=20000, bs=1, max_seqs=400, max_blocks_per_seq=capacity, strict=False)
    ids = start(m, o, [0, 1, 127, 128, 129, 513, 1000], rng)
    parents = [p for p, run in zip([6, 4, 0, 3, 5, 2, 1, 6, 4], [33, 1, 5, 32, 65, 31, 64, 3, 1]) for _ in range(run)]
    slots = m._free_slots[::-1][: len(parents)]
    ops.fork_pages(m, torch.tensor([m._sequences[ids[p]].slot for p in parents], dtype=torch.int32, device="cuda"),
                   torch.tensor(slots, dtype=torch.int32, device="cuda"))
    m.check()
    for p, s in zip(parents, slots):
        own = m._sequences[ids[p]].slot
        assert torch.equal(m._nblocks[:, s], m._nblocks[:, own]) and torch.equal(m._ntok[:, s], m._ntok[:, own])
        nb = int(m._nblocks[0, own])
        assert torch.equal(m._tables[:, s, :nb], m._tables[:, own, :nb])
    ops.free_pages(m, torch.tensor(slots, dtype=torch.int32, device="cuda"))
    same(m, o)
    for n in (1, 3, 4, 70):
        some = [ids[p] for p in parents[:n]]
        assert m.fork_sequences(some) == [o.fork_sequence(s) for s in some]
    same(m, o)
