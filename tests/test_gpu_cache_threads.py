"""Calls of two host threads at once, each on its own cache and stream: sizes of shared memory that differ
between ordinary calls of one kernel must not refuse each other's launches.

The threads make the C calls themselves: through the
Python layer, which holds the interpreter's lock for most of a call, two of them are hardly ever inside at once."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

ROUNDS = 3000


def together(*jobs):
    """Each job (a function of the stream) ROUNDS times on a thread and stream of its own; what they returned."""
    statuses, gate = [set() for _ in jobs], threading.Barrier(len(jobs))

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            gate.wait(30)
            for r in range(ROUNDS):
                statuses[i].add(jobs[i](stream.cuda_stream))
                if r % 200 == 199:
                    stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return statuses


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sparse_decode_of_different_sizes(dtype):
    from mentat_b200 import KVCacheView, PageIndex, _lib, ops
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((1, 64, 16, 2, 128), generator=g, device="cuda").to(dtype) for _ in range(2))
    tables = torch.randperm(64, generator=g, device="cuda").to(torch.int32).view(1, 1, 64)
    fn = _lib.call("mentat_sparse_decode")
    jobs, outs, wants, keep = [], [], [], []
    for max_len, budget in ((1024, 8), (131072, 8192)):  # the longest length is a limit, any above 1000 is right
        c = KVCacheView(k, v, tables, torch.full((1, 1), 1000, dtype=torch.int32, device="cuda"))
        x = PageIndex(c)
        ops.page_index(x, 0, torch.arange(64, dtype=torch.int32, device="cuda"))
        q = torch.randn((1, 8, 128), generator=g, device="cuda").to(dtype)
        slots = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.zeros_like(q)
        assert x.workspace_bytes(1, max_len, budget) == 0
        args = (c._desc_ptr, 0, x._ptr, slots.data_ptr(), 1, q.data_ptr(), q.stride(0), 8, out.data_ptr(), out.stride(0),
                ops.default_scale(128), max_len, budget, 1, 1, None, None, 0)
        wants.append(ops.sparse_decode(x, 0, slots, q, max_len, budget))
        jobs.append(lambda stream, args=args: fn(*args, stream))
        outs.append(out)
        keep.append((c, x, q, slots))
    assert together(*jobs) == [{0}, {0}]
    for got, want in zip(outs, wants):
        assert torch.equal(got, want)


def test_compaction_of_different_rows():
    from mentat_b200 import PagedKVCacheManager, _lib
    compact, free = _lib.call("mentat_kv_compact"), _lib.call("mentat_kv_free_batched")
    size = _lib.call("mentat_pages_workspace_bytes")
    jobs, caches, keep = [], [], []
    i32 = dict(dtype=torch.int32, device="cuda")
    for hkv, d in ((1, 64), (8, 128)):
        m = PagedKVCacheManager(2, hkv, d, max_blocks=64, block_size=16, device="cuda", dtype=torch.bfloat16, max_seqs=8)
        s = m.allocate_sequence()
        g = torch.Generator(device="cuda").manual_seed(hkv)
        for layer in range(2):
            m.append_tokens(s, layer, *(torch.randn((100, hkv, d), generator=g, device="cuda").to(torch.bfloat16)
                                        for _ in range(2)))
        src, dst = torch.tensor([m._sequences[s].slot], **i32), torch.tensor([m._free_slots[-1]], **i32)
        rows, cu = torch.arange(1, 100, **i32), torch.tensor([0, 99], **i32)
        nbytes = size(m._desc_ptr, 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        a = (m._desc_ptr, src.data_ptr(), dst.data_ptr(), 1, rows.data_ptr(), 0, 99, cu.data_ptr(), 99, 7, None, ws.data_ptr(),
             nbytes)
        b = (m._desc_ptr, dst.data_ptr(), 1, 7, ws.data_ptr(), nbytes)
        jobs.append(lambda stream, a=a, b=b: (compact(*a, stream), free(*b, stream)))
        caches.append((m, m.get_stats()["blocks_used"]))
        keep.append((src, dst, rows, cu, ws))
    assert together(*jobs) == [{(0, 0)}, {(0, 0)}]
    for m, used in caches:
        assert m.get_stats()["blocks_used"] == used  # no fresh block without a table
