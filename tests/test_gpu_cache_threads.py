"""Calls of two host threads at once, each on its own cache and stream: sizes of shared memory that differ
between ordinary calls of one kernel must not refuse each other's launches."""

import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

ROUNDS = 400


def together(*jobs):
    """Each job (a function of no arguments) ROUNDS times on a thread and stream of its own."""
    failed, gate = [], threading.Barrier(len(jobs))

    def work(job):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait(30)
                for _ in range(ROUNDS):
                    job()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - shown by the assertion
            failed.append(e)

    torch.cuda.synchronize()
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert not failed, failed


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sparse_decode_of_different_sizes(dtype):
    from mentat_b200 import KVCacheView, PageIndex, ops
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((1, 64, 16, 2, 128), generator=g, device="cuda").to(dtype) for _ in range(2))
    tables = torch.randperm(64, generator=g, device="cuda").to(torch.int32).view(1, 1, 64)
    jobs, outs, wants = [], [], []
    for max_len, budget in ((1024, 8), (131072, 8192)):  # the longest length is a limit, any above 1000 is right
        c = KVCacheView(k, v, tables, torch.full((1, 1), 1000, dtype=torch.int32, device="cuda"))
        x = PageIndex(c)
        ops.page_index(x, 0, torch.arange(64, dtype=torch.int32, device="cuda"))
        q = torch.randn((1, 8, 128), generator=g, device="cuda").to(dtype)
        slots = torch.zeros(1, dtype=torch.int32, device="cuda")

        def job(i=len(outs), x=x, slots=slots, q=q, max_len=max_len, budget=budget):
            outs[i] = ops.sparse_decode(x, 0, slots, q, max_len, budget)
        wants.append(ops.sparse_decode(x, 0, slots, q, max_len, budget))
        outs.append(None)
        jobs.append(job)
    together(*jobs)
    for got, want in zip(outs, wants):
        assert torch.equal(got, want)


def test_compaction_of_different_rows():
    from mentat_b200 import PagedKVCacheManager
    jobs, caches = [], []
    for hkv, d in ((1, 64), (8, 128)):
        m = PagedKVCacheManager(2, hkv, d, max_blocks=64, block_size=16, device="cuda", dtype=torch.bfloat16, max_seqs=8)
        s = m.allocate_sequence()
        g = torch.Generator(device="cuda").manual_seed(hkv)
        for layer in range(2):
            m.append_tokens(s, layer, *(torch.randn((100, hkv, d), generator=g, device="cuda").to(torch.bfloat16)
                                        for _ in range(2)))
        keep = list(range(1, 100))

        def job(m=m, s=s, keep=keep):
            m.free_sequences(m.compact_sequences([s], [keep], into_new=True))
        job()
        used = m.get_stats()["blocks_used"]
        jobs.append(job)
        caches.append((m, used))
    together(*jobs)
    for m, used in caches:
        assert m.get_stats()["blocks_used"] == used  # no fresh block without a table
