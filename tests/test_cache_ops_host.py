"""Rotary frequencies, and what the newer operators refuse, without a device."""

import ctypes as C
import math

import numpy as np
import pytest
import torch

from mentat_b200 import KVCacheView, Rotary, _lib, ops
from mentat_b200.rotary import frequencies


def test_plain_frequencies():
    f, scale = frequencies(8, 10000.0)
    np.testing.assert_allclose(f, [1.0, 10000 ** -0.25, 10000 ** -0.5, 10000 ** -0.75], rtol=1e-15)
    assert scale == 1.0


def _hf(kind, dim, base, **sc):
    """Frequencies of the model library's own rotary module for the same settings."""
    transformers = pytest.importorskip("transformers")
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    cfg = transformers.LlamaConfig(hidden_size=dim * 2, num_attention_heads=2, head_dim=dim,
                                   max_position_embeddings=sc.pop("max_position", 8192),
                                   rope_parameters=dict(rope_type=kind, rope_theta=base, **sc))
    inv, scale = ROPE_INIT_FUNCTIONS[kind](cfg, torch.device("cpu"))
    return inv.double().numpy(), float(scale)


@pytest.mark.parametrize("kind,extra", [
    ("linear", dict(factor=4.0)),
    ("llama3", dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)),
    ("yarn", dict(factor=4.0, original_max_position_embeddings=8192)),
    ("yarn", dict(factor=40.0, beta_fast=32.0, beta_slow=1.0, mscale=1.0, mscale_all_dim=0.7,
                  original_max_position_embeddings=4096)),
])
@pytest.mark.parametrize("dim,base", [(128, 5e5), (64, 1e4)])
def test_scaled_frequencies_are_the_models(kind, extra, dim, base):
    want, want_scale = _hf(kind, dim, base, **extra)
    got, scale = frequencies(dim, base, dict(rope_type=kind, **extra))
    # the module works in float: 2^-24 in the base's power, whose exponent is up to ln(5e5) = 13
    # times that, the quotient and a blend of two: below 32 * 2^-24
    np.testing.assert_allclose(got, want, rtol=32 * 2.0 ** -24)
    assert scale == pytest.approx(want_scale, rel=1e-6)


def test_dynamic_and_longrope():
    sc = dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=1024)
    np.testing.assert_array_equal(frequencies(64, 1e4, sc, seq_len=100)[0], frequencies(64, 1e4)[0])
    f, _ = frequencies(64, 1e4, sc, seq_len=4096)
    # the base grows by (2 * 4 - 1)^(64 / 62), so the slowest pair's angle by its inverse's 62 / 64th power
    assert f[-1] == pytest.approx(frequencies(64, 1e4)[0][-1] / 7.0, rel=1e-12)
    short, long = list(np.linspace(1, 2, 32)), list(np.linspace(1, 40, 32))
    sc = dict(rope_type="longrope", short_factor=short, long_factor=long, factor=16.0,
              original_max_position_embeddings=4096)
    f0 = frequencies(64, 1e4)[0]
    np.testing.assert_allclose(frequencies(64, 1e4, sc, seq_len=4096)[0], f0 / np.array(short))
    f, scale = frequencies(64, 1e4, sc)
    np.testing.assert_allclose(f, f0 / np.array(long))
    assert scale == pytest.approx(math.sqrt(1 + math.log(16) / math.log(4096)))


@pytest.mark.parametrize("kind,extra", [
    ("dynamic", dict(factor=2.0)),
    ("longrope", dict(factor=4.0, short_factor=[1.0] * 32, long_factor=[2.0] * 32, original_max_position_embeddings=512)),
])
def test_modules_that_change_with_the_length_are_refused(kind, extra):
    transformers = pytest.importorskip("transformers")
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding
    cfg = transformers.LlamaConfig(hidden_size=128, num_attention_heads=2, head_dim=64,
                                   max_position_embeddings=512 if kind == "dynamic" else 2048,
                                   rope_parameters=dict(rope_type=kind, rope_theta=1e4, **extra))
    module = LlamaRotaryEmbedding(cfg)
    before = module.inv_freq.clone()
    with pytest.raises(ValueError, match="seq_len"):
        Rotary.from_module(module, 64)
    module(torch.zeros(1, 2048, 128), torch.arange(2048)[None])
    assert not torch.equal(module.inv_freq, before)  # the reason
    with pytest.raises(ValueError, match="seq_len"):
        Rotary.from_module(module, 64)
    if kind == "dynamic":  # one length's angles, in float: as the comparison with the model's own above
        r = Rotary(64, base=1e4, scaling=dict(extra, rope_type=kind, original_max_position_embeddings=512), seq_len=2048,
                   device="cpu")
        np.testing.assert_allclose(r.inv_freq.numpy(), module.inv_freq.double().numpy(), rtol=32 * 2.0 ** -24)


@pytest.mark.parametrize("kind,extra", [
    ("default", {}), ("linear", dict(factor=4.0)),
    ("llama3", dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=512)),
    ("yarn", dict(factor=4.0, original_max_position_embeddings=512)),
])
def test_modules_with_fixed_angles(kind, extra):
    transformers = pytest.importorskip("transformers")
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding
    cfg = transformers.LlamaConfig(hidden_size=128, num_attention_heads=2, head_dim=64, max_position_embeddings=2048,
                                   rope_parameters=dict(rope_type=kind, rope_theta=1e4, **extra))
    module = LlamaRotaryEmbedding(cfg)
    r = Rotary.from_module(module, 64)
    assert torch.equal(r.inv_freq, module.inv_freq.double()) and r.attention_scaling == module.attention_scaling


def test_rotary_refusals():
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=72), dict(offset=-1),
                dict(rotary_dim=64, offset=1), dict(base=0.0), dict(scaling={"rope_type": "none such"}),
                dict(scaling={"rope_type": "linear"}), dict(rotary_dim=8, inv_freq=torch.ones(3)),
                dict(inv_freq=torch.ones(3, dtype=torch.int64)), dict(inv_freq=torch.ones(2, 2)),
                dict(inv_freq=torch.ones(3), scaling={"rope_type": "linear", "factor": 2.0}),
                dict(scaling={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
                              "original_max_position_embeddings": 8192})):
        with pytest.raises(ValueError):
            Rotary(64, device="cpu", **bad)
    with pytest.raises(ValueError):
        Rotary(1026, device="cpu")
    r = Rotary(64, rotary_dim=32, offset=16, device="cpu")
    assert (r.rotary_dim, r.offset) == (32, 16) and r.inv_freq.dtype == torch.float64


def test_row_operands_refused():
    r = Rotary(64, device="cpu")
    q, k, p = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.arange(3)
    for call in (lambda: ops.rotary(q[:, :, :32], None, p, r),
                 lambda: ops.rotary(q, k[:2], p, r),
                 lambda: ops.rotary(q, k, p[:2], r),
                 lambda: ops.rotary(q, k, p.double(), r),
                 lambda: ops.rotary(q, k, p, r, q_out=torch.zeros(3, 1, 64).expand(3, 4, 64)),
                 lambda: ops.rotary(q, k, p, r, q_out=torch.zeros(3, 4, 63)),
                 lambda: ops.rotary(torch.zeros(4, 4, 64)[:3], k, p, r, k_out=torch.zeros(3, 2, 64)[:, :1])):
        with pytest.raises(ValueError):
            call()
    base = torch.zeros(4, 4, 64)
    with pytest.raises(ValueError, match="not overlap"):
        ops.rotary(base[:3], None, p, r, q_out=base[1:])
    both = torch.zeros(3, 6, 64)
    for outs in (dict(q_out=both[:, :4], k_out=both[:, 3:5]), dict(q_out=torch.zeros(1), k_out=q[:, 1:3]),
                 dict(q_out=q, k_out=q[:, :2])):
        with pytest.raises(ValueError):
            ops.rotary(q, k, p, r, **outs)
    with pytest.raises(ValueError, match="q_out must not overlap k"):
        ops.rotary(q, q.clone()[:, :2], p, r, q_out=both[:, :4], k_out=both[:, 2:4])
    with pytest.raises(ValueError, match="q_out must not overlap k"):
        ops.rotary(both[:, 2:6].clone(), both[:, :4], p, r, q_out=both[:, :4])
    # parts of one buffer's rows are apart
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary(both[:, :4], both[:, 4:], p, r, q_out=both[:, :4], k_out=both[:, 4:])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary(q, k, p, r, q_out=both[:, 2:], k_out=both[:, :2])
    with pytest.raises(TypeError):
        ops.rotary(q, k.double(), p, r)
    with pytest.raises(TypeError):
        ops.rotary(q.long(), None, p, r)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary(q, k, p, r)
    with pytest.raises(ValueError):
        KVCacheView(torch.zeros(1, 4, 16, 1, 64), torch.zeros(1, 4, 16, 1, 64))  # not on a device


def _desc(**kw):
    """A descriptor whose pointers are never read: every call below is refused first."""
    d = _lib.KVCache()
    d.num_layers, d.num_blocks, d.block_size, d.num_kv_heads, d.head_dim = 2, 64, 16, 2, 64
    d.dtype, d.max_seqs, d.max_blocks_per_seq = _lib.MENTAT_BF16, 8, 16
    for f in ("k_pool", "v_pool", "refcounts", "free_ring", "ctrl", "tables", "nblocks", "ntok", "tail", "scratch"):
        setattr(d, f, 4096)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


ARG, UNSUPPORTED = -1, -3


def test_c_abi_refuses_rotary_arguments():
    lib = _lib.load()
    rows, none = _lib.Rows(4096, 128, 64, 2), _lib.Rows()
    r = _lib.Rotary(4096, 32, 0, 0, 0, 1.0)

    def apply(dtype=1, d=64, n=3, q=rows, qo=rows, k=none, ko=none, p=4096, rot=r):
        return lib.mentat_rotary_apply(dtype, d, n, q, qo, k, ko, p, rot, None)
    assert apply(n=0) == 0 and apply(q=none, qo=none) == 0
    assert apply(n=-1) == ARG and apply(p=None) == ARG and apply(qo=_lib.Rows(4096, 128, 64, 1)) == ARG
    assert apply(q=_lib.Rows(None, 128, 64, 2)) == ARG and apply(rot=_lib.Rotary(4096, 33, 0, 0, 0, 1.0)) == ARG
    assert apply(rot=_lib.Rotary(4096, 16, 33, 0, 0, 1.0)) == ARG and apply(rot=_lib.Rotary(None, 32, 0, 0, 0, 1.0)) == ARG
    assert apply(rot=_lib.Rotary(4096, 2 ** 30, 0, 0, 0, 1.0)) == ARG and apply(d=2048) == ARG
    assert apply(dtype=7) == UNSUPPORTED

    def append(c=_desc(), layer=0, n=3, where=4096, q=rows, qo=rows, k=rows, v=rows, p=4096):
        return lib.mentat_rotary_append(c, layer, n, where, q, qo, k, v, p, r, None)
    assert append(n=0) == 0
    assert append(layer=2) == ARG and append(where=None) == ARG and append(k=none) == ARG
    assert append(v=_lib.Rows(4096, 64, 64, 1)) == ARG and append(c=_desc(k_pool=None)) == ARG
    assert append(c=_desc(dtype=9)) == UNSUPPORTED

    def many(n=3, slots=4096, c=_desc()):
        return lib.mentat_kv_append_rotated_batched(c, 0, slots, n, rows, rows, rows, rows, None, r, None)
    assert many(n=0) == 0 and many(n=9) == ARG and many(slots=None) == ARG and many(c=_desc(dtype=9)) == UNSUPPORTED
    assert lib.mentat_kv_append_rotated(_desc(), 0, 8, 1, rows, rows, rows, rows, None, r, None) == ARG
    assert lib.mentat_kv_append_rotated(_desc(), 0, 0, 0, rows, rows, rows, rows, None, r, None) == 0


def test_c_abi_refuses_page_arguments():
    lib = _lib.load()
    c = _desc()
    need = lib.mentat_pages_workspace_bytes(c, 4)
    assert need >= 4 * (2 * 64 + 4 * 4 * 2) and lib.mentat_pages_workspace_bytes(c, 1025) == 0
    assert lib.mentat_kv_fork_batched(c, None, None, 0, None) == 0
    assert lib.mentat_kv_fork_batched(c, None, 4096, 1, None) == ARG
    assert lib.mentat_kv_fork_batched(c, 4096, 4096, 1025, None) == ARG
    assert lib.mentat_kv_fork_batched(_desc(max_seqs=1 << 20), 4096, 4096, 1, None) == UNSUPPORTED
    assert lib.mentat_kv_free_batched(c, None, 0, 0, None, 0, None) == 0
    assert lib.mentat_kv_free_batched(c, 4096, 4, 1, 4096, need - 1, None) == ARG
    assert lib.mentat_kv_free_batched(c, 4096, 4, 1, None, need, None) == ARG
    big = _desc(num_layers=64, max_blocks_per_seq=1 << 20)
    assert lib.mentat_kv_free_batched(big, 4096, 1024, 1, 4096, 1 << 40, None) == UNSUPPORTED

    def compact(c=c, n=4, keep=4096, cu=4096, most=5, rot=None, ws=need, ls=0, total=20):
        return lib.mentat_kv_compact(c, 4096, None, n, keep, ls, total, cu, most, 3, rot, 4096, ws, None)
    assert compact(n=0) == 0 and compact(n=1025) == ARG and compact(keep=None) == ARG and compact(cu=None) == ARG
    assert compact(ws=need - 1) == ARG and compact(most=-1) == ARG and compact(ls=-1) == ARG and compact(total=-1) == ARG
    assert compact(rot=C.byref(_lib.Rotary(4096, 33, 0, 0, 0, 1.0))) == ARG


def test_batches_are_split_where_a_call_cannot_take_them():
    """Releases of one call are numbered in 32 bits; a fork has no such limit."""
    from types import SimpleNamespace

    from mentat_b200 import PagedKVCacheManager
    lib = _lib.load()
    for layers, cap in ((80, 65536), (64, 1 << 20), (2, 16), (126, 33333332)):
        step = PagedKVCacheManager._pages_step(SimpleNamespace(num_layers=layers, _table_stride=cap))
        d = _desc(num_layers=layers, max_blocks_per_seq=cap)
        assert lib.mentat_kv_free_batched(d, 4096, step, 1, 4096, 0, None) == ARG  # only its workspace is missing
        if step < 1024:
            assert lib.mentat_kv_free_batched(d, 4096, step + 1, 1, 4096, 0, None) == UNSUPPORTED
        else:
            assert step == 1024


def test_c_abi_refuses_sparse_arguments():
    lib = _lib.load()
    x = _lib.PageIndex(4096, 4096)

    def decode(c=_desc(), layer=0, idx=x, slots=4096, n=2, hq=4, scale=0.1, longest=100, budget=8, sink=1, recent=1):
        return lib.mentat_sparse_decode(c, layer, idx, slots, n, 4096, hq * 64, hq, 4096, hq * 64, scale, longest,
                                        budget, sink, recent, None, None, 0, None)
    assert decode(n=0) == 0
    for bad in (dict(layer=2), dict(idx=_lib.PageIndex(None, 4096)), dict(idx=_lib.PageIndex(4097, 4096)),
                dict(slots=None), dict(hq=3), dict(scale=0.0), dict(scale=float("nan")), dict(longest=-1),
                dict(budget=0), dict(sink=-1), dict(recent=0), dict(sink=4, recent=5), dict(c=_desc(k_pool=4100)),
                dict(c=_desc(tables=None))):
        assert decode(**bad) == ARG, bad
    assert lib.mentat_sparse_workspace_bytes(_desc(), 2, 100, 8) == 0      # a small batch needs none
    long = _desc(max_blocks_per_seq=2000)
    need = lib.mentat_sparse_workspace_bytes(long, 500, 20000, 8)
    assert need >= 4 * 500 * 2 * (1250 + 8) and decode(c=long, n=500, longest=20000) == ARG
    assert decode(hq=34) == UNSUPPORTED and decode(budget=8193) == UNSUPPORTED
    assert decode(c=_desc(head_dim=96)) == UNSUPPORTED and decode(c=_desc(dtype=5)) == UNSUPPORTED
    assert lib.mentat_page_index_blocks(_desc(), 0, None, 1, x, None) == ARG
    assert lib.mentat_page_index_blocks(_desc(), 0, None, 0, x, None) == 0
    assert lib.mentat_page_index_seqs(_desc(), -2, 4096, 1, 0, 1, x, None) == ARG
    assert lib.mentat_page_index_seqs(_desc(), -1, 4096, 1, 0, 0, x, None) == 0
    for first, pages in ((0x7fffffff, 1), (0x7fffff00, 0x100), (1, 0x7fffffff)):  # a page's number would pass an int
        assert lib.mentat_page_index_seqs(_desc(), 0, 4096, 1, first, pages, x, None) == ARG
    assert lib.mentat_page_bounds(_desc(), 0, 4096, 1, x, None, 4096, 4096, None) == ARG


def test_rotated_appends_and_index_refuse_their_arguments():
    """What the kernels would read by: another model's rotary, slots of another type, length or shape, no index."""
    class Cache:  # what the checks look at
        def __init__(self, **kw):
            self.__dict__.update(kw)
    cpu = torch.device("cpu")
    cache = Cache(device=cpu, dtype=torch.bfloat16, head_dim=64, num_layers=2, num_key_value_heads=2,
                  page_index=None, table_capacity=16, _desc_ptr=0)
    cid = ops.register_cache(cache)
    rot, wide = Rotary(64, device="cpu"), Rotary(128, device="cpu")
    q, k = torch.zeros(4, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    slots = torch.arange(4, dtype=torch.int32)

    def append(slots=slots, q=q, rot=rot):
        return ops.append_rotated(k, k, slots, q, k, k, cid, 0, rot.op_id)
    with pytest.raises(RuntimeError, match="CUDA"):  # nothing to refuse but the device
        append()
    with pytest.raises(ValueError, match="heads of 128"):
        append(rot=wide)
    for bad in (slots.long(), slots[:3], slots.view(2, 2), torch.zeros(5, dtype=torch.int32)):
        with pytest.raises(ValueError, match="slots"):
            append(slots=bad)
    with pytest.raises(RuntimeError, match="enable_page_index"):
        ops.index_sequences(cache, slots, 0, 1)
    cache.page_index = Cache(_ptr=0)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.index_sequences(cache, slots, 0, 1)
    with pytest.raises(ValueError, match="slots"):
        ops.index_sequences(cache, slots.long(), 0, 1)
    for first, pages in ((-1, 1), (0, -1)):
        with pytest.raises(ValueError, match="range of pages"):
            ops.index_sequences(cache, slots, first, pages)


def test_operator_schemas():
    s = str(torch.ops.mentat_b200.append_rotated.default._schema)
    assert "Tensor(a0!) k_pool" in s and "Tensor(a1!) v_pool" in s and s.endswith("-> Tensor")
    s = str(torch.ops.mentat_b200.paged_sparse_decode.default._schema)
    assert s.startswith("mentat_b200::paged_sparse_decode(Tensor q, Tensor slots,") and s.endswith("-> Tensor")
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k = torch.empty(4, 8, 64, dtype=torch.bfloat16), torch.empty(4, 2, 64, dtype=torch.bfloat16)
        pool, slots = torch.empty(2, 16, 2, 64, dtype=torch.bfloat16), torch.empty(4, dtype=torch.int32)
        out = torch.ops.mentat_b200.append_rotated(pool, pool, slots, q, k, k, 1, 0, 2)
        assert out.shape == q.shape and out.dtype == q.dtype
        out = torch.ops.mentat_b200.paged_sparse_decode(q, slots, 100, 1, 0, 0.1, 8, 1, 1)
        assert out.shape == q.shape and out.dtype == q.dtype
