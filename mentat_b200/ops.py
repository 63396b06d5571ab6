"""torch custom operators over the C ABI (``torch.library``).

The three hot-path calls of the public Python API
(``PagedKVCacheManager.append_tokens_batched``, ``attention_backend.attn_decode``,
``gate.Gate``) are registered as torch operators with schemas and fake (meta)
implementations, so torch.compile can trace a caller that uses them.  The
public API calls them through ``paged_decode``, ``append_batched`` and
``gate_step`` below, which go through the operators while torch.compile traces
and call the implementation directly otherwise (eagerly and under CUDA-graph
capture), which saves the dispatcher's host time.  Each call launches on the
current torch stream and returns without synchronising.

A cache is passed as the integer id it registered under (``register_cache``),
because operator arguments are tensors and scalars.
"""

from __future__ import annotations

import ctypes as C
import itertools
import math
import struct
import threading
import weakref
from typing import Optional

import torch

from . import _lib

_caches: "weakref.WeakValueDictionary[int, object]" = weakref.WeakValueDictionary()
_ids = itertools.count(1)

MAX_SEQS_PER_LAUNCH = 1024  # mentat_paged_decode's per-launch sequence limit


def register_cache(mgr) -> int:
    """Registers a ``PagedKVCacheManager``; returns the id the operators take."""
    i = next(_ids)
    _caches[i] = mgr
    return i


def _cache(i: int):
    mgr = _caches.get(i)
    if mgr is None:
        raise RuntimeError(f"mentat_b200: no live cache with id {i}")
    return mgr


def _paged_decode(q: torch.Tensor, slots: torch.Tensor, max_len: int, cache: int, layer: int,
                  scale: float, reuse_plan: bool = False) -> torch.Tensor:
    """Tree-aware decode attention of ``q`` (N, Hq, D) over the cached sequences in
    ``slots`` (N,) int32 of layer ``layer``; ``max_len`` is the longest of their
    lengths (it sizes the workspace).  Wraps ``mentat_paged_decode``; with
    ``reuse_plan``, ``mentat_paged_decode_reuse_plan`` (the previous call on this
    cache planned the same sequences for another layer of the same step; batches
    above the per-launch limit always plan)."""
    mgr = _cache(cache)
    lib = _lib.load()
    n, hq, d = q.shape
    out = torch.empty((n, hq, d), device=q.device, dtype=q.dtype)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    fn = lib.mentat_paged_decode_reuse_plan if reuse_plan and n <= MAX_SEQS_PER_LAUNCH else lib.mentat_paged_decode
    for a in range(0, n, MAX_SEQS_PER_LAUNCH):
        b = min(n, a + MAX_SEQS_PER_LAUNCH)
        ws, wsb, parts = mgr.decode_workspace(b - a, hq, max_len)
        _lib.check(fn(
            mgr._descp, layer, slots.data_ptr() + 4 * a, b - a,
            q.data_ptr() + a * q.stride(0) * q.element_size(), q.stride(0), hq,
            out.data_ptr() + a * out.stride(0) * out.element_size(), out.stride(0), scale,
            ws.data_ptr(), wsb, parts, stream), "mentat_paged_decode")
    return out


paged_decode_op = torch.library.custom_op("mentat_b200::paged_decode", mutates_args=(),
                                          device_types="cuda")(_paged_decode)


@paged_decode_op.register_fake
def _paged_decode_fake(q, slots, max_len, cache, layer, scale, reuse_plan=False):
    return torch.empty_like(q)


def _append_batched(k_pool: torch.Tensor, v_pool: torch.Tensor, slots: torch.Tensor, k: torch.Tensor,
                    v: torch.Tensor, cache: int, layer: int) -> None:
    """Appends one token per sequence (rows of ``k``, ``v``: (N, Hkv, D)) to the
    sequences in ``slots`` of layer ``layer``, allocating and copying-on-write on
    the device.  ``k_pool`` / ``v_pool`` are the cache's pools, named so that
    torch knows what the operator writes.  Wraps ``mentat_kv_append_batched``."""
    mgr = _cache(cache)
    lib = _lib.load()
    n = k.shape[0]
    ks, vs = k.stride(0), v.stride(0)
    stream = torch.cuda.current_stream(k.device).cuda_stream
    for a in range(0, n, 1024):
        b = min(n, a + 1024)
        _lib.check(lib.mentat_kv_append_batched(
            mgr._descp, layer, slots.data_ptr() + 4 * a, b - a,
            k.data_ptr() + a * ks * k.element_size(), ks,
            v.data_ptr() + a * vs * v.element_size(), vs, stream), "append_tokens_batched")
    if mgr.page_index is not None:
        _index_tails(mgr, layer, slots, n)


append_batched_op = torch.library.custom_op("mentat_b200::append_batched", mutates_args=("k_pool", "v_pool"),
                                            device_types="cuda")(_append_batched)


@append_batched_op.register_fake
def _append_batched_fake(k_pool, v_pool, slots, k, v, cache, layer):
    return None


# The public API calls these wrappers.  Eagerly (and under CUDA-graph capture) they
# call the implementation directly: the dispatcher round trip of a custom
# operator costs about 15 us of host time per call, which a decode step pays
# for every layer.  While torch.compile traces they go through the operators.
def paged_decode(q, slots, max_len, cache, layer, scale, reuse_plan=False):
    if torch.compiler.is_compiling():
        return torch.ops.mentat_b200.paged_decode(q, slots, max_len, cache, layer, scale, reuse_plan)
    return _paged_decode(q, slots, max_len, cache, layer, scale, reuse_plan)


def append_batched(k_pool, v_pool, slots, k, v, cache, layer):
    if torch.compiler.is_compiling():
        return torch.ops.mentat_b200.append_batched(k_pool, v_pool, slots, k, v, cache, layer)
    return _append_batched(k_pool, v_pool, slots, k, v, cache, layer)


def _gate_step(logits: torch.Tensor, hist_ptr: torch.Tensor, hist_ids: torch.Tensor, ema_old: torch.Tensor,
               params: list[float], ints: list[int], out: torch.Tensor) -> None:
    """The fused entropy gate over ``logits`` (N, V) into ``out`` (N records of
    ``mentat_gate_out`` as bytes).  ``params`` = (temperature, penalty, alpha,
    multiplier, soft-explore initial), ``ints`` = (K, max_active, num_active,
    step, soft-explore window[, flags]).  Wraps ``mentat_gate_step``."""
    lib = _lib.load()
    n, V = logits.shape
    p = _lib.GateParams(*params, *ints[:5], ints[5] if len(ints) > 5 else 0)
    stream = torch.cuda.current_stream(logits.device).cuda_stream
    _lib.check(lib.mentat_gate_step(
        logits.data_ptr(), _DT[logits.dtype], n, V, logits.stride(0), hist_ptr.data_ptr(), hist_ids.data_ptr(),
        ema_old.data_ptr(), C.byref(p), out.data_ptr(), stream), "mentat_gate_step")


gate_step_op = torch.library.custom_op("mentat_b200::gate_step", mutates_args=("out",),
                                       device_types="cuda")(_gate_step)


@gate_step_op.register_fake
def _gate_step_fake(logits, hist_ptr, hist_ids, ema_old, params, ints, out):
    return None


def gate_step(logits, hist_ptr, hist_ids, ema_old, params, ints, out):
    if torch.compiler.is_compiling():
        return torch.ops.mentat_b200.gate_step(logits, hist_ptr, hist_ids, ema_old, params, ints, out)
    return _gate_step(logits, hist_ptr, hist_ids, ema_old, params, ints, out)


_DT = {torch.bfloat16: _lib.MENTAT_BF16, torch.float16: _lib.MENTAT_F16, torch.float32: _lib.MENTAT_F32}


def default_scale(d: int) -> float:
    return 1.0 / math.sqrt(d)


def paged_prefill(descp, layer: int, slot: torch.Tensor, pos0: int, q: torch.Tensor, scale: float,
                  out: torch.Tensor = None) -> torch.Tensor:
    """Causal prefill attention of ``q`` (n, Hq, D), query i at position pos0 + i
    of the sequence in ``slot`` (device int32[1]) of the cache described by
    ``descp`` (a ``ctypes.byref`` of ``_lib.KVCache``); its K/V must already be
    cached.  Wraps ``mentat_paged_prefill``, PREFILL_QUERIES_PER_LAUNCH queries
    per call (the workspace grows with queries x partials); the workspace comes
    from torch's caching allocator on the current stream."""
    lib = _lib.load()
    n, hq, d = q.shape
    if out is None:
        out = torch.empty((n, hq, d), device=q.device, dtype=q.dtype)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    for a in range(0, n, PREFILL_QUERIES_PER_LAUNCH):
        m = min(n - a, PREFILL_QUERIES_PER_LAUNCH)
        parts = int(lib.mentat_prefill_max_parts(descp, m, pos0 + a, hq))
        wsb = int(lib.mentat_decode_workspace_bytes(m, hq, d, parts))
        ws = torch.empty(wsb, device=q.device, dtype=torch.uint8)
        _lib.check(lib.mentat_paged_prefill(
            descp, layer, slot.data_ptr(), m, pos0 + a, q.data_ptr() + a * q.stride(0) * q.element_size(),
            q.stride(0), hq, out.data_ptr() + a * out.stride(0) * out.element_size(), out.stride(0), scale,
            ws.data_ptr(), wsb, parts, stream), "mentat_paged_prefill")
    return out


PREFILL_QUERIES_PER_LAUNCH = 8192


def prune_similar(sim: torch.Tensor, group_off: torch.Tensor, parent_key: torch.Tensor, logp: torch.Tensor,
                  threshold: float, max_group: int) -> torch.Tensor:
    """Pair resolution of semantic pruning (``generator.py:446-484``) on the device:
    ``sim`` (m, m) holds the cosine similarities of the leaves of several trees laid
    out tree after tree (``group_off`` int32, the trees' first rows and m);
    ``parent_key`` (int64) is equal for siblings; ``logp`` (float64) the leaves'
    cumulative log-probs.  Returns one uint8 per leaf, 1 for the pruned ones.
    Wraps ``mentat_prune_similar``; the threshold is rounded to ``sim``'s dtype,
    as torch's ``(sim * mask) > threshold`` compares in that dtype."""
    lib = _lib.load()
    m = sim.shape[0]
    out = torch.empty(m, dtype=torch.uint8, device=sim.device)
    if sim.stride(1) != 1:
        sim = sim.contiguous()
    thr = float(torch.tensor(threshold, dtype=sim.dtype).item())
    stream = torch.cuda.current_stream(sim.device).cuda_stream
    _lib.check(lib.mentat_prune_similar(sim.data_ptr(), _DT[sim.dtype], sim.stride(0), group_off.data_ptr(),
                                        group_off.numel() - 1, max_group, parent_key.data_ptr(), logp.data_ptr(),
                                        thr, out.data_ptr(), stream), "mentat_prune_similar")
    return out


# ---------------------------------------------------------------------------
# rotary positions, pages, sparse decode
# ---------------------------------------------------------------------------
try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
    from torch._C import _cuda_getDevice as _current_device
except ImportError:  # the same through the public calls, about a microsecond slower each
    _current_device = torch.cuda.current_device

    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def _call(device, name: str, *args) -> None:
    """Entry point ``name`` on the device's current torch stream, with the device current."""
    if device.type != "cuda":
        raise RuntimeError("mentat_b200 runs on CUDA devices only")
    fn = _lib.call(name)
    index = device.index
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(status, name)


class _RowArgs(threading.local):
    """Four ``mentat_rows`` of the calling thread, filled in one step and passed by address (a call
    has read them when it returns)."""

    def __init__(self):
        self.buf = bytearray(128)
        self._keep = (C.c_char * 128).from_buffer(self.buf)
        a = C.addressof(self._keep)
        self.at = (a, a + 32, a + 64, a + 96)


_row_args = _RowArgs()
_pack_rows = struct.Struct("@Pqqi4xPqqi4xPqqi4xPqqi4x").pack_into


_NO_ROWS = (0, 0, 0, 0)


def _rows(a, b, c, d) -> tuple:
    """Addresses of four ``mentat_rows``, given as (address, token stride, head stride, heads)."""
    r = _row_args
    _pack_rows(r.buf, 0, *a, *b, *c, *d)
    return r.at


def _operand(name: str, t: torch.Tensor, n: int, d: int, dtype, device) -> tuple:
    """``t`` checked as rows (n, heads, d), its last dimension made contiguous, and its ``mentat_rows``."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[0] != n or shape[2] != d:
        raise ValueError(f"{name} {tuple(shape)} is not ({n}, heads, {d})")
    if t.dtype is not dtype or dtype not in _DT:
        raise TypeError(f"{name} has dtype {t.dtype}, {dtype if dtype in _DT else 'float32, bfloat16 or float16'} expected")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, {device} expected")
    if stride[2] != 1 and d != 1:
        t = t.contiguous()
        stride = t.stride()
    return t, (t.data_ptr(), stride[0], stride[1], shape[1])


def _like(x: torch.Tensor) -> tuple:
    """A new tensor of x's shape, dtype and device, and its ``mentat_rows``."""
    _, h, d = x.shape
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    return out, (out.data_ptr(), h * d, d, h)


def _check_rows(name: str, t: torch.Tensor, n: int, d: int, dtype, device) -> torch.Tensor:
    return _operand(name, t, n, d, dtype, device)[0]


def _out_rows(name: str, out: Optional[torch.Tensor], x: torch.Tensor) -> tuple:
    """``out`` checked as the result of a row operation on ``x``: its own rows distinct, and
    either ``x`` itself or apart from it; a new tensor if None.  With its ``mentat_rows``."""
    if out is None:
        return _like(x)
    _check_out(name, out, x)
    return out, (out.data_ptr(), out.stride(0), out.stride(1), out.shape[1])


def _check_out(name: str, out: torch.Tensor, x: torch.Tensor) -> None:
    n, h, d = x.shape
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} must have the input's shape, dtype and device")
    if x.numel() == 0:
        return
    s0, s1 = out.stride(0), out.stride(1)
    if (d > 1 and out.stride(2) != 1) or not (
            ((h == 1 or s1 >= d) and (n == 1 or s0 >= (h - 1) * s1 * (h > 1) + d)) or
            ((n == 1 or s0 >= d) and (h == 1 or s1 >= (n - 1) * s0 * (n > 1) + d))):
        raise ValueError(f"{name} must hold rows of its own, each contiguous")
    if not (out.data_ptr() == x.data_ptr() and out.stride() == x.stride() or _apart(out, x)):
        raise ValueError(f"{name} must be the input itself or not overlap it")


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of rows share no byte: separate ranges of memory, or separate parts of
    the rows of one buffer (equal token strides)."""
    if a.numel() == 0 or b.numel() == 0:
        return True

    def reach(t, dims):
        return t.element_size() * (sum((m - 1) * s for m, s in zip(t.shape[dims:], t.stride()[dims:])) + 1)
    a0, b0 = a.data_ptr(), b.data_ptr()
    if a0 + reach(a, 0) <= b0 or b0 + reach(b, 0) <= a0:
        return True
    row = a.stride(0) * a.element_size()
    if row <= 0 or row != b.stride(0) * b.element_size():
        return False
    at = (b0 - a0) % row  # b's part, from the start of one of a's
    return reach(a, 1) <= at and at + reach(b, 1) <= row


def _check_apart(**tensors) -> None:
    """Refuses an output (the first, if given) that shares memory with another operand."""
    (name, out), *others = tensors.items()
    for other, t in others:
        if out is not None and t is not None and not _apart(out, t):
            raise ValueError(f"{name} must not overlap {other}")


def _check_positions(positions: torch.Tensor, n: int, device) -> torch.Tensor:
    dtype = positions.dtype
    if positions.shape != (n,) or (dtype is not torch.int64 and dtype is not torch.int32):
        raise ValueError(f"positions must be {n} int64 or int32 values")
    if positions.device != device:
        raise ValueError(f"positions are on {positions.device}, {device} expected")
    return positions if dtype is torch.int64 and positions.is_contiguous() else positions.to(torch.int64).contiguous()


def _check_layer(layer: int, cache) -> None:
    if not 0 <= layer < cache.num_layers:
        raise ValueError(f"layer {layer} is not within 0 .. {cache.num_layers - 1}")


def _check_rotary(rotary, d: int, device) -> None:
    if rotary.head_dim != d:
        raise ValueError(f"the rotary is for heads of {rotary.head_dim}, not {d}")
    if rotary.device != device:
        raise ValueError(f"the rotary is on {rotary.device}, {device} expected")


def _check_ids(name: str, t: torch.Tensor, device, n: Optional[int] = None, limit: Optional[int] = None) -> torch.Tensor:
    if t.dim() != 1 or t.dtype != torch.int32 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be a vector of {'' if n is None else str(n) + ' '}int32 values")
    if t.device != device:
        raise ValueError(f"{name} are on {t.device}, {device} expected")
    if limit is not None and t.shape[0] > limit:
        raise ValueError(f"{name}: {t.shape[0]} in one call, at most {limit}")
    return t.contiguous()


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary, *, inverse: bool = False,
           q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> tuple:
    """Turns ``q`` (N, Hq, D) and ``k`` (N, Hkv, D; may be None) to ``positions`` (N,)
    (``Rotary``); ``inverse`` turns back, which is also the gradient of the turn.
    Returns (q, k): new tensors, or ``q_out`` / ``k_out``, which may be the inputs
    themselves.  Any token and head strides; wraps ``mentat_rotary_apply``.  Gradients
    pass to ``q`` and ``k``; with outputs given, which torch could not follow, an input that
    requires one is refused."""
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        if q_out is not None or k_out is not None:
            raise RuntimeError("rotary: q_out and k_out pass no gradients on, and an input requires one")
        return _Turn.apply(q, k, positions, rotary, bool(inverse))
    n, _, d = q.shape
    dtype, dev = q.dtype, q.device
    q, rq = _operand("q", q, n, d, dtype, dev)
    _check_rotary(rotary, d, dev)
    positions = _check_positions(positions, n, dev)
    qo, rqo = _out_rows("q_out", q_out, q)
    ko, rk, rko = None, _NO_ROWS, _NO_ROWS
    if k is not None:
        k, rk = _operand("k", k, n, d, dtype, dev)
        ko, rko = _out_rows("k_out", k_out, k)
        if q_out is not None or k_out is not None:
            _check_apart(q_out=q_out, k=k, k_out=k_out)
            _check_apart(k_out=k_out, q=q)
    if n:
        _call(dev, "mentat_rotary_apply", _DT[dtype], d, n, *_rows(rq, rqo, rk, rko), positions.data_ptr(),
              rotary._ptrs[bool(inverse)])
    return qo, ko


class _Turn(torch.autograd.Function):
    """``rotary`` with gradients: the turn is linear, and turning back (with the same factor) is its transpose."""

    @staticmethod
    def forward(ctx, q, k, positions, rot, inverse):
        ctx.save_for_backward(positions)
        ctx.rot, ctx.inverse = rot, inverse
        ctx.set_materialize_grads(False)
        out = rotary(q, k, positions, rot, inverse=inverse)
        ctx.mark_non_differentiable(*(o for o, need in zip(out, ctx.needs_input_grad) if o is not None and not need))
        return out

    @staticmethod
    def backward(ctx, gq, gk):
        positions, = ctx.saved_tensors
        gq, gk = (g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad))
        if gq is None and gk is None:
            return (None,) * 5
        a, b = rotary(gk if gq is None else gq, None if gq is None else gk, positions, ctx.rot, inverse=not ctx.inverse)
        return (None, a, None, None, None) if gq is None else (a, b, None, None, None)


def rotary_append(cache, layer: int, rows: torch.Tensor, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                  positions: torch.Tensor, rotary, *, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Turns ``q`` (N, Hq, D; may be None) and ``k`` (N, Hkv, D) to ``positions`` (N,) and
    writes the keys and ``v`` into rows ``rows`` (N,) int64 of layer ``layer``
    of ``cache`` (a manager or a ``KVCacheView``): block * block_size + offset,
    distinct; -1 writes none.  Returns the turned queries.  The tables and lengths
    are not touched; ``PagedKVCacheManager.append_rotated`` keeps them.  Passes no
    gradients on, like every operator of a cache.  Wraps ``mentat_rotary_append``."""
    n, hkv, d = k.shape
    dev, dtype = cache.device, cache.dtype
    if d != cache.head_dim or hkv != cache.num_key_value_heads or v.shape[1] != hkv:
        raise ValueError("k or v shape does not match the cache geometry")
    _check_layer(layer, cache)
    k, rk = _operand("k", k, n, d, dtype, dev)
    v, rv = _operand("v", v, n, d, dtype, dev)
    _check_rotary(rotary, d, dev)
    positions = _check_positions(positions, n, dev)
    if rows.shape != (n,) or rows.dtype is not torch.int64 or rows.device != dev:
        raise ValueError(f"rows must be {n} int64 values on {dev}")
    rows = rows.contiguous()
    qo, rq, rqo = None, _NO_ROWS, _NO_ROWS
    if q is not None:
        q, rq = _operand("q", q, n, d, dtype, dev)
        qo, rqo = _out_rows("q_out", q_out, q)
        _check_apart(q_out=q_out, k=k, v=v)
    if n:
        _call(dev, "mentat_rotary_append", cache._desc_ptr, layer, n, rows.data_ptr(), *_rows(rq, rqo, rk, rv),
              positions.data_ptr(), rotary._ptrs[0])
    return qo


def _append_rotated(k_pool: torch.Tensor, v_pool: torch.Tensor, slots: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                    v: torch.Tensor, cache: int, layer: int, rotary: int) -> torch.Tensor:
    """``append_batched`` with ``q`` (N, Hq, D) and ``k`` turned to the index of their
    token in its sequence; returns the turned queries.  ``rotary`` is the id that
    ``register_cache`` gave a ``Rotary``.  Wraps ``mentat_kv_append_rotated_batched``."""
    mgr, rot = _cache(cache), _cache(rotary)
    n, d = k.shape[0], k.shape[2]
    dev = mgr.device
    _check_rotary(rot, mgr.head_dim, dev)
    slots = _check_ids("slots", slots, dev, n)
    (q, rq), (k, rk), (v, rv) = (_operand(name, t, n, d, mgr.dtype, dev) for name, t in (("q", q), ("k", k), ("v", v)))
    qo, rqo = _like(q)
    size = q.element_size()
    for a in range(0, n, 1024):
        part = [(p + a * s0 * size, s0, s1, h) for p, s0, s1, h in (rq, rqo, rk, rv)] if a else (rq, rqo, rk, rv)
        _call(dev, "mentat_kv_append_rotated_batched", mgr._desc_ptr, layer, slots.data_ptr() + 4 * a, min(n - a, 1024),
              *_rows(*part), None, rot._ptrs[0])
    if mgr.page_index is not None:
        _index_tails(mgr, layer, slots, n)
    return qo


append_rotated_op = torch.library.custom_op("mentat_b200::append_rotated", mutates_args=("k_pool", "v_pool"),
                                            device_types="cuda")(_append_rotated)


@append_rotated_op.register_fake
def _append_rotated_fake(k_pool, v_pool, slots, q, k, v, cache, layer, rotary):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def append_rotated(k_pool, v_pool, slots, q, k, v, cache, layer, rotary):
    if torch.compiler.is_compiling():
        return torch.ops.mentat_b200.append_rotated(k_pool, v_pool, slots, q, k, v, cache, layer, rotary)
    return _append_rotated(k_pool, v_pool, slots, q, k, v, cache, layer, rotary)


def _index_tails(mgr, layer: int, slots: torch.Tensor, n: int) -> None:
    """Indexes the pages that a batched append to ``slots`` has filled."""
    _call(mgr.device, "mentat_page_index_seqs", mgr._desc_ptr, layer, slots.data_ptr(),
          n, -1, 1, mgr.page_index._ptr)


def index_sequences(mgr, slots: torch.Tensor, first_page: int, max_pages: int, layer: int = -1) -> None:
    """Indexes the full pages ``first_page .. first_page + max_pages`` of the slots' sequences
    in ``layer`` (-1: every layer) into the cache's index.  Wraps ``mentat_page_index_seqs``."""
    index = _index_of(mgr)
    slots = _check_ids("slots", slots, mgr.device)
    if first_page < 0 or max_pages < 0:
        raise ValueError(f"pages {first_page} .. {first_page} + {max_pages} are no range of pages")
    first_page, max_pages = min(first_page, mgr.table_capacity), min(max_pages, mgr.table_capacity)  # no table has more
    step = max(1, 0x7fffffff // max(1, max_pages))
    for a in range(0, slots.shape[0], step):
        part = slots[a: a + step]
        _call(mgr.device, "mentat_page_index_seqs", mgr._desc_ptr, layer,
              part.data_ptr(), part.shape[0], first_page, max_pages, index._ptr)


def _workspace(cache, n: int) -> tuple:
    size = _lib.call("mentat_pages_workspace_bytes")(cache._desc_ptr, n)
    return torch.empty(size, dtype=torch.uint8, device=cache.device), size


MAX_SEQS_PER_PAGES_CALL = 1024


def fork_pages(cache, parents: torch.Tensor, children: torch.Tensor) -> None:
    """Every layer's table of slot ``parents[i]`` into slot ``children[i]``, with a
    reference on each page (int32 slots on the device; the children distinct, empty
    and no parents).  ``PagedKVCacheManager.fork_sequences`` keeps the host's mirror too.  Wraps
    ``mentat_kv_fork_batched``."""
    dev = cache.device
    parents = _check_ids("parents", parents, dev, limit=MAX_SEQS_PER_PAGES_CALL)
    children = _check_ids("children", children, dev, parents.shape[0])
    _call(dev, "mentat_kv_fork_batched", cache._desc_ptr, parents.data_ptr(), children.data_ptr(), parents.shape[0])


def free_pages(cache, slots: torch.Tensor, max_blocks: Optional[int] = None) -> None:
    """Releases every page of the (distinct) slots, as freeing them one after another
    would, the order of the free list included.  ``max_blocks``: the longest table, a
    launch-size hint.  Wraps ``mentat_kv_free_batched``."""
    dev = cache.device
    slots = _check_ids("slots", slots, dev, limit=MAX_SEQS_PER_PAGES_CALL)
    hint = cache.table_capacity if max_blocks is None else max_blocks
    ws, size = _workspace(cache, slots.shape[0])
    _call(dev, "mentat_kv_free_batched", cache._desc_ptr, slots.data_ptr(), slots.shape[0], hint,
          ws.data_ptr(), size)


def compact_pages(cache, src: torch.Tensor, dst: Optional[torch.Tensor], keep: torch.Tensor, cu: torch.Tensor,
                  max_keep: int, *, rotary=None, max_blocks: Optional[int] = None) -> None:
    """Sequence ``src[i]`` reduced to its positions ``keep[cu[i]:cu[i + 1]]``, which become
    positions 0, 1, ...: in place if ``dst`` is None, else as a new sequence in the
    empty slot ``dst[i]`` that shares the full pages at the front whose tokens stay
    where they are.  ``keep`` (total,) int32, or (layers, total) with a choice for each
    layer; ``cu`` (n + 1,) int32; ``max_keep`` the longest list.  With ``rotary``
    the keys are turned from their old position to the new one.
    ``PagedKVCacheManager.compact_sequences`` keeps the host's mirror too.  Wraps
    ``mentat_kv_compact``."""
    dev = cache.device
    src = _check_ids("src", src, dev, limit=MAX_SEQS_PER_PAGES_CALL)
    n = src.shape[0]
    dst = None if dst is None else _check_ids("dst", dst, dev, n)
    cu = _check_ids("cu", cu, dev, n + 1)
    if keep.dtype != torch.int32 or keep.device != dev or keep.dim() not in (1, 2) or \
            (keep.dim() == 2 and keep.shape[0] not in (1, cache.num_layers)):
        raise ValueError(f"keep must be int32 on {dev}, (total,) or (layers, total)")
    if keep.stride(-1) != 1:
        keep = keep.contiguous()
    per_layer = keep.dim() == 2 and keep.shape[0] > 1
    if rotary is not None:
        _check_rotary(rotary, cache.head_dim, dev)
    hint = cache.table_capacity if max_blocks is None else max_blocks
    ws, size = _workspace(cache, n)
    _call(dev, "mentat_kv_compact", cache._desc_ptr, src.data_ptr(),
          None if dst is None else dst.data_ptr(), n, keep.data_ptr(), keep.stride(0) if per_layer else 0, keep.shape[-1],
          cu.data_ptr(), max_keep, hint, None if rotary is None else rotary._ptrs[0], ws.data_ptr(), size)


def page_index(index, layer: int, blocks: torch.Tensor) -> None:
    """Indexes ``blocks`` (n,) int32 of layer ``layer`` from every row of each.  A
    manager's own index (``enable_page_index``) is kept by its appends.  Wraps
    ``mentat_page_index_blocks``."""
    c = index.cache
    blocks = _check_ids("blocks", blocks, c.device)
    _call(c.device, "mentat_page_index_blocks", c._desc_ptr, layer, blocks.data_ptr(),
          blocks.shape[0], index._ptr)


def page_bounds(index, layer: int, blocks: torch.Tensor) -> tuple:
    """What the index holds for ``blocks`` (n,): ``(low, high, exps)``, the bounds of their
    keys as float32 (n, Hkv, D) and their exponents int8 (n, Hkv).  Wraps
    ``mentat_page_bounds``."""
    c = index.cache
    blocks = _check_ids("blocks", blocks, c.device)
    n, h, d = blocks.shape[0], c.num_key_value_heads, c.head_dim
    low = torch.empty((n, h, d), dtype=torch.float32, device=c.device)
    high = torch.empty_like(low)
    exps = torch.empty((n, h), dtype=torch.int8, device=c.device)
    _call(c.device, "mentat_page_bounds", c._desc_ptr, layer, blocks.data_ptr(), n, index._ptr,
          low.data_ptr(), high.data_ptr(), exps.data_ptr())
    return low, high, exps


def sparse_decode(index, layer: int, slots: torch.Tensor, q: torch.Tensor, max_len: int, budget: int, *, sink: int = 1,
                  recent: int = 1, scale: Optional[float] = None, return_pages: bool = False):
    """Decode attention of ``q`` (N, Hq, D) over at most ``budget`` pages of each of the
    sequences in ``slots`` (N,) int32, chosen for each KV head by the scores of
    ``index`` (``PageIndex``): the first ``sink`` and last ``recent`` always, then the
    highest.  ``max_len``: the longest of the lengths.  Returns (N, Hq, D), with
    ``return_pages`` also the chosen pages, int32 (N, Hkv, budget), rising, then -1.
    Wraps ``mentat_sparse_decode``."""
    c = index.cache
    n, hq, d = q.shape
    if d != c.head_dim or hq % c.num_key_value_heads:
        raise ValueError("q shape does not match the cache geometry")
    q = _check_rows("q", q, n, d, c.dtype, c.device)
    if q.stride(1) != d:
        q = q.contiguous()
    slots = _check_ids("slots", slots, c.device, n)
    if recent < 1 or sink < 0 or sink + recent > budget:
        raise ValueError(f"sink {sink} >= 0 and recent {recent} >= 1 pages must fit in the budget of {budget}")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    pages = slots.new_empty((n, c.num_key_value_heads, budget)) if return_pages else None
    if n:
        size = index.workspace_bytes(n, max_len, budget)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        _call(c.device, "mentat_sparse_decode", c._desc_ptr, layer, index._ptr,
              slots.data_ptr(), n, q.data_ptr(), q.stride(0), hq, out.data_ptr(), out.stride(0),
              default_scale(d) if scale is None else scale, max_len, budget, sink, recent,
              None if pages is None else pages.data_ptr(), None if ws is None else ws.data_ptr(), size)
    return (out, pages) if return_pages else out


def _paged_sparse_decode(q: torch.Tensor, slots: torch.Tensor, max_len: int, cache: int, layer: int, scale: float,
                         budget: int, sink: int, recent: int) -> torch.Tensor:
    """``sparse_decode`` over a manager's own index, the cache given by its id."""
    return sparse_decode(_index_of(_cache(cache)), layer, slots, q, max_len, budget, sink=sink, recent=recent, scale=scale)


def _index_of(mgr):
    if mgr.page_index is None:
        raise RuntimeError("the cache has no page index: call enable_page_index() first")
    return mgr.page_index


paged_sparse_decode_op = torch.library.custom_op("mentat_b200::paged_sparse_decode", mutates_args=(),
                                                 device_types="cuda")(_paged_sparse_decode)


@paged_sparse_decode_op.register_fake
def _paged_sparse_decode_fake(q, slots, max_len, cache, layer, scale, budget, sink, recent):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def paged_sparse_decode(q, slots, max_len, cache, layer, scale, budget, sink, recent):
    if torch.compiler.is_compiling():
        return torch.ops.mentat_b200.paged_sparse_decode(q, slots, max_len, cache, layer, scale, budget, sink, recent)
    return _paged_sparse_decode(q, slots, max_len, cache, layer, scale, budget, sink, recent)
