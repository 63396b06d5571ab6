"""Rotary positions of the paged decode path.

:class:`Rotary` holds what the kernels read: the angle per position of every pair
of dimensions (64 bits, on the device) and how the pairs lie in a head.  The
operators that use it are ``ops.rotary`` (turn q and k),
``ops.rotary_append`` (turn q, write turned keys and the values into cache
rows), ``PagedKVCacheManager.append_rotated`` / ``append_rotated_batched`` and
``compact_sequences``.  The reference leaves rotary positions to the model's
modules (``qwen3_adapter.py:71-93,195-221``, ``llama_adapter.py:70,152``).
"""

from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import numpy as np
import torch

from . import _lib, ops

MAX_HEAD_DIM = 1024


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                seq_len: Optional[int] = None) -> tuple:
    """Angles per position of the ``rotary_dim / 2`` pairs (float64 array), and the
    factor that turned values are multiplied by, for a ``rope_scaling`` mapping
    of a model's configuration.  ``rope_type``:

    * ``"default"``: ``base ** (-2 i / rotary_dim)``.
    * ``"linear"``: positions divided by ``factor``.
    * ``"dynamic"``: the base raised so that the longest wavelength covers
      ``seq_len`` tokens (at least ``original_max_position_embeddings``).
    * ``"llama3"``: wavelengths above ``original / low_freq_factor`` divided by
      ``factor``, those below ``original / high_freq_factor`` kept, a linear blend
      between.
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times within the original
      context kept, fewer than ``beta_slow`` divided by ``factor``, a linear ramp
      over the pairs between; the factor is ``attention_factor`` or
      ``0.1 ln(factor) + 1``.
    * ``"longrope"``: every pair divided by its entry of ``long_factor``, or of
      ``short_factor`` where ``seq_len`` is within the original context; the
      factor is ``attention_factor`` or ``sqrt(1 + ln(factor) / ln(original))``.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} is not a positive even number")
    if not base > 0:
        raise ValueError(f"rotary base {base} is not positive")
    sc = dict(scaling or {})
    kind = sc.get("rope_type", sc.get("type", "default"))
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    f = np.float64(base) ** (-2.0 * i / rotary_dim)
    if kind == "default":
        return f, 1.0

    def need(key):
        if sc.get(key) is None:
            raise ValueError(f"rope_scaling of type {kind!r} needs {key!r}")
        return sc[key]

    if kind == "linear":
        return f / float(need("factor")), 1.0
    original = int(need("original_max_position_embeddings"))
    if kind == "dynamic":
        x = float(need("factor")) * max(seq_len or 0, original) / original - (float(sc["factor"]) - 1.0)
        if rotary_dim == 2:
            return f, 1.0
        return np.float64(base * x ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * i / rotary_dim), 1.0
    if kind == "llama3":
        factor, lo, hi = (float(need(k)) for k in ("factor", "low_freq_factor", "high_freq_factor"))
        if not hi > lo:
            raise ValueError("rope_scaling: high_freq_factor must be above low_freq_factor")
        turns = original * f / (2 * math.pi)  # within the original context
        keep = np.clip((turns - lo) / (hi - lo), 0.0, 1.0)
        return keep * f + (1.0 - keep) * f / factor, 1.0
    if kind == "yarn":
        factor = float(need("factor"))
        fast, slow = float(sc.get("beta_fast") or 32.0), float(sc.get("beta_slow") or 1.0)

        def pair_of(turns):  # the pair that turns so often within the original context
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        first, last = pair_of(fast), pair_of(slow)
        if sc.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotary_dim - 1)
        ramp = np.clip((i - first) / max(last - first, 1e-3), 0.0, 1.0)
        scale = sc.get("attention_factor")
        if scale is None:
            def strength(m):
                return 1.0 if factor <= 1.0 else 0.1 * float(m) * math.log(factor) + 1.0
            if sc.get("mscale") and sc.get("mscale_all_dim"):
                scale = strength(sc["mscale"]) / strength(sc["mscale_all_dim"])
            else:
                scale = strength(1.0)
        return f * (1.0 - ramp) + f / factor * ramp, float(scale)
    if kind == "longrope":
        long = seq_len is None or seq_len > original
        ext = np.asarray(need("long_factor" if long else "short_factor"), np.float64)
        if ext.shape != f.shape:
            raise ValueError(f"rope_scaling: {len(f)} factors are needed, {ext.size} are given")
        scale = sc.get("attention_factor")
        if scale is None:
            factor = float(need("factor"))
            scale = 1.0 if factor <= 1.0 else math.sqrt(1.0 + math.log(factor) / math.log(original))
        return f / ext, float(scale)
    raise ValueError(f"unknown rope_type {kind!r}")


class Rotary:
    """Rotary positions of heads of ``head_dim`` dimensions.

    Dimensions ``offset .. offset + rotary_dim`` of a head are turned; the others
    pass through.  ``interleaved`` pairs dimensions (2i, 2i + 1), otherwise
    (i, i + rotary_dim / 2).  The angles come from ``base`` and ``scaling``
    (:func:`frequencies`) or are given as ``inv_freq`` (radians per position, a
    tensor of rotary_dim / 2; kept in 64 bits), with ``attention_scaling`` the
    factor of the turned values."""

    def __init__(self, head_dim: int, *, rotary_dim: Optional[int] = None, offset: int = 0, base: float = 10000.0,
                 interleaved: bool = False, scaling: Optional[dict] = None, seq_len: Optional[int] = None,
                 inv_freq: Optional[torch.Tensor] = None, attention_scaling: Optional[float] = None,
                 device: str | torch.device = "cuda"):
        if not 0 < head_dim <= MAX_HEAD_DIM:
            raise ValueError(f"head_dim {head_dim} is not within 1 .. {MAX_HEAD_DIM}")
        if inv_freq is None:
            f, scale = frequencies(head_dim - offset if rotary_dim is None else rotary_dim, base, scaling, seq_len)
            inv_freq = torch.from_numpy(f).to(device)
            attention_scaling = scale if attention_scaling is None else attention_scaling
        elif scaling is not None:
            raise ValueError("give inv_freq or scaling, not both")
        elif rotary_dim is not None and rotary_dim != 2 * inv_freq.numel():
            raise ValueError(f"rotary_dim {rotary_dim} does not match {inv_freq.numel()} frequencies")
        if inv_freq.dim() != 1 or inv_freq.numel() == 0 or not inv_freq.is_floating_point():
            raise ValueError("inv_freq must be a vector of floating-point numbers")
        self.inv_freq = inv_freq.detach().to(torch.float64).contiguous()
        self.head_dim, self.rotary_dim, self.offset = head_dim, 2 * self.inv_freq.numel(), offset
        if offset < 0 or offset + self.rotary_dim > head_dim:
            raise ValueError(f"rotary dimensions {offset} .. {offset + self.rotary_dim} are outside a head of {head_dim}")
        self.interleaved = bool(interleaved)
        self.attention_scaling = 1.0 if attention_scaling is None else float(attention_scaling)
        self._args = tuple(_lib.Rotary(self.inv_freq.data_ptr(), self.rotary_dim // 2, offset, int(self.interleaved),
                                       inverse, self.attention_scaling) for inverse in (0, 1))
        self._ptrs = tuple(C.addressof(a) for a in self._args)
        self.op_id = ops.register_cache(self)  # the id that torch operators take

    @classmethod
    def from_module(cls, rotary_emb, head_dim: int) -> "Rotary":
        """The angles of a Hugging Face rotary module (its ``inv_freq`` and
        ``attention_scaling``; Llama and Qwen3 pair i with i + rotary_dim / 2).
        A module of type ``dynamic`` or ``longrope`` is refused: it replaces its
        frequencies while it runs, when a sequence passes the original context, and
        what it holds now is right for some lengths only.  For one length its
        angles are ``Rotary(head_dim, base=..., scaling=..., seq_len=...)``."""
        kind = getattr(rotary_emb, "rope_type", None)
        if kind in ("dynamic", "longrope"):
            raise ValueError(f"rope_type {kind!r} changes its frequencies with the length of the sequence: "
                             "give Rotary its base, scaling and seq_len instead")
        return cls(head_dim, inv_freq=rotary_emb.inv_freq,
                   attention_scaling=getattr(rotary_emb, "attention_scaling", 1.0))

    @property
    def device(self) -> torch.device:
        return self.inv_freq.device

    def __call__(self, q, k, positions, **kw):
        return ops.rotary(q, k, positions, self, **kw)
