"""Rotary positions on the device against the definition in 64 bits (``oracle.cache_ops``)."""

from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle.cache_ops import turn, turn_tolerance
from tests.gpu_util import TORCH_DT

pytestmark = pytest.mark.gpu


def _near(got, x, positions, rot, *, inverse=False, what=""):
    """got against x turned, element by element."""
    kw = dict(offset=rot.offset, interleaved=rot.interleaved, scale=rot.attention_scaling)
    f = rot.inv_freq.cpu().numpy()
    x = x.double().cpu().numpy()
    want = turn(x, positions.cpu().numpy(), f, inverse=inverse, **kw)
    tol = turn_tolerance(x, f, torch.finfo(got.dtype).eps, **kw)(want)
    # fp16 steps below 2^-14 are 2^-24 wide
    tol = tol + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    off = np.abs(got.double().cpu().numpy() - want) - tol
    assert np.all(off <= 0), (what, float(off.max()), np.unravel_index(off.argmax(), off.shape))
    passed = np.ones(rot.head_dim, bool)
    passed[rot.offset: rot.offset + rot.rotary_dim] = False
    np.testing.assert_array_equal(got.double().cpu().numpy()[..., passed], x[..., passed])


def _positions(n, rng):
    p = rng.integers(0, 1 << 20, n)
    special = [0, 1, -1, 131071, 1 << 20, -(1 << 20), (1 << 31) + 7, 1 << 33]
    p[: min(n, len(special))] = special[: n]
    return torch.tensor(p, device="cuda")


CASES = [  # tokens, query heads, kv heads, head_dim, rotary_dim, offset, interleaved
    (1, 16, 8, 128, 128, 0, False), (1, 1, 1, 2, 2, 0, True), (3, 4, 2, 64, 64, 0, True), (17, 5, 1, 64, 32, 0, False),
    (8, 8, 8, 80, 48, 16, True), (9, 3, 3, 96, 24, 72, False), (33, 2, 1, 37, 6, 3, True), (33, 2, 1, 37, 6, 3, False),
    (5, 64, 8, 256, 256, 0, False), (257, 32, 8, 128, 64, 64, True), (2, 1, 1, 1024, 1024, 0, False),
    (1000, 10, 2, 128, 126, 1, False),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_rotary_matches_definition(case, dtype):
    from mentat_b200 import Rotary, ops
    n, hq, hkv, d, rd, off, il = case
    rng = np.random.default_rng(d + n)
    rot = Rotary(d, rotary_dim=rd, offset=off, interleaved=il, base=5e5)
    pos = _positions(n, rng)
    # strided parts of one projection; with one element in front nothing is aligned
    for lead in (0, 1):
        flat = torch.from_numpy(rng.standard_normal(n * (hq + 2 * hkv) * d + lead)).cuda().to(TORCH_DT[dtype])
        qkv = flat[lead:].view(n, hq + 2 * hkv, d)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
        before = flat.clone()
        qo, ko = ops.rotary(q, k, pos, rot)
        _near(qo, q, pos, rot, what="q")
        _near(ko, k, pos, rot, what="k")
        assert torch.equal(flat, before)
        back, none = ops.rotary(q, None, pos.to(torch.int32) if int(pos.abs().max()) < 1 << 31 else pos, rot,
                                inverse=True)
        assert none is None
        _near(back, q, pos, rot, inverse=True, what="inverse")
        # in place: the same values, and what lies between the rows untouched
        r1, r2 = ops.rotary(q, k, pos, rot, q_out=q, k_out=k)
        assert r1 is q and r2 is k and torch.equal(q, qo) and torch.equal(k, ko)
        assert torch.equal(qkv[:, hq + hkv:], before[lead:].view(n, hq + 2 * hkv, d)[:, hq + hkv:])


def test_rotary_layouts_of_rows():
    """Heads outside tokens, rows repeated by a stride of zero, a tensor without tokens or heads, a
    last dimension that is not contiguous, outputs of another layout."""
    from mentat_b200 import Rotary, ops
    g = torch.Generator(device="cuda").manual_seed(0)
    rot, pos = Rotary(64), torch.arange(7, device="cuda") * 1000
    x = torch.randn((6, 7, 64), generator=g, device="cuda")
    _near(ops.rotary(x.transpose(0, 1), None, pos, rot)[0], x.transpose(0, 1), pos, rot)
    one = x[:1, :1].expand(7, 5, 64)
    _near(ops.rotary(one, one, pos, rot)[1], one, pos, rot)
    y = torch.randn((7, 3, 128), generator=g, device="cuda")[..., ::2]
    _near(ops.rotary(y, None, pos, rot)[0], y, pos, rot)
    out = torch.zeros((3, 7, 64), device="cuda").transpose(0, 1)
    assert ops.rotary(y.contiguous(), None, pos, rot, q_out=out)[0] is out
    _near(out, y, pos, rot)
    assert ops.rotary(y[:0], y[:0], pos[:0], rot)[0].shape == (0, 3, 64)
    assert ops.rotary(y[:, :0], None, pos, rot)[0].shape == (7, 0, 64)


def test_rotary_inverse_is_the_gradient():
    """<turn(x), y> = <x, inverse(y)>, and the slope of <turn(x), y> by differences."""
    from mentat_b200 import Rotary, ops
    g = torch.Generator(device="cuda").manual_seed(1)
    rot = Rotary(32, rotary_dim=24, offset=4, attention_scaling=1.3)
    pos = torch.tensor([0, 5, 70000], device="cuda")
    x, y, dx = (torch.randn((3, 2, 32), generator=g, device="cuda") for _ in range(3))
    grad = ops.rotary(y, None, pos, rot, inverse=True)[0].double()
    a = (ops.rotary(x, None, pos, rot)[0].double() * y.double()).sum()
    # 192 products of values below 6, each turned value off by less than 10 2^-24 * 2 * 6 * 1.3
    bound = 192 * 6 * 10 * 2.0 ** -24 * 12 * 1.3
    assert abs(a - (x.double() * grad).sum()) < bound
    h = 0.5  # the turn is linear: any step
    up, down = (ops.rotary(x + s * h * dx, None, pos, rot)[0].double() for s in (1, -1))
    slope = ((up - down) * y.double()).sum() / (2 * h)
    # the inputs' sums are rounded too: 2^-24 * 9 each, divided by the step
    assert abs(slope - (dx.double() * grad).sum()) < 3 * bound / h


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hkv,d,bs,rd,il", [(8, 128, 16, 128, False), (2, 64, 4, 64, True), (1, 37, 3, 10, False)])
def test_rotary_append_rows(dtype, hkv, d, bs, rd, il):
    from mentat_b200 import KVCacheView, Rotary, ops
    rng = np.random.default_rng(3)
    L, blocks, n, hq, layer = 2, 9, 11, 2 * hkv, 1
    g = torch.Generator(device="cuda").manual_seed(5)
    dt = TORCH_DT[dtype]
    kp, vp = (torch.randn((L, blocks, bs, hkv, d), generator=g, device="cuda").to(dt) for _ in range(2))
    kp0, vp0 = kp.clone(), vp.clone()
    c = KVCacheView(kp, vp)
    rot = Rotary(d, rotary_dim=rd, interleaved=il, attention_scaling=0.75)
    q, k, v = (torch.randn((n, h, d), generator=g, device="cuda").to(dt) for h in (hq, hkv, hkv))
    pos = _positions(n, rng)
    rows = torch.from_numpy(rng.permutation(blocks * bs)[:n]).cuda()
    rows[4] = -1
    rows[7] = blocks * bs - 1 if blocks * bs - 1 not in rows.tolist() else rows[7]
    qo = ops.rotary_append(c, layer, rows, q, k, v, pos, rot)
    _near(qo, q, pos, rot)
    live = rows >= 0
    at = rows[live]
    _near(kp[layer].view(-1, hkv, d)[at], k[live], pos[live], rot)
    assert torch.equal(vp[layer].view(-1, hkv, d)[at], v[live])
    # nothing else written
    kp[layer].view(-1, hkv, d)[at] = kp0[layer].view(-1, hkv, d)[at]
    vp[layer].view(-1, hkv, d)[at] = vp0[layer].view(-1, hkv, d)[at]
    assert torch.equal(kp, kp0) and torch.equal(vp, vp0)
    c.check()
    # rows outside the pool are recorded and not written
    bad = torch.tensor([blocks * bs, -2, 0], device="cuda")
    ops.rotary_append(c, layer, bad, None, k[:3], v[:3], pos[:3], rot)
    with pytest.raises(AssertionError, match="outside the pool"):
        c.check()
    assert torch.equal(vp[layer].view(-1, hkv, d)[0], v[2])


def test_rotary_on_another_stream_and_in_a_graph():
    from mentat_b200 import Rotary, ops
    g = torch.Generator(device="cuda").manual_seed(2)
    rot = Rotary(128, base=1e6)
    q = torch.randn((40, 8, 128), generator=g, device="cuda").bfloat16()
    pos = torch.arange(40, device="cuda")
    want = ops.rotary(q, None, pos, rot)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.rotary(q, None, pos, rot)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(q, None, pos, rot)[0]
    pos.add_(1000)
    graph.replay()
    assert torch.equal(out, ops.rotary(q, None, pos, rot)[0]) and not torch.equal(out, want)


# 1 / 2 pi to 60 digits
INV_TWO_PI = Fraction(159154943091895335768883763372514362034459645740456448747667, 10 ** 60)


@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_angles_of_any_position(scale):
    """Cosines and sines (the turn of (1, 0) and of (0, 1)) of near and far positions against exact arithmetic.

    The fraction of a turn is off by 2^-42, the angle by 2^-39.3.  sincospif is off by at most 2 units in the last
    place (2^-23 for values up to 1), the added remainder's product and sum by 2^-24 each of at most 1 and a second-order
    term of 2^-47; a power of two as the factor adds nothing and the products with 0 and 1 are exact.  Below
    2^-23 + 2^-24 + 2^-24 + 2^-38."""
    from mentat_b200 import Rotary, ops
    d = 128
    rot = Rotary(d, base=5e5, attention_scaling=scale)
    rng = np.random.default_rng(0)
    pos = [0, 1, -1, 7, 4095, 131071, 1 << 20, -(1 << 20) - 3, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, -(1 << 32) - 1,
           (1 << 40) + 12345, (1 << 53) + 1, -(1 << 53) - 1, (1 << 62) + 987654321, (1 << 63) - 1, -(1 << 63)]
    pos += [int(v) for v in rng.integers(-(1 << 62), 1 << 62, 20)] + [int(v) for v in rng.integers(0, 1 << 20, 200)]
    x = torch.zeros((len(pos), 2, d), device="cuda")
    x[:, 0, : d // 2] = 1.0
    x[:, 1, d // 2:] = 1.0
    got = ops.rotary(x, None, torch.tensor(pos, dtype=torch.int64, device="cuda"), rot)[0].double().cpu().numpy()
    back = ops.rotary(x, None, torch.tensor(pos, dtype=torch.int64, device="cuda"), rot, inverse=True)[0].double().cpu().numpy()
    turns = np.array([[float((lambda t: t - round(t))(p * Fraction(f) * INV_TWO_PI)) for f in rot.inv_freq.tolist()] for p in pos])
    cos, sin = np.cos(2 * np.pi * turns) * scale, np.sin(2 * np.pi * turns) * scale
    tol = (2.0 ** -23 + 2.0 ** -23 + 2.0 ** -38) * scale
    h = d // 2
    for out, s in ((got, sin), (back, -sin)):
        for part, want in ((out[:, 0, :h], cos), (out[:, 0, h:], s), (out[:, 1, :h], -s), (out[:, 1, h:], cos)):
            assert np.abs(part - want).max() <= tol, np.unravel_index(np.abs(part - want).argmax(), part.shape)


def test_rotary_passes_gradients_on():
    """Against the formula's transpose in 64 bits and against differences; q alone, k alone, both, neither."""
    from mentat_b200 import Rotary, ops
    g = torch.Generator(device="cuda").manual_seed(2)
    rot = Rotary(32, rotary_dim=24, offset=4, interleaved=True, attention_scaling=1.3)
    pos = torch.tensor([0, 5, 70000], device="cuda")
    q, gq = (torch.randn((3, 4, 32), generator=g, device="cuda") for _ in range(2))
    k, gk = (torch.randn((3, 2, 32), generator=g, device="cuda") for _ in range(2))
    plain = ops.rotary(q, k, pos, rot)
    for need_q, need_k in ((True, True), (True, False), (False, True)):
        a, b = q.clone().requires_grad_(need_q), k.clone().requires_grad_(need_k)
        oq, ok = ops.rotary(a, b, pos, rot)
        assert torch.equal(oq, plain[0]) and torch.equal(ok, plain[1])
        torch.autograd.backward([oq, ok] if need_q and need_k else [oq] if need_q else [ok],
                                [gq, gk] if need_q and need_k else [gq] if need_q else [gk])
        for x, up in ((a, gq), (b, gk)):
            if x.requires_grad:
                _near(x.grad, up, pos, rot, inverse=True, what="gradient")
            else:
                assert x.grad is None
    # turned back, alone, a gradient of stride zero, and one output that nothing uses
    a = q.clone().requires_grad_()
    out, none = ops.rotary(a, None, pos, rot, inverse=True)
    assert none is None
    out.sum().backward()
    _near(a.grad, torch.ones_like(q), pos, rot, what="gradient of the turn back")
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    ops.rotary(a, b, pos, rot)[1].backward(gk)
    assert a.grad is None
    _near(b.grad, gk, pos, rot, inverse=True)
    # the slope by differences: the turn is linear, so any step; 384 products of values below 6 * 1.3 * 2, each turned
    # value off by less than 10 2^-24 of that, and the inputs' sums by 2^-24 * 9, over the step
    a = q.clone().requires_grad_()
    (ops.rotary(a, None, pos, rot)[0] * gq).sum().backward()
    dx, h = torch.randn((3, 4, 32), generator=g, device="cuda"), 0.5
    up, down = (ops.rotary(q + s * h * dx, None, pos, rot)[0].double() for s in (1, -1))
    slope = ((up - down) * gq.double()).sum() / (2 * h)
    assert abs(slope - (dx.double() * a.grad.double()).sum()) < 3 * 384 * 6 * 10 * 2.0 ** -24 * 12 * 1.3 / h
    # second order: the gradient is a turn of its own
    a = q.clone().requires_grad_()
    y = gq.clone().requires_grad_()
    grad, = torch.autograd.grad((ops.rotary(a, None, pos, rot)[0] * y).sum(), a, create_graph=True)
    again, = torch.autograd.grad((grad * dx).sum(), y)
    _near(again, dx, pos, rot, what="second order")
    # outputs of the caller's take none; without gradients they are as before
    with pytest.raises(RuntimeError, match="q_out"):
        ops.rotary(q.clone().requires_grad_(), None, pos, rot, q_out=torch.empty_like(q))
    with torch.no_grad():
        assert torch.equal(ops.rotary(q.clone().requires_grad_(), None, pos, rot, q_out=torch.empty_like(q))[0], plain[0])


def test_gradients_in_a_graph():
    """Forward and backward pass captured together, beside an eager graph of the same leaves that is still alive, and
    replayed over new values."""
    from mentat_b200 import Rotary, ops
    g = torch.Generator(device="cuda").manual_seed(3)
    rot, pos = Rotary(64), torch.arange(5, device="cuda") * 1001
    q, k = (torch.randn((5, h, 64), generator=g, device="cuda").requires_grad_() for h in (4, 2))
    up = [torch.randn((5, h, 64), generator=g, device="cuda") for h in (4, 2)]

    def step():
        return torch.autograd.grad(ops.rotary(q, k, pos, rot), (q, k), up)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        alive = ops.rotary(q, k, pos, rot)
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    for _ in range(2):
        for t in up:
            t.normal_(generator=g)
        graph.replay()
        for a, b, name in zip(got, up, "qk"):
            _near(a, b, pos, rot, inverse=True, what=name)
    assert torch.equal(torch.autograd.grad(alive, (q, k), up)[0], got[0])


def test_outputs_require_gradients_as_their_inputs_do():
    from mentat_b200 import Rotary, ops
    rot, pos = Rotary(64), torch.arange(3, device="cuda")
    for need in ((True, False), (False, True), (True, True), (False, False)):
        q, k = (torch.ones((3, 2, 64), device="cuda").requires_grad_(n) for n in need)
        assert tuple(t.requires_grad for t in ops.rotary(q, k, pos, rot)) == need
