"""rope.rotary against the rotation in 64 bits.

Bound of a rotated value y = s (u cos a -+ w sin a): its rounding to the
output's type, half a step (finfo.eps / 2) of y; and, in fp32, the rounding of
the fraction of a turn (2^-25 of at most half a turn: pi 2^-25 radians), of sine
and cosine (4 steps of 2^-24), of their scaling, of two products and a sum:
together below 12 * 2^-24 of s (|u| + |w|)."""
from __future__ import annotations

import pytest
import torch

from pyramidkv import rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _ref(x, pos, freqs, axes, interleaved, scale, inverse):
    """[value, bound of the fp32 part] in 64 bits."""
    P = sum(axes)
    pos = pos.reshape(x.shape[0], -1).double()
    axis = [i for i, n in enumerate(axes) for _ in range(n)]
    a = (pos[:, axis] * freqs)[:, None] * (-1 if inverse else 1)
    y, e = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    iu, iw = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    u, w = x[..., iu].double(), x[..., iw].double()
    y[..., iu] = scale * (u * a.cos() - w * a.sin())
    y[..., iw] = scale * (u * a.sin() + w * a.cos())
    e[..., iu] = e[..., iw] = scale * (u.abs() + w.abs()) * 12 * 2.0 ** -24
    return y, e


def _check(got, x, *args):
    y, e = _ref(x, *args)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    # (fp16's smallest steps are absolute)
    u = torch.finfo(x.dtype).eps / 2
    bound = e + u * (y.abs() + e) + (2.0 ** -25 if x.dtype == HF else 0.0)
    over = (got.double() - y).abs() - bound
    assert (over <= 0).all(), over.max().item()
    P = sum(args[2])
    assert torch.equal(got[..., 2 * P:], x[..., 2 * P:])


CASES = [  # rows, heads, kv heads, D, axes, interleaved, far
    (1, 1, 0, 2, (1,), True, 10), (1, 1, 1, 2, (1,), False, 10),
    (5, 3, 1, 64, (32,), True, 1 << 20), (5, 3, 1, 64, (32,), False, 1 << 20),
    (333, 12, 0, 128, (22, 21, 21), True, 120), (333, 12, 3, 128, (22, 21, 21), False, 120),
    (17, 4, 4, 80, (16,), False, 5000), (17, 4, 4, 80, (16,), True, 5000),   # part of the head, 16-byte pieces
    (17, 4, 4, 80, (13,), False, 5000), (17, 4, 2, 80, (13,), True, 5000),   # part of it, odd pairs
    (1031, 5, 1, 96, (0, 48), True, 1 << 31), (2500, 2, 1, 256, (1, 2, 3, 122), False, 1 << 31),
    (4099, 1, 1, 512, (256,), True, 1000),
]


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=str)
@pytest.mark.parametrize("rows,heads,kv,D,axes,interleaved,far", CASES)
def test_rotary(rows, heads, kv, D, axes, interleaved, far, dtype):
    qkv = torch.randn(rows, heads + 2 * kv, D, device=DEV).to(dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv] if kv else None
    pos = torch.randint(-far, far, (rows, len(axes)), device=DEV)
    f = torch.cat([rope.rotary_frequencies(2 * n, device=DEV)[0] for n in axes if n])
    for inverse in (False, True):
        out = rope.rotary(q, pos, f, k=k, axes=axes, interleaved=interleaved, scale=1.25, inverse=inverse)
        args = (pos, f, axes, interleaved, 1.25, inverse)
        if kv:
            _check(out[0], q, *args)
            _check(out[1], k, *args)
        else:
            _check(out, q, *args)


@pytest.mark.parametrize("offset", [0, 1, 8], ids=lambda n: f"column{n}")
def test_rotary_strides(offset):
    """Rows and heads apart, beginning at a column that 16-byte reads allow or not."""
    buf = torch.randn(9, 11, 7, 200, device=DEV).to(BF)
    q = buf[:, 3, ::2, offset:offset + 128]
    pos = torch.randint(0, 50000, (9,), dtype=torch.int32, device=DEV)
    f, s = rope.rotary_frequencies(64, scaling="parts", factor=8.0, trained_length=2048, device=DEV)
    for interleaved in (True, False):
        _check(rope.rotary(q, pos, f, interleaved=interleaved, scale=s), q, pos, f, (32,), interleaved, s, False)


def test_rotary_of_more_rows_than_a_launch_has_workgroups():
    """256 pairs are a workgroup a row: more rows than 2^32 threads hold."""
    rows = 0xffffffff // 256 + 3
    q = torch.zeros(rows, 1, 512, device=DEV, dtype=BF)
    at = torch.tensor([0, 1, rows - 4, rows - 3, rows - 2, rows - 1], device=DEV)
    q[at] = torch.randn(6, 1, 512, device=DEV).to(BF)
    pos = torch.arange(rows, device=DEV)
    f = rope.rotary_frequencies(512, device=DEV)[0]
    got = rope.rotary(q, pos, f)
    _check(got[at], q[at], pos[at], f, (256,), True, 1.0, False)


def test_rotary_of_empty_inputs():
    f = rope.rotary_frequencies(64, device=DEV)[0]
    pos = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert rope.rotary(torch.empty(0, 4, 64, dtype=BF, device=DEV), pos, f).shape == (0, 4, 64)
    pos = torch.zeros(3, dtype=torch.int64, device=DEV)
    q, k = torch.empty(3, 0, 64, dtype=BF, device=DEV), torch.randn(3, 2, 64, device=DEV).to(BF)
    a, b = rope.rotary(q, pos, f, k=k)
    assert a.shape == q.shape and torch.equal(b, k)  # (position 0 turns nothing)


def test_rotary_keeps_infinities_to_their_pairs():
    x = torch.randn(4, 2, 64, device=DEV).to(BF)
    x[1, 0, 6], x[2, 1, 40] = float("inf"), float("nan")
    pos = torch.arange(4, device=DEV)
    f = rope.rotary_frequencies(64, device=DEV)[0]
    got = rope.rotary(x, pos, f)
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[1, 0, 6:8] = want[2, 1, 40:42] = True
    assert torch.equal(bad, want)


def test_rotary_agrees_with_the_packed_keys_rotation():
    """The rotation that the cache's keys get (fp32 tables): within half a step of bf16 and 12 * 2^-24 of the pair's sum each."""
    x = torch.randn(200, 1, 128, device=DEV).to(BF)
    pos = torch.stack([torch.randint(0, n, (200,), device=DEV) for n in (120, 30, 52)], dim=1)
    f = torch.cat([rope.rotary_frequencies(2 * n, device=DEV)[0] for n in (22, 21, 21)])
    a = rope.rotary(x, pos, f, axes=(22, 21, 21))
    b = rope.apply_rope_to_flat_k(x[:, 0], pos, rope.wan_freqs(128))
    y, e = _ref(x, pos, f, (22, 21, 21), True, 1.0, False)
    assert ((a[:, 0].double() - b.double()).abs() <= 2 * (e + 2.0 ** -8 * (y.abs() + e))[:, 0]).all()


# ---- gradients ------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_gradient(interleaved):
    """The gradient is the inverse rotation of the outputs', as the formula says
    and as differences measure it."""
    f, pos = rope.rotary_frequencies(48, device=DEV)[0], torch.randint(0, 9999, (31,), device=DEV)
    q = torch.randn(31, 6, 64, device=DEV, requires_grad=True)
    k = torch.randn(31, 2, 64, device=DEV, requires_grad=True)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    kw = dict(interleaved=interleaved, scale=1.5)
    out = rope.rotary(q, pos, f, k=k, **kw)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk))
    _check(dq, gq, pos, f, (24,), interleaved, 1.5, True)
    _check(dk, gk, pos, f, (24,), interleaved, 1.5, True)
    # the rotation is linear: a difference along d is exact but for rounding, at
    # most 12 * 2^-24 of each pair's sum on each of its two ends
    d = torch.randn_like(q)
    with torch.no_grad():
        diff = rope.rotary(q + d, pos, f, **kw).double() - rope.rotary(q - d, pos, f, **kw).double()
    size = (q.abs().max() + d.abs().max()).item() * 1.5 * 2 * 14 * 2.0 ** -24
    assert abs(((gq.double() * diff).sum() / 2 - (dq.double() * d.double()).sum()).item()) <= \
        size * gq.double().abs().sum().item() * 2
    # only one of the two is used; gradients that are not dense
    out = rope.rotary(q, pos, f, k=k, **kw)
    only, none = torch.autograd.grad(out[1], (k, q), gk, allow_unused=True)
    assert torch.equal(only, dk) and (none is None or not none.any())
    one = rope.rotary(q, pos, f, **kw)
    assert torch.equal(torch.autograd.grad(one, q, gq)[0], dq)
    wide = gq.expand(31, 6, 64) if gq.shape[0] == 1 else gq
    summed = torch.autograd.grad(rope.rotary(q, pos, f, **kw).sum(), q)[0]
    _check(summed, torch.ones_like(wide), pos, f, (24,), interleaved, 1.5, True)


def test_rotary_gradient_of_part_of_a_projection():
    """q and k out of one leaf: its gradient holds both, and zero for the rest."""
    f, pos = rope.rotary_frequencies(64, device=DEV)[0], torch.randint(0, 9999, (31,), device=DEV)
    qkv = torch.randn(31, 8, 64, device=DEV).to(BF).requires_grad_()
    q, k = rope.rotary(qkv[:, :4], pos, f, k=qkv[:, 4:6])
    (q.float().sum() + k.float().sum()).backward()
    ones = torch.ones(31, 6, 64, device=DEV, dtype=BF)
    _check(qkv.grad[:, :6].contiguous(), ones, pos, f, (32,), True, 1.0, True)
    assert not qkv.grad[:, 6:].any()


def test_rotary_second_gradient():
    f, pos = rope.rotary_frequencies(64, device=DEV)[0], torch.randint(0, 999, (7,), device=DEV)
    q = torch.randn(7, 2, 64, device=DEV, requires_grad=True)
    g = torch.randn(7, 2, 64, device=DEV, requires_grad=True)
    dq = torch.autograd.grad(rope.rotary(q, pos, f), q, g, create_graph=True)[0]
    h = torch.randn_like(q)
    _check(torch.autograd.grad(dq, g, h)[0], h, pos, f, (32,), True, 1.0, False)


# ---- streams, graphs, refusals ------------------------------------------------------
def test_rotary_replayed():
    f, pos = rope.rotary_frequencies(128, device=DEV)[0], torch.randint(0, 9999, (40,), device=DEV)
    q = torch.randn(40, 4, 128, device=DEV).to(BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope.rotary(q, pos, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope.rotary(q, pos, f)
    for i in range(4):
        q.copy_(torch.randn(40, 4, 128, device=DEV))
        pos.copy_(torch.randint(0, 9999, (40,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rope.rotary(q, pos, f))


def test_rotary_gradient_replayed():
    """Forward and backward in one graph, of leaves that no eager result uses."""
    f, pos = rope.rotary_frequencies(64, device=DEV)[0], torch.randint(0, 9999, (40,), device=DEV)

    def step(q, k, g):
        out = rope.rotary(q, pos, f, k=k, interleaved=False)
        return torch.autograd.grad(out, (q, k), g)

    def leaves():
        return [torch.randn(40, h, 64, device=DEV).to(BF).requires_grad_() for h in (4, 2)]

    g = [torch.randn(40, h, 64, device=DEV).to(BF) for h in (4, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves(), g)
    torch.cuda.synchronize()
    q, k = leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dq, dk = step(q, k, g)
    for i in range(4):
        for x in g:
            x.copy_(torch.randn_like(x))
        pos.copy_(torch.randint(0, 9999, (40,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        eq, ek = step(*leaves(), g)
        assert torch.equal(dq, eq) and torch.equal(dk, ek)


Z = lambda *s, dtype=BF, device=DEV: torch.zeros(s, dtype=dtype, device=device)
REFUSED = {
    "q of two dimensions": lambda: dict(q=Z(4, 64)),
    "q of float64": lambda: dict(q=Z(4, 2, 64, dtype=torch.float64)),
    "columns apart": lambda: dict(q=Z(4, 2, 128)[..., ::2]),
    "k of another type": lambda: dict(k=Z(4, 2, 64, dtype=HF)),
    "k of other rows": lambda: dict(k=Z(5, 2, 64)),
    "k of another head_dim": lambda: dict(k=Z(4, 2, 32)),
    "k on the host": lambda: dict(k=Z(4, 2, 64, device="cpu")),
    "positions on the host": lambda: dict(positions=Z(4, dtype=torch.int64, device="cpu")),
    "positions of float": lambda: dict(positions=Z(4, dtype=F32)),
    "positions of other rows": lambda: dict(positions=Z(3, dtype=torch.int64)),
    "positions of two columns": lambda: dict(positions=Z(4, 2, dtype=torch.int64)),
    "one column for two axes": lambda: dict(axes=(16, 16)),
    "frequencies of fp32": lambda: dict(freqs=Z(32, dtype=F32)),
    "frequencies on the host": lambda: dict(freqs=Z(32, dtype=torch.float64, device="cpu")),
    "fewer frequencies than pairs": lambda: dict(freqs=Z(31, dtype=torch.float64), axes=(32,)),
    "more pairs than columns": lambda: dict(freqs=Z(33, dtype=torch.float64)),
    "no axes": lambda: dict(axes=()),
    "an axis of -1": lambda: dict(axes=(33, -1), positions=Z(4, 2, dtype=torch.int64)),
}


@pytest.mark.parametrize("name", REFUSED)
def test_rotary_refuses(name):
    kw = dict(q=Z(4, 2, 64), positions=Z(4, dtype=torch.int64), freqs=Z(32, dtype=torch.float64))
    kw.update(REFUSED[name]())
    with pytest.raises(RuntimeError):
        rope.rotary(kw.pop("q"), kw.pop("positions"), kw.pop("freqs"), **kw)


# ---- forward derivatives, batches --------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF], ids=str)
def test_rotary_forward_derivative(dtype):
    """The rotation is linear: the derivative along a tangent is the rotated
    tangent, for q, for k, and for the one of them that has one."""
    from torch.autograd import forward_ad as fw
    f, pos = rope.rotary_frequencies(48, device=DEV)[0], torch.randint(0, 9999, (31,), device=DEV)
    q, tq = (torch.randn(31, 6, 64, device=DEV).to(dtype) for _ in range(2))
    k, tk = (torch.randn(31, 2, 64, device=DEV).to(dtype) for _ in range(2))
    kw = dict(interleaved=False, scale=1.5)
    args = (pos, f, (24,), False, 1.5, False)
    with fw.dual_level():
        out = fw.unpack_dual(rope.rotary(fw.make_dual(q, tq), pos, f, **kw))
        assert torch.equal(out.primal, rope.rotary(q, pos, f, **kw))
        _check(out.tangent, tq, *args)
        a, b = (fw.unpack_dual(x) for x in rope.rotary(fw.make_dual(q, tq), pos, f, k=fw.make_dual(k, tk), **kw))
        _check(a.tangent, tq, *args)
        _check(b.tangent, tk, *args)
        a, b = (fw.unpack_dual(x) for x in rope.rotary(q, pos, f, k=fw.make_dual(k, tk), **kw))
        assert a.tangent is None or not a.tangent.any()
        _check(b.tangent, tk, *args)
        a, b = (fw.unpack_dual(x) for x in rope.rotary(fw.make_dual(q, tq), pos, f, k=k, **kw))
        assert b.tangent is None or not b.tangent.any()
        _check(a.tangent, tq, *args)
    y, t = torch.func.jvp(lambda x: rope.rotary(x, pos, f, **kw), (q,), (tq,))
    assert torch.equal(y, rope.rotary(q, pos, f, **kw))
    _check(t, tq, *args)
    # forwards over backwards: the derivative of a gradient
    if dtype == F32:
        loss = lambda x: (rope.rotary(x, pos, f, **kw) ** 3).sum() / 3
        g, h = torch.func.jvp(torch.func.grad(loss), (q,), (tq,))
        y, t = rope.rotary(q, pos, f, **kw).double(), rope.rotary(tq, pos, f, **kw).double()
        # What is rotated back is rounded before: torch's (1/3) * (3 * y^2) for y^2
        # takes four roundings of 2^-24 (y^2, times 3, 1/3, the product), its
        # (1/3) * (3 * (2 y)) * t for 2 y t four (times 3, 1/3, two products); in
        # another order or with the factors apart at most four more.  A pair's
        # rounded values are off by 8 * 2^-24 of each, which turns into 8 * 2^-24 of
        # s (|u| + |w|): two thirds of e.
        for got, x in ((g, y * y), (h, 2 * y * t)):
            want, e = _ref(x, pos, f, (24,), False, 1.5, True)
            # (columns 48 on, where e is 0, are copied with the 8 * 2^-24 of their own)
            own = torch.where(torch.arange(64, device=DEV) < 48, 1, 8) * 2.0 ** -24
            assert ((got.double() - want).abs() <= e * (1 + 8 / 12) + own * (want.abs() + 2 * e)).all()


def test_rotary_of_batches():
    """torch.func.vmap over q, over q, k and positions, and over a gradient."""
    f = rope.rotary_frequencies(64, device=DEV)[0]
    pos = torch.randint(0, 9999, (5, 31), device=DEV)
    q, k = torch.randn(5, 31, 4, 64, device=DEV).to(BF), torch.randn(31, 5, 2, 64, device=DEV).to(BF)
    got = torch.func.vmap(lambda x: rope.rotary(x, pos[0], f))(q)
    assert torch.equal(got, torch.stack([rope.rotary(x, pos[0], f) for x in q]))
    a, b = torch.func.vmap(lambda x, y, p: rope.rotary(x, p, f, k=y), in_dims=(0, 1, 0))(q, k, pos)
    want = [rope.rotary(q[i], pos[i], f, k=k[:, i]) for i in range(5)]
    assert torch.equal(a, torch.stack([w[0] for w in want])) and torch.equal(b, torch.stack([w[1] for w in want]))
    g = torch.randn(5, 31, 4, 64, device=DEV).to(BF)
    grads = torch.func.vmap(lambda x, p, y: torch.func.vjp(lambda z: rope.rotary(z, p, f), x)[1](y)[0])(q, pos, g)
    assert torch.equal(grads, torch.stack([rope.rotary(g[i], pos[i], f, inverse=True) for i in range(5)]))
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.vmap(lambda x, y: rope.rotary(x, pos[0], y))(q, f.expand(5, 32))


def test_rotary_refuses_frequencies_that_want_gradients():
    f, pos = rope.rotary_frequencies(64, device=DEV)[0].requires_grad_(), torch.zeros(3, dtype=torch.int64, device=DEV)
    q = torch.randn(3, 2, 64, device=DEV)
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises((RuntimeError, ValueError)):
            rope.rotary(x, pos, f)
    with torch.no_grad():
        assert torch.equal(rope.rotary(q, pos, f), q)


@pytest.mark.parametrize("far", [1, 100, 1 << 20])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_rounds_sine_and_cosine_once(interleaved, far):
    """fp32, scale 1, u = 2^-24: c and s are off by u of themselves, one of the
    two products by u (the other goes into the sum as it is, or by u too), the sum
    by u of the result: 2 u (|a c| + |b s|) + u |y|.  The angle in 64 bits is off
    by 2^-51 of itself on either side.  Second-order terms: a factor 1 + 2^-20."""
    f, pos = rope.rotary_frequencies(128, device=DEV)[0], torch.randint(-far, far + 1, (3000,), device=DEV)
    x = torch.randn(3000, 2, 128, device=DEV)
    got = rope.rotary(x, pos, f, interleaved=interleaved).double()
    iu, iw = (slice(0, 128, 2), slice(1, 128, 2)) if interleaved else (slice(0, 64), slice(64, 128))
    a = (pos.double()[:, None] * f)[:, None]
    c, s, u, w = a.cos(), a.sin(), x[..., iu].double(), x[..., iw].double()
    off = 2.0 ** -50 * a.abs() * (u.abs() + w.abs())
    for at, y, size in ((iu, u * c - w * s, (u * c).abs() + (w * s).abs()), (iw, u * s + w * c, (u * s).abs() + (w * c).abs())):
        bound = 2.0 ** -24 * (2 * size + y.abs()) * (1 + 2.0 ** -20) + off
        assert ((got[..., at] - y).abs() <= bound).all()
