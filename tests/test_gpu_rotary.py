"""Rotary positions against the formula in 64 bits.

The fraction of a turn is rounded to fp32 once (an angle error of pi 2^-25), sine and cosine are within 2^-23, the
products with `size` and the two products and the sum round in fp32: together below 2^-21 (|a| + |b|) size, plus half
a step of the type at the end."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import AnncError, device  # noqa: E402

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def reference(plan, pos, x, layout, transposed=False):
    """(y, bound): turned by rotation as complex numbers, in 64 bits."""
    rot = plan.rot_dim
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    angle = pos.double()[:, None] * plan.freq * (-1 if transposed else 1)
    y = x.double().clone()
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous())
    size = torch.full_like(angle, plan.size)
    turned = z * torch.polar(size, angle)[:, None]
    tol = torch.zeros_like(y)
    # the 64-bit product of position and frequency has its own rounding: 2^-52 of the angle on either side
    far = (2.0 ** -50 * angle.abs() + 2.0 ** -21)[:, None]
    bound = (z.real.abs() + z.imag.abs()) * plan.size * far
    y[..., first], y[..., second] = turned.real, turned.imag
    tol[..., first], tol[..., second] = bound, bound
    f = torch.finfo(x.dtype)
    if x.dtype != torch.float32:
        tol[..., :rot] += f.eps / 2 * (y[..., :rot].abs() + tol[..., :rot]) + f.tiny * f.eps
    return y, tol


def check(plan, pos, x, out, layout, transposed=False):
    y, tol = reference(plan, pos, x, layout, transposed)
    assert bool(((out.double() - y).abs() <= tol).all())
    assert torch.equal(out[..., plan.rot_dim:], x[..., plan.rot_dim:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot", [(1, 1, 1, 2, 2), (1, 8, 2, 64, 64), (16, 16, 4, 128, 128), (7, 3, 1, 80, 80),
                                                     (33, 5, 0, 80, 40), (1000, 8, 8, 128, 64), (5000, 4, 1, 96, 96),
                                                     (3, 2, 1, 13, 6), (2, 1, 2, 600, 512), (2500, 1, 1, 20, 20)])
def test_turns(tokens, heads, kv, dim, rot, layout, dtype):
    plan = device.Rotary(rot, layout=layout)
    pos = torch.randint(-50, 5000, (tokens,), device="cuda", dtype=torch.int32)
    q = randn(tokens, heads, dim, seed=1, dtype=dtype)
    out = torch.empty_like(q)
    if kv == 0:
        plan.run(pos, q, out)
        check(plan, pos, q, out, layout)
        return
    k = randn(tokens, kv, dim, seed=2, dtype=dtype)
    out_k = torch.empty_like(k)
    plan.run(pos.long(), q, out, k, out_k)
    check(plan, pos, q, out, layout)
    check(plan, pos, k, out_k, layout)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_positions(layout, scaling):
    plan = device.Rotary(128, layout=layout, scaling=scaling, factor=16.0, base=500000.0)
    pos = torch.tensor([0, 1, 131071, 1 << 20, (1 << 31) - 1, 1 << 40, -(1 << 40)], device="cuda")
    x = randn(len(pos), 2, 128, seed=3)
    out = torch.empty_like(x)
    plan.run(pos, x, out)
    check(plan, pos, x, out, layout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_in_one_projection_buffer(layout, dtype):
    # queries, keys and values of a token side by side: strided views, turned in place; the values stay
    tokens, heads, kv, dim, rot = 300, 6, 2, 64, 32
    buf = randn(tokens, (heads + 2 * kv) * dim, seed=4, dtype=dtype)
    was = buf.clone()
    view = lambda b: (b[:, :heads * dim].view(tokens, heads, dim), b[:, heads * dim:(heads + kv) * dim].view(tokens, kv, dim))
    q, k = view(buf)
    plan = device.Rotary(rot, layout=layout, scaling="yarn", factor=4.0)
    pos = torch.arange(7, tokens + 7, device="cuda")
    plan.run(pos, q, q, k, k)
    for new, old in zip(view(buf), view(was)):
        check(plan, pos, old, new, layout)
    assert torch.equal(buf[:, (heads + kv) * dim:], was[:, (heads + kv) * dim:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_strides_and_odd_addresses(shift, layout, dtype):
    tokens, heads, dim, rot = 50, 3, 48, 32
    wide = randn(tokens, heads, dim + 9, seed=5, dtype=dtype)
    x = wide[:, :, shift:shift + dim]
    out = torch.full((tokens, heads, dim + 20), 9.0, dtype=dtype, device="cuda")
    o = out[:, :, 4:4 + dim]
    plan = device.Rotary(rot, layout=layout)
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32)
    plan.run(pos, x, o)
    check(plan, pos, x, o, layout)
    o.fill_(9.0)
    assert bool((out == 9.0).all())
    perm = wide.permute(1, 0, 2)[:, :, shift:shift + dim]  # tokens and heads exchanged
    res = torch.empty((tokens, heads, dim), dtype=dtype, device="cuda").permute(1, 0, 2)
    plan.run(pos[:heads], perm, res)
    check(plan, pos[:heads], perm, res, layout)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_transposed_undoes_and_takes_gradients_back(layout):
    plan = device.Rotary(64, layout=layout)
    pos = torch.randint(0, 100000, (40,), device="cuda")
    x, g = randn(40, 4, 80, seed=6), randn(40, 4, 80, seed=7)
    y, back, gx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    plan.run(pos, x, y)
    plan.run(pos, y, back, transposed=True)
    # two calls, each within 2^-21 (|a| + |b|), and |a| + |b| <= 2 times the pair's length, which a turn keeps
    length = x.double().abs().amax(-1, keepdim=True) * 2
    assert bool(((back - x).double().abs() <= 2 * 2.0 ** -21 * 2 * length).all())
    # <g, R x> = <R^T g, x>
    yarn = device.Rotary(64, layout=layout, scaling="yarn", factor=8.0)
    yarn.run(pos, x, y)
    yarn.run(pos, g, gx, transposed=True)
    check(yarn, pos, g, gx, layout, transposed=True)
    left, right = (g.double() * y.double()).sum(), (gx.double() * x.double()).sum()
    room = 2.0 ** -21 * yarn.size * 4 * (g.double().norm() * x.double().norm())
    assert abs(float(left - right)) <= float(room)


def test_no_tokens_and_other_stream():
    plan = device.Rotary(64)
    e = torch.empty((0, 4, 64), device="cuda")
    plan.run(torch.empty(0, device="cuda", dtype=torch.int64), e, e)
    x = randn(100, 4, 64, seed=8)
    pos, out, want = torch.arange(100, device="cuda"), torch.empty_like(x), torch.empty_like(x)
    plan.run(pos, x, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plan.run(pos, x, out)
    s.synchronize()
    assert torch.equal(out, want)


def test_refusals():
    plan = device.Rotary(64)
    x, k, pos = randn(4, 2, 64), randn(4, 1, 64), torch.arange(4, device="cuda")
    out, out_k = torch.empty_like(x), torch.empty_like(k)
    for args in ((pos, x, out, k), (pos[:3], x, out), (pos.float(), x, out), (pos, x[..., :32], out[..., :32]), (pos, x, out.half()),
                 (pos, x[0], out[0]), (pos, x, out, k.half(), out_k.half()), (pos, x.cpu(), out), (pos.cpu(), x, out),
                 (pos, x.transpose(1, 2), out.transpose(1, 2)), (pos, x.double(), out.double())):
        with pytest.raises(AnncError):
            plan.run(*args)
    for kw in (dict(layout="other"), dict(scaling="other"), dict(rot_dim=7), dict(scaling="linear", factor=0.0)):
        with pytest.raises(AnncError):
            device.Rotary(**{"rot_dim": 64, **kw})
