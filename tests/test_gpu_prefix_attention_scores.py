"""Shared-prefix attention where scores are infinite or far out: keys masked through an extra value of the head.

The queries hold 1 in the head's last place, the keys 0 there, or the mask.  A masked key has weight zero and adds
nothing to any sum, so that a row is held to the same row without its masked keys, under the bound of that row."""
import copy
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import device  # noqa: E402
from tests.test_gpu_prefix_attention import BF16, F16, Batch, some_of  # noqa: E402

INF = float("inf")


def maskable(*args, **kw):
    """A batch whose keys have a place for a mask."""
    b = Batch(*args, **kw)
    b.q[..., -1], b.kp[..., -1], b.ko[..., -1] = 1, 0, 0
    return b


def check_without(b, keep, tokens=None, own=True):
    """b has run; the prefix keys that are not in `keep` were masked."""
    c = some_of(b, tokens) if tokens is not None else copy.copy(b)
    c.kp, c.vp = b.kp[keep], b.vp[keep]
    c.check(own=own)


def run_of(first, count, prefix):
    keep = torch.ones(prefix, dtype=torch.bool, device="cuda")
    keep[first:first + count] = False
    return keep


# ---------------------------------------------------------------- scores of -inf

# (tokens, heads, key heads, prefix): items that one CTA has all of and items that are cut, one row tile (two chains that
# take the key tiles in turn) and two; each without own keys and with them
@pytest.mark.parametrize("tokens,heads,kv,prefix", [(3, 4, 2, 20000), (700, 4, 4, 1700), (600, 8, 1, 1300), (5, 2, 1, 1500)])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("own", [True, False])
def test_runs_of_hidden_keys(tokens, heads, kv, prefix, dim, dtype, own):
    some = np.unique(np.linspace(0, tokens - 1, 7).astype(int))
    for count in (128, 129, 1000):
        for first in (0, 128, 129, prefix // 2 // 128 * 128, prefix // 2 + 5, prefix - count):
            b = maskable([1] * tokens, [(i * 5) % 7 for i in range(tokens)], heads, kv, dim, prefix, dtype, seed=count + first)
            keep = run_of(first, count, prefix)
            b.kp[~keep, :, -1] = -INF
            b.run(own=own)
            check_without(b, keep, some, own)


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("tokens,kv,prefix", [(5, 2, 20000), (600, 1, 1300), (5, 2, 700), (4, 2, 40)])
def test_all_of_a_prefix_hidden(tokens, kv, prefix, dim, dtype):
    # the own keys alone are left; where there are none either, every score is -inf: NaN, and lse -inf
    no = np.array([(i * 5) % 7 for i in range(tokens)])
    b = maskable([1] * tokens, no, 4, kv, dim, prefix, dtype, seed=prefix)
    b.kp[..., -1] = -INF
    b.run()
    some = np.unique(np.linspace(0, tokens - 1, 30).astype(int))
    check_without(b, torch.zeros(prefix, dtype=torch.bool, device="cuda"), some[no[some] > 0])
    lost = torch.from_numpy(np.flatnonzero(no == 0)).cuda()
    assert bool(torch.isnan(b.out[lost]).all()) and bool((b.lse[lost] == -INF).all())
    b.run(own=False)
    assert bool(torch.isnan(b.out).all()) and bool((b.lse == -INF).all())


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (40, F16)])
@pytest.mark.parametrize("tokens", [2, 40, 1500])
def test_hidden_keys_of_a_short_prefix_and_of_sequences(tokens, dim, dtype):
    # the first keys of a short prefix, and the first own keys of every sequence, in steps around 16
    for hidden in (1, 15, 16, 17, 32, 47):
        no = np.array([(i * 11) % 50 for i in range(tokens)])
        for prefix, hidden_prefix in ((0, 0), (50, hidden), (50, 50), (700, 300)):
            b = maskable([1] * tokens, no, 4, 2, dim, prefix, dtype, seed=hidden)
            b.kp[:hidden_prefix, :, -1] = -INF
            for t in range(tokens):
                b.ko[int(b.begin[t]):int(b.begin[t]) + min(hidden, int(no[t])), :, -1] = -INF
            b.run()
            c = copy.copy(b)
            c.kp, c.vp = b.kp[hidden_prefix:], b.vp[hidden_prefix:]
            c.begin, c.no = b.begin + np.minimum(no, hidden), no - np.minimum(no, hidden)
            some = np.unique(np.linspace(0, tokens - 1, 60).astype(int))
            left = (prefix - hidden_prefix + c.no[some]) > 0
            some_of(c, some[left]).check()
            lost = [int(t) for t in some[~left] if prefix + no[t] > 0]  # keys, none of them with a finite score
            assert not lost or bool(torch.isnan(b.out[lost]).all()) and bool((b.lse[lost] == -INF).all())
            none = [int(t) for t in some[~left] if prefix + no[t] == 0]
            assert not none or bool((b.out[none] == 0).all()) and bool((b.lse[none] == -INF).all())


@pytest.mark.parametrize("dim,scale", [(136, 0.09), (60, 0.1), (64, -0.3)])
def test_hidden_keys_row_by_row(dim, scale):
    for first, count in ((0, 3), (0, 4), (0, 9), (40, 30), (96, 4)):
        b = maskable([1, 1, 3], [0, 9, 4], 4, 2, dim, 100, seed=count)
        keep = run_of(first, count, 100)
        b.kp[~keep, :, -1] = -math.copysign(INF, scale)
        b.run(scale=scale)
        c = copy.copy(b)
        c.kp, c.vp = b.kp[keep], b.vp[keep]
        c.check(scale=scale)
    b.kp[..., -1] = -math.copysign(INF, scale)
    b.run(own=False, scale=scale)
    assert bool(torch.isnan(b.out).all()) and bool((b.lse == -INF).all())


def test_a_hidden_key_with_an_infinite_value_shows():
    # weight zero times infinity is NaN, as the formula has it, in the row's other key heads nothing
    for prefix, hidden in ((700, 130), (40, 16)):
        b = maskable([1] * 3, [0] * 3, 4, 2, 64, prefix, seed=8)
        b.kp[:hidden, :, -1] = -INF
        b.vp[3, 0, 5] = INF
        b.run(own=False)
        bad = torch.isnan(b.out)
        assert bool(bad[:, :2, 5].all()) and int(bad.sum()) == 6


# ---------------------------------------------------------------- scores far out

@pytest.mark.parametrize("tokens,heads,kv,prefix", [(3, 4, 2, 20000), (700, 4, 4, 1700), (600, 8, 1, 1300), (5, 2, 1, 1500), (5, 2, 1, 60)])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("own", [True, False])
def test_runs_of_keys_with_the_lowest_value(tokens, heads, kv, prefix, dim, dtype, own):
    low = torch.finfo(dtype).min
    some = np.unique(np.linspace(0, tokens - 1, 7).astype(int))
    for count in (128, 129, 1000) if prefix > 1000 else (16, 17, 50):
        for first in (0, 128, prefix // 2 + 5, prefix - count) if prefix > 1000 else (0, 7, prefix - count):
            b = maskable([1] * tokens, [(i * 5) % 7 for i in range(tokens)], heads, kv, dim, prefix, dtype, seed=count + first)
            keep = run_of(first, count, prefix)
            b.kp[~keep, :, -1] = low
            b.run(own=own)
            check_without(b, keep, some, own)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 136])
@pytest.mark.parametrize("size", [1.0, -1.0, 0.37, -0.37])
@pytest.mark.parametrize("prefix,tokens", [(40, 5), (130, 5), (1300, 5), (1300, 500), (20000, 3)])
def test_equal_scores_of_any_size(prefix, tokens, size, dim, dtype):
    # the same score for every key, as far out as the type goes: the mean of the values
    heads, kv = 4, 2
    b = Batch([1] * tokens, [0] * tokens, heads, kv, dim, prefix, dtype, seed=3)
    f = torch.finfo(dtype)
    for power in (0, 10, 15, 30, 60, 100, 127):
        if 2.0 ** power > f.max:
            continue
        b.q.zero_()
        b.q[..., 0] = 1.0 if dtype == BF16 else f.max
        b.kp[..., 0] = size * 2.0 ** power
        b.run(own=False)
        v = b.vp.double().repeat_interleave(heads // kv, 1)
        want, mass = v.mean(0), v.abs().mean(0)
        # one weight for all keys of a part, 1 times a power of two where scores are large; the sums of a CTA's part,
        # their join, the quotient, and half a step of the type.  Small scores have the operands' rounding of the weights too, which
        # is the same for all keys and for their sum is not.
        u = f.eps / 2
        tol = mass * (u + 2.0 ** -17 + 2 * (prefix + 8) * 2.0 ** -24) + u * want.abs()
        assert bool(((b.out.double() - want).abs() <= tol).all()), power


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [1300, 20000])
def test_large_scores_are_compared_as_they_round(dim, prefix):
    # one key above all others by a step of the type, far out: it alone has weight
    b = Batch([1] * 5, [0] * 5, 4, 2, dim, prefix, BF16, seed=4)
    b.q.zero_()
    b.q[..., 0] = 1.0
    for size in (2.0 ** 28, 2.0 ** 60, -(2.0 ** 28)):
        for at in (0, 127, 128, 700, prefix - 1):
            b.kp[..., 0] = size
            b.kp[at, :, 0] = size * (1 + 2.0 ** -7) if size > 0 else size * (1 - 2.0 ** -8)
            b.run(own=False)
            want = b.vp[at].double().repeat_interleave(2, 0)
            assert bool(((b.out.double() - want).abs() <= 2.0 ** -8 * want.abs()).all()), (size, at)


@pytest.mark.parametrize("dtype,scale", [(BF16, 1.0), (BF16, 0.1), (F16, 1.0), (F16, 30000.0)])
@pytest.mark.parametrize("dim", [64, 128, 136])
@pytest.mark.parametrize("prefix,tokens", [(0, 3), (40, 3), (300, 3), (20000, 3), (300, 900)])
def test_every_key_with_the_lowest_value(prefix, tokens, dim, dtype, scale):
    # a row that is masked throughout by the type's lowest number is the mean of its values
    heads, kv, own = 4, 2, 21
    b = Batch([1] * tokens, [own] * tokens, heads, kv, dim, prefix, dtype, seed=5)
    f = torch.finfo(dtype)
    b.q.zero_()
    b.q[..., 0] = 1.0 if dtype == BF16 else f.max
    b.kp[..., 0] = f.min
    b.ko[..., 0] = f.min
    b.run(scale=scale)
    count, u = prefix + own, f.eps / 2
    vo = b.vo.double().view(tokens, own, kv, dim)
    both = lambda p, o: ((p.double().sum(0) + o.sum(1)) / count).repeat_interleave(heads // kv, 1)
    want, mass = both(b.vp, vo), both(b.vp.abs(), vo.abs())
    tol = mass * (u + 2.0 ** -17 + 2 * (count + 8) * 2.0 ** -24) + u * want.abs()
    assert bool(((b.out.double() - want).abs() <= tol).all())
    top = float(b.q[0, 0, 0].double() * f.min * scale)
    assert bool(((b.lse.double() - top).abs() <= 2.0 ** -22 * abs(top)).all())


@pytest.mark.parametrize("scale", [0.0, 1e-45, 1e-38, 1e-30, 3e38])
def test_scales_at_the_ends_of_their_range(scale):
    b = maskable([1] * 3, [0, 4, 1], 4, 2, 64, 400, BF16, seed=6)
    b.q[..., :-1] *= 1e-3
    keep = run_of(100, 40 if scale else 0, 400)
    b.kp[~keep, :, -1] = -INF
    if scale > 1:  # scores within the range of 32 bits
        b.q *= 2.0 ** -126
    b.run(scale=scale)
    c = copy.copy(b)
    c.kp, c.vp = b.kp[keep], b.vp[keep]
    c.check(scale=scale)


# ---------------------------------------------------------------- many small weights of f16

@pytest.mark.parametrize("dim,kv", [(64, 148), (128, 74)])
@pytest.mark.parametrize("at", [0, 50001, (1 << 17) - 1])
def test_many_small_weights_beside_a_large_one(dim, kv, at):
    # one key of weight 1 and 2^17 - 1 of some 2^-26 each, that a CTA has all or half of: they make up 1/512 of the sum, and
    # all of the output.  A numerator in f16 is off by at most 2^-25 of its unit, which is 2^-7 of the row's largest or less.
    prefix = 1 << 17
    b = Batch([1], [0], kv, kv, dim, prefix, F16, seed=at)
    b.q.zero_()
    b.q[..., 0] = 1.0
    b.kp[..., 0] = -18.0 + 0.3 * torch.sin(torch.arange(prefix, device="cuda"))[:, None]
    b.kp[at, :, 0] = 0
    b.vp.abs_()  # (every lost weight shows)
    b.vp[at] = 0
    b.run(own=False, scale=1.0)
    u = 2.0 ** -11
    for h in (0, 1, kv // 2, kv - 1):
        p, v = torch.softmax(b.kp[:, h, 0].double(), 0), b.vp[:, h].double()
        want = p @ v
        tol = want * (u + 2.0 ** -17 + 2 * (prefix + 8) * 2.0 ** -24) + prefix * 2.0 ** -32 * v.amax() * p.max() + u * want
        got = b.out[0, h].double()
        assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [0, 60])
def test_many_small_weights_of_own_keys(dim, prefix):
    rows = 200000
    b = Batch([1], [rows], 2, 1, dim, prefix, F16, seed=2)
    b.q.zero_()
    b.q[..., 0] = 1.0
    b.ko[..., 0] = -18.0
    b.kp[..., 0] = -18.0
    b.ko[77, :, 0] = 0
    b.vo.abs_()
    b.vo[77] = 0
    b.run(scale=1.0)
    s = torch.cat([b.kp[:, 0, 0], b.ko[:, 0, 0]]).double()
    v = torch.cat([b.vp[:, 0], b.vo[:, 0]]).double()
    want = torch.softmax(s, 0) @ v
    u, count = 2.0 ** -11, len(s)
    mass = torch.softmax(s, 0) @ v.abs()
    tol = mass * (u + 2.0 ** -17 + 2 * (count + 8) * 2.0 ** -24) + count * 2.0 ** -40 * v.abs().amax() + u * want.abs()
    got = b.out.double()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


# ---------------------------------------------------------------- lists

@pytest.mark.parametrize("prefix", [30, 500])
def test_lengths_far_below_zero(prefix):
    # a sequence of several tokens with the lowest length there is: no own keys for any of them
    b = Batch([1, 4, 3], [3, 5, 4], 4, 2, 64, prefix)
    b.own_len[1] = -(1 << 31)
    b.run()
    b.no[1] = 0
    b.check()
