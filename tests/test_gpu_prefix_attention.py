"""Shared-prefix attention against softmax attention in 64 bits.

Bound of an output value, with u = half a step of the type: the weights may be rounded to the type before they meet
the values (u each; f16 also loses up to 2^-25 of the row's largest weight where a small one is no longer normal),
scores are off by delta = scale * sum|q||k| * (dim + 2) 2^-24, exponentials and joins of partial sums by 2^-18, and a
sum of n positive terms in fp32 by n 2^-24 on either side of the quotient; the result is rounded once more (u)."""
import copy
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import AnncError, device  # noqa: E402

BF16, F16 = torch.bfloat16, torch.float16


class Batch:
    """Inputs of one call: nq tokens and no own keys per sequence, own keys packed or in slots of a wider buffer."""

    def __init__(self, nq, no, heads, kv, dim, prefix, dtype=BF16, seed=0, slots=0, size=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: (torch.randn(s, device="cuda", generator=g) * size).to(dtype)
        self.nq, self.no = np.asarray(nq, np.int64), np.asarray(no, np.int64)
        self.heads, self.kv, self.dim, self.dtype = heads, kv, dim, dtype
        tokens = int(self.nq.sum())
        if slots:
            begin, rows = np.arange(len(self.no)) * slots, slots * len(self.no)
        else:
            begin, rows = np.cumsum(self.no) - self.no, int(self.no.sum())
        self.begin = begin
        self.q, self.kp, self.vp = r(tokens, heads, dim), r(prefix, kv, dim), r(prefix, kv, dim)
        self.ko, self.vo = r(rows, kv, dim), r(rows, kv, dim)
        up = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")
        self.own_begin, self.own_len = up(begin, torch.int64), up(self.no, torch.int32)
        self.q_begin = up(np.concatenate([[0], np.cumsum(self.nq)]), torch.int32)
        self.out = torch.full((tokens, heads, dim), 77.0, dtype=dtype, device="cuda")
        self.lse = torch.full((tokens, heads), 77.0, device="cuda")

    def run(self, plan=None, own=True, ragged=None, lse=True, scale=None):
        ragged = bool((self.nq != 1).any()) if ragged is None else ragged
        plan = plan or device.PrefixAttention(self.heads, self.kv, self.dim, self.q.shape[0], dtype=self.dtype)
        kw = dict(k_own=self.ko, v_own=self.vo, own_begin=self.own_begin, own_len=self.own_len) if own else {}
        plan.run(self.q, self.kp, self.vp, self.out, q_begin=self.q_begin if ragged else None, scale=scale,
                 lse=self.lse if lse else None, **kw)

    def check(self, own=True, lse=True, scale=None):
        f = torch.finfo(self.dtype)
        u = f.eps / 2
        group = self.heads // self.kv
        scale = self.dim ** -0.5 if scale is None else scale
        spread = lambda x: x.double().repeat_interleave(group, 1).transpose(0, 1)  # [heads, rows, dim]
        kp, vp = spread(self.kp), spread(self.vp)
        ko, vo = spread(self.ko), spread(self.vo)
        seqs = [(int(t), int(n), int(b), int(m)) for t, n, b, m in
                zip(np.cumsum(self.nq) - self.nq, self.nq, self.begin, self.no)]
        for t0, n, b, m in seqs:
            for i in range(n):
                seen = max(0, m - (n - 1 - i)) if own else 0
                k = torch.cat([kp, ko[:, b:b + seen]], 1)
                v = torch.cat([vp, vo[:, b:b + seen]], 1)
                q = self.q[t0 + i].double()
                got, got_lse = self.out[t0 + i].double(), self.lse[t0 + i].double()
                if k.shape[1] == 0:
                    assert bool((got == 0).all())
                    assert not lse or bool((got_lse == -math.inf).all())
                    continue
                s = (k * q[:, None]).sum(-1) * scale
                delta = ((k.abs() * q[:, None].abs()).sum(-1) * abs(scale)).amax(-1) * (self.dim + 2) * 2.0 ** -24
                p = torch.softmax(s, -1)
                want = (p[..., None] * v).sum(1)
                mass = (p[..., None] * v.abs()).sum(1)
                count = k.shape[1]
                tol = mass * (u + 2 * (delta[:, None] + 2.0 ** -18 + (count + 8) * 2.0 ** -24))
                if self.dtype == F16:
                    tol = tol + count * 2.0 ** -25 * v.abs().amax(1)
                tol = tol + u * (want.abs() + tol) + f.tiny * f.eps
                bad = (got - want).abs() > tol
                assert not bool(bad.any()), (t0 + i, float(((got - want).abs() / tol).max()))
                if lse:
                    want = torch.logsumexp(s, -1)
                    room = delta + 2.0 ** -18 + (count + 8) * 2.0 ** -24 + 2.0 ** -22 * want.abs()
                    assert bool(((got_lse - want).abs() <= room).all()), float(((got_lse - want).abs() / room).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [1, 2, 63, 127, 128, 129, 255, 257, 320, 321, 383, 384, 385, 511, 513, 640, 1000])
def test_single_tokens(prefix, dim, dtype):
    b = Batch([1] * 5, [0, 1, 3, 17, 40], 8, 2, dim, prefix, dtype, seed=prefix)
    b.run()
    b.check()


@pytest.mark.parametrize("dim", [1, 7, 8, 16, 24, 32, 40, 72, 80, 96, 100, 120, 136, 192, 256])
@pytest.mark.parametrize("prefix", [300, 700])
def test_head_sizes(dim, prefix):
    b = Batch([1, 2, 3], [0, 2, 30], 4, 2, dim, prefix, seed=dim)
    b.run()
    b.check()


@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (3, 1), (5, 1), (6, 2), (7, 1), (12, 4), (32, 1), (64, 1), (40, 8), (96, 1),
                                      (128, 1), (130, 1), (300, 2)])
@pytest.mark.parametrize("dim,prefix", [(64, 200), (64, 500), (128, 500)])
def test_head_groups(heads, kv, dim, prefix):
    b = Batch([1] * 9, [4, 0, 9, 1, 2, 3, 5, 8, 13], heads, kv, dim, prefix, seed=heads)
    b.run()
    b.check()


@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 63, 64, 65, 130, 257])
@pytest.mark.parametrize("prefix", [90, 700])
def test_batch_sizes(tokens, prefix):
    b = Batch([1] * tokens, [(i * 7) % 12 for i in range(tokens)], 4, 1, 64, prefix, seed=tokens)
    b.run()
    b.check()


@pytest.mark.parametrize("heads,kv,dim,prefix", [(1, 1, 64, 200), (4, 2, 128, 300), (12, 4, 64, 70), (10, 2, 40, 129), (16, 2, 128, 40),
                                                 (40, 1, 64, 500), (2, 1, 64, 64), (3, 1, 128, 17)])
def test_many_tokens(heads, kv, dim, prefix):
    # enough tokens that a warp of the joining kernel takes the heads of several (groups below eight)
    tokens = 1400 // kv + 3
    b = Batch([1] * tokens, [(i * 7) % 23 for i in range(tokens)], heads, kv, dim, prefix, seed=heads)
    b.run()
    b.check()


def some_of(b, tokens):
    """The given tokens (each a sequence) of a batch that has run, to be checked."""
    c = copy.copy(b)
    at = torch.as_tensor(tokens, device="cuda")
    c.nq, c.no, c.begin = np.ones(len(tokens), np.int64), b.no[tokens], b.begin[tokens]
    c.q, c.out, c.lse = b.q[at], b.out[at], b.lse[at]
    return c


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 1), (4, 1), (5, 1), (2, 2), (8, 4), (12, 4), (16, 2)])
@pytest.mark.parametrize("dim,prefix", [(64, 40), (64, 129), (128, 700), (40, 300)])
def test_warps_with_the_heads_of_several_tokens(heads, kv, dim, prefix):
    tokens = 9700 // kv + 5
    b = Batch([1] * tokens, [(i * 7) % 23 if i % 3 else 0 for i in range(tokens)], heads, kv, dim, prefix, seed=heads + dim)
    b.run()
    some_of(b, np.unique(np.concatenate([np.arange(12), np.arange(60, 68), np.arange(0, tokens, 311), tokens - 1 - np.arange(9)]))).check()


def test_index_products_beyond_32_bits():
    # tokens * key heads * key heads is 5.2e9
    tokens, kv = 20000, 512
    b = Batch([1] * tokens, [0] * tokens, kv, kv, 8, 3, seed=5)
    b.run(own=False)
    some_of(b, np.array([0, 1, 7, 8, 9999, 16383, 16384, 19998, 19999])).check(own=False)


@pytest.mark.parametrize("nq", [[3] + [0] * 70 + [1] * 50 + [0] * 33 + [40] + [0] * 31 + [2, 0, 1],
                                [0] * 40 + [1] * 3 + [0, 0, 5] * 45 + [0] * 64, [31, 1, 32, 33, 0, 64, 7], [1] * 129 + [0] * 32 + [1] * 64,
                                [0] * 2000 + [1] * 70 + [0] * 1100 + [2] * 30])
def test_sequences_without_tokens(nq):
    # runs of empty sequences around the 32 tokens and the 32 entries that a warp looks at together
    b = Batch(nq, [(i * 13) % 29 for i in range(len(nq))], 2, 1, 64, 300, seed=len(nq))
    b.run()
    b.check()


def test_tokens_before_the_first_sequence():
    b = Batch([1] * 70 + [2] * 20, [(i * 13) % 29 for i in range(90)], 2, 1, 64, 300, seed=9)
    b.q_begin[:41] = 40  # the first 40 tokens belong to no sequence, sequences 0 to 39 have none
    b.run(ragged=True)
    assert bool((b.out[:40] == 77).all()) and bool((b.lse[:40] == 77).all())
    c = copy.copy(b)
    c.nq, c.no, c.begin, c.q, c.out, c.lse = b.nq[40:], b.no[40:], b.begin[40:], b.q[40:], b.out[40:], b.lse[40:]
    c.check()


def test_many_ragged_tokens():
    nq = [1 + (i * 5) % 9 for i in range(300)] + [0, 40, 1]
    b = Batch(nq, [(i * 11) % 30 for i in range(303)], 4, 2, 64, 260, F16, seed=2)
    b.run()
    b.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,tokens,prefix", [(8, 8, 1, 5000), (8, 2, 3, 20000), (8, 2, 40, 9000), (8, 1, 300, 2500), (4, 4, 300, 700),
                                                    (6, 2, 97, 3333), (4, 1, 5, 128), (2, 1, 700, 129), (96, 1, 4, 1500)])
def test_without_own_keys(heads, kv, tokens, prefix, dim):
    # items that one CTA has all of, and items that are cut between two, three or many
    b = Batch([1] * tokens, [0] * tokens, heads, kv, dim, prefix, seed=tokens)
    b.run(own=False)
    b.check(own=False)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefix", [0, 1, 130, 513, 1025])
def test_sequences_of_several_tokens(prefix, dtype):
    # no token, fewer own keys than tokens, as many, more; a long sequence
    nq = [1, 0, 3, 5, 2, 8, 1, 70, 0]
    no = [0, 4, 3, 2, 0, 40, 9, 75, 0]
    b = Batch(nq, no, 6, 2, 64, prefix, dtype, seed=prefix)
    b.run()
    b.check()


@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("prefix", [0, 77])
def test_rows_without_keys(prefix, own):
    b = Batch([1] * 6, [0, 3, 0, 0, 1, 0], 4, 2, 64, prefix)
    b.run(own=own)
    b.check(own=own)


def test_own_keys_long_and_in_slots():
    b = Batch([1, 1, 2, 1], [500, 0, 300, 129], 8, 2, 128, 260, slots=512)
    # what lies in a slot behind its sequence is never used
    for i, n in enumerate(b.no):
        b.ko[i * 512 + n:(i + 1) * 512] = float("nan")
        b.vo[i * 512 + n:(i + 1) * 512] = float("inf")
    b.run()
    b.check()


def test_tokens_behind_the_last_sequence_stay():
    b = Batch([2, 3, 4], [2, 3, 4], 4, 2, 64, 150)
    pad = 5
    q = torch.cat([torch.full((2, 4, 64), float("nan"), device="cuda").to(BF16), b.q,
                   torch.full((pad, 4, 64), float("nan"), device="cuda").to(BF16)])
    out = torch.full_like(q, 55.0)
    lse = torch.full((len(q), 4), 55.0, device="cuda")
    plan = device.PrefixAttention(4, 2, 64, 100)
    plan.run(q, b.kp, b.vp, out, k_own=b.ko, v_own=b.vo, own_begin=b.own_begin, own_len=b.own_len, q_begin=b.q_begin + 2, lse=lse)
    assert bool((out[:2] == 55).all()) and bool((out[-pad:] == 55).all())
    assert bool((lse[:2] == 55).all()) and bool((lse[-pad:] == 55).all())
    b.out, b.lse = out[2:-pad], lse[2:-pad]
    b.check()
    # and without own keys
    out.fill_(55.0)
    lse.fill_(55.0)
    plan.run(q, b.kp, b.vp, out, q_begin=b.q_begin + 2, lse=lse)
    assert bool((out[:2] == 55).all()) and bool((out[-pad:] == 55).all()) and bool((lse[-pad:] == 55).all())
    b.check(own=False)
    plan.run(q, b.kp, b.vp, out.fill_(55.0), q_begin=b.q_begin[:1])  # no sequence at all
    assert bool((out == 55).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size,scale", [(6.0, 1.0), (30.0, 0.125), (0.01, 0.125), (1.0, 0.0), (1.0, -0.3)])
def test_peaked_flat_and_odd_scales(size, scale, dtype):
    b = Batch([1] * 7 + [2], [5, 0, 1, 64, 3, 2, 9, 4], 8, 4, 64, 900, dtype, seed=11, size=size)
    b.run(scale=scale)
    b.check(scale=scale)


def test_rising_scores():
    # every key tops the one before it, in steps from tiny to large: running maxima move all the time
    b = Batch([1] * 4, [20, 0, 5, 9], 4, 2, 64, 1500)
    b.q.fill_(1.0)
    ramp = torch.linspace(0, 1, 1500, device="cuda") ** 3 * 6
    b.kp.copy_((ramp[:, None, None] * torch.ones_like(b.kp, dtype=torch.float32)).to(BF16))
    for sign in (1, -1):
        b.run(scale=sign * 0.5)
        b.check(scale=sign * 0.5)


@pytest.mark.parametrize("dim", [64, 128])
def test_infinities_and_nans_reach_only_their_rows(dim):
    b = Batch([1] * 200, [2] * 200, 2, 1, dim, 300, seed=3)
    b.q[5, 0] = float("nan")
    b.q[17, 1, 3] = float("inf")
    b.ko[2 * 40] = float("nan")   # own key of sequence 40
    b.vo[2 * 50 + 1] = float("inf")
    b.run()
    bad = {(5, 0), (17, 1), (40, 0), (40, 1), (50, 0), (50, 1)}
    finite = torch.isfinite(b.out.float()).all(-1)
    for t in range(200):
        for h in range(2):
            assert bool(finite[t, h]) == ((t, h) not in bad), (t, h)


@pytest.mark.parametrize("dim", [64, 128])
def test_infinities_and_nans_of_other_tokens_keys(dim):
    # tokens that share a warp, of sequences of one and of several tokens: what one may not see reaches it in no way
    nq = [1, 1, 3, 1, 4, 2] * 130
    b = Batch(nq, [3, 5, 6, 2, 4, 9] * 130, 2, 1, dim, 150, seed=4)
    hidden = {}
    starts = np.cumsum(b.nq) - b.nq
    for s in range(0, len(nq), 13):
        last = int(b.begin[s] + b.no[s] - 1)  # the own key that only the sequence's last token sees
        (b.ko if s % 2 else b.vo)[last] = float("nan") if s % 3 else float("inf")
        hidden[int(starts[s] + b.nq[s] - 1)] = True
    b.run()
    finite = torch.isfinite(b.out.float()).all(-1).all(-1).cpu().numpy()
    assert [t for t in range(len(finite)) if not finite[t]] == sorted(hidden)


def test_infinite_scores():
    # a row all of whose scores are -inf, or that has one of +inf, is one of NaN, as the formula has it; others stay
    for dim in (64, 128):
        b = Batch([1] * 130, [0] * 130, 2, 1, dim, 300, F16, seed=6)
        b.kp.fill_(0)
        b.kp[:, 0, 0] = 60000.0
        b.q.fill_(0)
        b.q[3, 0, 0] = -60000.0
        b.q[3, 1, 0] = 1.0
        b.kp[200, 0, 0] = float("inf")
        b.q[5, 0, 0] = 1.0
        b.q[6, 0, 0] = -1.0
        b.run(own=False, scale=1e35)  # scores of -3.6e44, 6e39 and +-inf
        bad = ~torch.isfinite(b.out.float()).all(-1)
        assert bool(bad[3].all()) and bool(bad[5, 0]) and bool(bad[6, 0])
        # (zero queries meet the infinite key: 0 * inf)
        assert bool(bad.all())
        b.kp[200, 0, 0] = 0
        b.run(own=False, scale=1e35)
        bad = ~torch.isfinite(b.out.float()).all(-1)
        assert sorted(map(tuple, bad.nonzero().tolist())) == [(3, 0), (3, 1), (5, 0), (6, 0)]


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    code = """
import torch
from annc_b200 import device as dev
torch.cuda.init()
x = torch.randn((40, 96), device="cuda")
q, s, w, ws = dev.i8_rows(40, 96), torch.empty(40, device="cuda"), dev.i8_rows(64, 96).fill_(1), torch.ones(64, device="cuda")
c = torch.empty((40, 64), dtype=torch.bfloat16, device="cuda")
rot, plan = dev.Rotary(32), dev.PrefixAttention(2, 1, 32, 40)
kv, out, pos = torch.randn((70, 1, 32), device="cuda").bfloat16(), torch.empty((40, 2, 32), dtype=torch.bfloat16, device="cuda"), torch.arange(40, device="cuda")
def calls():
    dev.quantize_rows(x, q, s)
    dev.gemm_i8(q, s, w, ws, c)
    rot.run(pos, c.view(40, 2, 32), c.view(40, 2, 32))
    plan.run(c.view(40, 2, 32), kv, kv, out)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
graph.replay()
got = out.clone()
calls()
assert torch.equal(got, out) and bool(torch.isfinite(out.float()).all())
print("fine")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_strided_operands():
    # one buffer [rows, 2, kv, dim] of keys and values, queries inside a projection, a padded output
    b = Batch([1, 3, 2], [1, 3, 20], 6, 2, 64, 333, seed=5)
    kv = torch.stack([b.kp, b.vp], 1)
    own = torch.stack([b.vo, b.ko], 2)  # [rows, kv, 2, dim]
    wide = torch.full((6, 10, 72), 3.0, dtype=BF16, device="cuda")
    wide[:, 2:8, :64] = b.q
    out = torch.full((6, 8, 80), 44.0, dtype=BF16, device="cuda")
    b.kp, b.vp, b.ko, b.vo, b.q, b.out = kv[:, 0], kv[:, 1], own[:, :, 1], own[:, :, 0], wide[:, 2:8, :64], out[:, 1:7, 8:72]
    b.run()
    b.check()
    out[:, 1:7, 8:72] = 44.0
    assert bool((out == 44).all())
    # heads first, and addresses off 16 bytes
    b.kp, b.vp = b.kp.transpose(0, 1).contiguous().transpose(0, 1), b.vp.transpose(0, 1).contiguous().transpose(0, 1)
    b.run()
    b.check()
    for name in ("kp", "vp", "ko", "vo", "q"):
        x = getattr(b, name)
        odd = torch.zeros(x.shape[:2] + (67,), dtype=BF16, device="cuda")[:, :, 3:]
        odd.copy_(x)
        setattr(b, name, odd)
        b.run()
        b.check()
    odd_out = torch.full((6, 6, 67), 4.0, dtype=BF16, device="cuda")
    b.out = odd_out[:, :, 1:65]
    b.run()
    b.check()


def test_bad_begins_and_lengths_stay_inside():
    b = Batch([1] * 5, [4] * 5, 4, 2, 64, 40)
    b.own_begin = torch.tensor([-3, 1 << 40, 18, 0, 19], device="cuda")
    b.own_len = torch.tensor([4, 4, 1 << 30, -5, 4], dtype=torch.int32, device="cuda")
    b.run()
    b.begin, b.no = np.array([0, 0, 18, 0, 19]), np.array([0, 0, 2, 0, 1])  # as clamped to the 20 rows
    b.check()


def test_one_plan_for_many_calls():
    plan = device.PrefixAttention(8, 2, 64, 300)
    for tokens, prefix, seed in ((300, 513, 1), (1, 4000, 2), (77, 0, 3), (300, 64, 4), (13, 20000, 5)):
        b = Batch([1] * tokens, [(i * 5) % 9 for i in range(tokens)], 8, 2, 64, prefix, seed=seed)
        b.run(plan)
        b.check()


@pytest.mark.parametrize("tokens,prefix", [(3, 5000), (600, 700)])
def test_another_stream_and_a_captured_graph(tokens, prefix):
    b = Batch([1] * tokens, [(i * 5) % 9 for i in range(tokens)], 8, 2, 128, prefix, seed=1)
    plan = device.PrefixAttention(8, 2, 128, tokens)
    b.run(plan)
    want, want_lse = b.out.clone(), b.lse.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.out.zero_()
        b.run(plan)
    s.synchronize()
    assert torch.equal(b.out, want) and torch.equal(b.lse, want_lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(plan)
    b.out.zero_()
    for _ in range(3):
        graph.replay()
    assert torch.equal(b.out, want) and torch.equal(b.lse, want_lse)
    b.q.copy_(b.q.flip(0))
    graph.replay()
    b.check()


def test_cache_beyond_32_bits():
    # rows whose offsets in the own cache pass 2^31 elements, and a prefix that lies there
    rows = (1 << 31) // 128 + 1000
    cache = torch.empty((rows, 1, 128), dtype=BF16, device="cuda")
    b = Batch([1, 2], [30, 12], 4, 1, 128, 600, seed=9)
    first = rows - 700
    cache[first:first + 600], cache[rows - 50:rows - 20], cache[rows - 20:rows - 8] = b.kp, b.ko[:30], b.ko[30:]
    b.kp = cache[first:first + 600]
    ko, b.ko = b.ko, cache
    vo, b.vo = b.vo, torch.empty_like(cache)
    b.vo[rows - 50:rows - 8] = vo
    b.own_begin += rows - 50
    b.run()
    b.ko, b.vo = ko, vo
    b.check()


def test_refusals():
    b = Batch([1] * 4, [2] * 4, 4, 2, 64, 40)
    plan = device.PrefixAttention(4, 2, 64, 4)
    own = dict(k_own=b.ko, v_own=b.vo, own_begin=b.own_begin, own_len=b.own_len)
    good = dict(q=b.q, k_prefix=b.kp, v_prefix=b.vp, out=b.out, **own)
    plan.run(**good)
    for bad in (dict(q=b.q[:, :2]), dict(q=b.q.half()), dict(k_prefix=b.kp[:30]), dict(v_prefix=b.vp[..., :32]), dict(k_own=None),
                dict(own_len=None), dict(own_len=b.own_len.long()), dict(own_begin=b.own_begin.int()), dict(own_len=b.own_len[:3]),
                dict(q_begin=b.q_begin), dict(q_begin=b.q_begin[:0]), dict(lse=b.lse.t()), dict(lse=b.lse[:, :2]),
                dict(out=b.out.float()), dict(q=b.q.cpu()), dict(v_own=b.vo[:5]), dict(scale=float("nan")),
                dict(q=torch.cat([b.q, b.q]), out=torch.cat([b.out, b.out]))):
        if "q_begin" in bad and len(bad["q_begin"]) == 5:
            bad["q_begin"] = bad["q_begin"][:4]  # three sequences, four lengths
        with pytest.raises(AnncError):
            plan.run(**{**good, **bad})
    for args in ((4, 3, 64, 4), (0, 0, 64, 4), (4, 2, 300, 4)):
        with pytest.raises(AnncError):
            p = device.PrefixAttention(*args)
            p.run(torch.empty((1, args[0], args[2]), dtype=BF16, device="cuda"),
                  torch.empty((5, args[1], args[2]), dtype=BF16, device="cuda"),
                  torch.empty((5, args[1], args[2]), dtype=BF16, device="cuda"),
                  torch.empty((1, args[0], args[2]), dtype=BF16, device="cuda"))
    with pytest.raises(AnncError):
        device.PrefixAttention(4, 2, 64, 4, dtype=torch.float32)
