"""8-bit integer layers against their definition in 64 bits.

Quantisation is exact: the step is the fp32 number next to max|x| / 127, a value goes to the whole number nearest to
x / step, halves to even.  Products: the integer sum is exact; it is rounded to fp32, scaled twice, the bias added
(one rounding each, 2^-24), then rounded to C's type (half a step of it)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import AnncError, device  # noqa: E402
from annc_b200._lib import ACT_NONE, ACT_RELU, ACT_SIGMOID  # noqa: E402

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------- quantisation

def quantize_ref(x):
    """scale f32 and q of the rows of x (fp64 throughout; the quotient of two fp32 numbers is never nearer to a half
    than 2^-32 of it unless it is one, so that rounding it to 53 bits decides nothing)."""
    x = x.double()
    top = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    bad = ~torch.isfinite(x).all(1)
    scale = torch.maximum(top / 127, torch.full_like(top, 2.0 ** -126)).float()
    scale[bad] = float("nan")
    q = torch.round(x / scale.double()[:, None])
    q[bad] = 0
    return scale, q.to(torch.int8)


def check_quantize(x, q=None):
    q = device.i8_rows(*x.shape) if q is None else q
    scale = torch.full((x.shape[0],), -1.0, device="cuda")
    device.quantize_rows(x, q, scale)
    want_scale, want_q = quantize_ref(x)
    assert torch.equal(scale.nan_to_num(-7.0), want_scale.nan_to_num(-7.0))
    assert torch.equal(q, want_q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8192), (3, 16), (16, 1000), (2, 8191), (5, 40000), (1024, 64), (1500, 1001),
                                       (1027, 2048), (1024, 2056), (1100, 17), (2, 0)])
def test_quantize(dtype, rows, cols):
    x = torch.randn((rows, cols), device="cuda", generator=gen(rows + cols))
    check_quantize((x * torch.rand((rows, 1), device="cuda", generator=gen(5)) * 3).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_and_odd_addresses(dtype):
    big = torch.randn((70, 300), device="cuda", generator=gen(1)).to(dtype)
    check_quantize(big[:, 1:258])
    check_quantize(big[::2, 16:272])
    check_quantize(big[:, 8:264], torch.empty((70, 257), dtype=torch.int8, device="cuda")[:, 1:])
    q = torch.full((70, 304), 99, dtype=torch.int8, device="cuda")
    check_quantize(big, q[:, :300])
    assert bool((q[:, 300:] == 99).all())  # what lies behind a row stays


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [1100, 1102, 1101])
def test_quantize_by_quads(dtype, pitch):
    # every alignment of a row and every rest of four, in registers and read again, one row and many
    big = torch.randn((40, pitch), device="cuda", generator=gen(pitch)).to(dtype)
    for rows in (1, 40):
        for cols in (1, 2, 3, 4, 5, 30, 255, 256, 257, 258, 1090):
            for first in range(5):
                q = torch.full((rows, 1104), 99, dtype=torch.int8, device="cuda")
                check_quantize(big[:rows, first:first + cols], q[:, :cols])
                assert bool((q[:, cols:] == 99).all())
    wide = torch.randn((2, 33001), device="cuda", generator=gen(1)).to(dtype)
    for first, cols in ((0, 33001), (1, 32999), (2, 32994)):
        check_quantize(wide[:, first:first + cols])


def test_quantize_at_the_borders_of_steps():
    # quotients next to a half: k + 1/2 steps and the fp32 neighbours of that, for steps that are not powers of two
    rows = []
    for top in (127.0, 1.0, 0.3, 3.3e-5, 1e30, 5e-38):
        scale = np.float32(top) / np.float32(127)
        h = ((np.arange(0, 127) + 0.5) * np.float64(scale)).astype(np.float32)
        row = np.concatenate([h, np.nextafter(h, np.float32(0)), np.nextafter(h, np.float32(np.inf)), -h, [np.float32(top)]])
        rows.append(row[np.abs(row) <= np.float32(top)][-500:])
    n = min(len(r) for r in rows)
    x = np.stack([np.concatenate([r[:n - 1], r[-1:]]) for r in rows]).astype(np.float32)
    check_quantize(torch.from_numpy(x).cuda())


def test_quantize_extremes():
    x = torch.zeros((8, 64), device="cuda")
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3, 63] = -float("inf")
    x[4] = 1e-45  # below every step: the step stays a normal number
    x[5, 0] = 3.4e38
    x[5, 1] = -3.4e38
    x[6] = -0.0
    x[7] = 2.0 ** -126
    check_quantize(x)


@pytest.mark.parametrize("k,n", [(1, 1), (64, 32), (1000, 33), (129, 1003), (2048, 512)])
def test_weight(k, n):
    w = torch.randn((k, n + 3), device="cuda", generator=gen(k + n))[:, :n]
    q, scale = device.i8_weight(w)
    want_scale, want_q = quantize_ref(w.t())
    assert torch.equal(scale, want_scale) and torch.equal(q, want_q) and q.stride(0) % 16 == 0


# ---------------------------------------------------------------- product

def operands(m, n, k, seed, extreme=False):
    g = gen(seed)

    def ints(r):
        v = (torch.randn((r, k), device="cuda", generator=g) * 40).round_().clamp_(-128, 127)
        if extreme:
            v = torch.full((r, k), -128.0, device="cuda")
        out = device.i8_rows(r, k)
        out.copy_(v)
        return out
    return (ints(m), torch.rand(m, device="cuda", generator=g) * 0.05 + 1e-3, ints(n),
            torch.rand(n, device="cuda", generator=g) * 1e-2 + 1e-4, torch.randn(n, device="cuda", generator=g))


def check_product(a, sa, b, sb, bias, act, dtype, c=None):
    m, n = a.shape[0], b.shape[0]
    if c is None:
        c = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    device.gemm_i8(a, sa, b, sb, c, bias=bias, activation=act)
    prod = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    y = prod + (bias.double() if bias is not None else 0)
    tol = 2.0 ** -24 * (3.01 * prod.abs() + y.abs()) + 1e-38
    if act == ACT_RELU:
        y = y.clamp_min(0)
    elif act == ACT_SIGMOID:  # slope at most 1/4; exp within 2 ulp, a sum and a quotient
        y = torch.sigmoid(y)
        tol = tol / 4 + 2.0 ** -21 * y
    f = torch.finfo(dtype)
    if dtype != torch.float32:
        tol = tol + f.eps / 2 * (y.abs() + tol) + f.tiny * f.eps
    assert bool(((c.double() - y).abs() <= tol).all()), float(((c.double() - y).abs() - tol).max())


SHAPES = [(1, 1, 1), (1, 1024, 8192), (1, 17, 100), (2, 64, 16), (7, 129, 1024), (16, 1024, 1024), (17, 100, 257),
          (33, 4096, 512), (64, 512, 2048), (65, 8, 4096), (128, 128, 128), (130, 260, 384), (200, 4096, 2048), (256, 256, 1),
          (300, 1003, 1001), (511, 1, 1024), (1999, 640, 130), (2048, 1024, 1024), (4100, 520, 96), (8192, 16, 64)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k):
    a, sa, b, sb, bias = operands(m, n, k, m + n + k)
    for i, dtype in enumerate(TYPES):
        act = (ACT_NONE, ACT_RELU, ACT_SIGMOID)[(i + m) % 3]
        check_product(a, sa, b, sb, bias if (m + i) % 2 else None, act, dtype)


@pytest.mark.parametrize("act", [ACT_NONE, ACT_RELU, ACT_SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(5, 70, 96), (150, 200, 300), (1300, 1030, 256)])
def test_epilogues(m, n, k, act, dtype):
    a, sa, b, sb, bias = operands(m, n, k, 3)
    check_product(a, sa, b, sb, bias, act, dtype)
    check_product(a, sa, b, sb, None, act, dtype)


@pytest.mark.parametrize("act", [ACT_NONE, ACT_RELU, ACT_SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(16384, 264, 640), (6000, 1001, 2048), (9001, 520, 1100), (4099, 1192, 1024), (16200, 640, 32)])
def test_tall_products(m, n, k, act, dtype):
    # tiles of CTA pairs one after the other; tails of both sides; rows of C that TMA stores, and rows that it does not
    a, sa, b, sb, bias = operands(m, n, k, 7)
    assert device.gemm_i8_kernel_name(a, sa, b, sb, torch.empty((m, n), dtype=dtype, device="cuda")) == "tcgen05_pair_i8"
    wide = torch.full((m + 2, n), 5.0, dtype=dtype, device="cuda")
    check_product(a, sa, b, sb, bias if n % 16 else None, act, dtype, wide[:m])
    assert bool((wide[m:] == 5.0).all())


@pytest.mark.parametrize("n", [24, 264])
def test_sigmoid_far_out(n):
    # values from -110 to 110: zero only where the smallest normal number is not reached, one at the other end
    m, k = 3000, 16
    a, b = device.i8_rows(m, k), device.i8_rows(n, k)
    a.zero_()
    b.zero_()
    bias = torch.linspace(-110, 110, n, device="cuda")
    c = torch.empty((m, n), device="cuda")
    device.gemm_i8(a, torch.ones(m, device="cuda"), b, torch.ones(n, device="cuda"), c, bias=bias, activation=ACT_SIGMOID)
    want = torch.sigmoid(bias.double())
    # the exponent's product rounds once (|x| 2^-24 of the power), its factor log2(e) is off by 0.23 2^-24; exp2, the sum and
    # the reciprocal within 2 ulp each
    tol = want * (bias.double().abs() * 1.25 * 2.0 ** -24 + 6 * 2.0 ** -23) + torch.finfo(torch.float32).tiny
    assert bool(((c.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("m,n,k", [(1, 40, 131071), (200, 300, 70000)])
def test_long_sums_are_exact(m, n, k):
    # all operands -128: the largest sum there is, 2^31 - 16384 at k = 131071
    a, sa, b, sb, _ = operands(m, n, k, 1, extreme=True)
    check_product(a, sa, b, sb, None, ACT_NONE, torch.float32)


def test_no_terms():
    a, sa, b, sb, bias = operands(3, 20, 0, 1)
    check_product(a, sa, b, sb, bias, ACT_RELU, torch.float32)


@pytest.mark.parametrize("m,n,k", [(5, 70, 96), (150, 200, 300), (1300, 600, 256)])
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_odd_addresses(m, n, k, dtype):
    a, sa, b, sb, bias = operands(m, n, k, 4)
    wide_a = torch.zeros((m, k + 37), dtype=torch.int8, device="cuda")
    wide_b = torch.zeros((n, k + 5), dtype=torch.int8, device="cuda")
    wide_a[:, 5:5 + k] = a
    wide_b[:, 1:1 + k] = b
    va, vb = wide_a[:, 5:5 + k], wide_b[:, 1:1 + k]
    for pa, pb in ((va, b), (a, vb), (va, vb)):
        for off, pitch in ((0, n), (3, n + 7), (0, (n + 15) // 16 * 16 + 16)):
            wide = torch.full((m + 1, pitch + off), 5.0, dtype=dtype, device="cuda")
            c = wide[:m, off:off + n]
            check_product(pa, sa, pb, sb, bias, ACT_NONE, dtype, c)
            c.fill_(5.0)
            assert bool((wide == 5.0).all())  # nothing beside C is written
    for off, pitch in ((3, n + 7), (0, (n + 15) // 16 * 16 + 16)):
        wide = torch.full((m + 1, pitch + off), 5.0, dtype=dtype, device="cuda")
        c = wide[:m, off:off + n]
        check_product(a, sa, b, sb, bias, ACT_NONE, dtype, c)
        c.fill_(5.0)
        assert bool((wide == 5.0).all())


def test_nan_scale_shows():
    a, sa, b, sb, bias = operands(40, 64, 64, 6)
    sa[7] = float("nan")
    c = torch.empty((40, 64), device="cuda")
    for act in (ACT_NONE, ACT_RELU, ACT_SIGMOID):
        device.gemm_i8(a, sa, b, sb, c, bias=bias, activation=act)
        assert bool(torch.isnan(c[7]).all()) and not bool(torch.isnan(c[:7]).any()) and not bool(torch.isnan(c[8:]).any())


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (40, 512, 1024), (1024, 2048, 512)])
def test_another_stream_and_a_captured_graph(m, n, k):
    a, sa, b, sb, bias = operands(m, n, k, 8)
    x = torch.randn((m, k), device="cuda", generator=gen(3))
    c, q, s = torch.empty((m, n), device="cuda"), device.i8_rows(m, k), torch.empty(m, device="cuda")
    want = torch.empty_like(c)
    device.quantize_rows(x, q, s)
    device.gemm_i8(q, s, b, sb, want, bias=bias)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        device.quantize_rows(x, q, s)
        device.gemm_i8(q, s, b, sb, c, bias=bias)
    stream.synchronize()
    assert torch.equal(c, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        device.quantize_rows(x, q, s)
        device.gemm_i8(q, s, b, sb, c, bias=bias)
    x.copy_(torch.randn((m, k), device="cuda", generator=gen(4)))
    for _ in range(3):
        c.zero_()
        graph.replay()
    device.quantize_rows(x, q, s)
    device.gemm_i8(q, s, b, sb, want, bias=bias)
    assert torch.equal(c, want)


def test_refusals():
    a, sa, b, sb, bias = operands(4, 32, 64, 9)
    c = torch.empty((4, 32), device="cuda")
    for bad in (dict(a=a[:, :32].t()), dict(a=a.float()), dict(scale_a=sa[:3]), dict(b=b.t()), dict(c=c.double()), dict(c=c.t()),
                dict(a=a.cpu()), dict(scale_b=sb[None]), dict(bias=bias[1:]), dict(activation=9)):
        kw = dict(a=a, scale_a=sa, b=b, scale_b=sb, c=c, bias=bias, activation=0)
        kw.update(bad)
        with pytest.raises(AnncError):
            device.gemm_i8(kw["a"], kw["scale_a"], kw["b"], kw["scale_b"], kw["c"], bias=kw["bias"], activation=kw["activation"])
    x = torch.empty((4, 8), device="cuda")
    for args in ((x.double(), a[:, :8], sa), (x, a, sa), (x, a[:, :8], sa[:2]), (x.cpu(), a[:, :8], sa), (x, x, sa),
                 (x.t(), a[:, :4], sa)):
        with pytest.raises(AnncError):
            device.quantize_rows(*args)
