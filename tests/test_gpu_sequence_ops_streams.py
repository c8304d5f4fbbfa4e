"""Sequence operators on two streams at once, each with its own plan: every call gives what it gives alone."""
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import device  # noqa: E402
from tests.test_gpu_gemm_i8 import operands  # noqa: E402
from tests.test_gpu_prefix_attention import BF16, F16, Batch  # noqa: E402


def product(m, n, k, seed):
    a, sa, b, sb, bias = operands(m, n, k, seed)
    c = torch.zeros((m, n), dtype=BF16, device="cuda")
    return (lambda: device.gemm_i8(a, sa, b, sb, c, bias=bias)), c


def attention(tokens, heads, kv, dim, prefix, dtype, seed):
    b = Batch([1] * tokens, [(i * 5) % 9 for i in range(tokens)], heads, kv, dim, prefix, dtype, seed=seed)
    plan = device.PrefixAttention(heads, kv, dim, tokens, dtype=dtype)
    return (lambda: b.run(plan)), b.out


def turns(tokens, seed):
    plan, pos = device.Rotary(128, scaling="yarn", factor=4.0), torch.arange(tokens, device="cuda")
    x = torch.randn((tokens, 8, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    out = torch.empty_like(x)
    return (lambda: plan.run(pos, x, out)), out


@pytest.mark.parametrize("captured", [False, True])
def test_two_streams(captured):
    sides = []
    for seed in (1, 2):
        sides.append([product(1, 1024, 4096, seed), attention(40, 8, 2, 64, 5000, BF16, seed), product(4096, 520, 1100, seed),
                      attention(700, 6, 2, 128, 700, F16, seed), turns(3000, seed), product(200, 1000, 2048, seed),
                      attention(300, 4, 4, 96, 40, BF16, seed)][::1 if seed == 1 else -1])
    want = []
    for side in sides:
        for run, out in side:
            run()
        torch.cuda.synchronize()
        want.append([out.clone() for _, out in side])
        for _, out in side:
            out.zero_()
    streams = [torch.cuda.Stream() for _ in sides]
    torch.cuda.synchronize()
    graphs = []
    if captured:
        for side, stream in zip(sides, streams):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                for run, _ in side:
                    run()
    for _ in range(20):
        for i, (side, stream) in enumerate(zip(sides, streams)):
            with torch.cuda.stream(stream):
                if captured:
                    graphs[i].replay()
                else:
                    for run, _ in side:
                        run()
    torch.cuda.synchronize()
    for side, outs in zip(sides, want):
        assert all(torch.equal(out, w) for (_, out), w in zip(side, outs))
