"""The sequence operators as a ranking model runs them: candidates, of one or a few tokens each, against a user's
history that is read in once.  Token rows are quantised and projected to queries, keys and values by the 8-bit
product, queries and keys get rotary positions, the candidates attend to the history and to themselves, and the
output projection and a score layer follow, all on one stream with nothing between the calls.

Every operator is held to its own bound by its own tests; here the chain is held to the same chain in 64 bits on the
same integers and weights: what the device rounds on the way (activations to 8 bits, queries, keys, values and the
attention's output to bf16) is rounded in the reference at the same places, so that only sums and functions differ.
An 8-bit value may then fall to the other side of a border: one step, 1/127 of its row's largest value."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import device as dev  # noqa: E402
from annc_b200._lib import ACT_NONE, ACT_SIGMOID  # noqa: E402

HEADS, KV, DIM, WIDTH = 8, 2, 64, 256


class Block:
    """Weights of one layer and the plans a program keeps."""

    def __init__(self, max_tokens, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda k, n: torch.randn((k, n), device="cuda", generator=g) * k ** -0.5
        self.qkv = dev.i8_weight(r(WIDTH, (HEADS + 2 * KV) * DIM))
        self.proj = dev.i8_weight(r(HEADS * DIM, WIDTH))
        self.score = dev.i8_weight(r(WIDTH, 1))
        self.bias = torch.randn(1, device="cuda", generator=g)
        self.rotary = dev.Rotary(DIM, base=10000.0, scaling="yarn", factor=4.0, original_len=2048)
        self.attention = dev.PrefixAttention(HEADS, KV, DIM, max_tokens)

    def linear(self, x, weight, dtype, bias=None, act=ACT_NONE):
        q, scale = dev.i8_rows(*x.shape), torch.empty(x.shape[0], device="cuda")
        y = torch.empty((x.shape[0], weight[0].shape[0]), dtype=dtype, device="cuda")
        dev.quantize_rows(x, q, scale)
        dev.gemm_i8(q, scale, weight[0], weight[1], y, bias=bias, activation=act)
        return y

    def heads(self, x, positions):
        """Rotated queries and keys, and values: views of one projection buffer, turned in place."""
        y = self.linear(x, self.qkv, torch.bfloat16).view(x.shape[0], HEADS + 2 * KV, DIM)
        q, k, v = y[:, :HEADS], y[:, HEADS:HEADS + KV], y[:, HEADS + KV:]
        self.rotary.run(positions, q, q, k, k)
        return q, k, v

    def run(self, history, candidates, begin, lengths, q_begin, positions):
        _, kp, vp = self.heads(history, torch.arange(history.shape[0], device="cuda"))
        q, k, v = self.heads(candidates, positions)
        out = torch.empty((candidates.shape[0], HEADS, DIM), dtype=torch.bfloat16, device="cuda")
        self.attention.run(q, kp, vp, out, k_own=k, v_own=v, own_begin=begin, own_len=lengths, q_begin=q_begin)
        y = self.linear(out.view(-1, HEADS * DIM), self.proj, torch.float32)
        return self.linear(y, self.score, torch.float32, bias=self.bias, act=ACT_SIGMOID)[:, 0], out


def ref_linear(x, weight):
    x = x.double()
    scale = torch.maximum(x.abs().amax(1) / 127, torch.tensor(2.0 ** -126, device="cuda", dtype=torch.float64)).float().double()
    return (torch.round(x / scale[:, None]) @ weight[0].double().T) * scale[:, None] * weight[1].double()


def ref_block(b, history, candidates, nq, positions):
    def heads(x, pos):
        y = ref_linear(x, b.qkv).bfloat16().double().view(x.shape[0], HEADS + 2 * KV, DIM)
        angle = pos.double()[:, None] * b.rotary.freq
        turn = torch.polar(torch.full_like(angle, b.rotary.size), angle)[:, None]
        z = torch.complex(y[:, :HEADS + KV, :DIM // 2].contiguous(), y[:, :HEADS + KV, DIM // 2:].contiguous()) * turn
        return torch.cat([torch.cat([z.real, z.imag], -1).bfloat16().double(), y[:, HEADS + KV:]], 1)
    h = heads(history, torch.arange(history.shape[0], device="cuda"))
    c = heads(candidates, positions)
    out = torch.empty((candidates.shape[0], HEADS, DIM), dtype=torch.float64, device="cuda")
    at = 0
    for n in nq:
        for i in range(n):
            for head in range(HEADS):
                g = HEADS + head // (HEADS // KV)
                k = torch.cat([h[:, g], c[at:at + i + 1, g]])
                v = torch.cat([h[:, g + KV], c[at:at + i + 1, g + KV]])
                out[at + i, head] = torch.softmax(k @ c[at + i, head] * DIM ** -0.5, 0) @ v
        at += n
    o = out.bfloat16()
    return torch.sigmoid(ref_linear(ref_linear(o.view(-1, HEADS * DIM), b.proj), b.score) + b.bias.double())[:, 0], out


def batch(nq, history, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = int(sum(nq))
    starts = np.cumsum(nq) - nq
    pos = torch.tensor(np.concatenate([history + np.arange(n) for n in nq]), device="cuda")
    return dict(history=torch.randn((history, WIDTH), device="cuda", generator=g).bfloat16(),
                candidates=torch.randn((tokens, WIDTH), device="cuda", generator=g).bfloat16(),
                begin=torch.tensor(starts, device="cuda"), lengths=torch.tensor(nq, dtype=torch.int32, device="cuda"),
                q_begin=torch.tensor(np.concatenate([[0], np.cumsum(nq)]), dtype=torch.int32, device="cuda"), positions=pos)


def close(got, want):
    # Most values agree to a few bf16 steps; a value of the 8-bit activations on the other side of a border moves a
    # projection by one part in 127 of one of 256 or 512 inputs, far below this.
    assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -6


@pytest.mark.parametrize("nq,history", [([1] * 7, 50), ([1, 3, 2, 8, 1], 333), ([4] * 40, 1000)])
def test_block(nq, history):
    b = Block(sum(nq), 1)
    x = batch(np.asarray(nq), history, 2)
    score, out = b.run(**x)
    want_score, want_out = ref_block(b, x["history"], x["candidates"], nq, x["positions"])
    close(out, want_out)
    close(score, want_score)


def test_block_in_a_graph_and_on_another_stream():
    nq = np.asarray([2, 1, 5, 1, 1, 3] * 10)
    b = Block(int(nq.sum()), 3)
    x = batch(nq, 700, 4)
    want, want_out = b.run(**x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got, got_out = b.run(**x)
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(got_out, want_out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_out = b.run(**x)
    y = batch(nq, 700, 5)
    for name in ("history", "candidates"):
        x[name].copy_(y[name])
    graph.replay()
    graph.replay()
    want, want_out = b.run(**x)
    assert torch.equal(got, want) and torch.equal(got_out, want_out)
