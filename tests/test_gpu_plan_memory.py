"""Memory that Rotary and PrefixAttention keep, used on another stream than the one it was made on."""
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import device  # noqa: E402
from tests.test_gpu_prefix_attention import Batch  # noqa: E402

LONG = 100_000_000  # cycles, some 50 ms


def rotary_case():
    x, pos = torch.randn((40, 2, 64), device="cuda"), torch.arange(40, device="cuda")
    out = torch.empty_like(x)
    return (lambda: device.Rotary(64)), (lambda plan: plan.run(pos, x, out)), (lambda plan: plan.freq), out


def attention_case():
    b = Batch([1] * 40, [(i * 5) % 9 for i in range(40)], 8, 2, 64, 3000)
    return (lambda: device.PrefixAttention(8, 2, 64, 40)), (lambda plan: b.run(plan)), (lambda plan: plan.ws), b.out


CASES = [rotary_case, attention_case]


@pytest.mark.parametrize("case", CASES)
def test_memory_is_not_handed_out_under_a_run(case):
    make, run, kept, out = case()
    run(make())
    want = out.clone()
    side = torch.cuda.Stream()
    plan = make()
    at, size, dtype = kept(plan).data_ptr(), kept(plan).numel(), kept(plan).dtype
    torch.cuda.synchronize()
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        run(plan)
    del plan
    others = [torch.empty(size, dtype=dtype, device="cuda") for _ in range(4)]  # (what would have taken its place)
    assert not side.query()
    assert all(t.data_ptr() != at for t in others)
    side.synchronize()
    assert torch.equal(out, want)
    torch.empty(1, device="cuda")  # (freed blocks whose streams are done come back)


@pytest.mark.parametrize("case", CASES)
def test_a_run_waits_for_what_had_the_memory_before(case):
    make, run, kept, out = case()
    run(make())
    want = out.clone()
    side, before = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    torch.cuda._sleep(LONG)
    before.record()
    plan = make()
    with torch.cuda.stream(side):
        run(plan)
        run(plan)
    side.synchronize()
    assert before.query()
    assert torch.equal(out, want)


@pytest.mark.parametrize("case", CASES)
def test_first_use_of_a_plan_in_a_capture_on_another_stream(case):
    make, run, kept, out = case()
    run(make())
    want = out.clone()
    plan = make()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(plan)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(plan)
    side.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("case", CASES)
def test_copies_of_a_plan(case):
    import copy
    import io
    make, run, kept, out = case()
    plan = make()
    run(plan)
    want = out.clone()
    stored = io.BytesIO()
    torch.save(plan, stored)
    stored.seek(0)
    side = torch.cuda.Stream()
    for other in (copy.deepcopy(plan), torch.load(stored, weights_only=False)):
        assert kept(other).data_ptr() != kept(plan).data_ptr()
        out.zero_()
        run(other)
        assert torch.equal(out, want)
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(other)
        side.synchronize()
        assert torch.equal(out, want)
