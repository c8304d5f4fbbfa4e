"""A bounded wait that ran out, as the sequence operators see it: launches that meet the raised error word end at once, leave
C as it is and are reported; once the word is cleared the same operands give the same results as before."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import device  # noqa: E402
from annc_b200._lib import lib  # noqa: E402
from tests.test_gpu_gemm_i8 import operands  # noqa: E402
from tests.test_gpu_prefix_attention import BF16, F16, Batch  # noqa: E402


def timed_out():
    flag = C.c_int(-1)
    assert lib.annc_gemm_check(C.c_void_p(torch.cuda.current_stream().cuda_stream), C.byref(flag)) == 0
    return flag.value


@pytest.fixture
def raised():
    """Raises and clears the word by hand; never leaves it raised."""
    def to(value):
        torch.cuda.synchronize()
        assert lib.annc_gemm_debug_set_error_word(value) == 0
    yield to
    to(0)


@pytest.mark.parametrize("m,n,k,kernel", [(1, 1024, 4096, "tcgen05_i8"), (200, 300, 256, "tcgen05_i8"), (16384, 264, 640, "tcgen05_pair_i8")])
def test_products(m, n, k, kernel, raised):
    a, sa, b, sb, bias = operands(m, n, k, 3)
    c = torch.empty((m, n), dtype=BF16, device="cuda")
    assert device.gemm_i8_kernel_name(a, sa, b, sb, c, bias) == kernel
    device.gemm_i8(a, sa, b, sb, c, bias=bias)
    want = c.clone()
    assert timed_out() == 0
    raised(1)
    c.fill_(5.0)
    for _ in range(3):
        device.gemm_i8(a, sa, b, sb, c, bias=bias)
    assert timed_out() == 1 and bool((c == 5.0).all())
    raised(0)
    device.gemm_i8(a, sa, b, sb, c, bias=bias)
    assert timed_out() == 0 and torch.equal(c, want)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("tokens,prefix", [(1, 1000), (40, 5000), (700, 700)])
@pytest.mark.parametrize("own", [True, False])
def test_attention(tokens, prefix, dim, dtype, own, raised):
    b = Batch([1] * tokens, [(i * 5) % 9 for i in range(tokens)], 8, 2, dim, prefix, dtype, seed=tokens)
    plan = device.PrefixAttention(8, 2, dim, tokens, dtype=dtype)
    b.run(plan, own=own)
    want, want_lse = b.out.clone(), b.lse.clone()
    raised(1)
    for _ in range(3):
        b.run(plan, own=own)
    assert timed_out() == 1
    raised(0)
    b.run(plan, own=own)
    assert timed_out() == 0 and torch.equal(b.out, want) and torch.equal(b.lse, want_lse)
