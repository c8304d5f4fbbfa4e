"""8-bit products with very many rows, or channels, in layouts that the tensor-core kernels do not take."""
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import device  # noqa: E402
from annc_b200._lib import ACT_RELU  # noqa: E402


def far_out(m, n, k, dtype):
    """The product of dense operands (rows k bytes apart), against integers and one rounding for each step."""
    g = torch.Generator(device="cuda").manual_seed(m + k)
    ints = lambda r: torch.randint(-128, 128, (r, k), device="cuda", generator=g, dtype=torch.int8)
    a, b = ints(m), ints(n)
    sa, sb = torch.rand(m, device="cuda", generator=g) + 0.1, torch.rand(n, device="cuda", generator=g) + 0.1
    bias = torch.randn(n, device="cuda", generator=g)
    c = torch.full((m, n), 7.0, dtype=dtype, device="cuda")
    assert device.gemm_i8_kernel_name(a, sa, b, sb, c, bias, ACT_RELU) == "simt_i8"
    device.gemm_i8(a, sa, b, sb, c, bias=bias, activation=ACT_RELU)
    for first in range(0, m, 1 << 20):  # (in pieces, for the memory)
        to = slice(first, first + (1 << 20))
        prod = (a[to].double() @ b.double().T) * sa[to].double()[:, None] * sb.double()
        want = (prod + bias.double()).clamp_min(0)
        tol = 2.0 ** -24 * (3.01 * prod.abs() + want)
        if dtype != torch.float32:
            tol = tol + torch.finfo(dtype).eps / 2 * (want + tol)
        assert bool(((c[to].double() - want).abs() <= tol).all()), first


@pytest.mark.parametrize("m,n,k,dtype", [(4194240, 16, 8, torch.bfloat16), (4194241, 16, 8, torch.bfloat16), (5000003, 65, 3, torch.bfloat16),
                                         (4194305, 2, 0, torch.float32), (3, 4194305, 8, torch.float32)])
def test_rows_beyond_65535_tiles(m, n, k, dtype):
    far_out(m, n, k, dtype)
