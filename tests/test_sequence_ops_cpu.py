"""Sequence operators without a GPU: what the entry points refuse before they touch the device, calls that have
nothing to do, and the rotary frequencies against their formulas."""
import ctypes as C
import math

import pytest

import annc_b200  # noqa: F401
from annc_b200._lib import (ANNC_BF16, ANNC_F16, ANNC_F32, ANNC_I32, ANNC_I64, GemmI8Desc, PrefixAttentionDesc, RotaryDesc,
                            lib)

INVALID, UNSUPPORTED = 3, 102
P = 1 << 20  # an aligned address that is never followed


def err():
    return lib.annc_last_error().decode()


# ---------------------------------------------------------------- product

def gemm_desc(**kw):
    d = GemmI8Desc(8, 16, 32, 32, 32, 16, P, P, P, P, None, P, ANNC_F32, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,code,text", [
    (dict(m=-1), INVALID, "extents"), (dict(n=(1 << 30) + 1), INVALID, "extents"),
    (dict(k=131072, lda=131072, ldb=131072), UNSUPPORTED, "131071"),
    (dict(lda=31), INVALID, "leading"), (dict(ldb=31), INVALID, "leading"), (dict(ldc=15), INVALID, "leading"),
    (dict(activation=3), INVALID, "activation"), (dict(activation=-1), INVALID, "activation"),
    (dict(c_dtype=6), INVALID, "C is"), (dict(a=None), INVALID, "null"), (dict(b=None), INVALID, "null"),
    (dict(c=None), INVALID, "null"), (dict(scale_a=None), INVALID, "null"), (dict(scale_b=None), INVALID, "null"),
    (dict(scale_a=P + 2), INVALID, "aligned"), (dict(bias=P + 1), INVALID, "aligned"),
    (dict(c=P + 2), INVALID, "aligned"), (dict(c=P + 1, c_dtype=ANNC_BF16), INVALID, "aligned"),
])
def test_gemm_i8_refuses(kw, code, text):
    assert lib.annc_gemm_i8_run(C.byref(gemm_desc(**kw)), None) == code
    assert text in err()


def test_gemm_i8_null_descriptor_and_empty_products():
    assert lib.annc_gemm_i8_run(None, None) == INVALID
    assert lib.annc_gemm_i8_kernel_name(None) == b""
    assert lib.annc_gemm_i8_run(C.byref(gemm_desc(m=0, a=None, c=None, scale_a=None)), None) == 0
    assert lib.annc_gemm_i8_run(C.byref(gemm_desc(n=0, b=None, c=None, scale_b=None)), None) == 0


@pytest.mark.parametrize("args,text", [
    ((P, 6, 4, 8, 8, P, 16, P), "f32, bf16 or f16"), ((P, ANNC_F32, -1, 8, 8, P, 16, P), "extents"),
    ((P, ANNC_F32, 4, 8, 7, P, 16, P), "extents"), ((P, ANNC_F32, 4, 8, 8, P, 7, P), "extents"),
    ((P, ANNC_F32, 4, 1 << 30, 1 << 30, P, 1 << 30, P), "extents"),
    ((None, ANNC_F32, 4, 8, 8, P, 16, P), "null"), ((P, ANNC_F32, 4, 8, 8, None, 16, P), "null"),
    ((P, ANNC_F32, 4, 8, 8, P, 16, None), "null"), ((P + 2, ANNC_F32, 4, 8, 8, P, 16, P), "aligned"),
    ((P + 1, ANNC_F16, 4, 8, 8, P, 16, P), "aligned"), ((P, ANNC_F32, 4, 8, 8, P, 16, P + 2), "aligned"),
])
def test_quantize_rows_refuses(args, text):
    assert lib.annc_quantize_rows_dev(*args, None) == INVALID
    assert text in err()


def test_quantize_no_rows():
    assert lib.annc_quantize_rows_dev(None, ANNC_F32, 0, 8, 8, None, 8, None, None) == 0


@pytest.mark.parametrize("args", [(None, 8, P, 8, P, 8, 8), (P, 8, None, 8, P, 8, 8), (P, 8, P, 8, None, 8, 8),
                                  (P, 7, P, 8, P, 8, 8), (P, 8, P, 7, P, 8, 8), (P, 8, P, 8, P, 0, 8), (P, 8, P, 8, P, 8, 0),
                                  (P + 2, 8, P, 8, P, 8, 8), (P, 8, P, 8, P + 1, 8, 8)])
def test_i8_weight_refuses(args):
    assert lib.annc_i8_weight_dev(*args, None) == INVALID


# ---------------------------------------------------------------- rotary

def rotary_desc(x0=None, x1=None, **kw):
    d = RotaryDesc(ANNC_BF16, 64, 64, 0, ANNC_I64, 0, 4, P, P, 1.0)
    d.x[0] = x0 if x0 is not None else (P, P, 8, 512, 64, 512, 64)
    if x1 is not None:
        d.x[1] = x1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=ANNC_I32), "f32, bf16 or f16"), (dict(layout=2), "layout"), (dict(positions_dtype=ANNC_F32), "i32 or i64"),
    (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=66), "rot_dim"),
    (dict(rot_dim=514, head_dim=1024), "rot_dim"), (dict(tokens=-1), "extents"), (dict(positions=None), "positions"),
    (dict(freq=None), "positions or freq"), (dict(freq=P + 4), "aligned"), (dict(positions=P + 4), "aligned"),
    (dict(x0=(None, P, 8, 512, 64, 512, 64)), "null"), (dict(x0=(P, None, 8, 512, 64, 512, 64)), "null"),
    (dict(x0=(P + 1, P, 8, 512, 64, 512, 64)), "aligned"), (dict(x0=(P, P, -1, 512, 64, 512, 64)), "heads"),
    (dict(x1=(P, None, 8, 512, 64, 512, 64)), "null"),
])
def test_rotary_refuses(kw, text):
    assert lib.annc_rotary_dev(C.byref(rotary_desc(**kw)), None) == INVALID
    assert text in err()


def test_rotary_nothing_to_do():
    assert lib.annc_rotary_dev(None, None) == INVALID
    assert lib.annc_rotary_dev(C.byref(rotary_desc(tokens=0, positions=None)), None) == 0
    assert lib.annc_rotary_dev(C.byref(rotary_desc(x0=(None, None, 0, 0, 0, 0, 0))), None) == 0


def frequencies(rot, base=10000.0, scaling=0, factor=1.0, original=4096, fast=32.0, slow=1.0):
    out, size = (C.c_double * max(rot // 2, 1))(), C.c_float()
    rc = lib.annc_rotary_frequencies(rot, base, scaling, factor, original, fast, slow, out, C.byref(size))
    return rc, list(out), size.value


def close(got, want):  # a handful of roundings in 64 bits, one of them under a power
    return all(abs(g - w) <= 1e-13 * abs(w) for g, w in zip(got, want))


@pytest.mark.parametrize("rot", [2, 20, 64, 128, 512])
def test_rotary_frequencies(rot):
    plain = [10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)]
    rc, got, size = frequencies(rot)
    assert rc == 0 and size == 1.0 and close(got, plain)
    rc, got, size = frequencies(rot, scaling=1, factor=4.0)
    assert rc == 0 and size == 1.0 and close(got, [f / 4 for f in plain])
    rc, got, size = frequencies(rot, scaling=2, factor=4.0)
    base = 10000.0 * 4.0 ** (rot / (rot - 2)) if rot > 2 else 10000.0
    assert rc == 0 and size == 1.0 and close(got, [base ** (-2.0 * j / rot) for j in range(rot // 2)])
    rc, got, size = frequencies(rot, scaling=3, factor=8.0)
    assert rc == 0 and abs(size - (0.1 * math.log(8.0) + 1)) <= 2.0 ** -23
    for j, (g, f) in enumerate(zip(got, plain)):
        turns = 4096 * f / (2 * math.pi)
        assert f / 8 * (1 - 1e-12) <= g <= f * (1 + 1e-12)
        if rot >= 64 and turns >= 2 * 32:  # a pair's step away from the ends of the ramp
            assert close([g], [f])
        if rot >= 64 and turns <= 0.5:
            assert close([g], [f / 8])
    assert all(a >= b for a, b in zip(got, got[1:]))


@pytest.mark.parametrize("kw", [dict(rot=3), dict(rot=0), dict(rot=514), dict(rot=64, base=1.0), dict(rot=64, base=float("inf")),
                                dict(rot=64, scaling=4), dict(rot=64, scaling=1, factor=0.5),
                                dict(rot=64, scaling=1, factor=float("nan")), dict(rot=64, scaling=3, factor=2.0, original=0),
                                dict(rot=64, scaling=3, factor=2.0, slow=0.0), dict(rot=64, scaling=3, factor=2.0, fast=0.5)])
def test_rotary_frequencies_refuses(kw):
    assert frequencies(**kw)[0] == INVALID


# ---------------------------------------------------------------- attention

def attention_desc(**kw):
    d = PrefixAttentionDesc(ANNC_BF16, 8, 2, 64, 4, 4, 100, 50, 0.125, 0, P, 512, 64, P, 128, 64, P, 128, 64, P, 128, 64, P, 128,
                            64, P, P, None, P, 512, 64, None, P, 1 << 30)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=ANNC_F32), "bf16 or f16"), (dict(heads=7), "multiple"), (dict(kv_heads=0), "multiple"),
    (dict(heads=1), "multiple"), (dict(head_dim=0), "head_dim"), (dict(head_dim=257), "head_dim"), (dict(tokens=-1), "extents"),
    (dict(prefix_len=-1), "extents"), (dict(own_rows=-1), "extents"), (dict(sequences=3), "q_begin"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(k_prefix=None), "null"), (dict(v_prefix=None), "null"), (dict(k_own=None), "own"), (dict(own_begin=None), "own"),
    (dict(q=P + 1), "aligned"), (dict(v_own=P + 1), "aligned"), (dict(lse=P + 2), "aligned"), (dict(own_begin=P + 4), "aligned"),
    (dict(q_begin=P + 2), "aligned"), (dict(workspace=None), "workspace"), (dict(workspace=P + 8), "workspace"),
    (dict(workspace_bytes=1000), "workspace"),
])
def test_prefix_attention_refuses(kw, text):
    assert lib.annc_prefix_attention_dev(C.byref(attention_desc(**kw)), None) == INVALID
    assert text in err()


def test_prefix_attention_no_tokens():
    assert lib.annc_prefix_attention_dev(None, None) == INVALID
    assert lib.annc_prefix_attention_dev(C.byref(attention_desc(tokens=0, sequences=0, q=None, out=None)), None) == 0


def test_prefix_attention_workspace():
    ws = lib.annc_prefix_attention_workspace_bytes
    assert ws(0, 8, 2, 64) == 0 and ws(4, 7, 2, 64) == 0 and ws(4, 8, 0, 64) == 0
    assert ws(4, 8, 2, 256) == 0  # taken row by row, without parts
    for heads, kv, dim in ((8, 2, 64), (8, 8, 128), (96, 1, 40)):
        sizes = [ws(t, heads, kv, dim) for t in (1, 2, 7, 100, 1000, 100000)]
        assert sizes == sorted(sizes) and sizes[0] > 0  # what serves many tokens serves few
