"""ctypes binding of libannc_b200.so.  There is no fallback: if the library has not
been built the import of the package fails, and every compute call fails with
ANNC_ERR_CUDA on a machine without a CUDA device."""
from __future__ import annotations

import ctypes as C
import os
import struct

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "lib", "libannc_b200.so")

ANNC_F32, ANNC_I32, ANNC_I64, ANNC_BOOL, ANNC_BF16, ANNC_F16, ANNC_U64 = 1, 3, 9, 10, 14, 19, 23
ERR_INVALID_ARGUMENT = 3
ACT_NONE, ACT_RELU, ACT_SIGMOID = 0, 1, 2
B_PLAIN, B_KN4 = 0, 1
MATH_AUTO, MATH_FP32, MATH_TF32, MATH_BF16 = 0, 1, 2, 3
ROTARY_HALF, ROTARY_INTERLEAVED = 0, 1
ROTARY_UNSCALED, ROTARY_LINEAR, ROTARY_NTK, ROTARY_YARN = 0, 1, 2, 3
IO_A_BF16, IO_B_BF16, IO_C_BF16, IO_SOFTMAX, IO_PAIR, IO_SINGLE = 1, 2, 4, 8, 16, 32


class AnncError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"[annc {code}] {message}")
        self.code = code
        self.message = message


class Tensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("dtype", C.c_int32), ("rank", C.c_int32),
                ("dims", C.c_int64 * 4)]


class BagTable(C.Structure):
    _fields_ = [("table", C.c_void_p), ("rows", C.c_int64), ("num_buckets", C.c_int64),
                ("ids", C.c_void_p), ("slice_input", C.c_void_p), ("nnz", C.c_int64),
                ("out", C.c_void_p), ("offsets", C.c_void_p)]


class GemmDesc(C.Structure):
    _fields_ = [("trans_a", C.c_int32), ("trans_b", C.c_int32),
                ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64), ("batch", C.c_int64),
                ("lda", C.c_int64), ("ldb", C.c_int64), ("ldc", C.c_int64), ("ld_addend", C.c_int64),
                ("stride_a", C.c_int64), ("stride_b", C.c_int64), ("stride_c", C.c_int64),
                ("stride_addend", C.c_int64),
                ("alpha", C.c_float), ("beta", C.c_float),
                ("a", C.c_void_p), ("b", C.c_void_p), ("c", C.c_void_p),
                ("addend", C.c_void_p), ("bias", C.c_void_p),
                ("activation", C.c_int32), ("b_format", C.c_int32), ("math", C.c_int32),
                ("io_flags", C.c_int32), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class GemmI8Desc(C.Structure):
    _fields_ = [("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
                ("lda", C.c_int64), ("ldb", C.c_int64), ("ldc", C.c_int64),
                ("a", C.c_void_p), ("b", C.c_void_p), ("scale_a", C.c_void_p), ("scale_b", C.c_void_p),
                ("bias", C.c_void_p), ("c", C.c_void_p), ("c_dtype", C.c_int32), ("activation", C.c_int32)]


class RotaryHeads(C.Structure):
    _fields_ = [("in_", C.c_void_p), ("out", C.c_void_p), ("heads", C.c_int64),
                ("in_token", C.c_int64), ("in_head", C.c_int64), ("out_token", C.c_int64), ("out_head", C.c_int64)]


class RotaryDesc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("head_dim", C.c_int32), ("rot_dim", C.c_int32), ("layout", C.c_int32),
                ("positions_dtype", C.c_int32), ("transposed", C.c_int32), ("tokens", C.c_int64),
                ("positions", C.c_void_p), ("freq", C.c_void_p), ("size", C.c_float), ("reserved", C.c_int32),
                ("x", RotaryHeads * 2)]


class PrefixAttentionDesc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32),
                ("tokens", C.c_int64), ("sequences", C.c_int64), ("prefix_len", C.c_int64), ("own_rows", C.c_int64),
                ("scale", C.c_float), ("reserved", C.c_int32)] + \
        [f for name in ("q", "k_prefix", "v_prefix", "k_own", "v_own")
         for f in ((name, C.c_void_p), (name + "_row", C.c_int64), (name + "_head", C.c_int64))] + \
        [("own_begin", C.c_void_p), ("own_len", C.c_void_p), ("q_begin", C.c_void_p),
         ("out", C.c_void_p), ("out_row", C.c_int64), ("out_head", C.c_int64), ("lse", C.c_void_p),
         ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


# The same layouts as bytes: the calls of device.py fill a descriptor in 0.5 us this way, a Structure takes 1.5 us.
PACK_GEMM_I8 = struct.Struct("@6q6P2i")
PACK_ROTARY = struct.Struct("@6iq2Pfi" + "2P5q" * 2)
PACK_PREFIX_ATTENTION = struct.Struct("@4i4qfi" + "P2q" * 5 + "3PP2q2PN")
for _pack, _desc in ((PACK_GEMM_I8, GemmI8Desc), (PACK_ROTARY, RotaryDesc), (PACK_PREFIX_ATTENTION, PrefixAttentionDesc)):
    assert _pack.size == C.sizeof(_desc)

ALLOC_FN = C.CFUNCTYPE(C.c_void_p, C.c_void_p, C.c_int, C.c_int32, C.c_int32, C.POINTER(C.c_int64))


def _load() -> C.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python annc_b200/build.py` "
            "(nvcc, sm_100a). annc_b200 has no CPU fallback.")
    lib = C.CDLL(LIB_PATH)
    lib.annc_last_error.restype = C.c_char_p
    lib.annc_version.restype = C.c_char_p
    lib.annc_get_stream.restype = C.c_void_p
    lib.annc_set_stream.argtypes = [C.c_void_p]
    lib.annc_lookup_custom_call.restype = C.c_void_p
    lib.annc_lookup_custom_call.argtypes = [C.c_char_p]
    lib.annc_select_gemm_target.restype = C.c_char_p
    lib.annc_gemm_kernel_name.restype = C.c_char_p
    lib.annc_gemm_run.argtypes = [C.POINTER(GemmDesc), C.c_void_p]
    lib.annc_gemm_i8_run.argtypes = [C.c_void_p, C.c_void_p]  # (a descriptor by reference, or its bytes)
    lib.annc_gemm_i8_kernel_name.restype = C.c_char_p
    lib.annc_gemm_i8_kernel_name.argtypes = [C.c_void_p]
    lib.annc_quantize_rows_dev.argtypes = [C.c_void_p, C.c_int32, C.c_int64, C.c_int64, C.c_int64, C.c_void_p,
                                           C.c_int64, C.c_void_p, C.c_void_p]
    lib.annc_i8_weight_dev.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64,
                                       C.c_int64, C.c_void_p]
    lib.annc_rotary_frequencies.argtypes = [C.c_int32, C.c_double, C.c_int32, C.c_double, C.c_int64, C.c_double,
                                            C.c_double, C.POINTER(C.c_double), C.POINTER(C.c_float)]
    lib.annc_rotary_dev.argtypes = [C.c_void_p, C.c_void_p]
    lib.annc_prefix_attention_workspace_bytes.restype = C.c_size_t
    lib.annc_prefix_attention_workspace_bytes.argtypes = [C.c_int64, C.c_int32, C.c_int32, C.c_int32]
    lib.annc_prefix_attention_dev.argtypes = [C.c_void_p, C.c_void_p]
    lib.annc_embed_bag_workspace_bytes.restype = C.c_size_t
    lib.annc_embed_bag_workspace_bytes.argtypes = [C.c_int, C.c_int64]
    lib.annc_kn4_offset.restype = C.c_int64
    lib.annc_kn4_offset.argtypes = [C.c_int64] * 4
    lib.annc_timer_create.restype = C.c_void_p
    lib.annc_timer_destroy.argtypes = [C.c_void_p]
    lib.annc_timer_elapsed_ms.argtypes = [C.c_void_p, C.c_void_p, C.POINTER(C.c_float)]
    lib.annc_embed_bag_set_timing_events.argtypes = [C.c_void_p, C.c_void_p]
    lib.annc_embed_bag_set_stream_ctas_per_sm.argtypes = [C.c_int]
    lib.annc_embed_bag_set_stream_ctas_per_sm.restype = None
    lib.annc_embed_bag_stream_registers.argtypes = [C.c_int64, C.POINTER(C.c_int)]
    lib.annc_peer_buffer_create.argtypes = [C.c_size_t, C.POINTER(C.c_void_p), C.c_void_p]
    lib.annc_peer_buffer_open.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    lib.annc_peer_buffer_close.argtypes = [C.c_void_p]
    lib.annc_peer_copy_dev.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
    lib.annc_peer_buffer_destroy.argtypes = [C.c_void_p]
    lib.annc_embed_bag_owner_mask_dev.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int64, C.c_int,
                                                  C.c_void_p, C.c_void_p]
    lib.annc_sum_partials_masked_dev.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int64, C.c_int64,
                                                 C.c_int, C.c_int64, C.c_void_p, C.c_void_p, C.c_int64,
                                                 C.c_int, C.c_void_p]
    lib.annc_synth_fill_rows_dev.argtypes = [C.c_void_p, C.c_int64, C.c_int64, C.c_uint64, C.c_int64,
                                             C.c_int64, C.c_int64, C.c_void_p]
    lib.annc_synth_fill_row_list_dev.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_uint64,
                                                 C.c_int64, C.c_void_p]
    lib.annc_set_operand_cache.argtypes = [C.c_int, C.c_size_t]
    lib.annc_staging_counters.argtypes = [C.POINTER(C.c_uint64)] * 3
    lib.annc_register_constant.argtypes = [C.c_void_p, C.c_size_t]
    lib.annc_unregister_constant.argtypes = [C.c_void_p]
    return lib


lib = _load()


def check(rc: int) -> None:
    if rc != 0:
        raise AnncError(rc, lib.annc_last_error().decode(errors="replace"))
