"""Device-pointer entry points (`*_dev`, annc_gemm_run) on torch CUDA tensors.

torch supplies device memory and the stream; every kernel that runs is from
libannc_b200.so.  Nothing here allocates inside a call: outputs and workspaces are
passed in, so the calls can sit in a timed loop or under stream capture."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch

from ._lib import (ACT_NONE, ANNC_BF16, ANNC_F16, ANNC_F32, ANNC_I32, ANNC_I64, B_PLAIN, ERR_INVALID_ARGUMENT, MATH_AUTO,
                   ROTARY_HALF, ROTARY_INTERLEAVED, ROTARY_LINEAR, ROTARY_NTK, ROTARY_UNSCALED, ROTARY_YARN, AnncError,
                   BagTable, GemmDesc, GemmI8Desc, PrefixAttentionDesc, RotaryDesc, check, lib)


def raw_stream() -> int:
    """Handle of torch's current stream, without the Stream object around it (0.2 us, not 3 us)."""
    if not torch.cuda.is_initialized():
        return torch.cuda.current_stream().cuda_stream
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _stream() -> C.c_void_p:
    return C.c_void_p(raw_stream())


class BagPlan:
    """Holds the host descriptor array and the device workspace of one grouped
    embedding-bag call (tables, id buffers, segment matrices and outputs fixed).  One run() at a
    time: runs on different streams that may overlap need a plan each (the workspace holds the
    counter from which the kernel hands out its work)."""

    def __init__(self, tables: Sequence[torch.Tensor], ids: Sequence[torch.Tensor],
                 slice_inputs: Sequence[torch.Tensor], out: torch.Tensor, out_slot0: int,
                 batch: int, id_kind: int = 2, col: int = 0, combiner: int = 0,
                 num_buckets: Optional[Sequence[int]] = None,
                 out_slots: Optional[Sequence[int]] = None):
        self.n = len(tables)
        self.dim = int(tables[0].shape[1])
        self.batch = int(batch)
        self.id_kind, self.col, self.combiner = id_kind, col, combiner
        self.ncols = int(slice_inputs[0].shape[1])
        self.out = out
        # out is [batch, slots, dim]; table t writes slot out_slot0 + t (or out_slot0 + out_slots[t])
        slots = int(out.shape[1]) if out.dim() == 3 else 1
        self.out_stride = slots * self.dim
        self.keep = (list(tables), list(ids), list(slice_inputs))
        self.desc = (BagTable * self.n)()
        esz = out.element_size()
        for t in range(self.n):
            d = self.desc[t]
            d.table = tables[t].data_ptr()
            d.rows = int(tables[t].shape[0])
            d.num_buckets = int(num_buckets[t]) if num_buckets is not None else int(tables[t].shape[0])
            d.ids = ids[t].data_ptr()
            d.slice_input = slice_inputs[t].data_ptr()
            d.nnz = int(ids[t].shape[0])
            d.out = out.data_ptr() + (out_slot0 + (out_slots[t] if out_slots is not None else t)) * self.dim * esz
        self.ws_bytes = int(lib.annc_embed_bag_workspace_bytes(self.n, self.batch))
        self.ws = torch.zeros(self.ws_bytes, dtype=torch.uint8, device=out.device)

    def run(self) -> None:
        check(lib.annc_embed_bags_dev(self.desc, C.c_int(self.n), C.c_int64(self.dim),
                                      C.c_int(self.id_kind), C.c_int64(self.ncols),
                                      C.c_int32(self.col), C.c_int(self.combiner),
                                      C.c_int64(self.batch), C.c_int64(self.out_stride),
                                      C.c_void_p(self.ws.data_ptr()), C.c_size_t(self.ws_bytes),
                                      _stream()))

    def error_bits(self) -> int:
        bits = C.c_int(0)
        check(lib.annc_embed_bag_check(C.c_void_p(self.ws.data_ptr()), _stream(), C.byref(bits)))
        return bits.value


def gemm(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, *, m: int, n: int, k: int,
         trans_a: bool = False, trans_b: bool = False, batch: int = 1,
         lda: Optional[int] = None, ldb: Optional[int] = None, ldc: Optional[int] = None,
         stride_a: int = 0, stride_b: int = 0, stride_c: int = 0,
         alpha: float = 1.0, beta: float = 0.0, addend: Optional[torch.Tensor] = None,
         ld_addend: Optional[int] = None, stride_addend: int = 0,
         bias: Optional[torch.Tensor] = None, activation: int = ACT_NONE,
         b_format: int = B_PLAIN, math: int = MATH_AUTO,
         workspace: Optional[torch.Tensor] = None, io_flags: int = 0,
         stream: Optional[int] = None) -> str:
    """annc_gemm_run on the current stream (or the one whose handle is given); returns the name of
    the kernel family that ran."""
    d = GemmDesc(1 if trans_a else 0, 1 if trans_b else 0, m, n, k, batch,
                 (m if trans_a else k) if lda is None else lda,
                 (k if trans_b else n) if ldb is None else ldb,
                 n if ldc is None else ldc, n if ld_addend is None else ld_addend,
                 stride_a, stride_b, stride_c, stride_addend, alpha, beta,
                 a.data_ptr(), b.data_ptr(), c.data_ptr(),
                 None if addend is None else addend.data_ptr(), None if bias is None else bias.data_ptr(),
                 activation, b_format, math, io_flags)
    if workspace is not None:
        d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    name = lib.annc_gemm_kernel_name(C.byref(d)).decode()
    rc = lib.annc_gemm_run(C.byref(d), raw_stream() if stream is None else stream)
    if rc:
        check(rc)
    return name


def softmax(x: torch.Tensor, out: torch.Tensor) -> None:
    ch = x.shape[-1]
    check(lib.annc_softmax_dev(C.c_void_p(x.data_ptr()), C.c_void_p(out.data_ptr()),
                               C.c_int64(x.numel() // ch), C.c_int64(ch), _stream()))


def gemv(a: torch.Tensor, x: torch.Tensor, y: torch.Tensor, m: int, n: int, trans_a=False,
         alpha=1.0, beta=0.0) -> None:
    check(lib.annc_gemv_dev(C.c_int(int(trans_a)), C.c_int64(m), C.c_int64(n), C.c_float(alpha),
                            C.c_void_p(a.data_ptr()), C.c_void_p(x.data_ptr()), C.c_float(beta),
                            C.c_void_p(y.data_ptr()), _stream()))


def dot_interaction(z: torch.Tensor, out: torch.Tensor, math: int = MATH_AUTO) -> None:
    """z f32[batch, F, D] -> out f32[batch, out_stride] = [z[:,0,:] | tril(z z^T, -1) | 0 pad]."""
    batch, F, D = z.shape
    check(lib.annc_dot_interaction_dev(C.c_void_p(z.data_ptr()), C.c_int64(batch), C.c_int(F),
                                       C.c_int(D), C.c_int64(F * D), C.c_void_p(out.data_ptr()),
                                       C.c_int64(out.shape[1]), C.c_int(math), _stream()))


def bf16_weight(b_kn: torch.Tensor) -> torch.Tensor:
    """fp32 [K,N] -> bf16 [N,K] for the BF16 route (annc_bf16_weight_dev)."""
    k, n = b_kn.shape
    out = torch.empty((n, k), dtype=torch.bfloat16, device=b_kn.device)
    check(lib.annc_bf16_weight_dev(C.c_void_p(b_kn.data_ptr()), C.c_int64(b_kn.stride(0)),
                                   C.c_void_p(out.data_ptr()), C.c_int64(k), C.c_int64(n), _stream()))
    return out


def cast_bf16(x: torch.Tensor) -> torch.Tensor:
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    check(lib.annc_cast_bf16_dev(C.c_void_p(x.data_ptr()), C.c_void_p(out.data_ptr()),
                                 C.c_int64(x.numel()), _stream()))
    return out


def kn4_pack(b_kn: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(b_kn)
    check(lib.annc_kn4_pack_dev(C.c_void_p(b_kn.data_ptr()), C.c_void_p(out.data_ptr()),
                                C.c_int64(b_kn.shape[0]), C.c_int64(b_kn.shape[1]), _stream()))
    return out


def kn4_unpack(b_packed: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(b_packed)
    check(lib.annc_kn4_unpack_dev(C.c_void_p(b_packed.data_ptr()), C.c_void_p(out.data_ptr()),
                                  C.c_int64(b_packed.shape[0]), C.c_int64(b_packed.shape[1]),
                                  _stream()))
    return out


def gemm_timed_out() -> bool:
    """True when a tensor-core GEMM CTA gave up on a bounded wait since the library was
    loaded (annc_gemm_check; synchronises the current stream)."""
    flag = C.c_int(0)
    check(lib.annc_gemm_check(_stream(), C.byref(flag)))
    return flag.value != 0


class BagLaunch:
    """Grouped embedding-bag launch over explicit (table, ids, segments, output) entries,
    optionally row-sharded (annc_embed_bags_sharded_dev).  Each entry is a tuple
    (table_ptr, local_rows, num_buckets, ids_ptr, seg_ptr, nnz, out_ptr[, offsets_ptr]); with
    offsets_ptr (i32[batch + 1] bag offsets) the segment matrix is not read."""

    def __init__(self, entries, dim: int, batch: int, ncols: int, out_stride: int,
                 device: torch.device, id_kind: int = 2, col: int = 0, combiner: int = 0,
                 shard_count: int = 1, shard_rank: int = 0, exchange: bool = False):
        self.exchange = exchange  # annc_embed_bags_exchange_dev: bags without an owned lookup are not written
        self.n = len(entries)
        self.dim, self.batch, self.ncols, self.out_stride = dim, batch, ncols, out_stride
        self.id_kind, self.col, self.combiner = id_kind, col, combiner
        self.shard_count, self.shard_rank = shard_count, shard_rank
        self.desc = (BagTable * self.n)()
        for i, e in enumerate(entries):
            tp, rows, nb, ip, sp, nnz, op = e[:7]
            d = self.desc[i]
            d.table, d.rows, d.num_buckets, d.ids, d.slice_input, d.nnz, d.out = \
                tp, int(rows), int(nb), ip, sp, int(nnz), op
            d.offsets = e[7] if len(e) > 7 else None
        self.ws_bytes = int(lib.annc_embed_bag_workspace_bytes(self.n, self.batch))
        self.ws = torch.zeros(self.ws_bytes, dtype=torch.uint8, device=device)

    def run(self) -> None:
        if self.exchange:
            check(lib.annc_embed_bags_exchange_dev(
                self.desc, C.c_int(self.n), C.c_int64(self.dim), C.c_int(self.id_kind),
                C.c_int(self.combiner), C.c_int64(self.batch), C.c_int64(self.out_stride),
                C.c_int(self.shard_count), C.c_int(self.shard_rank),
                C.c_void_p(self.ws.data_ptr()), C.c_size_t(self.ws_bytes), _stream()))
            return
        check(lib.annc_embed_bags_sharded_dev(
            self.desc, C.c_int(self.n), C.c_int64(self.dim), C.c_int(self.id_kind),
            C.c_int64(self.ncols), C.c_int32(self.col), C.c_int(self.combiner),
            C.c_int64(self.batch), C.c_int64(self.out_stride), C.c_int(self.shard_count),
            C.c_int(self.shard_rank), C.c_void_p(self.ws.data_ptr()), C.c_size_t(self.ws_bytes),
            _stream()))

    def error_bits(self) -> int:
        bits = C.c_int(0)
        check(lib.annc_embed_bag_check(C.c_void_p(self.ws.data_ptr()), _stream(), C.byref(bits)))
        return bits.value


def sum_partials(src: torch.Tensor, parts: int, part_stride: int, rows: int, width: int,
                 src_stride: int, out_ptr: int, out_stride: int) -> None:
    check(lib.annc_sum_partials_dev(C.c_void_p(src.data_ptr()), C.c_int(parts), C.c_int64(part_stride),
                                    C.c_int64(rows), C.c_int64(width), C.c_int64(src_stride),
                                    C.c_void_p(out_ptr), C.c_int64(out_stride), _stream()))


def sum_partials_ptr(src_ptr: int, parts: int, part_stride: int, rows: int, width: int,
                     src_stride: int, out_ptr: int, out_stride: int) -> None:
    check(lib.annc_sum_partials_dev(C.c_void_p(src_ptr), C.c_int(parts), C.c_int64(part_stride),
                                    C.c_int64(rows), C.c_int64(width), C.c_int64(src_stride),
                                    C.c_void_p(out_ptr), C.c_int64(out_stride), _stream()))


def peer_copy(dst_ptr: int, src_ptr: int, nbytes: int) -> None:
    """annc_peer_copy_dev on the current stream (raw pointers: either may be a peer mapping)."""
    check(lib.annc_peer_copy_dev(C.c_void_p(dst_ptr), C.c_void_p(src_ptr), C.c_size_t(nbytes), _stream()))


def cast_bf16_ptr(src_ptr: int, dst_ptr: int, n: int) -> None:
    check(lib.annc_cast_bf16_dev(C.c_void_p(src_ptr), C.c_void_p(dst_ptr), C.c_int64(n), _stream()))


class OwnerMask:
    """annc_embed_bag_owner_mask_dev over fixed id / offset buffers: which ranks hold a part
    of each bag of this rank's batch.  entries: (ids_ptr, nnz, num_buckets, offsets_ptr)."""

    def __init__(self, entries, batch: int, shard_count: int, device: torch.device, id_kind: int = 2):
        self.n, self.batch, self.shard_count, self.id_kind = len(entries), batch, shard_count, id_kind
        self.desc = (BagTable * self.n)()
        for i, (ip, nnz, nb, op) in enumerate(entries):
            d = self.desc[i]
            d.ids, d.nnz, d.num_buckets, d.offsets = ip, int(nnz), int(nb), op
        self.mask = torch.zeros(self.n * batch, dtype=torch.int32, device=device)

    def run(self) -> None:
        check(lib.annc_embed_bag_owner_mask_dev(self.desc, C.c_int(self.n), C.c_int(self.id_kind),
                                                C.c_int64(self.batch), C.c_int(self.shard_count),
                                                C.c_void_p(self.mask.data_ptr()), _stream()))


def sum_partials_masked(src_ptr: int, mask: torch.Tensor, parts: int, part_stride: int, rows: int,
                        slots: int, slot_width: int, out_ptr: int, out_stride: int,
                        mean_offsets_ptr: Optional[int] = None, out_bf16: bool = False) -> None:
    check(lib.annc_sum_partials_masked_dev(C.c_void_p(src_ptr), C.c_void_p(mask.data_ptr()),
                                           C.c_int(parts), C.c_int64(part_stride), C.c_int64(rows),
                                           C.c_int(slots), C.c_int64(slot_width),
                                           C.c_void_p(mean_offsets_ptr), C.c_void_p(out_ptr),
                                           C.c_int64(out_stride), C.c_int(int(out_bf16)), _stream()))


class PeerBuffers:
    """One receive buffer per rank, mapped into every rank (annc_peer_buffer_*).  `local` is
    this rank's buffer, `ptrs[p]` the address under which rank p's buffer is seen here.
    Handles travel through torch.distributed (host side); the data path is plain stores."""

    def __init__(self, nbytes: int, world: int, rank: int):
        import torch.distributed as dist
        ptr = C.c_void_p()
        handle = (C.c_ubyte * 64)()
        check(lib.annc_peer_buffer_create(C.c_size_t(nbytes), C.byref(ptr), handle))
        self.local = int(ptr.value)
        self.nbytes, self.rank = nbytes, rank
        handles = [None] * world
        dist.all_gather_object(handles, bytes(handle))
        self.ptrs = []
        for p in range(world):
            if p == rank:
                self.ptrs.append(self.local)
                continue
            q = C.c_void_p()
            buf = (C.c_ubyte * 64).from_buffer_copy(handles[p])
            check(lib.annc_peer_buffer_open(buf, C.byref(q)))
            self.ptrs.append(int(q.value))

    def close(self) -> None:
        """Unmaps the peers' buffers, waits for every rank to have done so, frees this one."""
        import torch.distributed as dist
        for p, q in enumerate(self.ptrs):
            if p != self.rank and q:
                check(lib.annc_peer_buffer_close(C.c_void_p(q)))
        self.ptrs = []
        if dist.is_initialized():
            dist.barrier()
        if self.local:
            check(lib.annc_peer_buffer_destroy(C.c_void_p(self.local)))
            self.local = 0


def copy_rows(dst_ptr: int, dst_stride: int, src_ptr: int, src_stride: int, width: int,
              rows: int) -> None:
    """2-D device copy of `rows` rows of `width` floats between pitched buffers."""
    check(lib.annc_copy_rows_dev(C.c_void_p(dst_ptr), C.c_int64(dst_stride), C.c_void_p(src_ptr),
                                 C.c_int64(src_stride), C.c_int64(width), C.c_int64(rows), _stream()))


class BagPrepass:
    """Segment prepass alone (annc_embed_bag_prepass_dev): bag offsets of every table's
    lookups into `ws` (512-byte header, then i32 offsets[tables][batch + 1])."""

    def __init__(self, slice_inputs: Sequence[torch.Tensor], batch: int, col: int = 0):
        self.n = len(slice_inputs)
        self.batch, self.col = int(batch), col
        self.ncols = int(slice_inputs[0].shape[1])
        self.desc = (BagTable * self.n)()
        for t, s in enumerate(slice_inputs):
            self.desc[t].slice_input = s.data_ptr()
            self.desc[t].nnz = int(s.shape[0])
        self.ws_bytes = int(lib.annc_embed_bag_workspace_bytes(self.n, self.batch))

    def run(self, ws: torch.Tensor) -> None:
        self.run_ptr(ws.data_ptr())

    def run_ptr(self, ws_ptr: int) -> None:
        check(lib.annc_embed_bag_prepass_dev(self.desc, C.c_int(self.n), C.c_int64(self.ncols),
                                             C.c_int32(self.col), C.c_int64(self.batch),
                                             C.c_void_p(ws_ptr), C.c_size_t(self.ws_bytes),
                                             _stream()))


# ---------------------------------------------------------------- sequence operators

_DTYPES = {torch.float32: ANNC_F32, torch.bfloat16: ANNC_BF16, torch.float16: ANNC_F16}


def _require(cond: bool, message: str) -> None:
    if not cond:
        raise AnncError(ERR_INVALID_ARGUMENT, message)


def _operand(name: str, t: torch.Tensor, dtypes, shape) -> None:
    """A tensor of the current device with one of the types and the shape (None: any extent), the values of its
    last dimension adjacent."""
    _require(t.is_cuda and t.device.index == torch.cuda.current_device(), f"{name}: not on the current CUDA device")
    _require(t.dtype in dtypes, f"{name}: bad type {t.dtype}")
    _require(t.dim() == len(shape) and all(w is None or w == g for w, g in zip(shape, t.shape)),
             f"{name}: bad shape {tuple(t.shape)}")
    _require(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: the values of the last dimension are not adjacent")


def _pitch(t: torch.Tensor) -> int:
    """Elements from row to row; a single row has any."""
    return max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)


def i8_rows(rows: int, cols: int, device=None) -> torch.Tensor:
    """i8[rows, cols] whose rows start on 16 bytes, as the tensor-core product wants its operands."""
    return torch.empty((rows, max(cols + 15, 16) // 16 * 16), dtype=torch.int8, device=device or "cuda")[:, :cols]


def quantize_rows(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """annc_quantize_rows_dev: x f32 / bf16 / f16 [rows, cols] -> q i8[rows, cols] (i8_rows), scale f32[rows]."""
    _operand("x", x, _DTYPES, (None, None))
    _operand("q", q, (torch.int8,), x.shape)
    _operand("scale", scale, (torch.float32,), (x.shape[0],))
    rc = lib.annc_quantize_rows_dev(x.data_ptr(), _DTYPES[x.dtype], x.shape[0], x.shape[1], _pitch(x), q.data_ptr(),
                                    _pitch(q), scale.data_ptr(), raw_stream())
    if rc:
        check(rc)


def i8_weight(b_kn: torch.Tensor):
    """f32 [K,N] -> (i8 [N,K] with rows on 16 bytes, f32 scale [N]) for gemm_i8 (annc_i8_weight_dev)."""
    _operand("b_kn", b_kn, (torch.float32,), (None, None))
    k, n = b_kn.shape
    q = i8_rows(n, k, b_kn.device)
    scale = torch.empty(n, dtype=torch.float32, device=b_kn.device)
    check(lib.annc_i8_weight_dev(b_kn.data_ptr(), _pitch(b_kn), q.data_ptr(), q.stride(0), scale.data_ptr(), k, n,
                                 raw_stream()))
    return q, scale


def gemm_i8_desc(a, scale_a, b, scale_b, c, bias=None, activation: int = ACT_NONE) -> GemmI8Desc:
    """The checked descriptor of gemm_i8."""
    m, n, k = a.shape[0], b.shape[0], a.shape[-1]
    _operand("a", a, (torch.int8,), (None, None))
    _operand("b", b, (torch.int8,), (None, k))
    _operand("scale_a", scale_a, (torch.float32,), (m,))
    _operand("scale_b", scale_b, (torch.float32,), (n,))
    _operand("c", c, _DTYPES, (m, n))
    if bias is not None:
        _operand("bias", bias, (torch.float32,), (n,))
    return GemmI8Desc(m, n, k, _pitch(a), _pitch(b), _pitch(c), a.data_ptr(), b.data_ptr(), scale_a.data_ptr(),
                      scale_b.data_ptr(), None if bias is None else bias.data_ptr(), c.data_ptr(), _DTYPES[c.dtype],
                      activation)


def gemm_i8(a: torch.Tensor, scale_a: torch.Tensor, b: torch.Tensor, scale_b: torch.Tensor, c: torch.Tensor, *,
            bias: Optional[torch.Tensor] = None, activation: int = ACT_NONE) -> None:
    """annc_gemm_i8_run on the current stream: c = act(a b^T * scale_a[:, None] * scale_b + bias); a i8[m,k], b
    i8[n,k], c f32 / bf16 / f16 [m,n]."""
    rc = lib.annc_gemm_i8_run(C.byref(gemm_i8_desc(a, scale_a, b, scale_b, c, bias, activation)), raw_stream())
    if rc:
        check(rc)


def gemm_i8_kernel_name(a, scale_a, b, scale_b, c, bias=None, activation: int = ACT_NONE) -> str:
    """Name of the kernel family that gemm_i8 takes for these operands."""
    return lib.annc_gemm_i8_kernel_name(C.byref(gemm_i8_desc(a, scale_a, b, scale_b, c, bias, activation))).decode()


class Rotary:
    """Rotary positions (annc_rotary_dev): holds the frequencies of annc_rotary_frequencies on the device.
    layout "half" or "interleaved"; scaling "none", "linear", "ntk" or "yarn" by `factor`."""

    def __init__(self, rot_dim: int, *, base: float = 10000.0, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original_len: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device=None):
        layouts = {"half": ROTARY_HALF, "interleaved": ROTARY_INTERLEAVED}
        scalings = {"none": ROTARY_UNSCALED, "linear": ROTARY_LINEAR, "ntk": ROTARY_NTK, "yarn": ROTARY_YARN}
        _require(layout in layouts, f"rotary: unknown layout {layout!r}")
        _require(scaling in scalings, f"rotary: unknown scaling {scaling!r}")
        self.rot_dim, self.layout = int(rot_dim), layouts[layout]
        host = (C.c_double * max(self.rot_dim // 2, 1))()
        size = C.c_float(0)
        check(lib.annc_rotary_frequencies(self.rot_dim, base, scalings[scaling], factor, original_len, beta_fast,
                                          beta_slow, host, C.byref(size)))
        self.size = size.value
        self.freq = torch.tensor(list(host), dtype=torch.float64, device=device or "cuda")

    def run(self, positions: torch.Tensor, q: torch.Tensor, out_q: torch.Tensor, k: Optional[torch.Tensor] = None,
            out_k: Optional[torch.Tensor] = None, *, transposed: bool = False) -> None:
        """q [tokens, heads, head_dim] -> out_q (q itself: in place), and k likewise in the same launch; positions
        i32 / i64 [tokens]."""
        _operand("q", q, _DTYPES, (None, None, None))
        tokens, _, dim = q.shape
        _operand("out_q", out_q, (q.dtype,), q.shape)
        _operand("positions", positions, (torch.int32, torch.int64), (tokens,))
        _require(self.freq.device == q.device, "q: not on the device of the frequencies")
        _require((k is None) == (out_k is None), "rotary: k and out_k go together")
        d = RotaryDesc(_DTYPES[q.dtype], dim, self.rot_dim, self.layout,
                       ANNC_I64 if positions.dtype == torch.int64 else ANNC_I32, int(transposed), tokens,
                       positions.data_ptr(), self.freq.data_ptr(), self.size)
        d.x[0] = (q.data_ptr(), out_q.data_ptr(), q.shape[1], q.stride(0), q.stride(1), out_q.stride(0), out_q.stride(1))
        if k is not None:
            _operand("k", k, (q.dtype,), (tokens, None, dim))
            _operand("out_k", out_k, (q.dtype,), k.shape)
            d.x[1] = (k.data_ptr(), out_k.data_ptr(), k.shape[1], k.stride(0), k.stride(1), out_k.stride(0),
                      out_k.stride(1))
        rc = lib.annc_rotary_dev(C.byref(d), raw_stream())
        if rc:
            check(rc)


class PrefixAttention:
    """Attention of up to max_tokens tokens that share one prefix (annc_prefix_attention_dev); holds the workspace.
    One run() at a time: runs on different streams that may overlap, captured graphs among them, need a plan each."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, max_tokens: int, *, dtype=torch.bfloat16, device=None):
        _require(dtype in (torch.bfloat16, torch.float16), f"prefix attention: bad type {dtype}")
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        self.max_tokens, self.dtype = int(max_tokens), dtype
        self.ws_bytes = int(lib.annc_prefix_attention_workspace_bytes(self.max_tokens, self.heads, self.head_dim))
        self.ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=device or "cuda")

    def run(self, q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, out: torch.Tensor, *,
            k_own: Optional[torch.Tensor] = None, v_own: Optional[torch.Tensor] = None,
            own_begin: Optional[torch.Tensor] = None, own_len: Optional[torch.Tensor] = None,
            q_begin: Optional[torch.Tensor] = None, scale: Optional[float] = None,
            lse: Optional[torch.Tensor] = None) -> None:
        """q, out [tokens, heads, head_dim]; k_prefix, v_prefix [prefix, kv_heads, head_dim]; k_own, v_own [rows,
        kv_heads, head_dim] with own_begin i64[sequences] and own_len i32[sequences]; q_begin i32[sequences + 1],
        without it a token is a sequence; scale head_dim ** -0.5 unless given; lse f32[tokens, heads]."""
        heads, kv, dim = self.heads, self.kv_heads, self.head_dim
        dt = (self.dtype,)
        _operand("q", q, dt, (None, heads, dim))
        tokens = q.shape[0]
        _require(tokens <= self.max_tokens, f"q: more than the plan's {self.max_tokens} tokens")
        _require(self.ws.device == q.device, "q: not on the plan's device")
        _operand("out", out, dt, q.shape)
        _operand("k_prefix", k_prefix, dt, (None, kv, dim))
        _operand("v_prefix", v_prefix, dt, k_prefix.shape)
        d = PrefixAttentionDesc(_DTYPES[self.dtype], heads, kv, dim, tokens, tokens, k_prefix.shape[0], 0,
                                dim ** -0.5 if scale is None else scale, 0,
                                q.data_ptr(), q.stride(0), q.stride(1),
                                k_prefix.data_ptr(), k_prefix.stride(0), k_prefix.stride(1),
                                v_prefix.data_ptr(), v_prefix.stride(0), v_prefix.stride(1))
        if q_begin is not None:
            _operand("q_begin", q_begin, (torch.int32,), (None,))
            _require(q_begin.shape[0] >= 1, "q_begin: has one entry more than there are sequences")
            d.sequences, d.q_begin = q_begin.shape[0] - 1, q_begin.data_ptr()
        given = [x is not None for x in (k_own, v_own, own_begin, own_len)]
        _require(all(given) or not any(given), "prefix attention: own keys need k_own, v_own, own_begin and own_len")
        if k_own is not None:
            _operand("k_own", k_own, dt, (None, kv, dim))
            _operand("v_own", v_own, dt, k_own.shape)
            _operand("own_begin", own_begin, (torch.int64,), (d.sequences,))
            _operand("own_len", own_len, (torch.int32,), (d.sequences,))
            d.own_rows = k_own.shape[0]
            d.k_own, d.k_own_row, d.k_own_head = k_own.data_ptr(), k_own.stride(0), k_own.stride(1)
            d.v_own, d.v_own_row, d.v_own_head = v_own.data_ptr(), v_own.stride(0), v_own.stride(1)
            d.own_begin, d.own_len = own_begin.data_ptr(), own_len.data_ptr()
        d.out, d.out_row, d.out_head = out.data_ptr(), out.stride(0), out.stride(1)
        if lse is not None:
            _operand("lse", lse, (torch.float32,), (tokens, heads))
            _require(lse.is_contiguous(), "lse: not contiguous")
            d.lse = lse.data_ptr()
        d.workspace, d.workspace_bytes = self.ws.data_ptr(), self.ws_bytes
        rc = lib.annc_prefix_attention_dev(C.byref(d), raw_stream())
        if rc:
            check(rc)
