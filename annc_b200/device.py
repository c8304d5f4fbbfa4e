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
                   BagTable, GemmDesc, PACK_GEMM_I8, PACK_PREFIX_ATTENTION, PACK_ROTARY, check, lib)


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

_F32_MAX = torch.finfo(torch.float32).max
_DTYPES = {torch.float32: ANNC_F32, torch.bfloat16: ANNC_BF16, torch.float16: ANNC_F16}


def _refuse(message: str) -> None:
    raise AnncError(ERR_INVALID_ARGUMENT, message)


def _current(name: str, t: torch.Tensor) -> int:
    """The current device, which is the tensor's."""
    dev = t.get_device()
    if dev < 0 or dev != torch._C._cuda_getDevice():
        _refuse(f"{name}: not on the current CUDA device")
    return dev


# The checks of an operand (some 0.7 us each: they are a good part of what a small call costs).  All operands are on
# the current device `dev`.

def _dense(name: str, t: torch.Tensor, dev: int, dtypes, dims: int):
    """(shape, strides) of a tensor of so many dimensions, the values of the last one adjacent."""
    if t.get_device() != dev:
        _refuse(f"{name}: not on the current CUDA device")
    if t.dtype not in dtypes:
        _refuse(f"{name}: bad type {t.dtype}")
    shape, strides = t.shape, t.stride()
    if len(shape) != dims:
        _refuse(f"{name}: bad shape {tuple(shape)}")
    if strides[-1] != 1 and shape[-1] > 1:
        _refuse(f"{name}: the values of the last dimension are not adjacent")
    return shape, strides


def _vector(name: str, t: torch.Tensor, dev: int, dtype, length: int) -> int:
    """Address of a vector of that length."""
    if t.get_device() != dev or t.dtype is not dtype or t.shape != (length,) or not t.is_contiguous():
        _refuse(f"{name}: has to be a vector of {length} {dtype} on the current CUDA device")
    return t.data_ptr()


def _alike(name: str, shape, want) -> None:
    if shape != want:
        _refuse(f"{name}: bad shape {tuple(shape)}, wanted {tuple(want)}")


def _pitch(shape, strides) -> int:
    """Elements from row to row; a single row has any."""
    return strides[0] if shape[0] > 1 else max(strides[0], shape[1])


_I8, _FLOATS = (torch.int8,), tuple(_DTYPES)


def i8_rows(rows: int, cols: int, device=None) -> torch.Tensor:
    """i8[rows, cols] whose rows start on 16 bytes, as the tensor-core product wants its operands."""
    return torch.empty((rows, max(cols + 15, 16) // 16 * 16), dtype=torch.int8, device=device or "cuda")[:, :cols]


def quantize_rows(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """annc_quantize_rows_dev: x f32 / bf16 / f16 [rows, cols] -> q i8[rows, cols] (i8_rows), scale f32[rows]."""
    dev = _current("x", x)
    shape, strides = _dense("x", x, dev, _FLOATS, 2)
    q_shape, q_strides = _dense("q", q, dev, _I8, 2)
    _alike("q", q_shape, shape)
    rc = lib.annc_quantize_rows_dev(x.data_ptr(), _DTYPES[x.dtype], shape[0], shape[1], _pitch(shape, strides), q.data_ptr(),
                                    _pitch(q_shape, q_strides), _vector("scale", scale, dev, torch.float32, shape[0]),
                                    torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc)


def i8_weight(b_kn: torch.Tensor):
    """f32 [K,N] -> (i8 [N,K] with rows on 16 bytes, f32 scale [N]) for gemm_i8 (annc_i8_weight_dev)."""
    shape, strides = _dense("b_kn", b_kn, _current("b_kn", b_kn), (torch.float32,), 2)
    k, n = shape
    q = i8_rows(n, k, b_kn.device)
    scale = torch.empty(n, dtype=torch.float32, device=b_kn.device)
    check(lib.annc_i8_weight_dev(b_kn.data_ptr(), _pitch(shape, strides), q.data_ptr(), q.stride(0), scale.data_ptr(), k, n,
                                 raw_stream()))
    return q, scale


def _gemm_i8_desc(dev, a, scale_a, b, scale_b, c, bias, activation) -> bytes:
    a_shape, a_strides = _dense("a", a, dev, _I8, 2)
    b_shape, b_strides = _dense("b", b, dev, _I8, 2)
    c_shape, c_strides = _dense("c", c, dev, _FLOATS, 2)
    m, k = a_shape
    n = b_shape[0]
    if b_shape[1] != k or c_shape != (m, n):
        _refuse(f"gemm_i8: a {tuple(a_shape)}, b {tuple(b_shape)} and c {tuple(c_shape)} do not belong together")
    return PACK_GEMM_I8.pack(m, n, k, _pitch(a_shape, a_strides), _pitch(b_shape, b_strides), _pitch(c_shape, c_strides),
                             a.data_ptr(), b.data_ptr(), _vector("scale_a", scale_a, dev, torch.float32, m),
                             _vector("scale_b", scale_b, dev, torch.float32, n),
                             0 if bias is None else _vector("bias", bias, dev, torch.float32, n), c.data_ptr(),
                             _DTYPES[c.dtype], activation)


def gemm_i8(a: torch.Tensor, scale_a: torch.Tensor, b: torch.Tensor, scale_b: torch.Tensor, c: torch.Tensor, *,
            bias: Optional[torch.Tensor] = None, activation: int = ACT_NONE) -> None:
    """annc_gemm_i8_run on the current stream: c = act(a b^T * scale_a[:, None] * scale_b + bias); a i8[m,k], b
    i8[n,k], c f32 / bf16 / f16 [m,n]."""
    dev = _current("a", a)
    rc = lib.annc_gemm_i8_run(_gemm_i8_desc(dev, a, scale_a, b, scale_b, c, bias, activation),
                              torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc)


def gemm_i8_kernel_name(a, scale_a, b, scale_b, c, bias=None, activation: int = ACT_NONE) -> str:
    """Name of the kernel family that gemm_i8 takes for these operands."""
    return lib.annc_gemm_i8_kernel_name(_gemm_i8_desc(_current("a", a), a, scale_a, b, scale_b, c, bias, activation)).decode()


class _Plan:
    """Device memory that a plan keeps: made on one stream, used on any."""

    def _keep(self, memory: torch.Tensor) -> torch.Tensor:
        stream = torch.cuda.current_stream(memory.device)
        self._memory, self._streams = memory, {stream.cuda_stream}
        self._made = None if torch.cuda.is_current_stream_capturing() else stream.record_event()
        return memory

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_streams", "_made")}

    def __setstate__(self, state) -> None:  # (a copy of a plan, made on the stream that is current now)
        self.__dict__.update(state)
        self._keep(self._memory)

    def _stream(self, dev: int) -> int:
        """The current stream of the device, which may use the memory from now on: behind what had it before the
        plan, and the allocator hands it out again only behind what is queued there when the plan is dropped."""
        raw = torch._C._cuda_getCurrentRawStream(dev)
        if raw not in self._streams:
            stream = torch.cuda.current_stream(dev)
            self._memory.record_stream(stream)
            if not torch.cuda.is_current_stream_capturing():  # (a capture cannot wait for what is outside it)
                if self._made is not None:
                    stream.wait_event(self._made)
                self._streams.add(raw)
        return raw


class Rotary(_Plan):
    """Rotary positions (annc_rotary_dev): holds the frequencies of annc_rotary_frequencies on the device.
    layout "half" or "interleaved"; scaling "none", "linear", "ntk" or "yarn" by `factor`.  Runs on any stream; a
    captured graph needs the plan as long as it is replayed."""

    def __init__(self, rot_dim: int, *, base: float = 10000.0, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original_len: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device=None):
        layouts = {"half": ROTARY_HALF, "interleaved": ROTARY_INTERLEAVED}
        scalings = {"none": ROTARY_UNSCALED, "linear": ROTARY_LINEAR, "ntk": ROTARY_NTK, "yarn": ROTARY_YARN}
        if layout not in layouts or scaling not in scalings:
            _refuse(f"rotary: unknown layout {layout!r} or scaling {scaling!r}")
        self.rot_dim, self.layout = int(rot_dim), layouts[layout]
        host = (C.c_double * max(self.rot_dim // 2, 1))()
        size = C.c_float(0)
        check(lib.annc_rotary_frequencies(self.rot_dim, base, scalings[scaling], factor, original_len, beta_fast,
                                          beta_slow, host, C.byref(size)))
        self.size = size.value
        self.freq = self._keep(torch.tensor(list(host), dtype=torch.float64, device=device or "cuda"))

    def run(self, positions: torch.Tensor, q: torch.Tensor, out_q: torch.Tensor, k: Optional[torch.Tensor] = None,
            out_k: Optional[torch.Tensor] = None, *, transposed: bool = False) -> None:
        """q [tokens, heads, head_dim] -> out_q (q itself: in place), and k likewise in the same launch; positions
        i32 / i64 [tokens]."""
        dev = _current("q", q)
        dtypes = (q.dtype,)
        shape, s = _dense("q", q, dev, _FLOATS, 3)
        out_shape, so = _dense("out_q", out_q, dev, dtypes, 3)
        _alike("out_q", out_shape, shape)
        tokens, heads, dim = shape
        if self.freq.get_device() != dev:
            _refuse("q: not on the device of the frequencies")
        if positions.dtype is torch.int64:
            pos, pos_type = _vector("positions", positions, dev, torch.int64, tokens), ANNC_I64
        else:
            pos, pos_type = _vector("positions", positions, dev, torch.int32, tokens), ANNC_I32
        second = (0, 0, 0, 0, 0, 0, 0)
        if k is not None:
            if out_k is None:
                _refuse("rotary: k and out_k go together")
            k_shape, sk = _dense("k", k, dev, dtypes, 3)
            out_shape, sko = _dense("out_k", out_k, dev, dtypes, 3)
            _alike("k", k_shape, (tokens, k_shape[1], dim))
            _alike("out_k", out_shape, k_shape)
            second = (k.data_ptr(), out_k.data_ptr(), k_shape[1], sk[0], sk[1], sko[0], sko[1])
        elif out_k is not None:
            _refuse("rotary: k and out_k go together")
        rc = lib.annc_rotary_dev(
            PACK_ROTARY.pack(_DTYPES[q.dtype], dim, self.rot_dim, self.layout, pos_type, 1 if transposed else 0, tokens, pos,
                             self.freq.data_ptr(), self.size, 0, q.data_ptr(), out_q.data_ptr(), heads, s[0], s[1], so[0],
                             so[1], *second),
            self._stream(dev))
        if rc:
            check(rc)


class PrefixAttention(_Plan):
    """Attention of up to max_tokens tokens that share one prefix (annc_prefix_attention_dev); holds the workspace.
    One run() at a time: runs on different streams that may overlap, captured graphs among them, need a plan each, and
    a captured graph needs it as long as it is replayed."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, max_tokens: int, *, dtype=torch.bfloat16, device=None):
        if dtype not in (torch.bfloat16, torch.float16):
            _refuse(f"prefix attention: bad type {dtype}")
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        self.max_tokens, self.dtype = int(max_tokens), dtype
        self.ws_bytes = int(lib.annc_prefix_attention_workspace_bytes(self.max_tokens, self.heads, self.kv_heads,
                                                                      self.head_dim))
        self.ws = self._keep(torch.empty(max(self.ws_bytes, 16), dtype=torch.uint8, device=device or "cuda"))

    def run(self, q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, out: torch.Tensor, *,
            k_own: Optional[torch.Tensor] = None, v_own: Optional[torch.Tensor] = None,
            own_begin: Optional[torch.Tensor] = None, own_len: Optional[torch.Tensor] = None,
            q_begin: Optional[torch.Tensor] = None, scale: Optional[float] = None,
            lse: Optional[torch.Tensor] = None) -> None:
        """q, out [tokens, heads, head_dim]; k_prefix, v_prefix [prefix, kv_heads, head_dim]; k_own, v_own [rows,
        kv_heads, head_dim] with own_begin i64[sequences] and own_len i32[sequences]; q_begin i32[sequences + 1],
        without it a token is a sequence; scale head_dim ** -0.5 unless given; lse f32[tokens, heads]."""
        heads, kv, dim, dtypes = self.heads, self.kv_heads, self.head_dim, (self.dtype,)
        scale = dim ** -0.5 if scale is None else scale
        if not -_F32_MAX <= scale <= _F32_MAX:
            _refuse(f"scale: {scale} is not a finite f32")
        dev = _current("q", q)
        shape, sq = _dense("q", q, dev, dtypes, 3)
        tokens = shape[0]
        _alike("q", shape, (tokens, heads, dim))
        if tokens > self.max_tokens:
            _refuse(f"q: more than the plan's {self.max_tokens} tokens")
        if self.ws.get_device() != dev:
            _refuse("q: not on the plan's device")
        out_shape, so = _dense("out", out, dev, dtypes, 3)
        _alike("out", out_shape, shape)
        k_shape, sk = _dense("k_prefix", k_prefix, dev, dtypes, 3)
        v_shape, sv = _dense("v_prefix", v_prefix, dev, dtypes, 3)
        prefix = k_shape[0]
        _alike("k_prefix", k_shape, (prefix, kv, dim))
        _alike("v_prefix", v_shape, k_shape)
        sequences, q_ptr = tokens, 0
        if q_begin is not None:
            sequences = q_begin.shape[0] - 1 if q_begin.dim() == 1 else -1
            if sequences < 0:
                _refuse("q_begin: a vector with one entry more than there are sequences")
            q_ptr = _vector("q_begin", q_begin, dev, torch.int32, sequences + 1)
        rows, own, lists = 0, (0, 0, 0, 0, 0, 0), (0, 0)
        if k_own is not None:
            if v_own is None or own_begin is None or own_len is None:
                _refuse("prefix attention: own keys need k_own, v_own, own_begin and own_len")
            k_shape, sko = _dense("k_own", k_own, dev, dtypes, 3)
            v_shape, svo = _dense("v_own", v_own, dev, dtypes, 3)
            rows = k_shape[0]
            _alike("k_own", k_shape, (rows, kv, dim))
            _alike("v_own", v_shape, k_shape)
            own = (k_own.data_ptr(), sko[0], sko[1], v_own.data_ptr(), svo[0], svo[1])
            lists = (_vector("own_begin", own_begin, dev, torch.int64, sequences),
                     _vector("own_len", own_len, dev, torch.int32, sequences))
        elif v_own is not None or own_begin is not None or own_len is not None:
            _refuse("prefix attention: own keys need k_own, v_own, own_begin and own_len")
        lse_ptr = 0
        if lse is not None:
            _alike("lse", _dense("lse", lse, dev, (torch.float32,), 2)[0], (tokens, heads))
            if not lse.is_contiguous():
                _refuse("lse: not contiguous")
            lse_ptr = lse.data_ptr()
        rc = lib.annc_prefix_attention_dev(
            PACK_PREFIX_ATTENTION.pack(_DTYPES[self.dtype], heads, kv, dim, tokens, sequences, prefix, rows,
                                       scale, 0, q.data_ptr(), sq[0], sq[1],
                                       k_prefix.data_ptr(), sk[0], sk[1], v_prefix.data_ptr(), sv[0], sv[1], *own, *lists,
                                       q_ptr, out.data_ptr(), so[0], so[1], lse_ptr, self.ws.data_ptr(), self.ws_bytes),
            self._stream(dev))
        if rc:
            check(rc)
