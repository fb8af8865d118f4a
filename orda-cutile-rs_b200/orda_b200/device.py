"""Device entry points of the C ABI for torch tensors (torch is used only for
device memory and streams; every computation runs in liborda_b200.so).
"""
from __future__ import annotations

import ctypes as C
import threading
from dataclasses import dataclass
from typing import Optional

import torch

from . import ChunkPlan, LossOptions, Reduction, TeacherMode, _abi, _check
from ._abi import load_library


def _lib():
    return load_library()


class DeviceContext:
    """Owns an `OrdaContext` (device workspace + status word)."""

    def __init__(self, device: int = 0):
        self.device = device
        h = C.c_void_p()
        buf = _abi.err_buf()
        _check(_lib().orda_context_create(device, C.byref(h), buf, len(buf)), buf)
        self.handle = h

    def close(self) -> None:
        if self.handle:
            _lib().orda_context_destroy(self.handle)
            self.handle = C.c_void_p()

    def check(self) -> None:
        buf = _abi.err_buf()
        _check(_lib().orda_context_check(self.handle, buf, len(buf)), buf)

    def workspace_bytes(self) -> int:
        return int(_lib().orda_context_workspace_bytes(self.handle))

    def inject_alloc_failures(self, count: int) -> None:
        _lib().orda_context_inject_alloc_failures(self.handle, count)

    def enable_timing(self, on: bool = True) -> None:
        _lib().orda_context_enable_timing(self.handle, int(on))

    def reset_timing(self) -> None:
        _lib().orda_context_reset_timing(self.handle)

    def phase_times(self) -> dict:
        """Milliseconds and kernel launches per phase since the last reset
        (events recorded on the launch stream; synchronizes)."""
        ms = (C.c_double * _abi.NUM_PHASES)()
        n = (C.c_uint64 * _abi.NUM_PHASES)()
        _lib().orda_context_phase_times(self.handle, ms, n)
        return {name: (float(ms[i]), int(n[i])) for i, name in enumerate(_abi.PHASE_NAMES)}

    def set_concurrency(self, spare_sms: int) -> None:
        """`orda_context_set_concurrency`: SMs the persistent GEMMs leave to the
        teacher statistics and the INT8 quantiser running beside them on an
        auxiliary stream (0, the default = every kernel serial on the caller's
        stream)."""
        _lib().orda_context_set_concurrency(self.handle, int(spare_sms))

    def launch_count(self) -> int:
        return int(_lib().orda_context_launch_count(self.handle))

    def slots_create(self, world: int, rank: int, total_rows: int, h: int, copies: int = 1) -> bytes:
        """`orda_context_slots_create`: allocates this rank's slot buffer for
        `total_rows` rows split over the owners (shard.owner_rows; `copies`
        sets of [world][slice][h] fp32) for the fused reduce-scatters;
        returns its 64-byte IPC handle."""
        hd = _abi.OrdaIpcHandle()
        buf = _abi.err_buf()
        _check(_lib().orda_context_slots_create(self.handle, world, rank, total_rows, h, copies, C.byref(hd), buf,
                                                len(buf)), buf)
        return C.string_at(C.addressof(hd), C.sizeof(hd))

    def slots_attach(self, handles: list) -> None:
        """`orda_context_slots_attach` with every rank's handle, by rank."""
        arr = (_abi.OrdaIpcHandle * len(handles))()
        for i, b in enumerate(handles):
            b = bytes(b)
            if len(b) != C.sizeof(_abi.OrdaIpcHandle):
                raise ValueError(f"IPC handle {i} has {len(b)} bytes")
            C.memmove(C.addressof(arr[i]), b, len(b))
        buf = _abi.err_buf()
        _check(_lib().orda_context_slots_attach(self.handle, arr, buf, len(buf)), buf)

    def reduce_slots(self, grad_w_slice: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                     quantize: bool = False, stochastic: bool = False, seed: int = 0,
                     q: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, stream=None,
                     int8_wire: bool = False) -> None:
        """`orda_reduce_slots_device`: this rank's grad_W rows, summed over
        the ranks' partials (and INT8 round trip when quantize); int8_wire
        when the partials were sent in the INT8 wire format."""
        buf = _abi.err_buf()
        _check(_lib().orda_reduce_slots_device(
            self.handle, grad_w_slice.data_ptr(), grad_w_slice.stride(0), labels.data_ptr(), labels.numel(),
            ignore_index, int(quantize), int(stochastic), seed, _ptr(q), _ptr(scale), int(int8_wire),
            _stream(stream), buf, len(buf)), buf)

    def reduce_slot_set(self, copy: int, out: torch.Tensor, stream=None) -> None:
        """`orda_reduce_slot_set_device`: rank-ordered sum of slot set `copy`."""
        buf = _abi.err_buf()
        _check(_lib().orda_reduce_slot_set_device(self.handle, copy, out.data_ptr(), out.stride(0), _stream(stream),
                                                  buf, len(buf)), buf)

    def set_l2_persisting(self, nbytes: int) -> int:
        """`orda_context_set_l2_persisting`: persisting-L2 carve-out for the
        evict-last GEMM operands; returns the bytes granted."""
        got = C.c_size_t()
        buf = _abi.err_buf()
        _check(_lib().orda_context_set_l2_persisting(self.handle, nbytes, C.byref(got), buf, len(buf)), buf)
        return int(got.value)

    def selftest_bounded_wait(self, limit_us: int = 50000, stream=None) -> None:
        """Runs the bounded-wait self-test kernel (a wait that expires)."""
        buf = _abi.err_buf()
        _check(_lib().orda_context_selftest_bounded_wait(self.handle, limit_us, _stream(stream), buf, len(buf)), buf)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


def dev_mat(t: Optional[torch.Tensor]) -> _abi.OrdaDeviceMat:
    m = _abi.OrdaDeviceMat()
    if t is None:
        return m
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError("device matrices must be 2-D with unit column stride")
    if t.dtype == torch.bfloat16:
        m.dtype = _abi.DTYPE_BF16
    elif t.dtype == torch.float32:
        m.dtype = _abi.DTYPE_F32
    else:
        raise ValueError(f"unsupported dtype {t.dtype}")
    m.data = t.data_ptr()
    m.rows, m.cols = t.shape
    m.ld = t.stride(0)
    return m


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


@dataclass
class DeviceLossResult:
    scalars: torch.Tensor  # device float[4]: loss, student_ce, teacher_ce, kl
    grad_student_hidden: Optional[torch.Tensor]
    grad_weight: Optional[torch.Tensor]
    grad_teacher_hidden: Optional[torch.Tensor]
    grad_teacher_weight: Optional[torch.Tensor]
    grad_weight_q: Optional[torch.Tensor]
    grad_weight_scale: Optional[torch.Tensor]
    chunk_plan: ChunkPlan


def _teacher_struct(teacher_mode, teacher_hidden, teacher_weight, teacher_logits):
    t = _abi.OrdaDeviceTeacher()
    t.mode = int(teacher_mode)
    t.hidden = dev_mat(teacher_hidden)
    t.weight = dev_mat(teacher_weight)
    t.logits = dev_mat(teacher_logits)
    return t


def _outputs(opts, teacher_mode, bt, h, v, ht, dev, out, want_int8, with_grad_weight=True, with_grad_hidden=True):
    """Output tensors (from `out` or newly allocated) and their C struct."""
    w_t = opts.teacher_ce_weight
    if w_t is None:
        w_t = 1.0 if teacher_mode == TeacherMode.Tied else 0.0
    live = teacher_mode in (TeacherMode.Tied, TeacherMode.Separate)
    out = dict(out or {})
    f32 = dict(device=dev, dtype=torch.float32)
    gsh = out.get("grad_student_hidden") if with_grad_hidden else None
    if gsh is None and with_grad_hidden:
        gsh = torch.empty(bt, h, **f32)
    gw = out.get("grad_weight") if with_grad_weight else None
    if gw is None and with_grad_weight:
        gw = torch.empty(v, h, **f32)
    gth = out.get("grad_teacher_hidden") if with_grad_hidden else None
    if gth is None and w_t > 0 and live and with_grad_hidden:
        gth = torch.empty(bt, ht, **f32)
    gtw = out.get("grad_teacher_weight")
    if gtw is None and w_t > 0 and teacher_mode == TeacherMode.Separate:
        gtw = torch.empty(v, ht, **f32)
    q = out.get("grad_weight_q")
    sc = out.get("grad_weight_scale")
    if want_int8 and opts.config.quantize_grad_weight:
        if q is None:
            q = torch.empty(v, h, device=dev, dtype=torch.int8)
        if sc is None:
            sc = torch.empty(v, **f32)
    scal = out.get("scalars")
    if scal is None:
        scal = torch.empty(4, **f32)
    o = _abi.OrdaDeviceOutputs()
    if gsh is not None:
        o.grad_student_hidden = gsh.data_ptr()
        o.ld_grad_student_hidden = gsh.stride(0)
    if gw is not None:
        o.grad_weight = gw.data_ptr()
        o.ld_grad_weight = gw.stride(0)
    if gth is not None:
        o.grad_teacher_hidden = gth.data_ptr()
        o.ld_grad_teacher_hidden = gth.stride(0)
    if gtw is not None:
        o.grad_teacher_weight = gtw.data_ptr()
        o.ld_grad_teacher_weight = gtw.stride(0)
    o.grad_weight_q = _ptr(q)
    o.grad_weight_scale = _ptr(sc)
    o.scalars = scal.data_ptr()
    tensors = dict(scalars=scal, grad_student_hidden=gsh, grad_weight=gw, grad_teacher_hidden=gth,
                   grad_teacher_weight=gtw, grad_weight_q=q, grad_weight_scale=sc)
    return o, tensors


def distillation_loss_device(
    ctx: DeviceContext,
    student_hidden: torch.Tensor,
    weight: torch.Tensor,
    labels: torch.Tensor,
    teacher_mode: TeacherMode,
    teacher_hidden: Optional[torch.Tensor] = None,
    teacher_weight: Optional[torch.Tensor] = None,
    teacher_logits: Optional[torch.Tensor] = None,
    opts: Optional[LossOptions] = None,
    out: Optional[dict] = None,
    global_non_ignore: int = 0,
    skip_quantize: bool = False,
    want_int8: bool = False,
    stream=None,
    scatter_grad_weight: bool = False,
    int8_wire: bool = False,
) -> DeviceLossResult:
    """`orda_distillation_loss_device`: bf16 device inputs, fp32 device grads.
    With scatter_grad_weight the grad_W partial goes to the slot buffers
    (see DeviceContext.slots_create) and the returned grad_weight is None;
    int8_wire sends it there as row-wise INT8 codes and scales."""
    opts = opts or LossOptions()
    bt, h = student_hidden.shape
    v = weight.shape[0]
    ht = teacher_hidden.shape[1] if teacher_mode == TeacherMode.Separate else h
    o, tensors = _outputs(opts, teacher_mode, bt, h, v, ht, student_hidden.device, out, want_int8,
                          with_grad_weight=not scatter_grad_weight)
    t = _teacher_struct(teacher_mode, teacher_hidden, teacher_weight, teacher_logits)
    shard = _abi.OrdaShardOptions(int(global_non_ignore), int(skip_quantize), int(scatter_grad_weight),
                                  int(int8_wire), 0)
    plan = _abi.OrdaChunkPlan()
    buf = _abi.err_buf()
    rc = _lib().orda_distillation_loss_device(
        ctx.handle,
        C.byref(dev_mat(student_hidden)),
        C.byref(dev_mat(weight)),
        labels.data_ptr(),
        labels.numel(),
        C.byref(t),
        C.byref(opts._c()),
        C.byref(o),
        C.byref(shard),
        _stream(stream),
        C.byref(plan),
        buf,
        len(buf),
    )
    _check(rc, buf)
    return DeviceLossResult(chunk_plan=ChunkPlan(int(plan.chunk_size), int(plan.num_chunks)), **tensors)


def vocab_forward_device(
    ctx: DeviceContext,
    student_hidden: torch.Tensor,
    weight_slice: torch.Tensor,
    labels: torch.Tensor,
    teacher_mode: TeacherMode,
    v_total: int,
    v0: int,
    teacher_hidden: Optional[torch.Tensor] = None,
    teacher_weight_slice: Optional[torch.Tensor] = None,
    teacher_logits_slice: Optional[torch.Tensor] = None,
    opts: Optional[LossOptions] = None,
    partials: Optional[torch.Tensor] = None,
    stream=None,
) -> torch.Tensor:
    """`orda_vocab_forward_device`: logits of this rank's vocabulary rows
    [v0, v0 + len(weight_slice)); returns the per-row partial statistics
    [bt, VOCAB_TUPLE] to all-gather."""
    opts = opts or LossOptions()
    bt = student_hidden.shape[0]
    if partials is None:
        partials = torch.empty(bt, _abi.VOCAB_TUPLE, device=student_hidden.device, dtype=torch.float32)
    t = _teacher_struct(teacher_mode, teacher_hidden, teacher_weight_slice, teacher_logits_slice)
    vs = _abi.OrdaVocabShard(int(v_total), int(v0), 1, 0, 0, 0)
    buf = _abi.err_buf()
    rc = _lib().orda_vocab_forward_device(
        ctx.handle, C.byref(dev_mat(student_hidden)), C.byref(dev_mat(weight_slice)), labels.data_ptr(),
        labels.numel(), C.byref(t), C.byref(opts._c()), C.byref(vs), partials.data_ptr(), _stream(stream), buf,
        len(buf))
    _check(rc, buf)
    return partials


def vocab_backward_device(
    ctx: DeviceContext,
    student_hidden: torch.Tensor,
    weight_slice: torch.Tensor,
    labels: torch.Tensor,
    teacher_mode: TeacherMode,
    v_total: int,
    v0: int,
    all_partials: torch.Tensor,
    include_rows: bool,
    teacher_hidden: Optional[torch.Tensor] = None,
    teacher_weight_slice: Optional[torch.Tensor] = None,
    teacher_logits_slice: Optional[torch.Tensor] = None,
    opts: Optional[LossOptions] = None,
    out: Optional[dict] = None,
    want_int8: bool = False,
    stream=None,
    scatter_grad_hidden: bool = False,
) -> DeviceLossResult:
    """`orda_vocab_backward_device`: all_partials [world, bt, VOCAB_TUPLE]
    are every rank's tuples by rank. grad_weight (and grad_teacher_weight)
    hold this slice's rows; grad_student_hidden, grad_teacher_hidden and
    scalars are this rank's partial sums (add them over the ranks)."""
    opts = opts or LossOptions()
    bt, h = student_hidden.shape
    v = weight_slice.shape[0]
    ht = teacher_hidden.shape[1] if teacher_mode == TeacherMode.Separate else h
    o, tensors = _outputs(opts, teacher_mode, bt, h, v, ht, student_hidden.device, out, want_int8,
                          with_grad_hidden=not scatter_grad_hidden)
    t = _teacher_struct(teacher_mode, teacher_hidden, teacher_weight_slice, teacher_logits_slice)
    vs = _abi.OrdaVocabShard(int(v_total), int(v0), int(all_partials.shape[0]), int(include_rows),
                             int(scatter_grad_hidden), 0)
    plan = _abi.OrdaChunkPlan()
    buf = _abi.err_buf()
    rc = _lib().orda_vocab_backward_device(
        ctx.handle, C.byref(dev_mat(student_hidden)), C.byref(dev_mat(weight_slice)), labels.data_ptr(),
        labels.numel(), C.byref(t), C.byref(opts._c()), C.byref(vs), all_partials.data_ptr(), C.byref(o),
        _stream(stream), C.byref(plan), buf, len(buf))
    _check(rc, buf)
    return DeviceLossResult(chunk_plan=ChunkPlan(int(plan.chunk_size), int(plan.num_chunks)), **tensors)


def _on_context(ctx: DeviceContext, **tensors: Optional[torch.Tensor]) -> None:
    """Every tensor lies on the context's GPU."""
    for name, t in tensors.items():
        if t is not None and t.get_device() != ctx.device:
            raise ValueError(f"{name} must be on cuda:{ctx.device}, the context's device, got {t.device}")


def _context_stream(ctx: DeviceContext, stream) -> int:
    """The given stream, else the current one of the context's device (the raw
    handle: a Stream object costs as much as a small kernel's launch)."""
    return torch._C._cuda_getCurrentRawStream(ctx.device) if stream is None else _stream(stream)


_DTYPE_CODES = {torch.bfloat16: _abi.DTYPE_BF16, torch.float32: _abi.DTYPE_F32}
_thread = threading.local()


def _err():
    """This thread's error buffer."""
    buf = getattr(_thread, "err", None)
    if buf is None:
        buf = _thread.err = _abi.err_buf()
    return buf


def _grad_dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPE_CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: unsupported dtype {t.dtype}")
    return code


def _row_major(rows: int, cols: int, dtype: torch.dtype, device) -> torch.Tensor:
    """[rows, cols] whose rows start on 16 bytes (what TMA stores address)."""
    step = 16 // dtype.itemsize
    if cols % step == 0:
        return torch.empty(rows, cols, device=device, dtype=dtype)
    return torch.empty(rows, -(-cols // step) * step, device=device, dtype=dtype)[:, :cols]


@dataclass
class LinearCrossEntropyResult:
    loss: torch.Tensor  # device float, 0-dim
    nll: torch.Tensor  # float [bt], 0 for ignored tokens
    lse: torch.Tensor  # float [bt], 0 for ignored tokens
    grad_hidden: Optional[torch.Tensor]
    grad_weight: Optional[torch.Tensor]


def linear_cross_entropy_device(
    ctx: DeviceContext,
    hidden: torch.Tensor,
    weight: torch.Tensor,
    labels: torch.Tensor,
    ignore_index: int = -100,
    label_smoothing: float = 0.0,
    reduction: Reduction = Reduction.Mean,
    need_grad_hidden: bool = True,
    need_grad_weight: bool = True,
    grad_dtype: torch.dtype = torch.float32,
    out: Optional[dict] = None,
    global_non_ignore: int = 0,
    piece_bytes: int = 0,
    stream=None,
) -> LinearCrossEntropyResult:
    """`orda_linear_cross_entropy_device`: softmax cross entropy of
    hidden [bt, H] @ weight [V, H]^T (bf16) against labels [bt] (int64), with
    the gradients of hidden and weight and without a teacher.

    need_grad_hidden / need_grad_weight select the gradients (neither: the
    losses alone, for scoring). grad_dtype (bf16 or f32) is the type of the
    gradients that are allocated here; `out` may hold loss (float [1]), nll,
    lse, grad_hidden and grad_weight to write into (their own types decide).
    piece_bytes bounds the 16-bit logits kept at once (0: 4 GiB); columns of
    the vocabulary beyond it are computed twice. nll and lse are those of
    each token, for log-probabilities (-nll without smoothing).
    Labels out of range are reported by ctx.check()."""
    if hidden.dim() != 2 or weight.dim() != 2 or labels.dim() != 1:
        raise ValueError("hidden and weight must be 2-D and labels 1-D")
    if labels.dtype != torch.int64 or not labels.is_contiguous():
        raise ValueError("labels must be contiguous int64")
    if out is not None:
        unknown = set(out) - {"loss", "nll", "lse", "grad_hidden", "grad_weight"}
        if unknown:
            raise ValueError(f"unknown outputs {sorted(unknown)}")
    dev = ctx.device
    if hidden.get_device() != dev or weight.get_device() != dev or labels.get_device() != dev:
        _on_context(ctx, hidden=hidden, weight=weight, labels=labels)
    h_mat, w_mat = _mat(_abi.OrdaDeviceMat, hidden, "hidden"), _mat(_abi.OrdaDeviceMat, weight, "weight")
    bt, h, v = h_mat.rows, h_mat.cols, w_mat.rows
    if out is None:
        # one allocation for the three
        store = torch.empty(2 * bt + 1, device=hidden.device, dtype=torch.float32)
        nll, lse, loss = store.split((bt, bt, 1))
        at = store.data_ptr()
        o = _abi.OrdaLinearCeOutputs(at + 8 * bt, at, at + 4 * bt)
    else:
        for name, need in (("grad_hidden", need_grad_hidden), ("grad_weight", need_grad_weight)):
            if not need and out.get(name) is not None:
                raise ValueError(f"out holds {name}, which need_{name}=False leaves out")
        _on_context(ctx, **out)
        given = []
        for name, n in (("loss", 1), ("nll", bt), ("lse", bt)):
            t = out.get(name)
            if t is None:
                t = torch.empty(n, device=hidden.device, dtype=torch.float32)
            elif t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous float32 of {n} element(s)")
            given.append(t)
        loss, nll, lse = given
        o = _abi.OrdaLinearCeOutputs(loss.data_ptr(), nll.data_ptr(), lse.data_ptr())

    def gradient(name, rows):
        t = None if out is None else out.get(name)
        if t is None:
            t = _row_major(rows, h, grad_dtype, hidden.device)
        elif tuple(t.shape) != (rows, h) or (h > 1 and t.stride(1) != 1):
            raise ValueError(f"{name} must be ({rows}, {h}) with unit column stride")
        # a row stride means nothing for a single row
        return t, t.data_ptr(), t.stride(0) if rows > 1 else max(t.stride(0), h), _grad_dtype(t, name)

    gh = gw = None
    if need_grad_hidden:
        gh, o.grad_hidden, o.ld_grad_hidden, o.grad_hidden_dtype = gradient("grad_hidden", bt)
    if need_grad_weight:
        gw, o.grad_weight, o.ld_grad_weight, o.grad_weight_dtype = gradient("grad_weight", v)
    opts = _abi.OrdaLinearCeOptions(ignore_index, label_smoothing, reduction, global_non_ignore, piece_bytes)
    buf = _err()
    rc = _lib().orda_linear_cross_entropy_device(ctx.handle, C.byref(h_mat), C.byref(w_mat), labels.data_ptr(),
                                                 labels.numel(), C.byref(opts), C.byref(o),
                                                 _context_stream(ctx, stream), buf, len(buf))
    if rc:
        _check(rc, buf)
    return LinearCrossEntropyResult(loss.view(()), nll, lse, gh, gw)


def _ids(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype != torch.int64 or not ids.is_contiguous():
        raise ValueError("ids must be contiguous int64")
    return ids


def _rows_of(t: torch.Tensor, n: int, h: int, name: str) -> torch.Tensor:
    """t [..., h] as [n, h] without a copy."""
    if t.dim() < 1 or t.shape[-1] != h or t.numel() != n * h:
        raise ValueError(f"{name} must have {n} rows of {h}, got {tuple(t.shape)}")
    try:
        return t.view(n, h)
    except RuntimeError:
        raise ValueError(f"{name} must be viewable as ({n}, {h}) without a copy") from None


def _mat(cls, t: torch.Tensor, name: str):
    """The C struct of a 2-D tensor with unit column stride."""
    rows, cols = t.shape
    ld, step = t.stride()
    if cols > 1 and step != 1:
        raise ValueError(f"{name} must have unit column stride")
    if rows <= 1 and ld < cols:  # a row stride means nothing for a single row
        ld = cols
    return cls(t.data_ptr(), rows, cols, ld, _grad_dtype(t, name))


def embedding_device(
    ctx: DeviceContext,
    table: torch.Tensor,
    ids: torch.Tensor,
    scale: float = 1.0,
    dtype: Optional[torch.dtype] = None,
    out: Optional[torch.Tensor] = None,
    stream=None,
) -> torch.Tensor:
    """`orda_embedding_device`: scale * table[ids] for table [V, H] (bf16 or
    f32) and ids of any shape (int64); the result has ids' shape and H, in
    `dtype` (default the table's) or written to `out`. Ids out of range give
    zeros and are reported by ctx.check()."""
    if table.dim() != 2:
        raise ValueError("table must be 2-D")
    _ids(ids)
    src = _mat(_abi.OrdaDeviceMat, table, "table")
    if table.get_device() != ctx.device or ids.get_device() != ctx.device or out is not None:
        _on_context(ctx, table=table, ids=ids, out=out)
    n, h = ids.numel(), src.cols
    if out is None:
        out = table.new_empty((*ids.shape, h), dtype=dtype)
        dst = _abi.OrdaDeviceMatMut(out.data_ptr(), n, h, h, _grad_dtype(out, "out"))
    elif dtype is not None and out.dtype != dtype:
        raise ValueError(f"out is {out.dtype}, not {dtype}")
    else:
        dst = _mat(_abi.OrdaDeviceMatMut, _rows_of(out, n, h, "out"), "out")
    buf = _err()
    rc = _lib().orda_embedding_device(ctx.handle, C.byref(src), ids.data_ptr(), n, scale, C.byref(dst),
                                      _context_stream(ctx, stream), buf, len(buf))
    if rc:
        _check(rc, buf)
    return out


def embedding_grad_device(
    ctx: DeviceContext,
    grad_out: torch.Tensor,
    ids: torch.Tensor,
    vocab: int,
    scale: float = 1.0,
    padding_id: Optional[int] = None,
    dtype: Optional[torch.dtype] = None,
    out: Optional[torch.Tensor] = None,
    accumulate: bool = False,
    stream=None,
) -> torch.Tensor:
    """`orda_embedding_grad_device`: the gradient [vocab, H] of the table, from
    grad_out (ids' shape and H, bf16 or f32). It is allocated in `dtype`
    (default grad_out's) or written to `out`; accumulate=True adds to what
    `out` holds (a shared table's output head gradient, say). Tokens of
    padding_id give no gradient. Ids out of range are reported by ctx.check()."""
    _ids(ids)
    _on_context(ctx, grad_out=grad_out, ids=ids, out=out)
    if grad_out.dim() < 1 or vocab < 1:
        raise ValueError("grad_out must have a last dimension H and vocab must be at least 1")
    n, h = ids.numel(), grad_out.shape[-1]
    g = grad_out if grad_out.dim() == 2 and grad_out.shape[0] == n else _rows_of(grad_out, n, h, "grad_out")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty(vocab, h, device=grad_out.device, dtype=dtype or grad_out.dtype)
    elif tuple(out.shape) != (vocab, h) or (h > 1 and out.stride(1) != 1):
        raise ValueError(f"out must be ({vocab}, {h}) with unit column stride")
    elif dtype is not None and out.dtype != dtype:
        raise ValueError(f"out is {out.dtype}, not {dtype}")
    buf = _err()
    rc = _lib().orda_embedding_grad_device(
        ctx.handle, C.byref(_mat(_abi.OrdaDeviceMat, g, "grad_out")), ids.data_ptr(), n, scale,
        padding_id is not None, padding_id or 0, C.byref(_mat(_abi.OrdaDeviceMatMut, out, "out")),
        accumulate, _context_stream(ctx, stream), buf, len(buf))
    _check(rc, buf)
    return out


def gemm_bf16(
    ctx: DeviceContext,
    a: torch.Tensor,
    a_kind: int,
    b: torch.Tensor,
    b_kind: int,
    c: torch.Tensor,
    m: int,
    n: int,
    k: int,
    alpha: float = 1.0,
    beta: float = 0.0,
    stream=None,
) -> torch.Tensor:
    """`orda_gemm_bf16_device`: C = alpha * op(A) @ op(B) + beta * C."""
    buf = _abi.err_buf()
    rc = _lib().orda_gemm_bf16_device(
        ctx.handle, a.data_ptr(), a.stride(0), a_kind, b.data_ptr(), b.stride(0), b_kind, c.data_ptr(), c.stride(0),
        m, n, k, alpha, beta, _stream(stream), buf, len(buf),
    )
    _check(rc, buf)
    return c


def quantize_grad_w(
    ctx: DeviceContext,
    grad_w: torch.Tensor,
    labels: torch.Tensor,
    ignore_index: int = -100,
    stochastic: bool = False,
    seed: int = 0,
    q: Optional[torch.Tensor] = None,
    scale: Optional[torch.Tensor] = None,
    stream=None,
):
    """`orda_quantize_grad_w_device`; grad_w is overwritten with the
    dequantised values, q / scale receive the INT8 body and scales."""
    v, h = grad_w.shape
    buf = _abi.err_buf()
    rc = _lib().orda_quantize_grad_w_device(
        ctx.handle, grad_w.data_ptr(), v, h, grad_w.stride(0), labels.data_ptr(), labels.numel(), ignore_index,
        int(stochastic), int(seed) & ((1 << 64) - 1), _ptr(q), _ptr(scale), _stream(stream), buf, len(buf),
    )
    _check(rc, buf)
    return grad_w, q, scale
