"""Bucketed ("grouped by expert") linear layers on 16-bit operands.

`GroupPlan` groups the rows of a batch by their bucket; `grouped_linear` multiplies every row with the weights of its own
bucket and has gradients for the rows, the weights and the bias.  Any number of buckets up to 1024, any layer size; the
reference multiplies every row with all buckets' weights and selects afterwards (model/modules/stacked_linear.py:38-66).

    plan = GroupPlan(bucket, count)                      # int64 or int32 [T]; -1: a padding row of no bucket
    y = grouped_linear(x, weight, bias, plan)            # x [T, K], weight [count * N, K], bias [count * N]

Operands are bf16 or fp16, sums fp32.  fp32 parameters (weight, bias) are allowed: the weights are rounded to the
rows' type for the products, their gradients come back in fp32, unrounded.  One plan serves every layer and direction
of its batch.
"""

from __future__ import annotations

import torch
from torch import autograd
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._launch import _NO_SPAN, _outside_graphs, _ptr, _require_cuda, _span, _stream

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}
HALF = (torch.bfloat16, torch.float16)


def _on(dev: torch.device):
    """Context in which `dev` is the current device (nothing to do when it already is)."""
    return _NO_SPAN if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _has_tangent(*tensors: torch.Tensor | None) -> bool:
    """True inside a forward-mode level where one of the tensors carries a tangent (such a tensor need not require a gradient)."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _pad4(n: int) -> int:
    return (n + 3) // 4 * 4


class GroupPlan:
    """Rows of a batch grouped by bucket (`nnue_group_plan`): a stable sort.

    order    int32 [T]: the rows by bucket, ascending inside a bucket, rows of no bucket (-1) last
    offsets  int32 [count + 1]: first place of every bucket in `order`, and the number of rows that have one

    An id below -1 or from `count` on is treated as -1 and recorded in the device status word
    (`_lib.device_status`).  The plan is built on the current stream and holds no reference to `bucket`."""

    __slots__ = ("rows", "count", "device", "buffer")

    @_outside_graphs
    def __init__(self, bucket: torch.Tensor, count: int):
        dev = _require_cuda(bucket)
        assert bucket.dtype in (torch.int64, torch.int32), "bucket ids are int64 or int32"
        count = int(count)
        assert 1 <= count <= 1024, "1 to 1024 buckets"
        bucket = bucket.detach().reshape(-1).contiguous()
        lib = _lib.load()
        self.rows, self.count, self.device = bucket.numel(), count, dev
        nbytes = lib.nnue_group_plan_bytes(self.rows, count)
        self.buffer = torch.empty(max(nbytes // 4, 4), dtype=torch.int32, device=dev)
        with _on(dev), _span("group_plan", dev):
            st = lib.nnue_group_plan(_ptr(bucket), bucket.dtype == torch.int64, self.rows, count, _ptr(self.buffer), nbytes,
                                     _stream(dev))
        _lib.check(st, "nnue_group_plan")

    @property
    def offsets(self) -> torch.Tensor:
        return self.buffer[4 : 5 + self.count]

    @property
    def order(self) -> torch.Tensor:
        at = 4 + _pad4(self.count + 2)
        return self.buffer[at : at + self.rows]

    def check(self, t: torch.Tensor) -> None:
        assert t.shape[0] == self.rows, f"the plan was built for {self.rows} rows, not {t.shape[0]}"
        assert t.device == self.device, "the plan lives on another device"


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(t, pitch of its rows) with neighbouring columns next to each other and rows that do not overlap.  The stride of a
    single row says nothing: a transposed column has 1."""
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1 or rows > 1 and t.stride(0) < cols:
        t = t.contiguous()
    return t, t.stride(0) if rows > 1 else cols


def _pitched(t: torch.Tensor, dtype: torch.dtype, lib, dev, whole: bool = False) -> tuple[torch.Tensor, int]:
    """(t as rows of `dtype` that start at multiples of 16 bytes, their pitch in elements): `t` itself where it is one,
    else a copy whose rows are padded with zeros (`nnue_pack_rows`).  `whole`: the last 16 bytes of every row may be read."""
    rows, cols = t.shape
    unit = 16 // dtype.itemsize
    if whole and cols % unit:
        pass
    elif t.dtype == dtype and (cols == 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0:
        pitch = t.stride(0)
        if pitch % unit == 0 and pitch >= cols:
            return t, pitch
        if rows == 1 and cols % unit == 0:
            return t, cols
    t, ld = _rows(t)
    pitch = (cols + unit - 1) // unit * unit
    out = torch.empty(rows, pitch, dtype=dtype, device=dev)
    st = lib.nnue_pack_rows(_ptr(t), TYPES[t.dtype], ld, _ptr(out), TYPES[dtype], pitch, rows, cols, _stream(dev))
    _lib.check(st, "nnue_pack_rows")
    return out, pitch


def _laid_out(t: torch.Tensor, dtype: torch.dtype, plan_buffer, E: int, lib, dev, sums: bool = False):
    """(t laid out by bucket as `dtype` (`nnue_group_rows`), the sums of its columns per tile or None)."""
    T, cols = t.shape
    t, ld = _rows(t)
    out = torch.empty(lib.nnue_group_rows_bytes(T, cols, E), dtype=torch.uint8, device=dev)
    part = torch.empty(lib.nnue_group_sums_bytes(T, cols, E) // 4, dtype=torch.float32, device=dev) if sums else None
    st = lib.nnue_group_rows(_ptr(t), TYPES[t.dtype], ld, _ptr(plan_buffer), _ptr(out), TYPES[dtype], _ptr(part), T, cols,
                             E, _stream(dev))
    _lib.check(st, "nnue_group_rows")
    return out, part


# Up to this many rows per bucket the products gather them as they lie; beyond it they are laid out by bucket first.  Kernels
# together, us, gathered against laid out (8 bits in brackets):
#   8 buckets of 1024 -> 1024, bf16     16 rows 21, 26 (18, 20)    32 rows 25, 26 (19, 20)    64 rows 33, 29 (22, 20)
#   64 of 2048 -> 1024                  16 rows 65, 73 (51, 53)    32 rows 66, 75 (58, 54)    64 rows 72, 78 (77, 56)
#   8 of 4096 -> 2048                    8 rows 53, 57 (40, 40)    16 rows 61, 57 (44, 40)    32 rows 78, 58 (52, 40)
GATHERED_ROWS = 16


def _forward(x, weight, bias, plan, out_dtype, keep_rows):
    """y, x as the product read it, the weights as it read them and their pitch.  `keep_rows`: x is laid out by bucket whatever
    its length, as the weight gradient reads it."""
    dev = _require_cuda(x, weight) if bias is None else _require_cuda(x, weight, bias)
    dtype = x.dtype
    assert dtype in HALF, "rows are bf16 or fp16"
    assert weight.dtype in (dtype, torch.float32), "weights have the rows' type or are fp32"
    out_dtype = out_dtype or dtype
    assert out_dtype in (dtype, torch.float32), "the output has the rows' type or is fp32"
    assert x.dim() == 2 and weight.dim() in (2, 3)
    plan.check(x)
    E = plan.count
    w2 = weight.detach().flatten(0, 1) if weight.dim() == 3 else weight.detach()
    T, K = x.shape
    N = w2.shape[0] // E
    assert K >= 1 and N >= 1 and w2.shape == (E * N, K) and (weight.dim() == 2 or weight.shape[0] == E), \
        f"weight {tuple(weight.shape)} does not hold {E} layers of {K} inputs"
    if bias is not None:
        assert bias.dtype in (dtype, torch.float32) and bias.numel() == E * N
        bias = bias.detach().contiguous()
    lib = _lib.load()
    y = torch.empty(T, N, dtype=out_dtype, device=dev)
    laid = keep_rows or T > GATHERED_ROWS * E
    with _on(dev), _span("grouped_linear_fwd", dev):
        s = _stream(dev)
        if laid:
            xr, ldx = _laid_out(x.detach(), dtype, plan.buffer, E, lib, dev)[0], 0
        else:
            xr, ldx = _pitched(x.detach(), dtype, lib, dev)
        wr, ldw = _pitched(w2, dtype, lib, dev)
        st = lib.nnue_grouped_linear_fwd(
            _ptr(xr), ldx, laid, _ptr(wr), ldw, _ptr(bias), 0 if bias is None else TYPES[bias.dtype], _ptr(plan.buffer), _ptr(y),
            TYPES[out_dtype], T, K, N, E, TYPES[dtype], s)
    _lib.check(st, "nnue_grouped_linear_fwd")
    return y, xr, wr, ldw


class GroupedLinearFunction(autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, plan, out_dtype=None):
        y, xr, wr, ldw = _forward(x, weight, bias, plan, out_dtype, ctx.needs_input_grad[1])
        ctx.save_for_backward(xr if ctx.needs_input_grad[1] else None, wr if ctx.needs_input_grad[0] else None, plan.buffer)
        ctx.dims, ctx.w_read = (*x.shape, y.shape[1], plan.count), (wr.stride(), ldw)
        ctx.dtype, ctx.w_like, ctx.b_like = x.dtype, (weight.dtype, weight.shape), None if bias is None else (bias.dtype, bias.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, plan = ctx.saved_tensors
        T, K, N, E = ctx.dims
        dev, dtype = dy.device, ctx.dtype
        lib = _lib.load()
        need_x, need_w, need_b = ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        dx = dw = db = None
        with _on(dev), _span("grouped_linear_bwd", dev):
            s = _stream(dev)
            # saved-tensor hooks may give the same numbers back with other strides
            plan, x = plan.contiguous(), None if x is None else x.contiguous()
            if need_w or need_b or T > GATHERED_ROWS * E:
                dyr, part = _laid_out(dy, dtype, plan, E, lib, dev, sums=need_b)
                laid, lddy = 1, 0
            else:
                dyr, lddy = _pitched(dy, dtype, lib, dev)
                laid = 0
            if need_x:
                strides, ldw = ctx.w_read
                if w.stride() != strides:
                    w, ldw = _pitched(w, dtype, lib, dev)
                dx = torch.empty(T, K, dtype=dtype, device=dev)
                _lib.check(lib.nnue_grouped_linear_bwd_input(_ptr(dyr), lddy, laid, _ptr(w), ldw, _ptr(plan), _ptr(dx), T, K, N, E,
                                                             TYPES[dtype], s), "nnue_grouped_linear_bwd_input")
            if need_b:
                db = torch.empty(ctx.b_like[1], dtype=ctx.b_like[0], device=dev)
            if need_w:
                w_dtype, w_shape = ctx.w_like
                dw = torch.empty(w_shape, dtype=w_dtype, device=dev)
                _lib.check(lib.nnue_grouped_linear_bwd_weight(
                    _ptr(dyr), _ptr(part), _ptr(x), _ptr(plan), _ptr(dw), TYPES[w_dtype], _ptr(db),
                    0 if db is None else TYPES[db.dtype], T, K, N, E, TYPES[dtype], s), "nnue_grouped_linear_bwd_weight")
            elif need_b:
                _lib.check(lib.nnue_group_sums(_ptr(part), _ptr(plan), _ptr(db), TYPES[db.dtype], T, N, E, s), "nnue_group_sums")
        return dx, dw, db, None, None


@_outside_graphs  # ctypes launches: runs eagerly inside a compiled model
def grouped_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, plan: GroupPlan,
                   out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[p] = weight[b(p)] x[p] + bias[b(p)], zeros for rows of no bucket.

    x       bf16 or fp16 [T, K], any strides
    weight  [count * N, K] or [count, N, K], of x's type or fp32
    bias    count * N numbers of x's type or fp32, or None
    out_dtype  x's type (default) or float32

    Gradients: those of the formula, with dy rounded to x's type where it is fp32; each in its tensor's own type.  They have
    no gradients of their own, and there is no forward mode: tensors with tangents are refused.  Everything runs on the
    current stream and can be captured into a CUDA graph; as for any operator, no eager autograd graph of the same leaves
    may be alive when a backward pass is captured."""
    if (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))) \
            or _has_tangent(x, weight, bias):  # the function has no forward mode and says so
        return GroupedLinearFunction.apply(x, weight, bias, plan, out_dtype)
    return _forward(x, weight, bias, plan, out_dtype, False)[0]
