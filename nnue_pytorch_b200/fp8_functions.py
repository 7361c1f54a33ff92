"""8-bit floating point with one scale per block of 128, and the linear layer that multiplies it.

`quantize_fp8_rows` quantises activations (a scale per 128 consecutive numbers of a row), `quantize_fp8_tiles` weights (a
scale per 128 x 128 tile of each bucket's matrix).  Scales are powers of two: 2^ceil(log2(a / MAX)) for a block whose
largest finite number is a (MAX 448 for e4m3, 57344 for e5m2), 1 for a block of zeros; the only rounding is the one to
8 bits.  Numbers that are not finite become NaN in e4m3 and stay what they are in e5m2, without touching the scale.

`linear_fp8` multiplies them, dense or bucketed (with a `GroupPlan`), for evaluation: it has no gradient.  Blocks are constants:
quantised weights do not lead back to the parameters they were made of, and rows that would need a gradient are refused.

    w8 = quantize_fp8_tiles(weight, count)               # once per export
    y = linear_fp8(x, w8, bias, plan)                    # x bf16, fp16 or fp32: quantised on the way in
"""

from __future__ import annotations

import torch

from . import _lib
from ._launch import _outside_graphs, _ptr, _require_cuda, _span, _stream
from .grouped_linear_functions import GATHERED_ROWS, TYPES, GroupPlan, _has_tangent, _on, _pitched, _rows

FORMATS = (torch.float8_e4m3fn, torch.float8_e5m2)
BLOCK = 128


class Fp8Blocks:
    """Quantised numbers and their scales.

    q      float8 [rows, K] (rows at any pitch; the quantisers leave multiples of 16 bytes)
    scale  float32 [rows, ceil(K / 128)] (row blocks), or [count, ceil(N / 128), ceil(K / 128)] (tiles of `count`
           matrices of N rows each)"""

    __slots__ = ("q", "scale")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        assert q.dim() == 2 and q.dtype in FORMATS, "q is a float8_e4m3fn or float8_e5m2 matrix"
        assert scale.dtype == torch.float32 and scale.dim() in (2, 3) and scale.device == q.device
        blocks = (q.shape[1] + BLOCK - 1) // BLOCK
        if scale.dim() == 2:
            want = (q.shape[0], blocks)
        else:
            count = scale.shape[0]
            assert count >= 1 and q.shape[0] % count == 0, "the matrices' rows do not divide"
            want = (count, (q.shape[0] // count + BLOCK - 1) // BLOCK, blocks)
        assert tuple(scale.shape) == want, f"scales {tuple(scale.shape)} where {want} are needed"
        self.q, self.scale = q, scale.contiguous()

    def dequantize(self) -> torch.Tensor:
        """float32 [rows, K]: the numbers the blocks stand for."""
        rows, K = self.q.shape
        if self.scale.dim() == 2:
            return self.q.float() * self.scale.repeat_interleave(BLOCK, 1)[:, :K]
        count = self.scale.shape[0]
        s = self.scale.repeat_interleave(BLOCK, 1)[:, : rows // max(count, 1)].repeat_interleave(BLOCK, 2)[:, :, :K]
        return self.q.float() * s.reshape(rows, K)


def _check_source(t: torch.Tensor, format: torch.dtype) -> None:
    assert t.dim() == 2 and t.shape[1] >= 1, "a matrix with at least one column"
    assert t.dtype in (torch.float32, torch.bfloat16, torch.float16), "fp32, bf16 or fp16"
    assert format in FORMATS, "float8_e4m3fn or float8_e5m2"


def _check_no_gradient(what: str, *tensors: torch.Tensor | None) -> None:
    wanted = _has_tangent(*tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            wanted |= t is not None and t.requires_grad
    assert not wanted, f"{what} has no gradient: call it under torch.no_grad()"


def _empty_q(rows: int, K: int, format: torch.dtype, dev) -> tuple[torch.Tensor, int]:
    pitch = (K + 15) // 16 * 16
    q = torch.empty(rows, pitch, dtype=format, device=dev)
    return (q if pitch == K else q[:, :K]), pitch


@_outside_graphs
def quantize_fp8_rows(x: torch.Tensor, format: torch.dtype = torch.float8_e4m3fn) -> Fp8Blocks:
    """x [T, K] (fp32, bf16 or fp16) in 8 bits, one scale per 128 consecutive numbers of a row.  Has no gradient."""
    _check_no_gradient("quantize_fp8_rows", x)
    dev = _require_cuda(x)
    _check_source(x, format)
    x, ldx = _rows(x.detach())
    T, K = x.shape
    q, ldq = _empty_q(T, K, format, dev)
    scale = torch.empty(T, (K + BLOCK - 1) // BLOCK, dtype=torch.float32, device=dev)
    with _on(dev), _span("fp8_rows", dev):
        st = _lib.load().nnue_fp8_quantize_rows(_ptr(x), TYPES[x.dtype], ldx, _ptr(q), ldq, _ptr(scale), 0, T, K,
                                                TYPES[format], None, 0, _stream(dev))
    _lib.check(st, "nnue_fp8_quantize_rows")
    return Fp8Blocks(q, scale)


@_outside_graphs
def quantize_fp8_tiles(weight: torch.Tensor, count: int = 1, format: torch.dtype = torch.float8_e4m3fn) -> Fp8Blocks:
    """weight [count * N, K] (fp32, bf16 or fp16; `count` matrices below one another) in 8 bits, one scale per tile of
    128 x 128 of each matrix.  The blocks are constants, also those of a parameter."""
    assert not _has_tangent(weight), "quantize_fp8_tiles has no gradient: no tangent passes it"
    dev = _require_cuda(weight)
    _check_source(weight, format)
    count = int(count)
    assert 1 <= count <= 1024 and weight.shape[0] % count == 0, "the matrices' rows do not divide"
    weight, ldw = _rows(weight.detach())
    rows, K = weight.shape
    N = rows // count
    assert N >= 1, "empty matrices"
    q, ldq = _empty_q(rows, K, format, dev)
    scale = torch.empty(count, (N + BLOCK - 1) // BLOCK, (K + BLOCK - 1) // BLOCK, dtype=torch.float32, device=dev)
    with _on(dev), _span("fp8_tiles", dev):
        st = _lib.load().nnue_fp8_quantize_tiles(_ptr(weight), TYPES[weight.dtype], ldw, _ptr(q), ldq, _ptr(scale), count, N, K,
                                                 TYPES[format], _stream(dev))
    _lib.check(st, "nnue_fp8_quantize_tiles")
    return Fp8Blocks(q, scale)


@_outside_graphs
def linear_fp8(x: torch.Tensor | Fp8Blocks, weight: Fp8Blocks, bias: torch.Tensor | None = None,
               plan: GroupPlan | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[p] = weight[b(p)] x[p] + bias[b(p)] on 8-bit operands, fp32 sums; zeros for rows of no bucket.

    x       [T, K]: fp32, bf16 or fp16 (quantised to the weight's format first), or `Fp8Blocks` of rows in it
    weight  `Fp8Blocks` of tiles, [count * N, K]
    bias    fp32, count * N numbers, or None
    plan    the rows' `GroupPlan`; None for a single matrix (count 1)
    out_dtype  float32, bfloat16 or float16; x's type by default (bfloat16 for `Fp8Blocks`)"""
    assert isinstance(weight, Fp8Blocks) and weight.scale.dim() == 3, "the weight is an Fp8Blocks of tiles"
    _check_no_gradient("linear_fp8", x if isinstance(x, torch.Tensor) else x.scale, weight.scale, bias)
    format = weight.q.dtype
    E = weight.scale.shape[0]
    given = not isinstance(x, torch.Tensor)
    if given:
        assert x.scale.dim() == 2 and x.q.dtype == format, "the rows are Fp8Blocks of rows in the weight's format"
        rows, out_dtype = x.q, out_dtype or torch.bfloat16
    else:
        _check_source(x, format)
        rows, out_dtype = x, out_dtype or x.dtype
    assert out_dtype in (torch.float32, torch.bfloat16, torch.float16)
    dev = _require_cuda(rows, weight.q, weight.scale)
    if given:
        _require_cuda(rows, x.scale)
    T, K = rows.shape
    N = weight.q.shape[0] // E
    assert weight.q.shape[1] == K, f"rows of {K} inputs against weights of {weight.q.shape[1]}"
    if plan is not None:
        plan.check(rows)
        assert plan.count == E, f"a plan of {plan.count} buckets for {E} matrices"
    else:
        assert E == 1, "several matrices need a plan"
    if bias is not None:
        _require_cuda(rows, bias)
        assert bias.dtype == torch.float32 and bias.numel() == E * N
        bias = bias.detach().contiguous()
    lib = _lib.load()
    laid = plan is not None and T > GATHERED_ROWS * E  # few rows per bucket are gathered by the product itself
    buffer = None if plan is None else _ptr(plan.buffer)
    y = torch.empty(T, N, dtype=out_dtype, device=dev)
    with _on(dev), _span("linear_fp8", dev):
        s = _stream(dev)
        wr, ldw = _pitched(weight.q, format, lib, dev)
        C = (K + BLOCK - 1) // BLOCK
        if not given:
            xs, ldx = _rows(x.detach())
            if laid:
                nbytes = lib.nnue_group_rows_bytes(T, (K + 15) // 16 * 8, E)
                xr, pitch, places = torch.empty(nbytes, dtype=torch.uint8, device=dev), 0, nbytes // ((K + 15) // 16 * 16)
            else:
                (xr, pitch), places = _empty_q(T, K, format, dev), T
            # scales by block, four rows at a time, where the product's rows are neighbours; by row where it gathers them
            scale_ld = (places + 3) // 4 * 4 if laid or plan is None else 0
            scale = torch.empty(C * (scale_ld or T), dtype=torch.float32, device=dev)
            _lib.check(lib.nnue_fp8_quantize_rows(_ptr(xs), TYPES[xs.dtype], ldx, _ptr(xr), pitch, _ptr(scale), scale_ld, T, K,
                                                  TYPES[format], buffer if laid else None, E, s), "nnue_fp8_quantize_rows")
            ldx = pitch
        else:
            scale, scale_ld = x.scale, 0
            xr, ldx = _pitched(x.q, format, lib, dev, whole=laid)
            if laid:  # pairs of bytes as 16-bit numbers, moved as they are
                src, xr = xr, torch.empty(lib.nnue_group_rows_bytes(T, (K + 15) // 16 * 8, E), dtype=torch.uint8, device=dev)
                _lib.check(lib.nnue_group_rows(_ptr(src), TYPES[torch.bfloat16], ldx // 2, buffer, _ptr(xr), TYPES[torch.bfloat16],
                                               None, T, (K + 15) // 16 * 8, E, s), "nnue_group_rows")
        st = lib.nnue_fp8_linear_fwd(_ptr(xr), ldx, laid, _ptr(scale), scale_ld, _ptr(wr), ldw, _ptr(weight.scale), _ptr(bias), buffer,
                                     _ptr(y), TYPES[out_dtype], T, K, N, E, TYPES[format], s)
    _lib.check(st, "nnue_fp8_linear_fwd")
    return y
