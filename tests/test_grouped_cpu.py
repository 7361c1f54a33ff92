"""Refusals of the bucketed and 8-bit operators, checked on the host before any CUDA call."""

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nnue_pytorch_b200 import _build, _lib

    _build.build()
    return _lib.load()


def _message(lib):
    return lib.nnue_b200_last_error().decode()


def test_plan_arguments(lib):
    f = lib.nnue_group_plan_bytes
    assert f(0, 1) > 0 and f(-1, 4) == 0 and f(10, 0) == 0 and f(10, 1025) == 0 and f((1 << 30) + 1, 8) == 0
    assert f(1000, 8) >= 4 * (4 + 12 + 1000) and f(100000, 8) < f(100000, 64)
    g = lib.nnue_group_plan
    assert g(None, 1, -1, 4, None, 0, None) == -1
    assert g(None, 1, 4, 0, None, 0, None) == -1
    assert g(None, 1, 4, 1025, None, 0, None) == -4
    assert g(None, 1, (1 << 30) + 1, 8, None, 0, None) == -4
    assert g(None, 1, 4, 8, None, 0, None) == -1 and "null bucket" in _message(lib)
    assert g(64, 1, 4, 8, 64, 8, None) == -3 and "too small" in _message(lib)
    assert g(64, 1, 4, 8, 68, 1 << 20, None) == -3


def test_grouped_linear_arguments(lib):
    BF16, F16, F32, E4M3 = 1, 2, 0, 3
    P = 1 << 20  # an aligned address that no refused call reads

    def fwd(x=P, ldx=64, laid=0, w=P, ldw=64, bias=None, bt=0, plan=P, y=P, yt=BF16, T=8, K=64, N=16, E=2, type=BF16):
        return lib.nnue_grouped_linear_fwd(x, ldx, laid, w, ldw, bias, bt, plan, y, yt, T, K, N, E, type, None)

    assert fwd(T=0) == 0  # an empty batch needs no device
    assert fwd(T=-1) == -1 and fwd(K=0) == -1 and fwd(N=0) == -1 and fwd(E=0) == -1
    assert fwd(E=1025) == -4 and fwd(K=1 << 24, ldx=1 << 24, ldw=1 << 24) == -4
    assert fwd(type=F32) == -4 and fwd(type=E4M3) == -4 and fwd(yt=F16) == -4 and fwd(bias=P, bt=E4M3) == -4
    assert fwd(plan=None) == -1 and fwd(x=None) == -1 and fwd(w=None) == -1
    assert fwd(ldx=63) == -1 and "pitch" in _message(lib)
    assert fwd(ldx=66) == -2 and fwd(x=P + 2) == -2 and fwd(ldw=68) == -2 and fwd(y=P + 4) == -2
    assert "16 bytes" in _message(lib) or "unaligned" in _message(lib)

    def dx(dy=P, lddy=16, laid=0, w=P, ldw=64, plan=P, out=P, T=8, K=64, N=16, E=2, type=F16):
        return lib.nnue_grouped_linear_bwd_input(dy, lddy, laid, w, ldw, plan, out, T, K, N, E, type, None)

    assert dx(T=0) == 0 and dx(dy=None) == -1 and dx(lddy=17) == -2 and dx(lddy=15) == -1 and dx(out=None) == -2 and dx(type=7) == -4

    def dw(dy=P, sums=P, x=P, plan=P, out=P, ot=F32, db=None, bt=0, T=8, K=64, N=16, E=2, type=F16):
        return lib.nnue_grouped_linear_bwd_weight(dy, sums, x, plan, out, ot, db, bt, T, K, N, E, type, None)

    assert dw(ot=BF16) == -4 and dw(db=P, bt=E4M3) == -4 and dw(x=None) == -1 and dw(dy=P + 2) == -2 and dw(out=None) == -2
    assert dw(db=P, sums=None) == -1 and "sums" in _message(lib)
    rows = lambda **k: lib.nnue_group_rows(*({**dict(s=P, st=F32, ld=64, plan=P, d=P, t=BF16, sums=None, T=4, c=64, E=2), **k}.values()), None)  # noqa: E731
    assert rows(T=0) == 0 and rows(T=-1) == -1 and rows(ld=63) == -1 and rows(c=0) == -1 and rows(E=0) == -1 and rows(E=1025) == -4
    assert rows(st=E4M3) == -4 and rows(t=F32) == -4 and rows(s=None) == -1 and rows(d=P + 8) == -2 and rows(plan=P + 4) == -2
    assert lib.nnue_group_rows_bytes(100, 20, 8) >= 100 * 24 * 2 and lib.nnue_group_rows_bytes(-1, 20, 8) == 0
    assert lib.nnue_group_sums_bytes(300, 20, 8) >= 4 * 20 * 4 and lib.nnue_group_sums_bytes(300, 0, 8) == 0
    assert lib.nnue_group_sums(None, P, P, F32, 4, 8, 2, None) == -1 and lib.nnue_group_sums(P, P, P, E4M3, 4, 8, 2, None) == -4
    assert lib.nnue_pack_rows(P, F32, 4, P, E4M3, 4, 1, 4, None) == -4
    assert lib.nnue_pack_rows(P, F32, 3, P, BF16, 4, 1, 4, None) == -1
    assert lib.nnue_pack_rows(None, F32, 4, None, BF16, 8, 1, 4, None) == -1
    assert lib.nnue_pack_rows(None, F32, 4, None, BF16, 8, 0, 4, None) == 0


def test_fp8_arguments(lib):
    P = 1 << 20
    rows = lambda **k: lib.nnue_fp8_quantize_rows(*({**dict(x=P, t=1, ldx=64, q=P, ldq=64, s=P, sl=0, T=4, K=64, f=3, plan=None, E=0), **k}.values()), None)  # noqa: E731
    assert rows(T=0) == 0 and rows(T=-1) == -1 and rows(K=0) == -1 and rows(ldx=63) == -1 and rows(ldq=63) == -1 and rows(ldq=129) == -1
    assert rows(plan=P) == -1 and rows(plan=P, E=1025) == -1 and rows(plan=P + 4, E=2) == -1 and rows(plan=P, E=2, ldq=0, T=0) == 0
    assert rows(t=3) == -4 and rows(f=1) == -4 and rows(x=None) == -1 and rows(s=None) == -1
    assert rows(sl=3) == -1 and rows(sl=4, T=0) == 0 and rows(plan=P, E=2, sl=4) == -1
    tiles = lambda **k: lib.nnue_fp8_quantize_tiles(*({**dict(x=P, t=1, ldx=64, q=P, ldq=64, s=P, E=1, N=4, K=64, f=3), **k}.values()), None)  # noqa: E731
    assert tiles(E=0) == -1 and tiles(N=0) == 0 and tiles(f=0) == -4 and tiles(q=None) == -1
    lin = lambda **k: lib.nnue_fp8_linear_fwd(*({**dict(x=P, ldx=64, laid=0, sx=P, sl=0, w=P, ldw=64, sw=P, b=None, plan=P, y=P, yt=1, T=4, K=64, N=8, E=2, f=3), **k}.values()), None)  # noqa: E731
    assert lin(T=0) == 0 and lin(plan=None) == -1 and lin(plan=None, E=1, T=0) == 0 and lin(plan=None, E=1, laid=1) == -1 and lin(f=1) == -4 and lin(yt=4) == -4
    assert lin(sx=None) == -1 and lin(sw=None) == -1 and lin(y=None) == -1 and lin(ldx=65) == -2 and lin(ldw=72) == -2
    assert lin(w=P + 8) == -2 and lin(y=P + 1) == -2 and lin(ldx=48) == -1 and lin(E=2000) == -4
    assert lin(sl=8) == -1 and lin(sl=4, laid=1) == -1 and lin(sl=3, plan=None, E=1) == -1


def test_python_refusals():
    """No CPU path; types and shapes are checked where a CPU tensor can show it."""
    from nnue_pytorch_b200 import Fp8Blocks, GroupPlan, grouped_linear, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        GroupPlan(torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        grouped_linear(torch.zeros(2, 8).bfloat16(), torch.zeros(8, 8).bfloat16(), None, None)
    for f in (quantize_fp8_rows, quantize_fp8_tiles):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            f(torch.zeros(4, 16))
    q = torch.zeros(4, 130).to(torch.float8_e4m3fn)
    with pytest.raises(AssertionError):
        Fp8Blocks(q.float(), torch.ones(4, 2))
    with pytest.raises(AssertionError, match="scales"):
        Fp8Blocks(q, torch.ones(4, 1))
    with pytest.raises(AssertionError, match="scales"):
        Fp8Blocks(q, torch.ones(2, 2, 2))
    with pytest.raises(AssertionError, match="divide"):
        Fp8Blocks(q, torch.ones(3, 1, 2))
    tiles = Fp8Blocks(q, torch.ones(1, 1, 2))
    rows = Fp8Blocks(q, torch.ones(4, 2))
    assert torch.equal(tiles.dequantize(), torch.zeros(4, 130))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        linear_fp8(rows, tiles)
    with pytest.raises(AssertionError, match="tiles"):
        linear_fp8(rows, rows)
    with pytest.raises(AssertionError, match="no gradient"):
        linear_fp8(torch.zeros(2, 130, requires_grad=True), tiles)
    with pytest.raises(AssertionError, match="format"):
        linear_fp8(Fp8Blocks(torch.zeros(4, 130).to(torch.float8_e5m2), torch.ones(4, 2)), tiles)
