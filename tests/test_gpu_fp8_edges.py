"""8-bit linear layer where its scales are extreme, against the definition in 64 bits."""

import pytest
import torch

from _grouped_util import close, linear_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    return torch.device("cuda:0")


def _values(blocks, count=1):
    """float64: a scale times an 8-bit number is exact there."""
    q, s = blocks.q.cpu().double(), blocks.scale.cpu().double()
    if s.dim() == 3:
        s = s.repeat_interleave(128, 1)[:, : q.shape[0] // count].reshape(q.shape[0], -1)
    return q * s.repeat_interleave(128, 1)[:, : q.shape[1]]


SIZES = [(3, 1, 40), (300, 3, 200), (5000, 8, 520), (20000, 3, 1000)]  # split sums, single CTAs, pairs


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("T,count,N", SIZES)
def test_scales_whose_product_leaves_the_range(dev, T, count, N, dense):
    """Products of two scales that are subnormal, zero or infinite where the sums they belong to are not: among them a block
    of zeros under two scales of 1e20."""
    from nnue_pytorch_b200 import Fp8Blocks, GroupPlan, linear_fp8

    format, K = torch.float8_e5m2, 300
    g = torch.Generator().manual_seed(T)
    count = 1 if dense else count
    qx, sx = torch.zeros(T, K), torch.ones(T, 3)
    kind = torch.arange(T) % 3
    large = lambda *shape: torch.randint(-57344, 57345, shape, generator=g).float()  # noqa: E731
    qx[kind != 1, :128] = large(int((kind != 1).sum()), 128)
    sx[kind == 0, 0], sx[kind == 2, 0] = 1.7e-22, 2.6e-23  # times 1.3e-22: 4 significant bits, and 2
    sx[:, 1] = 1e20                                         # a block of zeros, and one too large times it
    qx[kind == 1, 256:] = 2.0**-16                          # the smallest numbers, the scales' product is infinite
    sx[kind == 1, 2] = 1e20
    qw = large(count * N, K)
    qw[:, 256:] = 2.0**-16 * torch.randint(-1, 2, (count * N, 44), generator=g)
    sw = torch.tensor([1.3e-22, 1e20, 1e20]).expand(count, -(-N // 128), 3)
    x8 = Fp8Blocks(qx.to(format).to(dev), sx.to(dev))
    w8 = Fp8Blocks(qw.to(format).to(dev), sw.to(dev))
    b = torch.zeros(T, dtype=torch.int64) if dense else torch.randint(-1, count, (T,), generator=g)
    y = linear_fp8(x8, w8, None, None if dense else GroupPlan(b.to(dev), count), torch.float32)
    ref, mag, _ = linear_ref(_values(x8), _values(w8, count), None, b, count)["y"]
    close(y, ref, mag, K + 3 * 3, "y")
    assert (y.cpu()[(b >= 0) & (kind == 0)].abs().max(1).values > 0).all()  # nothing vanished


@pytest.mark.parametrize("T,count,N", SIZES)
def test_rows_and_weights_of_extreme_size(dev, T, count, N):
    """fp32 rows and weights whose largest numbers meet zeros: the quantisers' own scales multiply to more than fp32 holds."""
    from nnue_pytorch_b200 import GroupPlan, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    g = torch.Generator().manual_seed(T + 1)
    K = 256
    x, w = torch.randn(T, K, generator=g), torch.randn(count * N, K, generator=g)
    x[:, 0], w[:, 0] = 3e36, 0.0
    x[:, 1], w[:, 1] = 0.0, 2e18
    b = torch.randint(-1, count, (T,), generator=g)
    xd, w8 = x.to(dev), quantize_fp8_tiles(w.to(dev), count)
    x8 = quantize_fp8_rows(xd)
    assert float(x8.scale.max()) * float(w8.scale.max()) > 3.5e38
    y = linear_fp8(xd, w8, None, GroupPlan(b.to(dev), count))
    ref, mag, _ = linear_ref(_values(x8), _values(w8, count), None, b, count)["y"]
    close(y, ref, mag, K + 3 * 2, "y")
