"""8-bit quantisation by blocks of 128 and the 8-bit linear layer against their definitions in 64 bits."""

import pytest
import torch

from _grouped_util import close, linear_ref, quantize_ref

pytestmark = pytest.mark.gpu

FORMATS = [torch.float8_e4m3fn, torch.float8_e5m2]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    return torch.device("cuda:0")


def _values(rows, K, seed):
    """Numbers over a wide range: rows of very different sizes, zeros, a block of zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-30, 12, (rows, 1), generator=g).float())
    x[torch.rand(rows, K, generator=g) < 0.3] = 0.0
    x[rows // 2] = 0.0
    return x


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K", [(1, 1), (3, 16), (5, 127), (4, 128), (7, 129), (33, 1000), (2, 4104)])
def test_rows(dev, T, K, dtype, format):
    from nnue_pytorch_b200 import quantize_fp8_rows

    x = _values(T, K, T + K).to(dtype)
    got = quantize_fp8_rows(x.to(dev), format)
    q, s = quantize_ref(x, 1, format)
    assert torch.equal(got.q.float().cpu(), q) and torch.equal(got.scale.cpu(), s)
    assert got.q.stride(0) % 16 == 0 and torch.equal(got.dequantize().cpu(), q * s.repeat_interleave(128, 1)[:, :K])


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("count,N,K", [(1, 1, 1), (3, 5, 40), (1, 128, 128), (2, 129, 257), (5, 200, 1000), (8, 32, 1024)])
def test_tiles(dev, count, N, K, dtype, format):
    from nnue_pytorch_b200 import quantize_fp8_tiles

    w = _values(count * N, K, N + K).to(dtype)
    got = quantize_fp8_tiles(w.to(dev), count, format)
    for e in range(count):
        q, s = quantize_ref(w[e * N : (e + 1) * N], 128, format)
        assert torch.equal(got.q[e * N : (e + 1) * N].float().cpu(), q) and torch.equal(got.scale[e].cpu(), s)


@pytest.mark.parametrize("format", FORMATS)
def test_borders_of_the_scale(dev, format):
    """Largest numbers at, just below and just above MAX times a power of two; the smallest and largest of fp32."""
    from nnue_pytorch_b200 import quantize_fp8_rows

    top = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}[format]
    rows = []
    for k in (-140, -127, -126, -100, -10, 0, 1, 30, 100):
        a = torch.tensor(top * 2.0**k, dtype=torch.float32)
        if not torch.isfinite(a):
            continue
        rows += [a, torch.nextafter(a, torch.tensor(0.0)), torch.nextafter(a, torch.tensor(float("inf"))), -a]
    rows += [torch.tensor(v) for v in (1e-45, 1.1754944e-38, 3.4028235e38, -3.4028235e38, 0.0, -0.0)]
    x = torch.zeros(len(rows), 130)
    x[:, 5] = torch.stack(rows)
    x[:, 77] = torch.stack(rows) * 0.37
    x[:, 129] = torch.stack(rows)
    got = quantize_fp8_rows(x.to(dev), format)
    q, s = quantize_ref(x, 1, format)
    assert torch.equal(got.scale.cpu(), s) and torch.equal(got.q.float().cpu(), q)


@pytest.mark.parametrize("format", FORMATS)
def test_every_rounding(dev, format):
    """All numbers of the format, the midpoints between neighbours and their fp32 neighbours on either side."""
    from nnue_pytorch_b200 import quantize_fp8_rows

    all8 = torch.arange(256, dtype=torch.uint8).view(format).float()
    all8 = torch.unique(all8[torch.isfinite(all8)])
    mid = (all8[1:] + all8[:-1]) / 2
    inf = torch.tensor(float("inf"))
    v = torch.cat([all8, mid, torch.nextafter(mid, inf), torch.nextafter(mid, -inf)])
    x = torch.zeros((len(v) + 126) // 127, 128)
    x[:, 0] = float(all8.max())  # scale 1
    x[:, 1:] = torch.nn.functional.pad(v, (0, x.shape[0] * 127 - len(v))).view(-1, 127)
    got = quantize_fp8_rows(x.to(dev), format)
    assert (got.scale == 1).all() and torch.equal(got.q.float().cpu(), x.to(format).float())


@pytest.mark.parametrize("format", FORMATS)
def test_not_finite_numbers(dev, format):
    from nnue_pytorch_b200 import quantize_fp8_rows, quantize_fp8_tiles

    x = torch.randn(6, 300)
    x[1, 3], x[2, 140], x[3, 299], x[4] = float("nan"), float("inf"), float("-inf"), float("nan")
    for got, (q, s) in ((quantize_fp8_rows(x.to(dev), format), quantize_ref(x, 1, format)),
                        (quantize_fp8_tiles(x.to(dev), 1, format), quantize_ref(x, 128, format))):
        assert torch.equal(got.scale.view(s.shape).cpu(), s)
        assert torch.equal(torch.nan_to_num(got.q.float().cpu(), nan=7e7, posinf=8e7, neginf=-8e7),
                           torch.nan_to_num(q, nan=7e7, posinf=8e7, neginf=-8e7))


def test_strided_sources(dev):
    from nnue_pytorch_b200 import quantize_fp8_rows, quantize_fp8_tiles

    big = torch.randn(64, 700, device=dev)
    for x in (big[:, 3:303], big[::2, :300], big.t(), big[:1].expand(5, 700), big[:, 5:6]):
        a, b = quantize_fp8_rows(x), quantize_fp8_rows(x.contiguous())
        assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale, b.scale)
        a, b = quantize_fp8_tiles(x), quantize_fp8_tiles(x.contiguous())
        assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale, b.scale)


def _linear(dev, T, count, K, N, format, out_dtype, seed, arbitrary_scales=False, dense=False):
    from nnue_pytorch_b200 import Fp8Blocks, GroupPlan, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    w = torch.randn(count * N, K, generator=g) / K**0.5
    bias = torch.randn(count * N, generator=g)
    b = torch.zeros(T, dtype=torch.int64) if dense else torch.randint(-1, count, (T,), generator=g)
    x8, w8 = quantize_fp8_rows(x.to(dev), format), quantize_fp8_tiles(w.to(dev), count, format)
    if arbitrary_scales:
        x8 = Fp8Blocks(x8.q, torch.rand(x8.scale.shape, generator=g).to(dev) + 0.1)
        w8 = Fp8Blocks(w8.q, torch.rand(w8.scale.shape, generator=g).to(dev) - 0.4)
    y = linear_fp8(x8, w8, bias.to(dev), None if dense else GroupPlan(b.to(dev), count), out_dtype)
    assert y.dtype == out_dtype
    # values in 64 bits: a scale times an 8-bit number is exact there
    def value(blocks):
        q, s, K = blocks.q.cpu().double(), blocks.scale.cpu().double(), blocks.q.shape[1]
        if s.dim() == 3:
            s = s.repeat_interleave(128, 1)[:, : q.shape[0] // s.shape[0]].reshape(q.shape[0], -1)
        return q * s.repeat_interleave(128, 1)[:, :K]

    ref, mag, _ = linear_ref(value(x8), value(w8), bias, b, count)["y"]
    # K products, and for each block the product of the scales, the scaling and its sum
    close(y, ref, mag, K + 3 * (-(-K // 128)), "y")
    assert not y.cpu()[b < 0].any()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("T,count,K,N", [(1, 1, 16, 1), (1, 8, 128, 64), (2, 3, 40, 7), (130, 1, 129, 129), (300, 5, 512, 200),
                                         (64, 70, 200, 33), (1000, 8, 1024, 32), (257, 2, 1000, 300), (4, 2, 4100, 130),
                                         (9000, 8, 300, 2100), (20000, 3, 1000, 520), (5000, 40, 130, 520)])
def test_linear(dev, T, count, K, N, format):
    for i, out in enumerate((torch.bfloat16, torch.float16, torch.float32) if T < 5000 else (torch.bfloat16,)):
        _linear(dev, T, count, K, N, format, out, T + i)
    _linear(dev, T, count, K, N, format, torch.float32, T + 5, arbitrary_scales=True)
    _linear(dev, T, 1, K, N, format, torch.float32, T + 6, dense=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K", [(77, 200), (30, 200), (900, 208), (900, 1030)])
def test_linear_quantises_its_rows(dev, dtype, T, K):
    from nnue_pytorch_b200 import GroupPlan, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, K, generator=g).to(dev, dtype)
    w8 = quantize_fp8_tiles(torch.randn(3 * 50, K, generator=g).to(dev), 3)
    plan = GroupPlan(torch.randint(-1, 3, (T,), generator=g).to(dev), 3)
    y = linear_fp8(x, w8, None, plan)
    assert y.dtype == dtype
    assert torch.equal(y, linear_fp8(quantize_fp8_rows(x), w8, None, plan, dtype))
    assert torch.equal(y, linear_fp8(x, w8, None, plan))  # the same bits again
    wide = torch.randn(T, 2 * K, generator=g).to(dev, dtype)
    assert torch.equal(linear_fp8(wide[:, 1::2], w8, None, plan), linear_fp8(wide[:, 1::2].contiguous(), w8, None, plan))
    assert torch.equal(linear_fp8(wide[:, 3 : 3 + K], w8, None, plan), linear_fp8(wide[:, 3 : 3 + K].contiguous(), w8, None, plan))


def test_linear_with_unaligned_operands(dev):
    from nnue_pytorch_b200 import Fp8Blocks, GroupPlan, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    g = torch.Generator().manual_seed(5)
    x8 = quantize_fp8_rows(torch.randn(40, 130, generator=g).to(dev))
    w8 = quantize_fp8_tiles(torch.randn(30, 130, generator=g).to(dev))
    want = linear_fp8(x8, w8)
    plan = GroupPlan(torch.randint(-1, 1, (40,), generator=g).to(dev), 1)
    tight = lambda q: q.view(torch.uint8).contiguous().view(q.dtype)  # noqa: E731  rows of 130 bytes
    assert torch.equal(want, linear_fp8(Fp8Blocks(tight(x8.q), x8.scale), Fp8Blocks(tight(w8.q), w8.scale)))
    assert torch.equal(linear_fp8(x8, w8, None, plan), linear_fp8(Fp8Blocks(tight(x8.q), x8.scale), w8, None, plan))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("T,count,K,N", [(3000, 3, 400, 700), (20000, 3, 136, 1000)])
def test_given_rows_equal_quantised_ones(dev, T, count, K, N, format):
    """Rows quantised on the way in (scales by block) and rows given with their scales by row: the same bits, also where pairs
    of SMs share a tile and where rows of no bucket are among them; and the dense product of the same rows."""
    from nnue_pytorch_b200 import GroupPlan, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    g = torch.Generator().manual_seed(31)
    x = (torch.randn(T, K, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).half().to(dev)
    w8 = quantize_fp8_tiles(torch.randn(count * N, K, generator=g).to(dev), count, format)
    b = torch.randint(-1, count, (T,), generator=g).to(dev)
    plan = GroupPlan(b, count)
    bias = torch.randn(count * N, generator=g).to(dev)
    y = linear_fp8(x, w8, bias, plan)
    assert torch.equal(y, linear_fp8(quantize_fp8_rows(x, format), w8, bias, plan, torch.float16))
    one = quantize_fp8_tiles(torch.randn(N, K, generator=g).to(dev), 1, format)
    d = linear_fp8(x, one, bias[:N])
    assert torch.equal(d, linear_fp8(quantize_fp8_rows(x, format), one, bias[:N], None, torch.float16))
    assert torch.equal(d, linear_fp8(x, one, bias[:N], GroupPlan(torch.zeros(T, dtype=torch.int32, device=dev), 1)))


def test_not_finite_rows(dev):
    from nnue_pytorch_b200 import GroupPlan, linear_fp8, quantize_fp8_tiles

    x = torch.randn(200, 256, device=dev)
    b = torch.randint(0, 4, (200,), device=dev)
    b[:20] = -1
    x[:20], x[50, 200] = float("nan"), float("nan")
    y = linear_fp8(x, quantize_fp8_tiles(torch.randn(4 * 40, 256, device=dev), 4), None, GroupPlan(b, 4))
    assert not y[:20].any() and torch.isnan(y[50]).all() and torch.isfinite(y[51:]).all() and torch.isfinite(y[20:50]).all()


def test_empty_batch(dev):
    from nnue_pytorch_b200 import GroupPlan, linear_fp8, quantize_fp8_tiles

    w8 = quantize_fp8_tiles(torch.randn(2 * 9, 40, device=dev), 2)
    x = torch.empty(0, 40, device=dev)
    assert linear_fp8(x, w8, None, GroupPlan(torch.empty(0, dtype=torch.int32, device=dev), 2)).shape == (0, 9)


def test_stream_and_replayed_graph(dev):
    from nnue_pytorch_b200 import GroupPlan, linear_fp8, quantize_fp8_tiles

    g = torch.Generator().manual_seed(6)
    w8 = quantize_fp8_tiles(torch.randn(4 * 200, 384, generator=g).to(dev), 4)
    data = [(torch.randn(300, 384, generator=g).bfloat16().to(dev), torch.randint(-1, 4, (300,), generator=g).to(dev)) for _ in range(2)]
    step = lambda x, b: linear_fp8(x, w8, None, GroupPlan(b, 4))  # noqa: E731
    want = [step(*d) for d in data]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = step(*data[0])
    side.synchronize()
    assert torch.equal(got, want[0])
    hold = [t.clone() for t in data[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*hold)
    for i in (1, 0):
        for h, t in zip(hold, data[i]):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    del graph
