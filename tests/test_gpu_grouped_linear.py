"""Bucketed linear layer on 16-bit operands: the plan, the products and their gradients against 64-bit forms."""

import pytest
import torch

from _grouped_util import close, linear_ref, plan_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    return torch.device("cuda:0")


def _ids(T, count, seed, padding=False, skew=False):
    g = torch.Generator().manual_seed(seed)
    b = torch.randint(0, count, (T,), generator=g)
    if skew:
        b = torch.minimum(b, torch.randint(0, count, (T,), generator=g)) // 2
    if padding:
        b[torch.rand(T, generator=g) < 0.2] = -1
    return b


# ---- the plan
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("T,count", [(0, 3), (1, 1), (1, 1024), (31, 2), (32, 8), (33, 8), (1000, 257), (1025, 1024), (16384, 8),
                                     (2048, 3), (2049, 1024), (16385, 8), (40961, 5), (65536, 2), (65537, 700), (70000, 1024)])
def test_plan(dev, T, count, wide):
    from nnue_pytorch_b200 import GroupPlan

    b = _ids(T, count, T + count, padding=True, skew=count > 4)
    plan = GroupPlan(b.to(dev, torch.int64 if wide else torch.int32), count)
    order, offsets = plan_ref(b, count)
    assert torch.equal(plan.order.cpu(), order) and torch.equal(plan.offsets.cpu(), offsets)


def test_plan_of_one_bucket_and_of_padding_only(dev):
    from nnue_pytorch_b200 import GroupPlan

    for b, count in ((torch.full((5000,), 6), 8), (torch.full((300,), -1), 8), (torch.full((20000,), -1), 2)):
        plan = GroupPlan(b.to(dev), count)
        order, offsets = plan_ref(b, count)
        assert torch.equal(plan.order.cpu(), order) and torch.equal(plan.offsets.cpu(), offsets)


def test_plan_records_ids_out_of_range(dev):
    from nnue_pytorch_b200 import GroupPlan, _launch, _lib

    _launch.device_status(dev)
    for T in (100, 20000):
        b = _ids(T, 4, 1)
        b[7], b[50], b[99] = 4, -2, 1 << 40
        plan = GroupPlan(b.to(dev), 4)
        with pytest.raises(_lib.NnueB200Error, match="3 feature indices"):
            _launch.device_status(dev)
        order, offsets = plan_ref(b, 4)
        assert torch.equal(plan.order.cpu(), order) and torch.equal(plan.offsets.cpu(), offsets)
        _launch.device_status(dev)


# ---- the products
CASES = [
    # T, count, K, N
    (1, 1, 1, 1), (1, 8, 64, 32), (2, 3, 17, 5), (5, 2, 8, 1), (40, 8, 100, 1), (127, 1, 64, 31), (128, 1, 128, 128), (129, 1, 130, 129),
    (300, 3, 96, 200), (257, 64, 72, 40), (1000, 8, 1000, 32), (700, 5, 264, 520), (64, 70, 520, 33), (3, 1, 4099, 260),
    (2000, 2, 40, 300), (515, 4, 1032, 257),
    # more tiles than SMs, in every direction
    (9000, 8, 256, 2100), (24000, 3, 1000, 520), (5000, 40, 520, 520),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,count,K,N", CASES)
def test_forward_and_gradients(dev, T, count, K, N, dtype):
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(T * 7 + K)
    b = _ids(T, count, K + N, padding=T > 4, skew=count > 3)
    x = torch.randn(T, K, generator=g).to(dtype)
    master = (T + K) % 2 == 0
    w = torch.randn(count * N, K, generator=g) / K**0.5
    bias = torch.randn(count * N, generator=g)
    if not master:
        w, bias = w.to(dtype), bias.to(dtype)
    dy = torch.randn(T, N, generator=g).to(dtype)
    ref = linear_ref(x, w.to(dtype), bias, b, count, dy)
    xd, wd, bd = (t.to(dev).requires_grad_(True) for t in (x, w, bias))
    plan = GroupPlan(b.to(dev), count)
    y = grouped_linear(xd, wd, bd, plan)
    assert y.dtype == dtype
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(dev))
    assert dx.dtype == dtype and dw.dtype == w.dtype and db.dtype == bias.dtype
    for name, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        close(t, *ref[name], name)
    # rows of no bucket: exact zeros
    none = b < 0
    assert not y.detach().cpu()[none].any() and not dx.cpu()[none].any()
    # the same bits again
    y2 = grouped_linear(xd, wd, bd, plan)
    again = torch.autograd.grad(y2, (xd, wd, bd), dy.to(dev))
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("K,N", [(64, 48), (33, 7)])
def test_fp32_output_and_no_bias(dev, K, N):
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(3)
    T, count = 200, 4
    b = _ids(T, count, 5, padding=True)
    x = torch.randn(T, K, generator=g).bfloat16()
    w = torch.randn(count, N, K, generator=g).bfloat16()
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = grouped_linear(xd, wd, None, GroupPlan(b.to(dev), count), out_dtype=torch.float32)
    assert y.dtype == torch.float32
    dy = torch.randn(T, N, generator=g)
    y.backward(dy.to(dev))
    assert wd.grad.shape == w.shape
    ref = linear_ref(x, w, None, b, count, dy.bfloat16())
    close(y, *ref["y"], "y")
    close(xd.grad, *ref["dx"], "dx")
    close(wd.grad.view(-1, K), *ref["dw"], "dw")


def test_each_gradient_alone(dev):
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(13)
    for T in (20, 700):  # few rows per bucket, and many
        count, K, N = 4, 96, 72
        b = _ids(T, count, T, padding=True)
        x = torch.randn(T, K, generator=g).half()
        w, bias = torch.randn(count * N, K, generator=g).half(), torch.randn(count * N, generator=g).half()
        dy = torch.randn(T, N, generator=g).half()
        ref = linear_ref(x, w, bias, b, count, dy)
        plan = GroupPlan(b.to(dev), count)
        for i, name in enumerate(("dx", "dw", "db")):
            ts = [t.to(dev).requires_grad_(i == j) for j, t in enumerate((x, w, bias))]
            y = grouped_linear(*ts, plan)
            y.backward(dy.to(dev))
            close(y, *ref["y"], "y")
            close(ts[i].grad, *ref[name], name)
            assert all(t.grad is None for j, t in enumerate(ts) if j != i)


def test_strides_and_alignments(dev):
    """Column slices at every offset, transposed and expanded operands."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(4)
    T, count, K, N = 150, 3, 48, 40
    b = _ids(T, count, 6, padding=True)
    plan = GroupPlan(b.to(dev), count)
    wide = torch.randn(T, 2 * K, generator=g).bfloat16().to(dev)
    w = torch.randn(count * N, 2 * K, generator=g).bfloat16().to(dev)
    for off in (0, 1, 2, 5, 8):
        x, ws = wide[:, off : off + K].detach().requires_grad_(True), w[:, off : off + K].detach().requires_grad_(True)
        y = grouped_linear(x, ws, None, plan)
        dyt = torch.randn(N, T, generator=g).bfloat16().to(dev).t()
        dx, dw = torch.autograd.grad(y, (x, ws), dyt)
        ref = linear_ref(x, ws, None, b, count, dyt)
        close(y, *ref["y"], f"y at {off}")
        close(dx, *ref["dx"], f"dx at {off}")
        close(dw, *ref["dw"], f"dw at {off}")
    xt = torch.randn(K, T, generator=g).bfloat16().to(dev).t()
    wt = torch.randn(K, count * N, generator=g).bfloat16().to(dev).t()
    close(grouped_linear(xt, wt, None, plan), *linear_ref(xt, wt, None, b, count)["y"], "transposed")
    one = torch.randn(1, K, generator=g).bfloat16().to(dev).expand(T, K)
    close(grouped_linear(one, wt, None, plan), *linear_ref(one, wt, None, b, count)["y"], "expanded")
    x = wide[:, :K].detach().requires_grad_(True)
    grouped_linear(x, wt, None, plan).sum().backward()  # an expanded gradient
    close(x.grad, *linear_ref(x, wt, None, b, count, torch.ones(T, N))["dx"], "dx of a sum")


def test_one_row_of_any_stride(dev):
    """A single row's own stride says nothing: a transposed column has 1."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(21)
    plan = GroupPlan(torch.ones(1, dtype=torch.int64, device=dev), 2)
    for K, N in ((64, 8), (33, 5)):
        x = torch.randn(K, 1, generator=g).bfloat16().to(dev).t()
        w = torch.randn(2 * N, K, generator=g).to(dev).requires_grad_(True)
        dy = torch.randn(N, 1, generator=g).bfloat16().to(dev).t()
        assert x.stride(0) == 1 and dy.stride(0) == 1
        b = torch.ones(1, dtype=torch.int64)
        ref = linear_ref(x, w.detach().bfloat16(), None, b, 2, dy)
        with torch.no_grad():
            close(grouped_linear(x, w, None, plan), *ref["y"], "y")
        xg = x.detach().requires_grad_(True)
        y = grouped_linear(xg, w, None, plan)
        dx, dw = torch.autograd.grad(y, (xg, w), dy)
        close(y, *ref["y"], "y")
        close(dx, *ref["dx"], "dx")
        close(dw, *ref["dw"], "dw")
    w1 = torch.randn(64, 1, generator=g).bfloat16().to(dev).t()  # one output: a weight matrix of one row
    one = GroupPlan(torch.zeros(3, dtype=torch.int64, device=dev), 1)
    x = torch.randn(3, 64, generator=g).bfloat16().to(dev)
    close(grouped_linear(x, w1, None, one), *linear_ref(x, w1, None, torch.zeros(3, dtype=torch.int64), 1)["y"], "one output")


def test_inside_a_compiled_model(dev):
    """The calls run eagerly inside a function that torch.compile traces, with their gradients."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(22)
    b = _ids(200, 4, 22, padding=True).to(dev)
    plan = GroupPlan(b, 4)
    x = torch.randn(200, 48, generator=g).bfloat16().to(dev).requires_grad_(True)
    w = torch.randn(4 * 24, 48, generator=g).to(dev).requires_grad_(True)

    def layer(x, w):
        return grouped_linear(x * 2, w, None, plan).clamp(0, 1) * 3

    want = layer(x, w)
    got = torch.compile(layer, backend="eager")(x, w)
    assert torch.equal(want, got)
    for p, q in zip(torch.autograd.grad(want.sum(), (x, w)), torch.autograd.grad(got.sum(), (x, w))):
        assert torch.equal(p, q)


def test_trained_layers_then_evaluated_in_8_bits(dev):
    """One plan through two bucketed layers, forward and backward, then the same layers exported to 8 bits.

    With dyadic inputs (multiples of 1/4 of at most 1, weights of -1, 0, 1 over 8, few terms) every sum and every rounding
    on the way is exact, in 16 and in 8 bits: both paths have to equal the 64-bit network to the bit."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear, linear_fp8, quantize_fp8_tiles

    g = torch.Generator().manual_seed(23)
    T, count, K, H, N = 5000, 8, 160, 40, 16
    b = _ids(T, count, 23, padding=True)
    x = torch.randint(0, 5, (T, K), generator=g) / 4 * (torch.rand(T, K, generator=g) < 0.05)
    w1 = torch.randint(-1, 2, (count * H, K), generator=g) / 4.0
    w2 = torch.randint(-1, 2, (count * N, H), generator=g) / 4.0
    plan = GroupPlan(b.to(dev), count)
    clip = lambda t: (t * 4).round().clamp(0, 4) / 4  # noqa: E731  an activation on the same quarters

    h64 = clip(linear_ref(x, w1, None, b, count)["y"][0])
    ref = linear_ref(h64, w2, None, b, count, torch.ones(T, N))
    xd = x.bfloat16().to(dev)
    w1d, w2d = w1.to(dev), w2.to(dev).requires_grad_(True)
    h = clip(grouped_linear(xd, w1d, None, plan))
    assert torch.equal(h.cpu().double(), h64)
    y = grouped_linear(h, w2d, None, plan, out_dtype=torch.float32)
    assert torch.equal(y.detach().cpu().double(), ref["y"][0])
    dw, = torch.autograd.grad(y.sum(), w2d)
    assert torch.equal(dw.cpu().double(), ref["dw"][0])
    with torch.no_grad():
        a = clip(linear_fp8(xd, quantize_fp8_tiles(w1d, count), None, plan))
        assert torch.equal(a, h)
        e = linear_fp8(a, quantize_fp8_tiles(w2d, count), None, plan, out_dtype=torch.float32)
    assert torch.equal(e, y.detach())


def test_not_finite_values_stay_where_they_are(dev):
    """NaN and infinities in padding rows reach nothing; in a row they reach that row, in a bucket that bucket."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(8)
    T, count, K, N = 300, 5, 72, 24
    b = _ids(T, count, 9, padding=True)
    b[3], b[b == 4] = -1, 2
    x = torch.randn(T, K, generator=g)
    dy = torch.randn(T, N, generator=g)
    clean = linear_ref(x.half(), torch.ones(count * N, K).half(), None, b, count, dy.half())
    x[b < 0], dy[b < 0] = float("nan"), float("inf")
    xd = x.half().to(dev).requires_grad_(True)
    wd = torch.ones(count * N, K, dtype=torch.float16, device=dev, requires_grad=True)
    bd = torch.zeros(count * N, dtype=torch.float16, device=dev, requires_grad=True)
    plan = GroupPlan(b.to(dev), count)
    y = grouped_linear(xd, wd, bd, plan)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.half().to(dev))
    for name, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        close(t, *clean[name], name)
    assert not dw.view(count, -1)[4].any() and not db.view(count, -1)[4].any()  # the empty bucket
    row = int(torch.nonzero(b == 1)[0])
    x[row] = float("inf")
    y = grouped_linear(x.half().to(dev), wd.detach(), bd.detach(), plan).cpu()
    assert torch.isinf(y[row]).all()
    keep = torch.arange(T) != row
    assert torch.isfinite(y[keep]).all()
    wn = wd.detach().clone()
    wn[2 * N] = float("nan")  # first output of bucket 2
    y = grouped_linear(torch.zeros(T, K, dtype=torch.float16, device=dev), wn, None, plan).cpu()
    assert torch.equal(torch.isnan(y), (b == 2)[:, None] & (torch.arange(N) == 0))


def test_empty_batch(dev):
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    x = torch.empty(0, 16, dtype=torch.bfloat16, device=dev, requires_grad=True)
    w = torch.randn(3 * 8, 16, device=dev, requires_grad=True)
    b = torch.randn(3 * 8, device=dev, requires_grad=True)
    y = grouped_linear(x, w, b, GroupPlan(torch.empty(0, dtype=torch.int64, device=dev), 3))
    assert y.shape == (0, 8)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == w.shape and db.shape == b.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_against_differences(dev, dtype):
    """The layer is linear in x, in the weights and in the bias, so f(v + d) - f(v) = f'(v) d exactly; with whole-number
    inputs every value below 2^8 and every sum is exact in fp32, and <dy, f(v + d) - f(v)> = <gradient, d> holds to the bit."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(10)
    T, count, K, N = 90, 4, 40, 24
    b = _ids(T, count, 11, padding=True)
    plan = GroupPlan(b.to(dev), count)

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=g).float().to(dev)

    x, w, bias, dy = whole(T, K), whole(count * N, K), whole(count * N), whole(T, N)
    xd, wd, bd = x.to(dtype).requires_grad_(True), w.clone().requires_grad_(True), bias.clone().requires_grad_(True)
    y = grouped_linear(xd, wd, bd, plan, out_dtype=torch.float32)
    grads = torch.autograd.grad(y, (xd, wd, bd), dy)
    for i, base in enumerate((x, w, bias)):
        for _ in range(3):
            d = torch.zeros_like(base)
            d.view(-1)[torch.randint(0, d.numel(), (5,), generator=g).to(dev)] = 1.0
            moved = [x, w, bias]
            moved[i] = base + d
            diff = grouped_linear(moved[0].to(dtype), moved[1], moved[2], plan, out_dtype=torch.float32) - y.detach()
            # dx is rounded to 16 bits: whole numbers below 2^8 survive that
            assert grads[i].abs().max() < 256 or grads[i].dtype == torch.float32
            assert float((dy.double() * diff.double()).sum()) == float((grads[i].double() * d.double()).sum())


def test_other_stream_and_replayed_graph(dev):
    """Forward and backward on a side stream, then captured once and replayed on other inputs."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    T, count, K, N = 260, 4, 96, 64

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        return (_ids(T, count, seed, padding=True).to(dev), torch.randn(T, K, generator=g).bfloat16().to(dev),
                torch.randn(count * N, K, generator=g).to(dev), torch.randn(count * N, generator=g).to(dev),
                torch.randn(T, N, generator=g).bfloat16().to(dev))

    def step(b, x, w, bias, dy):
        x, w, bias = (t.detach().requires_grad_(True) for t in (x, w, bias))
        y = grouped_linear(x, w, bias, GroupPlan(b, count))
        return (y.detach(), *torch.autograd.grad(y, (x, w, bias), dy))

    want = [step(*inputs(s)) for s in (1, 2)]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = step(*inputs(1))
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want[0], got))
    hold = [t.clone() for t in inputs(1)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(*hold)
    for s in (2, 1):
        for h, t in zip(hold, inputs(s)):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want[s - 1], out))
    del graph


def test_from_threads_of_their_own(dev):
    """Threads that have made no CUDA call yet (as autograd's are), two at a time."""
    import threading

    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(12)
    b = _ids(256, 4, 12).to(dev)
    x, w = torch.randn(256, 64, generator=g).bfloat16().to(dev), torch.randn(4 * 64, 64, generator=g).bfloat16().to(dev)
    plan = GroupPlan(b, 4)
    want = grouped_linear(x, w, None, plan)
    got = [None, None]

    def work(i):
        with torch.no_grad():
            got[i] = [grouped_linear(x, w, None, plan) for _ in range(20)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(y, want) for ys in got for y in ys)


def test_offsets_beyond_32_bits(dev):
    """x and y of more than 2^31 numbers; the last rows are looked at."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    T, K, N, count = 1 << 20, 2056, 16, 2
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    x[-200:] = torch.randn(200, K, generator=g, device=dev).bfloat16()
    b = (torch.arange(T, device=dev) >= T - 77).long()
    w = torch.randn(count * N, K, generator=g, device=dev).bfloat16()
    y = grouped_linear(x, w, None, GroupPlan(b, count))
    assert not y[:-200].any()
    close(y[-200:], *linear_ref(x[-200:], w, None, b[-200:], count)["y"], "y")
    del y
    wide = torch.randn(count * K, 16, generator=g, device=dev).bfloat16()
    y = grouped_linear(x[:, :16], wide, None, GroupPlan(b, count))  # the output is the large one, rows pitched
    close(y[-200:], *linear_ref(x[-200:, :16], wide, None, b[-200:], count)["y"], "wide y")
