"""Bucketed linear layer where a call is allowed and out of the ordinary, against 64-bit forms."""

import pytest
import torch

from _grouped_util import close, linear_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("T", [20, 700])  # gathered, and laid out by bucket
def test_saved_tensors_kept_on_the_host(dev, T):
    """`save_on_cpu` gives tensors back without the strides they were saved with: a column slice of the weights, rows of any
    stride, the plan."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator().manual_seed(41)
    count, K, N = 4, 64, 40
    b = torch.randint(-1, count, (T,), generator=g)
    wide = torch.randn(count * N, 2 * K, generator=g).bfloat16().to(dev)
    rows = torch.randn(T, 2 * K, generator=g).bfloat16().to(dev)
    dy = torch.randn(T, N, generator=g).bfloat16()
    plan = GroupPlan(b.to(dev), count)
    for train_weights in (False, True):
        x, w = rows[:, K:].detach().requires_grad_(True), wide[:, :K].detach().requires_grad_(train_weights)
        with torch.autograd.graph.save_on_cpu():
            y = grouped_linear(x, w, None, plan)
        y.backward(dy.to(dev))
        ref = linear_ref(x, w, None, b, count, dy)
        close(y, *ref["y"], "y")
        close(x.grad, *ref["dx"], "dx")
        if train_weights:
            close(w.grad, *ref["dw"], "dw")


# ---- accuracy of long sums.  One addition of the tensor core takes 16 terms: each loses what lies below a quarter of the
# last bit of the largest, their sum what lies below its own last bit, together less than 5 * 2^-23 of the sum.  A run of 512
# terms of one sign is 32 additions to partial sums that are no larger than the run.  Runs are added rounding to nearest, at
# most 2^-24 of the sum each, and where a sum is split over ranks, up to 8 additions more.
def _long_sum_bound(terms):
    return 32 * 5 * 2.0**-23 + (-(-terms // 512) + 8) * 2.0**-24


def _near(ours, ref, terms, what):
    bound = ref.abs() * _long_sum_bound(terms)
    if ours.dtype != torch.float32:
        bound += (ref.abs() + bound) * (torch.finfo(ours.dtype).eps / 2)
    off = (ours.double() - ref).abs()
    assert (off <= bound).all(), f"{what}: off by {float((off / ref.abs()).max()):.3e} of the sum, allowed {float((bound / ref.abs()).max()):.3e}"


def _one_sign(g, dev, *shape):
    return (torch.rand(*shape, generator=g, device=dev) * 0.5 + 0.25).bfloat16()


@pytest.mark.parametrize("T,K,N", [(60, 16384, 40), (300, 16384, 1000), (2500, 8192, 2100), (20000, 8192, 200)])
def test_long_sums_of_the_forward_in_fp32(dev, T, K, N):
    """One, several and all-SM tiles, single CTAs and pairs."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator(device=dev).manual_seed(51)
    x, w = _one_sign(g, dev, T, K), _one_sign(g, dev, N, K)
    plan = GroupPlan(torch.zeros(T, dtype=torch.int64, device=dev), 1)
    _near(grouped_linear(x, w, None, plan, out_dtype=torch.float32), x.double() @ w.double().T, K, "y")


@pytest.mark.parametrize("K,N", [(64, 40), (2048, 200), (1280, 2100)])  # split sums, single CTAs, pairs
def test_long_sums_of_the_weight_gradient_in_fp32(dev, K, N):
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    T = 16000
    g = torch.Generator(device=dev).manual_seed(52)
    x, dy = _one_sign(g, dev, T, K), _one_sign(g, dev, T, N)
    w = torch.zeros(N, K, device=dev, requires_grad=True)
    y = grouped_linear(x, w, None, GroupPlan(torch.zeros(T, dtype=torch.int64, device=dev), 1))
    dw, = torch.autograd.grad(y, w, dy)
    _near(dw, dy.double().T @ x.double(), T, "dw")


@pytest.mark.parametrize("direction", ["y", "dx", "dw"])
def test_very_long_sums_in_16_bits(dev, direction):
    """2^20 terms: what is cut off may not outgrow the one rounding to fp16."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator(device=dev).manual_seed(53)
    long, T, K, N = 1 << 20, 48, 16, 24
    T, K, N = {"y": (T, long, N), "dx": (T, K, long), "dw": (long, K, N)}[direction]
    small = 2.0**-8  # 2^20 products near 1/4 stay within fp16
    x, w, dy = ((_one_sign(g, dev, *s) * small).half().requires_grad_(True) for s in ((T, K), (N, K), (T, N)))
    if direction == "y":
        y = grouped_linear(x.detach(), w.detach() / small, None, GroupPlan(torch.zeros(T, dtype=torch.int64, device=dev), 1))
        _near(y, x.detach().double() @ (w.detach() / small).double().T, long, "y")
        return
    y = grouped_linear(x, w, None, GroupPlan(torch.zeros(T, dtype=torch.int64, device=dev), 1))
    if direction == "dx":
        dx, = torch.autograd.grad(y, x, dy.detach() / small)
        _near(dx, (dy.detach() / small).double() @ w.detach().double(), long, "dx")
    else:
        dw, = torch.autograd.grad(y, w, dy.detach() / small)
        _near(dw, (dy.detach() / small).double().T @ x.detach().double(), long, "dw")


def test_status_of_a_device_without_an_index(dev):
    from nnue_pytorch_b200 import _launch

    for device in (None, torch.device("cuda"), "cuda", "cuda:0", 0):
        _launch.device_status(device)
        assert _launch._stream(device) == torch.cuda.current_stream(device).cuda_stream
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        assert _launch._stream(torch.device("cuda")) == _launch._stream(dev) == side.cuda_stream


# Tiles of every width, of one CTA and of pairs, split and whole, in each direction: (rows, buckets, inputs, outputs), and the
# columns of the tiles that 148 SMs get in forward, dx and dw.
FORMS = [
    (24000, 8, 512, 1000),  # pairs, pairs, 128
    (3000, 8, 2560, 264),  # 32, pairs, pairs
    (4000, 40, 1000, 1000),  # 256, 256, pairs
    (3000, 40, 1000, 100),  # 32, 256, 256
    (2000, 20, 1000, 1000),  # 128, 128, pairs
    (3000, 20, 1000, 100),  # 32, pairs, 128
    (1000, 10, 1000, 1000),  # 64, 64, pairs
    (800, 8, 1000, 600),  # 32, 64, pairs
    (3000, 8, 1000, 100),  # 32, 128, 64
    (12000, 3, 4096, 72),  # 64, pairs, 64
    (3000, 2, 300, 40),  # 32 split in 2, 64, 64 split in 8
    (100, 2, 300, 600),  # 32 split in 2, 64 split in 4, 64
]


@pytest.mark.parametrize("weights", ["own", "fp32"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,count,K,N", FORMS)
def test_whole_numbers_in_every_form(dev, T, count, K, N, dtype, weights):
    """Whole numbers of at most 2 in size: no sum reaches 2^24, so every sum is exact in fp32, in any order and where
    additions cut off, and each result is the 64-bit one rounded once."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator(device=dev).manual_seed(T + K + N)
    whole = lambda *shape: torch.randint(-2, 3, shape, generator=g, device=dev).float()  # noqa: E731
    x, w, bias, dy = whole(T, K), whole(count * N, K), whole(count * N), whole(T, N)
    b = torch.randint(-1, count, (T,), generator=g, device=dev)
    w_dtype = torch.float32 if weights == "fp32" else dtype
    xd, wd, bd = x.to(dtype).requires_grad_(True), w.to(w_dtype).requires_grad_(True), bias.to(w_dtype).requires_grad_(True)
    y = grouped_linear(xd, wd, bd, GroupPlan(b, count))
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(dtype))
    y32 = grouped_linear(xd.detach(), wd.detach(), bd.detach(), GroupPlan(b, count), out_dtype=torch.float32)
    x, w, dy = x.double(), w.double().view(count, N, K), dy.double()
    for e in range(count):
        r = torch.nonzero(b == e).view(-1)
        ref = x[r] @ w[e].T + bias.view(count, N)[e].double()
        assert torch.equal(y[r], ref.to(dtype)) and torch.equal(y32[r].double(), ref), f"y of bucket {e}"
        assert torch.equal(dx[r], (dy[r] @ w[e]).to(dtype)), f"dx of bucket {e}"
        assert torch.equal(dw.view(count, N, K)[e], (dy[r].T @ x[r]).to(w_dtype)), f"dw of bucket {e}"
        assert torch.equal(db.view(count, N)[e], dy[r].sum(0).to(w_dtype)), f"dbias of bucket {e}"
    none = b < 0
    assert not y[none].any() and not y32[none].any() and not dx[none].any()


def test_plan_and_8_bit_layer_inside_a_compiled_model(dev):
    """A plan depends on the batch, so a compiled model makes its own; the 8-bit layer runs in one too."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear, linear_fp8, quantize_fp8_tiles

    g = torch.Generator().manual_seed(61)
    count, K, N = 4, 48, 24
    w = torch.randn(count * N, K, generator=g).to(dev).requires_grad_(True)
    w8 = quantize_fp8_tiles(w, count)

    def train(x, b, w):
        return grouped_linear(x * 2, w, None, GroupPlan(b, count)).clamp(0, 1) * 3

    def evaluate(x, b):
        return linear_fp8(x * 2, w8, None, GroupPlan(b, count)).clamp(0, 1) * 3

    compiled = torch.compile(train, backend="eager"), torch.compile(evaluate, backend="eager")
    for T in (200, 200, 37):  # the second batch runs what the first compiled, the third has another length
        b = torch.randint(-1, count, (T,), generator=g).to(dev)
        x = torch.randn(T, K, generator=g).bfloat16().to(dev).requires_grad_(True)
        want, got = train(x, b, w), compiled[0](x, b, w)
        assert torch.equal(want, got)
        for p, q in zip(torch.autograd.grad(want.sum(), (x, w)), torch.autograd.grad(got.sum(), (x, w))):
            assert torch.equal(p, q)
        with torch.no_grad():
            assert torch.equal(evaluate(x, b), compiled[1](x, b))


def test_two_captured_graphs_replayed_in_any_order(dev):
    """Two graphs of one process, each with a plan, both directions and the 8-bit layer, replayed in turn and side by side on
    two streams: they share no buffer."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear, linear_fp8, quantize_fp8_tiles

    def inputs(T, count, K, N, seed):
        g = torch.Generator().manual_seed(seed)
        return (torch.randint(-1, count, (T,), generator=g).to(dev), torch.randn(T, K, generator=g).bfloat16().to(dev),
                torch.randn(count * N, K, generator=g).to(dev), torch.randn(T, N, generator=g).bfloat16().to(dev), count)

    def step(b, x, w, dy, count):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        plan = GroupPlan(b, count)
        y = grouped_linear(x, w, None, plan)
        out = (y.detach(), *torch.autograd.grad(y, (x, w), dy))
        with torch.no_grad():
            return (*out, linear_fp8(x, quantize_fp8_tiles(w, count), None, plan))

    data = [inputs(3000, 3, 256, 300, 71), inputs(900, 8, 320, 96, 72)]
    want = [step(*d) for d in data]
    graphs, outs = [], []
    for d in data:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*d))
        graphs.append(graph)
    streams = [torch.cuda.Stream(dev) for _ in data]
    for order in ((0, 1), (1, 0), (0, 0), (1, 1)):
        for t in (t for o in outs for t in o):
            t.fill_(7)
        torch.cuda.synchronize()
        for i in order:
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in set(order):
            assert all(torch.equal(p, q) for p, q in zip(want[i], outs[i]))
    del graphs


@pytest.mark.parametrize("T", [30, 3000])
def test_broadcast_weights_and_repeated_leaves(dev, T):
    """One matrix expanded over all buckets, its gradient the sum over them; the same layer twice in a graph; checkpointed."""
    from torch.utils.checkpoint import checkpoint

    from nnue_pytorch_b200 import GroupPlan, grouped_linear

    g = torch.Generator(device=dev).manual_seed(81)
    count, K = 5, 72
    whole = lambda *shape: torch.randint(-1, 2, shape, generator=g, device=dev).float()  # noqa: E731
    b = torch.randint(-1, count, (T,), generator=g, device=dev)
    plan = GroupPlan(b, count)
    x = (whole(T, K) * (torch.rand(T, K, generator=g, device=dev) < 0.1)).bfloat16().requires_grad_(True)
    one = whole(K, K).requires_grad_(True)
    dy = whole(T, K).bfloat16()

    def twice(x, one):
        w = one.expand(count, K, K)
        return grouped_linear(grouped_linear(x, w, None, plan), w, None, plan, out_dtype=torch.float32)

    live = (b >= 0).double()[:, None]
    h = (x.detach().double() @ one.detach().double().T) * live
    want = (h @ one.detach().double().T) * live
    dh = (dy.double() * live) @ one.detach().double()
    assert h.abs().max() < 256 and dh.abs().max() < 256  # exact in bf16 on the way
    dx, dw = dh @ one.detach().double() * live, (dy.double() * live).T @ h + dh.T @ (x.detach().double() * live)
    for run in (twice, lambda x, one: checkpoint(twice, x, one, use_reentrant=False)):
        y = run(x, one)
        got = torch.autograd.grad(y, (x, one), dy.float())
        assert torch.equal(y.double(), want)
        assert torch.equal(got[0], dx.bfloat16()) and torch.equal(got[1].double(), dw)


# ---- offsets beyond 32 bits and many rows
@pytest.mark.parametrize("T,count", [(3_000_001, 1000), (20_000_000, 7)])
def test_plan_of_many_rows(dev, T, count):
    from nnue_pytorch_b200 import GroupPlan

    g = torch.Generator(device=dev).manual_seed(91)
    b = torch.randint(-1, count, (T,), generator=g, device=dev)
    plan = GroupPlan(b, count)
    key = torch.where(b < 0, count, b)
    assert torch.equal(plan.order.long(), torch.sort(key, stable=True).indices)
    sizes = torch.bincount(key, minlength=count + 1)
    assert torch.equal(plan.offsets.long(), torch.cat([sizes.new_zeros(1), sizes[:count].cumsum(0)]))


def test_weights_and_gradients_of_more_than_2_31_numbers(dev):
    """1024 matrices of 2056 x 1024, in 16 and in 8 bits; rows of the first, a middle and the last bucket."""
    from nnue_pytorch_b200 import GroupPlan, grouped_linear, linear_fp8, quantize_fp8_tiles

    count, N, K, T = 1024, 2056, 1024, 96
    g = torch.Generator(device=dev).manual_seed(92)
    some = torch.tensor([0, 500, 1023], device=dev)
    whole = lambda *shape: torch.randint(-2, 3, shape, generator=g, device=dev)  # noqa: E731
    w = torch.zeros(count, N, K, dtype=torch.bfloat16, device=dev)
    w[some] = whole(3, N, K).bfloat16()
    w.requires_grad_(True)
    b = some.repeat(T // 3)
    x, dy = whole(T, K).bfloat16().requires_grad_(True), whole(T, N).bfloat16()
    y = grouped_linear(x, w, None, GroupPlan(b, count))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        y8 = linear_fp8(x, quantize_fp8_tiles(w.flatten(0, 1), count), None, GroupPlan(b, count), torch.float32)
        for e in some.tolist():
            r = torch.nonzero(b == e).view(-1)
            ref = x[r].double() @ w[e].double().T
            assert torch.equal(y[r], ref.bfloat16()) and torch.equal(y8[r].double(), ref)  # quantising whole numbers is exact
            assert torch.equal(dx[r], (dy[r].double() @ w[e].double()).bfloat16())
            assert torch.equal(dw[e], (dy[r].double().T @ x[r].double()).bfloat16())
        assert not dw[1:500].any() and not dw[501:1023].any()


@pytest.mark.parametrize("dense", [False, True])
def test_8_bit_rows_of_more_than_2_31_numbers(dev, dense):
    from nnue_pytorch_b200 import GroupPlan, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    T, K, N = 1 << 20, 2064, 16
    count = 1 if dense else 2
    g = torch.Generator(device=dev).manual_seed(93)
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=dev)
    x[-200:] = torch.randint(-2, 3, (200, K), generator=g, device=dev).bfloat16()
    w = torch.randint(-2, 3, (count * N, K), generator=g, device=dev).bfloat16()
    b = (torch.arange(T, device=dev) >= T - 77).long() if not dense else torch.zeros(T, dtype=torch.int64, device=dev)
    w8, plan = quantize_fp8_tiles(w, count), None if dense else GroupPlan(b, count)
    want = torch.stack([x[p].double() @ w.view(count, N, K)[b[p]].double().T for p in range(T - 200, T)])
    for rows in (x, quantize_fp8_rows(x)):
        y = linear_fp8(rows, w8, None, plan, torch.float32)
        assert not y[:-200].any() and torch.equal(y[-200:].double(), want)
        del y
    wide = torch.randint(-2, 3, (count * K, 16), generator=g, device=dev).bfloat16()  # the output is the large one
    y = linear_fp8(x[:, -16:].contiguous(), quantize_fp8_tiles(wide, count), None, plan)
    want = torch.stack([x[p, -16:].double() @ wide.view(count, K, 16)[b[p]].double().T for p in range(T - 200, T)])
    assert not y[:-200].any() and torch.equal(y[-200:], want.bfloat16())
