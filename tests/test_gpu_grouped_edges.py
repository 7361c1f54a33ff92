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
