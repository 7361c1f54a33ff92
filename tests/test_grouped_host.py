"""Host side of the bucketed and 8-bit operators, without a GPU: what the C entries are called with, and rules on the sources."""

import contextlib
import re
import types
from pathlib import Path

import pytest
import torch


class _Recorder:
    """In place of the native library: sizes that are large enough, and the arguments of every launch."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *args: 1 << 16
        return lambda *args: self.calls.setdefault(name, []).append(args) or 0


@pytest.fixture
def recorder(monkeypatch):
    """The operators on CPU tensors: their checks and their calls, no kernel."""
    from nnue_pytorch_b200 import fp8_functions, grouped_linear_functions

    lib = _Recorder()
    monkeypatch.setattr(grouped_linear_functions._lib, "load", lambda: lib)
    for module in (grouped_linear_functions, fp8_functions):
        monkeypatch.setattr(module, "_require_cuda", lambda *tensors: tensors[0].device)
        monkeypatch.setattr(module, "_on", lambda dev: contextlib.nullcontext())
        monkeypatch.setattr(module, "_stream", lambda dev: 0)
    return lib


def _plan(rows, count):
    return types.SimpleNamespace(rows=rows, count=count, buffer=torch.zeros(1 << 14, dtype=torch.int32), check=lambda t: None)


@pytest.mark.parametrize("rows", [4, 400])  # gathered, and laid out by bucket
@pytest.mark.parametrize("hooks", ["none", "contiguous", "columns"])
def test_backward_reads_the_weights_at_the_pitch_they_have(recorder, rows, hooks):
    """Saved-tensor hooks may give a column slice of the weights back with other strides than it was saved with."""
    from nnue_pytorch_b200 import grouped_linear

    count, N, K = 2, 8, 64
    x = torch.zeros(rows, K, dtype=torch.bfloat16, requires_grad=True)
    wide = torch.zeros(count * N, 2 * K, dtype=torch.bfloat16)
    seen = []

    def columns(t):  # column-major, where it is a matrix
        seen.append(t.t().contiguous().t() if t.dim() == 2 else t)
        return seen[-1]

    def tight(t):
        seen.append(t.contiguous().clone())
        return seen[-1]

    unpack = {"contiguous": tight, "columns": columns}.get(hooks)
    context = contextlib.nullcontext() if unpack is None else torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack)
    with context:
        y = grouped_linear(x, wide[:, :K], None, _plan(rows, count))
    assert recorder.calls["nnue_grouped_linear_fwd"][0][4] == 2 * K  # the slice itself was read
    y.backward(torch.zeros(rows, N, dtype=torch.bfloat16))
    address, pitch = recorder.calls["nnue_grouped_linear_bwd_input"][0][3:5]
    if hooks == "none":
        assert (address, pitch) == (wide.data_ptr(), 2 * K)
    elif hooks == "contiguous":
        assert address in [t.data_ptr() for t in seen] and pitch == K
    else:  # rows of one number next to each other: a copy of tight rows
        assert address not in [t.data_ptr() for t in seen] and pitch == K


def test_waits_for_tensor_memory_name_their_registers():
    """A wait without operands orders memory only: arithmetic on the registers that a read fills may move before it."""
    csrc = Path(__file__).parent.parent / "nnue_pytorch_b200" / "csrc"
    for name in ("tc.cuh", "grouped_tc.cuh", "grouped_linear.cu", "fp8_linear.cu"):
        source = (csrc / name).read_text()
        for wait in re.finditer(r'asm volatile\(\s*"tcgen05\.wait::ld[^;]*;"([^;]*);', source):
            named = wait.group(1).count('"+r"')
            assert named == 32, f"{name}: the wait for a read of 32 registers names {named}"
        assert "tmem_wait_ld()" not in source, name


def test_forward_mode_is_refused(recorder):
    """A dual tensor does not require a gradient; its tangent may not get lost, with gradients on or off."""
    from torch.autograd import forward_ad

    from nnue_pytorch_b200 import Fp8Blocks, grouped_linear, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    x, w, bias = torch.zeros(4, 64), torch.zeros(2 * 8, 64), torch.zeros(2 * 8)
    w8 = Fp8Blocks(torch.zeros(8, 64).to(torch.float8_e4m3fn), torch.ones(1, 1, 1))
    for mode in (contextlib.nullcontext, torch.no_grad):
        with mode(), forward_ad.dual_level():
            for i in range(3):
                args = [t.bfloat16() for t in (x, w, bias)]
                args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                assert not args[i].requires_grad
                with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                    grouped_linear(*args, _plan(4, 2))
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            for call in (lambda: quantize_fp8_rows(dual), lambda: quantize_fp8_tiles(dual), lambda: linear_fp8(dual, w8),
                         lambda: linear_fp8(x, w8, forward_ad.make_dual(bias[:8], bias[:8]))):
                with pytest.raises(AssertionError, match="no gradient"):
                    call()
            assert grouped_linear(x.bfloat16(), w.bfloat16(), None, _plan(4, 2)).shape == (4, 8)  # no tangent: as ever
            assert linear_fp8(x, w8).shape == (4, 8)


def test_rows_that_need_a_gradient_are_not_quantised(recorder):
    from nnue_pytorch_b200 import Fp8Blocks, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles

    x = torch.zeros(4, 64, requires_grad=True)
    with pytest.raises(AssertionError, match="no gradient"):
        quantize_fp8_rows(x)
    with torch.no_grad():
        assert quantize_fp8_rows(x).q.shape == (4, 64)
    blocks = quantize_fp8_tiles(torch.nn.Parameter(torch.zeros(4, 64)))  # weights are exported as constants
    assert not blocks.q.requires_grad and not blocks.scale.requires_grad
    with pytest.raises(AssertionError, match="no gradient"):  # scales of one's own
        linear_fp8(torch.zeros(4, 64), Fp8Blocks(blocks.q, torch.ones(1, 1, 1, requires_grad=True)))


def test_stream_of_a_device_without_an_index(monkeypatch):
    """`device_status` and others pass on the device they are given: without an index, a string, a number or none."""
    from nnue_pytorch_b200 import _launch

    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: types.SimpleNamespace(cuda_stream=("stream of", device)))
    assert _launch._stream(torch.device("cuda", 3)) == 103
    for device in (torch.device("cuda"), "cuda", "cuda:0", 0, None):
        assert _launch._stream(device) == ("stream of", device)
