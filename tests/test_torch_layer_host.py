"""The torch side of the 4-bit layer and of orthogonalised updates where no GPU is needed: what is recorded by a
trace, what forward-mode differentiation is told, which stream a call names, what the optimiser keeps.  The
library's entries are replaced by stand-ins that write through the raw pointer, as the kernels do, so that nothing torch
could see or record happens in them."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import cake_on_cpu_amd as cake
from cake_on_cpu_amd import _lib, api
from cake_on_cpu_amd import torch_linear as tl

pytestmark = pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")

N, K = 5, 8


def _at(t, n):
    return np.ctypeslib.as_array((ctypes.c_float * n).from_address(t.data_ptr()))


def _packed(values):
    """Stand-in weights: the first byte says by what the sum of a row of x is multiplied."""
    data = torch.zeros(cake.q4_size(N, K, 32), dtype=torch.uint8)
    data[0] = values
    return data


@pytest.fixture
def stand_in(monkeypatch):
    def linear(x, q, bias, y, M, workspace=None, timed=True):
        out = _at(y, M * q.N).reshape(M, q.N)
        out[:] = _at(x, M * q.K).reshape(M, q.K).sum(1, keepdims=True) * int(q.data.flatten()[0])
        if bias is not None:
            out += _at(bias, q.N)

    monkeypatch.setattr(api, "linear_q4_forward", linear)


def _layer(values, bias):
    return tl.cake_linear_q4(cake.q4_of(_packed(values), N, K, 32, "float32", False), torch.arange(float(N)) if bias else None)


def test_a_tangent_is_not_dropped(stand_in):
    """Forward mode has no formula here and says so, also where nothing requires a gradient."""
    import torch.autograd.forward_ad as fa
    q, x = cake.q4_of(_packed(3), N, K, 32, "float32", False), torch.randn(2, K)
    layer = _layer(3, True)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fa.dual_level():
            dual = fa.make_dual(x, torch.ones_like(x))
            for call in (lambda: tl.forward_q4(dual, q), lambda: layer(dual), lambda: tl.forward_q4(x, q, fa.make_dual(torch.ones(N), torch.ones(N)))):
                with pytest.raises(NotImplementedError):
                    call()
            assert torch.equal(tl.forward_q4(x, q), tl.forward_q4(x.clone(), q))      # without a tangent it is a call like any other
    for transform in (lambda: torch.func.jvp(lambda v: tl.forward_q4(v, q), (x,), (x,)), lambda: torch.func.vmap(lambda v: tl.forward_q4(v, q))(x[None])):
        with pytest.raises(RuntimeError):
            transform()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_a_traced_layer_computes(stand_in, bias, grad):
    """A trace records the layer itself, not the memory of the result it had then."""
    gen = torch.Generator().manual_seed(1)
    layer, x = _layer(3, bias), torch.randn(2, 3, K, generator=gen)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(layer, (x,), check_trace=False)
        alone = torch.jit.trace(lambda v: tl.forward_q4(v, layer.weight_q4), (x[0],), check_trace=False)
        for rows in (3, 3, 5):
            x = torch.randn(2, rows, K, generator=gen)
            keep = [torch.full((2 * rows, N), float("nan")) for _ in range(8)]   # memory that an unwritten result would take over
            del keep
            assert torch.equal(traced(x), layer(x))
            assert torch.equal(alone(x[0]), tl.forward_q4(x[0], layer.weight_q4))
        # the packed bytes are the traced layer's own buffer
        traced.load_state_dict({**traced.state_dict(), "packed": _packed(7)})
        want = _layer(7, bias)
        assert torch.equal(traced(x), want(x))


@pytest.fixture
def stand_ins(monkeypatch, stand_in):
    def dequantize(q, w, timed=False):
        _at(w, q.N * q.K)[:] = int(q.data.flatten()[0])

    def orthogonalize(g, out, batch, rows, cols, steps, coefficients, eps, workspace=None, timed=True):
        _at(out, batch * rows * cols)[:] = _at(g, batch * rows * cols) * steps

    monkeypatch.setattr(api, "q4_dequantize", dequantize)
    monkeypatch.setattr(api, "orthogonalize", orthogonalize)


@pytest.mark.parametrize("grad", [False, True])
def test_a_traced_update_computes(stand_ins, grad):
    """orthogonalize and dequantize_q4 are recorded as themselves; what packs weights is refused in a trace."""
    gen = torch.Generator().manual_seed(2)
    g = torch.randn(2, 4, 6, generator=gen, requires_grad=grad)
    q = cake.q4_of(_packed(3), N, K, 32, "float32", False)
    update = torch.jit.trace(lambda v: tl.orthogonalize(v, steps=4), (g,), check_trace=False)
    weights = torch.jit.trace(lambda v: v @ tl.dequantize_q4(q).t(), (torch.randn(2, K),), check_trace=False)
    for _ in range(3):
        g = torch.randn(2, 4, 6, generator=gen, requires_grad=grad)
        keep = [torch.full(s, float("nan")) for s in ((2, 4, 6), (N, K)) for _ in range(8)]
        del keep
        out = update(g)
        assert torch.equal(out, 4 * g.detach()) and not out.requires_grad and not tl.orthogonalize(g).requires_grad
        x = torch.randn(2, K, generator=gen)
        assert torch.equal(weights(x), x @ torch.full((K, N), 3.0))
    for call in (lambda w: tl.dequantize_q4(tl.quantize_q4(w)), lambda s: tl.dequantize_q4(tl.pack_q4(torch.zeros(4, 8, dtype=torch.uint8), s[:, :1], None, 16))):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (torch.randn(4, 16),), check_trace=False)


def test_a_call_names_torchs_default_stream(monkeypatch):
    """The handle of torch's default stream is 0, which the C entries take for the current context's own stream: a call
    on tensors names the null stream instead, so that it runs behind the work that made them."""
    class Torch:
        class _C:
            handle = 0
            _cuda_getCurrentRawStream = staticmethod(lambda index: Torch._C.handle)

        class cuda:
            current_stream = staticmethod(lambda device: type("Stream", (), {"cuda_stream": Torch._C.handle}))

    for device in (torch.device("cuda:0"), torch.device("cuda")):
        for Torch._C.handle, want in ((0, _lib.NULL_STREAM), (0x1234, 0x1234)):
            assert api._torch_stream(Torch, device) == want
    assert _lib.NULL_STREAM != 0 and api._stream(np.zeros(1, np.float32), torch.zeros(1)) == 0   # host operands: the context's own
