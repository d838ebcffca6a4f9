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


@pytest.fixture
def signs(monkeypatch):
    """In place of the iterations something as blunt that torch computes the same everywhere; returns the calls' batches."""
    calls = []

    def orthogonalize(g, out, batch, rows, cols, steps, coefficients, eps, workspace=None, timed=True):
        assert g.shape == out.shape and g.dtype == out.dtype and g.is_contiguous()
        calls.append((batch, rows, cols, g.dtype))
        out.copy_(g.sign() * 0.25)

    monkeypatch.setattr(api, "orthogonalize", orthogonalize)
    return calls


def _grads(shape, dtype, steps, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=gen).to(dtype) for _ in range(steps)]


def _formula(w, grads, lr, mu, nesterov, decay):
    """The optimiser's formula in 64 bits on the stand-in: weights and momentum after every step"""
    w, b, out = w.double(), torch.zeros_like(w, dtype=torch.float64), []
    for g in grads:
        b = mu * b + g.double()
        u = g.double() + mu * b if nesterov else b
        w = w - lr * decay * w - lr * max(1.0, w.size(0) / w.size(1)) ** 0.5 * u.sign() * 0.25
        out.append((w, b))
    return out


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_optimiser_keeps_its_state_in_32_bits(signs, dtype, nesterov):
    """200 steps of every type of parameter against the formula: momentum to 32 bits (two roundings a step of at most the
    largest |b|, of which 1 / (1 - mu) count together), a 16-bit weight to one rounding of the formula's."""
    start, lr, mu, decay = torch.randn(7, 3, generator=torch.Generator().manual_seed(3)).to(dtype), 0.01, 0.95, 0.1
    w = torch.nn.Parameter(start.clone())
    opt = tl.cake_muon([w], lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay)
    grads = _grads((7, 3), dtype, 200)
    formula = _formula(start, grads, lr, mu, nesterov, decay)
    widest = max(float(b.abs().max()) for _, b in formula)
    for i, (g, (want, b)) in enumerate(zip(grads, formula)):
        w.grad = g.clone()
        opt.step()
        held = opt.state[w]["momentum"]
        assert held.dtype == torch.float32
        assert float((held.double() - b).abs().max()) <= 2 * 2.0 ** -24 * widest / (1 - mu), i
        # two roundings of a step of the 32-bit weight, 200 steps of values below 4, then the type's
        bar = 2 * (i + 1) * 2.0 ** -24 * 4 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (want.abs() + 1e-4))
        assert bool(((w.detach().double() - want).abs() <= bar).all()), i
    assert all(c[3] == torch.float32 for c in signs)


def test_decay_below_a_16_bit_step_is_not_lost(signs):
    """1000 steps of weights w = w - 0.001 w: every single one is below half a step of bfloat16."""
    w = torch.nn.Parameter(torch.ones(4, 4, dtype=torch.bfloat16))
    opt = tl.cake_muon([w], lr=0.01, weight_decay=0.1)
    for _ in range(1000):
        w.grad = torch.zeros_like(w)
        opt.step()
    assert bool(((w.detach().double() - 0.999 ** 1000).abs() <= 2.0 ** -9 * 0.37).all())


def test_a_16_bit_weight_set_from_elsewhere_is_what_counts(signs):
    """Loaded or clipped weights are not undone by what the optimiser kept of the old ones."""
    w = torch.nn.Parameter(torch.ones(4, 4, dtype=torch.bfloat16))
    opt = tl.cake_muon([w], lr=0.0, momentum=0.0, weight_decay=0.0)
    for _ in range(3):
        w.grad = torch.ones_like(w)
        opt.step()
    with torch.no_grad():
        w[1].fill_(-2.0)
        w[2, 2] = float("nan")
    opt.step()
    want = torch.ones(4, 4)
    want[1] = -2.0
    want[2, 2] = float("nan")
    assert torch.equal(w.detach().float().nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_stored_optimiser_goes_on_where_it_was(signs, tmp_path, dtype):
    """Loading does not round the state to the parameters' type, whatever group a parameter is in."""
    def made():
        ws = [torch.nn.Parameter(torch.full(s, 0.5, dtype=dtype)) for s in ((4, 6), (6, 4), (4, 6))]
        return ws, tl.cake_muon([{"params": ws[:1]}, {"params": ws[1:], "lr": 0.003}], lr=0.01, weight_decay=0.05)

    def steps(ws, opt, seeds):
        for seed in seeds:
            for i, w in enumerate(ws):
                w.grad = _grads(tuple(w.shape), dtype, 1, 10 * seed + i)[0]
            opt.step()

    ws, opt = made()
    steps(ws, opt, range(5))
    torch.save((opt.state_dict(), [w.detach() for w in ws]), tmp_path / "o")
    held, weights = torch.load(tmp_path / "o", weights_only=True)
    others, other = made()
    with torch.no_grad():
        for a, b in zip(others, weights):
            a.copy_(b)
    other.load_state_dict(held)
    for a, b in zip(ws, others):
        assert all(torch.equal(opt.state[a][k], other.state[b][k]) and other.state[b][k].dtype == torch.float32 for k in opt.state[a])
    steps(ws, opt, range(5, 9))
    steps(others, other, range(5, 9))
    assert all(torch.equal(a, b) for a, b in zip(ws, others))
    kept = held["state"][0]["momentum"].clone()
    assert torch.equal(kept, torch.load(tmp_path / "o", weights_only=True)[0]["state"][0]["momentum"])   # and steps do not reach into what was loaded


def test_the_optimisers_copies_do_not_grow_with_the_number_of_large_matrices(signs):
    """Matrices of one shape go together up to 2^26 values."""
    ws = [torch.nn.Parameter(torch.zeros(2048, 4096)) for _ in range(11)] + [torch.nn.Parameter(torch.zeros(3, 5)) for _ in range(7)]
    opt = tl.cake_muon(ws, lr=1.0, momentum=0.0)
    for i, w in enumerate(ws):
        w.grad = torch.full_like(w, 1.0 if i % 3 else -1.0)
    opt.step()
    assert [c[0] for c in signs] == [8, 3, 7]
    assert all(bool((w == (-0.25 if i % 3 else 0.25)).all()) for i, w in enumerate(ws))


def test_a_refused_step_changes_nothing(signs):
    a, b = torch.nn.Parameter(torch.ones(3, 4)), torch.nn.Parameter(torch.ones(4, 4))
    for bad, error in ((dict(steps=0), cake.CakeHipError), (dict(steps=1001), cake.CakeHipError), (dict(coefficients=(40.0, 0.0, 0.0)), cake.CakeHipError),
                       (dict(eps=-1.0), cake.CakeHipError), (dict(coefficients=(1.0, 2.0)), ValueError)):
        opt = tl.cake_muon([{"params": [a]}, {"params": [b], **bad}])
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
        with pytest.raises(error):
            opt.step()
        assert bool((a == 1).all()) and not opt.state
    for other in (torch.nn.Parameter(torch.ones(4, 4, dtype=torch.float64)), torch.nn.Parameter(torch.ones(4, 4, dtype=torch.complex64))):
        opt = tl.cake_muon([a, other])
        other.grad = torch.ones_like(other)
        with pytest.raises(TypeError):
            opt.step()
        assert bool((a == 1).all()) and not opt.state
    opt = tl.cake_muon([a, b])
    b.grad = torch.ones(4, 4).to_sparse()
    with pytest.raises(TypeError):
        opt.step()
    assert bool((a == 1).all()) and not opt.state
    assert not signs


def test_packed_weights_stay_what_they_were_made_as(stand_in):
    """What a kernel reads follows from these numbers, so they do not change behind their check; bytes that shrank are refused."""
    q = cake.q4_of(_packed(3), N, K, 32, "float32", False)
    for name, value in (("data", torch.zeros(16, dtype=torch.uint8)), ("N", 500), ("K", 64), ("group", 64), ("scale_type", 1), ("with_zeros", True)):
        with pytest.raises(AttributeError):
            setattr(q, name, value)
    x = torch.ones(2, K)
    tl.forward_q4(x, q)
    q.data.resize_(q.data.numel() - 1)
    for call in (lambda: tl.forward_q4(x, q), lambda: tl.forward_q4(x.clone().requires_grad_(), q), lambda: tl.dequantize_q4(q)):
        with pytest.raises(ValueError):
            call()


def test_shrunk_bytes_are_refused_by_the_plain_interface():
    q = cake.q4_of(_packed(3), N, K, 32, "float32", False)
    q.data.resize_(q.data.numel() - 1)
    x, y = torch.ones(2, K), torch.full((2, N), 7.0)
    for call in (lambda: cake.linear_q4_forward(x, q, None, y, 2), lambda: cake.q4_dequantize(q, torch.zeros(N, K))):
        with pytest.raises(ValueError):
            call()
    assert bool((y == 7).all())


def test_packed_weights_are_copied_and_stored_whole():
    import copy
    import pickle
    q = cake.q4_of(_packed(3), N, K, 32, "float32", False)
    for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert torch.equal(other.data, q.data) and (other.N, other.K, other.group, other.scale_type, other.with_zeros) == (N, K, 32, _lib.F32, False)
    assert copy.deepcopy(q).data.data_ptr() != q.data.data_ptr()


@pytest.mark.parametrize("grad", [False, True])
def test_a_trace_compares_equal_with_the_next_one(stand_ins, grad):
    """torch.jit.trace's own check, which records everything twice and refuses what differs."""
    layer, q = _layer(3, True), cake.q4_of(_packed(3), N, K, 32, "float32", False)
    with torch.set_grad_enabled(grad):
        for call in (layer, lambda v: tl.forward_q4(v, layer.weight_q4), lambda v: tl.orthogonalize(v), lambda v: v @ tl.dequantize_q4(q).t()):
            traced = torch.jit.trace(call, (torch.randn(4, K),))
            x = torch.randn(6, K)
            assert torch.equal(traced(x), call(x))


def test_packed_weights_stored_attribute_by_attribute_load():
    """As pickle stores an object with slots by itself, which is how they were stored before their numbers were fixed."""
    q = cake.q4_of(_packed(3), N, K, 32, "float32", False)
    other = cake.Q4Weight.__new__(cake.Q4Weight)
    other.__setstate__((None, {name: getattr(q, name) for name in ("data", "N", "K", "group", "scale_type", "with_zeros")}))
    assert other.data is q.data and other.bytes == q.bytes and repr(other) == repr(q)
