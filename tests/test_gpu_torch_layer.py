"""GPU checks of the torch side of the 4-bit layer, of orthogonalize and of the linear layer: the order of a call and
the work that makes its operands, and traces."""
import pytest

torch = pytest.importorskip("torch")

import cake_on_cpu_amd as cake
from cake_on_cpu_amd import torch_linear as tl

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")]


def _calls():
    """name -> (a call of one argument, the shape of its argument)"""
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(384, 640, device="cuda", generator=gen)
    q = tl.quantize_q4(w, 64, True)
    layer = tl.cake_linear(640, 384).cuda()
    calls = {"one token": (lambda x: tl.forward_q4(x, q), (1, 640)), "a few": (lambda x: tl.forward_q4(x, q), (9, 640)),
             "a prompt": (lambda x: tl.forward_q4(x, q), (300, 640)), "one launch": (tl.orthogonalize, (64, 64)),
             "many launches": (tl.orthogonalize, (300, 700)), "pack": (lambda x: tl.dequantize_q4(tl.quantize_q4(x, 32)), (200, 300)),
             "layer": (lambda x: layer(x).detach(), (50, 640))}

    def gradient(x):
        x = x.clone().requires_grad_()
        return torch.autograd.grad(tl.forward_q4(x, q).sum(), x)[0]

    calls["gradient"] = (gradient, (30, 640))
    return calls


def test_inside_a_context_a_call_follows_the_work_that_makes_its_operands():
    """The operand is written on torch's default stream behind some milliseconds of other work, and the memory that a
    call gives back is written over right after it."""
    calls = _calls()
    gen = torch.Generator(device="cuda").manual_seed(2)
    busy = torch.randn(4096, 4096, device="cuda", generator=gen)
    want, fresh = {}, {}
    for name, (call, shape) in calls.items():
        fresh[name] = torch.randn(shape, device="cuda", generator=gen)
        want[name] = call(fresh[name])
    torch.cuda.synchronize()
    with cake.Context() as cx:
        assert cx.stream
        for name, (call, shape) in calls.items():
            for _ in range(2):
                x = torch.zeros(shape, device="cuda")
                torch.cuda.synchronize()
                for _ in range(4):
                    busy = busy @ busy * 1e-2
                x.copy_(fresh[name])
                got = call(x)
                x.fill_(float("nan"))
                over = [torch.full((1 << k,), 0xFF, dtype=torch.uint8, device="cuda") for k in range(9, 24)]
                assert torch.equal(got, want[name]), name
                del over


@pytest.mark.parametrize("rows", [1, 7, 100])
def test_a_traced_layer_computes_on_the_device(rows):
    layer = tl.cake_linear_q4.of(tl.cake_linear(300, 130).cuda(), group=64, zeros=True)
    update = torch.jit.trace(lambda g: tl.orthogonalize(g), (torch.randn(40, 60, device="cuda"),), check_trace=False)
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(layer, (torch.randn(rows, 300, device="cuda"),), check_trace=False)
            for _ in range(3):
                x, g = torch.randn(rows, 300, device="cuda"), torch.randn(40, 60, device="cuda")
                assert torch.equal(traced(x), layer(x)) and torch.equal(update(g), tl.orthogonalize(g))


@pytest.mark.parametrize("rows", [1, 7, 100])
def test_gradients_through_a_traced_layer(rows):
    layer = tl.cake_linear_q4.of(tl.cake_linear(300, 130).cuda(), group=64, zeros=True)
    traced = torch.jit.trace(layer, (torch.randn(rows, 300, device="cuda"),))
    for _ in range(3):
        x, gy = torch.randn(rows, 300, device="cuda", requires_grad=True), torch.randn(rows, 130, device="cuda")
        want = torch.autograd.grad(layer(x), (x, layer.bias), gy)
        got = torch.autograd.grad(traced(x), (x, layer.bias), gy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("grad", [False, True])
def test_a_compiled_model_calls_the_layer(grad):
    """torch.compile leaves the calls as they are and compiles around them."""
    layer = tl.cake_linear_q4.of(tl.cake_linear(300, 130).cuda(), group=64)

    def model(x):
        return torch.relu(layer(x * 2)) + 1

    compiled = torch.compile(model, backend="eager")
    with torch.set_grad_enabled(grad):
        for rows in (1, 7, 7, 100):
            x = torch.randn(rows, 300, device="cuda")
            assert torch.equal(compiled(x), model(x))
