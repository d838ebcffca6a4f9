"""Refusals and sizes of the 4-bit linear layer and of orthogonalize that need no GPU: every check of an
argument comes before the device is touched."""
import numpy as np
import pytest

import cake_on_cpu_amd as cake
from cake_on_cpu_amd import _lib

F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16


def _buf(n=64):
    return np.zeros(n, np.float32)


@pytest.mark.parametrize("N,K,group,st,zeros,want", [
    (16, 128, 128, F32, 0, 1024 + 256),                  # one tile, one block, 16 scales of 4 bytes on a multiple of 256
    (1, 1, 32, F16, 1, 1024 + 256 + 256),                # padded to the same tile; 64 scales of 2 bytes; zero points likewise
    (17, 129, 64, BF16, 0, 4 * 1024 + 256),              # two tiles, two blocks: 4 x 16 x 2 scales of 2 bytes
    (4096, 4096, 128, BF16, 0, 4096 * 4096 // 2 + 4096 * 32 * 2),
    (0, 128, 128, F32, 0, 0), (16, 0, 128, F32, 1, 0),
])
def test_packed_size(N, K, group, st, zeros, want):
    assert cake.load().cake_hip_q4_size(N, K, group, st, zeros) == want


@pytest.mark.parametrize("N,K,group,st", [(-1, 8, 32, F32), (8, -1, 32, F32), (8, 8, 16, F32), (8, 8, 0, F32), (8, 8, 256, F32),
                                          (8, 8, 32, 3), (8, 8, 32, -1)])
def test_q4_entry_points_refuse(N, K, group, st):
    lib = cake.load()
    b = _buf().ctypes.data
    assert lib.cake_hip_q4_size(N, K, group, st, 0) == 0
    assert lib.cake_hip_last_error()
    assert lib.cake_hip_q4_pack(b, b, None, b, N, K, group, st, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_q4_quantize(b, F32, b, N, K, group, st, 0, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_q4_dequantize(b, b, F32, N, K, group, st, 0, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_linear_q4_forward(b, b, None, b, F32, 1, N, K, group, st, 0, None, None, None) == _lib.ERR_ARG


def test_q4_null_type_and_range():
    lib = cake.load()
    b = _buf().ctypes.data
    assert lib.cake_hip_q4_pack(None, b, None, b, 8, 8, 32, F32, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_q4_pack(b, None, None, b, 8, 8, 32, F32, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_q4_quantize(b, 7, b, 8, 8, 32, F32, 0, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_q4_quantize(None, F32, b, 8, 8, 32, F32, 0, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_q4_dequantize(b, None, F32, 8, 8, 32, F32, 0, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_linear_q4_forward(None, b, None, b, F32, 1, 8, 8, 32, F32, 0, None, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_linear_q4_forward(b, b, None, None, F32, 1, 8, 8, 32, F32, 0, None, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_linear_q4_forward(b, b, None, b, 5, 1, 8, 8, 32, F32, 0, None, None, None) == _lib.ERR_ARG
    assert lib.cake_hip_linear_q4_forward(b, b, None, b, F32, -1, 8, 8, 32, F32, 0, None, None, None) == _lib.ERR_ARG
    for N, K in ((65536, 32768), (0x7FFFFFFE, 1), (1, 0x7FFFFFFE)):
        assert lib.cake_hip_q4_size(N, K, 32, F32, 0) == 0
        assert lib.cake_hip_q4_quantize(b, F32, b, N, K, 32, F32, 0, None, None) == _lib.ERR_RANGE
    assert lib.cake_hip_linear_q4_forward(b, b, None, b, F32, 1 << 20, 8, 4096, 32, F32, 0, None, None, None) == _lib.ERR_RANGE
    assert lib.cake_hip_linear_q4_forward(b, b, None, b, F32, 0x7FFFFF80, 1, 1, 32, F32, 0, None, None, None) == _lib.ERR_RANGE
    # nothing to do: no device is asked for
    assert lib.cake_hip_linear_q4_forward(None, None, None, None, F32, 0, 8, 8, 32, F32, 0, None, None, None) == _lib.OK
    assert lib.cake_hip_q4_quantize(None, F32, None, 0, 8, 32, F32, 0, None, None) == _lib.OK


def _orth(batch=1, rows=4, cols=4, steps=5, c=(3.4445, -4.775, 2.0315), eps=1e-7, t=F32, g=True):
    b = _buf().ctypes.data
    return cake.load().cake_hip_orthogonalize(b if g else None, b, t, batch, rows, cols, steps, *c, eps, None, None, None)


def test_orthogonalize_refuses():
    for bad in (dict(batch=-1), dict(rows=-1), dict(cols=-2), dict(steps=0), dict(steps=-3), dict(t=3), dict(eps=-1.0),
                dict(eps=float("nan")), dict(eps=float("inf")), dict(g=False)):
        assert _orth(**bad) == _lib.ERR_ARG, bad
    assert _orth(batch=65536) == _lib.ERR_RANGE
    assert _orth(rows=65536, cols=32768) == _lib.ERR_RANGE
    assert _orth(rows=1, cols=0x7FFFFFF0) == _lib.ERR_RANGE and _orth(rows=0x7FFFFFF0, cols=1) == _lib.ERR_RANGE
    assert _orth(batch=0) == _lib.OK and _orth(rows=0) == _lib.OK and _orth(cols=0, g=False) == _lib.OK
    # polynomials that drive singular values away from 1 without bound
    assert _orth(c=(40.0, 0.0, 0.0)) == _lib.ERR_ARG
    assert b"singular value" in cake.load().cake_hip_last_error()
    assert _orth(c=(40.0, 0.0, 0.0), steps=1, rows=0) == _lib.OK
    assert _orth(c=(float("nan"), 0.0, 0.0)) == _lib.ERR_ARG
    assert _orth(c=(2.0, 1e30, 0.0), steps=1) == _lib.ERR_ARG


def test_orthogonalize_workspace_covers_its_parts():
    ws = cake.orthogonalize_workspace
    assert ws(0, 4, 4) == 0 and ws(1, 0, 4) == 0 and ws(-1, 4, 4) == 0 and ws(1, 1 << 20, 1 << 20) == 0
    # at least three copies of x and two of the small square, each 4 bytes a padded value; the same on every call
    for batch, rows, cols in ((2, 300, 200), (2, 200, 300), (1, 1024, 4096)):
        m, n = (-(-v // 32) * 32 for v in sorted((rows, cols)))
        assert ws(batch, rows, cols) >= batch * (3 * m * n * 4 + 2 * m * m * 4) and ws(batch, rows, cols) == ws(batch, rows, cols)


def test_python_refusals():
    f, u = _buf(64), np.zeros(4096, np.uint8)
    with pytest.raises(TypeError):
        cake.q4_quantize(np.zeros(64, np.float64), 8, 8)
    with pytest.raises(ValueError):
        cake.q4_quantize(f, 9, 8)
    with pytest.raises(cake.CakeHipError):
        cake.q4_quantize(f, 8, 8, group=48)
    with pytest.raises(TypeError):
        cake.q4_pack(f, f, None, 8, 8, 32)                       # codes are bytes
    with pytest.raises(ValueError):
        cake.q4_pack(u[:16], f, None, 8, 8, 32)                  # too few codes
    with pytest.raises(ValueError):
        cake.q4_pack(u, f[:7], None, 8, 8, 32)                   # too few scales
    with pytest.raises(TypeError):
        cake.q4_pack(u, f, f.astype(np.float16), 8, 8, 32)       # zeros of another type than scales
    with pytest.raises(ValueError):
        cake.q4_of(u[:100], 8, 8, 32, "float32", False)
    q = cake.q4_of(np.zeros(4096, np.uint8), 8, 8, 32, "float32", False)
    with pytest.raises(ValueError):
        cake.linear_q4_forward(f[:7], q, None, f, 1)
    with pytest.raises(TypeError):
        cake.linear_q4_forward(f, q, f.astype(np.float16), f, 1)
    with pytest.raises(TypeError):
        cake.linear_q4_forward(f.reshape(8, 8).T, q, None, f, 1)
    with pytest.raises(ValueError):
        cake.orthogonalize(f, f, 2, 8, 8)
    with pytest.raises(TypeError):
        cake.orthogonalize(f, f.astype(np.float16), 1, 8, 8)


def test_torch_layer_refusals():
    torch = pytest.importorskip("torch")
    from cake_on_cpu_amd import torch_linear as tl
    q = cake.q4_of(torch.zeros(4096, dtype=torch.uint8), 8, 8, 32, torch.float32, False)
    for x, bias in ((torch.zeros(2, 9), None), (torch.zeros(8), None), (torch.zeros(2, 8), torch.zeros(7)),
                    (torch.zeros(2, 8), torch.zeros(8, dtype=torch.float16))):
        with pytest.raises(ValueError):
            tl.forward_q4(x, q, bias)
    with pytest.raises(TypeError):
        tl.forward_q4(torch.zeros(2, 8, dtype=torch.float64), q)
    codes, s = torch.zeros(8, 4, dtype=torch.uint8), torch.zeros(8, 1)
    for bad in ((codes, s, None, 10), (codes, s[:7], None, 8), (codes, s, s[:, :0], 8)):
        with pytest.raises(ValueError):
            tl.pack_q4(*bad, 32)
    with pytest.raises(ValueError):
        tl.quantize_q4(torch.zeros(2, 3, 4))
    with pytest.raises(ValueError):
        tl.orthogonalize(torch.zeros(5))
    with pytest.raises(ValueError):
        tl.cake_muon([torch.nn.Parameter(torch.zeros(5))])
    assert tl.orthogonalize(torch.zeros(0, 5)).shape == (0, 5)


def test_sides_beyond_a_launch_are_refused():
    """What would take 2^32 threads or more never reaches a launch."""
    lib = cake.load()
    b = _buf().ctypes.data
    assert lib.cake_hip_q4_size(0x3FFFFF01, 1, 32, F32, 0) == 0 and lib.cake_hip_q4_size(0x3FFFFF00, 1, 32, F32, 0) > 0
    assert lib.cake_hip_q4_pack(b, b, None, b, 0x3FFFFF01, 1, 32, F32, None, None) == _lib.ERR_RANGE
    assert lib.cake_hip_linear_q4_forward(b, b, None, b, F32, 0x1FFFFF01, 1, 1, 32, F32, 0, None, None, None) == _lib.ERR_RANGE
    assert lib.cake_hip_linear_q4_workspace(0x1FFFFF01, 1, 1, F32) == 0 < lib.cake_hip_linear_q4_workspace(0x1FFFFF00, 1, 1, F32)
    assert _orth(rows=1, cols=0x3FFFFF01) == _lib.ERR_RANGE and _orth(rows=0x3FFFFF01, cols=1) == _lib.ERR_RANGE


def test_steps_without_end_are_refused():
    """A small matrix takes all its steps in one launch, which has to end."""
    assert _orth(steps=1001) == _lib.ERR_ARG and _orth(steps=0x7FFFFFFF) == _lib.ERR_ARG
    assert b"steps" in cake.load().cake_hip_last_error()


def test_packed_weights_hold_what_they_say():
    """Sizes are checked where packed weights are made and where the layer's function is applied by itself."""
    torch = pytest.importorskip("torch")
    from cake_on_cpu_amd import torch_linear as tl
    held = torch.zeros(cake.q4_size(8, 8, 32), dtype=torch.uint8)
    for bad in ((held[:-1], 8, 8, 32, F32, False), (held, 17, 8, 32, F32, False), (held, 8, 8, 32, F32, True)):
        with pytest.raises(ValueError):
            cake.Q4Weight(*bad)
    for bad in ((held, 8, 8, 48, F32, False), (held, 8, 8, 32, 9, False), (held, -8, 8, 32, F32, False)):
        with pytest.raises(cake.CakeHipError):
            cake.Q4Weight(*bad)
    with pytest.raises(TypeError):
        cake.Q4Weight(held.float(), 8, 8, 32, F32, False)
    q = cake.Q4Weight(held, 8, 8, 32, F32, False)
    for x, bias in ((torch.zeros(2, 7), None), (torch.zeros(2, 8), torch.zeros(7))):
        with pytest.raises(ValueError):
            tl.cake_linear_q4_function.apply(x.requires_grad_(), q, bias)


def test_layer_refuses_what_is_not_its_own():
    """Stored bytes of another group size, type of scales or kind are other weights, also where their number is the same."""
    torch = pytest.importorskip("torch")
    from cake_on_cpu_amd import torch_linear as tl

    def layer(N=16, K=128, group=32, dtype=torch.bfloat16, zeros=False):
        return tl.cake_linear_q4(cake.q4_of(torch.zeros(cake.q4_size(N, K, group, dtype, zeros), dtype=torch.uint8), N, K, group, dtype, zeros))

    stored = layer().state_dict()
    assert all(isinstance(v, torch.Tensor) for v in stored.values())
    layer().load_state_dict(stored)
    for other in (layer(dtype=torch.float16), layer(group=64), layer(N=15)):
        with pytest.raises((ValueError, RuntimeError)):
            other.load_state_dict(stored)
    for x in (torch.zeros(3, 64), torch.zeros(3, 256), torch.zeros(128, 3), torch.tensor(1.0)):
        with pytest.raises(ValueError):
            layer()(x)


def test_optimiser_takes_matrices_alone_also_later():
    torch = pytest.importorskip("torch")
    from cake_on_cpu_amd import torch_linear as tl
    w = torch.nn.Parameter(torch.zeros(3, 4))
    opt = tl.cake_muon(iter([w]))
    for shape in ((5,), (2, 3, 4)):
        with pytest.raises(ValueError):
            opt.add_param_group({"params": torch.nn.Parameter(torch.zeros(shape))})
        with pytest.raises(ValueError):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(shape))], "lr": 0.1})
    opt.add_param_group({"params": (v for v in [torch.nn.Parameter(torch.zeros(4, 4))]), "lr": 0.5})
    assert [len(g["params"]) for g in opt.param_groups] == [1, 1] and opt.param_groups[1]["lr"] == 0.5
    for bad in ([3], {torch.nn.Parameter(torch.zeros(2, 2))}):
        with pytest.raises(TypeError):
            tl.cake_muon(bad) if isinstance(bad, list) else opt.add_param_group({"params": bad})
    with pytest.raises(ValueError):
        tl.cake_muon([("bias", torch.nn.Parameter(torch.zeros(2)))])
    assert len(tl.cake_muon(torch.nn.Linear(3, 4, bias=False).named_parameters()).param_groups[0]["params"]) == 1
    for group in (0, 48):
        with pytest.raises(ValueError):
            tl.pack_q4(torch.zeros(8, 4, dtype=torch.uint8), torch.zeros(8, 1), None, 8, group)


def test_a_refused_load_changes_nothing():
    torch = pytest.importorskip("torch")
    from cake_on_cpu_amd import torch_linear as tl

    def layer(fill, dtype):
        data = torch.full((cake.q4_size(16, 128, 32, dtype, False),), fill, dtype=torch.uint8)
        return tl.cake_linear_q4(cake.q4_of(data, 16, 128, 32, dtype, False), torch.zeros(16))

    held, stored = layer(1, torch.bfloat16), layer(2, torch.float16).state_dict()
    with pytest.raises(ValueError):
        held.load_state_dict(stored)
    assert bool((held.packed == 1).all())
    model, other = torch.nn.Sequential(layer(1, torch.float16)), torch.nn.Sequential(layer(2, torch.float16))
    model.load_state_dict(other.state_dict())
    assert bool((model[0].packed == 2).all())
    with pytest.raises(RuntimeError):       # strict: what the bytes were made for has to be there
        model.load_state_dict({k: v for k, v in other.state_dict().items() if "extra" not in k})


def test_a_workspace_does_not_grow_with_the_number_of_large_matrices():
    """Beyond 2^26 values a batch is taken some matrices at a time: 16 bytes a value of a pass (x three times in
    pairs, once in fp32), 8 a value of its squares, and the sums of slices."""
    ws = cake.orthogonalize_workspace
    assert ws(64, 4096, 4096) <= 1.1 * 24 * 2 ** 26 and ws(4, 4096, 4096) >= 20 * 2 ** 26
    assert ws(32, 14336, 4096) == ws(1, 14336, 4096) and ws(65535, 300, 300) <= 1.1 * 24 * 2 ** 26
    assert ws(65535, 64, 64) == 0
