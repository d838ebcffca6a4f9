"""GPU checks of the 4-bit linear layer against its definition in 64 bits.

Quantising and dequantising are exact statements (codes, scales and zero points are determined), so
their values have to be equal.  A product's bar: with S = sum_k s (code + |zero|) |x| the sum of everything that
is added in fp32, every result is within R 2^-24 S of the 64-bit sum, R counting the roundings in a row:
at most 16 for a block of 128 columns (four matrix instructions that round their sum of 32 products no more than
twice, for the codes and for the column of ones, and two operations per group of 32) and 48 for the joining of
waves and pieces and the bias; then half a step of the output's type, and half of fp16's last subnormal step."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import cake_on_cpu_amd as cake
from cake_on_cpu_amd import _lib
from cake_on_cpu_amd import torch_linear as tl

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _weights(N, K, group, zeros, scale_dtype, seed):
    """codes as bytes and as numbers [N][K], scales, zero points, the values in 64 bits, and s (code + |zero|)"""
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // group)
    packed = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, dtype=torch.uint8)
    s = (0.01 * torch.randn(N, groups, generator=g).exp()).to(scale_dtype)
    z = (torch.rand(N, groups, generator=g) * 15).to(scale_dtype) if zeros else None     # no whole numbers
    k = torch.arange(K)
    code = ((packed[:, k // 2].int() >> (4 * (k % 2)).int()) & 15).double()
    s64, z64 = s.double()[:, k // group], (z.double()[:, k // group] if zeros else torch.full((N, K), 8.0, dtype=torch.float64))
    return packed, s, z, (code - z64) * s64, s64.abs() * (code + z64.abs())


def _check(y, x, v64, mass, bias, K):
    x64 = x.double().cpu()
    want = x64 @ v64.t()
    S = x64.abs() @ mass.t()
    if bias is not None:
        want = want + bias.double().cpu()
        S = S + bias.double().cpu().abs()
    R = 16 * (-(-K // 128)) + 48
    tol = R * 2.0 ** -24 * S + 2.0 ** -40
    if y.dtype != torch.float32:
        tol = tol + torch.finfo(y.dtype).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    far = (y.double().cpu() - want).abs() - tol
    assert y.shape == want.shape and bool((far <= 0).all()), float(far.max())


# M, N, K: one token to many, odd sizes, a single row or column, one group, short last groups and blocks
SHAPES = [(1, 1, 1), (1, 16, 128), (1, 17, 33), (1, 100, 1000), (1, 1024, 4096), (2, 31, 129), (3, 256, 257), (4, 40, 512), (5, 33, 640),
          (6, 50, 300), (7, 64, 96), (10, 48, 1111), (11, 65, 256), (16, 130, 384), (17, 47, 2048), (21, 32, 500), (22, 33, 128),
          (32, 96, 1000), (33, 70, 2111), (64, 48, 130), (65, 40, 77), (100, 111, 960), (130, 260, 520), (257, 300, 384), (600, 96, 200)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_q4_against_64_bits(shape, kind):
    M, N, K = shape
    for i, (group, zeros, scale) in enumerate(((32, True, "f32"), (64, False, "bf16"), (128, True, "f16"), (128, False, "f32"), (32, False, "f16"),
                                               (64, True, "bf16"))):
        print(f"linear_q4 M={M} N={N} K={K} {kind} group={group} zeros={zeros} scales={scale}", flush=True)
        packed, s, z, v64, mass = _weights(N, K, group, zeros, TYPES[scale], 7 * i + M)
        q = tl.pack_q4(packed.cuda(), s.cuda(), None if z is None else z.cuda(), K, group)
        x = torch.randn(M, K, generator=torch.Generator().manual_seed(i)).to(TYPES[kind]).cuda()
        bias = torch.randn(N, generator=torch.Generator().manual_seed(50 + i)).to(TYPES[kind]).cuda() if i % 2 else None
        y = tl.forward_q4(x, q, bias)
        _check(y, x, v64, mass, bias, K)
        # the packed weights stand for the codes they were made of, bit for bit
        assert torch.equal(tl.dequantize_q4(q).cpu(), v64.float() if not zeros else _product32(packed, s, z, K, group))
        # and the result does not change from call to call
        assert torch.equal(y, tl.forward_q4(x, q, bias))


def _product32(packed, s, z, K, group):
    k = torch.arange(K)
    code = ((packed[:, k // 2].int() >> (4 * (k % 2)).int()) & 15).float()
    return (code - z.float()[:, k // group]) * s.float()[:, k // group]


@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_of_x_off_alignment_and_guards_around_y(kind):
    """x that starts one element behind a 16-byte border, and y inside a larger buffer that stays as it was."""
    t = TYPES[kind]
    for M, N, K in ((1, 33, 264), (9, 47, 1000), (70, 50, 136)):
        packed, s, z, v64, mass = _weights(N, K, 64, True, torch.float32, M)
        q = tl.pack_q4(packed.cuda(), s.cuda(), z.cuda(), K, 64)
        flat = torch.randn(M * K + 1, generator=torch.Generator().manual_seed(3)).to(t).cuda()
        x = flat[1:].view(M, K)
        around = torch.full((M * N + 64,), 7.0, dtype=t, device="cuda")
        y = around[32:32 + M * N].view(M, N)
        print(f"linear_q4 unaligned M={M} N={N} K={K} {kind}", flush=True)
        cake.linear_q4_forward(x, q, None, y, M, timed=False)
        _check(y, x, v64, mass, None, K)
        assert bool((around[:32] == 7).all()) and bool((around[32 + M * N:] == 7).all())


def test_views_are_made_contiguous_and_values_of_every_size_survive():
    N, K, M = 48, 256, 6
    packed, s, z, v64, mass = _weights(N, K, 128, False, torch.float32, 1)
    q = tl.pack_q4(packed.cuda(), s.cuda(), None, K, 128)
    wide = torch.randn(K, M, generator=torch.Generator().manual_seed(3)).cuda()
    _check(tl.forward_q4(wide.t(), q), wide.t(), v64, mass, None, K)
    # fp32 and bf16 reach beyond fp16: nothing overflows or vanishes on the way to the matrix pipe
    for scale in (1e-30, 1e30):
        for t in (torch.float32, torch.bfloat16):
            x = (torch.randn(M, K, generator=torch.Generator().manual_seed(4)) * scale).to(t)
            want = x.double() @ v64.t()
            tol = (16 * 2 + 48) * 2.0 ** -24 * (x.double().abs() @ mass.t()) + torch.finfo(t).eps * want.abs()
            assert bool(((tl.forward_q4(x.cuda(), q).double().cpu() - want).abs() <= tol).all()), (scale, t)
    # one token's NaN is that token's alone
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(5)).cuda()
    y0 = tl.forward_q4(x, q)
    x[2, 17] = float("nan")
    y1 = tl.forward_q4(x, q)
    keep = [0, 1, 3, 4, 5]
    assert bool(torch.isnan(y1[2]).all()) and torch.equal(y1[keep], y0[keep])


def test_empty_dimensions_and_host_operands():
    f32 = np.float32
    y = np.full((3, 5), np.nan, f32)
    bias = np.arange(5, dtype=f32)
    empty = cake.q4_of(np.zeros(16, np.uint8)[:0], 5, 0, 32, "float32", False)
    cake.linear_q4_forward(np.zeros(1, f32), empty, bias, y, 3)          # K = 0: y = bias
    assert np.array_equal(y, np.broadcast_to(bias, (3, 5)))
    cake.linear_q4_forward(np.zeros(1, f32), empty, None, y, 3)
    assert not y.any()
    many = np.full((700, 5), np.nan, f32)                                # and for many rows
    cake.linear_q4_forward(np.zeros(1, f32), empty, bias, many, 700)
    assert np.array_equal(many, np.broadcast_to(bias, (700, 5)))
    N, K, M = 70, 333, 5
    packed, s, z, v64, mass = _weights(N, K, 32, True, torch.float32, 2)
    q = cake.q4_pack(packed.numpy(), s.numpy(), z.numpy(), N, K, 32)
    x = np.random.default_rng(1).standard_normal((M, K)).astype(f32)
    y = np.full((M, N), np.nan, f32)
    secs = cake.linear_q4_forward(x, q, None, y, M)
    assert secs > 0
    _check(torch.from_numpy(y), torch.from_numpy(x), v64, mass, None, K)
    w = np.full((N, K), np.nan, f32)
    cake.q4_dequantize(q, w)
    assert np.array_equal(w, _product32(packed, s, z, K, 32).numpy())


def _quantized64(w, group, zeros, scale_dtype):
    """The definition in 64 bits: scales, zero points and the values of the codes"""
    w = w.double()
    N, K = w.shape
    out = torch.empty(N, K, dtype=torch.float64)
    for k0 in range(0, K, group):
        run = w[:, k0:k0 + group]
        hi, lo = run.amax(1).clamp(min=0), run.amin(1).clamp(max=0)
        s = ((hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7).float().to(scale_dtype).double()[:, None]
        z = torch.where(s > 0, torch.round(-lo[:, None] / s), 8.0).clamp(0, 15) if zeros else 8.0
        c = torch.where(s > 0, torch.round(run / s), 0.0).add(z).clamp(0, 15)
        out[:, k0:k0 + group] = (c - z) * s
    return out


@pytest.mark.parametrize("shape", [(1, 1), (16, 128), (17, 129), (5, 31), (33, 1000), (100, 4099), (257, 264), (2111, 40)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("zeros", [False, True], ids=["plain", "zeros"])
def test_quantize_is_the_definition(shape, zeros):
    N, K = shape
    for i, (kind, scale, group) in enumerate((("f32", "f32", 32), ("f32", "bf16", 128), ("bf16", "f32", 64), ("f16", "f16", 32), ("bf16", "bf16", 128),
                                              ("f16", "f32", 64))):
        print(f"quantize N={N} K={K} {kind} scales={scale} group={group} zeros={zeros}", flush=True)
        g = torch.Generator().manual_seed(11 + i)
        w = torch.randn(N, K, generator=g) * 0.02
        w[N // 2] = 0                                                       # a row of zeros
        w[0] = w[0].abs()                                                   # a row of one sign
        # whole numbers: quotients that are ties
        if N > 3:
            w[3] = torch.randint(-7, 8, (K,), generator=g) * 0.25
        w = w.to(TYPES[kind])
        q = tl.quantize_q4(w.cuda(), group, zeros, TYPES[scale])
        want = _quantized64(w, group, zeros, TYPES[scale])
        assert torch.equal(tl.dequantize_q4(q, torch.float32).cpu(), want.float())
        for t in (torch.float16, torch.bfloat16):
            assert torch.equal(tl.dequantize_q4(q, t).cpu(), want.float().to(t))


def test_quantize_small_and_large_weights():
    for scale in (1e-42, 1e-38, 1e-30, 1e30, 1e38):
        w = (torch.randn(40, 256, generator=torch.Generator().manual_seed(1)).clamp(-2, 2) * scale).float()
        for zeros in (False, True):
            q = tl.quantize_q4(w.cuda(), 64, zeros, torch.float32)
            assert torch.equal(tl.dequantize_q4(q).cpu(), _quantized64(w, 64, zeros, torch.float32).float()), (scale, zeros)
    # a run with a NaN or an infinity comes back as such, its neighbours as they are
    w = torch.randn(20, 256, generator=torch.Generator().manual_seed(2))
    clean = tl.dequantize_q4(tl.quantize_q4(w.cuda(), 64)).cpu()
    w[3, 70] = float("nan")
    w[5, 200] = float("inf")
    back = tl.dequantize_q4(tl.quantize_q4(w.cuda(), 64)).cpu()
    bad = torch.zeros(20, 256, dtype=torch.bool)
    bad[3, 64:128] = True
    bad[5, 192:256] = True
    assert torch.equal(back[~bad], clean[~bad]) and not bool(torch.isfinite(back[bad]).any())


def test_gradients_of_the_layer():
    """Input and bias gradients against the formula in 64 bits and against differences."""
    M, N, K = 9, 50, 200
    packed, s, z, v64, mass = _weights(N, K, 64, True, torch.float32, 3)
    q = tl.pack_q4(packed.cuda(), s.cuda(), z.cuda(), K, 64)
    for t in (torch.float32, torch.bfloat16):
        x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).to(t).cuda().requires_grad_()
        b = torch.randn(N, generator=torch.Generator().manual_seed(2)).to(t).cuda().requires_grad_()
        gy = torch.randn(M, N, generator=torch.Generator().manual_seed(3)).to(t).cuda()
        tl.forward_q4(x, q, b).backward(gy)
        g64 = gy.double().cpu()
        # N products and the rounding of each weight to 32 bits, then the type
        tol = (N + 8) * 2.0 ** -24 * (g64.abs() @ v64.abs()) + torch.finfo(t).eps / 2 * (g64 @ v64).abs() * 1.01
        assert bool(((x.grad.double().cpu() - g64 @ v64).abs() <= tol).all())
        tol = M * 2.0 ** -24 * g64.abs().sum(0) + torch.finfo(t).eps / 2 * g64.sum(0).abs() * 1.01
        assert bool(((b.grad.double().cpu() - g64.sum(0)).abs() <= tol).all())
    # y is linear in x: a difference is exact up to the bar of the two products
    x0 = torch.randn(M, K, generator=torch.Generator().manual_seed(4))
    d = torch.randn(M, K, generator=torch.Generator().manual_seed(5))
    gy = torch.randn(M, N, generator=torch.Generator().manual_seed(6))
    x = x0.cuda().requires_grad_()
    tl.forward_q4(x, q).backward(gy.cuda())
    up, down = tl.forward_q4((x0 + d).cuda(), q), tl.forward_q4((x0 - d).cuda(), q)
    slope = float(((up - down).double().cpu() * gy.double()).sum() / 2)
    want = float((x.grad.double().cpu() * d.double()).sum())
    bar = (16 * 2 + 48) * 2.0 ** -24 * float(((x0.abs() + d.abs()).double() @ mass.t() * gy.double().abs()).sum()) * 2
    assert abs(slope - want) <= bar


def test_layer_modules_round_trip():
    torch.manual_seed(0)
    layer = tl.cake_linear(300, 130).cuda()
    held = tl.cake_linear_q4.of(layer, group=64, zeros=True)
    x = torch.randn(2, 7, 300, device="cuda")
    y = held(x)
    assert y.shape == (2, 7, 130)
    w = tl.dequantize_q4(held.weight_q4).double().cpu()
    want = x.double().cpu() @ w.t() + layer.bias.double().cpu()
    assert float((y.double().cpu() - want).abs().max()) <= (16 * 3 + 48) * 2.0 ** -24 * 300 * 4 * float(w.abs().max()) * 15
    other = tl.cake_linear_q4.of(tl.cake_linear(300, 130).cuda(), group=64, zeros=True)
    other.load_state_dict(held.state_dict())
    assert torch.equal(other(x), y)
    assert held(x.bfloat16()).dtype == torch.bfloat16
    cpu = tl.cake_linear_q4(cake.q4_of(held.packed.cpu(), 130, 300, 64, torch.bfloat16, True), held.bias.cpu())
    assert torch.equal(cpu(x.cpu()), y.cpu())


@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_captured_calls_on_two_graphs_and_streams(M):
    """Two graphs captured from the same weights replay side by side on streams of their own, with eager
    calls between, and every replay gives the eager result for the inputs of that moment."""
    N, K = 520, 1500
    packed, s, z, _, _ = _weights(N, K, 32, True, torch.float16, 5)
    q = tl.pack_q4(packed.cuda(), s.cuda(), z.cuda(), K, 32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(M, K, device="cuda", generator=gen) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            tl.forward_q4(x, q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, st in zip(xs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(tl.forward_q4(x, q))
        graphs.append(g)
    for replay in range(4):
        for x in xs:
            x.copy_(torch.randn(M, K, device="cuda", generator=gen))
        want = [tl.forward_q4(x, q) for x in xs]
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), replay


def test_refusals_on_the_device():
    N, K = 32, 128
    q = tl.quantize_q4(torch.ones(N, K, device="cuda"), 128)
    x, y = torch.ones(2, K, device="cuda"), torch.full((2, N), 7.0, device="cuda")
    lib = cake.load()
    off = torch.zeros(q.data.numel() + 16, dtype=torch.uint8, device="cuda")[4:]
    st = lib.cake_hip_linear_q4_forward(x.data_ptr(), off.data_ptr(), None, y.data_ptr(), _lib.F32, 2, N, K, 128, _lib.BF16, 0, None, None, None)
    assert st == _lib.ERR_ARG and b"aligned" in lib.cake_hip_last_error()
    assert lib.cake_hip_q4_quantize(x.data_ptr(), _lib.F32, off.data_ptr(), 2, K, 128, _lib.BF16, 0, None, None) == _lib.ERR_ARG
    host = np.zeros(1 << 16, np.uint8)
    st = lib.cake_hip_linear_q4_forward(x.data_ptr(), q.data.data_ptr(), None, y.data_ptr(), _lib.F32, 2, N, K, 128, _lib.BF16, 0,
                                        off.data_ptr(), None, None)
    assert st == _lib.ERR_ARG
    with pytest.raises(ValueError):
        tl.forward_q4(x.cpu(), q)
    torch.cuda.synchronize()
    assert bool((y == 7).all())
    del host


def test_operands_beyond_4_gb():
    """Weights of 4.2 GB (2.1 billion, as many as an operand may have): the last rows as good as the first."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    N, K = 65536, 32000
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(N, K, dtype=torch.bfloat16, device="cuda").normal_(0, 0.02, generator=gen)
    q = tl.quantize_q4(w, 64, True, torch.bfloat16)
    rows = torch.cat([torch.arange(0, 40), torch.arange(N - 40, N)]).cuda()
    v = _quantized64(w[rows].cpu(), 64, True, torch.bfloat16)
    back = tl.dequantize_q4(q, torch.bfloat16)
    assert torch.equal(back[rows].cpu(), v.float().bfloat16())
    del back
    for M in (1, 40):
        x = torch.randn(M, K, device="cuda", generator=gen)
        print(f"linear_q4 beyond 4 GB M={M}", flush=True)
        y = tl.forward_q4(x, q)[:, rows]
        # codes and zero points are at most 15, so s (code + zero) is at most 30 s, and s at most a fifteenth of twice the largest weight
        mass = x.double().cpu().abs().sum(1, keepdim=True) * (30 * 2 / 15 * float(w.abs().max()) * (1 + 2.0 ** -7))
        assert bool(((y.double().cpu() - x.double().cpu() @ v.t()).abs() <= (16 * (K // 128) + 48) * 2.0 ** -24 * mass).all())


def test_an_input_of_tiny_values():
    """Products of values down to 2^-100 keep their relative accuracy; below that pieces leave bf16's normal range."""
    N, K, M = 40, 256, 3
    packed, s, z, v64, mass = _weights(N, K, 64, True, torch.float32, 4)
    q = tl.pack_q4(packed.cuda(), s.cuda(), z.cuda(), K, 64)
    for rows in (M, 30):
        x = torch.randn(rows, K, generator=torch.Generator().manual_seed(4)) * 2.0 ** -100
        want = x.double() @ v64.t()
        tol = (16 * 2 + 48) * 2.0 ** -24 * (x.double().abs() @ mass.t())
        assert bool(((tl.forward_q4(x.cuda(), q).double().cpu() - want).abs() <= tol).all()), rows


def test_layer_without_tokens_or_columns():
    held = tl.cake_linear_q4.of(tl.cake_linear(300, 130).cuda(), group=64, zeros=True)
    assert held(torch.zeros(2, 0, 300, device="cuda")).shape == (2, 0, 130)
    assert held(torch.zeros(300, device="cuda")).shape == (130,)
    none = tl.cake_linear_q4(cake.q4_of(torch.zeros(0, dtype=torch.uint8, device="cuda"), 5, 0, 32, torch.float32, False), torch.arange(5.0, device="cuda"))
    for shape in ((2, 3, 0), (40, 0)):
        assert torch.equal(none(torch.zeros(shape, device="cuda")), torch.arange(5.0, device="cuda").expand(*shape[:-1], 5))


def test_weights_changed_before_the_backward_pass_are_noticed():
    q = tl.quantize_q4(torch.randn(32, 128, device="cuda"), 64)
    x = torch.randn(3, 128, device="cuda", requires_grad=True)
    y = tl.forward_q4(x, q)
    q.data.zero_()
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_captured_forward_and_backward_replay():
    """The whole step in one graph, replayed on changed inputs with eager work of the same sizes in between."""
    M, N, K = 40, 96, 320
    q = tl.quantize_q4(torch.randn(N, K, generator=torch.Generator().manual_seed(1)).cuda(), 64, True)
    x = torch.zeros(M, K, device="cuda", requires_grad=True)
    gy = torch.zeros(M, N, device="cuda")

    def eager(xs, g):
        leaf = xs.clone().requires_grad_()
        y = tl.forward_q4(leaf, q)
        return y.detach(), torch.autograd.grad(y, leaf, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(tl.forward_q4(x, q), x, gy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tl.forward_q4(x, q)
        gx, = torch.autograd.grad(y, x, gy)
    for i in range(4):
        gen = torch.Generator().manual_seed(10 + i)
        with torch.no_grad():
            x.copy_(torch.randn(M, K, generator=gen))
            gy.copy_(torch.randn(M, N, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        want, want_g = eager(x.detach(), gy)
        assert torch.equal(y, want) and torch.equal(gx, want_g), i


@pytest.mark.parametrize("kind", list(TYPES))
def test_few_rows_of_every_number_and_many_outputs(kind):
    """More outputs than 512 tiles, an odd number of tiles, and either side of every number of rows and columns at
    which the kernel changes."""
    N = 8200
    for K, group, zeros, rows in ((1111, 32, True, (1, 3, 4, 5, 6, 9, 10, 11, 16, 17, 24, 25, 31, 32, 33)), (300, 128, False, (2, 6, 10, 17, 32)),
                                  (640, 64, True, (5, 8, 20, 29))):
        packed, s, z, v64, mass = _weights(N, K, group, zeros, torch.float32 if group == 32 else torch.bfloat16, K)
        q = tl.pack_q4(packed.cuda(), s.cuda(), None if z is None else z.cuda(), K, group)
        for M in rows:
            print(f"linear_q4 M={M} N={N} K={K} {kind} group={group}", flush=True)
            x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(TYPES[kind]).cuda()
            _check(tl.forward_q4(x, q), x, v64, mass, None, K)
    for K in (8192, 8193):
        packed, s, z, v64, mass = _weights(40, K, 64, False, torch.float16, K)
        q = tl.pack_q4(packed.cuda(), s.cuda(), None, K, 64)
        for M in (10, 24, 25, 32):
            print(f"linear_q4 M={M} K={K} {kind}", flush=True)
            x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(TYPES[kind]).cuda()
            _check(tl.forward_q4(x, q), x, v64, mass, None, K)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_an_input_of_huge_values(kind):
    """Products of x and whole codes, or the sum of a row of x, pass 32 bits long before what they stand for does."""
    N, K = 40, 300
    for group, zeros in ((32, True), (64, False), (128, True), (128, False)):
        packed, s, z, v64, mass = _weights(N, K, group, zeros, torch.float32, 5)
        q = tl.pack_q4(packed.cuda(), s.cuda(), None if z is None else z.cuda(), K, group)
        for M in (1, 4, 9, 20, 30, 70, 200):
            x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).clamp(-3, 3)
            x = (x * (2.5e38 / float((x.double().abs() @ v64.abs().t()).max()))).to(TYPES[kind])      # no order of the sums overflows
            assert float(x.abs().max()) > 1e36
            print(f"linear_q4 huge M={M} {kind} group={group} zeros={zeros}", flush=True)
            _check(tl.forward_q4(x.cuda(), q), x, v64, mass, None, K)


def _on_device(y, x, v64, mass, bias, K, R=None):
    """_check with the 64-bit sums on the device"""
    x64, v, s = x.double(), v64.cuda(), mass.cuda()
    want = x64 @ v.t().contiguous()
    S = x64.abs() @ s.t().contiguous()
    if bias is not None:
        want, S = want + bias.double(), S + bias.double().abs()
    tol = (R or 16 * (-(-K // 128)) + 48) * 2.0 ** -24 * S + 2.0 ** -40
    if y.dtype != torch.float32:
        tol = tol + torch.finfo(y.dtype).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    far = (y.double() - want).abs() - tol
    assert y.shape == want.shape and bool((far <= 0).all()), float(far.max())


KINDS = [(group, zeros, scale) for zeros in (False, True) for group, scale in ((32, "bf16"), (64, "f16"), (128, "f32"))]


@pytest.mark.parametrize("shape", [(300, 16500, 200), (600, 8200, 200), (1100, 8200, 300), (2050, 4100, 300), (1030, 4111, 1500)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(TYPES))
def test_prompts_in_wide_bands(shape, kind):
    """What fills the device is taken in bands of 128 rows, or 256 for 16-bit x without zero points: last bands and strips
    that are partly filled, blocks that end inside K, every group size, with and without zero points."""
    M, N, K = shape
    for i, (group, zeros, scale) in enumerate(KINDS):
        packed, s, z, v64, mass = _weights(N, K, group, zeros, TYPES[scale], i)
        q = tl.pack_q4(packed.cuda(), s.cuda(), None if z is None else z.cuda(), K, group)
        gen = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randn(M, K, device="cuda", generator=gen).to(TYPES[kind])
        bias = torch.randn(N, device="cuda", generator=gen).to(TYPES[kind]) if i % 2 else None
        around = torch.full((M * N + 64,), 7.0, dtype=TYPES[kind], device="cuda")
        y = around[:M * N].view(M, N)
        print(f"linear_q4 M={M} N={N} K={K} {kind} group={group} zeros={zeros}", flush=True)
        cake.linear_q4_forward(x, q, bias, y, M, timed=False)
        _on_device(y, x, v64, mass, bias, K)
        assert bool((around[M * N:] == 7).all())


@pytest.mark.parametrize("rows", [1, 2, 5, 6, 10, 11, 40, 600])
def test_every_bit_of_a_32_bit_input_counts(rows):
    """One element of 24 significant bits a row, at the ends of steps, runs and blocks: a result is s (code - z) x with
    no more than 12 roundings in a row (three pieces' sums, zero points and scales, and their joining); without the last
    8 bits of x it would be off by up to 256 times 2^-24."""
    K, N = (200, 8200) if rows == 600 else (300, 75)
    columns = [c for c in (0, 7, 8, 31, 32, 63, 64, 95, 96, 127, 128, 191, 199, 255, 256, 287, 288, 299) if c < K]
    for i, (group, zeros, scale) in enumerate(KINDS):
        packed, s, z, v64, mass = _weights(N, K, group, zeros, TYPES[scale], 20 + i)
        q = tl.pack_q4(packed.cuda(), s.cuda(), None if z is None else z.cuda(), K, group)
        for turn in range(len(columns) if rows < 3 else 3):
            x = torch.zeros(rows, K)
            gen = torch.Generator().manual_seed(turn)
            bits = torch.randint(1 << 22, 1 << 23, (rows,), generator=gen) * 2 + 1      # 24 bits, the first and the last set
            for m in range(rows):
                x[m, columns[(turn + m) % len(columns)]] = float(bits[m]) * 2.0 ** -22 * (-1) ** m
            print(f"linear_q4 24 bits M={rows} group={group} zeros={zeros}", flush=True)
            _on_device(tl.forward_q4(x.cuda(), q), x.cuda(), v64, mass, None, K, R=12)


@pytest.mark.parametrize("kind", list(TYPES))
def test_inputs_with_outliers_and_an_offset(kind):
    """Columns a thousand times the others, some of them where every code is the zero point, and rows that do not sum to
    nothing: within the bar, whose S counts code and zero point apart."""
    N, K = 130, 700
    for group, zeros in ((32, True), (64, False), (128, True), (128, False)):
        packed, s, z, _, _ = _weights(N, K, group, zeros, torch.float32, 6)
        packed[:, 5::16] = 0x88
        k = torch.arange(K)
        code = ((packed[:, k // 2].int() >> (4 * (k % 2)).int()) & 15).double()
        if zeros:
            z = z.round()
            z[::2] = 8
        z64 = z.double()[:, k // group] if zeros else torch.full((N, K), 8.0, dtype=torch.float64)
        s64 = s.double()[:, k // group]
        q = tl.pack_q4(packed.cuda(), s.cuda(), z.cuda() if zeros else None, K, group)
        for M in (1, 4, 9, 20, 33, 200):
            x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)) + 3
            x[:, 10::32] *= 1000
            x = x.to(TYPES[kind]).cuda()
            print(f"linear_q4 outliers M={M} {kind} group={group} zeros={zeros}", flush=True)
            _on_device(tl.forward_q4(x, q), x, (code - z64) * s64, s64 * (code + z64), None, K)


@pytest.mark.parametrize("kind", list(TYPES))
def test_gradients_of_larger_layers(kind):
    """A layer of a thousand columns, rows from none to some hundreds, either gradient alone."""
    N, K, t = 1001, 1300, TYPES[kind]
    packed, s, z, v64, _ = _weights(N, K, 32, True, torch.bfloat16, 9)
    q = tl.pack_q4(packed.cuda(), s.cuda(), z.cuda(), K, 32)
    v = v64.cuda()
    for M in (0, 1, 17, 300):
        gen = torch.Generator(device="cuda").manual_seed(M)
        x0, gy = torch.randn(M, K, device="cuda", generator=gen).to(t), torch.randn(M, N, device="cuda", generator=gen).to(t)
        b0 = torch.randn(N, device="cuda", generator=gen).to(t)
        for need_x, need_b in ((True, True), (True, False), (False, True)):
            x, b = x0.clone().requires_grad_(need_x), b0.clone().requires_grad_(need_b)
            print(f"backward M={M} {kind} {need_x} {need_b}", flush=True)
            tl.forward_q4(x, q, b).backward(gy)
            g64 = gy.double()
            if need_x:
                want = g64 @ v
                # N products and the rounding of each weight to 32 bits, then the type (and fp16's last subnormal step)
                tol = (N + 8) * 2.0 ** -24 * (g64.abs() @ v.abs()) + (torch.finfo(t).eps / 2 * want.abs() * 1.01 + 2.0 ** -25 if t != torch.float32 else 0)
                assert x.grad.dtype == t and x.grad.shape == x.shape and bool(((x.grad.double() - want).abs() <= tol).all())
            if need_b:
                want = g64.sum(0)
                tol = M * 2.0 ** -24 * g64.abs().sum(0) + (torch.finfo(t).eps / 2 * want.abs() * 1.01 + 2.0 ** -25 if t != torch.float32 else 0)
                assert b.grad.dtype == t and bool(((b.grad.double() - want).abs() <= tol).all())


def test_a_workspace_in_host_memory_is_refused():
    N, K, M = 64, 128, 50
    q = tl.quantize_q4(torch.ones(N, K, device="cuda"), 128)
    x, y = torch.ones(M, K, device="cuda"), torch.full((M, N), 7.0, device="cuda")
    lib = cake.load()
    need = lib.cake_hip_linear_q4_workspace(M, N, K, _lib.F32)
    host = np.zeros(need + 16, np.uint8)
    at = host.ctypes.data + (-host.ctypes.data % 16)
    st = lib.cake_hip_linear_q4_forward(x.data_ptr(), q.data.data_ptr(), None, y.data_ptr(), _lib.F32, M, N, K, 128, _lib.BF16, 0, at, None, None)
    assert need > 0 and st == _lib.ERR_ARG and b"workspace" in lib.cake_hip_last_error()
    torch.cuda.synchronize()
    assert bool((y == 7).all()) and not host.any()


@pytest.mark.parametrize("N", [50, 8200])
@pytest.mark.parametrize("kind", list(TYPES))
def test_few_rows_under_every_kind_of_weights(kind, N):
    """Every group size with every type of scales, for the numbers of rows that fill a result register, one tile and two."""
    K = 300
    for group in (32, 64, 128):
        for i, scale in enumerate(TYPES):
            zeros = (group // 32 + i) % 2 == 0
            packed, s, z, v64, mass = _weights(N, K, group, zeros, TYPES[scale], 40 + i)
            q = tl.pack_q4(packed.cuda(), s.cuda(), None if z is None else z.cuda(), K, group)
            for M in (1, 5, 9, 18):
                x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(TYPES[kind]).cuda()
                print(f"linear_q4 M={M} N={N} {kind} group={group} scales={scale} zeros={zeros}", flush=True)
                _on_device(tl.forward_q4(x, q), x, v64, mass, None, K)
