"""GPU checks of orthogonalize (Newton-Schulz iterations) and of the optimiser on it, against the definition
in 64 bits.

The bar.  One iteration commits an error of at most C 2^-24 of its result's Frobenius norm -- each kept value to
2^-23 and each product to 2^-22, of either sign, sums over a side of which the random part grows with its root; C = 32 allows for sides up to
some hundreds -- and every later iteration enlarges a perturbation by at most the largest of |p(s)| / s
and |p'(s)| over the singular values it meets, L = 3.4445 for the usual coefficients (both at 0) and 1.5 for
(1.5, -0.5, 0).  So |x - x64|_F <= C 2^-24 sum_i |x_i|_F L^(steps - i), plus half a step of the type per entry.
All entries that a case can get wrong are of the order of the mean entry or above, far beyond that."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import cake_on_cpu_amd as cake
from cake_on_cpu_amd import _lib
from cake_on_cpu_amd import torch_linear as tl

pytestmark = pytest.mark.gpu

USUAL = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _reference(g, steps, c, eps, L):
    """x after `steps` in 64 bits, and the bar on the Frobenius norm of fp32 work"""
    x = g.double().cpu()
    norm = float(x.square().sum().sqrt())
    x = x / (norm + eps) if norm + eps > 0 else x
    tall = x.size(0) > x.size(1)
    if tall:
        x = x.t()
    bar = float(x.norm()) * L ** steps
    for i in range(1, steps + 1):
        a = x @ x.t()
        x = c[0] * x + (c[1] * a + c[2] * a @ a) @ x
        bar += float(x.norm()) * L ** (steps - i)
    return (x.t() if tall else x), 32 * 2.0 ** -24 * bar


def _check(out, g, steps, c=USUAL, eps=1e-7, L=3.4445):
    want, bar = _reference(g, steps, c, eps, L)
    t = out.dtype
    half_step = torch.finfo(t).eps / 2 * want.abs() if t != torch.float32 else torch.zeros_like(want)
    if t == torch.float16:
        half_step = half_step + 2.0 ** -25
    far = ((out.double().cpu() - want).abs() - half_step).clamp(min=0)
    assert out.shape == want.shape and float(far.norm()) <= bar * (1 + torch.finfo(t).eps), (float(far.norm()), bar)


def _gradient(m, n, seed, rank=None):
    g = torch.Generator().manual_seed(seed)
    r = rank or max(1, min(m, n) // 2)
    return torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g) * 1e-3 + 1e-4 * torch.randn(m, n, generator=g)


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (7, 1), (2, 2), (16, 16), (17, 15), (31, 33), (32, 32), (33, 32), (64, 64), (65, 200), (200, 65),
                                   (128, 128), (129, 130), (96, 500), (500, 96), (260, 300), (1, 3000), (3000, 2), (40, 4099)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(TYPES))
def test_orthogonalize_against_64_bits(shape, kind):
    for steps in (1, 2, 5):
        g = _gradient(*shape, seed=steps).to(TYPES[kind])
        print(f"orthogonalize {shape} {kind} steps={steps}", flush=True)
        out = tl.orthogonalize(g.cuda(), steps=steps)
        _check(out, g, steps)
        assert torch.equal(out, tl.orthogonalize(g.cuda(), steps=steps))


@pytest.mark.parametrize("shape", [(512, 1024), (1030, 520), (1100, 1100), (2100, 300)], ids=lambda s: "x".join(map(str, s)))
def test_orthogonalize_many_tiles(shape):
    for kind in ("f32", "bf16"):
        g = _gradient(*shape, seed=3).to(TYPES[kind])
        print(f"orthogonalize {shape} {kind}", flush=True)
        _check(tl.orthogonalize(g.cuda()), g, 5)


@pytest.mark.parametrize("shape", [(3, 20, 50), (2, 3, 130, 96), (5, 1, 9), (17, 64, 64)], ids=lambda s: "x".join(map(str, s)))
def test_batches_are_their_matrices(shape):
    flat = torch.stack([_gradient(*shape[-2:], seed=i) * 10.0 ** (i - 2) for i in range(int(np.prod(shape[:-2])))])
    g = flat.view(shape).cuda()
    print(f"orthogonalize batch {shape}", flush=True)
    out = tl.orthogonalize(g).view(flat.shape)
    for i, each in enumerate(flat):
        assert torch.equal(out[i], tl.orthogonalize(each.cuda())), i
        _check(out[i], each, 5)


def test_other_coefficients_and_convergence():
    g = _gradient(60, 90, 1, rank=60)
    _check(tl.orthogonalize(g.cuda(), steps=12, coefficients=(1.5, -0.5, 0.0)), g, 12, (1.5, -0.5, 0.0), L=1.5)
    # singular values that are all alike stay alike; the usual polynomial takes them near 1
    q = torch.linalg.qr(torch.randn(80, 80, generator=torch.Generator().manual_seed(2)))[0]
    s = torch.linalg.svdvals(tl.orthogonalize(q.cuda()).double().cpu())
    assert float(s.min()) > 0.6 and float(s.max()) < 1.3
    # a growing polynomial: values up to 5^3, kept under a smaller power of two
    g = _gradient(33, 70, 4)
    _check(tl.orthogonalize(g.cuda(), steps=3, coefficients=(5.0, 0.0, 0.0)), g, 3, (5.0, 0.0, 0.0), L=5.0)


def test_norms_of_every_size():
    """Squares that over- or underflow 32 bits; eps against the norm; zeros."""
    g = _gradient(40, 60, 5)
    for scale in (1e-30, 1e-12, 1e20, 1e33):
        each = (g.double() * scale).float()
        _check(tl.orthogonalize(each.cuda(), eps=0.0), each, 5, eps=0.0)
    small = (g.double() / float(g.double().norm()) * 1e-7).float()      # eps as large as the norm
    _check(tl.orthogonalize(small.cuda(), eps=1e-7), small, 5, eps=1e-7)
    for eps in (0.0, 1e-7):
        assert not bool(tl.orthogonalize(torch.zeros(33, 20, device="cuda"), eps=eps).any())


def test_nan_stays_in_its_matrix():
    g = torch.stack([_gradient(40, 70, i) for i in range(4)])
    clean = tl.orthogonalize(g.cuda())
    g[1, 3, 5] = float("nan")
    g[2, 0, 0] = float("inf")
    out = tl.orthogonalize(g.cuda())
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(out[2]).all())
    assert torch.equal(out[0], clean[0]) and torch.equal(out[3], clean[3])


def test_in_place_views_and_host_operands():
    g = _gradient(50, 77, 6)
    want = tl.orthogonalize(g.cuda())
    assert torch.equal(tl.orthogonalize(g.cuda().t().contiguous().t()), want)      # not contiguous
    same = g.cuda()
    cake.orthogonalize(same, same, 1, 50, 77, timed=False)
    assert torch.equal(same, want)
    around = torch.full((50 * 77 + 64,), 7.0, device="cuda")
    cake.orthogonalize(g.cuda(), around[32:32 + 50 * 77], 1, 50, 77, timed=False)
    assert torch.equal(around[32:32 + 50 * 77].view(50, 77), want)
    assert bool((around[:32] == 7).all()) and bool((around[32 + 50 * 77:] == 7).all())
    host = np.full((50, 77), np.nan, np.float32)
    assert cake.orthogonalize(np.ascontiguousarray(g.numpy()), host, 1, 50, 77) > 0
    assert np.array_equal(host, want.cpu().numpy())
    # a workspace that is not device memory, or off its alignment, is refused and nothing is written
    lib, out = cake.load(), torch.full((50, 77), 7.0, device="cuda")
    need = cake.orthogonalize_workspace(1, 50, 77)
    off = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    where = np.empty(need + 256, np.uint8)
    for ws in (off.data_ptr() + 16, where.ctypes.data + (-where.ctypes.data % 256)):
        assert lib.cake_hip_orthogonalize(g.cuda().data_ptr(), out.data_ptr(), _lib.F32, 1, 50, 77, 5, *USUAL, 1e-7, ws, None, None) == _lib.ERR_ARG
    torch.cuda.synchronize()
    assert bool((out == 7).all())


def test_captured_updates_side_by_side():
    gen = torch.Generator(device="cuda").manual_seed(1)
    for shape in ((3, 60, 100), (300, 200), (2100, 2300)):
        gs = [torch.randn(*shape, device="cuda", generator=gen) for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        for g, st in zip(gs, streams):
            with torch.cuda.stream(st):
                tl.orthogonalize(g)
        torch.cuda.synchronize()
        graphs, outs = [], []
        for g, st in zip(gs, streams):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                outs.append(tl.orthogonalize(g))
            graphs.append(graph)
        for replay in range(4):
            for g in gs:
                g.copy_(torch.randn(*shape, device="cuda", generator=gen))
            want = [tl.orthogonalize(g) for g in gs]
            torch.cuda.synchronize()
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
            torch.cuda.synchronize()
            for o, w in zip(outs, want):
                assert torch.equal(o, w), (shape, replay)


def test_contexts_take_turns_on_their_own_workspaces():
    g = _gradient(120, 200, 7).cuda()
    want = tl.orthogonalize(g)
    torch.cuda.synchronize()
    with cake.Context():
        out = torch.empty_like(g)
        cake.orthogonalize(g, out, 1, 120, 200)          # the context's buffer
        assert torch.equal(out, want)


def test_optimiser_steps_are_the_formula():
    """Three steps of cake_muon on matrices of like and unlike shapes, from gradients of the linear layer,
    against the same steps in 64 bits."""
    torch.manual_seed(0)
    shapes = [(40, 24), (40, 24), (24, 56)]
    layers = [tl.cake_linear(n, m, bias=False).cuda() for m, n in shapes]
    opt = tl.cake_muon([p for l in layers for p in l.parameters()], lr=0.05, momentum=0.9, weight_decay=0.1)
    w64 = [l.weight.detach().double().cpu() for l in layers]
    b64 = [torch.zeros_like(w) for w in w64]
    for step in range(3):
        opt.zero_grad()
        for layer in layers:
            x = torch.randn(30, layer.input_features, device="cuda")
            (layer(x) - 1).square().mean().backward()
        grads = [l.weight.grad.double().cpu() for l in layers]
        opt.step()
        bars = []
        for i, (m, n) in enumerate(shapes):
            b64[i] = 0.9 * b64[i] + grads[i]
            o, bar = _reference(grads[i] + 0.9 * b64[i], 5, USUAL, 1e-7, 3.4445)
            w64[i] = w64[i] * (1 - 0.05 * 0.1) - 0.05 * max(1.0, m / n) ** 0.5 * o
            bars.append(bar)
        for layer, w, bar in zip(layers, w64, bars):
            # the orthogonal part's bar, enlarged by what u's own rounding adds (2^-23 of its norm, L^5), and w's rounding
            tol = 0.05 * 1.4 * (bar + 2.0 ** -22 * 3.4445 ** 5) + 4 * 2.0 ** -24 * float(w.norm())
            assert float((layer.weight.detach().double().cpu() - w).norm()) <= tol * (step + 1), step


def test_a_layer_is_trained_held_in_4_bits_and_served():
    torch.manual_seed(1)
    layer = tl.cake_linear(192, 130).cuda()
    opt = tl.cake_muon([layer.weight], lr=0.02)
    target = torch.randn(192, 130, device="cuda") / 14
    for _ in range(4):
        x = torch.randn(256, 192, device="cuda")
        loss = (layer(x) - x @ target).square().mean()
        layer.zero_grad()
        loss.backward()
        opt.step()
    held = tl.cake_linear_q4.of(layer, group=64, zeros=True)
    w = layer.weight.detach().double().cpu()
    v = tl.dequantize_q4(held.weight_q4).double().cpu()
    # a code is off by half a step of its run, and the scale's bf16 rounding (2^-8) adds up to 2^-8 of 15 steps at the ends
    runs = w.view(130, 3, 64)
    step = (runs.amax(2).clamp(min=0) - runs.amin(2).clamp(max=0)) / 15
    assert bool(((w - v).view(130, 3, 64).abs() <= (0.5 + 0.5 + 15 * 2.0 ** -8) * step[:, :, None] * (1 + 2.0 ** -7)).all())
    for rows in (1, 6, 100):                             # one token, a few, a prompt
        x = torch.randn(rows, 192, device="cuda")
        want = x.double().cpu() @ v.t() + layer.bias.double().cpu()
        mass = x.double().cpu().abs() @ (step[:, torch.arange(192) // 64] * 31).t() + layer.bias.double().cpu().abs()
        assert bool(((held(x).double().cpu() - want).abs() <= (16 * 2 + 48) * 2.0 ** -24 * mass).all()), rows


def test_a_batch_beyond_4_gb():
    """2.2 billion values in one call: the last matrix as good as the first."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of device memory")
    batch, m, n = 530, 2048, 2048
    g = torch.empty(batch, m, n, dtype=torch.bfloat16, device="cuda").normal_(0, 1e-3, generator=torch.Generator(device="cuda").manual_seed(1))
    print("orthogonalize batch beyond 4 GB", flush=True)
    out = tl.orthogonalize(g, steps=2)
    for i in (0, batch - 1):
        x = g[i].double()
        x = x / (x.norm() + 1e-7)
        bar = float(x.norm()) * 3.4445 ** 2
        for step in (1, 2):
            a = x @ x.t().contiguous()
            x = USUAL[0] * x + (USUAL[1] * a + USUAL[2] * (a @ a)) @ x
            bar += float(x.norm()) * 3.4445 ** (2 - step)
        far = ((out[i].double() - x).abs() - 2.0 ** -8 * x.abs()).clamp(min=0)
        assert float(far.norm()) <= 32 * 2.0 ** -24 * bar * (1 + 2.0 ** -7), i
    torch.cuda.empty_cache()


def test_optimiser_leaves_empty_and_untouched_parameters_alone():
    a, b, c = (torch.nn.Parameter(torch.ones(s, device="cuda")) for s in ((4, 6), (0, 6), (5, 3)))
    opt = tl.cake_muon([a, b, c])
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    assert bool((c == 1).all()) and not bool((a == 1).any())


def test_a_row_of_more_than_2_to_the_25_columns():
    """Operands whose block rows pass 32 bits.  One row of norm 1 stays a multiple of itself, x (c0 + b) in every step; its
    pair, b's and the sum are off by 2^-23 each, relative to |c0| + |b|, which is at most 10 |c0 + b| on the way of 1."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    n = (1 << 25) + (1 << 20) + 5
    gen = torch.Generator(device="cuda").manual_seed(3)
    for shape in ((1, n), (n, 1)):
        g = torch.randn(shape, device="cuda", generator=gen)
        print(f"orthogonalize {shape}", flush=True)
        out = tl.orthogonalize(g).double().flatten()
        unit = g.double().flatten() / g.double().norm()
        along = float(out @ unit)
        assert 0.6 < along < 1.3
        assert float((out - along * unit).abs().max()) <= 5 * 10 * 3 * 2.0 ** -23 * 1.3 * float(unit.abs().max())
        del g, out, unit
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(64, 544), (64, 545), (30, 1216), (1217, 30), (50, 270), (20, 520), (33, 97), (97, 129), (96, 320), (90, 321), (128, 160), (110, 161)],
                         ids=lambda s: "x".join(map(str, s)))
def test_orthogonalize_at_the_ends_of_one_launch(shape):
    """The largest matrices that one workgroup takes, the smallest that it does not, and every kind of units between."""
    for kind in TYPES:
        g = _gradient(*shape, seed=sum(shape)).to(TYPES[kind])
        print(f"orthogonalize {shape} {kind}", flush=True)
        _check(tl.orthogonalize(g.cuda()), g, 5)
    three = torch.stack([_gradient(*shape, seed=s) for s in range(3)])
    out = tl.orthogonalize(three.cuda())
    for i in range(3):
        _check(out[i], three[i], 5)


@pytest.mark.parametrize("shape", [(300, 500), (700, 260), (3, 200, 330), (1, 5000), (40, 60)], ids=lambda s: "x".join(map(str, s)))
def test_the_first_step_reads_x_in_32_bits(shape):
    """With b = 0 a step is x = c0 x: x0's rounding and the product's, whatever the size of a row beside the others'."""
    for tall in (False, True):
        g = torch.randn(shape, generator=torch.Generator().manual_seed(4))
        if shape[-2] > 1:
            g[..., ::3, :] *= 1e-6
        g = g.transpose(-2, -1).contiguous() if tall else g
        print(f"orthogonalize c0 alone {tuple(g.shape)}", flush=True)
        out = tl.orthogonalize(g.cuda(), steps=1, coefficients=(1.5, 0.0, 0.0)).double().cpu()
        want = g.double()
        want = 1.5 * want / (want.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
        assert bool(((out - want).abs() <= 2.0 ** -23 * (1 + 2.0 ** -20) * want.abs()).all())


@pytest.mark.parametrize("shape", [(37, 1024, 2048), (35, 2048, 1000), (3, 6000, 5700)], ids=lambda s: "x".join(map(str, s)))
def test_a_batch_taken_in_passes(shape):
    """More values than one pass takes (37 matrices in 19 and 18, three singly): every matrix against the 64-bit iteration,
    in place as well, and nothing behind the last one is written."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of device memory")
    batch, m, n = shape
    gen = torch.Generator(device="cuda").manual_seed(5)
    room = torch.full((batch * m * n + 64,), 7.0, device="cuda")
    out = room[:-64].view(shape)
    g = torch.randn(shape, device="cuda", generator=gen) * torch.logspace(-4, 4, batch, device="cuda")[:, None, None]
    print(f"orthogonalize in passes {shape}", flush=True)
    ws = torch.empty(cake.orthogonalize_workspace(*shape), dtype=torch.uint8, device="cuda")
    cake.orthogonalize(g, out, *shape, steps=2, workspace=ws, timed=False)
    assert torch.equal(tl.orthogonalize(g, steps=2), out) and bool((room[-64:] == 7).all())
    for i in range(batch):
        x = g[i].double() if m <= n else g[i].double().t().contiguous()
        x = x / (x.norm() + 1e-7)
        bar = float(x.norm()) * 3.4445 ** 2
        for step in (1, 2):
            a = x @ x.t().contiguous()
            x = USUAL[0] * x + (USUAL[1] * a + USUAL[2] * (a @ a)) @ x
            bar += float(x.norm()) * 3.4445 ** (2 - step)
        assert float((out[i].double() - (x if m <= n else x.t())).norm()) <= 32 * 2.0 ** -24 * bar, i
    cake.orthogonalize(g, g, *shape, steps=2, workspace=ws, timed=False)
    assert torch.equal(g, out)
    del room, out, g, ws, x, a
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(2100, 2300), (2300, 2100), (1030, 4111), (4111, 1030), (4000, 4100), (5000, 3333)], ids=lambda s: "x".join(map(str, s)))
def test_orthogonalize_large_tiles(shape):
    """Every size of tile, sliced and not, with sides that are no multiple of it, after one step, two and five.  Few large
    singular values, so that the products weigh as much as x itself: a part left out of one of them is 2^-12 of the result.
    C of the bar above allows for sides of some 400; the random part of longer sums grows with their root."""
    m, n = shape
    gen = torch.Generator(device="cuda").manual_seed(m)
    g = torch.randn(m, 5, device="cuda", generator=gen) @ torch.randn(5, n, device="cuda", generator=gen) + 0.3 * torch.randn(m, n, device="cuda", generator=gen)
    for steps in (1, 2, 5):
        print(f"orthogonalize {shape} steps={steps}", flush=True)
        out = tl.orthogonalize(g, steps=steps)
        x = (g if m <= n else g.t().contiguous()).double()
        x = x / (x.norm() + 1e-7)
        bar = float(x.norm()) * 3.4445 ** steps
        for i in range(1, steps + 1):
            a = x @ x.t().contiguous()
            x = USUAL[0] * x + (USUAL[1] * a + USUAL[2] * (a @ a)) @ x
            bar += float(x.norm()) * 3.4445 ** (steps - i)
        far = float((out.double() - (x if m <= n else x.t())).norm())
        assert far <= 32 * max(1.0, (max(m, n) / 400) ** 0.5) * 2.0 ** -24 * bar, (far, bar)


def test_rows_of_very_different_size():
    """Rows down to 1e-7 of the others: each value within 2^-39 of the norm a kept value may be off by, enlarged as the bar
    above enlarges it, and the whole within that bar."""
    for shape in ((60, 100), (300, 500)):
        g = _gradient(*shape, seed=8) * torch.logspace(0, -7, shape[0])[:, None]
        print(f"orthogonalize rows of different size {shape}", flush=True)
        for steps in (1, 5):
            _check(tl.orthogonalize(g.cuda(), steps=steps), g, steps)


def test_the_optimiser_on_16_bit_layers():
    """Steps on bf16 and fp16 matrices, some of one shape, against the formula in 64 bits: state to 32 bits, weights to one rounding."""
    for t in (torch.bfloat16, torch.float16):
        gen = torch.Generator().manual_seed(1)
        shapes = [(40, 24), (40, 24), (200, 300)]
        ws = [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(t).cuda()) for s in shapes]
        w64 = [w.detach().double().cpu() for w in ws]
        b64 = [torch.zeros_like(w) for w in w64]
        opt = tl.cake_muon(ws, lr=0.05, momentum=0.9, weight_decay=0.1)
        bars = [0.0] * 3
        for step in range(3):
            for i, (m, n) in enumerate(shapes):
                ws[i].grad = _gradient(m, n, 10 * step + i).to(t).cuda()
                b64[i] = 0.9 * b64[i] + ws[i].grad.double().cpu()
                o, bar = _reference(ws[i].grad.double().cpu() + 0.9 * b64[i], 5, USUAL, 1e-7, 3.4445)
                scale = 0.05 * max(1.0, m / n) ** 0.5
                w64[i] = w64[i] * (1 - 0.05 * 0.1) - scale * o
                # the orthogonal part's bar, enlarged by what u's own rounding adds (2^-22 of its norm, L^5), and the 32-bit weight's roundings
                bars[i] += scale * (bar + 2.0 ** -22 * 3.4445 ** 5) + 4 * 2.0 ** -24 * float(w64[i].norm())
            opt.step()
            for w, want, bar in zip(ws, w64, bars):
                assert opt.state[w]["momentum"].dtype == opt.state[w]["weight"].dtype == torch.float32
                assert float((opt.state[w]["weight"].double().cpu() - want).norm()) <= bar, step
                assert torch.equal(w.detach(), opt.state[w]["weight"].to(t))
