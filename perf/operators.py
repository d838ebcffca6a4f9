"""Operators of large language models around the linear layer, as cases that can be timed and checked.

Three operators that belong to one weight matrix w[N][K] of a linear layer:

* `linear_q4`: y[M][N] = x[M][K] . v[N][K]^T (+ bias[N]) where the weights are held in 4 bits.  Code
  q[n][k] in 0..15 stands for v = (q - z) * s with one scale s and one zero point z for each run of
  `group` weights of a row (z = 8 where a layer keeps none).  The input rows are one token (a step of
  generation), a few (several users' steps) or many (a prompt).
* `quantize_q4`: w[N][K] to such codes, scales and zero points.  Without zero points
  s = max|w| / 7 and q = clamp(round(w / s), -8, 7) + 8; with them, lo = min(w, 0), hi = max(w, 0),
  s = (hi - lo) / 15, z = clamp(round(-lo / s), 0, 15) and q = clamp(round(w / s) + z, 0, 15); s is
  rounded to 32 bits and to the type it is kept in before anything is divided by it, and the
  ratios are rounded as real numbers, ties to even.  The codes are returned as the values v that
  they stand for.
* `orthogonalize`: Newton-Schulz iterations on the update g[m][n] of a weight matrix.
  x = g / (|g|_F + eps), then `steps` times a = x x^T, x = c0 x + (c1 a + c2 a a) x; for m > n the
  same on the transpose.  A batch of matrices of one shape is one call.

`own` is False for the plain forms (elementary torch operations in 32 bits) and True for this
package's kernels."""
import math

import torch

own = False

GROUPS = (32, 64, 128)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one token of one user through a square projection: the launch is most of the time
        {"name": "token_4096", "op": "linear_q4", "M": 1, "N": 4096, "K": 4096, "group": 128, "zeros": False, "bias": False, "type": "bfloat16", "scales": "bfloat16"},
        # one token through the wide half of a feed-forward layer, weights of a checkpoint with zero points
        {"name": "token_14336", "op": "linear_q4", "M": 1, "N": 14336, "K": 4096, "group": 64, "zeros": True, "bias": False, "type": "float16", "scales": "float16"},
        # one token in full precision through the largest matrix of the matrix-vector benchmark, the smallest groups
        {"name": "token_16384", "op": "linear_q4", "M": 1, "N": 16384, "K": 16384, "group": 32, "zeros": True, "bias": True, "type": "float32", "scales": "float32"},
        # the steps of eight users together, down projection of a feed-forward layer
        {"name": "batch_8", "op": "linear_q4", "M": 8, "N": 4096, "K": 14336, "group": 128, "zeros": False, "bias": False, "type": "bfloat16", "scales": "bfloat16"},
        # a batch and a layer of odd sizes: rows that no vector load divides, a last group that is short
        {"name": "batch_33_odd", "op": "linear_q4", "M": 33, "N": 8190, "K": 4099, "group": 64, "zeros": True, "bias": True, "type": "float32", "scales": "float32"},
        # a prompt
        {"name": "prompt_2048", "op": "linear_q4", "M": 2048, "N": 14336, "K": 4096, "group": 128, "zeros": False, "bias": False, "type": "bfloat16", "scales": "bfloat16"},
        # a trained layer made ready for serving, and one of odd sizes with zero points
        {"name": "quantize_14336", "op": "quantize_q4", "N": 14336, "K": 4096, "group": 128, "zeros": False, "type": "float32", "scales": "bfloat16"},
        {"name": "quantize_odd", "op": "quantize_q4", "N": 2111, "K": 4099, "group": 32, "zeros": True, "type": "bfloat16", "scales": "float32"},
        # the updates of many small projections of one shape, together
        {"name": "update_small", "op": "orthogonalize", "batch": 16, "m": 96, "n": 130, "steps": 5, "type": "float32"},
        # a projection's update in mixed precision
        {"name": "update_1024", "op": "orthogonalize", "batch": 1, "m": 1024, "n": 4096, "steps": 5, "type": "bfloat16"},
        # a square projection's update
        {"name": "update_4096", "op": "orthogonalize", "batch": 1, "m": 4096, "n": 4096, "steps": 5, "type": "float32"},
        # a feed-forward layer's update: more rows than columns
        {"name": "update_14336", "op": "orthogonalize", "batch": 1, "m": 14336, "n": 4096, "steps": 5, "type": "float32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("linear_q4", "linear_q4", "quantize_q4", "orthogonalize"))
    some = rng.choice(("float32", "float16", "bfloat16"))
    if kind == "orthogonalize":
        largest = work(listed()[-1])["flops"]
        while True:
            case = {"op": kind, "batch": _log(rng, 1, 16), "m": _log(rng, 16, 14336), "n": _log(rng, 16, 14336), "steps": rng.randint(1, 6), "type": some}
            if work(case)["flops"] <= largest and case["batch"] * case["m"] * case["n"] <= 14336 * 4096:
                return case
    N, K = _log(rng, 64, 16384), _log(rng, 64, 16384)
    case = {"op": kind, "N": N, "K": K, "group": rng.choice(GROUPS), "zeros": rng.random() < 0.5, "type": some,
            "scales": rng.choice(("float32", "bfloat16") if kind == "quantize_q4" else ("float32", "float16", "bfloat16"))}
    if kind == "linear_q4":
        M = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
        case |= {"M": max(1, min(M, 2048 * 14336 * 4096 // (N * K))), "bias": rng.random() < 0.5}
    return case


def _width(name):
    return 4 if name == "float32" else 2


def work(case):
    if case["op"] == "orthogonalize":
        # a and a a are symmetric: half of each is computed
        m, n = sorted((case["m"], case["n"]))
        values = case["batch"] * case["m"] * case["n"]
        return {"bytes": 2 * values * _width(case["type"]), "flops": case["batch"] * case["steps"] * (3 * m * m * n + m * m * m)}
    N, K = case["N"], case["K"]
    groups = N * -(-K // case["group"])
    held = N * K // 2 + groups * _width(case["scales"]) * (2 if case["zeros"] else 1)
    if case["op"] == "quantize_q4":
        return {"bytes": N * K * _width(case["type"]) + 2 * held + N * K * 4, "flops": 6 * N * K}
    M = case["M"]
    values = M * K + M * N + (N if case["bias"] else 0)
    return {"bytes": held + values * _width(case["type"]), "flops": 2 * M * N * K}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    if case["op"] == "orthogonalize":
        # a gradient: a sum over samples with falling weights, and noise
        b, m, n = case["batch"], case["m"], case["n"]
        rank = max(1, min(m, n, 256) // 2)
        falling = torch.linspace(0, -3, rank, device="cuda").exp()
        g = 1e-3 * (torch.bmm(normal(b, m, rank) * falling, normal(b, rank, n)) + 0.5 * normal(b, m, n))
        return {"case": case, "g": (g if b > 1 else g[0]).to(kind)}
    N, K = case["N"], case["K"]
    if case["op"] == "quantize_q4":
        # weights of rows of different sizes
        return {"case": case, "w": (normal(N, K) * (0.02 * (0.5 * normal(N, 1)).exp())).to(kind)}
    groups = -(-K // case["group"])
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (0.005 * (0.3 * normal(N, groups)).exp()).to(TYPES[case["scales"]])
    zeros = torch.randint(4, 12, (N, groups), generator=gen, device="cuda").to(scales.dtype) if case["zeros"] else None
    state = {"case": case, "x": normal(case["M"], K).to(kind), "bias": normal(N).to(kind) if case["bias"] else None}
    if own:
        from cake_on_cpu_amd import torch_linear
        return state | {"weight": torch_linear.pack_q4(codes, scales, zeros, K, case["group"])}
    return state | {"codes": codes, "scales": scales, "zeros": zeros}


def run(state):
    return {"linear_q4": _linear_q4, "quantize_q4": _quantize_q4, "orthogonalize": _orthogonalize}[state["case"]["op"]](state)


def _linear_q4(state):
    case, x = state["case"], state["x"]
    if own:
        from cake_on_cpu_amd import torch_linear
        return torch_linear.forward_q4(x, state["weight"], state["bias"])
    codes, K = state["codes"], case["K"]
    q = torch.stack((codes & 15, codes >> 4), dim=2).flatten(1)[:, :K].float()
    s = state["scales"].float().repeat_interleave(case["group"], dim=1)[:, :K]
    z = state["zeros"].float().repeat_interleave(case["group"], dim=1)[:, :K] if case["zeros"] else 8.0
    y = torch.matmul(x.float(), ((q - z) * s).t())
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(x.dtype)


def _quantize_q4(state):
    case, w = state["case"], state["w"]
    if own:
        from cake_on_cpu_amd import torch_linear
        held = torch_linear.quantize_q4(w, group=case["group"], zeros=case["zeros"], scale_dtype=TYPES[case["scales"]])
        return torch_linear.dequantize_q4(held, torch.float32)
    N, K, group = case["N"], case["K"], case["group"]
    groups = -(-K // group)
    padded = torch.zeros((N, groups * group), device=w.device)
    padded[:, :K] = w
    # 64 bits: a ratio next to a half must not be rounded onto it
    g = padded.view(N, groups, group).double()
    if case["zeros"]:
        lo, hi = g.amin(2, keepdim=True).clamp(max=0), g.amax(2, keepdim=True).clamp(min=0)
        s = ((hi - lo) / 15).float().to(TYPES[case["scales"]]).double()
        z = torch.where(s > 0, torch.round(-lo / s), 8.0).clamp(0, 15)
    else:
        s = (g.abs().amax(2, keepdim=True) / 7).float().to(TYPES[case["scales"]]).double()
        z = 8.0
    q = torch.where(s > 0, torch.round(g / s), 0.0).add(z).clamp(0, 15)
    return ((q - z) * s).view(N, -1)[:, :K].float()


def _orthogonalize(state):
    g, steps = state["g"], state["case"]["steps"]
    if own:
        from cake_on_cpu_amd import torch_linear
        return torch_linear.orthogonalize(g, steps=steps, coefficients=COEFFICIENTS, eps=EPS)
    c0, c1, c2 = COEFFICIENTS
    tall = g.size(-2) > g.size(-1)
    x = g.float()
    if tall:
        x = x.transpose(-2, -1).contiguous()
    norm = x.double().square().sum(dim=(-2, -1), keepdim=True).sqrt()
    x = (x / (norm + EPS)).float()
    for _ in range(steps):
        a = torch.matmul(x, x.transpose(-2, -1))
        x = c0 * x + torch.matmul(c1 * a + c2 * torch.matmul(a, a), x)
    if tall:
        x = x.transpose(-2, -1).contiguous()
    return x.to(g.dtype)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "orthogonalize":
        x = state["g"].double()
        left = x.size(-2) <= x.size(-1)
        x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + EPS)
        for _ in range(case["steps"]):
            t = x.transpose(-2, -1).contiguous()
            # the small square is x x^T on the left of x, or x^T x on its right: the same polynomial
            a = x @ t if left else t @ x
            p = COEFFICIENTS[2] * (a @ a) + COEFFICIENTS[1] * a
            p.diagonal(dim1=-2, dim2=-1).add_(COEFFICIENTS[0])
            x = p @ x if left else x @ p
        return x
    K, group = case["K"], case["group"]
    at = torch.arange(K, device="cuda") // group
    if case["op"] == "quantize_q4":
        w = state["w"].double()
        small = torch.full((case["N"], int(at[-1]) + 1), 0.0, device="cuda", dtype=torch.float64)
        each = at.expand(case["N"], K)
        hi, lo = small.scatter_reduce(1, each, w, "amax"), small.scatter_reduce(1, each, w, "amin")
        s = ((hi - lo) / 15 if case["zeros"] else torch.maximum(hi, -lo) / 7).float().to(TYPES[case["scales"]]).double()
        ratio = torch.where(s[:, at] > 0, w / s[:, at], 0.0).round()
        z = torch.where(s > 0, (-lo / s).round(), 8.0).clamp(0, 15)[:, at] if case["zeros"] else 8
        return (torch.clamp(ratio + z, 0, 15) - z) * s[:, at]
    k = torch.arange(K, device="cuda")
    q = (state["codes"][:, k // 2].int() >> (4 * (k % 2)).int()) & 15
    z = state["zeros"].double()[:, at] if case["zeros"] else 8
    y = state["x"].double() @ ((q.double() - z) * state["scales"].double()[:, at]).t().contiguous()
    return y + state["bias"].double() if case["bias"] else y
