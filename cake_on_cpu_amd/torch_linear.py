"""PyTorch operator over the C-ABI: the linear layer of the reference's only
framework binding (src/linear.cpp:12-107, python/cake.py:18-49), with the same
names -- forward / backward, cake_linear_function, cake_linear.

Tensors on a ROCm device are used in place through their device pointers on
torch's current stream; CPU tensors are staged by the library.  torch only
provides memory, streams and autograd bookkeeping; every product, transpose and
reduction runs in libcake_hip.so.

Beside it stand the same layer with 4-bit weights for serving (forward_q4, cake_linear_q4) and the
orthogonalised update of its weight in training (orthogonalize, cake_muon), which the reference lacks."""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd import forward_ad

from . import api


def _f32c(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype != torch.float32:
        raise TypeError(f"{what} must be float32, got {t.dtype}")
    return t.detach().contiguous()


def forward(cache_sz, input, weight, bias=None, weight_t=None):
    """output[M][N] = input[M][K] . weight[N][K]^T (+ bias).  `cache_sz` (the
    reference passes the host's L2/L3 sizes, src/linear.cpp:37) is accepted and
    unused: block sizes come from the device.  weight_t: the weights already
    transposed ([K][N]), from a caller that holds them that way; the library itself reads
    `weight` as it lies and needs no such copy."""
    if input.dim() != 2 or weight.dim() != 2 or input.size(1) != weight.size(1):
        raise ValueError(f"linear forward: input {tuple(input.shape)} does not match weight {tuple(weight.shape)}")
    M, K = input.shape
    N = weight.size(0)
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"linear forward: bias {tuple(bias.shape)} does not match {N} outputs")
    x = _f32c(input, "input")
    b = None if bias is None else _f32c(bias, "bias")
    out = torch.empty((M, N), dtype=torch.float32, device=input.device)
    # device tensors: no event timing, so the call only enqueues work on torch's current stream
    timed = not input.is_cuda
    if weight_t is not None:
        if tuple(weight_t.shape) != (K, N):
            raise ValueError(f"linear forward: weight_t {tuple(weight_t.shape)} is not {(K, N)}")
        api.linear_forward_wt(x, _f32c(weight_t, "weight_t"), b, out, M, N, K, timed=timed)
    else:
        api.linear_forward(x, _f32c(weight, "weight"), b, out, M, N, K, timed=timed)
    return out


def backward(cache_sz, grad_output, input, weight, bias=None, needs=(True, True, True)):
    """(grad_input, grad_weight, grad_bias) for grad_output[M][N]; entries whose
    `needs` flag is false (or grad_bias when bias is None) are returned as None."""
    M, K = input.shape
    N = weight.size(0)
    if tuple(grad_output.shape) != (M, N):
        raise ValueError(f"linear backward: grad_output {tuple(grad_output.shape)} is not {(M, N)}")
    g = _f32c(grad_output, "grad_output")
    x, w = _f32c(input, "input"), _f32c(weight, "weight")
    dev = grad_output.device
    gx = torch.empty((M, K), dtype=torch.float32, device=dev) if needs[0] else None
    gw = torch.empty((N, K), dtype=torch.float32, device=dev) if needs[1] else None
    gb = torch.empty((N,), dtype=torch.float32, device=dev) if (needs[2] and bias is not None) else None
    api.linear_backward(g, x if gw is not None else None, w if gx is not None else None, gx, gw, gb, M, N, K,
                        timed=not grad_output.is_cuda)
    return gx, gw, gb


class cake_linear_function(torch.autograd.Function):
    @staticmethod
    def forward(ctx, data, weight, bias=None, weight_t=None):
        ctx.save_for_backward(data, weight, bias)
        return forward(None, data, weight, bias, weight_t)

    @staticmethod
    def backward(ctx, grad_output):
        data, weight, bias = ctx.saved_tensors
        return (*backward(None, grad_output, data, weight, bias, ctx.needs_input_grad[:3]), None)


class cake_linear(nn.Module):
    """Drop-in for the reference's cake_linear (python/cake.py:33-49): weight
    [output_features][input_features] and bias drawn from U(-0.1, 0.1)."""

    def __init__(self, input_features, output_features, bias=True):
        super().__init__()
        self.input_features = input_features
        self.output_features = output_features
        self.weight = nn.Parameter(torch.empty(output_features, input_features).uniform_(-0.1, 0.1))
        if bias:
            self.bias = nn.Parameter(torch.empty(output_features).uniform_(-0.1, 0.1))
        else:
            self.register_parameter("bias", None)

    def forward(self, data):
        lead = data.shape[:-1]
        flat = data.reshape(-1, self.input_features)
        out = cake_linear_function.apply(flat, self.weight, self.bias)
        return out.reshape(*lead, self.output_features)

    def extra_repr(self):
        return f"input_features={self.input_features}, output_features={self.output_features}, bias={self.bias is not None}"


# ---- the layer with 4-bit weights -------------------------------------------------------


_is_tracing = torch._C._is_tracing   # (a lookup less: one token is bound by the host's call)


def _watched():
    """Whether torch has to see an operator although nothing needs its gradient: a trace records what becomes of
    tensors and not what is written through a pointer, and a dual tensor's tangent is not to be lost in silence."""
    return _is_tracing() or forward_ad._current_level >= 0


def _not_in_a_trace(what):
    if _is_tracing():
        raise RuntimeError(f"{what}: a trace cannot record what packs weights; pack them before it and trace the layer")


def pack_q4(codes, scales, zeros, in_features, group=128):
    """Packed weights from an existing checkpoint's tensors: codes[N][(K + 1) // 2] (uint8, even columns in the low
    half of a byte), scales and zeros (or None: 8) [N][ceil(K / group)]."""
    _not_in_a_trace("pack_q4")
    if codes.dim() != 2 or codes.size(1) != (in_features + 1) // 2:
        raise ValueError(f"pack_q4: codes {tuple(codes.shape)} do not hold {in_features} columns")
    if group not in (32, 64, 128):
        raise ValueError(f"pack_q4: group of {group} (32, 64 or 128)")
    want = (codes.size(0), -(-in_features // group))
    for t, what in ((scales, "scales"), (zeros, "zeros")):
        if t is not None and tuple(t.shape) != want:
            raise ValueError(f"pack_q4: {what} {tuple(t.shape)} are not {want}")
        if t is not None and t.device != codes.device:
            raise ValueError(f"pack_q4: {what} on {t.device}, codes on {codes.device}")
    return api.q4_pack(codes.contiguous(), scales.detach().contiguous(), None if zeros is None else zeros.detach().contiguous(),
                       codes.size(0), in_features, group)


def quantize_q4(weight, group=128, zeros=False, scale_dtype=torch.bfloat16):
    """A weight matrix in 4 bits with one scale (and, with `zeros`, one zero point) for `group` columns of a row."""
    _not_in_a_trace("quantize_q4")
    if weight.dim() != 2:
        raise ValueError(f"quantize_q4: weight {tuple(weight.shape)} is no matrix")
    return api.q4_quantize(weight.detach().contiguous(), *weight.shape, group=group, zeros=zeros, scale_dtype=scale_dtype)


def dequantize_q4(q, dtype=torch.float32):
    """The values that packed weights stand for, as a tensor [N][K]."""
    call = _dequantize_q4_function.apply if _is_tracing() else _dequantize_q4
    return call(q.data, q.N, q.K, q.group, q.scale_type, q.with_zeros, dtype)


def _dequantize_q4(packed, N, K, group, scale_type, with_zeros, dtype):
    w = torch.empty((N, K), dtype=dtype, device=packed.device)
    api.q4_dequantize(api.Q4Weight(packed, N, K, group, scale_type, with_zeros), w)
    return w


class _dequantize_q4_function(torch.autograd.Function):
    """As one operation of a trace, on plain numbers, which are the same in every trace; packed weights are constants."""

    @staticmethod
    def forward(ctx, packed, *args):
        return _dequantize_q4(packed, *args)


def _forward_q4(input, q, bias):
    if input.dim() != 2 or input.size(1) != q.K:
        raise ValueError(f"forward_q4: input {tuple(input.shape)} does not match {q.K} columns of weights")
    if not q.data.is_contiguous():
        raise TypeError("forward_q4: packed weights must be contiguous")
    if q.data.numel() < q.bytes:   # resized since they were made
        raise ValueError(f"forward_q4: packed weights hold {q.data.numel()} bytes, {q.bytes} needed")
    if bias is not None and (tuple(bias.shape) != (q.N,) or bias.dtype != input.dtype):
        raise ValueError(f"forward_q4: bias {tuple(bias.shape)} of {bias.dtype} does not match {q.N} outputs of {input.dtype}")
    if input.device != q.data.device or (bias is not None and bias.device != input.device):
        raise ValueError(f"forward_q4: input on {input.device}, weights on {q.data.device}")
    x, bias = input.contiguous(), None if bias is None else bias.contiguous()
    M = x.size(0)
    y = x.new_empty((M, q.N))
    if not x.is_cuda:
        api.linear_q4_forward(x, q, bias, y, M)
        return y
    # one token is a few microseconds of device time: straight into the C entry, which checks sizes, types and
    # devices itself
    t = api.element_type(x.dtype)
    lib = api.load()
    # a workspace from torch's allocator belongs to this call's stream, and to a graph if one is captured
    need = lib.cake_hip_linear_q4_workspace(M, q.N, q.K, t) if M > 1 else 0
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    api.check(lib.cake_hip_linear_q4_forward(x.data_ptr(), q.data.data_ptr(), None if bias is None else bias.data_ptr(), y.data_ptr(), t,
                                             M, q.N, q.K, q.group, q.scale_type, q.with_zeros, None if ws is None else ws.data_ptr(),
                                             api._torch_stream(torch, x.device), None), "forward_q4")
    return y


class cake_linear_q4_function(torch.autograd.Function):
    """Gradients of the layer for its input and bias; the packed weights are constants."""

    @staticmethod
    def forward(ctx, data, q, bias, packed=None):
        """packed: q's bytes once more, as a tensor that a trace connects with where they come from."""
        if packed is not None and packed is not q.data:   # replayed
            q = api.Q4Weight(packed, q.N, q.K, q.group, q.scale_type, q.with_zeros)
        ctx.q, ctx.dtype = q, data.dtype
        ctx.save_for_backward(q.data if packed is None else packed)   # to notice a change before the backward pass reads it
        return _forward_q4(data.detach(), q, None if bias is None else bias.detach())

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        _, q, M = ctx.saved_tensors, ctx.q, grad_output.size(0)
        g = grad_output.detach().float().contiguous()
        gx = torch.empty((M, q.K), dtype=torch.float32, device=g.device) if ctx.needs_input_grad[0] else None
        gb = torch.empty((q.N,), dtype=torch.float32, device=g.device) if ctx.needs_input_grad[2] else None
        w = dequantize_q4(q) if gx is not None else None
        api.linear_backward(g, None, w, gx, None, gb, M, q.N, q.K, timed=not g.is_cuda)
        return None if gx is None else gx.to(ctx.dtype), None, None if gb is None else gb.to(ctx.dtype), None


def forward_q4(input, q, bias=None):
    """output[M][N] = input[M][K] . v[N][K]^T (+ bias) with v in 4 bits (pack_q4, quantize_q4).  input is float32,
    float16 or bfloat16, bias and output likewise; sums are fp32, of codes and of zero points apart (include/cake_hip.h
    says what that leaves of outliers).  Differentiable in input and bias (reverse mode; a tangent of forward mode is refused)."""
    if (torch.is_grad_enabled() and (input.requires_grad or (bias is not None and bias.requires_grad))) or _watched():
        return cake_linear_q4_function.apply(input, q, bias, q.data)
    return _forward_q4(input, q, bias)


class cake_linear_q4(nn.Module):
    """cake_linear with its weight held in 4 bits: cake_linear_q4.of(layer) for a trained layer, or of
    packed weights.  The packed bytes are a buffer, so .to(device) and state_dict carry them."""

    def __init__(self, q, bias=None):
        super().__init__()
        self.input_features, self.output_features = q.K, q.N
        self.group, self.scale_type, self.with_zeros = q.group, q.scale_type, q.with_zeros
        self.register_buffer("packed", q.data)
        self.bias = None if bias is None else nn.Parameter(bias.detach().clone())

    @classmethod
    def of(cls, layer, group=128, zeros=False, scale_dtype=torch.bfloat16):
        """From a layer with .weight and .bias (cake_linear, nn.Linear)."""
        return cls(quantize_q4(layer.weight, group, zeros, scale_dtype), layer.bias)

    @property
    def weight_q4(self):
        return api.Q4Weight(self.packed, self.output_features, self.input_features, self.group, self.scale_type, self.with_zeros)

    def get_extra_state(self):
        """What the packed bytes were made for, a tensor as everything else that is stored."""
        return torch.tensor([self.output_features, self.input_features, self.group, self.scale_type, int(self.with_zeros)])

    def set_extra_state(self, state):
        pass   # compared before anything is copied

    def _load_from_state_dict(self, state_dict, prefix, *args):
        state = state_dict.get(prefix + "_extra_state")
        if state is not None and state.tolist() != self.get_extra_state().tolist():
            raise ValueError(f"cake_linear_q4: stored weights are {state.tolist()} (outputs, inputs, group, scale type, zeros), "
                             f"this layer's {self.get_extra_state().tolist()}")
        super()._load_from_state_dict(state_dict, prefix, *args)

    def forward(self, data):
        if data.dim() == 0 or data.size(-1) != self.input_features:
            raise ValueError(f"cake_linear_q4: input {tuple(data.shape)} does not match {self.input_features} columns of weights")
        flat = data.flatten(0, -2) if data.dim() > 1 else data.unsqueeze(0)   # (no number of rows that a trace would keep)
        bias = None if self.bias is None else self.bias.to(data.dtype)
        return forward_q4(flat, self.weight_q4, bias).reshape(*data.shape[:-1], self.output_features)

    def extra_repr(self):
        return (f"input_features={self.input_features}, output_features={self.output_features}, bias={self.bias is not None}, "
                f"group={self.group}, zeros={self.with_zeros}")


# ---- the update of a weight matrix in training ---------------------------------------------


def orthogonalize(grad, steps=5, coefficients=api.NEWTON_SCHULZ, eps=1e-7):
    """Newton-Schulz iterations on the last two dimensions (leading ones are a batch): a tensor like `grad` whose
    matrices have their singular values moved close to 1.  Not differentiable.  Rows and columns down to 1e-3 of the others
    are as exact as these, smaller ones less (include/cake_hip.h)."""
    if grad.dim() < 2:
        raise ValueError(f"orthogonalize: {tuple(grad.shape)} is no matrix")
    call = _orthogonalize_function.apply if _is_tracing() else _orthogonalize
    return call(grad.detach(), steps, coefficients, eps)


class _orthogonalize_function(torch.autograd.Function):
    """As one operation of a trace."""

    @staticmethod
    def forward(ctx, grad, steps, coefficients, eps):
        return _orthogonalize(grad, steps, coefficients, eps)


def _orthogonalize(grad, steps, coefficients, eps):
    rows, cols = grad.shape[-2:]
    g = grad.contiguous()
    out = torch.empty_like(g)
    if g.numel() == 0:
        return out
    batch = g.numel() // (rows * cols)
    ws = torch.empty(api.orthogonalize_workspace(batch, rows, cols), dtype=torch.uint8, device=g.device) if g.is_cuda else None
    api.orthogonalize(g, out, batch, rows, cols, steps, coefficients, eps, workspace=ws, timed=not g.is_cuda)
    return out


# Values of matrices that the optimiser copies together for one call: what the library takes in one pass, too
_TOGETHER = 1 << 26


class cake_muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates for weight matrices (cake_linear.weight and the like; biases and
    other vectors belong to another optimiser):
        b = momentum * b + grad,  u = grad + momentum * b  (b without nesterov)
        w = w - lr * weight_decay * w - lr * sqrt(max(1, rows / cols)) * orthogonalize(u)
    Matrices of one shape are orthogonalised together, up to 2^26 values in a call.  The state is kept in fp32 whatever the
    parameters' type (float32, float16, bfloat16): the momentum, and of a 16-bit w an fp32 copy that the formula runs on and
    w is rounded from, so that updates below a step of w's type add up.  A w that was set from elsewhere counts as it was set."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=api.NEWTON_SCHULZ,
                 eps=1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps))

    def add_param_group(self, param_group):
        params = param_group["params"]
        if not isinstance(params, set):   # (which the base class refuses: it has no order)
            params = [params] if isinstance(params, torch.Tensor) else list(params)
            for w in params:
                w = w[1] if isinstance(w, tuple) else w   # (name, parameter)
                if isinstance(w, torch.Tensor) and w.dim() != 2:
                    raise ValueError(f"cake_muon: parameter {tuple(w.shape)} is no matrix")
        super().add_param_group({**param_group, "params": params})

    def load_state_dict(self, state_dict):
        """As the base class does, but without rounding the state to the parameters' type."""
        given = []
        hook = self.register_load_state_dict_pre_hook(lambda _, d: given.append(d))   # what other hooks made of it
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
        given = given[-1]
        names = [n for group in given["param_groups"] for n in group["params"]]
        for n, w in zip(names, (w for group in self.param_groups for w in group["params"])):
            for key, value in given["state"].get(n, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[w][key] = value.detach().to(device=w.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check()
        for group in self.param_groups:
            alike = {}
            for w in group["params"]:
                if w.grad is not None and w.numel() != 0:
                    alike.setdefault((tuple(w.shape), w.dtype, w.device), []).append(w)
            for (shape, _, _), ws in alike.items():
                some = max(1, _TOGETHER // (shape[0] * shape[1]))
                for i in range(0, len(ws), some):
                    self._update(group, ws[i:i + some])
        return loss

    def _check(self):
        """Raises for what cannot be taken, before anything is changed."""
        for group in self.param_groups:
            api.orthogonalize_check(group["steps"], group["coefficients"], group["eps"])
            for w in group["params"]:
                if w.grad is None or w.numel() == 0:
                    continue
                if w.grad.layout != torch.strided or w.grad.shape != w.shape:
                    raise TypeError(f"cake_muon: gradient {tuple(w.grad.shape)} of {w.grad.layout} for a matrix {tuple(w.shape)}")
                api.element_type(w.dtype)
                if w.is_cuda and w.device.index != api.device_info().device:
                    raise ValueError(f"cake_muon: parameter on {w.device}, the library works on device {api.device_info().device}")

    def _update(self, group, ws):
        rows, cols = ws[0].shape
        momentum, rate = group["momentum"], group["lr"] * max(1.0, rows / cols) ** 0.5
        us = torch.empty((len(ws), rows, cols), dtype=torch.float32, device=ws[0].device)
        for u, w in zip(us, ws):
            state = self.state[w]
            if "momentum" not in state:
                state["momentum"] = torch.zeros_like(w, dtype=torch.float32)
            b = state["momentum"].mul_(momentum).add_(w.grad)
            if group["nesterov"]:
                torch.add(w.grad, b, alpha=momentum, out=u)
            else:
                u.copy_(b)
        for w, done in zip(ws, orthogonalize(us, group["steps"], group["coefficients"], group["eps"])):
            full = w if w.dtype == torch.float32 else self._in_32_bits(w)
            if group["weight_decay"]:
                full.mul_(1 - group["lr"] * group["weight_decay"])
            full.add_(done, alpha=-rate)
            if full is not w:
                w.copy_(full)

    def _in_32_bits(self, w):
        state = self.state[w]
        if "weight" not in state:
            state["weight"] = w.float()
        else:   # entries that are no longer what was rounded from here
            state["weight"].copy_(torch.where(state["weight"].to(w.dtype) == w, state["weight"], w.float()))
        return state["weight"]
