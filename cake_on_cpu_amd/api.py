"""Host-side mirror of the reference's operator interface for the fp32 GEMM path.

Names, argument order and meaning follow include/cake.h, include/tiling.h,
include/packing.h, examples/cake_gemv.cpp and examples/cake_conv.cpp of
vnatesh/CAKE_on_CPU, so code (and tests) written against the reference read the
same here.  Matrices are float32, C-contiguous numpy arrays (host memory, staged
by the library) or torch ROCm tensors (used in place through their device
pointer, on torch's current stream)."""
from __future__ import annotations

import ctypes as C
import os
import re
import subprocess

import numpy as np

from . import _lib
from ._lib import KMN, MKN, NKM, NA, BlkDims, CakeHipError, CpuCntx, DeviceInfo, Plan, check, load


# ----------------------------------------------------------------------------
# array plumbing
# ----------------------------------------------------------------------------
def _is_torch(a) -> bool:
    return hasattr(a, "data_ptr") and hasattr(a, "is_contiguous")


def _ptr(a, what: str) -> int:
    if a is None:
        raise ValueError(f"{what} is None")
    if _is_torch(a):
        import torch
        if a.dtype != torch.float32 or not a.is_contiguous():
            raise TypeError(f"{what} must be a contiguous float32 tensor")
        return a.data_ptr()
    if not isinstance(a, np.ndarray) or a.dtype != np.float32 or not a.flags["C_CONTIGUOUS"]:
        raise TypeError(f"{what} must be a C-contiguous float32 numpy array or torch tensor")
    return a.ctypes.data


def _stream(*arrays) -> int:
    """torch's current HIP stream when any operand lives on the GPU, else the default stream."""
    for a in arrays:
        if _is_torch(a) and a.is_cuda:
            import torch
            return _torch_stream(torch, a.device)
    return 0


def _torch_stream(torch, device) -> int:
    """The handle of torch's current stream on `device`, without the stream object where this torch
    has the short way (0.1 us instead of 1.7: a short kernel's call is bound by the host).  The default stream's
    is 0 in torch and has a name of its own here: a 0 would be the stream of the current context, which does not
    wait for what torch has enqueued."""
    short = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if short is None or device.index is None:
        return torch.cuda.current_stream(device).cuda_stream or _lib.NULL_STREAM
    return short(device.index) or _lib.NULL_STREAM


def _numel(a) -> int:
    return a.numel() if _is_torch(a) else a.size


def _empty_like_kind(ref, shape):
    if _is_torch(ref):
        import torch
        return torch.empty(shape, dtype=torch.float32, device=ref.device)
    return np.empty(shape, dtype=np.float32)


def _need(a, n: int, what: str):
    if _numel(a) < n:
        raise ValueError(f"{what} holds {_numel(a)} elements, {n} needed")


# ----------------------------------------------------------------------------
# machine description and block sizing (include/tiling.h:15-41)
# ----------------------------------------------------------------------------
def _lscpu_cache(level: int) -> int:
    try:
        col = "ONE-SIZE" if level < 3 else "ALL-SIZE"
        out = subprocess.run(["lscpu", f"--caches=NAME,{col}"], capture_output=True, text=True, timeout=10).stdout
        for line in out.splitlines():
            if line.strip().startswith(f"L{level}"):
                m = re.search(r"(\d+)([KMG])", line)
                if m:
                    return int(m.group(1)) << {"K": 10, "M": 20, "G": 30}[m.group(2)]
    except Exception:
        pass
    return 0


def _physical_cores() -> int:
    logical = os.cpu_count() or 1
    try:
        out = subprocess.run(["lscpu"], capture_output=True, text=True, timeout=10).stdout
        tpc = int(re.search(r"Thread\(s\) per core:\s*(\d+)", out).group(1))
        sockets = int(re.search(r"Socket\(s\):\s*(\d+)", out).group(1))
        return max(1, logical // (tpc * sockets))
    except Exception:
        return logical


def cake_query_cntx() -> CpuCntx:
    """cake_query_cntx (src/block_sizing.cpp:40-75): host cache sizes and physical core
    count, m_r x n_r = 6 x 16.  On the GPU these only shape the reference-compatible
    blk_dims_t / packed layouts; the kernels are planned from the device instead."""
    cx = CpuCntx()
    cx.alpha_n = 1.0
    cx.mr, cx.nr = 6, 16
    cx.L1 = _lscpu_cache(1) or (32 << 10)
    cx.L2 = _lscpu_cache(2) or (1 << 20)
    cx.L3 = _lscpu_cache(3) or (32 << 20)
    cx.ncores = _physical_cores()
    return cx


_DEFAULT_CNTX = None


def _default_cntx() -> CpuCntx:
    """What a NULL cake_cntx stands for (src/cake_sgemm.cpp:14-16): the host's own description,
    queried once per process here instead of on every call."""
    global _DEFAULT_CNTX
    if _DEFAULT_CNTX is None:
        _DEFAULT_CNTX = cake_query_cntx()
    cx = CpuCntx()
    C.memmove(C.byref(cx), C.byref(_DEFAULT_CNTX), C.sizeof(CpuCntx))
    return cx


def update_mr_nr(cake_cntx: CpuCntx, m_r: int, n_r: int) -> None:
    """update_mr_nr (src/block_sizing.cpp:78-83)."""
    cake_cntx.mr, cake_cntx.nr = m_r, n_r


def init_block_dims(M, N, K, p, cake_cntx: CpuCntx, sch=NA, argv=None, type_size=4,
                    mcu=0, kcu=0, ncu=0, x: BlkDims | None = None) -> BlkDims:
    """init_block_dims (src/block_sizing.cpp:465-595).  Returns (and fills) blk_dims_t."""
    x = BlkDims() if x is None else x
    check(load().cake_hip_init_block_dims(M, N, K, p, C.byref(cake_cntx), sch, mcu, kcu, ncu, C.byref(x)),
          "init_block_dims")
    return x


def grid_dims_2d(M, N, K, p, ncores=0) -> int:
    """pn of the reference's pm x pn grid of cores (src/block_sizing.cpp:596-634): the factor of p
    closest to sqrt(p N / M).  Host arithmetic."""
    return load().cake_hip_grid_dims_2d(M, N, K, p, ncores)


def init_block_dims_2d(M, N, K, p, cake_cntx: CpuCntx, sch=NA, argv=None, type_size=4,
                       mcu=0, kcu=0, ncu=0) -> BlkDims:
    """init_block_dims_2d (include/tiling.h:43-45, src/block_sizing.cpp:639-779)."""
    x = BlkDims()
    check(load().cake_hip_init_block_dims_2d(M, N, K, p, C.byref(cake_cntx), sch, float(type_size), mcu, kcu, ncu,
                                             C.byref(x)), "init_block_dims_2d")
    return x


def init_block_dims_2d_small(M, N, K, p, cake_cntx: CpuCntx, sch=NA, argv=None, type_size=4) -> BlkDims:
    """init_block_dims_2d_small (include/tiling.h:47-49, src/block_sizing.cpp:785-841)."""
    x = BlkDims()
    check(load().cake_hip_init_block_dims_2d_small(M, N, K, p, C.byref(cake_cntx), sch, float(type_size), C.byref(x)),
          "init_block_dims_2d_small")
    return x


def init_block_dims_conv(Wf, Hf, Win, Hin, Wout, Hout, Cin, Cout, s, p, cake_cntx: CpuCntx, sch=KMN,
                         argv=None, density=0.0, type_size=4) -> BlkDims:
    """init_block_dims_conv (examples/cake_conv.cpp:333-425): blocks of the direct convolution, K-first."""
    x = BlkDims()
    check(load().cake_hip_init_block_dims_conv(Wf, Hf, Win, Hin, Wout, Hout, Cin, Cout, s, p, C.byref(cake_cntx),
                                               C.byref(x)), "init_block_dims_conv")
    return x


def plan(M, N, K, sch=NA, tile=None) -> Plan:
    """The GPU planner's decision for one product (tile, wave layout, reuse order, split-K)."""
    out = Plan()
    ov = (C.c_int * 4)(*tile) if tile is not None else None
    check(load().cake_hip_plan(M, N, K, sch, ov, C.byref(out)), "plan")
    return out


def _tile_override(M, N, K, sch, mcu, kcu, ncu):
    """mcu,kcu,ncu ask for a block of m x k x n; honoured when a macro-tile of that shape exists."""
    if not (mcu and kcu and ncu):
        return None
    ov = (C.c_int * 4)(mcu, ncu, kcu, 0)
    if load().cake_hip_plan(M, N, K, sch, ov, C.byref(Plan())) != _lib.OK:
        return None
    return ov


# ----------------------------------------------------------------------------
# cake_sgemm (include/cake.h:12-14)
# ----------------------------------------------------------------------------
def cake_sgemm(A, B, Cm, M, N, K, p, cake_cntx: CpuCntx | None = None, argv=None,
               packedA=False, packedB=False, alpha=1.0, beta=0.0, sch=NA,
               mcu=0, kcu=0, ncu=0) -> float:
    """C = A.B in place, returns seconds (device time of the kernels).

    Semantics follow src/cake_sgemm.cpp:9-175: alpha is ignored; K-first assigns
    C; for M-/N-first beta != 0 means "start from the existing C".  With
    packedA/packedB the operand is a buffer written by pack_A/pack_B for the same
    (M,N,K,p,cake_cntx,sch)."""
    lib = load()
    _need(Cm, M * N, "C")
    secs = C.c_double(0.0)
    stream = _stream(A, B, Cm)
    if packedA or packedB:
        cx = cake_cntx if cake_cntx is not None else _default_cntx()
        x = init_block_dims(M, N, K, p, cx, sch, argv, 4, mcu, kcu, ncu)
        accumulate = int(x.sch != KMN and beta != 0)
        check(lib.cake_hip_sgemm_packed(_ptr(A, "A"), _ptr(B, "B"), _ptr(Cm, "C"), M, N, K, p,
                                        C.byref(x), C.byref(cx), int(packedA), int(packedB),
                                        accumulate, stream, C.byref(secs)), "cake_sgemm")
        return secs.value
    _need(A, M * K, "A")
    _need(B, K * N, "B")
    # beta != 0 means "start from C" only under the schedule the reference resolves from the
    # caller's cntx and p (src/cake_sgemm.cpp:34-35,114); the GPU's tile order stays the planner's.
    resolved = sch
    if M > 0 and N > 0 and K > 0:
        cx = cake_cntx if cake_cntx is not None else _default_cntx()
        resolved = init_block_dims(M, N, K, p, cx, sch, argv, 4, mcu, kcu, ncu).sch
    elif sch == NA:
        resolved = KMN
    accumulate = int(resolved != KMN and beta != 0)
    ov = _tile_override(M, N, K, sch, mcu, kcu, ncu)
    check(lib.cake_hip_sgemm(_ptr(A, "A"), _ptr(B, "B"), _ptr(Cm, "C"), M, N, K, sch, accumulate, ov,
                             stream, C.byref(secs)), "cake_sgemm")
    return secs.value


# ----------------------------------------------------------------------------
# packing (include/packing.h:6-13,70-72)
# ----------------------------------------------------------------------------
def cake_sgemm_packed_A_size(M, K, p, x, cake_cntx, sch) -> int:
    return load().cake_hip_packed_a_size(M, K, p, C.byref(x), C.byref(cake_cntx), sch)


def cake_sgemm_packed_B_size(K, N, p, x, cake_cntx) -> int:
    return load().cake_hip_packed_b_size(K, N, p, C.byref(x), C.byref(cake_cntx))


def cake_sgemm_packed_C_size(M, N, p, x, cake_cntx, sch) -> int:
    return load().cake_hip_packed_c_size(M, N, p, C.byref(x), C.byref(cake_cntx), sch)


def pack_A(A, A_p, M, K, p, x, cake_cntx, sch) -> float:
    _need(A, M * K, "A")
    _need(A_p, cake_sgemm_packed_A_size(M, K, p, x, cake_cntx, sch) // 4, "A_p")
    secs = C.c_double(0.0)
    check(load().cake_hip_pack_a(_ptr(A, "A"), _ptr(A_p, "A_p"), M, K, p, C.byref(x), C.byref(cake_cntx),
                                 sch, _stream(A, A_p), C.byref(secs)), "pack_A")
    return secs.value


def pack_B(B, B_p, K, N, p, x, cake_cntx, sch) -> float:
    _need(B, K * N, "B")
    _need(B_p, cake_sgemm_packed_B_size(K, N, p, x, cake_cntx) // 4, "B_p")
    secs = C.c_double(0.0)
    check(load().cake_hip_pack_b(_ptr(B, "B"), _ptr(B_p, "B_p"), K, N, p, C.byref(x), C.byref(cake_cntx),
                                 sch, _stream(B, B_p), C.byref(secs)), "pack_B")
    return secs.value


def pack_C(Cm, C_p, M, N, p, x, cake_cntx, sch) -> float:
    _need(Cm, M * N, "C")
    _need(C_p, cake_sgemm_packed_C_size(M, N, p, x, cake_cntx, sch) // 4, "C_p")
    secs = C.c_double(0.0)
    check(load().cake_hip_pack_c(_ptr(Cm, "C"), _ptr(C_p, "C_p"), M, N, p, C.byref(x), C.byref(cake_cntx),
                                 sch, _stream(Cm, C_p), C.byref(secs)), "pack_C")
    return secs.value


def unpack_C(Cm, C_p, M, N, p, x, cake_cntx, sch) -> float:
    _need(Cm, M * N, "C")
    _need(C_p, cake_sgemm_packed_C_size(M, N, p, x, cake_cntx, sch) // 4, "C_p")
    secs = C.c_double(0.0)
    check(load().cake_hip_unpack_c(_ptr(Cm, "C"), _ptr(C_p, "C_p"), M, N, p, C.byref(x), C.byref(cake_cntx),
                                   sch, _stream(Cm, C_p), C.byref(secs)), "unpack_C")
    return secs.value


def packed_offset(which, row, col, M, N, K, p, x, cake_cntx, sch) -> int:
    """Host evaluation of the packed index map (which: 0 A, 1 B, 2 C); -1 when out of range."""
    return load().cake_hip_packed_offset(which, row, col, M, N, K, p, C.byref(x), C.byref(cake_cntx), sch)


# ----------------------------------------------------------------------------
# cake_sgemv (examples/cake_gemv.cpp:7-9)
# ----------------------------------------------------------------------------
def cake_sgemv(A, B, Cv, M, K, p, cake_cntx=None, argv=None, packedA=False, alpha=1.0, beta=0.0,
               sch=NA, *, row_major=False, accumulate=True) -> float:
    """y += A.x with A column-major (A[k*M + m]), as examples/cake_gemv.cpp:716-767 does.
    row_major=True reads A[m*K + k]; accumulate=False overwrites y.  Returns seconds."""
    _need(A, M * K, "A")
    _need(B, K, "x")
    _need(Cv, M, "y")
    secs = C.c_double(0.0)
    check(load().cake_hip_sgemv(_ptr(A, "A"), _ptr(B, "x"), _ptr(Cv, "y"), M, K, int(not row_major),
                                int(accumulate), _stream(A, B, Cv), C.byref(secs)), "cake_sgemv")
    return secs.value


# ----------------------------------------------------------------------------
# convolution through im2col (examples/cake_conv.cpp:24-25,1007-1066)
# ----------------------------------------------------------------------------
def im2col(inp, cols, batch, Cin, Hin, Win, Hf, Wf, stride=1, pad=0) -> float:
    Hout = (Hin + 2 * pad - Hf) // stride + 1
    Wout = (Win + 2 * pad - Wf) // stride + 1
    _need(inp, batch * Cin * Hin * Win, "input")
    _need(cols, Cin * Hf * Wf * batch * Hout * Wout, "cols")
    secs = C.c_double(0.0)
    check(load().cake_hip_im2col(_ptr(inp, "input"), _ptr(cols, "cols"), batch, Cin, Hin, Win, Hf, Wf,
                                 stride, pad, _stream(inp, cols), C.byref(secs)), "im2col")
    return secs.value


def im_2_col(In, Wf, Hf, Win, Hin, Wout, Hout, Cin, Cout=0, s=1):
    """im_2_col (examples/cake_conv.cpp:1178-1213): one CHW image, no padding; the
    stride argument is accepted and unused, as in the reference.  Returns the new
    [Cin*Hf*Wf, Hout*Wout] matrix."""
    if Hout != Hin - Hf + 1 or Wout != Win - Wf + 1:
        raise ValueError("im_2_col needs Hout = Hin - Hf + 1 and Wout = Win - Wf + 1")
    cols = _empty_like_kind(In, (Cin * Hf * Wf, Hout * Wout))
    im2col(In, cols, 1, Cin, Hin, Win, Hf, Wf, 1, 0)
    return cols


def conv2d(inp, weights, out, batch, Cin, Hin, Win, Cout, Hf, Wf, stride=1, pad=0,
           out_nchw=False, workspace=None, explicit_im2col=False) -> float:
    """weights[Cout x Cin*Hf*Wf] . im2col(inp): the im2col path of
    examples/cake_conv.cpp:1007-1066.  out is [Cout][batch*Hout*Wout] or NCHW.
    By default the column matrix is gathered inside the GEMM when the geometry
    allows; explicit_im2col=True always materialises it first, as the reference does."""
    Hout = (Hin + 2 * pad - Hf) // stride + 1
    Wout = (Win + 2 * pad - Wf) // stride + 1
    _need(inp, batch * Cin * Hin * Win, "input")
    _need(weights, Cout * Cin * Hf * Wf, "weights")
    _need(out, Cout * batch * Hout * Wout, "out")
    ws = 0
    if workspace is not None:
        need = load().cake_hip_conv2d_workspace(batch, Cin, Hin, Win, Cout, Hf, Wf, stride, pad)
        _need(workspace, (need + 3) // 4, "workspace")
        ws = _ptr(workspace, "workspace")
    secs = C.c_double(0.0)
    fn = load().cake_hip_conv2d_im2col if explicit_im2col else load().cake_hip_conv2d
    check(fn(_ptr(inp, "input"), _ptr(weights, "weights"), _ptr(out, "out"),
                                 batch, Cin, Hin, Win, Cout, Hf, Wf, stride, pad, int(out_nchw), ws,
                                 _stream(inp, weights, out), C.byref(secs)), "conv2d")
    return secs.value


def pack_filters(A, A_p, M, K, p, x, cake_cntx, taps=9) -> float:
    """pack_filters (examples/cake_conv.cpp:536-610): filters A[M = Cout][K = Cin * taps] into the K-first
    blocks of init_block_dims_conv; A_p holds x.M_padded * K floats.  The reference is written for
    3 x 3 filters (taps = 9)."""
    _need(A, M * K, "filters")
    _need(A_p, x.M_padded * K, "packed filters")
    secs = C.c_double(0.0)
    check(load().cake_hip_pack_filters(_ptr(A, "filters"), _ptr(A_p, "packed filters"), M, K // taps, taps, p,
                                       C.byref(x), C.byref(cake_cntx), _stream(A, A_p), C.byref(secs)), "pack_filters")
    return secs.value


def cake_sconv(A, B, Cm, Wf, Hf, Win, Hin, Wout, Hout, Cin, Cout, s, p, cake_cntx=None, argv=None,
               packedA=False, sch=NA) -> float:
    """cake_sconv (examples/cake_conv.cpp:5-8,765-848): C[Cout][Hout][Wout] += A[Cout][Cin][Hf][Wf] * B[Cin][Hin][Win],
    one CHW image, no padding; sch is accepted and unused (the reference always runs it K-first).
    With packedA the filters are in the layout of pack_filters for the blocks that
    init_block_dims_conv derives from the same geometry, p and cake_cntx (:791-799).  Returns seconds."""
    _need(B, Cin * Hin * Win, "input")
    _need(Cm, Cout * Hout * Wout, "output")
    secs = C.c_double(0.0)
    if packedA:
        cx = cake_cntx if cake_cntx is not None else _default_cntx()
        x = init_block_dims_conv(Wf, Hf, Win, Hin, Wout, Hout, Cin, Cout, s, p, cx)
        _need(A, x.M_padded * Cin * Hf * Wf, "packed filters")
        check(load().cake_hip_sconv_packed(_ptr(A, "filters"), _ptr(B, "input"), _ptr(Cm, "output"), Wf, Hf, Win, Hin,
                                           Wout, Hout, Cin, Cout, s, p, C.byref(x), C.byref(cx), _stream(A, B, Cm),
                                           C.byref(secs)), "cake_sconv")
        return secs.value
    _need(A, Cout * Cin * Hf * Wf, "filters")
    check(load().cake_hip_sconv(_ptr(A, "filters"), _ptr(B, "input"), _ptr(Cm, "output"), Wf, Hf, Win, Hin, Wout, Hout,
                                Cin, Cout, s, _stream(A, B, Cm), C.byref(secs)), "cake_sconv")
    return secs.value


def last_conv_route() -> int:
    """Which route this thread's last convolution call took (_lib.CONV_*)."""
    return load().cake_hip_last_conv_route()


# ----------------------------------------------------------------------------
# device contexts
# ----------------------------------------------------------------------------
class Context:
    """A device context of its own (cake_hip_ctx_create): workspaces, events and a stream that calls
    made while it is current do not share with the default context or with other contexts.

        with cake.Context() as ctx:          # current on this thread inside the block
            cake.cake_sgemm(...)             # torch tensors on the GPU: on torch's current stream, host operands
                                             # on ctx.stream
    """

    def __init__(self):
        h = C.c_void_p()
        check(load().cake_hip_ctx_create(C.byref(h)), "cake_hip_ctx_create")
        self.handle = h.value
        self._before = []

    @property
    def stream(self) -> int:
        return load().cake_hip_ctx_stream(self.handle) or 0

    def make_current(self) -> None:
        check(load().cake_hip_ctx_set_current(self.handle), "cake_hip_ctx_set_current")

    def __enter__(self):
        self._before.append(load().cake_hip_ctx_get_current())
        self.make_current()
        return self

    def __exit__(self, *exc):
        check(load().cake_hip_ctx_set_current(self._before.pop()), "cake_hip_ctx_set_current")
        return False

    def destroy(self) -> None:
        if self.handle:
            check(load().cake_hip_ctx_destroy(self.handle), "cake_hip_ctx_destroy")
            self.handle = None


def transpose_mat(A_old, At, K, N, Kt=0, Nt=0) -> float:
    """At[n][k] = A_old[k][n] for a K x N matrix (src/transpose.cpp:5-29; the
    blocking arguments Kt, Nt are accepted and unused).  Returns seconds."""
    _need(A_old, K * N, "A_old")
    _need(At, K * N, "At")
    secs = C.c_double(0.0)
    check(load().cake_hip_transpose(_ptr(A_old, "A_old"), _ptr(At, "At"), K, N, _stream(A_old, At),
                                    C.byref(secs)), "transpose_mat")
    return secs.value


def _opt_ptr(a, what):
    return None if a is None else _ptr(a, what)


def linear_forward(x, w, bias, y, M, N, K, timed=True) -> float:
    """y[M][N] = x[M][K] . w[N][K]^T + bias[N] (bias may be None): linear_forward of
    src/linear.cpp:12-50.  Returns seconds; timed=False skips the event timing, which makes
    the call asynchronous on device operands (it then returns 0)."""
    _need(x, M * K, "x")
    _need(w, N * K, "w")
    _need(y, M * N, "y")
    if bias is not None:
        _need(bias, N, "bias")
    secs = C.c_double(0.0)
    check(load().cake_hip_linear_forward(_ptr(x, "x"), _ptr(w, "w"), _opt_ptr(bias, "bias"), _ptr(y, "y"),
                                         M, N, K, _stream(x, w, y), C.byref(secs) if timed else None), "linear_forward")
    return secs.value


def sgemm_nt(A, Bt, Cm, M, N, K, accumulate=False, tile=None, timed=True) -> float:
    """C[M][N] = (C if accumulate else 0) + A[M][K] . Bt[N][K]^T with Bt read as it lies (the
    product of linear_forward, src/linear.cpp:38, without its transposed copy and bias).
    tile = (tile_m, tile_n, tile_k, split_k) forces the macro-tile kernel.  Returns seconds."""
    _need(A, M * K, "A")
    _need(Bt, N * K, "Bt")
    _need(Cm, M * N, "C")
    secs = C.c_double(0.0)
    ov = (C.c_int * 4)(*tile) if tile is not None else None
    check(load().cake_hip_sgemm_nt(_ptr(A, "A"), _ptr(Bt, "Bt"), _ptr(Cm, "C"), M, N, K, int(accumulate), ov,
                                   _stream(A, Bt, Cm), C.byref(secs) if timed else None), "sgemm_nt")
    return secs.value


def linear_forward_wt(x, wt, bias, y, M, N, K, timed=True) -> float:
    """The same with the weights already transposed: wt is [K][N] (transpose_mat of w), for callers
    that keep the transposed copy while the weights stay the same."""
    _need(x, M * K, "x")
    _need(wt, N * K, "wt")
    _need(y, M * N, "y")
    if bias is not None:
        _need(bias, N, "bias")
    secs = C.c_double(0.0)
    check(load().cake_hip_linear_forward_wt(_ptr(x, "x"), _ptr(wt, "wt"), _opt_ptr(bias, "bias"), _ptr(y, "y"),
                                            M, N, K, _stream(x, wt, y), C.byref(secs) if timed else None), "linear_forward_wt")
    return secs.value


def linear_backward(grad_y, x, w, grad_x, grad_w, grad_bias, M, N, K, timed=True) -> float:
    """grad_x = grad_y . w, grad_w = grad_y^T . x, grad_bias = column sums of grad_y
    (src/linear.cpp:53-102).  Outputs passed as None are skipped.  Returns seconds (0 with timed=False)."""
    _need(grad_y, M * N, "grad_y")
    for a, n, what in ((x, M * K, "x"), (w, N * K, "w"), (grad_x, M * K, "grad_x"),
                       (grad_w, N * K, "grad_w"), (grad_bias, N, "grad_bias")):
        if a is not None:
            _need(a, n, what)
    secs = C.c_double(0.0)
    check(load().cake_hip_linear_backward(_ptr(grad_y, "grad_y"), _opt_ptr(x, "x"), _opt_ptr(w, "w"),
                                          _opt_ptr(grad_x, "grad_x"), _opt_ptr(grad_w, "grad_w"),
                                          _opt_ptr(grad_bias, "grad_bias"), M, N, K,
                                          _stream(grad_y, x, w), C.byref(secs) if timed else None), "linear_backward")
    return secs.value


# ----------------------------------------------------------------------------
# the linear layer with 4-bit weights, orthogonalised updates
# ----------------------------------------------------------------------------
_TYPE_CODES = {"float32": _lib.F32, "float16": _lib.F16, "bfloat16": _lib.BF16}


def element_type(dtype) -> int:
    """CAKE_HIP_F32 / F16 / BF16 of a torch or numpy dtype or its name."""
    code = _TYPE_CODES.get(dtype)
    if code is None:
        name = np.dtype(dtype).name if isinstance(dtype, (type, np.dtype)) else str(dtype).replace("torch.", "")
        if name not in _TYPE_CODES:
            raise TypeError(f"element type {dtype}: float32, float16 or bfloat16 needed")
        code = _TYPE_CODES[dtype] = _TYPE_CODES[name]
    return code


def _any_ptr(a, what: str, of: int | None = None) -> int:
    """Address of a contiguous array of any element type (uint8, or `of` = an element type's code)."""
    if _is_torch(a):
        ok = a.is_contiguous()
        where = a.data_ptr()
    elif isinstance(a, np.ndarray):
        ok = a.flags["C_CONTIGUOUS"]
        where = a.ctypes.data
    else:
        raise TypeError(f"{what} must be a numpy array or torch tensor")
    if not ok:
        raise TypeError(f"{what} must be contiguous")
    if of is None:
        if str(a.dtype).replace("torch.", "") != "uint8":
            raise TypeError(f"{what} must be uint8, got {a.dtype}")
    elif element_type(a.dtype) != of:
        raise TypeError(f"{what} is {a.dtype}, another element type than its companions")
    return where


class Q4Weight:
    """A weight matrix v[N][K] in 4 bits, v = (code - zero) * scale per run of `group` columns: the packed
    bytes (numpy or torch uint8, in the library's own order) and what they hold.  It is made by q4_pack
    or q4_quantize; q4_of wraps bytes that were stored.  What it holds does not change: other bytes are
    another Q4Weight."""
    __slots__ = ("data", "N", "K", "group", "scale_type", "with_zeros", "bytes")

    def __init__(self, data, N, K, group, scale_type, with_zeros):
        _any_ptr(data, "packed weights")
        size = _q4_bytes(N, K, group, scale_type, with_zeros)
        _need(data, size, "packed weights")
        for name, value in zip(self.__slots__, (data, N, K, group, scale_type, bool(with_zeros), size)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"packed weights are made for one {name}; q4_of wraps other bytes")

    def __repr__(self):   # of what is in it and not of where it lies: a trace compares it with the next one's
        return f"Q4Weight(N={self.N}, K={self.K}, group={self.group}, scale_type={self.scale_type}, with_zeros={self.with_zeros})"

    def __reduce__(self):
        return Q4Weight, (self.data, self.N, self.K, self.group, self.scale_type, self.with_zeros)

    def __setstate__(self, state):   # what was stored attribute by attribute
        self.__init__(**state[1])


def _q4_bytes(N, K, group, scale_type, zeros) -> int:
    n = load().cake_hip_q4_size(N, K, group, scale_type, bool(zeros))
    if n == 0 and N != 0 and K != 0:
        raise CakeHipError(_lib.ERR_ARG, "q4_size", load().cake_hip_last_error().decode())
    return n


def q4_size(N, K, group=128, scale_dtype="float32", zeros=False) -> int:
    """Bytes of the packed form."""
    return _q4_bytes(N, K, group, element_type(scale_dtype), zeros)


def _bytes_like(ref, n):
    if _is_torch(ref):
        import torch
        return torch.empty(n, dtype=torch.uint8, device=ref.device)
    # a little more than needed, so that the packed bytes can start on 16
    raw = np.empty(n + 16, np.uint8)
    skip = -raw.ctypes.data % 16
    return raw[skip:skip + n]


def q4_of(data, N, K, group, scale_dtype, zeros) -> Q4Weight:
    """Packed bytes that an earlier q4_pack or q4_quantize made, with what they were made for."""
    return Q4Weight(data, N, K, group, element_type(scale_dtype), zeros)


def q4_pack(codes, scales, zeros, N, K, group=128, timed=False) -> Q4Weight:
    """codes[N][(K + 1) // 2] (uint8, even columns in the low half of a byte), scales and zeros
    [N][ceil(K / group)] of one element type (zeros None: 8 everywhere) as packed weights."""
    st = element_type(scales.dtype)
    q = Q4Weight(_bytes_like(codes, q4_size(N, K, group, scales.dtype, zeros is not None)), N, K, group, st, zeros is not None)
    runs = N * -(-K // group)
    _need(codes, N * ((K + 1) // 2), "codes")
    _need(scales, runs, "scales")
    if zeros is not None:
        _need(zeros, runs, "zeros")
    secs = C.c_double(0.0)
    check(load().cake_hip_q4_pack(_any_ptr(codes, "codes"), _any_ptr(scales, "scales", st),
                                  None if zeros is None else _any_ptr(zeros, "zeros", st), _any_ptr(q.data, "q"), N, K, group, st,
                                  _stream(codes, scales), C.byref(secs) if timed else None), "q4_pack")
    return q


def q4_quantize(w, N, K, group=128, zeros=False, scale_dtype="float32", timed=False) -> Q4Weight:
    """w[N][K] in 4 bits: scales max|w| / 7 around code 8, or with `zeros` the range's / 15 and a zero point
    (the full definition is in include/cake_hip.h)."""
    _need(w, N * K, "w")
    st, wt = element_type(scale_dtype), element_type(w.dtype)
    q = Q4Weight(_bytes_like(w, q4_size(N, K, group, scale_dtype, zeros)), N, K, group, st, zeros)
    secs = C.c_double(0.0)
    check(load().cake_hip_q4_quantize(_any_ptr(w, "w", wt), wt, _any_ptr(q.data, "q"), N, K, group, st, int(q.with_zeros),
                                      _stream(w), C.byref(secs) if timed else None), "q4_quantize")
    return q


def q4_dequantize(q: Q4Weight, w, timed=False) -> float:
    """The values that packed weights stand for, into w[N][K] of any element type.  Returns seconds (0 with timed=False)."""
    _need(w, q.N * q.K, "w")
    _need(q.data, q.bytes, "packed weights")
    wt = element_type(w.dtype)
    secs = C.c_double(0.0)
    check(load().cake_hip_q4_dequantize(_any_ptr(q.data, "q"), _any_ptr(w, "w", wt), wt, q.N, q.K, q.group, q.scale_type,
                                        int(q.with_zeros), _stream(w, q.data), C.byref(secs) if timed else None), "q4_dequantize")
    return secs.value


def linear_q4_workspace(M, N, K, dtype="float32") -> int:
    """Bytes of device memory linear_q4_forward wants for M rows of x (0 for a few)."""
    return load().cake_hip_linear_q4_workspace(M, N, K, element_type(dtype))


def linear_q4_forward(x, q: Q4Weight, bias, y, M, workspace=None, timed=True) -> float:
    """y[M][N] = x[M][K] . v[N][K]^T + bias[N] (bias may be None); x, bias and y of one element type.
    workspace: a uint8 device tensor of linear_q4_workspace bytes, or None for the library's own
    (calls on several streams at once need one each).
    Returns seconds (0 with timed=False, which makes the call asynchronous on device operands)."""
    t = element_type(x.dtype)
    N, K = q.N, q.K
    _need(x, M * K, "x")
    _need(y, M * N, "y")
    _need(q.data, q.bytes, "packed weights")
    if bias is not None:
        _need(bias, N, "bias")
    if workspace is not None:
        _need(workspace, load().cake_hip_linear_q4_workspace(M, N, K, t), "workspace")
    secs = C.c_double(0.0)
    check(load().cake_hip_linear_q4_forward(_any_ptr(x, "x", t), _any_ptr(q.data, "q"),
                                            None if bias is None else _any_ptr(bias, "bias", t), _any_ptr(y, "y", t), t, M, N, K,
                                            q.group, q.scale_type, int(q.with_zeros),
                                            None if workspace is None else _any_ptr(workspace, "workspace"),
                                            _stream(x, q.data, y), C.byref(secs) if timed else None), "linear_q4_forward")
    return secs.value


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def orthogonalize_workspace(batch, rows, cols) -> int:
    """Bytes of device memory orthogonalize wants."""
    return load().cake_hip_orthogonalize_workspace(batch, rows, cols)


def orthogonalize_check(steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7) -> None:
    """Raises for what orthogonalize refuses whatever the matrices."""
    c0, c1, c2 = coefficients
    check(load().cake_hip_orthogonalize(None, None, _lib.F32, 0, 0, 0, steps, c0, c1, c2, eps, None, None, None), "orthogonalize")


def orthogonalize(g, out, batch, rows, cols, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, workspace=None, timed=True) -> float:
    """Newton-Schulz iterations on g[batch][rows][cols] into out (of g's element type; may be g):
    x = g / (|g| + eps), then `steps` times a = x x^T, x = c0 x + (c1 a + c2 a a) x.
    workspace: a uint8 device tensor of orthogonalize_workspace bytes, or None for the library's own
    (calls on several streams at once need one each).  Returns seconds (0 with timed=False)."""
    t = element_type(g.dtype)
    _need(g, batch * rows * cols, "g")
    _need(out, batch * rows * cols, "out")
    if workspace is not None:
        _need(workspace, load().cake_hip_orthogonalize_workspace(batch, rows, cols), "workspace")
    c0, c1, c2 = coefficients
    secs = C.c_double(0.0)
    check(load().cake_hip_orthogonalize(_any_ptr(g, "g", t), _any_ptr(out, "out", t), t, batch, rows, cols, steps, c0, c1, c2, eps,
                                        None if workspace is None else _any_ptr(workspace, "workspace"),
                                        _stream(g, out), C.byref(secs) if timed else None), "orthogonalize")
    return secs.value


# ----------------------------------------------------------------------------
# autotuner (successor of mcu,kcu,ncu + src/autotune_sa.cpp)
# ----------------------------------------------------------------------------
def autotune(M, N, K, budget_seconds=2.0):
    """Measure the macro-tile / split-K candidates for an M x N x K product and keep the
    fastest for later calls.  Returns (plan, best_seconds, default_seconds)."""
    out = Plan()
    best, base = C.c_double(0.0), C.c_double(0.0)
    check(load().cake_hip_autotune(M, N, K, float(budget_seconds), C.byref(out), C.byref(best), C.byref(base)),
          "autotune")
    return out, best.value, base.value


def tune_save(path) -> None:
    check(load().cake_hip_tune_save(os.fsencode(path)), "tune_save")


def tune_load(path) -> int:
    n = C.c_int(0)
    check(load().cake_hip_tune_load(os.fsencode(path), C.byref(n)), "tune_load")
    return n.value


def tune_clear() -> None:
    check(load().cake_hip_tune_clear(), "tune_clear")


def tune_count() -> int:
    return load().cake_hip_tune_count()


# ----------------------------------------------------------------------------
# utilities
# ----------------------------------------------------------------------------
def fill_uniform(dst, seed: int) -> None:
    """dst[i] = uniform[-1,1) value i of stream `seed` (replaces rand_init, src/util.cpp:259-267)."""
    check(load().cake_hip_fill_uniform(_ptr(dst, "dst"), _numel(dst), seed, _stream(dst)), "fill_uniform")


def device_info() -> DeviceInfo:
    info = DeviceInfo()
    check(load().cake_hip_device_info(C.byref(info)), "device_info")
    return info


def last_kernel_seconds() -> dict:
    arr = (C.c_double * 5)()
    check(load().cake_hip_last_kernel_seconds(C.byref(arr)), "last_kernel_seconds")
    return dict(zip(("gemm", "splitk_reduce", "gemv", "im2col", "pack"), arr))
