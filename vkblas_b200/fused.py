"""Fused language-model products on torch CUDA tensors: the gated feed-forward
block, the cross entropy of a linear head, and decode products with 4-bit
weights (include/vkblas_b200.h).

Matrices are 2-D float16 or bfloat16 tensors of one type on one device whose
rows are contiguous (any row stride of at least the row length); weights hold
one row of inputs per output, as torch.nn.Linear stores them.  Calls run on
``stream`` (a torch.cuda.Stream, a raw handle or None for torch's current
stream); results and scratch are allocated from torch's pool of that stream, so
calls can be captured into a CUDA graph.  On a stream other than the one that its inputs were
made on, the caller orders the two and keeps the inputs until the call's work is done
(Tensor.record_stream).  A misfit raises ValueError before
anything is launched, a non-OK status VkblasError.  Autograd is not involved:
the backward passes are calls of their own.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import vkblas_b200 as _vk

_u32, _i64, _vp, _i32 = C.c_uint32, C.c_int64, C.c_void_p, C.c_int

ACT_SILU, ACT_GELU, ACT_GELU_TANH = 0, 1, 2
ACTS = {"silu": ACT_SILU, "gelu": ACT_GELU, "gelu_tanh": ACT_GELU_TANH}


def _mats(*names):
    return [f for n, ld in names for f in ((n, _vp), (ld, _u32))]


class Gated(C.Structure):
    _fields_ = [("dtype", _i32), ("act", _i32), ("M", _u32), ("F", _u32), ("H", _u32)] + _mats(
        ("x", "ldx"), ("w_gate", "ldwg"), ("w_up", "ldwu"), ("h", "ldh"), ("g", "ldg"), ("u", "ldu"))


class GatedBackward(C.Structure):
    _fields_ = [("dtype", _i32), ("act", _i32), ("M", _u32), ("F", _u32), ("H", _u32)] + _mats(
        ("dh", "lddh"), ("g", "ldg"), ("u", "ldu"), ("x", "ldx"), ("w_gate", "ldwg"),
        ("w_up", "ldwu"), ("dx", "lddx"), ("dw_gate", "lddwg"), ("dw_up", "lddwu"))


class LinearXent(C.Structure):
    _fields_ = [("dtype", _i32), ("T", _u32), ("V", _u32), ("H", _u32)] + _mats(
        ("x", "ldx"), ("w", "ldw")) + [("targets", _vp), ("ignore_index", _i64), ("loss", _vp),
                                       ("lse", _vp)]


class LinearXentBackward(C.Structure):
    _fields_ = [("dtype", _i32), ("T", _u32), ("V", _u32), ("H", _u32), ("dloss", _vp),
                ("lse", _vp)] + _mats(("x", "ldx"), ("w", "ldw")) + [
        ("targets", _vp), ("ignore_index", _i64)] + _mats(("dx", "lddx"), ("dw", "lddw"))


class Q4(C.Structure):
    _fields_ = [("dtype", _i32), ("N", _u32), ("K", _u32), ("group", _u32), ("has_zeros", _i32),
                ("packed", _vp)]


def declare(lib) -> None:
    """Argument types of this module's entry points."""
    sz = C.c_size_t
    for name, st in (("gated", Gated), ("gated_backward", GatedBackward), ("linear_xent", LinearXent),
                     ("linear_xent_backward", LinearXentBackward)):
        ws, fn = getattr(lib, f"vkblas_b200_{name}_workspace"), getattr(lib, f"vkblas_b200_{name}")
        ws.argtypes, ws.restype = [C.POINTER(st)], sz
        fn.argtypes, fn.restype = [C.POINTER(st), _vp, sz, _vp], _i32
    lib.vkblas_b200_q4_bytes.argtypes = [C.POINTER(Q4)]
    lib.vkblas_b200_q4_bytes.restype = sz
    lib.vkblas_b200_q4_pack.argtypes = [C.POINTER(Q4), _vp, _u32, _vp, _u32, _vp, _u32, _vp, _vp]
    lib.vkblas_b200_gemv_q4.argtypes = [C.POINTER(Q4), _u32, C.c_float, _vp, _u32, C.c_float, _vp,
                                        _u32, _vp]
    for fn in (lib.vkblas_b200_q4_pack, lib.vkblas_b200_gemv_q4):
        fn.restype = _i32


# ------------------------------------------------------------------------------ checks
# These run before every call, some of which take a few microseconds on the
# GPU: they look at each tensor once.
_DTYPES = {}


def _dtype(t) -> int:
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float16: _vk.DT_F16, torch.bfloat16: _vk.DT_BF16})
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"float16 or bfloat16 wanted, got {t.dtype}")
    return d


def _device(**ts):
    """The one CUDA device of the tensors given (None is left out)."""
    first = None
    for name, t in ts.items():
        if t is None:
            continue
        if not getattr(t, "is_cuda", False):
            raise ValueError(f"{name} must be a CUDA tensor")
        if first is None:
            first, index = t, t.get_device()
        elif t.get_device() != index:
            raise ValueError(f"devices differ: {first.device}, {t.device} ({name})")
    return first.device


def _mat(name, t, rows, cols, dtype):
    """(pointer, leading dimension) of a rows x cols matrix."""
    if t.dtype != dtype:
        raise ValueError(f"dtypes differ: {name} is {t.dtype}, not {dtype}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name} is {tuple(t.shape)}, not {(rows, cols)}")
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous")
    # One row is never stepped from: any leading dimension says the same.
    ld = t.stride(0) if rows > 1 else (cols + 7) // 8 * 8
    if not cols <= ld < 1 << 32:
        raise ValueError(f"{name}'s row stride {ld} is below {cols} or does not fit 32 bits")
    return t.data_ptr(), ld


def _sizes(*ns):
    for n in ns:
        if not 0 < n < 1 << 32:
            raise ValueError(f"sizes must be positive and fit 32 bits, got {ns}")


def _vec(name, t, n, dtype):
    if t.dtype != dtype or t.shape != (n,):
        raise ValueError(f"{name} must be {dtype} of shape ({n},), is {t.dtype} {tuple(t.shape)}")
    return t


def _enter(device, stream):
    """Makes `device` current, and `stream` (or torch's current one there) torch's
    current stream, so that allocations belong to it.  Returns the stream's handle and
    what undoes it: a call, or None where all of that was so already."""
    import torch
    if stream is None and torch._C._cuda_getDevice() == device.index:
        # torch.cuda.current_stream() without building the Stream object
        return torch._C._cuda_getCurrentRawStream(device.index), None
    if stream is None:
        stream = torch.cuda.current_stream(device)
    elif not hasattr(stream, "cuda_stream"):
        with torch.cuda.device(device):
            stream = (torch.cuda.ExternalStream(stream, device) if stream
                      else torch.cuda.default_stream(device))
    if stream.device != device:
        raise ValueError(f"the stream is of {stream.device}, the tensors of {device}")
    stack = contextlib.ExitStack()
    stack.enter_context(torch.cuda.device(device))
    stack.enter_context(torch.cuda.stream(stream))
    return stream.cuda_stream, stack.close


def _new(rows, cols, like):
    """A new matrix and its (pointer, leading dimension)."""
    t = like.new_empty((rows, cols))
    return t, (t.data_ptr(), cols)


def _given(t, rows, cols, like, **ins):
    """(pointer, leading dimension) of the caller's output; it may share no element with `ins`,
    2-D tensors of its type, which the kernels read while they write it.  Column blocks of one
    buffer are apart."""
    p, ld = _mat("out", t, rows, cols, like.dtype)
    size = t.element_size()
    end = p + size * ((rows - 1) * ld + cols)
    for name, x in ins.items():
        r, c = x.shape
        q, lx = x.data_ptr(), x.stride(0)
        if q >= end or p >= q + size * ((r - 1) * lx + c):
            continue
        pitch = ld if r == 1 else lx if rows == 1 else ld if ld == lx else 0
        at = (q - p) // size % pitch if pitch else 0     # x's first column, counted from out's
        if not (pitch and cols <= at and at + c <= pitch):
            raise ValueError(f"out overlaps {name}, which is read while it is written")
    return p, ld


_FNS = {}


def _run(name, args, dev, handle):
    if name not in _FNS:
        _FNS[name] = (getattr(_vk.lib, f"vkblas_b200_{name}_workspace"), getattr(_vk.lib, f"vkblas_b200_{name}"))
    size, fn = _FNS[name]
    ref = C.byref(args)
    n = size(ref)
    if n:
        import torch
        ws = torch.empty(n, device=dev, dtype=torch.uint8)
        st = fn(ref, ws.data_ptr(), n, handle)
    else:
        st = fn(ref, None, 0, handle)
    if st != _vk.VKBLAS_OK:
        raise _vk.VkblasError(f"vkblas_b200_{name} returned status {st}")


def _act(act) -> int:
    if act not in ACTS:
        raise ValueError(f"act is one of {sorted(ACTS)}, not {act!r}")
    return ACTS[act]


def _shape2(name, t):
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, is {tuple(t.shape)}")
    return t.shape


# ------------------------------------------------------------------------------ gated block
def gated_tensors(x, w_gate, w_up, act="silu", out=None, save=False, stream=None):
    """h = act(x w_gate^T) * (x w_up^T) for x (M, H) and weights (F, H), in one
    kernel.  ``act``: "silu", "gelu" or "gelu_tanh".  Returns h (M, F) (``out``
    where given, which shares no element with the inputs), or (h, g, u) with ``save``: g and u are the two projections,
    which :func:`gated_backward_tensors` reads."""
    (M, H), (F, _) = _shape2("x", x), _shape2("w_gate", w_gate)
    _sizes(M, F, H)
    dev, code = _device(x=x, w_gate=w_gate, w_up=w_up, out=out), _act(act)
    dt = _dtype(x)
    a = (_mat("x", x, M, H, x.dtype), _mat("w_gate", w_gate, F, H, x.dtype),
         _mat("w_up", w_up, F, H, x.dtype))
    h, hm = out, _given(out, M, F, x, x=x, w_gate=w_gate, w_up=w_up) if out is not None else None
    s, undo = _enter(dev, stream)
    try:
        if h is None:
            h, hm = _new(M, F, x)
        g, u, gm, um = None, None, (None, 0), (None, 0)
        if save:
            g, gm = _new(M, F, x)
            u, um = _new(M, F, x)
        _run("gated", Gated(dt, code, M, F, H, *a[0], *a[1], *a[2], *hm, *gm, *um), dev, s)
    finally:
        if undo:
            undo()
    return (h, g, u) if save else h


def gated_backward_tensors(dh, g, u, x, w_gate, w_up, act="silu", need_dx=True, need_dw=True,
                           stream=None):
    """Gradients (dx, dw_gate, dw_up) of :func:`gated_tensors` from the gradient
    ``dh`` of h and the saved g and u; those not needed are None."""
    (M, F), (_, H) = _shape2("dh", dh), _shape2("x", x)
    _sizes(M, F, H)
    if not (need_dx or need_dw):
        raise ValueError("no gradient is asked for")
    dev, code = _device(dh=dh, g=g, u=u, x=x, w_gate=w_gate, w_up=w_up), _act(act)
    dt, t = _dtype(dh), dh.dtype
    ins = [*_mat("dh", dh, M, F, t), *_mat("g", g, M, F, t), *_mat("u", u, M, F, t),
           *_mat("x", x, M, H, t), *_mat("w_gate", w_gate, F, H, t), *_mat("w_up", w_up, F, H, t)]
    none = (None, (None, 0))
    s, undo = _enter(dev, stream)
    try:
        dx, dxm = _new(M, H, dh) if need_dx else none
        dwg, dwu, dwgm, dwum = None, None, (None, 0), (None, 0)
        if need_dw:
            # one buffer, both matrices on 16 bytes: the library then computes them in one grid
            pad = -(F * H) % 8
            buf = dh.new_empty(2 * F * H + pad)
            dwg, dwu = buf[:F * H].view(F, H), buf[F * H + pad:].view(F, H)
            dwgm, dwum = (dwg.data_ptr(), H), (dwu.data_ptr(), H)
        _run("gated_backward", GatedBackward(dt, code, M, F, H, *ins, *dxm, *dwgm, *dwum), dev, s)
    finally:
        if undo:
            undo()
    return dx, dwg, dwu


# ------------------------------------------------------------------------------ cross entropy
def linear_xent_tensors(x, w, targets, ignore_index=-100, stream=None):
    """(loss, lse), fp32 of shape (T,): softmax cross entropy of the logits
    x w^T for x (T, H) and w (V, H) against int64 ``targets``, and the rows'
    log-sum-exp, which the backward pass takes.  The logits are not kept.  Rows
    of ``ignore_index`` have loss 0, rows of another target outside [0, V) NaN."""
    import torch
    (T, H), (V, _) = _shape2("x", x), _shape2("w", w)
    _sizes(T, V, H)
    dev, dt = _device(x=x, w=w, targets=targets), _dtype(x)
    a = (*_mat("x", x, T, H, x.dtype), *_mat("w", w, V, H, x.dtype))
    _vec("targets", targets, T, torch.int64)
    s, undo = _enter(dev, stream)
    try:
        targets = targets.contiguous()
        loss, lse = (torch.empty(T, device=dev, dtype=torch.float32) for _ in range(2))
        _run("linear_xent", LinearXent(dt, T, V, H, *a, targets.data_ptr(), ignore_index,
                                       loss.data_ptr(), lse.data_ptr()), dev, s)
    finally:
        if undo:
            undo()
    return loss, lse


def linear_xent_backward_tensors(dloss, lse, x, w, targets, ignore_index=-100, need_dx=True,
                                 need_dw=True, stream=None):
    """Gradients (dx, dw) of :func:`linear_xent_tensors` from the gradients
    ``dloss`` of the losses and the forward pass's ``lse``; those not needed are
    None.  The logits are computed again, in pieces of the vocabulary."""
    import torch
    (T, H), (V, _) = _shape2("x", x), _shape2("w", w)
    _sizes(T, V, H)
    if not (need_dx or need_dw):
        raise ValueError("no gradient is asked for")
    dev, dt = _device(x=x, w=w, targets=targets, dloss=dloss, lse=lse), _dtype(x)
    a = (*_mat("x", x, T, H, x.dtype), *_mat("w", w, V, H, x.dtype))
    _vec("targets", targets, T, torch.int64)
    _vec("dloss", dloss, T, torch.float32)
    _vec("lse", lse, T, torch.float32)
    none = (None, (None, 0))
    s, undo = _enter(dev, stream)
    try:
        # A gradient of a sum comes as one value expanded over the rows.
        targets, dloss, lse = targets.contiguous(), dloss.contiguous(), lse.contiguous()
        dx, dxm = _new(T, H, x) if need_dx else none
        dw, dwm = _new(V, H, x) if need_dw else none
        _run("linear_xent_backward",
             LinearXentBackward(dt, T, V, H, dloss.data_ptr(), lse.data_ptr(), *a,
                                targets.data_ptr(), ignore_index, *dxm, *dwm), dev, s)
    finally:
        if undo:
            undo()
    return dx, dw


# ------------------------------------------------------------------------------ 4-bit weights
class Q4Weight:
    """A matrix of 4-bit weights laid out for :func:`gemv_q4_tensors`."""

    def __init__(self, dtype, N, K, group, has_zeros, packed):
        self.dtype, self.N, self.K, self.group = dtype, N, K, group
        self.has_zeros, self.packed = has_zeros, packed
        self._code = None

    def struct(self):
        if self._code is None:
            import torch
            self._code = _vk.DT_F16 if self.dtype == torch.float16 else _vk.DT_BF16
        return Q4(self._code, self.N, self.K, self.group, self.has_zeros,
                  self.packed.data_ptr() if self.packed is not None else None)


def q4_pack_tensors(q, scales, zeros, K, group, stream=None) -> Q4Weight:
    """Lays out 4-bit weights for the decode product, once.  Weight (n, k) is
    scales[n, k // group] * (q[n, k] - zeros[n, k // group]); ``q`` (N,
    ceil(K / 2)) uint8 holds two weights a byte, the even k in the low half;
    ``scales`` (N, ceil(K / group)) float16 or bfloat16, the type of the
    activations; ``zeros`` uint8 of the same shape, or None for 8.  Of a zero point
    only the low 4 bits are kept: formats that store it less 1 may give 16 after their
    offset, which would become 0.  ``group`` is a multiple of 32."""
    import torch
    N = _shape2("q", q)[0]
    _sizes(N, K, group)
    if group % 32:
        raise ValueError(f"group must be a multiple of 32, is {group}")
    dev = _device(q=q, scales=scales, zeros=zeros)
    _dtype(scales)
    ng = -(-K // group)
    qp, ldq = _mat("q", q, N, -(-K // 2), torch.uint8)
    sp, lds = _mat("scales", scales, N, ng, scales.dtype)
    zp, ldz = (None, 0) if zeros is None else _mat("zeros", zeros, N, ng, torch.uint8)
    w = Q4Weight(scales.dtype, N, K, group, zeros is not None, None)
    s, undo = _enter(dev, stream)
    try:
        st = w.struct()
        w.packed = torch.empty(_vk.lib.vkblas_b200_q4_bytes(C.byref(st)), device=dev, dtype=torch.uint8)
        rc = _vk.lib.vkblas_b200_q4_pack(C.byref(st), qp, ldq, sp, lds, zp, ldz, w.packed.data_ptr(), s)
    finally:
        if undo:
            undo()
    if rc != _vk.VKBLAS_OK:
        raise _vk.VkblasError(f"vkblas_b200_q4_pack returned status {rc}")
    return w


def gemv_q4_tensors(x, w: Q4Weight, out=None, alpha=1.0, beta=0.0, stream=None):
    """out = alpha x W^T + beta out for x (M, K), M <= 16, and packed 4-bit
    weights W (N, K).  Returns out (M, N), which shares no element with x; without
    ``out``, beta must be 0."""
    M, _ = _shape2("x", x)
    if not 0 < M <= 16:
        raise ValueError(f"M must be positive and at most 16 rows, got {M}")
    if out is None and beta != 0.0:
        raise ValueError("beta needs out")
    dev = _device(x=x, w=w.packed, out=out)
    xp, ldx = _mat("x", x, M, w.K, w.dtype)
    ym = _given(out, M, w.N, x, x=x) if out is not None else None
    s, undo = _enter(dev, stream)
    try:
        if ym is None:
            out, ym = _new(M, w.N, x)
        yp, ldy = ym
        rc = _vk._get().vkblas_b200_gemv_q4(C.byref(w.struct()), M, alpha, xp, ldx, beta, yp, ldy, s)
    finally:
        if undo:
            undo()
    if rc != _vk.VKBLAS_OK:
        raise _vk.VkblasError(f"vkblas_b200_gemv_q4 returned status {rc}")
    return out
