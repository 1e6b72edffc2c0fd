"""Dense operators of the guidance network's layers and of its training step: hand-written HIP kernels of libnirrt_hip.so
(csrc/nnops.hip, C ABI include/nirrt_nnops.h), launched on the current torch stream, differentiable where a gradient makes sense.

    linear_act            act(x W^T + b) + r in one kernel, with its backward pass
    linear_cross_entropy  a classification head with softmax cross entropy; the scores are never kept, forward or backward
    grad_norm             2-norm over many tensors
    clip_grad_norm_       the same, and the clipping by it (in place, or into other tensors)

float32, bfloat16 and float16; sums are held in 32 bits and rounded once.  In 16 bits the backward passes have roundings of their own: the
pre-activation is kept in the tensors' type, and the gradient in front of a product (dz, or probability minus target) is rounded to it, as
matrix instructions multiply 16-bit operands - dx and dW are 2.4e-3 off in bfloat16 (2-norm) where the rounding of the result alone is
1.7e-3, and a float16 gradient above 5.8e4 may overflow in dz.  Tensors must live on the GPU (a CPU tensor is an error,
there is no other implementation); rows may have any stride, other layouts are copied.  Results are the same bits for the same input
(no atomics).  Backward passes are differentiable once; there is no forward mode, and a call cannot be traced (torch.jit.trace, make_fx):
both are refused.

Everything can be captured into a graph; a backward pass through torch.autograd.grad, or with .backward() while no eager graph of the same
leaves is alive (torch's accumulators of a leaf remember the stream they were made on, and adding to them from a capture ends the
process).
"""
import contextlib
import ctypes as C
import operator

import numpy as np
import torch
from torch.autograd import forward_ad

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_DIM_MAX = (1 << 31) - 4096


_library = None


def _lib():
    global _library
    if _library is None:
        from . import _hip
        L = _hip.load()
        vp, i, l, f = C.c_void_p, C.c_int, C.c_int64, C.c_float
        L.nirrt_nn_linear_workspace.argtypes = [i, vp, l, vp, l, l, l, l]
        L.nirrt_nn_linear.argtypes = [i, i, vp, l, vp, l, vp, vp, l, vp, l, vp, l, l, l, vp, vp]
        L.nirrt_nn_linear_backward_workspace.argtypes = [i, i, vp, l, vp, l, vp, l, l, l, l]
        L.nirrt_nn_linear_backward.argtypes = [i, i, vp, l, vp, l, vp, vp, l, vp, vp, vp, l, l, l, vp, vp]
        L.nirrt_nn_cross_entropy_workspace.argtypes = [i, l, l, l]
        L.nirrt_nn_cross_entropy.argtypes = [i, vp, l, vp, l, vp, vp, vp, l, vp, vp, vp, l, l, l, vp, vp]
        L.nirrt_nn_cross_entropy_backward_workspace.argtypes = [i, l, l, l]
        L.nirrt_nn_cross_entropy_backward.argtypes = [i, vp, l, vp, l, vp, vp, vp, l, vp, vp, i, vp, vp, vp, vp, l, l, l, vp, vp]
        L.nirrt_nn_norm_workspace.argtypes = [vp, C.c_int32]
        L.nirrt_nn_norm.argtypes = [vp, C.c_int32, vp, vp, vp]
        L.nirrt_nn_scale_by_norm.argtypes = [vp, C.c_int32, vp, f, vp]
        for name in ("linear", "linear_backward", "cross_entropy", "cross_entropy_backward", "norm"):
            getattr(L, "nirrt_nn_%s_workspace" % name).restype = l
            getattr(L, "nirrt_nn_%s" % name).restype = i
        L.nirrt_nn_scale_by_norm.restype = i
        _library = L
    return _library


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # (the stream object costs 2 us per call)


def _stream(device):
    return _raw_stream(device.index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _check(rc, what):
    if rc != 0:
        raise RuntimeError("libnirrt_hip %s failed (%d)" % (what, rc))


_HERE = contextlib.nullcontext()


def _on(device):
    """the C functions launch on the calling thread's current device"""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


_is_tracing = torch._C._is_tracing
_dispatch_modes = torch._C._len_torch_dispatch_stack


def _not_recorded(name):
    """torch.jit.trace and make_fx see the allocation of a result and not the kernel that fills it: what they record returns whatever
    the memory holds"""
    recorded = _is_tracing()
    if not recorded and _dispatch_modes():
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        recorded = get_proxy_mode() is not None
    if recorded:
        raise RuntimeError("nirrt_star_amd.nnops.%s cannot be traced: its kernels are launched through the C library" % name)


def _need(name, first, **others):
    """one device (a GPU) and one element type for all of them"""
    if _is_tracing() or _dispatch_modes():
        _not_recorded(name)
    if not first.is_cuda:
        raise RuntimeError("nirrt_star_amd.nnops.%s got a CPU tensor: the package only has the HIP kernels (move it to 'cuda')" % name)
    if first.dtype not in _TYPES:
        raise ValueError("%s: float32, bfloat16 or float16, not %s" % (name, first.dtype))
    for key, t in others.items():
        if t is None:
            continue
        if t.device != first.device:
            raise ValueError("%s: %s is on %s, the input on %s" % (name, key, t.device, first.device))
        if t.dtype != first.dtype:
            raise ValueError("%s: %s is %s, the input %s" % (name, key, t.dtype, first.dtype))


def _rows(t):
    """(..., k) -> (rows, k) with unit column stride and rows that do not overlap (a copy if need be), and its row stride"""
    if t.dim() != 2:
        k = t.shape[-1]
        t = t.reshape(t.numel() // k if k else _prod(t.shape[:-1]), k)
    m, k = t.shape
    ld, one = t.stride()
    if one == 1 and ld >= k > 0:
        return t, ld
    if m <= 1 or k == 0:
        return (t if k <= 1 or one == 1 else t.contiguous()), max(k, 1)
    if k > 1 or ld < k:
        t = t.contiguous()
    return t, t.stride(0)


def _prod(shape):
    n = 1
    for s in shape:
        n *= int(s)
    return n


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, device):
    if nbytes < 0:
        raise RuntimeError("libnirrt_hip: bad sizes for a workspace")
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _sizes_ok(name, *dims):
    if max(dims) > _DIM_MAX:
        raise ValueError("%s: a dimension of %d is beyond %d" % (name, max(dims), _DIM_MAX))


# ---- linear layer ---------------------------------------------------------------------------------------------------------------------
def _linear_forward(x, w, b, r, act, keep):
    """-> y, z (what the backward pass needs of the pre-activation: None, y itself, or a tensor of its own)"""
    n, k = w.shape
    x2, ldx = _rows(x)
    w2, ldw = _rows(w)
    m = x2.shape[0]
    device, dtype = x.device, x.dtype
    y = torch.empty((m, n) if x.dim() == 2 else x.shape[:-1] + (n,), dtype=dtype, device=device)
    r2, ldr = _rows(r) if r is not None else (None, n)
    z = None
    if keep and act:
        z = y if act == 1 and r is None else torch.empty(m, n, dtype=dtype, device=device)
    if m and n:
        L, dt, px, pw = _lib(), _TYPES[dtype], x2.data_ptr(), w2.data_ptr()
        ws = _workspace(L.nirrt_nn_linear_workspace(dt, px, ldx, pw, ldw, m, n, k), device)
        _check(L.nirrt_nn_linear(dt, act, px, ldx, pw, ldw, None if b is None else b.data_ptr(), None if r2 is None else r2.data_ptr(), ldr, y.data_ptr(), n,
                                 None if z is None or z is y else z.data_ptr(), m, n, k, _ptr(ws), _stream(device)), "linear")
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, r, act):
        keep = ctx.needs_input_grad[0] or ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        with _on(x.device):
            y, z = _linear_forward(x, w, b, r, act, keep)
        ctx.act = act
        if keep:
            ctx.save_for_backward(x, w, z)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            x, w, z = ctx.saved_tensors
            m, n, k = _prod(x.shape[:-1]), w.shape[0], w.shape[1]
            with _on(x.device):
                dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
                dw = torch.empty(n, k, dtype=x.dtype, device=x.device) if need[1] else None
                db = torch.empty(n, dtype=x.dtype, device=x.device) if need[2] else None
                if n == 0 and dx is not None:
                    dx.zero_()
                dy2, lddy = _rows(dy)
                x2, ldx = _rows(x)
                w2, ldw = _rows(w)
                L, dt = _lib(), _TYPES[x.dtype]
                ws = _workspace(L.nirrt_nn_linear_backward_workspace(dt, ctx.act, x2.data_ptr(), ldx, w2.data_ptr(), ldw, dy2.data_ptr(), lddy,
                                                                     m, n, k), x.device)
                if n:
                    _check(L.nirrt_nn_linear_backward(dt, ctx.act, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(z), dy2.data_ptr(), lddy, _ptr(dx),
                                                      _ptr(dw), _ptr(db), m, n, k, _ptr(ws), _stream(x.device)), "linear_backward")
        return dx, dw, db, (dy if need[3] else None), None


def linear_act(x, weight, bias=None, residual=None, activation="none"):
    """act(x weight^T + bias) + residual: x (..., k), weight (n, k), bias (n,), residual (..., n) -> (..., n), all of one type.
    activation: "none", "relu", "gelu" (with erf) or "silu".  Gradients for x, weight, bias and residual."""
    if activation not in ACTIVATIONS:
        raise ValueError("linear_act: activation %r is not one of %s" % (activation, ", ".join(ACTIVATIONS)))
    _need("linear_act", x, weight=weight, bias=bias, residual=residual)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError("linear_act: x %s and weight %s do not fit" % (tuple(x.shape), tuple(weight.shape)))
    n = weight.shape[0]
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError("linear_act: bias %s, expected (%d,)" % (tuple(bias.shape), n))
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise ValueError("linear_act: residual %s, expected %s" % (tuple(residual.shape), tuple(x.shape[:-1] + (n,))))
    _sizes_ok("linear_act", _prod(x.shape[:-1]), n, weight.shape[1])
    if bias is not None:
        bias = bias.contiguous()
    act = ACTIVATIONS[activation]
    # (dual numbers go through autograd too, which refuses them: there is no forward mode)
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act)
    with _on(x.device):
        return _linear_forward(x, weight, bias, residual, act, False)[0]


# ---- head with softmax cross entropy ---------------------------------------------------------------------------------------------------
def _copy_not_made(address, n, row, apart):
    """the bytes of a copy of n rows of `row` bytes that cross entropy of many classes leaves out of its workspaces where they lie in whole aligned
    16-byte chunks, at most 4 MB apart (include/nirrt_nnops.h)"""
    return 0 if (address | row | apart) & 15 or apart > 1 << 22 else (n * row + 255) & ~255


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, target, cw, ignore, mode):
        rows, (v, k), dev, dtype = target.numel(), w.shape, x.device, x.dtype
        with _on(dev):
            x2, ldx = _rows(x)
            w2, ldw = _rows(w)
            lse = torch.empty(rows, 2, dtype=torch.float32, device=dev)
            nll = torch.empty(target.shape, dtype=torch.float32, device=dev)
            total = torch.empty(3, dtype=torch.float32, device=dev)
            L, dt, px, pw = _lib(), _TYPES[dtype], x2.data_ptr(), w2.data_ptr()
            most = L.nirrt_nn_cross_entropy_workspace(dt, rows, v, k)
            if v > 8:
                e = 2 if dt else 4
                most -= _copy_not_made(px, rows, k * e, ldx * e) + _copy_not_made(pw, v, k * e, ldw * e)
            ws = _workspace(most, dev)
            _check(L.nirrt_nn_cross_entropy(dt, px, ldx, pw, ldw, _ptr(b), target.data_ptr(), _ptr(cw), ignore, lse.data_ptr(),
                                            nll.data_ptr(), total.data_ptr(), rows, v, k, _ptr(ws), _stream(dev)), "cross_entropy")
        ctx.ignore, ctx.mode = ignore, mode
        ctx.save_for_backward(x, w, b, target, cw, lse, total)
        # (.data: no view of `total` for autograd, with a version of its own, so that a caller may scale or add to the loss in place; of
        # `total` the backward pass reads the sum of the weights only)
        return nll if mode == "none" else total[2 if mode == "mean" else 0].data

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, w, b, target, cw, lse, total = ctx.saved_tensors
        rows, (v, k), dev, dtype = target.numel(), w.shape, x.device, x.dtype
        need = ctx.needs_input_grad
        with _on(dev):
            dx = torch.empty(x.shape, dtype=dtype, device=dev) if need[0] else None
            dw = torch.empty(v, k, dtype=dtype, device=dev) if need[1] else None
            db = torch.empty(v, dtype=dtype, device=dev) if need[2] else None
            x2, ldx = _rows(x)
            w2, ldw = _rows(w)
            dloss = dloss.float().contiguous()
            L, dt, pw = _lib(), _TYPES[dtype], w2.data_ptr()
            most = L.nirrt_nn_cross_entropy_backward_workspace(dt, rows, v, k)
            if v > 8:
                e = 2 if dt else 4
                most -= _copy_not_made(pw, v, k * e, ldw * e)
            ws = _workspace(most, dev)
            _check(L.nirrt_nn_cross_entropy_backward(dt, x2.data_ptr(), ldx, pw, ldw, _ptr(b), target.data_ptr(), _ptr(cw), ctx.ignore,
                                                     lse.data_ptr(), dloss.data_ptr(), 1 if ctx.mode == "none" else 0,
                                                     total.data_ptr() if ctx.mode == "mean" else None, _ptr(dx), _ptr(dw), _ptr(db), rows, v, k,
                                                     _ptr(ws), _stream(dev)), "cross_entropy_backward")
        return dx, dw, db, None, None, None, None


def linear_cross_entropy(x, weight, target, bias=None, class_weight=None, ignore_index=-100, reduction="mean"):
    """softmax cross entropy of the scores x weight^T + bias against target, without keeping the scores: x (..., k), weight (classes, k),
    target int64 (...), bias (classes,), class_weight float32 (classes,).  Rows whose target is ignore_index count for nothing (their
    gradients are zero, whatever they hold); any other target outside [0, classes) gives NaN.  reduction: "mean" = sum of weight x loss
    over the sum of weights (NaN if no row counts), "sum", or "none" (the shape of target); the loss is float32.  Gradients for x, weight
    and bias; in float16 they are held relative to the largest dloss x weight of the call, so that rows with 1e-8 of it and less lose digits."""
    name = "linear_cross_entropy"
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("%s: reduction %r is not mean, sum or none" % (name, reduction))
    _need(name, x, weight=weight, bias=bias)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.shape[0] < 1:
        raise ValueError("%s: x %s and weight %s do not fit" % (name, tuple(x.shape), tuple(weight.shape)))
    if target.dtype != torch.int64 or target.device != x.device or target.shape != x.shape[:-1]:
        raise ValueError("%s: target must be int64 %s on %s" % (name, tuple(x.shape[:-1]), x.device))
    v = weight.shape[0]
    if bias is not None and tuple(bias.shape) != (v,):
        raise ValueError("%s: bias %s, expected (%d,)" % (name, tuple(bias.shape), v))
    if class_weight is not None and (class_weight.dtype != torch.float32 or class_weight.device != x.device or tuple(class_weight.shape) != (v,)
                                     or class_weight.requires_grad):
        raise ValueError("%s: class_weight must be float32 (%d,) on %s, without a gradient" % (name, v, x.device))
    rows, k = target.numel(), weight.shape[1]
    _sizes_ok(name, rows, v, k)
    if k > (1 << 20 if x.dtype is torch.float32 else 1 << 21):
        raise ValueError("%s: %d inputs are more than 4 MB" % (name, k))
    if v > 8 and rows >= 1 << 29:
        raise ValueError("%s: %d rows of more than 8 classes" % (name, rows))
    return _LinearCrossEntropy.apply(x, weight, bias.contiguous() if bias is not None else None, target.contiguous(),
                                     class_weight.contiguous() if class_weight is not None else None, int(ignore_index), reduction)


# ---- norm and clipping of many tensors -------------------------------------------------------------------------------------------------
_dtype_of, _layout_of, _wants_grad = operator.attrgetter("dtype"), operator.attrgetter("layout"), operator.attrgetter("requires_grad")
_TENSOR = np.dtype([("data", "<u8"), ("out", "<u8"), ("n", "<i8"), ("dtype", "<i4"), ("out_dtype", "<i4")])   # nirrt_nn_tensor


def _tensor_list(name, tensors):
    """-> the tensors that are not None, their device, their element types if they differ (else the one they share)"""
    _not_recorded(name)
    ts = [t for t in tensors if t is not None]
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError("%s: no forward mode" % name)
    if not ts:
        raise ValueError("%s: no tensors" % name)
    # (one pass per property, without a step of the interpreter per tensor: with hundreds of small tensors the host's time is what counts)
    where = set(map(torch.Tensor.get_device, ts))
    if where == {-1}:
        raise RuntimeError("nirrt_star_amd.nnops.%s got a CPU tensor: the package only has the HIP kernels (move it to 'cuda')" % name)
    types = list(map(_dtype_of, ts))
    kinds = set(types)
    if len(where) != 1 or set(map(_layout_of, ts)) != {torch.strided} or not kinds <= _TYPES.keys():
        raise ValueError("%s: dense float32, bfloat16 or float16 tensors of one device" % name)
    return ts, ts[0].device, _TYPES[types[0]] if len(kinds) == 1 else [_TYPES[t] for t in types]


def _dense(ts):
    return ts if all(map(torch.Tensor.is_contiguous, ts)) else [t if t.is_contiguous() else t.contiguous() for t in ts]


def _table(ts, types):
    tab = np.zeros(len(ts), dtype=_TENSOR)
    tab["data"] = list(map(torch.Tensor.data_ptr, ts))
    tab["n"] = list(map(torch.Tensor.numel, ts))
    tab["dtype"] = types
    return tab


def _norm(tab, dev):
    L = _lib()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = _workspace(L.nirrt_nn_norm_workspace(tab.ctypes.data, len(tab)), dev)
    _check(L.nirrt_nn_norm(tab.ctypes.data, len(tab), norm.data_ptr(), _ptr(ws), _stream(dev)), "norm")
    return norm


@torch.no_grad()
def grad_norm(tensors):
    """2-norm of all elements of the tensors (None entries are skipped), summed in 64 bits in a fixed order -> float32 scalar on their device"""
    ts, dev, types = _tensor_list("grad_norm", tensors)
    with _on(dev):
        return _norm(_table(_dense(ts), types), dev)


@torch.no_grad()
def clip_grad_norm_(grads, max_norm, out=None):
    """scales the tensors by min(1, max_norm / (norm + 1e-6)), norm as grad_norm gives it, and returns the norm (float32 scalar on their
    device; nothing waits for it).  In place, or into `out`: as many contiguous tensors of as many elements each, of any of the three types
    (half-precision gradients into float32 ones, say).  It takes the gradients themselves: a leaf that requires a gradient (a parameter) is
    refused as a tensor to write into.  None entries are skipped (in `out` too).  A tensor may be named once only, and an
    `out` tensor may share memory with its own gradient (of the same type) but not with another one."""
    name = "clip_grad_norm_"
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("%s: max_norm %r" % (name, max_norm))
    grads = list(grads)
    if out is not None:
        out = list(out)
        if len(out) != len(grads) or any((g is None) != (o is None) for g, o in zip(grads, out)):
            raise ValueError("%s: %d gradients, %d outputs (None where the gradient is)" % (name, len(grads), len(out)))
    ts, dev, types = _tensor_list(name, grads)
    src = _dense(ts)
    tab = _table(src, types)
    dst = ts
    if out is None:
        tab["out"], tab["out_dtype"] = tab["data"], tab["dtype"]
    else:
        dst, dev_o, types = _tensor_list(name, out)
        if dev_o != dev or list(map(torch.Tensor.numel, dst)) != tab["n"].tolist() or not all(map(torch.Tensor.is_contiguous, dst)):
            raise ValueError("%s: outputs must be contiguous, of as many elements as the gradients and on their device" % name)
        tab["out"], tab["out_dtype"] = list(map(torch.Tensor.data_ptr, dst)), types
    full = tab[tab["n"] > 0]
    places = set(full["out"].tolist())
    if len(places) != len(full):
        raise ValueError("%s: a tensor is named twice" % name)
    if out is not None and not places.isdisjoint(full["data"].tolist()):
        own = full["out"] == full["data"]
        if not places.isdisjoint(full["data"][~own].tolist()) or ((full["dtype"] != full["out_dtype"]) & own).any():
            raise ValueError("%s: an output shares memory with another gradient, or with its own of another type" % name)
    if any(map(_wants_grad, dst)) and any(t.requires_grad and t.is_leaf for t in dst):
        raise ValueError("%s: a leaf that requires a gradient would be scaled: pass the gradients (p.grad), not the parameters" % name)
    with _on(dev):
        norm = _norm(tab, dev)
        _check(_lib().nirrt_nn_scale_by_norm(tab.ctypes.data, len(tab), norm.data_ptr(), max_norm, _stream(dev)), "scale_by_norm")
        if out is None and src is not ts:
            for t, s in zip(ts, src):
                if s is not t:
                    t.copy_(s)
    # the kernel writes where autograd does not see it: a graph that saved one of these tensors has to find out
    torch.autograd.graph.increment_version(dst)
    return norm
