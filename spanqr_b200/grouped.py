"""Matrix products grouped by expert: rows sorted by expert, a ragged number of them each (no reference counterpart; the
layers whose gradients clip_grads and orth_batched then take).

    from spanqr_b200 import mm_grouped, mm_grouped_wgrad
    y = mm_grouped(x, w, offsets)                 # y[t] = w[e(t)] @ x[t], differentiable in x and w
    dw = mm_grouped_wgrad(dy, x, offsets)         # dw[e] = sum over e's rows of dy[t] x[t]^T, fp32: orth's input type
    mm_check()                                    # raises if a kernel of theirs gave up a wait (synchronises)

x is [T, K] with the rows of expert e at offsets[e - 1] .. offsets[e] (offsets: int32 on the GPU, the cumulative sum of
the rows per expert), w is [E, N, K], bf16 or fp16.  Everything runs on libspanqr's kernels on the current stream of x's
device; the offsets are only read on the device, so nothing synchronises with the host.
"""
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .grads import DTYPES

MAX_EXPERTS = 1024
INT_MAX = 2 ** 31 - 1


@functools.lru_cache(maxsize=4096)
def _ws_bytes(fn, *sizes):
    n = _lib.ctypes.c_size_t(0)
    _lib.check(getattr(_lib.lib(), fn)(*sizes, _lib.ctypes.byref(n)), f"{fn}{sizes}")
    return n.value


def _workspace(fn, x, *sizes):
    """a workspace for one call (None where it needs none), its address and size: from torch's allocator each time, so that
    calls on different streams and captured graphs never share one"""
    n = _ws_bytes(fn, *sizes)
    if n == 0:
        return None, None, 0
    ws = x.new_empty(n, dtype=torch.uint8)
    return ws, ws.data_ptr(), n


def _rows(x):
    """x [T, K] with contiguous rows, its address and row stride, and whether the library has to copy it to read it (rows
    off 16 bytes or over one another)"""
    if x.is_neg():   # (z.conj().imag: its memory holds the values negated)
        x = x.resolve_neg()
    ld, step = x.stride()
    if step != 1 and x.shape[1] > 1 or ld < 0:
        x = x.contiguous()
        ld = x.stride(0)
    ptr = x.data_ptr()
    return x, ptr, ld, ptr % 16 != 0 or x.shape[0] > 1 and (ld % 8 != 0 or ld < x.shape[1])


def _weights(w):
    """w [E, N, K] with one of its last two dimensions contiguous, its address, row stride, expert stride, whether it is
    stored [E, K, N], and whether the library has to copy it to read it"""
    if w.is_neg():
        w = w.resolve_neg()
    E, N, K = w.shape
    plane, sn, sk = w.stride()
    if sk == 1 or K == 1:
        rows, cols, ld, transposed = N, K, sn, False
    elif sn == 1 or N == 1:
        rows, cols, ld, transposed = K, N, sk, True
    else:
        return _weights(w.contiguous())
    ptr = w.data_ptr()
    copy = (ptr % 16 != 0 or rows > 1 and (ld % 8 != 0 or ld < cols) or
            E > 1 and (plane % 8 != 0 or plane < (rows - 1) * ld + cols))
    return w, ptr, ld, plane, transposed, copy


def _span(t):
    a = t.data_ptr()
    if t.numel() == 0:
        return a, a
    return a, a + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _side_by_side(a, b):
    """whether two matrices are different columns of one: rows of one stride that never meet"""
    if a.dim() != 2 or b.dim() != 2 or a.dtype != b.dtype or a.stride(0) != b.stride(0) or a.stride(1) != 1 or b.stride(1) != 1:
        return False
    step = a.stride(0) * a.element_size()
    gap = (b.data_ptr() - a.data_ptr()) % step if step else 0   # from a row of a to the next start of one of b
    return a.shape[1] * a.element_size() <= gap and gap + b.shape[1] * b.element_size() <= step


def _check_out(out, **others):
    """refuses an output that cannot be written as it lies: one that autograd follows (its gradient would go to what it held
    before), negated lazily, or over one of the other tensors"""
    if _tracked(out, out):
        raise RuntimeError("out requires a gradient, and its values would come from outside autograd: give out.detach(), or "
                           "use torch.no_grad()")
    if out.is_neg():
        raise ValueError("out is a lazily negated view (out.resolve_neg() gives a tensor of its own)")
    _no_overlap(out, **others)


def _no_overlap(out, **others):
    a, b = _span(out)
    for name, t in others.items():
        c, d = _span(t)
        if a < d and c < b and not _side_by_side(out, t):
            raise ValueError(f"out overlaps {name}")


def _check_sizes(name, *sizes):
    """the library's error for sizes beyond its int arguments, which would reach it cut to 32 bits (2^32 + 5 rows as 5); it
    checks its own lower limits itself"""
    if max(sizes) > INT_MAX:
        raise _lib.SpanqrError(1, f"{name} {'x'.join(map(str, sizes))}")   # SPANQR_ERR_SHAPE


def _check_rows(x, name):
    if not torch.is_tensor(x) or x.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor")
    rows, cols = x.shape
    if rows > INT_MAX or cols > INT_MAX:
        _check_sizes(name, rows, cols)
    if x.dtype not in (torch.bfloat16, torch.float16) or not x.is_cuda:
        raise TypeError(f"{name} must be a bf16 or fp16 CUDA tensor (got {x.dtype} on {x.device})")
    if cols < 1:
        raise ValueError(f"{name} has no columns")
    return rows, cols


def _check_offsets(offsets, x, E=None):
    if not torch.is_tensor(offsets) or offsets.dim() != 1:
        raise ValueError("offsets must be a 1-D tensor: the end of each expert's rows")
    if offsets.dtype != torch.int32 or offsets.get_device() != x.get_device():
        raise TypeError(f"offsets must be int32 on {x.device} (got {offsets.dtype} on {offsets.device})")
    n = offsets.shape[0]
    if E is not None and n != E:
        raise ValueError(f"offsets must have one end per expert: {E} (got {n})")
    if not 1 <= n <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts (got {n})")
    return offsets if offsets.stride(0) == 1 or n == 1 else offsets.contiguous()


def _product(rows, weights, offsets, T, E, N, K, out=None):
    """y [T, N] of operands as _rows and _weights give them, the weights [E, N, K]"""
    x, px, ldx, copy_x = rows
    w, pw, ldw, plane, transposed, copy_w = weights
    y = x.new_empty((T, N)) if out is None else out
    if T == 0:
        return y
    ws, pws, n = _workspace("spanqr_mm_grouped_workspace_bytes", x, T, E, N, K, copy_x + 2 * copy_w + 4 * transposed)
    _lib.launch(x.get_device(), _lib.lib().spanqr_mm_grouped, lambda: f"mm_grouped({T}x{K}, {E} experts of {N}x{K})", px, ldx,
                pw, ldw, plane, transposed, offsets.data_ptr(), y.data_ptr(), y.stride(0), DTYPES[x.dtype], T, E, N, K,
                out is None, pws, n)
    return y


def _wgrad(rows_dy, rows_x, offsets, T, E, N, K, dtype, out=None):
    """dw [E, N, K] of operands as _rows gives them"""
    dy, pdy, lddy, copy_dy = rows_dy
    x, px, ldx, copy_x = rows_x
    dw = x.new_empty((E, N, K), dtype=dtype) if out is None else out
    ws, pws, n = _workspace("spanqr_mm_grouped_wgrad_workspace_bytes", x, T, E, N, K, copy_dy + 2 * copy_x)
    _lib.launch(x.get_device(), _lib.lib().spanqr_mm_grouped_wgrad,
                lambda: f"mm_grouped_wgrad({T} rows, {E} experts of {N}x{K})", pdy, lddy, px, ldx, offsets.data_ptr(),
                dw.data_ptr(), DTYPES[x.dtype], DTYPES[dw.dtype], T, E, N, K, pws, n)
    return dw


def _tracked(x, w):
    """whether autograd follows either of them: backward, or forward with a tangent (make_dual)"""
    return torch.is_grad_enabled() and (x.requires_grad or w.requires_grad) or _dual(x, w)


def _dual(x, w):
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (x, w))


def _backward(ctx, dy):
    x, w, offsets = ctx.saved_tensors
    T, N = dy.shape
    E, _, K = w.shape
    rows_dy, dx, dw = _rows(dy), None, None
    if ctx.needs_input_grad[0]:
        v, ptr, ld, plane, transposed, copy = _weights(w)
        dx = _product(rows_dy, (v, ptr, ld, plane, not transposed, copy), offsets, T, E, K, N)
    if ctx.needs_input_grad[1]:
        dw = _wgrad(rows_dy, _rows(x), offsets, T, E, N, K, w.dtype)
    return dx, dw, None


_backward_once = once_differentiable(_backward)


class _MmGrouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        ctx.save_for_backward(x, w, offsets)
        T, K = x.shape
        E, N, _ = w.shape
        return _product(_rows(x), _weights(w), offsets, T, E, N, K)

    @staticmethod
    def backward(ctx, dy):
        # (under create_graph the gradients say that they cannot be differentiated again)
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def mm_grouped(x, w, offsets, *, out=None):
    """y [T, N] with y[t] = w[e(t)] @ x[t] for the expert e(t) whose rows hold t: x [T, K] and w [E, N, K] of one type
    (bf16 or fp16), offsets int32 [E], the end of each expert's rows.  Experts may be empty; w may be stored [E, N, K] or
    [E, K, N] (pass its transposed view).  Rows from offsets[-1] on belong to no expert: they are zero in a new y and
    left as they are in `out`, a [T, N] tensor of x's type with contiguous rows that overlaps neither input and needs no
    gradient.  The products are summed in fp32 by the tensor cores, which round toward zero (about 1e-9 K of the result),
    and rounded once; N and K are at most 2^18.

    Operands whose rows do not start on 16 bytes (K not a multiple of 8, odd strides or addresses), or that are contiguous
    along neither dimension, are copied first, at each call.  Ends that decrease or lie outside [0, T] are clamped to
    the nearest that do not, on the device.

    Differentiable once in x and w, backward only (without `out`; forward-mode tangents are refused): dx is this product with
    the transposed weights, dw is mm_grouped_wgrad in w's type; rows behind the last expert get a zero gradient and give
    none."""
    T, K = _check_rows(x, "x")
    if not torch.is_tensor(w) or w.dim() != 3 or w.shape[2] != K:
        raise ValueError(f"w must be a 3-D tensor [E, N, {K}]")
    E, N, _ = w.shape
    if N > INT_MAX:
        _check_sizes("w", E, N, K)
    if w.dtype != x.dtype or w.get_device() != x.get_device():
        raise TypeError(f"w must be {x.dtype} on {x.device}, as x (got {w.dtype} on {w.device})")
    if N < 1:
        raise ValueError("w has no rows")
    offsets = _check_offsets(offsets, x, E)
    grad = _tracked(x, w)
    if out is None:
        if grad and _dual(x, w):
            raise RuntimeError("mm_grouped has no forward-mode derivative (forward AD): it is differentiable backward only")
        return _MmGrouped.apply(x, w, offsets) if grad else _product(_rows(x), _weights(w), offsets, T, E, N, K)
    if grad:
        raise RuntimeError("mm_grouped with out= is not differentiable: leave out away, or use torch.no_grad()")
    if not torch.is_tensor(out) or out.shape != (T, N):
        raise ValueError(f"out must have shape {(T, N)}")
    if out.dtype != x.dtype or out.device != x.device:
        raise TypeError(f"out must be {x.dtype} on {x.device} (got {out.dtype} on {out.device})")
    if N > 1 and out.stride(1) != 1 or T > 1 and out.stride(0) < N:
        raise ValueError("out must have contiguous rows that do not overlap")
    _check_out(out, x=x, w=w, offsets=offsets)
    _product(_rows(x), _weights(w), offsets, T, E, N, K, out)
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return out


def mm_grouped_wgrad(dy, x, offsets, *, out=None, dtype=None):
    """dw [E, N, K] with dw[e] = sum over expert e's rows t of dy[t] x[t]^T: the weight gradient of mm_grouped.  dy [T, N]
    and x [T, K] of one type (bf16 or fp16), offsets int32 [E] as there; an expert without rows gets zeros, and rows from
    offsets[-1] on count nowhere.  dtype is fp32 (the default: what clip_grads and orth_batched take) or the inputs' type;
    `out`, a contiguous [E, N, K] tensor of either type that overlaps neither input and needs no gradient, is overwritten.
    Summed in fp32 (over 512 rows, or 2048 for 16-bit results, by the tensor cores, those sums to nearest) and rounded
    once.  Not differentiable."""
    T, N = _check_rows(dy, "dy")
    rows, K = _check_rows(x, "x")
    if rows != T:
        raise ValueError(f"dy and x must have as many rows (got {T} and {rows})")
    if dy.dtype != x.dtype or dy.get_device() != x.get_device():
        raise TypeError(f"dy must be {x.dtype} on {x.device}, as x (got {dy.dtype} on {dy.device})")
    offsets = _check_offsets(offsets, x)
    E = offsets.shape[0]
    if out is None:
        dtype = torch.float32 if dtype is None else dtype
        if dtype not in (torch.float32, x.dtype):
            raise TypeError(f"dtype must be fp32 or {x.dtype} (got {dtype})")
        return _wgrad(_rows(dy), _rows(x), offsets, T, E, N, K, dtype)
    if dtype is not None:
        raise ValueError("give dtype or out, not both")
    if not torch.is_tensor(out) or out.shape != (E, N, K) or not out.is_contiguous():
        raise ValueError(f"out must be contiguous with shape {(E, N, K)}")
    if out.dtype not in (torch.float32, x.dtype) or out.device != x.device:
        raise TypeError(f"out must be fp32 or {x.dtype} on {x.device} (got {out.dtype} on {out.device})")
    _check_out(out, dy=dy, x=x, offsets=offsets)
    _wgrad(_rows(dy), _rows(x), offsets, T, E, N, K, None, out)
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return out


def mm_check(device=None):
    """Raises SpanqrError if a kernel of mm_grouped or mm_grouped_wgrad gave up one of its device waits (2 s each) on this
    device since the last check, whichever stream it ran on; its results, and any after it, must not be used.  The calls
    themselves cannot say so without waiting: check where a program synchronises anyway, before it keeps what it computed
    (a step's loss, a checkpoint).  Waits for the device's current stream: other streams' calls are reported once they have
    ended.  Not inside a capture.  device: an index, a torch.device or its name; the current one by default."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"device must be a CUDA device (got {device})")
    index = torch.cuda.current_device() if device.index is None else device.index
    with torch.cuda.device(index):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("mm_check waits for the stream, which a capture does not allow")
        status = _lib.ctypes.c_int(0)
        rc = _lib.lib().spanqr_mm_read_status(torch._C._cuda_getCurrentRawStream(index), _lib.ctypes.byref(status))
    if rc:
        raise _lib.SpanqrError(rc, f"mm_check(cuda:{index}): a product's wait ran out (status 0x{status.value:x})" if
                               rc == 5 else f"mm_check(cuda:{index})")   # SPANQR_ERR_DEVICE
