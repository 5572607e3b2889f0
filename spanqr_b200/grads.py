"""The global norm of a list of gradients and its clipping: the step before orth in an optimizer (no reference
counterpart; the reference orthonormalises what it is given).

    from spanqr_b200 import grad_norm, clip_grads
    n = grad_norm(grads)                              # 0-dim fp32 tensor: sqrt of the sum of all squares
    clipped, n = clip_grads(grads, 1.0)               # new tensors; grads untouched
    clip_grads(grads, 1.0, out=grads)                 # in place

Both run on libspanqr's kernels on the current stream of the tensors' device, with no host synchronisation; the
workspace comes from torch's allocator per call, so calls on different streams and captured graphs never share one.
"""
from array import array
from operator import attrgetter, methodcaller

import torch
import torch.distributed as dist

from . import _lib

# SPANQR_F32, SPANQR_F16, SPANQR_BF16
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_dtype, _contiguous = attrgetter("dtype"), methodcaller("is_contiguous")
_ptr, _numel, _device = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device


def _dense(t):
    """whether t's elements fill one block of memory without holes, in any order of its dimensions"""
    n = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != n:
            return False
        n *= size
    return True


def _check(tensors, name):
    """the list as a list, and its device (None when empty)"""
    if torch.is_tensor(tensors):
        raise TypeError(f"{name} must be a list of tensors (got one tensor)")
    ts = list(tensors)
    if not all(map(torch.is_tensor, ts)):
        raise TypeError(f"{name} must hold tensors only")
    bad = set(map(_dtype, ts)) - DTYPES.keys()
    if bad:
        raise TypeError(f"{name} must be fp32, fp16 or bf16 (got {', '.join(map(str, bad))})")
    devs = set(map(_device, ts))
    if -1 in devs:
        raise TypeError(f"{name} must be CUDA tensors")
    if len(devs) > 1:
        raise ValueError(f"{name} must be on one device (got cuda:{', cuda:'.join(map(str, sorted(devs)))})")
    return ts, (torch.device("cuda", devs.pop()) if devs else None)


def _types(ts):
    kinds = set(map(_dtype, ts))
    if len(kinds) == 1:
        return array("i", [DTYPES[kinds.pop()]]) * len(ts)
    return array("i", [DTYPES[d] for d in map(_dtype, ts)])


def _at(a):
    return a.buffer_info()[0]


def _workspace(dev, count):
    n = _lib.ctypes.c_size_t(0)
    _lib.check(_lib.lib().spanqr_grad_workspace_bytes(count, _lib.ctypes.byref(n)), f"grad_workspace_bytes({count})")
    return torch.empty(n.value, dtype=torch.uint8, device=dev)


def _run_norm(ts, dev, sumsq, norm, stream):
    """the norm's kernels for contiguous tensors ts; sumsq and norm are tensors or None"""
    ws = _workspace(dev, len(ts))
    ptrs, kinds, sizes = array("Q", map(_ptr, ts)), _types(ts), array("q", map(_numel, ts))
    _lib.check(_lib.lib().spanqr_grad_norm(_at(ptrs), _at(kinds), _at(sizes), len(ts),
                                           None if sumsq is None else sumsq.data_ptr(),
                                           None if norm is None else norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                           stream), f"grad_norm({len(ts)} tensors)")


def _run_clip(ins, outs, dev, max_norm, sumsq, norm, stream):
    ws = _workspace(dev, len(ins))
    pi, po, sizes = array("Q", map(_ptr, ins)), array("Q", map(_ptr, outs)), array("q", map(_numel, ins))
    ki, ko = _types(ins), _types(outs)
    rc = _lib.lib().spanqr_grad_clip(_at(pi), _at(ki), _at(po), _at(ko), _at(sizes), len(ins), max_norm,
                                     None if sumsq is None else sumsq.data_ptr(), norm.data_ptr(), ws.data_ptr(),
                                     ws.numel(), stream)
    if rc == 7:   # SPANQR_ERR_OVERLAP
        raise ValueError("clip_grads: an output overlaps another tensor of the call (the same tensor listed twice?)")
    _lib.check(rc, f"clip_grads({len(ins)} tensors)")


def _group_sumsq(ts, dev, group, stream):
    """the list's sum of squares (fp64), summed over the group's ranks"""
    sumsq = torch.empty((), dtype=torch.float64, device=dev)
    _run_norm(ts, dev, sumsq, None, stream)
    dist.all_reduce(sumsq, group=group)
    return sumsq


def grad_norm(tensors, *, group=None):
    """The L2 norm over all elements of a list of fp32, fp16 or bf16 CUDA tensors on one device, as a 0-dim fp32 tensor.
    A tensor listed twice counts twice; an empty list gives 0.  With `group` (a torch.distributed process group whose
    ranks each hold their own part of the gradients) the norm is over all ranks' lists, through one 8-byte all-reduce
    of the sum of squares; every rank of the group must call, with an empty list if it holds nothing.  Without it the
    norm is of this process's list alone.  Deterministic; large and small values do not overflow or vanish in their
    squares.  Not differentiable."""
    ts, dev = _check(tensors, "tensors")
    if dev is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    ts = [t if t.is_contiguous() or _dense(t) else t.contiguous() for t in ts]
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        norm = torch.empty((), dtype=torch.float32, device=dev)
        if group is None:
            _run_norm(ts, dev, None, norm, stream)
        else:
            _run_clip([], [], dev, 0.0, _group_sumsq(ts, dev, group, stream), norm, stream)   # its square root
    return norm


def clip_grads(tensors, max_norm, *, out=None, group=None):
    """(clipped, norm): every tensor scaled by min(1, max_norm / (norm + 1e-6)), norm the list's L2 norm before it (as
    grad_norm gives it; `group` as there).  max_norm is a number >= 0.

    `out`: None for new tensors of the inputs' types, or a list of tensors of the inputs' shapes, each of its input's
    type or fp32 (so that bf16 gradients reach orth as fp32 in one pass).  An output may be its own input (in place),
    but overlaps no other tensor of the call.  Outputs must be contiguous, or dense with their input's strides.  An
    infinite gradient gives the coefficient 0 (finite values become 0, infinite ones NaN) and a NaN makes every output
    NaN, so a step can be skipped by looking at the norm alone.  A finite norm above fp32's largest value reads as
    infinity, but the scaling uses its fp64 value.  Autograd does not see the scaling."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number >= 0 (got {max_norm})")
    ts, dev = _check(tensors, "tensors")
    if out is None:
        ins = ts if all(map(_contiguous, ts)) else [t.contiguous() for t in ts]
        res = outs = [torch.empty_like(t, memory_format=torch.contiguous_format, requires_grad=False) for t in ins]
    else:
        res, odev = _check(out, "out")
        outs = res
        if len(res) != len(ts):
            raise ValueError(f"out must hold {len(ts)} tensors (got {len(res)})")
        if odev != dev:
            raise ValueError(f"out must be on the tensors' device (got {odev} and {dev})")
        ins = []
        for i, (t, o) in enumerate(zip(ts, outs)):
            if t is not o:
                if o.shape != t.shape:
                    raise ValueError(f"out[{i}] has shape {tuple(o.shape)}, its input {tuple(t.shape)}")
                if o.dtype != t.dtype and o.dtype != torch.float32:
                    raise TypeError(f"out[{i}] must be {t.dtype} or fp32 (got {o.dtype})")
            if not (t.is_contiguous() and o.is_contiguous()):
                if t.stride() == o.stride() and _dense(t):
                    pass
                elif not o.is_contiguous():
                    raise ValueError(f"out[{i}] must be contiguous, or dense with its input's strides")
                else:
                    t = t.contiguous()
            ins.append(t)
    if dev is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        norm = torch.empty((), dtype=torch.float32, device=dev)
        sumsq = None if group is None else _group_sumsq(ins, dev, group, stream)
        _run_clip(ins, outs, dev, max_norm, sumsq, norm, stream)
    if out is not None and res:
        torch.autograd.graph.increment_version([o for o in res if not o.is_inference()])
    return res, norm
