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
from itertools import compress
from operator import attrgetter

import torch
import torch.distributed as dist

from . import _lib

# SPANQR_F32, SPANQR_F16, SPANQR_BF16
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_dtype, _same_size = attrgetter("dtype"), torch.Tensor.is_same_size
_contiguous = torch.Tensor.is_contiguous
_neg = torch.Tensor.is_neg
_PLAIN = {torch.Tensor, torch.nn.Parameter}
_ptr, _numel, _device = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device


def _dense(t):
    """whether t's elements fill one block of memory without holes, in any order of its dimensions"""
    n = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != n:
            return False
        n *= size
    return True


def _check(tensors, name, like=None):
    """the list as a list, its types, its device's index (None when empty) and its dtypes; like: types and dtypes of another
    list, whose types are these where the dtypes are"""
    if torch.is_tensor(tensors):
        raise TypeError(f"{name} must be a list of tensors (got one tensor)")
    ts = list(tensors)
    if not set(map(type, ts)) <= _PLAIN and not all(map(torch.is_tensor, ts)):
        raise TypeError(f"{name} must hold tensors only")
    dtypes = list(map(_dtype, ts))
    kinds = set(dtypes)
    if not kinds <= DTYPES.keys():
        raise TypeError(f"{name} must be fp32, fp16 or bf16 (got {', '.join(map(str, kinds - DTYPES.keys()))})")
    devs = set(map(_device, ts))
    if -1 in devs:
        raise TypeError(f"{name} must be CUDA tensors")
    if len(devs) > 1:
        raise ValueError(f"{name} must be on one device (got cuda:{', cuda:'.join(map(str, sorted(devs)))})")
    if like is not None and dtypes == like[1]:
        types = like[0]
    else:
        types = array("i", [DTYPES[kinds.pop()]]) * len(ts) if len(kinds) == 1 else array("i", map(DTYPES.get, dtypes))
    return ts, types, devs.pop() if devs else None, dtypes


def _at(a):
    return a.buffer_info()[0]


_WS_BYTES = {}


def _norm_like(ts, dev):
    """where the norm goes"""
    return ts[0].new_empty((), dtype=torch.float32) if ts else torch.empty((), dtype=torch.float32, device=dev)


def _workspace(like, count):
    bytes_ = _WS_BYTES.get(count)
    if bytes_ is None:
        n = _lib.ctypes.c_size_t(0)
        _lib.check(_lib.lib().spanqr_grad_workspace_bytes(count, _lib.ctypes.byref(n)), f"grad_workspace_bytes({count})")
        bytes_ = _WS_BYTES[count] = n.value
    return like.new_empty(bytes_, dtype=torch.uint8)


def _run_norm(ts, types, dev, sumsq, norm):
    """the norm's kernels for contiguous tensors ts; sumsq and norm are tensors or None"""
    ws = _workspace(sumsq if norm is None else norm, len(ts))
    ptrs, sizes = array("Q", map(_ptr, ts)), array("q", map(_numel, ts))
    _lib.launch(dev, _lib.lib().spanqr_grad_norm, lambda: f"grad_norm({len(ts)} tensors)", _at(ptrs), _at(types),
                _at(sizes), len(ts), None if sumsq is None else sumsq.data_ptr(), None if norm is None else norm.data_ptr(),
                ws.data_ptr(), ws.numel())


def _run_clip(ins, in_types, outs, out_types, dev, max_norm, sumsq, norm):
    ws = _workspace(norm, len(ins))
    pi, po, sizes = array("Q", map(_ptr, ins)), array("Q", map(_ptr, outs)), array("q", map(_numel, ins))
    try:
        _lib.launch(dev, _lib.lib().spanqr_grad_clip, lambda: f"clip_grads({len(ins)} tensors)", _at(pi), _at(in_types),
                    _at(po), _at(out_types), _at(sizes), len(ins), max_norm, None if sumsq is None else sumsq.data_ptr(),
                    norm.data_ptr(), ws.data_ptr(), ws.numel())
    except _lib.SpanqrError as e:
        if e.code != 7:   # SPANQR_ERR_OVERLAP
            raise
        raise ValueError("clip_grads: an output overlaps another tensor of the call (one tensor listed twice?)") from None


def _any_negated(ts, types):
    """whether a tensor's memory holds its values negated, as that of z.conj().imag does (no bf16 one can: there is no complex
    type of such parts)"""
    bf16 = types.count(2)   # SPANQR_BF16
    if bf16 == 0:
        return True in map(_neg, ts)
    return bf16 < len(ts) and True in map(_neg, compress(ts, [t != 2 for t in types]))


def _signs(ins, in_types, outs, out_types):
    """ins, with those resolved that are negated lazily where their output is not (two such are scaled as they lie)"""
    if not (_any_negated(ins, in_types) or _any_negated(outs, out_types)):
        return ins
    ins = list(ins)
    for i, (t, o) in enumerate(zip(ins, outs)):
        if t.is_neg() != o.is_neg():
            if o.is_neg():
                raise ValueError(f"out[{i}] is a lazily negated view and its input is not: give a tensor of its own")
            ins[i] = t.resolve_neg()
    return ins


def _refused(group):
    """this rank's part in the all-reduce of a call that it is about to raise from: a NaN for its sum.  The other ranks do not
    wait for it then, and see by their norm that something was wrong"""
    if group is not None:
        dev = torch.cuda.current_device() if torch.cuda.is_available() else "cpu"
        dist.all_reduce(torch.full((), float("nan"), dtype=torch.float64, device=dev), group=group)


def _group_sumsq(ts, types, dev, group):
    """the list's sum of squares (fp64), summed over the group's ranks"""
    with torch.cuda.device(dev):
        try:
            sumsq = torch.empty((), dtype=torch.float64, device=dev)
            _run_norm(ts, types, dev, sumsq, None)
        except Exception:
            _refused(group)
            raise
        dist.all_reduce(sumsq, group=group)
    return sumsq


def grad_norm(tensors, *, group=None):
    """The L2 norm over all elements of a list of fp32, fp16 or bf16 CUDA tensors on one device, as a 0-dim fp32 tensor.
    A tensor listed twice counts twice; an empty list gives 0.  With `group` (a torch.distributed process group whose
    ranks each hold their own part of the gradients) the norm is over all ranks' lists, through one 8-byte all-reduce
    of the sum of squares; every rank of the group must call, with an empty list if it holds nothing (where one's list is
    refused the others get NaN).  Without it the norm is of this process's list alone.  Deterministic; large and small
    values do not overflow or vanish in their squares.  Not differentiable."""
    try:
        ts, types, dev, _ = _check(tensors, "tensors")
    except Exception:
        _refused(group)
        raise
    if dev is None:
        dev = torch.cuda.current_device()
    if not all(map(_contiguous, ts)):
        ts = [t if _dense(t) else t.contiguous() for t in ts]
    norm = _norm_like(ts, dev)
    if group is None:
        _run_norm(ts, types, dev, None, norm)
    else:   # an empty list's clipping gives the sum's square root
        none = array("i")
        _run_clip([], none, [], none, dev, 0.0, _group_sumsq(ts, types, dev, group), norm)
    return norm


def _clip_operands(tensors, max_norm, out):
    """the checked operands of a clipping: max_norm, the inputs as the kernels read them, their types and device, the
    outputs and their types, and where the norm goes"""
    if torch.is_tensor(max_norm):
        raise TypeError("max_norm must be a number (reading a tensor would wait for the device)")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number >= 0 (got {max_norm})")
    ts, types, dev, dtypes = _check(tensors, "tensors")
    if out is None:
        ins = ts if all(map(_contiguous, ts)) else [t.contiguous() for t in ts]
        res, out_types = [torch.empty_like(t, requires_grad=False) for t in ins], types
    else:
        res, out_types, odev, _ = _check(out, "out", (types, dtypes))
        if len(res) != len(ts):
            raise ValueError(f"out must hold {len(ts)} tensors (got {len(res)})")
        if odev != dev:
            raise ValueError(f"out must be on the tensors' device (got cuda:{odev} and cuda:{dev})")
        if not all(map(_same_size, ts, res)):
            i = next(i for i, (t, o) in enumerate(zip(ts, res)) if t.shape != o.shape)
            raise ValueError(f"out[{i}] has shape {tuple(res[i].shape)}, its input {tuple(ts[i].shape)}")
        if out_types is not types:
            for i, (t, o) in enumerate(zip(ts, res)):
                if o.dtype != t.dtype and o.dtype != torch.float32:
                    raise TypeError(f"out[{i}] must be {t.dtype} or fp32 (got {o.dtype})")
        ins = ts
        if not (all(map(_contiguous, ts)) and all(map(_contiguous, res))):
            ins = [_like_output(i, t, o) for i, (t, o) in enumerate(zip(ts, res))]
    if out is not tensors:
        ins = _signs(ins, types, res, out_types)
    if dev is None:
        dev = torch.cuda.current_device()
    return max_norm, ins, types, dev, res, out_types, _norm_like(ts, dev)


def clip_grads(tensors, max_norm, *, out=None, group=None):
    """(clipped, norm): every tensor scaled by min(1, max_norm / (norm + 1e-6)), norm the list's L2 norm before it (as
    grad_norm gives it; `group` as there).  max_norm is a number >= 0.

    `out`: None for new tensors of the inputs' types, or a list of tensors of the inputs' shapes, each of its input's
    type or fp32 (so that bf16 gradients reach orth as fp32 in one pass).  An output may be its own input (in place),
    but overlaps no other tensor of the call.  Outputs must be contiguous, or dense with their input's strides.  An
    infinite gradient gives the coefficient 0 (finite values become 0, infinite ones NaN) and a NaN makes every output
    NaN, so a step can be skipped by looking at the norm alone.  A finite norm above fp32's largest value reads as
    infinity, but the scaling uses its fp64 value.  Autograd does not see the scaling.  Lazily negated inputs (z.conj().imag)
    are resolved, and such outputs refused unless their input is one too."""
    try:
        max_norm, ins, types, dev, res, out_types, norm = _clip_operands(tensors, max_norm, out)
    except Exception:
        _refused(group)
        raise
    sumsq = None if group is None else _group_sumsq(ins, types, dev, group)
    _run_clip(ins, types, res, out_types, dev, max_norm, sumsq, norm)
    if out is not None and res:
        try:
            torch.autograd.graph.increment_version(res)
        except RuntimeError:   # tensors of inference mode have no version
            torch.autograd.graph.increment_version([o for o in res if not o.is_inference()])
    return res, norm


def _like_output(i, t, o):
    """t, or a contiguous copy of it, with its elements in o's order in memory"""
    if t.stride() == o.stride() and _dense(t):
        return t
    if not o.is_contiguous():
        raise ValueError(f"out[{i}] must be contiguous, or dense with its input's strides")
    return t.contiguous()
