"""spanqr_b200: spanqr's orth(X) rebuilt for NVIDIA B200 (sm_100a).

    from spanqr_b200 import orth, orth_batched
    Q = orth(X)                  # X: fp32 CUDA [K, r] -> Q, Q^T Q = I, span(Q) = span(X)
    Qs = orth_batched([X1, X2])  # many layers at once; across GPUs under torch.distributed
    grads, n = clip_grads(grads, 1.0)   # the list's global norm, and the list scaled to it (grad_norm: the norm alone)
    y = mm_grouped(x, w, offsets)       # products grouped by expert; mm_grouped_wgrad: their weight gradients in fp32
    mm_check()                          # raises if a product's kernel gave up waiting (synchronises)

The compute runs in libspanqr.so (CUDA kernels behind the C ABI of include/spanqr.h); this package only binds it.
"""
from .core import orth, zdust, workspace, TB, MAX_R, DUST_SEED
from .batched import orth_batched, partition
from .grads import grad_norm, clip_grads
from .grouped import mm_grouped, mm_grouped_wgrad, mm_check
from ._lib import SpanqrError, workspace_bytes

__all__ = ["orth", "orth_batched", "grad_norm", "clip_grads", "mm_grouped",
           "mm_grouped_wgrad", "mm_check", "partition", "zdust", "workspace", "workspace_bytes", "SpanqrError",
           "register_qrbench", "TB", "MAX_R", "DUST_SEED"]


def register_qrbench(name="b200"):
    """Register orth with the reference harness's method registry (qrbench/methods.py:15-20), so that
    `python -m qrbench.check -m b200` and `python -m qrbench.bench -m b200` run this implementation."""
    from qrbench.methods import register
    register(name)(lambda X: orth(X))
    return name
