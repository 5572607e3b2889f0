"""mm_grouped and mm_grouped_wgrad without a GPU: the Python layer's refusals, how it reads operands' layouts, and the C
ABI's argument checks, which come before any device work."""
import ctypes

import pytest
import torch

from spanqr_b200 import _lib, mm_grouped, mm_grouped_wgrad
from spanqr_b200 import grouped as g

OK, SHAPE, ARG = 0, 1, 2
A = 1 << 40             # a device address that no call below dereferences
BF16, FP16 = 2, 1


def test_refusals_on_host_tensors():
    x, w, off = torch.zeros(4, 8).bfloat16(), torch.zeros(2, 8, 8).bfloat16(), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        mm_grouped(x, w, off)
    with pytest.raises(TypeError, match="CUDA"):
        mm_grouped_wgrad(x, x, off)
    with pytest.raises(ValueError, match="2-D"):
        mm_grouped(x[0], w, off)
    with pytest.raises(ValueError, match="2-D"):
        mm_grouped_wgrad(w, x, off)


def test_offset_checks():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="1-D"):
        g._check_offsets(torch.zeros(2, 2, dtype=torch.int32), x)
    with pytest.raises(TypeError, match="int32"):
        g._check_offsets(torch.zeros(2, dtype=torch.int64), x)
    with pytest.raises(ValueError, match="one end per expert"):
        g._check_offsets(torch.zeros(2, dtype=torch.int32), x, 3)
    for n in (0, 1025):
        with pytest.raises(ValueError, match="experts"):
            g._check_offsets(torch.zeros(n, dtype=torch.int32), x)
    o = torch.arange(6, dtype=torch.int32)[::2]
    assert g._check_offsets(o, x).is_contiguous()


@pytest.mark.parametrize("make,copied,ld", [
    (lambda: torch.zeros(5, 64), False, 64), (lambda: torch.zeros(5, 61), True, 64),
    (lambda: torch.zeros(5, 128)[:, :61], False, 128), (lambda: torch.zeros(5, 128)[:, 1:62], True, 64),
    (lambda: torch.zeros(64, 5).t(), True, 64), (lambda: torch.zeros(1, 64).expand(5, 64), True, 64),
    (lambda: torch.zeros(5, 100)[:, :64], True, 64), (lambda: torch.zeros(9, 64)[::2], False, 128),
    (lambda: torch.zeros(1, 61), False, 64), (lambda: torch.zeros(5, 1), True, 8)])
def test_row_operands(make, copied, ld):
    base = make()
    x = torch.zeros(4096, dtype=torch.bfloat16).as_strided(base.shape, base.stride(), base.storage_offset())
    y, got = g._rows(x)
    assert (y.data_ptr() != x.data_ptr()) is copied and got == ld
    assert got % 8 == 0 and y.data_ptr() % 16 == 0


@pytest.mark.parametrize("shape,stride,copied,transposed", [
    ((3, 32, 64), (2048, 64, 1), False, False),        # [E, N, K]
    ((3, 64, 32), (2048, 1, 64), False, True),         # [E, K, N] seen as [E, N, K]
    ((3, 32, 61), (32 * 61, 61, 1), True, False),      # odd rows
    ((3, 61, 32), (61 * 32, 32, 1), False, False),     # odd N only
    ((3, 61, 32), (61 * 32, 1, 61), True, True),       # odd rows of the transposed storage
    ((3, 32, 64), (0, 64, 1), True, False),            # one matrix for all experts
    ((1, 32, 64), (5, 64, 1), False, False),           # a single expert's stride is free
    ((3, 32, 64), (2052, 64, 1), True, False),         # experts off 16 bytes
    ((3, 32, 64), (4096, 128, 2), True, False)])       # contiguous along neither
def test_weight_operands(shape, stride, copied, transposed):
    w = torch.zeros(1 << 15, dtype=torch.bfloat16).as_strided(shape, stride)
    v, ld, plane, tr = g._weights(w)
    assert (v.data_ptr() != w.data_ptr()) is copied and tr is transposed
    E, N, K = shape
    rows, cols = (K, N) if tr else (N, K)
    assert ld % 8 == 0 and plane % 8 == 0 and ld >= cols and plane >= (rows - 1) * ld + cols


def test_overlap():
    b = torch.zeros(64, 64)
    g._no_overlap(b[:32], x=b[32:])
    with pytest.raises(ValueError, match="overlaps x"):
        g._no_overlap(b[:33], x=b[32:])
    g._no_overlap(b[:0], x=b)


def mm(x=A, ldx=64, w=A, ldw=64, sw=64 * 128, tr=0, off=A, y=A, ldy=128, type=BF16, T=16, E=2, N=128, K=64):
    return _lib.lib().spanqr_mm_grouped(x, ldx, w, ldw, sw, tr, off, y, ldy, type, T, E, N, K, 1, None, 0, None)


def wgrad(dy=A, lddy=128, x=A, ldx=64, off=A, dw=A, type=BF16, out=0, T=16, E=2, N=128, K=64):
    return _lib.lib().spanqr_mm_grouped_wgrad(dy, lddy, x, ldx, off, dw, type, out, T, E, N, K, None, 0, None)


def test_argument_checks_before_any_device_work():
    for bad in (dict(T=-1), dict(T=(1 << 30) + 1), dict(E=0), dict(E=1025), dict(N=0), dict(K=0), dict(K=(1 << 24) + 1)):
        assert mm(**bad) == SHAPE, bad
        assert wgrad(**bad) == SHAPE, bad
    for bad in (dict(x=None), dict(x=A + 2), dict(ldx=63), dict(ldx=56), dict(ldx=68), dict(w=None), dict(w=A + 8),
                dict(ldw=60), dict(ldw=56), dict(sw=64 * 127), dict(sw=64 * 128 + 4), dict(off=None), dict(off=A + 2),
                dict(y=None), dict(y=A + 1), dict(ldy=127), dict(type=0), dict(type=3), dict(tr=1, ldw=120)):
        assert mm(**bad) == ARG, bad
    for bad in (dict(dy=None), dict(dy=A + 8), dict(lddy=120), dict(lddy=132), dict(x=None), dict(ldx=60), dict(off=None),
                dict(dw=None), dict(dw=A + 2), dict(out=2, dw=A + 1), dict(out=1), dict(out=3), dict(type=0)):
        assert wgrad(**bad) == ARG, bad
    pad = lambda src=A + 2, plane=999, ld=37, planes=2, rows=27, cols=37, dst=A, ldd=40: _lib.lib().spanqr_mm_pad_rows(  # noqa: E731
        src, plane, ld, planes, rows, cols, dst, ldd, None)
    for bad in (dict(planes=-1), dict(planes=1025), dict(rows=-1), dict(cols=0)):
        assert pad(**bad) == SHAPE, bad
    for bad in (dict(src=None), dict(src=A + 1), dict(plane=-1), dict(ld=-1), dict(dst=None), dict(dst=A + 8), dict(ldd=36),
                dict(ldd=32)):
        assert pad(**bad) == ARG, bad
    assert pad(rows=0) == OK
    assert mm(T=0) == OK                 # nothing to do
    assert _lib.lib().spanqr_mm_read_status(None, None) == ARG
