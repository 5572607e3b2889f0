"""mm_grouped and mm_grouped_wgrad without a GPU: the Python layer's refusals, how it reads operands' layouts, and the C
ABI's argument checks, which come before any device work."""
import ctypes

import pytest
import torch

from spanqr_b200 import _lib, mm_check, mm_grouped, mm_grouped_wgrad
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


@pytest.mark.parametrize("make,contiguous,copied", [
    (lambda: torch.zeros(5, 64), False, False), (lambda: torch.zeros(5, 61), False, True),
    (lambda: torch.zeros(5, 128)[:, :61], False, False), (lambda: torch.zeros(5, 128)[:, 1:62], False, True),
    (lambda: torch.zeros(64, 5).t(), True, False), (lambda: torch.zeros(1, 64).expand(5, 64), False, True),
    (lambda: torch.zeros(5, 100)[:, :64], False, True), (lambda: torch.zeros(9, 64)[::2], False, False),
    (lambda: torch.zeros(1, 61), False, False), (lambda: torch.zeros(5, 1), False, True)])
def test_row_operands(make, contiguous, copied):
    """made contiguous where its rows are not; left to the library to copy where its rows are off 16 bytes or overlap"""
    base = make()
    x = torch.zeros(4096, dtype=torch.bfloat16).as_strided(base.shape, base.stride(), base.storage_offset())
    y, ptr, ld, copy = g._rows(x)
    assert (y is not x) is contiguous and ptr == y.data_ptr() and ld == y.stride(0) and copy is copied


@pytest.mark.parametrize("shape,stride,contiguous,copied,transposed", [
    ((3, 32, 64), (2048, 64, 1), False, False, False),        # [E, N, K]
    ((3, 64, 32), (2048, 1, 64), False, False, True),         # [E, K, N] seen as [E, N, K]
    ((3, 32, 61), (32 * 61, 61, 1), False, True, False),      # odd rows
    ((3, 61, 32), (61 * 32, 32, 1), False, False, False),     # odd N only
    ((3, 61, 32), (61 * 32, 1, 61), False, True, True),       # odd rows of the transposed storage
    ((3, 32, 64), (0, 64, 1), False, True, False),            # one matrix for all experts
    ((1, 32, 64), (5, 64, 1), False, False, False),           # a single expert's stride is free
    ((3, 32, 64), (2052, 64, 1), False, True, False),         # experts off 16 bytes
    ((3, 32, 64), (4096, 128, 2), True, False, False)])       # contiguous along neither
def test_weight_operands(shape, stride, contiguous, copied, transposed):
    w = torch.zeros(1 << 15, dtype=torch.bfloat16).as_strided(shape, stride)
    v, ptr, ld, plane, tr, copy = g._weights(w)
    assert (v is not w) is contiguous and ptr == v.data_ptr() and plane == v.stride(0)
    assert tr is transposed and copy is copied and ld == (v.stride(2) if tr else v.stride(1))


def test_overlap():
    b = torch.zeros(64, 64)
    g._no_overlap(b[:32], x=b[32:])
    with pytest.raises(ValueError, match="overlaps x"):
        g._no_overlap(b[:33], x=b[32:])
    g._no_overlap(b[:0], x=b)
    g._no_overlap(b[:, :40], x=b[:, 40:])                 # columns side by side in one buffer
    g._no_overlap(b[:, 40:], x=b[3:, :40])
    for out, x in ((b[:, :41], b[:, 40:]), (b[:, 40:], b[:, :41]), (b[:, 20:], b[:, :30]), (b, b[:, :1]), (b[:, 5:9], b)):
        with pytest.raises(ValueError, match="overlaps x"):
            g._no_overlap(out, x=x)
    with pytest.raises(ValueError, match="overlaps x"):   # other strides: by their spans
        g._no_overlap(b.view(-1)[:64 * 32].view(32, 64)[:, :8], x=b.view(-1)[8:8 + 32 * 32].view(32, 32)[:, :8])


def mm(x=A, ldx=64, w=A, ldw=64, sw=64 * 128, tr=0, off=A, y=A, ldy=128, type=BF16, T=16, E=2, N=128, K=64):
    return _lib.lib().spanqr_mm_grouped(x, ldx, w, ldw, sw, tr, off, y, ldy, type, T, E, N, K, 1, None, 0, None)


def wgrad(dy=A, lddy=128, x=A, ldx=64, off=A, dw=A, type=BF16, out=0, T=16, E=2, N=128, K=64):
    return _lib.lib().spanqr_mm_grouped_wgrad(dy, lddy, x, ldx, off, dw, type, out, T, E, N, K, None, 0, None)


def test_argument_checks_before_any_device_work():
    for bad in (dict(T=-1), dict(T=(1 << 30) + 1), dict(E=0), dict(E=1025), dict(N=0), dict(K=0), dict(K=(1 << 24) + 1)):
        assert mm(**bad) == SHAPE, bad
        assert wgrad(**bad) == SHAPE, bad
    for big in (dict(K=(1 << 18) + 1, ldx=1 << 19, ldw=1 << 19), dict(N=(1 << 18) + 1, ldy=1 << 19)):   # sums of products
        assert mm(**big) == SHAPE, big
    for bad in (dict(x=None), dict(x=A + 1), dict(ldx=-64), dict(w=None), dict(w=A + 1), dict(ldw=-64), dict(sw=-8),
                dict(off=None), dict(off=A + 2), dict(y=None), dict(y=A + 1), dict(ldy=127), dict(type=0), dict(type=3)):
        assert mm(**bad) == ARG, bad
    for bad in (dict(dy=None), dict(dy=A + 1), dict(lddy=-8), dict(x=None), dict(ldx=-8), dict(off=None), dict(dw=None),
                dict(dw=A + 2), dict(out=2, dw=A + 1), dict(out=1), dict(out=3), dict(type=0)):
        assert wgrad(**bad) == ARG, bad
    assert mm(T=0) == OK                 # nothing to do
    assert _lib.lib().spanqr_mm_read_status(None, None) == ARG


def test_workspace_bytes():
    L, n = _lib.lib(), ctypes.c_size_t(0)

    def size(fn, *a):
        assert getattr(L, fn)(*a, ctypes.byref(n)) == OK, a
        return n.value
    mm_, wg = "spanqr_mm_grouped_workspace_bytes", "spanqr_mm_grouped_wgrad_workspace_bytes"
    assert size(mm_, 4096, 8, 1024, 1024, 0) == 0 and size(mm_, 0, 8, 1024, 1024, 7) == 0
    assert size(mm_, 64, 1, 768, 17408, 0) > 0                      # few tiles: partial sums
    assert size(wg, 32768, 1, 768, 512, 0) > 0 and size(wg, 4096, 32, 768, 512, 0) == 0
    one, two, tr = (size(mm_, 4096, 8, 1001, 1111, c) for c in (1, 2, 6))
    assert one >= 4096 * 1112 * 2 and two >= 8 * 1001 * 1112 * 2 and tr >= 8 * 1111 * 1008 * 2
    assert size(mm_, 4096, 8, 1001, 1111, 3) == one + two
    assert size(wg, 4096, 32, 1001, 1111, 3) >= 4096 * (1008 + 1112) * 2
    for fn, bad in ((mm_, 8), (mm_, -1), (wg, 4)):
        assert getattr(L, fn)(16, 2, 64, 64, bad, ctypes.byref(n)) == ARG
    assert L.spanqr_mm_grouped_workspace_bytes(16, 0, 64, 64, 0, ctypes.byref(n)) == SHAPE
    assert L.spanqr_mm_grouped_workspace_bytes(16, 1, 64, 64, 0, None) == ARG


def negated(*shape):
    """fp16 values 1, 2, ... as the imaginary part of a conjugate: the memory holds their negatives, two elements apart"""
    z = torch.zeros(shape, dtype=torch.complex32)
    z.imag.copy_(-torch.arange(1.0, z.numel() + 1).view(shape))
    return z.conj().imag


def test_lazily_negated_operands_are_resolved():
    """one column of such a view needs no copy for its strides"""
    for make in (lambda: negated(5, 1), lambda: negated(1, 1), lambda: negated(5, 3)):
        x = make()
        assert x.is_neg()
        y, ptr, _, _ = g._rows(x)
        assert not y.is_neg() and ptr == y.data_ptr() and torch.equal(y.float(), torch.arange(1.0, x.numel() + 1).view(x.shape))
    for shape in ((2, 3, 1), (2, 1, 3), (2, 3, 4), (1, 1, 1)):
        w = negated(*shape)
        v, ptr = g._weights(w)[:2]
        assert not v.is_neg() and ptr == v.data_ptr() and torch.equal(v.float(), torch.arange(1.0, w.numel() + 1).view(shape))
    with pytest.raises(ValueError, match="lazily negated"):
        g._check_out(negated(5, 1), x=torch.zeros(5, 1))


def test_what_autograd_follows():
    from torch.autograd import forward_ad
    x, r = torch.zeros(3), torch.zeros(3, requires_grad=True)
    assert not g._tracked(x, x) and g._tracked(x, r)
    with torch.no_grad():
        assert not g._tracked(x, r)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones(3))
        assert g._tracked(d, x) and g._tracked(x, d) and not g._tracked(x, x)
        with torch.no_grad():
            assert g._tracked(x, d)                       # tangents pass through no_grad


def test_sizes_beyond_32_bits_are_refused():
    """an int argument of the library keeps the low 32 bits alone: 2^32 + 5 rows would be 5"""
    assert _lib._I(2 ** 32 + 5).value == 5
    one, off = torch.zeros(1, 1).bfloat16(), torch.zeros(1, dtype=torch.int32)
    long, wide = one.expand(2 ** 32 + 5, 1), one.expand(1, 2 ** 32 + 5)
    w = one[None]
    for call in (lambda: mm_grouped(long, w, off), lambda: mm_grouped(wide, w, off), lambda: mm_grouped_wgrad(long, long, off),
                 lambda: g._check_rows(wide, "x"), lambda: mm_grouped_wgrad(wide, one, off),
                 lambda: g._check_sizes("w", 1, 2 ** 32 + 8, 1)):
        with pytest.raises(_lib.SpanqrError, match="unsupported shape") as e:
            call()
        assert e.value.code == SHAPE
    g._check_sizes("w", 1024, 2 ** 31 - 1, 1)


def test_an_output_that_autograd_follows_is_refused():
    """written over, it would still hand its gradient to what it held before"""
    leaf = torch.zeros(4, 8, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(RuntimeError, match="out requires a gradient"):
            g._check_out(out)
        g._check_out(out.detach())
        with torch.no_grad():
            g._check_out(out)


def test_selftest_argument_checks():
    for limit in (0, -1, 10 ** 8 + 1):
        assert _lib.lib().spanqr_mm_selftest_timeout(limit, 0, None) == ARG


@pytest.mark.parametrize("device,index", [(None, 1), ("cuda", 1), ("cuda:3", 3), (2, 2), (torch.device("cuda", 0), 0)])
def test_check_raises_what_the_device_reports(monkeypatch, device, index):
    """of the device that is asked for, on its current stream; nothing when there is nothing to report"""
    state = {"current": 1}

    class Device:
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            self.was, state["current"] = state["current"], self.i

        def __exit__(self, *a):
            state["current"] = self.was

    class Library:
        rc, word, seen = OK, 0, None

        def spanqr_mm_read_status(self, stream, out):
            Library.seen = state["current"], stream
            out._obj.value = self.word
            return self.rc

        def spanqr_strerror(self, code):
            return b"device reported a failure"
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(_lib, "lib", Library)
    assert mm_check(device) is None
    assert Library.seen == (index, 100 + index) and state["current"] == 1
    Library.rc, Library.word = 5, 0x100
    with pytest.raises(_lib.SpanqrError, match=f"cuda:{index}.*wait ran out .status 0x100.*reported a failure") as e:
        mm_check(device)
    assert e.value.code == 5 and state["current"] == 1
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        mm_check(device)


def test_check_refuses_other_devices():
    with pytest.raises(ValueError, match="CUDA device"):
        mm_check("cpu")
