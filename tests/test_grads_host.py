"""grad_norm and clip_grads without a GPU: the Python layer's refusals and the C ABI's argument checks, which come before
any device work."""
import ctypes
from array import array

import pytest
import torch

from spanqr_b200 import _lib, clip_grads, grad_norm
from spanqr_b200.grads import _dense, _signs

OK, ARG, WS, OVERLAP = 0, 2, 3, 7
BASE = 1 << 40          # device addresses that no call below dereferences: each fails its checks first


def test_refusals():
    cpu = torch.zeros(4)
    with pytest.raises(TypeError, match="list of tensors"):
        grad_norm(cpu)
    with pytest.raises(TypeError, match="tensors only"):
        grad_norm([1.0])
    with pytest.raises(TypeError, match="CUDA"):
        grad_norm([cpu])
    with pytest.raises(TypeError, match="float64"):
        grad_norm([cpu.double()])
    with pytest.raises(TypeError, match="CUDA"):
        clip_grads([cpu], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grads([], bad)
    with pytest.raises(TypeError, match="number"):
        clip_grads([], torch.tensor(1.0))


@pytest.mark.parametrize("make,want", [
    (lambda: torch.zeros(4, 6), True), (lambda: torch.zeros(4, 6).t(), True), (lambda: torch.zeros(4, 6)[:, :3], False),
    (lambda: torch.zeros(4, 1, 6).permute(2, 1, 0), True), (lambda: torch.zeros(4, 1).expand(4, 3), False),
    (lambda: torch.zeros(4, 6)[::2], False), (lambda: torch.zeros(()), True), (lambda: torch.zeros(7)[2:3], True)])
def test_dense(make, want):
    assert _dense(make()) is want


def test_workspace_bytes():
    n = ctypes.c_size_t(0)
    L = _lib.lib()
    assert L.spanqr_grad_workspace_bytes(-1, ctypes.byref(n)) == ARG
    assert L.spanqr_grad_workspace_bytes(1, None) == ARG
    last = 0
    for count in (0, 1, 64, 65, 900, 901, 5000):
        assert L.spanqr_grad_workspace_bytes(count, ctypes.byref(n)) == OK
        assert n.value >= max(last, 256)
        last = n.value


def _at(a):
    return a.buffer_info()[0]


def _clip(ins, outs, kinds=None, okinds=None, sizes=None, max_norm=1.0, ws=BASE, ws_bytes=1 << 30, norm=BASE):
    n = len(ins)
    pi, po = array("Q", ins), array("Q", outs)
    ki = array("i", kinds or [0] * n)
    ko = array("i", okinds or list(ki))
    sz = array("q", sizes or [64] * n)
    return _lib.lib().spanqr_grad_clip(_at(pi), _at(ki), _at(po), _at(ko), _at(sz), n, max_norm, None, norm, ws, ws_bytes,
                                       None)


def test_clip_argument_checks_before_any_device_work():
    a, b, c = BASE, BASE + 4096, BASE + 8192
    assert _clip([a], [a], kinds=[3]) == ARG                       # no such type
    assert _clip([a], [b], kinds=[0], okinds=[1]) == ARG           # fp32 to fp16
    assert _clip([a], [b], kinds=[1], okinds=[2]) == ARG           # fp16 to bf16
    assert _clip([a + 2], [b]) == ARG                              # fp32 off its alignment
    assert _clip([a], [b + 1], kinds=[1]) == ARG
    assert _clip([0], [b]) == ARG
    assert _clip([a], [0]) == ARG
    assert _clip([a], [b], sizes=[-1]) == ARG
    assert _clip([a], [b], max_norm=-1.0) == ARG
    assert _clip([a], [b], max_norm=float("nan")) == ARG
    assert _clip([a], [b], norm=BASE + 2) == ARG
    assert _clip([a], [b], ws=BASE + 16) == WS
    assert _clip([a], [b], ws=None) == WS
    assert _clip([a], [b], ws_bytes=256) == WS
    # overlaps: 64 fp32 elements are 256 bytes
    assert _clip([a, a], [a, a]) == OVERLAP                        # one tensor twice, in place
    assert _clip([a, c], [b, b]) == OVERLAP                        # two inputs to one output
    assert _clip([a], [a + 128]) == OVERLAP                        # shifted against its own input
    assert _clip([a, b], [b, c]) == OVERLAP                        # an output on another input
    assert _clip([a, b], [c, a]) == OVERLAP
    assert _clip([a], [a], kinds=[1], okinds=[0]) == OVERLAP       # fp16 widened in place
    # overlapping inputs alone are no race: the call gets as far as its workspace
    assert _clip([a, a + 128], [b, c], ws=None) == WS


def test_norm_argument_checks_before_any_device_work():
    L = _lib.lib()
    p, k, n = array("Q", [BASE]), array("i", [0]), array("q", [64])
    assert L.spanqr_grad_norm(_at(p), _at(k), _at(n), 1, None, None, BASE, 1 << 30, None) == ARG     # no result wanted
    assert L.spanqr_grad_norm(_at(p), _at(k), _at(n), -1, None, BASE, BASE, 1 << 30, None) == ARG
    assert L.spanqr_grad_norm(None, _at(k), _at(n), 1, None, BASE, BASE, 1 << 30, None) == ARG
    assert L.spanqr_grad_norm(_at(p), _at(k), _at(n), 1, BASE + 4, BASE, BASE, 1 << 30, None) == ARG  # fp64 off 8 bytes
    assert L.spanqr_grad_norm(_at(p), _at(k), _at(n), 1, None, BASE, BASE, 64, None) == WS


@pytest.mark.parametrize("current,index", [(0, 0), (0, 3), (2, 1)])
def test_a_launch_is_on_the_tensors_device_and_its_stream(monkeypatch, current, index):
    """with the tensors' device current (entered only where it is not), on that device's current stream"""
    state = {"current": current}

    class Device:
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            self.was, state["current"] = state["current"], self.i

        def __exit__(self, *a):
            state["current"] = self.was

    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    calls = []

    def fn(*args):
        calls.append((state["current"], args))
        return args[0]
    _lib.launch(index, fn, lambda: "never asked", 0, "x")
    assert calls == [(index, (0, "x", 100 + index))] and state["current"] == current
    with pytest.raises(_lib.SpanqrError, match="the call"):
        _lib.launch(index, fn, lambda: "the call", 2)
    assert state["current"] == current


def test_lazily_negated_tensors_keep_their_sign():
    """the imaginary part of a conjugate holds its values negated: one element of it has no gaps and passes as contiguous"""
    z = torch.tensor([3.0 + 4.0j]).conj().imag
    plain, two = torch.tensor([7.0]), torch.zeros(2)
    assert z.is_neg() and z.is_contiguous() and z.item() == -4.0
    strided = torch.tensor([1.0 + 2.0j, 3.0 + 4.0j]).conj().imag.as_strided((3,), (1,), 1)    # without gaps, of any length
    assert strided.is_neg() and strided.is_contiguous() and strided.tolist() == [-2.0, -3.0, -4.0]
    ins, types = [two, z, plain, strided], array("i", [0] * 4)
    got = _signs(ins, types, [torch.empty_like(t) for t in ins], types)
    assert not got[1].is_neg() and got[1].item() == -4.0 and got[0] is two and got[2] is plain and ins[1] is z
    assert not got[3].is_neg() and got[3].tolist() == [-2.0, -3.0, -4.0]
    one = types[:1]
    assert _signs([z], one, [z], one)[0] is z                    # two of them: scaled as they lie
    with pytest.raises(ValueError, match=r"out\[0\] is a lazily negated"):
        _signs([plain], one, [z], one)
    with pytest.raises(ValueError, match=r"out\[1\] is a lazily negated"):
        _signs([two.bfloat16(), two.bfloat16()], array("i", [2, 2]), [two, strided], types[:2])


# ---- group=: gloo ranks on CPU, the library's two entry points replaced by the formulas over the same pointers ----

def _fake_library(monkeypatch):
    """grads on CPU tensors of fp32: what it hands to the library is read from and written to their memory"""
    import contextlib

    import numpy as np
    from spanqr_b200 import grads
    real = _lib.lib()

    def view(address, ctype, n):
        return np.frombuffer((ctype * n).from_address(address), dtype=ctype) if n else np.zeros(0)

    def launch(index, fn, what, *args):
        clip = fn == real.spanqr_grad_clip
        ptrs, types, *rest = args
        if clip:
            outs, out_types, sizes, count, max_norm, sumsq, norm, ws, _ = rest
        else:
            sizes, count, sumsq, norm, ws, _ = rest
        assert ws and (not count or set(view(types, ctypes.c_int32, count)) == {0})
        ns = view(sizes, ctypes.c_longlong, count)
        ins = [view(int(p), ctypes.c_float, int(n)) for p, n in zip(view(ptrs, ctypes.c_ulonglong, count), ns)]
        total = sum(float((x.astype(np.float64) ** 2).sum()) for x in ins)
        if clip:
            if sumsq:
                total = float(view(sumsq, ctypes.c_double, 1)[0])
            c = min(1.0, max_norm / (total ** 0.5 + 1e-6)) if total == total else total
            for x, p, n in zip(ins, view(outs, ctypes.c_ulonglong, count), ns):
                view(int(p), ctypes.c_float, int(n))[:] = x * c
        elif sumsq:
            view(sumsq, ctypes.c_double, 1)[0] = total
        if norm:
            view(norm, ctypes.c_float, 1)[0] = total ** 0.5
    monkeypatch.setattr(_lib, "launch", launch)
    monkeypatch.setattr(grads, "_device", lambda t: torch.device("cpu"))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: torch.device("cpu"))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())


def _rank(rank, port, work):
    from datetime import timedelta

    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=3,
                            timeout=timedelta(seconds=20))
    try:
        with pytest.MonkeyPatch.context() as m:
            _fake_library(m)
            work(rank, dist)
    finally:
        dist.destroy_process_group()


def _ranks(work):
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as free:
        free.bind(("127.0.0.1", 0))
        port = free.getsockname()[1]
    mp.spawn(_rank, args=(port, work), nprocs=3, join=True)


def _refusals_of_one_rank(rank, dist):
    world = dist.group.WORLD
    good, bad = [torch.tensor([3.0, 4.0])], [torch.zeros(4, dtype=torch.float64)]
    for call, error in ((lambda ts: grad_norm(ts, group=world), TypeError),
                        (lambda ts: clip_grads(ts, 1.0, group=world)[1], TypeError),
                        (lambda ts: clip_grads(ts, 1.0, out=good + bad if ts is bad else None, group=world)[1], TypeError),
                        (lambda ts: clip_grads(good, -1.0 if ts is bad else 1.0, group=world)[1], ValueError)):
        if rank == 1:
            with pytest.raises(error):
                call(bad)
        else:
            assert call(good).isnan().item()
        assert abs(grad_norm(good, group=world).item() - 75 ** 0.5) < 1e-5       # the next call of all ranks is right


def test_a_rank_whose_list_is_refused_leaves_no_other_waiting():
    _ranks(_refusals_of_one_rank)


def _norms_of_all_ranks(rank, dist):
    """rank 0 holds two tensors, rank 1 nothing, rank 2 one: 9 + 16 + 144 = 13 squared"""
    world = dist.group.WORLD
    part = [[torch.tensor([3.0]), torch.tensor([[0.0, 4.0]])], [], [torch.tensor([12.0])]][rank]
    for _ in range(2):
        assert grad_norm(part, group=world).item() == 13.0
        own = sum(float((t ** 2).sum()) for t in part) ** 0.5
        assert abs(grad_norm(part).item() - own) < 1e-6              # without the group: this process's own
        ys, n = clip_grads(part, 6.5, group=world)
        assert n.item() == 13.0 and len(ys) == len(part)
        for y, t in zip(ys, part):
            assert torch.allclose(y, t / 2, rtol=1e-6, atol=0)
    pair = dist.new_group([0, 2])                                    # (every rank makes it)
    if rank != 1:
        assert grad_norm(part, group=pair).item() == 13.0
        mine = [t.clone() for t in part]
        _, n = clip_grads(mine, 1.3, out=mine, group=pair)
        assert n.item() == 13.0 and all(torch.allclose(y, t / 10, rtol=1e-6, atol=0) for y, t in zip(mine, part))


def test_norm_and_clipping_over_ranks():
    _ranks(_norms_of_all_ranks)
