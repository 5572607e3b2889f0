"""mm_grouped and mm_grouped_wgrad on the GPU against the definition in fp64.

Most cases use whole numbers of at most 2 in size: their products and sums are exact in fp32 in any order (below 2^24),
so the results must equal the exact ones rounded once, bit for bit.  With Gaussian inputs an element may be off by half a
step of its type, plus what the fp32 sums lose: the tensor core rounds toward zero at each product of 16 elements (at
most 2^-22 of S, the sum of the absolute terms, each time), and mm_grouped_wgrad adds its sums of 512 rows (32 such
additions) to nearest."""
import ctypes
from pathlib import Path

import pytest
import torch

from spanqr_b200 import _lib, SpanqrError, clip_grads, mm_check, mm_grouped, mm_grouped_wgrad, orth_batched

pytestmark = pytest.mark.gpu
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    st = ctypes.c_int(-1)
    assert _lib.lib().spanqr_mm_read_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(st)) == 0


def ints(shape, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-2, 3, shape, device="cuda", generator=g).to(dtype)


def offsets(counts):
    return torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)


def spread(T, E, seed=0):
    """T rows over E experts, unevenly, some without any"""
    g = torch.Generator().manual_seed(seed + 17 * E + T)
    share = torch.softmax(2.0 * torch.randn(E, generator=g), 0)
    return torch.bincount(torch.multinomial(share, T, replacement=True, generator=g), minlength=E).tolist() if T else [0] * E


def rows_of(off, T):
    a = 0
    for e, b in enumerate(off.tolist()):
        b = min(max(b, a), T)
        yield e, a, b
        a = b


def exact_mm(x, w, off):
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    for e, a, b in rows_of(off, x.shape[0]):
        y[a:b] = x[a:b].double() @ w[e].double().t()
    return y


def exact_wgrad(dy, x, off):
    dw = torch.zeros(off.shape[0], dy.shape[1], x.shape[1], dtype=torch.float64, device="cuda")
    for e, a, b in rows_of(off, x.shape[0]):
        dw[e] = dy[a:b].double().t() @ x[a:b].double()
    return dw


SHAPES = [   # T, E, N, K: one row, one tile and its edges, odd sides, many experts, both sides of every variant's border
    (1, 1, 1, 1), (1, 1, 128, 64), (2, 3, 8, 16), (16, 1, 128, 64), (17, 1, 129, 72), (33, 2, 136, 200), (5, 2, 100, 37),
    (31, 1, 256, 4096), (64, 4, 384, 1000), (65, 4, 130, 320), (100, 3, 257, 65), (200, 128, 64, 128), (7, 1024, 40, 24),
    (129, 2, 256, 64), (257, 1, 264, 128), (300, 2, 500, 77), (511, 5, 768, 512), (1000, 7, 250, 1111), (2049, 4, 1001, 640),
    (4096, 16, 512, 256)]


@pytest.mark.parametrize("T,E,N,K", SHAPES)
@pytest.mark.parametrize("dtype,transposed", [(BF16, False), (FP16, True)])
def test_product_exact(T, E, N, K, dtype, transposed):
    x = ints((T, K), T, dtype)
    w = ints((E, K, N), K, dtype).transpose(1, 2) if transposed else ints((E, N, K), K, dtype)
    off = offsets(spread(T, E))
    assert torch.equal(mm_grouped(x, w, off), exact_mm(x, w, off).to(dtype))


@pytest.mark.parametrize("T,E,N,K", SHAPES)
@pytest.mark.parametrize("dtype,out", [(BF16, F32), (FP16, FP16)])
def test_wgrad_exact(T, E, N, K, dtype, out):
    dy, x = ints((T, N), T, dtype), ints((T, K), T + 1, dtype)
    off = offsets(spread(T, E, 1))
    assert torch.equal(mm_grouped_wgrad(dy, x, off, dtype=out), exact_wgrad(dy, x, off).to(out))


@pytest.mark.parametrize("T,E,N,K", [(6000, 300, 64, 64), (12000, 600, 40, 72), (20000, 1024, 64, 256), (9000, 150, 300, 520)])
def test_many_small_ragged_experts(T, E, N, K):
    """one CTA pair after another takes experts whose few rows end inside a product's 16: its two CTAs run apart by
    several such tiles"""
    dy, x, w = ints((T, N), 1, BF16), ints((T, K), 2, BF16), ints((E, N, K), 3, BF16)
    g = torch.Generator().manual_seed(T)
    off = offsets(torch.bincount(torch.randint(0, E, (T,), generator=g), minlength=E).tolist())
    for _ in range(3):
        assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy, x, off).to(F32))
    assert torch.equal(mm_grouped(x, w, off), exact_mm(x, w, off).to(BF16))


@pytest.mark.parametrize("T,E,N,K", [(64, 1, 768, 17408), (1, 1, 300, 9000), (33, 2, 100, 8192), (200, 3, 260, 5001),
                                     (5, 1, 4096, 4096)])
def test_few_tiles_split_over_the_contracted_dimension(T, E, N, K):
    x, w = ints((T, K), T, BF16), ints((E, N, K), K, BF16)
    off = offsets(spread(T, E))
    want = exact_mm(x, w, off).to(BF16)
    for _ in range(2):
        assert torch.equal(mm_grouped(x, w, off), want)


@pytest.mark.parametrize("T,E,N,K", [(20000, 1, 300, 77), (30000, 2, 256, 512), (9000, 3, 41, 260), (16385, 1, 768, 500)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_tiles_split_over_the_rows(T, E, N, K, dtype):
    dy, x = ints((T, N), T, BF16), ints((T, K), K, BF16)
    for counts in (spread(T, E), [T] + [0] * (E - 1)):
        off = offsets(counts)
        assert torch.equal(mm_grouped_wgrad(dy, x, off, dtype=dtype), exact_wgrad(dy, x, off).to(dtype))


@pytest.mark.parametrize("N,K", [(2048, 2048), (2048, 1999), (2040, 2056)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_wgrad_in_16_bits_over_several_drains(N, K, dtype):
    """experts of more rows than are summed in one accumulator (2048), too many tiles to split the rows: the accumulators are
    taken in turn several times within a tile, at whole and ragged ends, and stored in both ways"""
    counts = [7001, 2049, 0, 4101, 2048, 4096]
    T, off = sum(counts), offsets(counts)
    dy, x = ints((T, N), 1, dtype), ints((T, K), 2, dtype)
    want = exact_wgrad(dy, x, off).to(dtype)
    assert torch.equal(mm_grouped_wgrad(dy, x, off, dtype=dtype), want)
    assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy, x, off).to(F32))
    w = ints((len(counts), N, K), 3, dtype).requires_grad_()
    dw, = torch.autograd.grad(mm_grouped(x, w, off), w, dy)
    assert torch.equal(dw, want)


@pytest.mark.parametrize("T,E,N,K", [(24, 8, 512, 2048), (700, 16, 384, 1024), (3000, 4, 640, 4096), (5000, 3, 256, 17408)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_product_gaussian(T, E, N, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, K, device="cuda", generator=g).to(dtype)
    w = (torch.randn(E, N, K, device="cuda", generator=g) / K ** 0.5).to(dtype)
    off = offsets(spread(T, E))
    want, S = exact_mm(x, w, off), exact_mm(x.abs(), w.abs(), off)
    tol = want.abs() * torch.finfo(dtype).eps / 2 * 1.001 + S * (K / 16 + 4) * 2.0 ** -22 + torch.finfo(dtype).tiny
    assert bool(((mm_grouped(x, w, off).double() - want).abs() <= tol).all())


@pytest.mark.parametrize("T,E,N,K", [(1000, 4, 300, 200), (30000, 2, 256, 512), (4000, 64, 128, 256)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_wgrad_gaussian(T, E, N, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(T)
    dy, x = (torch.randn(T, n, device="cuda", generator=g).abs().to(dtype) for n in (N, K))   # all terms positive
    off = offsets(spread(T, E))
    want = exact_wgrad(dy, x, off)
    most = max(b - a for _, a, b in rows_of(off, T))
    tol = want * (32 * 2.0 ** -22 + (most / 512 + 2) * 2.0 ** -24)
    assert bool(((mm_grouped_wgrad(dy, x, off).double() - want).abs() <= tol).all())


@pytest.mark.parametrize("T", [1000, 20000, 100000])
def test_wgrad_does_not_drift_with_the_rows(T):
    """sums of random sign: the tensor core's rounding toward zero stays that of 512 rows (32 additions of at most half a
    unit of 2^-23 on average, 32 * 2^-24 = 1.9e-6 of the result at the most), the sums of those are to nearest"""
    g = torch.Generator(device="cuda").manual_seed(T)
    x, dy = (torch.randn(T, n, device="cuda", generator=g).to(BF16) for n in (256, 512))
    off = offsets([T // 3, T - T // 3])
    want, got = exact_wgrad(dy, x, off), mm_grouped_wgrad(dy, x, off).double()
    assert float((got - want).norm() / want.norm()) <= 2e-6
    assert abs(float(((got - want) * want.sign()).sum() / want.abs().sum())) <= 2e-6


def test_product_over_a_long_contracted_dimension():
    g = torch.Generator(device="cuda").manual_seed(3)
    K = 1 << 18
    x, w = torch.randn(40, K, device="cuda", generator=g).to(BF16), torch.randn(1, 64, K, device="cuda", generator=g).to(BF16)
    off = offsets([40])
    want = exact_mm(x, w, off)
    err = (mm_grouped(x, w, off).double() - want).norm() / want.norm()
    assert float(err) <= 2.0 ** -8 + K / 16 * 2.0 ** -24          # half a step, and the additions toward zero


@pytest.mark.parametrize("counts", [[0, 0, 40], [40, 0, 0], [0, 40, 0], [13, 14, 13], [0, 0, 0], [1, 0, 1]])
@pytest.mark.parametrize("scale", [1, 20])
def test_uneven_experts(counts, scale):
    counts = [c * scale for c in counts]
    T = sum(counts)
    x, w, dy = ints((T, 96), 1, BF16), ints((3, 200, 96), 2, BF16), ints((T, 200), 3, BF16)
    off = offsets(counts)
    assert torch.equal(mm_grouped(x, w, off), exact_mm(x, w, off).to(BF16))
    assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy, x, off).to(F32))


@pytest.mark.parametrize("N", [136, 8, 2051])
def test_padded_batch(N):
    """a batch padded far behind its last row"""
    x, w = ints((5000, 64), 1, BF16), ints((2, N, 64), 2, BF16)
    off = torch.tensor([7, 100], dtype=torch.int32, device="cuda")
    y = mm_grouped(x, w, off)
    assert torch.equal(y, exact_mm(x, w, off).to(BF16))


@pytest.mark.parametrize("T,end", [(50, 33), (50, 0), (700, 450), (700, 0)])
def test_rows_behind_the_last_expert(T, end):
    """zero in a new result, untouched in a given one; infinities and NaN there reach nothing"""
    x, w, dy = ints((T, 64), 1, BF16), ints((2, 136, 64), 2, BF16), ints((T, 136), 3, BF16)
    x[end:], dy[end:] = float("nan"), float("inf")
    off = torch.tensor([end // 3, end], dtype=torch.int32, device="cuda")
    want = exact_mm(x[:end], w, off).to(BF16)
    y = mm_grouped(x, w, off)
    assert torch.equal(y[:end], want) and bool((y[end:] == 0).all())
    out = torch.full((T, 136), 7.0, dtype=BF16, device="cuda")
    assert mm_grouped(x, w, off, out=out) is out
    assert torch.equal(out[:end], want) and bool((out[end:] == 7).all())
    assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy[:end], x[:end], off).to(F32))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(mm_grouped(xg, wg, off), (xg, wg), dy)
    assert bool((dx[end:] == 0).all()) and bool(dw.isfinite().all())


@pytest.mark.parametrize("T", [40, 900])
def test_nan_rows_stay_in_their_expert(T):
    x, w, dy = ints((T, 64), 1, FP16), ints((3, 128, 64), 2, FP16), ints((T, 128), 3, FP16)
    a, b = T // 3 + 1, T // 2 + 3
    x[a:b], dy[a:b] = float("nan"), float("-inf")
    off = torch.tensor([a, b, T], dtype=torch.int32, device="cuda")
    y, dw = mm_grouped(x, w, off), mm_grouped_wgrad(dy, x, off)
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[a:b] = False
    clean, dclean = x.clone(), dy.clone()
    clean[a:b], dclean[a:b] = 0, 0
    assert torch.equal(y[keep], exact_mm(clean, w, off)[keep].to(FP16)) and bool(y[a:b].isnan().all())
    want = exact_wgrad(dclean, clean, off)
    assert torch.equal(dw[0], want[0].float()) and torch.equal(dw[2], want[2].float()) and bool(dw[1].isnan().all())


@pytest.mark.parametrize("ends", [[30, 10, 50], [-5, 20, 60], [100, 100, 100], [0, -3, 10 ** 9]])
def test_ends_out_of_order_or_range_are_clamped(ends):
    T = 50
    x, w, dy = ints((T, 64), 1, BF16), ints((3, 128, 64), 2, BF16), ints((T, 128), 3, BF16)
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    assert torch.equal(mm_grouped(x, w, off), exact_mm(x, w, off).to(BF16))
    assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy, x, off).to(F32))


@pytest.mark.parametrize("T", [30, 600])
def test_strides_and_alignment(T):
    N, K, E = 136, 88, 2
    off = offsets([T // 3, T - T // 3])
    big, wbig = ints((T, 2, 256), 1, BF16), ints((E, 256, 256), 2, BF16)
    xs = [big[:, 0, :K], big[:, 1, 8:8 + K], big[:, 0, 3:3 + K], ints((K, T), 4, BF16).t(), ints((1, K), 5, BF16).expand(T, K),
          ints((2 * T, K), 6, BF16)[::2]]
    ws = [wbig[:, :N, :K], wbig[:, 8:8 + N, 16:16 + K], wbig[:, 1:1 + N, 5:5 + K], wbig.transpose(1, 2)[:, :N, :K],
          wbig[:1, :N, :K].expand(E, N, K), wbig[:, ::2][:, :100, :K], wbig[:, :, ::2][:, :N, :K]]
    for x in xs:
        assert torch.equal(mm_grouped(x, ws[0], off), exact_mm(x, ws[0], off).to(BF16))
        assert torch.equal(mm_grouped_wgrad(big[:, 1, 1:1 + N], x, off), exact_wgrad(big[:, 1, 1:1 + N], x, off).to(F32))
    for w in ws:
        assert torch.equal(mm_grouped(xs[0], w, off), exact_mm(xs[0], w, off).to(BF16))


@pytest.mark.parametrize("T", [30, 600])
@pytest.mark.parametrize("ld,at", [(136, 0), (144, 8), (145, 1), (301, 5)])
def test_given_output_rows(T, ld, at):
    N = 135
    x, w = ints((T, 64), 1, FP16), ints((2, N, 64), 2, FP16)
    off = offsets([T // 2, T - T // 2])
    buf = torch.full((T, ld), 9.0, dtype=FP16, device="cuda")
    out = buf[:, at:at + N]
    mm_grouped(x, w, off, out=out)
    assert torch.equal(out, exact_mm(x, w, off).to(FP16))
    assert bool((buf[:, :at] == 9).all()) and bool((buf[:, at + N:] == 9).all())


@pytest.mark.parametrize("at", [0, 1, 2, 3, 5, 7, 8])
@pytest.mark.parametrize("K,extra", [(1, 0), (7, 0), (61, 0), (64, 1), (100, 3), (777, 0)])
def test_operands_at_every_alignment(at, K, extra):
    """x, w and dy up to the last element of their allocation, NaN between their rows"""
    T, E, N = 37, 2, 19

    def operand(planes, rows, cols, seed):
        ld = cols + extra
        flat = torch.full((at + (planes * rows - 1) * ld + cols,), float("nan"), dtype=FP16, device="cuda")
        t = flat.as_strided((planes, rows, cols), (rows * ld, ld, 1), at)
        t.copy_(ints((planes, rows, cols), seed, FP16))
        return t
    x, w, dy, wt = operand(1, T, K, 1)[0], operand(E, N, K, 2), operand(1, T, N, 3)[0], operand(E, K, N, 4).transpose(1, 2)
    off = offsets([20, 17])
    for v in (w, wt):
        assert torch.equal(mm_grouped(x, v, off), exact_mm(x, v, off).to(FP16))
    assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy, x, off).to(F32))


def test_operand_and_output_side_by_side_in_one_buffer():
    T, K, N = 300, 72, 136
    buf = torch.full((T, K + N + 8), 3.0, dtype=BF16, device="cuda")
    x, out = buf[:, :K], buf[:, K:K + N]
    x.copy_(ints((T, K), 1, BF16))
    w, off = ints((2, N, K), 2, BF16), offsets([100, 200])
    x0 = x.clone()
    mm_grouped(x, w, off, out=out)
    assert torch.equal(out, exact_mm(x0, w, off).to(BF16)) and torch.equal(x, x0) and bool((buf[:, K + N:] == 3).all())


def test_inference_mode():
    with torch.inference_mode():
        x, w, off = ints((90, 64), 1, BF16), ints((2, 72, 64), 2, BF16), offsets([40, 50])
        out = torch.empty(90, 72, dtype=BF16, device="cuda")
        want = exact_mm(x, w, off).to(BF16)
        assert torch.equal(mm_grouped(x, w, off), want) and torch.equal(mm_grouped(x, w, off, out=out), want)
        dw = mm_grouped_wgrad(out, x, off)
        assert torch.equal(dw, exact_wgrad(out, x, off).to(F32))
        n0 = float(dw.double().norm())
        _, n = clip_grads([dw], 1.0, out=[dw])
        assert abs(n.item() - n0) <= 1e-6 * n0 and abs(float(dw.double().norm()) - 1.0) <= 1e-6


def test_wgrad_into_given_output():
    dy, x = ints((200, 72), 1, BF16), ints((200, 136), 2, BF16)
    off = offsets([90, 110])
    want = exact_wgrad(dy, x, off)
    for dt in (F32, BF16):
        buf = torch.full((2 * 72 * 136 + 3,), 5.0, dtype=dt, device="cuda")
        out = buf[1:-2].view(2, 72, 136)
        assert mm_grouped_wgrad(dy, x, off, out=out) is out
        assert torch.equal(out, want.to(dt)) and buf[0] == 5 and bool((buf[-2:] == 5).all())


def test_no_rows_at_all():
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    x, w = ints((0, 64), 1, BF16).requires_grad_(), ints((3, 128, 64), 2, BF16).requires_grad_()
    y = mm_grouped(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 128) and dx.shape == (0, 64) and bool((dw == 0).all())
    assert bool((mm_grouped_wgrad(y.detach(), x, off) == 0).all())


@pytest.mark.parametrize("T,E,N,K", [(40, 3, 72, 104), (900, 4, 200, 96), (333, 2, 75, 41)])
def test_gradients_against_formula_and_differences(T, E, N, K):
    """whole numbers: the loss is exact, so differences of it equal the gradients' products exactly"""
    x, w, dy = ints((T, K), 1, FP16).requires_grad_(), ints((E, N, K), 2, FP16).requires_grad_(), ints((T, N), 3, FP16)
    off = offsets(spread(T, E, 3))
    y = mm_grouped(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dx, exact_mm(dy, w.detach().transpose(1, 2), off).to(FP16))
    assert torch.equal(dw, exact_wgrad(dy, x.detach(), off).to(FP16))
    loss = lambda xx, ww: float((mm_grouped(xx, ww, off).double() * dy.double()).sum())   # noqa: E731
    vx, vw = ints((T, K), 4, FP16), ints((E, N, K), 5, FP16)
    with torch.no_grad():
        assert loss(x + vx, w) - loss(x - vx, w) == 2 * float((dx.double() * vx.double()).sum())
        assert loss(x, w + vw) - loss(x, w - vw) == 2 * float((dw.double() * vw.double()).sum())


def test_gradients_of_shared_and_partial_inputs():
    x, w1, dy = ints((60, 64), 1, BF16), ints((1, 72, 64), 2, BF16).requires_grad_(), ints((60, 72), 3, BF16)
    off = offsets([20, 25, 15])
    mm_grouped(x, w1.expand(3, 72, 64), off).backward(dy)          # one matrix for all experts: their gradients' sum
    parts = exact_wgrad(dy, x, off).to(BF16).double()
    assert float((w1.grad[0].double() - parts.sum(0)).abs().max()) <= 2 * 2.0 ** -8 * float(parts.abs().sum(0).max())
    xg = x.clone().requires_grad_()
    mm_grouped(xg, w1.detach().expand(3, 72, 64), off).sum().backward()   # only x; a broadcast dy
    assert torch.equal(xg.grad, exact_mm(torch.ones_like(dy), w1.detach().expand(3, 72, 64).transpose(1, 2), off).to(BF16))
    with pytest.raises(RuntimeError):
        gx, = torch.autograd.grad(mm_grouped(xg, w1.expand(3, 72, 64), off).sum(), xg, create_graph=True)
        gx.sum().backward()


def test_refusals():
    x, w, off = ints((8, 16), 1, BF16), ints((2, 24, 16), 2, BF16), offsets([4, 4])
    for bad, err, msg in [((x.float(), w.float(), off), TypeError, "bf16 or fp16"), ((x, w.half(), off), TypeError, "as x"),
                          ((x, w[:, :, :8], off), ValueError, "3-D"), ((x, w, off.long()), TypeError, "int32"),
                          ((x, w, off[:1]), ValueError, "one end"), ((x, w, off.cpu()), TypeError, "int32 on")]:
        with pytest.raises(err, match=msg):
            mm_grouped(*bad)
    out = torch.empty(8, 24, dtype=BF16, device="cuda")
    for bad, err, msg in [(out[:4], ValueError, "shape"), (out.half(), TypeError, "must be"),
                          (torch.empty(24, 8, dtype=BF16, device="cuda").t(), ValueError, "contiguous rows"),
                          (out[:1].expand(8, 24), ValueError, "contiguous rows")]:
        with pytest.raises(err, match=msg):
            mm_grouped(x, w, off, out=bad)
    flat = ints((1000,), 1, BF16)
    with pytest.raises(ValueError, match="overlaps x"):
        mm_grouped(flat[:128].view(8, 16), w, off, out=flat[120:312].view(8, 24))
    with pytest.raises(RuntimeError, match="not differentiable"):
        mm_grouped(x.clone().requires_grad_(), w, off, out=out)
    dy = ints((8, 24), 3, BF16)
    for kw, err, msg in [(dict(dtype=torch.float16), TypeError, "fp32 or"), (dict(out=torch.empty(2, 24, 8, device="cuda")), ValueError, "contiguous with"),
                         (dict(out=torch.empty(2, 24, 16, device="cuda"), dtype=F32), ValueError, "not both"),
                         (dict(out=torch.empty(2, 24, 16, dtype=FP16, device="cuda")), TypeError, "fp32 or")]:
        with pytest.raises(err, match=msg):
            mm_grouped_wgrad(dy, x, off, **kw)
    with pytest.raises(ValueError, match="as many rows"):
        mm_grouped_wgrad(dy[:4], x, off)


def test_fp16_overflow_is_infinite():
    x, w = torch.full((20, 64), 200.0, dtype=FP16, device="cuda"), torch.full((1, 8, 64), 200.0, dtype=FP16, device="cuda")
    off = offsets([20])
    assert bool((mm_grouped(x, w, off) == float("inf")).all())
    assert bool((mm_grouped_wgrad(x, -x, off, dtype=FP16) == float("-inf")).all())
    assert bool((mm_grouped_wgrad(x, -x, off) == -200.0 * 200.0 * 20).all())


@pytest.mark.parametrize("dtype,tiny", [(FP16, 2.0 ** -24), (BF16, 2.0 ** -133)])
def test_subnormal_values(dtype, tiny):
    """whole multiples of the type's smallest value: exact sums, none of them flushed to zero"""
    T, N, K = 70, 40, 64
    x, w, dy = (ints((T, K), 1, F32) * tiny).to(dtype), ints((2, N, K), 2, dtype), ints((T, N), 3, dtype)
    off = offsets([30, 40])
    assert bool((x != 0).any())
    assert torch.equal(mm_grouped(x, w, off), exact_mm(x, w, off).to(dtype))
    assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy, x, off).to(F32))


@pytest.mark.parametrize("T", [48, 2000])
def test_streams_graphs_and_same_bits(T):
    E, N, K = 4, 264, 512
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(T, n, device="cuda", generator=g).to(BF16) for n in (K, N))
    w = torch.randn(E, N, K, device="cuda", generator=g).to(BF16)
    off = offsets(spread(T, E))
    y, dw = mm_grouped(x, w, off), mm_grouped_wgrad(dy, x, off)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ys = [mm_grouped(x, w, off) for _ in range(3)]
    y2, dw2 = mm_grouped(x, w, off), mm_grouped_wgrad(dy, x, off)
    torch.cuda.synchronize()
    assert all(torch.equal(y, t) for t in ys + [y2]) and torch.equal(dw, dw2)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mm_grouped(x, w, off), mm_grouped_wgrad(dy, x, off)
        graphs.append((graph, out))
    half = off.clone()
    off.copy_(torch.tensor([T, T, T, T]))                # the replays read the present offsets
    torch.cuda.synchronize()
    for (graph, _), st in zip(graphs, (s, torch.cuda.current_stream())):
        with torch.cuda.stream(st):
            graph.replay()
    torch.cuda.synchronize()
    y3, dw3 = mm_grouped(x, w, off), mm_grouped_wgrad(dy, x, off)
    for _, (a, b) in graphs:
        assert torch.equal(a, y3) and torch.equal(b, dw3)
    off.copy_(half)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], y) and torch.equal(graphs[0][1][1], dw)


def test_captured_training_step():
    """forward and backward in one captured graph, replayed on new data"""
    T, E, N, K = 300, 3, 136, 128
    x, w, dy = ints((T, K), 1, BF16), ints((E, N, K), 2, BF16).requires_grad_(), ints((T, N), 3, BF16)
    off = offsets(spread(T, E))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw, = torch.autograd.grad(mm_grouped(x, w, off), w, dy)
    x.copy_(ints((T, K), 9, BF16))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dw, exact_wgrad(dy, x, off).to(BF16))


def test_optimizer_step_of_an_expert_layer():
    """rows -> products -> fp32 weight gradients -> clipped -> an orthonormal basis per expert, as one trainer's step"""
    T, E, N, K = 3000, 4, 768, 128
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(T, K, device="cuda", generator=g).to(BF16)
    w = (torch.randn(E, N, K, device="cuda", generator=g) / K ** 0.5).to(BF16)
    off = offsets([1000, 500, 700, 800])
    y = mm_grouped(x, w, off)
    dw = mm_grouped_wgrad(y, x, off)
    grads, norm = clip_grads(list(dw), 1.0)
    assert abs(norm.item() - float(dw.double().norm())) <= 1e-6 * norm.item()
    assert abs(float(torch.stack(grads).double().norm()) - 1.0) <= 2e-6
    for q, d in zip(orth_batched(grads), dw):
        q, d = q.double(), d.double()
        assert float((q.t() @ q - torch.eye(K, device="cuda")).abs().max()) <= 3e-7
        assert float((d - q @ (q.t() @ d)).norm() / d.norm()) <= 1e-5


def test_results_past_two_to_the_31_elements():
    T, N, K = 1_100_003, 2048, 64
    x, w = ints((T, K), 1, BF16), ints((2, N, K), 2, BF16)
    off = torch.tensor([T - 300, T], dtype=torch.int32, device="cuda")
    y = mm_grouped(x, w, off)
    for rows, e in ((slice(0, 300), 0), (slice(T - 700, T - 300), 0), (slice(T - 300, T), 1)):
        assert torch.equal(y[rows], (x[rows].double() @ w[e].double().t()).to(BF16))
    del y
    E, N, K = 1024, 2048, 1104                           # 2.3e9 results of 4 bytes
    dy, x = ints((3000, N), 3, BF16), ints((3000, K), 4, BF16)
    off = torch.zeros(E, dtype=torch.int32, device="cuda")
    off[10:], off[E - 2:], off[E - 1] = 17, 1500, 3000
    dw = mm_grouped_wgrad(dy, x, off)
    for e, a, b in ((10, 0, 17), (E - 2, 17, 1500), (E - 1, 1500, 3000)):
        assert torch.equal(dw[e], (dy[a:b].double().t() @ x[a:b].double()).float())
    assert bool((dw[11:E - 2] == 0).all()) and bool((dw[:10] == 0).all())


def test_offsets_inside_a_larger_tensor():
    x, w = ints((50, 64), 1, BF16), ints((3, 72, 64), 2, BF16)
    ends = torch.tensor([0, 20, 20, 50, 0], dtype=torch.int32, device="cuda")
    want = exact_mm(x, w, ends[1:4]).to(BF16)
    assert torch.equal(mm_grouped(x, w, ends[1:4]), want)
    assert torch.equal(mm_grouped(x, w, ends[1:4].repeat_interleave(2)[::2]), want)


def test_two_streams_at_once():
    """calls in flight together on two streams, with workspaces (split products, copied operands): each its own"""
    ws = [ints((1, 768, 8193), i, BF16) for i in range(2)]
    xs = [ints((40, 8193), 5 + i, BF16) for i in range(2)]
    big = [(ints((9000, 200), 7 + i, BF16), ints((9000, 131), 9 + i, BF16)) for i in range(2)]
    off, boff = offsets([40]), offsets([9000])
    want = [exact_mm(x, w, off).to(BF16) for x, w in zip(xs, ws)]
    bwant = [exact_wgrad(d, x, boff).to(F32) for d, x in big]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((mm_grouped(xs[i], ws[i], off), mm_grouped_wgrad(*big[i], boff)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) and torch.equal(d, bwant[i]) for y, d in got[i])


def test_first_call_of_a_process_inside_a_capture():
    """nothing a first call sets up is refused by a capture"""
    import subprocess
    import sys
    code = """
import torch
from spanqr_b200 import clip_grads, grad_norm, mm_grouped, mm_grouped_wgrad
x = torch.ones(40, 64, dtype=torch.bfloat16, device="cuda")
w = torch.ones(2, 72, 64, dtype=torch.bfloat16, device="cuda")
off = torch.tensor([15, 40], dtype=torch.int32, device="cuda")
g = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    y = mm_grouped(x, w, off)
    dw = mm_grouped_wgrad(y, x, off)
    (c,), n = clip_grads([dw], 1.0)
    m = grad_norm([dw])
g.replay()
torch.cuda.synchronize()
assert bool((y == 64).all()) and bool((dw[0] == 15 * 64).all()) and bool((dw[1] == 25 * 64).all())
assert n.item() == m.item() > 1 and abs(c.norm().item() - 1) < 1e-5
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)


def test_lazily_negated_operands():
    """fp16 imaginary parts of conjugates, whose memory holds the values negated: one column of them has usable strides"""
    def negated(t):
        z = torch.zeros(t.shape, dtype=torch.complex32, device="cuda")
        z.imag.copy_(-t)
        assert z.conj().imag.is_neg()
        return z.conj().imag
    off = offsets([20, 17])
    for N, K in ((24, 1), (1, 24), (24, 40), (1, 1)):
        x, w, dy = ints((37, K), 1, FP16), ints((2, N, K), 2, FP16), ints((37, N), 3, FP16)
        want, dwant = exact_mm(x, w, off).to(FP16), exact_wgrad(dy, x, off).to(F32)
        for a, b in ((negated(x), w), (x, negated(w)), (negated(x), negated(w))):
            assert torch.equal(mm_grouped(a, b, off), want)
        for a, b in ((negated(dy), x), (dy, negated(x))):
            assert torch.equal(mm_grouped_wgrad(a, b, off), dwant)
    with pytest.raises(ValueError, match="lazily negated"):
        mm_grouped(x, w, off, out=negated(dy))


def test_forward_mode_is_refused():
    """a tangent is not dropped: every call with one raises"""
    from torch.autograd import forward_ad
    x, w, off = ints((40, 64), 1, BF16), ints((2, 72, 64), 2, BF16), offsets([15, 25])
    want = exact_mm(x, w, off).to(BF16)
    out = torch.full((40, 72), 3.0, dtype=BF16, device="cuda")
    with forward_ad.dual_level():
        xd, wd = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for a, b in ((xd, w), (x, wd), (xd, wd)):
            with pytest.raises(RuntimeError, match="forward AD"):
                mm_grouped(a, b, off)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward AD"):
                mm_grouped(a, b, off)
            with pytest.raises(RuntimeError, match="not differentiable"):
                mm_grouped(a, b, off, out=out)
        assert torch.equal(mm_grouped(x, w, off), want)      # nothing to follow
    assert bool((out == 3).all())


def test_outputs_that_autograd_follows_are_refused():
    x, w, dy, off = ints((40, 64), 1, BF16), ints((2, 72, 64), 2, BF16), ints((40, 72), 3, BF16), offsets([15, 25])
    leaf, dleaf = torch.ones(40, 72, dtype=BF16, device="cuda"), torch.ones(2, 72, 64, device="cuda")
    leaf.requires_grad_(), dleaf.requires_grad_()
    for out, dout in ((leaf, dleaf), (leaf * 2, dleaf * 2)):
        held = out.detach().clone(), dout.detach().clone()
        with pytest.raises(RuntimeError, match="out requires a gradient"):
            mm_grouped(x, w, off, out=out)
        with pytest.raises(RuntimeError, match="out requires a gradient"):
            mm_grouped_wgrad(dy, x, off, out=dout)
        assert torch.equal(out, held[0]) and torch.equal(dout, held[1])
    with torch.no_grad():
        mm_grouped(x, w, off, out=leaf), mm_grouped_wgrad(dy, x, off, out=dleaf)
    assert torch.equal(leaf, exact_mm(x, w, off).to(BF16)) and torch.equal(dleaf, exact_wgrad(dy, x, off).to(F32))


def test_no_report_is_lost_between_two_reads():
    """a kernel of another stream reports while the word is read: one of the reads, or one after both, has it (two, where one
    comes between the pair's two CTAs)"""
    L, status = _lib.lib(), ctypes.c_int(0)
    mine, other = torch.cuda.current_stream().cuda_stream, torch.cuda.Stream()
    read = lambda: L.spanqr_mm_read_status(mine, ctypes.byref(status))   # noqa: E731
    assert read() == 0
    for i in range(60):
        assert L.spanqr_mm_selftest_timeout(1_000 + 200 * i, 0, other.cuda_stream) == 0
        reports = 0
        while not other.query():
            reports += read() != 0
        reports += read() != 0
        assert 1 <= reports <= 2, (i, reports)


def test_a_pair_whose_waits_ran_out_stays_until_what_it_issued_has_landed():
    """10 ms, where the waits alone take a few microseconds; nothing stays where all arrived"""
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    a, b, c = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    assert L.spanqr_mm_selftest_timeout(100_000_000, 1, st) == 0          # (loaded)
    a.record()
    assert L.spanqr_mm_selftest_timeout(1_000, 0, st) == 0
    b.record()
    assert L.spanqr_mm_selftest_timeout(100_000_000, 1, st) == 0
    c.record()
    with pytest.raises(SpanqrError):
        mm_check()
    assert 9.9 <= a.elapsed_time(b) < 100 and b.elapsed_time(c) < 5


def test_waits_that_run_out_are_reported_and_leave_the_context_usable():
    """one pair of CTAs whose roles wait for what does not come, each for at most a millisecond"""
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    x, w, dy, off = ints((300, 64), 1, BF16), ints((2, 72, 64), 2, BF16), ints((300, 72), 3, BF16), offsets([115, 185])
    mm_check()
    assert L.spanqr_mm_selftest_timeout(100_000_000, 1, st) == 0          # everything arrives
    mm_check()
    for device in (None, "cuda", torch.cuda.current_device()):
        assert L.spanqr_mm_selftest_timeout(1_000_000, 0, st) == 0
        with pytest.raises(SpanqrError, match="wait ran out .status 0x100"):
            mm_check(device)
        mm_check()                                                        # reported once
        assert torch.equal(mm_grouped(x, w, off), exact_mm(x, w, off).to(BF16))
        assert torch.equal(mm_grouped_wgrad(dy, x, off), exact_wgrad(dy, x, off).to(F32))
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        assert L.spanqr_mm_selftest_timeout(1_000_000, 0, other.cuda_stream) == 0
    other.synchronize()
    with pytest.raises(SpanqrError):                                      # a word for the device, not for the stream
        mm_check()
    mm_check()
