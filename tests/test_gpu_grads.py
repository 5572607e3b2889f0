"""grad_norm and clip_grads on the GPU against the formula in fp64.

Tolerances.  The kernel sums a vector of at most 16 squares in fp32 (relative error below 16 * 2^-24, all terms
positive) and the rest in fp64, so the norm is within 8 * 2^-24 of the exact one before its rounding to fp32 (2^-24):
NORM_TOL = 9 * 2^-24.  A scaled value carries the norm's 8, the coefficient's rounding, the product's rounding (1 each)
and, in 16 bits, the rounding of the result: half a step of the type."""
import pytest
import torch

from spanqr_b200 import clip_grads, grad_norm, orth_batched

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NORM_TOL = 9 * U
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def norm64(ts):
    # scaled so that squares of fp32's largest values stay inside fp64 comfortably (they do: 2^256)
    return float(sum((t.double().cpu() ** 2).sum() for t in ts) ** 0.5)


def coef64(n, max_norm):
    return min(1.0, max_norm / (n + 1e-6))


def check_norm(got, want):
    assert got.dtype == F32 and got.dim() == 0
    assert abs(got.item() - want) <= NORM_TOL * want, (got.item(), want)


def check_clipped(got, x, coef):
    want = x.double().cpu() * coef
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2    # half a subnormal step
    err = (got.double().cpu() - want).abs()
    tol = want.abs() * (half * (1 + 10 * U) + 10 * U) + tiny * 1.01
    assert got.shape == x.shape and bool((err <= tol).all()), float((err - tol).max())


def rand(shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def mixed(seed=0):
    """odd sizes around the vector (8 or 16 elements) and chunk (8192 or 16384) borders, empty tensors and scalars"""
    sizes = [(), (1,), (0,), (7,), (8,), (9,), (15, 3), (16,), (17,), (33, 5), (8191,), (8192,), (8193,), (16385,), (0, 4),
             (3, 16384), (129, 257)]
    return [rand(s, (F32, BF16, F16)[i % 3], seed + i, 10.0 ** (i % 5 - 3)) for i, s in enumerate(sizes)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [1, 7, 8, 31, 8192, 8193, 100003, 3 << 20])
def test_norm_and_clip_of_one_tensor(dtype, n):
    x = rand((n,), dtype, n)
    want = norm64([x])
    check_norm(grad_norm([x]), want)
    x0 = x.clone()
    (y,), norm = clip_grads([x], 0.5)
    assert y.dtype == dtype and torch.equal(x, x0)
    check_norm(norm, want)
    check_clipped(y, x, coef64(want, 0.5))


def test_mixed_list_new_tensors_in_place_and_fp32_out():
    ts = mixed()
    want = norm64(ts)
    check_norm(grad_norm(ts), want)
    c = coef64(want, 1.0)
    ys, norm = clip_grads(ts, 1.0)
    check_norm(norm, want)
    for y, x in zip(ys, ts):
        assert y.dtype == x.dtype
        check_clipped(y, x, c)
    wide = [torch.full(t.shape, float("nan"), device="cuda") for t in ts]
    res, _ = clip_grads(ts, 1.0, out=wide)
    for y, x, o in zip(res, ts, wide):
        assert y is o
        check_clipped(y, x, c)
    inplace = [t.clone() for t in ts]
    res, _ = clip_grads(inplace, 1.0, out=inplace)
    for a, b in zip(res, ys):
        assert torch.equal(a, b)


@pytest.mark.parametrize("count", [63, 64, 65, 900, 901, 2003])
def test_long_lists(count):
    big = rand((count * 37,), F32, count)
    ts = [big[37 * i:37 * i + 1 + i % 37] for i in range(count)]
    want = norm64(ts)
    check_norm(grad_norm(ts), want)
    ys, norm = clip_grads(ts, 0.1)
    check_norm(norm, want)
    c = coef64(want, 0.1)
    check_clipped(torch.cat(ys), torch.cat(ts), c)


@pytest.mark.parametrize("dtype,off_in,off_out", [(F32, 1, 0), (F32, 3, 5), (BF16, 1, 0), (BF16, 0, 3), (F16, 7, 7)])
def test_misaligned_views(dtype, off_in, off_out):
    n = 50021
    src = rand((n + 64,), dtype, 5)
    x = src[off_in:off_in + n]
    guard = torch.full((n + 64,), 7.0, dtype=dtype, device="cuda")
    o = guard[off_out:off_out + n]
    want = norm64([x])
    check_norm(grad_norm([x]), want)
    clip_grads([x], 0.25, out=[o])
    check_clipped(o, x, coef64(want, 0.25))
    assert bool((guard[:off_out] == 7).all()) and bool((guard[off_out + n:] == 7).all())


@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-30, 1e-20, 1e-12, 1e15, 1e19, 1e30, 3e37])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_squares_outside_fp32(scale, dtype):
    x = rand((40001,), dtype, 3, scale)
    for ts in ([x], [x, rand((513,), dtype, 4, 1.0)]):
        want = norm64(ts)
        n = grad_norm(ts)
        if want > torch.finfo(F32).max:      # 200 * 3e37 = 6e39: the norm's nearest fp32 value is infinity
            assert n.item() == float("inf")
        else:                                # a norm below fp32's normal range is rounded to a subnormal step
            assert abs(n.item() - want) <= NORM_TOL * want + 2.0 ** -150, (n.item(), want)
        ys, _ = clip_grads(ts, 1.0)          # the coefficient comes from the fp64 norm
        for y, t in zip(ys, ts):
            check_clipped(y, t, coef64(want, 1.0))


def test_norm_of_many_equal_values_does_not_drift():
    x = torch.full((1 << 26,), 0.1, device="cuda")
    want = (float(x[0].item()) ** 2 * x.numel()) ** 0.5
    check_norm(grad_norm([x]), want)


def test_a_tensor_past_two_to_the_31_elements():
    n = (1 << 31) + 12345
    x = torch.zeros(n, dtype=BF16, device="cuda")
    x[7], x[n - 1], x[1 << 31] = 3.0, 4.0, 12.0
    assert grad_norm([x]).item() == 13.0
    clip_grads([x], 6.5, out=[x])                        # 6.5 / (13 + 1e-6): half, to fp32's last bits
    assert x[7].item() == 1.5 and x[n - 1].item() == 2.0 and x[1 << 31].item() == 6.0 and int((x != 0).sum()) == 3


def test_zero_empty_and_unclipped():
    z = [torch.zeros(1000, device="cuda"), torch.zeros(0, device="cuda")]
    assert grad_norm(z).item() == 0.0 and grad_norm([]).item() == 0.0
    ys, n = clip_grads(z, 1.0)
    assert n.item() == 0.0 and bool((ys[0] == 0).all()) and ys[1].numel() == 0
    assert clip_grads([], 1.0)[1].item() == 0.0
    x = rand((3000,), BF16, 1)
    for m in (1e6, float("inf")):
        (y,), _ = clip_grads([x], m)
        assert torch.equal(x, y)
        w = x.clone()
        clip_grads([w], m, out=[w])
        assert torch.equal(x, w)
    (y,), _ = clip_grads([x], 0.0)
    assert bool((y == 0).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_infinite_and_nan_gradients(dtype):
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = rand((20000,), dtype, 2)
        x[12345] = bad
        n = grad_norm([x]).item()
        (y,), norm = clip_grads([x], 1.0)
        if bad != bad:
            assert n != n and bool(y.isnan().all())
        else:
            assert n == float("inf") and bool(y[12345].isnan()) and int((y == 0).sum()) == 19999


def test_strides():
    base = rand((300, 200), F32, 8)
    col, tr, ex = base[:, 3:50], base.t(), base[:1].expand(9, 200)
    for t in (col, tr, ex):
        want = norm64([t])
        check_norm(grad_norm([t]), want)
        (y,), _ = clip_grads([t], 1.0)
        assert y.is_contiguous()
        check_clipped(y, t, coef64(want, 1.0))
    want = coef64(norm64([base]), 1.0) * base.double()
    clip_grads([tr], 1.0, out=[tr])                      # dense: in place through its transposed view
    assert float((base.double() - want).abs().max()) <= 10 * U * float(want.abs().max())
    with pytest.raises(ValueError, match="contiguous"):
        clip_grads([col], 1.0, out=[col])
    with pytest.raises(ValueError, match="contiguous"):
        clip_grads([rand((300, 47))], 1.0, out=[col])


def test_refusals():
    x, y = rand((64,)), rand((64,))
    with pytest.raises(ValueError, match="overlap"):
        clip_grads([x, x], 1.0, out=[x, x])
    with pytest.raises(ValueError, match="overlap"):
        clip_grads([x[:32], x[16:48]], 1.0, out=[x[:32], x[16:48]])
    with pytest.raises(ValueError, match="overlap"):
        clip_grads([x, y], 1.0, out=[y, x])
    with pytest.raises(ValueError, match="2 tensors"):
        clip_grads([x, y], 1.0, out=[x])
    with pytest.raises(ValueError, match="shape"):
        clip_grads([x], 1.0, out=[y.view(8, 8)])
    with pytest.raises(TypeError, match="fp32"):
        clip_grads([x], 1.0, out=[y.half()])
    n = grad_norm([x, x])                                # listed twice: counts twice
    check_norm(n, norm64([x, x]))


def test_deterministic_and_version_counter():
    ts = mixed(100)
    a, na = clip_grads(ts, 1.0)
    for _ in range(3):
        b, nb = clip_grads(ts, 1.0)
        assert torch.equal(na, nb) and all(torch.equal(p, q) for p, q in zip(a, b))
    v = ts[3]._version
    clip_grads(ts, 1.0, out=ts)
    assert ts[3]._version > v


def test_streams_and_captured_graphs():
    """calls on two streams, and two graphs captured one after the other and replayed at the same time, keep apart"""
    a, b = rand((5 << 20,), F32, 1), rand((5 << 20,), F32, 2, 3.0)
    oa, ob = torch.empty_like(a), torch.empty_like(b)
    wa, wb = norm64([a]), norm64([b])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g1, stream=s1):
        _, n1 = clip_grads([a], 1.0, out=[oa])
    with torch.cuda.graph(g2, stream=s1):
        _, n2 = clip_grads([b], 2.0, out=[ob])
    torch.cuda.synchronize()
    for _ in range(5):
        oa.zero_(), ob.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
            n3 = grad_norm([a])
        torch.cuda.synchronize()
        check_norm(n1, wa), check_norm(n2, wb), check_norm(n3, wa)
        check_clipped(oa, a, coef64(wa, 1.0)), check_clipped(ob, b, coef64(wb, 2.0))
    a.mul_(2.0)                                          # a replay reads the tensors' present values
    g1.replay()
    torch.cuda.synchronize()
    check_norm(n1, 2 * wa)


def test_under_a_process_group():
    import socket

    import torch.distributed as dist
    with socket.socket() as free:
        free.bind(("127.0.0.1", 0))
        port = free.getsockname()[1]
    dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    try:
        ts = mixed(7)
        want = norm64(ts)
        check_norm(grad_norm(ts, group=dist.group.WORLD), want)
        ys, n = clip_grads(ts, 1.0, group=dist.group.WORLD)
        check_norm(n, want)
        for y, x in zip(ys, ts):
            check_clipped(y, x, coef64(want, 1.0))
        assert grad_norm([], group=dist.group.WORLD).item() == 0.0
    finally:
        dist.destroy_process_group()


def test_clipped_gradients_go_to_orth():
    """bf16 layer gradients -> clipped fp32 -> orth_batched: the clipped step's basis is the gradients' own"""
    gs = [rand((768, 128), BF16, 20 + i, 4.0) for i in range(3)]
    wide = [torch.empty(g.shape, device="cuda") for g in gs]
    fs, _ = clip_grads(gs, 1.0, out=wide)
    for q, g in zip(orth_batched(fs), gs):
        q, g = q.double(), g.double()
        assert float((q.t() @ q - torch.eye(128, device="cuda")).abs().max()) <= 3e-7
        assert float((g - q @ (q.t() @ g)).norm() / g.norm()) <= 1e-5


def test_lazily_negated_tensors():
    """the imaginary part of a conjugate (the gradient of b in complex(a, b).conj() is one) into new and given tensors, in
    place, and refused as another tensor's output"""
    z = torch.tensor([3.0 + 4.0j], device="cuda")
    x, y = z.conj().imag, torch.zeros(1, device="cuda")
    assert x.is_neg() and x.is_contiguous() and x.item() == -4.0
    (a,), n = clip_grads([x], 8.0)
    clip_grads([x], 8.0, out=[y])
    assert a.item() == y.item() == -4.0 and n.item() == 4.0 and x.item() == -4.0
    (a,), _ = clip_grads([x], 2.0)
    check_clipped(a, x, coef64(4.0, 2.0))
    with pytest.raises(ValueError, match="lazily negated"):
        clip_grads([y], 1.0, out=[x])
    want = x.clone()
    clip_grads([x], 2.0, out=[x])
    check_clipped(x, want, coef64(4.0, 2.0))
    assert z.item().real == 3.0
    v = torch.arange(1.0, 6.0, device="cuda").to(torch.cfloat).mul(1j).conj().imag      # with gaps
    (c,), _ = clip_grads([v], 100.0)
    assert c.tolist() == [-1.0, -2.0, -3.0, -4.0, -5.0]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("max_norm", [1e-12, 1e-18, 1e-19, 1e-20, 1e-25, 1e-31, 1e-38, 1e-41, 1e-44, 1e-60, 1e-300, 5e-324])
@pytest.mark.parametrize("scale", [1.0, 1e30, 3e37])
def test_small_maximal_norms(scale, max_norm, dtype):
    """coefficients down to and past those whose products all round to zero (1e-60 / 6e39 is 2^-331)"""
    ts = [rand((40001,), dtype, 3, scale), rand((70,), dtype, 4, scale)]
    want = norm64(ts)
    for out in (None, [torch.empty(t.shape, device="cuda") for t in ts]):
        ys, _ = clip_grads(ts, max_norm, out=out)
        for y, t in zip(ys, ts):
            check_clipped(y, t, coef64(want, max_norm))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_infinite_gradient_and_infinite_maximal_norm(dtype):
    """the coefficient of an infinite norm is 0 whatever max_norm is: inf / inf is not left to become NaN everywhere"""
    x = rand((20000,), dtype, 2)
    x[12345] = float("-inf")
    for out in (None, [x.clone()]):
        ins = [x] if out is None else out
        (y,), n = clip_grads(ins, float("inf"), out=out)
        assert n.item() == float("inf") and bool(y[12345].isnan()) and int((y == 0).sum()) == 19999
    x[777] = float("nan")
    (y,), n = clip_grads([x], float("inf"))
    assert n.isnan().item() and bool(y.isnan().all())


def test_a_group_adds_the_sums_of_squares_in_fp64(monkeypatch):
    """another rank's part, added where the all-reduce would: to the fp64 sum of squares on the tensors' device, once per call"""
    import torch.distributed as dist
    ts, other, group, seen = mixed(11), rand((5001,), F32, 12, 3.0), object(), []

    def all_reduce(t, op=None, group=None):
        assert t.dtype == torch.float64 and t.dim() == 0 and t.is_cuda
        seen.append(group)
        t += other.double().square().sum()
    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    both, alone = norm64(ts + [other]), norm64([other])
    check_norm(grad_norm(ts, group=group), both)
    check_norm(grad_norm([], group=group), alone)
    for out in (None, [torch.empty(t.shape, device="cuda") for t in ts]):
        ys, n = clip_grads(ts, 1.0, out=out, group=group)
        check_norm(n, both)
        for y, x in zip(ys, ts):
            check_clipped(y, x, coef64(both, 1.0))
    _, n = clip_grads([], 1.0, group=group)
    check_norm(n, alone)
    assert seen == [group] * 5
    with pytest.raises(TypeError):
        grad_norm([other.double()], group=group)
    assert len(seen) == 6                                 # a refused list takes part too


def test_lazily_negated_tensors_of_any_length():
    """as_strided lays a view without gaps over the memory of a conjugate's imaginary part"""
    for dtype, part in ((torch.complex64, F32), (torch.complex32, F16)):
        z = torch.zeros(3000, dtype=dtype, device="cuda")
        z.imag.copy_(rand((3000,), part, 1)), z.real.copy_(rand((3000,), part, 2))
        x = z.conj().imag.as_strided((5999,), (1,), 1)
        assert x.dtype == part and x.is_neg() and x.is_contiguous()
        c = coef64(norm64([x]), 2.0)
        (y,), n = clip_grads([x], 2.0)
        check_norm(n, norm64([x]))
        check_clipped(y, x, c)
        wide = [torch.empty(5999, device="cuda"), torch.empty(7, device="cuda")]
        ones = torch.ones(7, device="cuda")
        clip_grads([x, ones], 2.0, out=wide)
        check_clipped(wide[0], x, coef64(norm64([x, ones]), 2.0))
        want = x.clone()
        clip_grads([x], 2.0, out=[x])
        check_clipped(x, want, c)
        with pytest.raises(ValueError, match="lazily negated"):
            clip_grads([y], 1.0, out=[x])
