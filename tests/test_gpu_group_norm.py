"""ops.group_norm / group_norm_bwd against the formulas in float64.

Tolerances.  u = 2^-24 is half a unit in the last place of fp32 relative to the value.  No fp32 sum of the kernels adds more than 300
terms one after the other (256 of a thread and the joining of a workgroup's threads; longer ones are joined in 64 bits), so a mean of values bounded by A is off by at most 300 u A, and
so are the others (variance: twice, it is a mean of squares of deviations that are themselves off; its root halves that again).  With
A = max |x - mean| in units of sigma the normalised value is off by (300 + 300 A^2 + 8) u relative to its largest magnitude; the affine map and
the activation (slope at most 1.1) add a few u of their own magnitudes.  A result in 16 bits adds half a unit of its type, eps / 2, of itself."""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # eps / 2: 2^-24, 2^-8, 2^-11
TERMS = 300


def oracle(x, dy, groups, gamma, beta, eps, act, slope):
    """Everything in float64 on the CPU: y, mean, rstd, z, xhat, dx, dgamma, dbeta (sums), their absolute sums."""
    n, c = x.shape[0], x.shape[-1]
    xd = x.double().cpu().reshape(n, -1, groups, c // groups)
    mean = xd.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((xd - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xh = (xd - mean) * rstd
    ga = torch.ones(c) if gamma is None else gamma.cpu()
    be = torch.zeros(c) if beta is None else beta.cpu()
    ga, be = ga.double().view(groups, -1), be.double().view(groups, -1)
    z = xh * ga + be
    if act == "lrelu":
        d = torch.where(z > 0, 1.0, slope).double()
        y = z * d
    elif act == "silu":
        s = torch.sigmoid(z)
        y, d = z * s, s * (1 + z * (1 - s))
    else:
        y, d = z, torch.ones_like(z)
    out = dict(y=y, mean=mean.view(n, groups), rstd=rstd.view(n, groups), z=z, xh=xh)
    if dy is not None:
        dz = dy.double().cpu().reshape(xd.shape) * d
        t = dz * ga
        out["dx"] = rstd * (t - t.mean((1, 3), keepdim=True) - xh * (t * xh).mean((1, 3), keepdim=True))
        out["t"] = t
        out["dgamma"], out["dbeta"] = (dz * xh).sum((0, 1)).view(c), dz.sum((0, 1)).view(c)
        out["agamma"], out["abeta"] = (dz * xh).abs().sum((0, 1)).view(c), dz.abs().sum((0, 1)).view(c)
    return out


def make(shape, dtype, groups, seed=0, offset=0.0, affine=True, kink_free=True, slope=0.01):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g) * (torch.rand(c, generator=g) + 0.5) + offset).to(dtype)
    gamma = (torch.rand(c, generator=g) + 0.5) if affine else None
    beta = (torch.randn(c, generator=g) * 0.2) if affine else None
    dy = torch.randn(shape, generator=g)
    if kink_free and x.numel():       # where z is within rounding of the kink its derivative is not defined: no gradient arrives there
        z = oracle(x, None, groups, gamma, beta, 1e-5, "none", slope)["z"].reshape(shape)
        dy = torch.where(z.abs() < 1e-4, 0.0, dy)
    dy = dy.to(dtype)
    dev = [None if t is None else t.cuda() for t in (x, gamma, beta, dy)]
    return dev


def check(x, dy, groups, gamma, beta, act, slope=0.01, eps=1e-5):
    from coarse3d_amd import ops
    y, mean, rstd = ops.group_norm(x, groups, gamma, beta, eps=eps, act=act, slope=slope)
    dx, dgamma, dbeta = ops.group_norm_bwd(dy, x, mean, rstd, gamma, beta, act=act, slope=slope)
    assert y.shape == x.shape and y.dtype == x.dtype and dx.shape == x.shape and dx.dtype == x.dtype and y.is_contiguous() and dx.is_contiguous()
    o = oracle(x, dy, groups, gamma, beta, eps, act, slope)
    h = HALF[x.dtype] if x.dtype != torch.float32 else 0.0
    A = float(o["xh"].abs().max()) + 1
    far = float(x.double().abs().max()) * float(o["rstd"].max()) * 4 * U       # x - mean where both are large
    rel = (TERMS + TERMS * A * A + 8) * U + far
    gmax = 1.0 if gamma is None else float(gamma.abs().max())
    zerr = rel * A * gmax + 8 * U * float(o["z"].abs().max())
    yd, yo = y.double().cpu().reshape(o["y"].shape), o["y"]
    assert ((yd - yo).abs() <= 1.1 * zerr + h * yo.abs() + 1e-30 + (2.0 ** -25 if x.dtype == torch.float16 else 0)).all(), float((yd - yo).abs().max())
    assert ((mean.double().cpu() - o["mean"]).abs() * o["rstd"] <= TERMS * U * A + far).all()
    assert ((rstd.double().cpu() / o["rstd"] - 1).abs() <= (2 * TERMS + 8) * U * A * A).all()
    # dx: each term is off by rel of its own size, and by act' times that (its slope is at most 0.5 for SiLU, 0 away from the kink)
    tm = float(o["t"].abs().max())
    amp = float(o["rstd"].max()) * tm * (2 + 2 * A * A)
    dxd, dxo = dx.double().cpu().reshape(o["dx"].shape), o["dx"]
    tol = amp * (2 * rel + zerr) + h * dxo.abs() + 1e-30 + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    assert ((dxd - dxo).abs() <= tol).all(), float(((dxd - dxo).abs() - tol).max())
    if gamma is None:
        assert dgamma is None and dbeta is None
    else:
        assert ((dgamma.double().cpu() - o["dgamma"]).abs() <= (TERMS * U + 2 * rel + zerr) * (o["agamma"] + A * o["abeta"]) + 1e-30).all()
        assert ((dbeta.double().cpu() - o["dbeta"]).abs() <= (TERMS * U + zerr) * (o["abeta"] * (1 + A)) + 1e-30).all()


SHAPES = [
    ((1, 1, 1, 8), 4), ((1, 1, 1, 1), 1), ((2, 1, 3, 6), 2), ((1, 5, 7, 20), 5), ((3, 4, 9, 33), 11), ((2, 8, 16, 32), 8), ((1, 3, 5, 32), 32),
    ((2, 7, 13, 22), 1), ((4, 1, 1, 64), 16), ((2, 16, 33, 64), 16), ((1, 9, 11, 704), 32), ((1, 3, 7, 2056), 8), ((2, 2, 2, 1030), 5),
    ((1, 40, 91, 20), 5), ((5, 64), 8), ((2, 301, 48), 6), ((17, 2, 3, 16), 2), ((1, 64, 128, 32), 4),
]


@pytest.mark.parametrize("act", ["none", "lrelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_against_float64(shape, groups, dtype, act):
    x, gamma, beta, dy = make(shape, dtype, groups, seed=len(shape) * 100 + shape[-1])
    check(x, dy, groups, gamma, beta, act)


# more channels than a workgroup takes: tiles of whole groups (the last one short), groups in several parts, both without a common vector,
# a tile of one pixel
WIDE = [((1, 30, 30, 2100), 100), ((2, 5, 9, 4104), 3), ((2, 3, 5, 8200), 2), ((1, 9, 70, 4099), 1), ((1, 70, 30, 4096), 32), ((1, 8, 9, 4095), 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", WIDE)
def test_many_channels(shape, groups, dtype):
    x, gamma, beta, dy = make(shape, dtype, groups, seed=shape[-1])
    check(x, dy, groups, gamma, beta, "lrelu")


@pytest.mark.parametrize("slope", [0.0, 0.1, 1.0])
def test_slopes_and_no_affine(slope):
    x, _, _, dy = make((2, 9, 17, 24), torch.float32, 3, seed=5, affine=False)
    check(x, dy, 3, None, None, "lrelu", slope=slope)
    x, gamma, _, dy = make((2, 9, 17, 24), torch.float32, 3, seed=6)
    from coarse3d_amd import ops
    y, mean, rstd = ops.group_norm(x, 3, gamma, None, act="none")
    dx, dgamma, dbeta = ops.group_norm_bwd(dy, x, mean, rstd, gamma, None, act="none")
    assert dbeta is None and dgamma is not None and torch.isfinite(dx).all()


@pytest.mark.parametrize("offset", [100.0, -3000.0])
def test_mean_far_from_zero_keeps_the_variance(offset):
    """The variance of values around 3000 sigma: the sum of squares in fp32 would leave nothing of it."""
    x, gamma, beta, dy = make((2, 16, 64, 32), torch.float32, 8, seed=9, offset=offset)
    check(x, dy, 8, gamma, beta, "silu")


def test_constant_group_gives_beta():
    from coarse3d_amd import ops
    x = torch.full((2, 4, 5, 8), 3.25, device="cuda")
    beta = torch.arange(8, device="cuda", dtype=torch.float32)
    y, mean, rstd = ops.group_norm(x, 2, torch.ones(8, device="cuda"), beta, act="none")
    assert torch.equal(y, beta.expand_as(y)) and torch.equal(mean, torch.full_like(mean, 3.25))
    torch.testing.assert_close(rstd, torch.full_like(rstd, 1e-5 ** -0.5))


def test_not_finite_stays_in_its_group():
    from coarse3d_amd import ops
    for bad in (float("inf"), float("-inf"), float("nan")):
        for where in ((1, 0, 0), (1, 3, 5)):
            x, gamma, beta, dy = make((3, 4, 6, 16), torch.float32, 4, seed=3)
            clean, _, _ = ops.group_norm(x, 4, gamma, beta, act="silu")
            x[where[0], where[1], where[2], 6] = bad
            y, mean, rstd = ops.group_norm(x, 4, gamma, beta, act="silu")
            assert torch.isnan(y[1, :, :, 4:8]).all()
            keep = torch.ones_like(y, dtype=torch.bool)
            keep[1, :, :, 4:8] = False
            assert torch.equal(y[keep], clean[keep])
            dx, _, _ = ops.group_norm_bwd(dy, x, mean, rstd, gamma, beta, act="silu")
            assert torch.isnan(dx[1, :, :, 4:8]).all() and torch.isfinite(dx[keep]).all()


def test_strides_slices_and_alignment():
    """Channel slices, cropped pixels, samples of a larger batch, addresses off the vector grid: the same bits as on a dense copy (sums are
    taken in the same order whatever the vector width only if the plan is the same, so values are compared with the plan's tolerance)."""
    from coarse3d_amd import ops
    big = torch.randn(6, 10, 12, 40, device="cuda")
    gb = torch.randn(6, 10, 12, 40, device="cuda")
    for sl in ((slice(None), slice(None), slice(None), slice(4, 36)), (slice(None), slice(None), slice(None), slice(1, 33)),
               (slice(0, 6, 2), slice(2, 9), slice(None), slice(0, 16)), (slice(1, 2), slice(3, 4), slice(0, 11), slice(0, 40)),
               (slice(None), slice(0, 1), slice(0, 1), slice(8, 24))):
        x, dy = big[sl], gb[sl]
        c = x.shape[-1]
        gamma, beta = torch.rand(c, device="cuda") + 0.5, torch.randn(c, device="cuda")
        y, mean, rstd = ops.group_norm(x, 4, gamma, beta, act="silu")
        yc, mc, rc = ops.group_norm(x.contiguous(), 4, gamma, beta, act="silu")
        torch.testing.assert_close(y, yc, rtol=2e-5, atol=2e-5)
        for got, want in zip(ops.group_norm_bwd(dy, x, mean, rstd, gamma, beta, act="silu"),
                             ops.group_norm_bwd(dy.contiguous(), x.contiguous(), mc, rc, gamma, beta, act="silu")):
            torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)
    flat = torch.randn(4 * 5 * 6 * 16 + 1, device="cuda")[1:].view(4, 5, 6, 16)
    y, _, _ = ops.group_norm(flat, 4)
    yc, _, _ = ops.group_norm(flat.clone(), 4)
    torch.testing.assert_close(y, yc, rtol=2e-5, atol=2e-5)


@pytest.mark.parametrize("shape", [(0, 4, 5, 8), (2, 0, 5, 8), (0, 8)])
def test_empty(shape):
    from coarse3d_amd import ops
    x = torch.empty(shape, device="cuda")
    ga = torch.ones(8, device="cuda")
    y, mean, rstd = ops.group_norm(x, 4, ga, ga)
    assert y.shape == x.shape and mean.shape == (shape[0], 4)
    dx, dgamma, dbeta = ops.group_norm_bwd(x, x, mean, rstd, ga, ga)
    assert dx.shape == x.shape and not dgamma.any() and not dbeta.any()


def test_equal_inputs_give_equal_bits_and_other_memory_is_left_alone():
    from coarse3d_amd import ops
    x, gamma, beta, dy = make((3, 33, 65, 48), torch.float32, 6, seed=8)
    first = None
    for _ in range(3):
        y, mean, rstd = ops.group_norm(x, 6, gamma, beta)
        got = (y, mean, rstd) + ops.group_norm_bwd(dy, x, mean, rstd, gamma, beta)
        if first is None:
            first = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_gradient_against_differences():
    """Central differences of sum(y * dy), in the float64 oracle's forward, against the kernel's gradients."""
    x, gamma, beta, dy = make((1, 2, 3, 8), torch.float32, 2, seed=21)
    from coarse3d_amd import ops
    y, mean, rstd = ops.group_norm(x, 2, gamma, beta, act="silu")
    dx, dgamma, dbeta = ops.group_norm_bwd(dy, x, mean, rstd, gamma, beta, act="silu")
    f = lambda x_, g_, b_: float((oracle(x_, None, 2, g_, b_, 1e-5, "silu", 0.01)["y"].reshape(x.shape) * dy.double().cpu()).sum())  # noqa: E731
    h = 1e-4
    args = [x.double().cpu(), gamma.double().cpu(), beta.double().cpu()]
    for k, got in enumerate((dx, dgamma, dbeta)):
        for i in range(got.numel()):
            hi, lo = [a.clone() for a in args], [a.clone() for a in args]
            hi[k].view(-1)[i] += h
            lo[k].view(-1)[i] -= h
            # truncation h^2 |f'''| / 6 ~ 1e-8 * 100, rounding 2^-53 |f| / h ~ 1e-11; the kernel's own 1e-5
            assert abs((f(*hi) - f(*lo)) / (2 * h) - float(got.view(-1)[i])) < 1e-4 * (1 + abs(float(got.view(-1)[i])))


def test_on_another_stream_and_in_a_graph():
    from coarse3d_amd import ops
    x, gamma, beta, dy = make((2, 16, 40, 32), torch.bfloat16, 8, seed=4)

    def both():
        y, mean, rstd = ops.group_norm(x, 8, gamma, beta)
        return (y, mean, rstd) + ops.group_norm_bwd(dy, x, mean, rstd, gamma, beta)
    want = [t.clone() for t in both()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = both()
    with torch.cuda.graph(g2, pool=g1.pool()):
        o2 = both()
    keep = x.clone()
    for k in range(4):
        x.copy_(keep * (1 + k))
        torch.cuda.synchronize()
        want = [t.clone() for t in both()]
        g1.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, o1)), k
        g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, o2)), k


def test_two_streams_at_once():
    """Workspaces belong to a call: two calls in flight on two streams do not meet."""
    from coarse3d_amd import ops
    xs = [torch.randn(4, 64, 256, 32, device="cuda") for _ in range(2)]
    want = [ops.group_norm(x, 8)[0] for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(ops.group_norm(x, 8)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_more_than_2_31_elements():
    from coarse3d_amd import ops
    n, hw, c = 2, (1 << 20) + 77, 1032
    x = torch.empty(n, hw, c, device="cuda", dtype=torch.bfloat16)
    for i in range(n):
        x[i].normal_(mean=float(i), std=1.0 + i)
    assert x.numel() > 1 << 31
    y, mean, rstd = ops.group_norm(x, 8, act="none")
    tail = x[1, -1000:].double().view(1000, 8, -1)
    # 1.35e8 values a group: the mean is within 5 / sqrt(1.35e8) sigma of the distribution's, and the values that come back follow from the saved numbers
    assert (mean[1].double() - 1).abs().max() < 2e-3 and (rstd[1].double() - 0.5).abs().max() < 1e-3
    want = (tail - mean[1].double().view(1, 8, 1)) * rstd[1].double().view(1, 8, 1)
    got = y[1, -1000:].double().view_as(want)
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()
    dx, _, _ = ops.group_norm_bwd(x, x, mean, rstd, act="none")
    xh = want
    # dy = x = mu + xhat / rstd: t - mean(t) - xhat mean(t xhat) = 0 up to eps in the variance and rounding of the sums
    assert dx[1, -1000:].abs().max() < 1e-2 and torch.isfinite(dx[0, :1000]).all()


def test_long_rows_keep_their_accuracy():
    """Samples of half a million and of two million pixels: the mean error of long sums stays that of short ones (the worst case is 300 u =
    2e-5 of the terms; in the 2-norm over many independent roundings a tenth of it is far from reached)."""
    for shape in ((1, 64, 8192, 8), (1, 1, 2100003, 2)):
        long_rows(shape)


def long_rows(shape):
    from coarse3d_amd import ops
    x, gamma, beta, dy = make(shape, torch.float32, 2, seed=12, offset=2.0)
    y, mean, rstd = ops.group_norm(x, 2, gamma, beta, act="lrelu")
    dx, dgamma, dbeta = ops.group_norm_bwd(dy, x, mean, rstd, gamma, beta, act="lrelu")
    o = oracle(x, dy, 2, gamma, beta, 1e-5, "lrelu", 0.01)
    for got, name in ((y, "y"), (dx, "dx"), (dgamma, "dgamma"), (dbeta, "dbeta")):
        want = o[name].reshape(got.shape)
        assert float((got.double().cpu() - want).norm() / want.norm()) < 1e-5, name
