"""ops.grad_norm / clip_grad_norm_ / adamw_step / adamw8_step against float64, and the 8-bit states bit for bit against a restatement of their
rule in numpy: scales from float32 operations that are each rounded once (as the kernel's are), codes from float64.

Tolerances: u = 2^-24.  m is two products and a sum (3 roundings), v three products and a sum (4), the new parameter carries one rounding of
the decay product, one of the sum, and the update's own: m 3 u, the root u (half of v's 4, plus its own) and eps' sum, the division (at most
2 units: an approximate reciprocal is allowed) and the step size: 12 u of the update covers them."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [(3, 5), (1,), (256,), (257,), (0,), (64, 32, 3, 3), (4096,), (4097,), (5, 1, 7), (20000,), (2,), (1023,)]


def rand(shape, scale, seed, dtype=torch.float32):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def make(sizes, pdt, gdt, master, seed=0):
    w = [rand(s, 0.1, seed + 10 * i) for i, s in enumerate(sizes)]
    p = [t.to(pdt) for t in w]
    if pdt == torch.float32:
        w = p
    g = [rand(s, 1e-3 * 4 ** (i % 3), seed + 10 * i + 1, gdt) for i, s in enumerate(sizes)]
    m = [rand(s, 3e-4, seed + 10 * i + 2) for i, s in enumerate(sizes)]
    v = [rand(s, 1e-3, seed + 10 * i + 3) ** 2 for i, s in enumerate(sizes)]
    return p, g, m, v, (w if master else None)


def reference(p, g, m, v, t, lr, b1, b2, eps, wd, scale=1.0):
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    g = g * scale
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    upd = lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p * (1 - lr * wd) - upd, m, v, upd, g


COMBOS = [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, True), (torch.bfloat16, torch.float32, True),
          (torch.bfloat16, torch.bfloat16, False), (torch.float16, torch.float16, True), (torch.float16, torch.float32, False)]


@pytest.mark.parametrize("t", [1, 2, 1000])
@pytest.mark.parametrize("pdt,gdt,master", COMBOS)
def test_step_against_float64(pdt, gdt, master, t):
    from coarse3d_amd import ops
    lr, b1, b2, eps, wd = 1e-3, 0.9, 0.999, 1e-8, 1e-2
    p, g, m, v, w = make(SIZES, pdt, gdt, master)
    before = [[x.clone() for x in l] for l in (w if master else p, g, m, v)]
    ops.adamw_step(p, g, m, v, step=t, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, masters=w)
    for i in range(len(SIZES)):
        rp, rm, rv, upd, gs = reference(*[l[i] for l in before], t, lr, b1, b2, eps, wd)
        assert torch.equal(g[i], before[1][i])
        assert ((m[i].double().cpu() - rm).abs() <= 4 * U * (before[2][i].double().cpu().abs() + gs.abs())).all()
        assert ((v[i].double().cpu() - rv).abs() <= 5 * U * rv + 1e-44).all()
        # (m is a sum that may cancel: its error counts as that of its terms)
        loose = lr / (1 - b1 ** t) * (before[2][i].double().cpu().abs() + gs.abs()) / (torch.sqrt(rv / (1 - b2 ** t)) + eps)
        tol = 3 * U * rp.abs() + 3 * U * before[0][i].double().cpu().abs() + 14 * U * (upd.abs() + loose)
        if master:
            assert ((w[i].double().cpu() - rp).abs() <= tol).all()
            assert torch.equal(p[i], w[i].to(pdt))
        else:
            assert ((p[i].double().cpu() - rp).abs() <= tol + (HALF[pdt] * rp.abs() * 1.01 + 2.0 ** -25 if pdt != torch.float32 else 0)).all()


@pytest.mark.parametrize("lr,betas,eps,wd", [(1e-2, (0.0, 0.0), 1e-8, 0.0), (3e-4, (0.95, 0.98), 1e-6, 0.1), (0.0, (0.9, 0.999), 1e-8, 0.0)])
def test_hyperparameters_and_many_steps_like_torch(lr, betas, eps, wd):
    """Twenty steps next to torch.optim.AdamW in float64 on the same gradients."""
    from coarse3d_amd import ops
    p, _, _, _, _ = make(SIZES, torch.float32, torch.float32, False, seed=3)
    ref = [torch.nn.Parameter(x.double().cpu()) for x in p]
    opt = torch.optim.AdamW(ref, lr=lr, betas=betas, eps=eps, weight_decay=wd)
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    for t in range(1, 21):
        g = [rand(x.shape, 1e-2, 7000 + 100 * t + i) for i, x in enumerate(p)]
        for r, x in zip(ref, g):
            r.grad = x.double().cpu()
        opt.step()
        ops.adamw_step(p, g, m, v, step=t, lr=lr, betas=betas, eps=eps, weight_decay=wd)
    for a, b in zip(p, ref):
        # per step: 3 u of the value, 40 u of an update of at most lr * 5 (with beta 0 exactly lr)
        assert ((a.double().cpu() - b).abs() <= 20 * (3 * U * b.abs() + 40 * U * 5 * lr) + 1e-12).all()


def np_mix(h):
    h = (h ^ (h >> np.uint32(16))) * np.uint32(0x9E3779B1)
    h = (h ^ (h >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return h ^ (h >> np.uint32(16))


def np_bits(blocks_before, n, step, seed):
    """Random bits of n elements whose first 256-block is number blocks_before of the call."""
    key = np_mix(np.array([(seed + step * 0x9E3779B9) % 2 ** 32], np.uint32))
    quad = (np.arange((n + 3) // 4, dtype=np.uint64) + blocks_before * 64).astype(np.uint32)
    x = np_mix(quad + key)
    cols = []
    for _ in range(4):
        cols.append(x)
        x = x ^ (x << np.uint32(13))
        x = x ^ (x >> np.uint32(17))
        x = x ^ (x << np.uint32(5))
    return np.stack(cols, 1).reshape(-1)[:n]


E4M3 = np.array([float(x) for x in torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()], np.float32)


def np_encode(x, wide, rnd16, floor):
    """x: the float32 values, which decide the scale; wide: the same in float64, which decide the codes: the grid point below
    |wide| / scale, or the one above where the fraction plus rnd16 / 2^16 reaches one."""
    n = x.size
    codes, scales = np.zeros(n, np.uint8), np.zeros((n + 255) // 256, np.float32)
    grid = E4M3[:127].astype(np.float64)
    for b in range(scales.size):
        s = slice(b * 256, min(n, b * 256 + 256))
        xs, r = x[s], rnd16[s].astype(np.float64)
        fin = np.isfinite(xs)
        top = float(np.max(np.abs(xs[fin]), initial=0.0))
        k = -100
        while top > 448.0 * 2.0 ** k:
            k += 1
        scales[b] = 2.0 ** k
        a = np.minimum(np.abs(np.where(fin, wide[s], 0)) / 2.0 ** k, 448.0)
        i = np.searchsorted(grid, a, side="right") - 1
        width = np.where(i < 126, grid[np.minimum(i + 1, 126)] - grid[i], 32.0)
        c = np.minimum(i + ((a - grid[i]) / width + r / 65536.0 >= 1.0), 126)
        if floor:
            c = np.where((xs > 0) & (c == 0), 1, c)
        c = np.where(fin, c, 127).astype(np.uint8)
        codes[s] = c if floor else c | (np.signbit(xs).astype(np.uint8) << 7)
    return codes, scales


def np_step8(g, m8, ms, r8, rs, before, step, seed, b1=0.9, b2=0.999, scale=np.float32(1)):
    f = np.float32
    n = g.size
    rep = lambda s: np.repeat(s, 256)[:n]  # noqa: E731
    with np.errstate(all="ignore"):
        x = g * f(scale)
        m = E4M3[m8] * rep(ms) * f(b1) + x * f(1 - b1)
        old = E4M3[r8] * rep(rs)
        r = np.sqrt((old * old) * f(b2) + (x * x) * f(1 - b2))
        d = np.float64
        wide_m = (E4M3[m8] * rep(ms)).astype(d) * b1 + x.astype(d) * (1 - b1)
        wide_r = np.sqrt(old.astype(d) ** 2 * b2 + x.astype(d) ** 2 * (1 - b2))
    bits = np_bits(before, n, step, seed)
    return m, r, np_encode(m, wide_m, bits & 0xFFFF, False), np_encode(r, wide_r, bits >> np.uint32(16), True)


def state8(sizes):
    z = lambda s: torch.zeros(s, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # noqa: E731
    sc = lambda s: torch.zeros((math.prod(s) + 255) // 256, device="cuda")  # noqa: E731
    return [z(s) for s in sizes], [sc(s) for s in sizes], [z(s) for s in sizes], [sc(s) for s in sizes]


def same_codes(a, b):
    """NaN codes of either sign are one value."""
    a, b = a.copy(), b.copy()
    a[(a & 127) == 127] = 127
    b[(b & 127) == 127] = 127
    return np.array_equal(a, b)


@pytest.mark.parametrize("pdt,gdt,master", COMBOS)
def test_8bit_states_bit_for_bit(pdt, gdt, master):
    from coarse3d_amd import ops
    lr, eps, wd = 1e-3, 1e-8, 1e-2
    p, _, _, _, w = make(SIZES, pdt, gdt, master, seed=40)
    m8, ms, r8, rs = state8(SIZES)
    for t in range(1, 5):
        g = [rand(s, 1e-3 * 10.0 ** (i % 4 - 2), 900 * t + i, gdt) for i, s in enumerate(SIZES)]
        g[8].view(-1)[::3] = 0.0
        old = [[x.clone() for x in l] for l in (w if master else p, m8, ms, r8, rs)]
        ops.adamw8_step(p, g, m8, ms, r8, rs, step=t, lr=lr, eps=eps, weight_decay=wd, masters=w, seed=11)
        blocks = 0
        for i, s in enumerate(SIZES):
            n = math.prod(s)
            if n:
                u8 = lambda x: x.view(torch.uint8).cpu().numpy().reshape(-1)  # noqa: E731
                m, r, (mc, msc), (rc, rsc) = np_step8(g[i].float().cpu().numpy().reshape(-1), u8(old[1][i]), old[2][i].cpu().numpy(), u8(old[3][i]),
                                                      old[4][i].cpu().numpy(), blocks, t, 11)
                assert np.array_equal(ms[i].cpu().numpy(), msc) and np.array_equal(rs[i].cpu().numpy(), rsc), (t, i)
                assert same_codes(u8(m8[i]), mc) and same_codes(u8(r8[i]), rc), (t, i)
                # the parameter moves by the unrounded moments
                pb = old[0][i].double().cpu().numpy().reshape(-1)
                upd = lr / (1 - 0.9 ** t) * m.astype(np.float64) / (r.astype(np.float64) / math.sqrt(1 - 0.999 ** t) + eps)
                want = pb * (1 - lr * wd) - upd
                got = (w if master else p)[i].double().cpu().numpy().reshape(-1)
                tol = 6 * U * np.abs(pb) + 14 * U * np.abs(upd)
                if not master and pdt != torch.float32:
                    tol = tol + HALF[pdt] * 1.01 * np.abs(want) + 2.0 ** -25
                assert (np.abs(got - want) <= tol).all(), (t, i)
                if master:
                    assert torch.equal(p[i], w[i].to(pdt))
            blocks += (n + 255) // 256


def test_8bit_extremes():
    """One block each: zeros, denormals, huge values, one outlier over tiny neighbours (roots stay above zero), inf and NaN."""
    from coarse3d_amd import ops
    n = 256
    cases = [torch.zeros(n), torch.full((n,), 1e-44), torch.full((n,), 1e18), torch.linspace(-1, 1, n), torch.full((n,), 1e-12)]
    cases[4][7] = 5.0
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.linspace(-1, 1, n)
        x[100] = bad
        cases.append(x)
    g = [c.cuda() for c in cases]
    p = [torch.ones(n, device="cuda") for _ in cases]
    m8, ms, r8, rs = state8([(n,)] * len(cases))
    for t in (1, 2, 3):
        old = [[x.clone() for x in l] for l in (m8, ms, r8, rs)]
        ops.adamw8_step(p, g, m8, ms, r8, rs, step=t, lr=1e-3, weight_decay=0.0, seed=0xFFFFFFFF)
        for i in range(len(cases)):
            u8 = lambda x: x.view(torch.uint8).cpu().numpy()  # noqa: E731
            m, r, (mc, msc), (rc, rsc) = np_step8(g[i].cpu().numpy(), u8(old[0][i]), old[1][i].cpu().numpy(), u8(old[2][i]), old[3][i].cpu().numpy(), i, t,
                                                  0xFFFFFFFF)
            assert np.array_equal(ms[i].cpu().numpy(), msc) and np.array_equal(rs[i].cpu().numpy(), rsc), (t, i)
            assert same_codes(u8(m8[i]), mc) and same_codes(u8(r8[i]), rc), (t, i)
    assert (r8[4].view(torch.uint8) > 0).all()                     # the outlier's neighbours keep a root
    for i in (5, 6, 7):
        ok = torch.ones(n, dtype=torch.bool, device="cuda")
        ok[100] = False
        assert torch.isfinite(p[i][ok]).all() and torch.isfinite(m8[i].float()[ok]).all() and torch.isnan(r8[i].float()[100])
    assert torch.equal(p[0], torch.ones_like(p[0]))


def test_8bit_rounding_is_unbiased_and_states_follow_a_change():
    """The mean over steps and seeds of a constant's stored value is the constant; after the gradient drops by 100 the second moment
    decays as in 32 bits, although one step changes it by a hundredth of a code."""
    from coarse3d_amd import ops
    n, steps = 65536, 400
    g = torch.full((n,), 0.37, device="cuda")
    g[::256] = 1.0
    p = torch.zeros(n, device="cuda")
    m8, ms, r8, rs = (x[0] for x in state8([(n,)]))
    for t in range(1, steps + 1):
        ops.adamw8_step([p], [g], [m8], [ms], [r8], [rs], step=t, lr=0.0, betas=(0.5, 0.99), weight_decay=0.0, seed=3)
    body = torch.arange(n, device="cuda") % 256 != 0
    r = (r8.float().view(-1, 256) * rs[:, None]).view(-1)[body]
    m = (m8.float().view(-1, 256) * ms[:, None]).view(-1)[body]
    # a code step at 0.37 of a block whose largest is 1 is 2^-4 relative at most 2^-5 / 0.37: over 65k values the mean's error is below 1e-3; the root's square has
    # the (positive) variance of its noise on top: (1 / (1 - 0.99^2)) / 4 * (2^-4 / 2)^2 / ... < 5 %
    assert abs(float(m.mean()) - 0.37) < 2e-3 and abs(float(r.mean()) - 0.37) < 0.02
    g *= 0.01
    start = float(r.mean())
    for t in range(steps + 1, steps + 201):
        ops.adamw8_step([p], [g], [m8], [ms], [r8], [rs], step=t, lr=0.0, betas=(0.5, 0.99), weight_decay=0.0, seed=3)
    r = (r8.float().view(-1, 256) * rs[:, None]).view(-1)[body]
    assert abs(float(r.mean()) / start / math.sqrt(0.99 ** 200) - 1) < 0.1


def test_same_call_same_bits_and_the_seed_matters():
    from coarse3d_amd import ops
    def once(seed):
        p, g, m, v, _ = make(SIZES, torch.float32, torch.float32, False, seed=8)
        s = state8(SIZES)
        for t in (1, 2, 3):
            ops.adamw8_step(p, g, *s, step=t, lr=1e-3, seed=seed)
        return [x.clone() for l in (p, *s) for x in l]
    raw = lambda x: x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x  # noqa: E731
    a, b, c = once(1), once(1), once(2)
    assert all(torch.equal(raw(x), raw(y)) for x, y in zip(a, b))
    assert not all(torch.equal(raw(x), raw(y)) for x, y in zip(a, c))


@pytest.mark.parametrize("bits", [8, 32])
def test_device_scalars_equal_host_numbers_and_a_captured_step_reads_them(bits):
    from coarse3d_amd import ops

    def fresh():
        p, g, m, v, _ = make(SIZES, torch.float32, torch.float32, False, seed=5)
        return p, g, (m, v) if bits == 32 else state8(SIZES)
    fn = ops.adamw_step if bits == 32 else ops.adamw8_step
    p1, g1, s1 = fresh()
    p2, g2, s2 = fresh()
    t_dev, lr_dev = torch.zeros((), device="cuda"), torch.zeros((), device="cuda")
    scale = torch.tensor(0.25, device="cuda")
    lrs = [float(torch.tensor(x)) for x in (1e-3, 5e-4, 2e-3, 1e-3, 1e-4)]        # fp32 numbers
    graph = torch.cuda.CUDAGraph()
    for t, lr in enumerate(lrs, 1):
        fn(p1, g1, *s1, step=t, lr=lr, grad_scale=scale)
        t_dev.fill_(t)
        lr_dev.fill_(lr)
        if t == 2:
            with torch.cuda.graph(graph):
                fn(p2, g2, *s2, step=t_dev, lr=lr_dev, grad_scale=scale)
        if t >= 2:
            graph.replay()
        else:
            fn(p2, g2, *s2, step=t_dev, lr=lr_dev, grad_scale=scale)
        torch.cuda.synchronize()
        for a, b in zip(p1, p2):
            # the two sides form 1 - beta^t in float64 by different libraries: one unit of the step size, a few of the update
            assert ((a - b).abs() <= 8 * U * t * lr * 10 + 2 * U * a.abs()).all()
        for a, b in zip([x for l in s1 for x in l], [x for l in s2 for x in l]):
            raw = (lambda x: x.view(torch.uint8)) if a.dtype == torch.float8_e4m3fn else (lambda x: x)
            assert torch.equal(raw(a), raw(b))


def test_layouts_and_unaligned_addresses():
    """Channels-last weights, transposed matrices and tensors that start anywhere: elementwise, so the same numbers as on copies."""
    from coarse3d_amd import ops
    base = torch.randn(8, 6000, device="cuda")
    def build(aligned):
        out = []
        for r in range(4):
            row = base[r].clone()
            a = row[0:288].view(8, 4, 3, 3).contiguous(memory_format=torch.channels_last)
            b = row[300:340].view(5, 8).t()
            c = (row[341:341 + 1000] if not aligned else row[341:1341].clone())
            d = (row[1343:1343 + 4999 - 1343] if not aligned else row[1343:4999].clone())
            out.append([a, b, c, d])
        out[3] = [x.square_() for x in out[3]]
        return out
    p1, g1, m1, v1 = build(True)
    p2, g2, m2, v2 = build(False)
    assert p2[2].data_ptr() % 16 != 0
    ops.adamw_step(p1, g1, m1, v1, step=3, lr=1e-2)
    ops.adamw_step(p2, g2, m2, v2, step=3, lr=1e-2)
    for a, b in zip(p1 + m1 + v1, p2 + m2 + v2):
        torch.testing.assert_close(a, b, rtol=0, atol=0)
    s1, s2 = state8([x.shape for x in p1]), None
    raw = torch.zeros(20000, dtype=torch.uint8, device="cuda")
    at, lists = 1, ([], [])
    for l in lists:
        for x in p1:
            l.append(torch.as_strided(raw.view(torch.float8_e4m3fn), x.shape, x.stride(), at))
            at += x.numel() + 1
    s1 = (([torch.empty_strided(x.shape, x.stride(), device="cuda", dtype=torch.uint8).zero_().view(torch.float8_e4m3fn) for x in p1]), s1[1],
          ([torch.empty_strided(x.shape, x.stride(), device="cuda", dtype=torch.uint8).zero_().view(torch.float8_e4m3fn) for x in p1]), s1[3])
    sc = state8([x.shape for x in p1])
    s2 = (lists[0], sc[1], lists[1], sc[3])
    for t in (1, 2):
        ops.adamw8_step(p1, g1, *s1, step=t, lr=1e-2)
        ops.adamw8_step(p2, g2, *s2, step=t, lr=1e-2)
    for a, b in zip(p1, p2):
        torch.testing.assert_close(a, b, rtol=0, atol=0)
    for l1, l2 in zip(s1, s2):
        for a, b in zip(l1, l2):
            assert torch.equal(a.float(), b.float())
    assert int(raw[0]) == 0 and not raw[at:].any()                 # what lies around the tensors stays


def test_more_tensors_than_a_launch_takes():
    from coarse3d_amd import ops
    sizes = [(7 + i % 300,) for i in range(500)]
    p, g, m, v, _ = make(sizes, torch.float32, torch.float32, False, seed=2)
    want = [reference(*x, 1, 1e-3, 0.9, 0.999, 1e-8, 1e-2)[0] for x in zip(p, g, m, v)]
    total = math.sqrt(sum(float((x.double() ** 2).sum()) for x in g))
    norm, scale = ops.grad_norm(g, 0.5 * total)
    assert abs(float(norm) / total - 1) <= 2 * U and abs(float(scale) / (0.5 * total / (total + 1e-6)) - 1) <= 2 * U
    ops.adamw_step(p, g, m, v, step=1, lr=1e-3)
    for a, b in zip(p, want):
        assert (a.double().cpu() - b).abs().max() < 1e-7
    p, g, m, v, _ = make(sizes, torch.float32, torch.float32, False, seed=2)
    s = state8(sizes)
    ops.adamw8_step(p, g, *s, step=1, lr=1e-3, seed=5)
    blocks = 0
    for i, sz in enumerate(sizes):
        n = sz[0]
        z = np.zeros(n, np.uint8)
        _, _, (mc, msc), (rc, rsc) = np_step8(g[i].cpu().numpy(), z, np.zeros((n + 255) // 256, np.float32), z, np.zeros((n + 255) // 256, np.float32), blocks, 1, 5)
        assert same_codes(s[0][i].view(torch.uint8).cpu().numpy(), mc) and same_codes(s[2][i].view(torch.uint8).cpu().numpy(), rc), i
        blocks += (n + 255) // 256


LISTS = {"short": SIZES, "one value": [(1,)], "full": [(64 * 256,)], "over": [(64 * 256,), (1,)], "many": [(3,)] * 241, "most": [(256,)] * 64, "sixteen": [(64 * 512,)],
         "long": [(300000,), (7,), (0,), (65537,)]}


@pytest.mark.parametrize("sizes", LISTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_and_clip(dtype, sizes):
    """Lists on both sides of what one workgroup takes by itself (64 blocks of 16 bytes a lane)."""
    from coarse3d_amd import ops
    g = [rand(s, 3.0, 60 + i, dtype) for i, s in enumerate(LISTS[sizes])]
    total = math.sqrt(sum(float((x.double() ** 2).sum()) for x in g))
    norm, scale = ops.grad_norm(g)
    assert abs(float(norm) / total - 1) <= 2 * U and float(scale) == 1.0
    old = [x.clone() for x in g]
    versions = [x._version for x in g]
    limit = total * 0.4
    n2 = ops.clip_grad_norm_(g, limit)
    assert float(n2) == float(norm) and all(x._version > v for x, v in zip(g, versions))
    f = limit / (total + 1e-6)
    for a, b in zip(g, old):
        want = b.double() * f
        assert ((a.double() - want).abs() <= (HALF[dtype] * 1.01 + 3 * U) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
    old = [x.clone() for x in g]
    ops.clip_grad_norm_(g, 1e9)
    assert all(torch.equal(a, b) for a, b in zip(g, old))
    assert abs(float(ops.clip_grad_norm_(g, 0.0)) / limit - 1) < 0.01 and all(not x.any() for x in g)


def test_norm_of_what_fp32_squares_lose():
    from coarse3d_amd import ops
    big, small = torch.full((1000,), 1e30, device="cuda"), torch.full((1000,), 1e-30, device="cuda")
    assert abs(float(ops.grad_norm([big])[0]) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    assert abs(float(ops.grad_norm([small])[0]) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    big[3] = float("inf")
    norm, scale = ops.grad_norm([big], 1.0)
    assert math.isinf(float(norm)) and float(scale) == 0.0
    big[3] = float("nan")
    norm, scale = ops.grad_norm([big], 1.0)
    assert math.isnan(float(norm)) and math.isnan(float(scale))
    assert float(ops.grad_norm([torch.empty(0, device="cuda"), torch.empty(3, 0, device="cuda")], 1.0)[0]) == 0.0


def test_one_tensor_longer_than_a_record():
    """Longer than 2^30 elements: cut into two records, whose blocks keep their numbers."""
    from coarse3d_amd import ops
    n = (1 << 30) + 5000
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-6000:] = rand((6000,), 1e-2, 1, torch.bfloat16)
    g[:4] = 2.0
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    m8 = torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    r8 = torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    ms, rs = torch.zeros((n + 255) // 256, device="cuda"), torch.zeros((n + 255) // 256, device="cuda")
    ops.adamw8_step([p], [g], [m8], [ms], [r8], [rs], step=1, lr=1e-3, seed=2)
    lo = (n - 6000) // 256 * 256
    z8, zs = np.zeros(n - lo, np.uint8), np.zeros((n - lo + 255) // 256, np.float32)
    _, _, (mc, msc), (rc, rsc) = np_step8(g[lo:].float().cpu().numpy(), z8, zs, z8, zs, lo // 256, 1, 2)
    assert same_codes(m8[lo:].view(torch.uint8).cpu().numpy(), mc) and same_codes(r8[lo:].view(torch.uint8).cpu().numpy(), rc)
    assert np.array_equal(ms[lo // 256:].cpu().numpy(), msc) and np.array_equal(rs[lo // 256:].cpu().numpy(), rsc)
    assert not p[4:lo].any() and (p[:4] != 0).all()
    want = math.sqrt(16.0 + float((g[-6000:].double() ** 2).sum()))
    assert abs(float(ops.clip_grad_norm_([g], 1.0)) / want - 1) <= 2 * U
    assert abs(float(ops.grad_norm([g])[0]) - 1.0) < 2.0 ** -8


def test_on_another_stream_and_two_graphs():
    from coarse3d_amd import ops
    g = [rand(s, 1.0, 5 + i) for i, s in enumerate(SIZES)]
    keep = [x.clone() for x in g]
    want = ops.grad_norm(g, 1.0)
    off = torch.zeros(4000, device="cuda")[1:3501]           # an address off the vector grid
    off.normal_()
    assert abs(float(ops.grad_norm([off])[0]) / float(off.double().norm()) - 1) <= 2 * U
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.grad_norm(g, 1.0)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a = ops.clip_grad_norm_(g, 1.0)
    with torch.cuda.graph(g2):
        b, _ = ops.grad_norm(g, 1.0)
    for k in (1.0, 3.0, 0.5, 2.0):
        for x, y in zip(g, keep):
            x.copy_(y * k)
        torch.cuda.synchronize()
        n0 = ops.grad_norm(g)[0].clone()
        g2.replay()
        torch.cuda.synchronize()
        g1.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, n0) and torch.equal(b, n0)
        for x, y in zip(g, keep):
            torch.testing.assert_close(x, y * k * min(1.0, 1.0 / (float(n0) + 1e-6)), rtol=1e-6, atol=0)
