"""The cases that the small-batch training operators are measured by: group normalisation with an activation over channels-last
images, the global norm of many gradients with its clipping, and the AdamW step over many tensors with states in 32 or in 8 bits.

``own`` False computes them from elementary torch operations, ``own`` True calls ``coarse3d_amd.ops``."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS_NORM = 1e-5
SLOPE = 0.01
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 1.0
BLOCK = 256                    # elements that share a scale of the 8-bit states
SEED = 20                      # of the 8-bit states' rounding


def listed():
    return [
        # the deepest level of the encoder on one scan, in the mixed-precision mode: the smallest call, all latency
        dict(name="gn infer 1x4x128x256 bf16", kind="gn", train=False, n=1, h=4, w=128, c=256, groups=32, dtype="bf16", act="lrelu", offset=0.0),
        # the full-resolution level of a 64 x 2048 batch of eight, 32 channels, fp32
        dict(name="gn infer 8x64x2048x32 f32", kind="gn", train=False, n=8, h=64, w=2048, c=32, groups=8, dtype="f32", act="lrelu", offset=0.0),
        # one scan per GPU at the third level, forward and backward: what replaces batch statistics at batch size one
        dict(name="gn train 1x8x256x128 f32", kind="gn", train=True, n=1, h=8, w=256, c=128, groups=16, dtype="f32", act="lrelu", offset=0.0),
        # the first decoder level of a batch of eight
        dict(name="gn train 8x32x1024x64 f32", kind="gn", train=True, n=8, h=32, w=1024, c=64, groups=16, dtype="f32", act="lrelu", offset=0.0),
        # odd everything: three 40-row scans cropped to an odd width, twenty class channels in five groups, no vector of eight fits
        dict(name="gn train 3x40x903x20 f32", kind="gn", train=True, n=3, h=40, w=903, c=20, groups=5, dtype="f32", act="silu", offset=4.0),
        # the projector's hidden layer (704 channels, 22 per group) on two half-resolution scans, mixed precision
        dict(name="gn train 2x32x1024x704 bf16", kind="gn", train=True, n=2, h=32, w=1024, c=704, groups=32, dtype="bf16", act="lrelu", offset=0.0),
        # the projector alone: six tensors (704 -> 704 -> 256), where latency counts
        dict(name="adamw32 projector", kind="adamw", bits=32, clip=False, layout="projector", width=704, blocks=1, param="f32"),
        # a backbone of 192 tensors from 32 to 256 channels, gradients clipped by their global norm
        dict(name="adamw32 clip 192 tensors", kind="adamw", bits=32, clip=True, layout="net", width=32, blocks=48, param="f32"),
        # the same backbone with the states in 8 bits
        dict(name="adamw8 192 tensors", kind="adamw", bits=8, clip=False, layout="net", width=32, blocks=48, param="f32"),
        # a deep backbone of 64 to 512 channels (208 tensors, 41 M), parameters and gradients in bf16 with fp32 masters, 8-bit states
        dict(name="adamw8 clip 208 tensors bf16", kind="adamw", bits=8, clip=True, layout="net", width=64, blocks=52, param="bf16m"),
        # clipping as a call of its own, in place: the backbone in fp32, the deep one in bf16
        dict(name="clip 192 tensors f32", kind="clip", layout="net", width=32, blocks=48, param="f32"),
        dict(name="clip 208 tensors bf16", kind="clip", layout="net", width=64, blocks=52, param="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gn", "gn", "gn", "adamw", "adamw", "clip"])
    if kind == "gn":
        groups = rng.choice([1, 2, 4, 5, 8, 16, 32])
        c = groups * _log_uniform(rng, 1, max(1, 704 // groups))
        n = rng.randint(1, 16)
        h = rng.randint(1, 64)
        w = max(1, min(_log_uniform(rng, 1, 2048), 30_000_000 // (n * h * c)))
        w = max(w, -(-16 * groups // (h * c)))               # with a handful of values in a group the gradient is a difference of equal numbers
        return dict(kind="gn", train=rng.random() < 0.7, n=n, h=h, w=w, c=c, groups=groups, dtype=rng.choice(["f32", "bf16", "f16"]),
                    act=rng.choice(["lrelu", "silu", "none"]), offset=rng.choice([0.0, 0.5, 4.0]))
    layout = rng.choice(["net", "net", "projector"])
    if layout == "net":
        width, blocks = _log_uniform(rng, 3, 48), _log_uniform(rng, 1, 52)
    else:
        width, blocks = _log_uniform(rng, 16, 1500), 1
    param = rng.choice(["f32", "f32", "bf16", "f16"] if kind == "clip" else ["f32", "f32", "bf16m", "f16m"])
    d = dict(kind=kind, layout=layout, width=width, blocks=blocks, param=param)
    if kind == "adamw":
        d.update(bits=rng.choice([8, 32]), clip=rng.random() < 0.5)
    return d


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _shapes(case):
    """The parameter tensors of the case, in order."""
    w = case["width"]
    if case["layout"] == "projector":
        out = max(1, w * 4 // 11)
        return [(w, w, 1, 1), (w,), (w,), (w,), (out, w, 1, 1), (out,)]
    shapes = []
    for b in range(case["blocks"]):
        c = w << (b % 4)
        shapes += [(c, c, 3, 3), (c,), (c,), (c,)]
    return shapes


def _offsets(case):
    """[(first element, elements)] of the tensors in one buffer, and its length; every tensor starts at a multiple of BLOCK."""
    at, spans = 0, []
    for s in _shapes(case):
        n = math.prod(s)
        spans.append((at, n))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return spans, at


def _quantised(x):
    """x [blocks, BLOCK] >= 0 or signed -> (e4m3 codes, scales): a starting state, rounded to the nearest code."""
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(1).clamp_min(1e-30) / 448.0)))
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def _prepare_gn(case, seed):
    g = _generator(seed)
    n, h, w, c, groups = case["n"], case["h"], case["w"], case["c"], case["groups"]
    dt = DTYPES[case["dtype"]]
    spread = torch.rand(c, device="cuda", generator=g) + 0.5
    centre = torch.randn(c, device="cuda", generator=g) * 0.3 + case["offset"]
    x = torch.randn(n, h, w, c, device="cuda", generator=g).mul_(spread).add_(centre).to(dt)
    gamma = torch.rand(c, device="cuda", generator=g) + 0.5
    beta = torch.randn(c, device="cuda", generator=g) * 0.2
    state = dict(case=case, x=x, gamma=gamma, beta=beta)
    if case["train"]:
        dy = torch.randn(n, h, w, c, device="cuda", generator=g)
        if case["act"] == "lrelu":
            # at the kink the derivative has no value to agree on: no gradient arrives within rounding of it
            z = x.double().view(n, h * w, groups, c // groups)
            var, mean = torch.var_mean(z, dim=(1, 3), keepdim=True, correction=0)
            z = ((z - mean) * torch.rsqrt(var + EPS_NORM)).view(n, h, w, c) * gamma + beta
            dy.masked_fill_(z.abs() < 1e-5, 0.0)
        state["dy"] = dy.to(dt)
    return state


def _prepare_tensors(case, seed):
    g = _generator(seed)
    spans, total = _offsets(case)
    shapes = _shapes(case)
    dt = DTYPES[case["param"].rstrip("m")]
    size = torch.zeros(total, device="cuda")              # the gradients' scale differs from tensor to tensor; 0 between tensors
    scales = np.exp(np.random.RandomState(seed % (1 << 32)).randn(len(spans)) * 0.7) * 2e-3
    for (at, k), s in zip(spans, scales):
        size[at:at + k] = float(s)
    draw_one = lambda: torch.randn(total, device="cuda", generator=g)  # noqa: E731
    flat = {"grad": (draw_one() * size).to(dt)}
    state = dict(case=case, flat=flat)
    if case["kind"] == "adamw":
        p = draw_one() * 0.05 * (size > 0)
        flat["param"] = p.to(dt)
        if case["param"].endswith("m"):
            flat["master"] = p
        m = draw_one() * size * 0.3
        r = (draw_one().abs() * 0.3 + 0.7) * size
        if case["bits"] == 8:
            flat["m8"], flat["m_scale"] = _quantised(m.view(-1, BLOCK))
            flat["r8"], flat["r_scale"] = _quantised(r.view(-1, BLOCK))
            flat["m8"], flat["r8"] = flat["m8"].view(-1), flat["r8"].view(-1)
        else:
            flat["m"], flat["v"] = m, r * r
        state["step"] = 100
    state["lists"] = {name: [t[at // BLOCK:at // BLOCK + (k + BLOCK - 1) // BLOCK] if name.endswith("_scale") else t[at:at + k].view(s)
                             for (at, k), s in zip(spans, shapes)] for name, t in flat.items()}
    return state


def prepare(case, seed):
    return _prepare_gn(case, seed) if case["kind"] == "gn" else _prepare_tensors(case, seed)


# ------------------------------------------------------------------------------------------------ the plain forms
def _act(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    return torch.where(z > 0, z, z * SLOPE) if act == "lrelu" else z


def _act_grad(z, act):
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.where(z > 0, 1.0, SLOPE) if act == "lrelu" else torch.ones_like(z)


def _plain_gn(state):
    case, x = state["case"], state["x"]
    n, c, groups = x.shape[0], x.shape[3], case["groups"]
    gamma, beta = state["gamma"], state["beta"]
    xf = x.float().view(n, -1, groups, c // groups)
    mean = xf.mean(dim=(1, 3), keepdim=True)
    xc = xf - mean
    rstd = torch.rsqrt((xc * xc).mean(dim=(1, 3), keepdim=True) + EPS_NORM)
    xhat = (xc * rstd).view(n, -1, c)
    z = xhat * gamma + beta
    y = _act(z, case["act"]).to(x.dtype).view_as(x)
    if not case["train"]:
        return y
    dz = state["dy"].float().view(n, -1, c) * _act_grad(z, case["act"])
    dgamma, dbeta = (dz * xhat).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    t = (dz * gamma).view_as(xf)
    xh = xhat.view_as(xf)
    dx = rstd * (t - t.mean(dim=(1, 3), keepdim=True) - xh * (t * xh).mean(dim=(1, 3), keepdim=True))
    return y, dx.to(x.dtype).view_as(x), dgamma, dbeta


def _plain_norm(grad):
    """(norm, factor) in 64 bits: the sum is long, and the factor decides roundings further on."""
    norm = grad.double().square().sum().sqrt()
    return norm, torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0).float()


def _plain_clip(state):
    grad = state["flat"]["grad"]
    norm, factor = _plain_norm(grad)
    grad.copy_(grad.float() * factor)
    return norm.float(), grad


def _mix(h):
    """Mixes the 32 bits of whole numbers held in int64."""
    h = ((h ^ (h >> 16)) * 0x9E3779B1) & 0xFFFFFFFF
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _xorshift(h):
    h = h ^ ((h << 13) & 0xFFFFFFFF)
    h = h ^ (h >> 17)
    return h ^ ((h << 5) & 0xFFFFFFFF)


def _random_bits(elements, step, device):
    """32 random bits for each element, from (SEED, step, number of its quad): one mix a quad, then a shift register."""
    key = torch.tensor((SEED + step * 0x9E3779B9) & 0xFFFFFFFF, device=device)
    a = _mix(torch.arange(elements // 4, device=device) + _mix(key) & 0xFFFFFFFF)
    b = _xorshift(a)
    c = _xorshift(b)
    return torch.stack([a, b, c, _xorshift(c)], dim=1).view(-1)


def _to_e4m3(x, rnd, floor):
    """x [blocks, BLOCK] -> (codes, scales): one power of two a block, such that its largest finite value is in (224, 448]; between two codes the
    16 random bits decide. floor: what is not zero does not become zero."""
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), 0.0).amax(1)
    f, e = torch.frexp(amax)                                        # amax = f * 2^e, f in [0.5, 1)
    k = torch.where(f > 0.875, e - 8, e - 9).clamp_min(-100)
    scale = torch.ldexp(torch.ones_like(amax), k)
    a = x.abs() * torch.ldexp(torch.ones_like(amax), -k)[:, None]
    low = a < 2.0 ** -6
    z = torch.where(low, a + 2.0 ** -6, a)
    ulp = torch.ldexp(torch.ones_like(z), torch.frexp(z)[1] - 4)
    q = torch.floor(z / ulp + rnd.float() * 2.0 ** -16) * ulp
    q = torch.where(low, q - 2.0 ** -6, q).clamp_max(448.0)
    if floor:
        q = torch.where(x > 0, q.clamp_min(2.0 ** -9), q)
    return torch.where(finite, torch.copysign(q, x), float("nan")).to(torch.float8_e4m3fn), scale


def _plain_adamw(state):
    case, f = state["case"], state["flat"]
    state["step"] += 1
    step = state["step"]
    g = f["grad"].float()
    out = {}
    if case["clip"]:
        norm, factor = _plain_norm(f["grad"])
        out["norm"] = norm.float()
        g = g * factor
    if case["bits"] == 8:
        m = (f["m8"].float().view(-1, BLOCK) * f["m_scale"][:, None]).view(-1)
        r = (f["r8"].float().view(-1, BLOCK) * f["r_scale"][:, None]).view(-1)
        m = m * BETA1 + g * (1 - BETA1)
        root = torch.sqrt((r * r) * BETA2 + (g * g) * (1 - BETA2))
        bits = _random_bits(m.numel(), step, m.device).view(-1, BLOCK)
        codes, scales = _to_e4m3(m.view(-1, BLOCK), bits & 0xFFFF, False)
        f["m8"].copy_(codes.view(-1))
        f["m_scale"].copy_(scales)
        codes, scales = _to_e4m3(root.view(-1, BLOCK), bits >> 16, True)
        f["r8"].copy_(codes.view(-1))
        f["r_scale"].copy_(scales)
    else:
        m = f["m"].mul_(BETA1).add_(g * (1 - BETA1))
        root = torch.sqrt(f["v"].mul_(BETA2).add_((g * g) * (1 - BETA2)))
    root = root / math.sqrt(1 - BETA2 ** step) + EPS
    p = f["master"] if "master" in f else f["param"].float()
    p = p * (1 - LR * DECAY) - (LR / (1 - BETA1 ** step)) * (m / root)
    if "master" in f:
        f["master"].copy_(p)
    f["param"].copy_(p)
    return _adamw_outputs(f, out)


def _adamw_outputs(f, out):
    """The updated buffers themselves; 8-bit states as the e4m3 values they are."""
    out.update({k: t for k, t in f.items() if k != "grad"})
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_gn(state):
    from coarse3d_amd import ops
    case = state["case"]
    y, mean, rstd = ops.group_norm(state["x"], case["groups"], state["gamma"], state["beta"], eps=EPS_NORM, act=case["act"], slope=SLOPE)
    if not case["train"]:
        return y
    dx, dgamma, dbeta = ops.group_norm_bwd(state["dy"], state["x"], mean, rstd, state["gamma"], state["beta"], act=case["act"], slope=SLOPE)
    return y, dx, dgamma, dbeta


def _own_clip(state):
    from coarse3d_amd import ops
    return ops.clip_grad_norm_(state["lists"]["grad"], MAX_NORM), state["flat"]["grad"]


def _own_adamw(state):
    from coarse3d_amd import ops
    case, t = state["case"], state["lists"]
    state["step"] += 1
    out, scale = {}, None
    if case["clip"]:
        out["norm"], scale = ops.grad_norm(t["grad"], MAX_NORM)
    more = dict(step=state["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, grad_scale=scale, masters=t.get("master"))
    if case["bits"] == 8:
        ops.adamw8_step(t["param"], t["grad"], t["m8"], t["m_scale"], t["r8"], t["r_scale"], seed=SEED, **more)
    else:
        ops.adamw_step(t["param"], t["grad"], t["m"], t["v"], **more)
    return _adamw_outputs(state["flat"], out)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own_gn(state) if kind == "gn" else _own_clip(state) if kind == "clip" else _own_adamw(state)
    return _plain_gn(state) if kind == "gn" else _plain_clip(state) if kind == "clip" else _plain_adamw(state)


# ------------------------------------------------------------------------------------------------ work and the definition in 64 bits
def work(case):
    if case["kind"] == "gn":
        n = case["n"] * case["h"] * case["w"] * case["c"]
        e = DTYPES[case["dtype"]].itemsize
        if case["train"]:
            return {"bytes": 4 * n * e + 16 * case["c"], "flops": 24 * n}
        return {"bytes": 2 * n * e + 8 * case["c"], "flops": 8 * n}
    n = sum(math.prod(s) for s in _shapes(case))
    e = DTYPES[case["param"].rstrip("m")].itemsize
    if case["kind"] == "clip":
        return {"bytes": 2 * n * e, "flops": 3 * n}
    moved = e + 2 * e + (8 if case["param"].endswith("m") else 0) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    if case["param"].endswith("m"):
        moved -= e                                          # the 16-bit parameter is written only
    return {"bytes": n * moved, "flops": (16 if case["bits"] == 32 else 40) * n}


def _exact_gn(case, state):
    n, c, groups = case["n"], case["c"], case["groups"]
    x = state["x"].to(torch.float64).reshape(n, -1, groups, c // groups)
    gamma, beta = state["gamma"].double().view(groups, -1), state["beta"].double().view(groups, -1)
    count = x.shape[1] * x.shape[3]
    mu = x.sum((1, 3), keepdim=True) / count
    sigma = torch.sqrt(((x - mu) ** 2).sum((1, 3), keepdim=True) / count + EPS_NORM)
    u = (x - mu) / sigma
    z = gamma * u + beta
    if case["act"] == "silu":
        gate = 1 / (1 + torch.exp(-z))
        y, slope = z * gate, gate + z * gate * (1 - gate)
    elif case["act"] == "lrelu":
        slope = torch.where(z > 0, torch.ones_like(z), torch.full_like(z, SLOPE))
        y = z * slope
    else:
        y, slope = z, torch.ones_like(z)
    y = y.view(n, case["h"], case["w"], c)
    if not case["train"]:
        return y
    d = state["dy"].to(torch.float64).view_as(x) * slope
    dgamma, dbeta = (d * u).sum((0, 1)).reshape(-1), d.sum((0, 1)).reshape(-1)
    d = d * gamma
    first, second = d.sum((1, 3), keepdim=True) / count, (d * u).sum((1, 3), keepdim=True) / count
    return y, ((d - first - u * second) / sigma).view_as(y), dgamma, dbeta


def _exact_bits(quads, step):
    """The rounding's random bits [quads, 4], in numpy's 32-bit arithmetic, which wraps by itself."""
    one = np.uint32

    def mixed(v):
        v = v ^ (v >> one(16))
        v = v * one(0x9E3779B1)
        v = v ^ (v >> one(15))
        v = v * one(0xBB67AE85)
        return v ^ (v >> one(16))

    key = mixed(np.array([(SEED + step * 0x9E3779B9) % 2 ** 32], dtype=np.uint32))
    v = mixed(np.arange(quads, dtype=np.uint64).astype(np.uint32) + key)
    cols = [v]
    for _ in range(3):
        v = v ^ (v << one(13))
        v = v ^ (v >> one(17))
        v = v ^ (v << one(5))
        cols.append(v)
    return np.stack(cols, 1)


def _exact_codes(x, rnd, floor):
    """Stochastic rounding to e4m3 from its definition: the neighbour above is taken where the fraction plus rnd / 2^16 reaches one."""
    top = x.abs().amax(1, keepdim=True)
    k = torch.ceil(torch.log2(top.clamp_min(1e-60) / 448.0)).clamp_min(-100.0)
    a = x.abs() / torch.exp2(k)
    e = torch.floor(torch.log2(a.clamp_min(1e-30))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    down = torch.floor(a / step)
    q = (down + ((a / step - down) + rnd / 65536.0 >= 1.0)) * step
    if floor:
        q = torch.where(x > 0, torch.clamp(q, min=2.0 ** -9), q)
    return (torch.sign(x) * q.clamp(max=448.0)).view(-1), torch.exp2(k).view(-1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "gn":
        return _exact_gn(case, state)
    f = {k: t.double() for k, t in state["flat"].items()}
    g = f["grad"]
    norm = torch.sqrt((g * g).sum())
    factor = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    if case["kind"] == "clip":
        return norm, g * factor
    out = {}
    if case["clip"]:
        out["norm"], g = norm, g * factor
    t = state["step"] + 1
    eight = case["bits"] == 8
    if eight:
        m = (f["m8"].view(-1, BLOCK) * f["m_scale"].view(-1, 1)).view(-1)
        v = (f["r8"].view(-1, BLOCK) * f["r_scale"].view(-1, 1)).view(-1) ** 2
    else:
        m, v = f["m"], f["v"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = f.get("master", f["param"])
    p = (1 - LR * DECAY) * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    out["param"] = p
    if "master" in f:
        out["master"] = p
    if eight:
        rnd = torch.from_numpy(_exact_bits(g.numel() // 4, t).astype(np.int64)).to(g.device).view(-1, BLOCK)
        out["m8"], out["m_scale"] = _exact_codes(m.view(-1, BLOCK), rnd % 65536, False)
        out["r8"], out["r_scale"] = _exact_codes(torch.sqrt(v).view(-1, BLOCK), rnd // 65536, True)
    else:
        out["m"], out["v"] = m, v
    return out
