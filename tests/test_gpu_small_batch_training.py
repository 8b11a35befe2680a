"""The operators of small-batch training as a user has them: ``optim.AdamW`` / ``clip_grad_norm_``, ``group_norm.GroupNormAct``,
``ProjectionV1(norm="group")``, ``TrainStep`` with the many-tensor optimiser, and a run of them together."""
import copy

import pytest
import torch
import torch.nn as nn

import weights as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def tensors(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    shapes = [(16, 8, 3, 3), (16,), (8, 4, 3, 3), (300, 7), (1,), (0, 4), (5, 11)]
    ps = [nn.Parameter((torch.randn(s, generator=g) * 0.1).to(DEV, dtype)) for s in shapes]
    ps[2].data = ps[2].data.contiguous(memory_format=torch.channels_last)
    return ps


def set_grads(ps, seed, skip=(), scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    for i, p in enumerate(ps):
        x = (torch.randn(p.shape, generator=g) * scale).to(DEV, p.dtype)
        p.grad = None if i in skip else x           # contiguous, also where the parameter is channels last


def test_adamw_follows_torch_over_groups_schedules_and_missing_gradients():
    from coarse3d_amd.optim import AdamW
    a, b = tensors(1), [nn.Parameter(p.detach().double().clone()) for p in tensors(1)]
    groups = lambda ps: [dict(params=ps[:3]), dict(params=ps[3:], lr=3e-3, weight_decay=0.0, betas=(0.8, 0.99))]  # noqa: E731
    oa, ob = AdamW(groups(a), lr=1e-3), torch.optim.AdamW(groups(b), lr=1e-3)
    sa, sb = torch.optim.lr_scheduler.StepLR(oa, 3, 0.5), torch.optim.lr_scheduler.StepLR(ob, 3, 0.5)
    for t in range(9):
        skip = () if t in (0, 6, 7) else (1, 3) if t < 4 else (0, 1, 6)
        set_grads(a, 50 + t, skip)
        for p, q in zip(a, b):
            q.grad = None if p.grad is None else p.grad.double()
        versions = [p._version for p in a]
        oa.step()
        ob.step()
        assert all(p._version > v for i, (p, v) in enumerate(zip(a, versions)) if i not in skip)
        sa.step()
        sb.step()
    for p, q in zip(a, b):
        # nine steps of at most 3 roundings of the value and 40 u of an update that is at most 5 lr (test_gpu_adamw_many.py)
        assert ((p.double() - q).abs() <= 9 * (3 * U * q.abs() + 40 * U * 5 * 3e-3) + 1e-12).all()
    da, db = oa.state_dict(), ob.state_dict()
    assert da["state"].keys() == db["state"].keys()
    for i in db["state"]:
        assert float(da["state"][i]["step"]) == float(db["state"][i]["step"])
        assert set(da["state"][i]) == set(db["state"][i])


def test_checkpoints_move_between_torch_and_here():
    from coarse3d_amd.optim import AdamW
    a = tensors(2)
    oa = AdamW(a, lr=2e-3)
    for t in range(4):
        set_grads(a, 70 + t, skip=(3,) if t == 1 else ())
        oa.step()
    b = [nn.Parameter(p.detach().clone()) for p in a]
    ob = torch.optim.AdamW(b, lr=1.0)
    sd = copy.deepcopy(oa.state_dict())
    sd.pop("state_bits")
    ob.load_state_dict(sd)
    c = [nn.Parameter(p.detach().clone()) for p in a]
    oc = AdamW(c, lr=5.0)
    oc.load_state_dict(ob.state_dict())
    assert oc.param_groups[0]["lr"] == 2e-3
    set_grads(a, 99)
    for q, r, p in zip(b, c, a):
        q.grad, r.grad = p.grad.clone(), p.grad.clone()
    for o in (oa, ob, oc):
        o.step()
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, r)
        assert ((p - q).abs() <= 4 * U * q.abs() + 40 * U * 2e-3 * 5).all()
    with pytest.raises(ValueError, match="8-bit states"):
        AdamW(c, state_bits=8).load_state_dict(oa.state_dict())
    with pytest.raises(ValueError, match="parameter groups differ"):
        oc.load_state_dict(AdamW(a[:3]).state_dict())


@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, False)])
def test_8bit_states_resume_bit_for_bit(dtype, master):
    from coarse3d_amd.optim import AdamW
    a = tensors(3, dtype)
    make = lambda ps: AdamW(ps, lr=1e-3, state_bits=8, master_weights=master, max_grad_norm=0.05, seed=4)  # noqa: E731
    oa = make(a)
    for t in range(6):
        if t == 3:
            b = [nn.Parameter(p.detach().clone()) for p in a]
            ob = make(b)
            ob.load_state_dict(copy.deepcopy(oa.state_dict()))
        set_grads(a, 30 + t, skip=(2,) if t == 1 else ())
        if t >= 3:
            for q, p in zip(b, a):
                q.grad = p.grad.clone()
            ob.step()
        oa.step()
        if t >= 3:
            assert torch.equal(ob.last_grad_norm, oa.last_grad_norm)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    sa, sb = oa.state_dict()["state"], ob.state_dict()["state"]
    assert sa.keys() == sb.keys()
    for i in sa:
        assert set(sa[i]) == {"step", "exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale"} | ({"master"} if master else set())
        for k in sa[i]:
            raw = lambda x: x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x  # noqa: E731
            assert torch.equal(raw(sa[i][k]), raw(sb[i][k])), (i, k)
    if master:
        assert all(torch.equal(p, oa.state[p]["master"].to(dtype)) for p in a)


def test_clipping_on_load_equals_clipping_ahead():
    from coarse3d_amd import optim
    a, b = tensors(5), [nn.Parameter(p.detach().clone()) for p in tensors(5)]
    oa, ob = optim.AdamW(a, lr=1e-3, max_grad_norm=0.3), optim.AdamW(b, lr=1e-3)
    for t in range(3):
        set_grads(a, 200 + t, scale=0.1)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        before = [p.grad.clone() for p in a]
        oa.step()
        assert all(torch.equal(p.grad, g) for p, g in zip(a, before))
        want = torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for g in before]))
        got = optim.clip_grad_norm_(b, 0.3)
        assert abs(float(got / want) - 1) <= 2 * U and torch.equal(got, oa.last_grad_norm) and float(want) > 0.3
        ob.step()
    # the same factor, applied to the gradient and rounded once either way
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    mixed = [nn.Parameter(torch.ones(5, device=DEV)), nn.Parameter(torch.ones(5, device=DEV, dtype=torch.bfloat16))]
    om = optim.AdamW(mixed, max_grad_norm=1.0)
    for p in mixed:
        p.grad = torch.full_like(p, 2.0)
    om.step()
    assert abs(float(om.last_grad_norm) - 40 ** 0.5) < 1e-5
    with pytest.raises(ValueError, match="several types"):
        optim.clip_grad_norm_(mixed, 1.0)
    assert float(optim.clip_grad_norm_([nn.Parameter(torch.ones(2, device=DEV))], 1.0)) == 0.0


@pytest.mark.parametrize("capturable", [False, True])
def test_a_copied_or_saved_optimiser_goes_on_alike(capturable):
    import copy
    import io
    from coarse3d_amd.optim import AdamW
    torch.manual_seed(6)
    net = nn.Sequential(nn.Linear(40, 33), nn.Linear(33, 7)).to(DEV)
    opt = AdamW(net.parameters(), lr=1e-2, state_bits=8, max_grad_norm=0.7, capturable=capturable, seed=5)
    x = torch.randn(9, 40, device=DEV)

    def step(n, o, which=slice(None)):
        for p in n.parameters():
            p.grad = None
        n(x).square().sum().backward()
        for p in list(n.parameters())[which]:
            p.grad = None
        o.step()
    step(net, opt, slice(0, 1))                    # (two cohorts)
    step(net, opt, slice(0, 0))
    file = io.BytesIO()
    torch.save((net, opt), file)                   # (pickle by itself cannot take torch's 8-bit floats)
    file.seek(0)
    others = [copy.deepcopy((net, opt)), torch.load(file, weights_only=False)]
    for _ in range(3):
        step(net, opt, slice(0, 0))
    for n, o in others:
        for _ in range(3):
            step(n, o, slice(0, 0))
        assert all(torch.equal(a, b) for a, b in zip(net.parameters(), n.parameters()))
        assert [float(v["step"]) for v in o.state_dict()["state"].values()] == [float(v["step"]) for v in opt.state_dict()["state"].values()]


def test_optimiser_refusals():
    from coarse3d_amd.optim import AdamW
    p = [nn.Parameter(torch.ones(3, device=DEV))]
    for kw in (dict(state_bits=4), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(max_grad_norm=-1.0), dict(weight_decay=float("nan"))):
        with pytest.raises(ValueError):
            AdamW(p, **kw)
    q = nn.Parameter(torch.ones(4, 4))
    q.grad = torch.ones(4, 4)
    with pytest.raises(ValueError, match="not on a GPU"):
        AdamW([q]).step()
    e = nn.Embedding(5, 3, sparse=True).to(DEV)
    e(torch.tensor([1], device=DEV)).sum().backward()
    with pytest.raises(RuntimeError, match="sparse"):
        AdamW(e.parameters()).step()
    o = AdamW(p)
    assert o.step() is None and not o.state_dict()["state"]                   # no gradients: nothing happens


def test_step_between_forward_and_backward_is_noticed():
    """The kernels write through raw pointers; autograd has to learn of it all the same."""
    from coarse3d_amd.optim import AdamW
    w = nn.Parameter(torch.randn(8, 8, device=DEV))
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    y = (x @ w).square().sum()
    w.grad = torch.ones_like(w)
    AdamW([w], lr=0.1).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits,norm", [(8, 0.5), (32, None)])
def test_captured_training_step_equals_the_eager_one(bits, norm):
    """TrainStep(graph=True) with the many-tensor optimiser: losses, parameters and states of replayed steps equal the steps issued launch
    by launch, bit for bit, over a learning-rate schedule and a checkpoint round trip."""
    from coarse3d_amd.optim import AdamW
    from coarse3d_amd.pc_processor.models import SalsaNextProto
    from coarse3d_amd.trainer import TrainStep
    b, h, w, ncls = 2, 32, 128, 20
    batches = [W.synthetic_batch(b, h, w, ncls, 300 + i, 0.02, gh=8, gw=16) for i in range(9)]
    runs = []
    for warm in (1000, 2):
        torch.manual_seed(51)
        m = SalsaNextProto(5, ncls, 20, 0, use_prototype=True).to(DEV).train()
        opt = AdamW(m.parameters(), lr=2e-3, state_bits=bits, max_grad_norm=norm, capturable=True, seed=9)
        sched = torch.optim.lr_scheduler.ExponentialLR(opt, 0.9)
        ts = TrainStep(m, ncls, proto_loss=True, num_anchor=32, graph=True, graph_warmup=warm, optimizer=opt, scheduler=sched)
        torch.manual_seed(52)
        losses = []
        for i, (x, tr, ev) in enumerate(batches):
            if i == 6:
                gen = opt.generation
                ts.flush()
                opt.load_state_dict(opt.state_dict())
                assert opt.generation == gen + 1
            res = ts.step(x.to(DEV), tr.to(DEV), ev.to(DEV), epoch=10)
            losses.append({k: res[k].clone() for k in ("loss", "ce", "lov", "contrast")})
            torch.cuda.synchronize()
        ts.flush()
        runs.append((losses, {k: v.detach().clone() for k, v in m.state_dict().items()}, opt.state_dict(), ts))
    assert runs[0][3]._captures == 0 and runs[1][3]._captures == 2 and runs[1][3]._replays >= 5
    for i, (la, lb) in enumerate(zip(runs[0][0], runs[1][0])):
        for k in la:
            assert torch.equal(la[k], lb[k]), (i, k)
    for k, v in runs[0][1].items():
        assert torch.equal(v, runs[1][1][k]), k
    sa, sb = runs[0][2]["state"], runs[1][2]["state"]
    assert sa.keys() == sb.keys() and len(sa) == 192
    for i in sa:
        assert float(sa[i]["step"]) == float(sb[i]["step"]) == len(batches)
        for k in sa[i]:
            raw = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t  # noqa: E731
            assert torch.equal(raw(sa[i][k]), raw(sb[i][k])), (i, k)


def test_a_captured_step_needs_a_capturable_optimiser():
    from coarse3d_amd.optim import AdamW
    from coarse3d_amd.pc_processor.models import SalsaNextProto
    from coarse3d_amd.trainer import TrainStep
    m = SalsaNextProto(5, 20, 20, 0, use_prototype=True).to(DEV).train()
    ts = TrainStep(m, 20, graph=True, optimizer=AdamW(m.parameters()))
    x, tr, ev = W.synthetic_batch(2, 32, 128, 20, 1, 0.02, gh=8, gw=16)
    with pytest.raises(RuntimeError, match="capturable"):
        ts.step(x.to(DEV), tr.to(DEV), ev.to(DEV), epoch=10)


def rel(a, b):
    return float((a.detach().double().cpu() - b.detach().double().cpu()).norm() / b.detach().double().cpu().norm())


@pytest.mark.parametrize("channels_last", [False, True])
@pytest.mark.parametrize("act", ["none", "lrelu", "silu"])
def test_group_norm_module_like_torch(act, channels_last):
    from coarse3d_amd.group_norm import GroupNormAct
    torch.manual_seed(3)
    m = GroupNormAct(4, 24, act=act, negative_slope=0.2)
    with torch.no_grad():
        m.weight.uniform_(0.5, 1.5)
        m.bias.normal_(std=0.3)
    ref = nn.Sequential(nn.GroupNorm(4, 24), {"none": nn.Identity(), "lrelu": nn.LeakyReLU(0.2), "silu": nn.SiLU()}[act]).double()
    ref[0].load_state_dict({k: v.double() for k, v in m.state_dict().items()})
    x = torch.randn(3, 24, 9, 21)
    if channels_last:
        x = x.contiguous(memory_format=torch.channels_last)
    dy = torch.randn(3, 24, 9, 21)
    xr = x.double().requires_grad_(True)
    z = ref[0](xr)
    dy = torch.where(z.detach().abs() < 1e-4, 0.0, dy)       # no gradient within rounding of the kink
    (ref(xr) * dy.double()).sum().backward()
    m.to(DEV)
    xd = x.to(DEV).requires_grad_(True)
    y = m(xd)
    (y * dy.to(DEV).float()).sum().backward()
    assert y.shape == x.shape
    # sums of at most 300 terms in fp32: 300 u in the mean, as much in the variance's root, 5 sigma at most (test_gpu_group_norm.py)
    tol = 2000 * U
    assert rel(y, ref(xr)) < tol and rel(xd.grad, xr.grad) < tol
    assert rel(m.weight.grad, ref[0].weight.grad) < tol and rel(m.bias.grad, ref[0].bias.grad) < tol
    y = m(xd)
    g, = torch.autograd.grad(y.sum(), xd, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(ValueError):
        m(x.to(DEV)[:, :8])
    with pytest.raises(ValueError):
        GroupNormAct(5, 24)


def test_group_norm_gradients_only_where_asked():
    from coarse3d_amd.group_norm import group_norm_act
    x = torch.randn(2, 5, 7, 16, device=DEV)
    w = torch.ones(16, device=DEV, requires_grad=True)
    group_norm_act(x, 4, w, None).square().sum().backward()
    assert w.grad is not None and torch.isfinite(w.grad).all()
    xg = x.clone().requires_grad_(True)
    group_norm_act(xg, 4).sum().backward()                    # an expanded gradient, no affine
    assert torch.isfinite(xg.grad).all()
    with torch.no_grad():
        assert not group_norm_act(x, 4, w).requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_group_norm_module_in_16_bits(dtype):
    from coarse3d_amd.group_norm import GroupNormAct
    torch.manual_seed(4)
    m = GroupNormAct(4, 24, act="silu").to(DEV, dtype)
    x = torch.randn(2, 24, 6, 10, device=DEV, dtype=dtype, requires_grad=True)
    y = m(x)
    y.square().sum().backward()
    ref = nn.functional.silu(nn.functional.group_norm(x.detach().double(), 4))
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    assert y.dtype == dtype and ((y.double() - ref).abs() <= 1.01 * half * ref.abs() + 2000 * U).all()
    assert x.grad.dtype == dtype and m.weight.grad.dtype == dtype and torch.isfinite(m.weight.grad).all()


def test_projector_with_group_norm_like_torch():
    from coarse3d_amd.pc_processor.models import ProjectionV1
    torch.manual_seed(6)
    proj = ProjectionV1(48, 32, norm="group", num_groups=6)
    with torch.no_grad():
        proj.proj[1].weight.uniform_(0.5, 1.5)
        proj.proj[1].bias.normal_(std=0.3)
    ref = nn.Sequential(nn.Conv2d(48, 48, 1), nn.GroupNorm(6, 48), nn.LeakyReLU(), nn.Conv2d(48, 32, 1)).double()
    ref.load_state_dict({k[len("proj."):]: v.double() for k, v in proj.state_dict().items()})
    x, dy = torch.randn(2, 48, 8, 64), torch.randn(2, 32, 8, 64)
    xr = x.double().requires_grad_(True)
    (ref(xr) * dy.double()).sum().backward()
    proj.to(DEV).train()
    xd, dyd = x.to(DEV).requires_grad_(True), dy.to(DEV)
    keep = dyd.clone()
    y = proj(xd)
    y.backward(dyd)
    assert torch.equal(dyd, keep)
    # the engine's bound for this module (test_gpu_heads.py)
    assert rel(y, ref(xr)) < 1e-4 and rel(xd.grad, xr.grad) < 1e-4
    for (n, p), (_, pr) in zip(proj.proj.named_parameters(), ref.named_parameters()):
        assert rel(p.grad, pr.grad) < 1e-4, n
    with torch.no_grad():
        y2 = proj(x.to(DEV))
        assert not y2.requires_grad and rel(y2, ref(x.double())) < 1e-4
        proj.eval()
        assert torch.equal(proj(x.to(DEV)), y2)               # no running statistics: evaluation is the same function
        # and one scan does not depend on what else is in the batch
        assert rel(proj(x.to(DEV)[:1]), y2[:1]) < 1e-5
    for kw in (dict(norm="layer"), dict(norm="group", num_groups=7)):
        with pytest.raises(ValueError):
            ProjectionV1(48, 32, **kw)


@pytest.mark.parametrize("bits", [8, 32])
def test_the_operators_together(bits):
    """A projector with group norm behind a group-normed layer, trained on one scan a step with clipping and the many-tensor optimiser,
    next to the same in float64 torch.  With states in 32 bits the parameters stay within rounding; in 8 bits the first step (from
    zero states) does, and afterwards a moment and a root are each off by one code step at most, an eighth: the update by 9/8 : 7/8 - 1
    < 0.3 of it."""
    from coarse3d_amd.group_norm import GroupNormAct
    from coarse3d_amd.optim import AdamW
    from coarse3d_amd.pc_processor.models import ProjectionV1
    torch.manual_seed(8)
    ours = nn.Sequential(GroupNormAct(8, 32, act="silu"), ProjectionV1(32, 16, norm="group", num_groups=8))
    ref = nn.Sequential(nn.GroupNorm(8, 32), nn.SiLU(), nn.Conv2d(32, 32, 1), nn.GroupNorm(8, 32), nn.LeakyReLU(), nn.Conv2d(32, 16, 1)).double()
    with torch.no_grad():
        for p, q in zip(ours.parameters(), ref.parameters()):
            q.copy_(p)
    ours.to(DEV).train()
    lr, clip, steps = 1e-3, 0.5, 6
    oa = AdamW(ours.parameters(), lr=lr, state_bits=bits, max_grad_norm=clip)
    ob = torch.optim.AdamW(ref.parameters(), lr=lr)
    for t in range(steps):
        x, dy = torch.randn(1, 32, 16, 48), torch.randn(1, 16, 16, 48)
        oa.zero_grad()
        ob.zero_grad()
        (ours(x.to(DEV)) * dy.to(DEV)).sum().backward()
        (ref(x.double()) * dy.double()).sum().backward()
        if t == 0:
            for p, q in zip(ours.parameters(), ref.parameters()):
                assert rel(p.grad, q.grad) < 1e-4
        norm = nn.utils.clip_grad_norm_(ref.parameters(), clip)
        oa.step()
        ob.step()
        if t == 0:
            assert abs(float(oa.last_grad_norm) / float(norm) - 1) < 1e-4
        for p, q in zip(ours.parameters(), ref.parameters()):
            d = (p.detach().double().cpu() - q.detach()).abs()
            # the first step moves every parameter by lr times the sign of its gradient: gradients within their own error of zero may differ
            loose = 2 * lr * (t + 1)
            assert float(d.max()) <= loose + 1e-6
            tight = (1e-2 if bits == 32 or t == 0 else 0.3) * lr * (t + 1)
            assert float((d > tight).double().mean()) < 0.03, (t, tuple(p.shape), float(d.max()))
