"""What the group-norm and many-tensor entry points refuse, checked on the host before anything is launched (no GPU needed: a call
whose only fault is that its tensors are on the CPU says so, and says it last)."""
import ctypes

import pytest
import torch


def _ops():
    from coarse3d_amd import ops
    return ops


def test_record_layouts_match_the_header():
    from coarse3d_amd import _lib as L
    out = (ctypes.c_int32 * 2)()
    assert L.lib().c3d_opt_abi_sizes(out) == 0
    assert list(out) == [ctypes.sizeof(L.OptTensor), ctypes.sizeof(L.AdamWDesc)]
    assert _ops().ADAMW8_BLOCK == 256


@pytest.mark.parametrize("kw,match", [
    (dict(groups=3), "divide"), (dict(groups=0), "divide"), (dict(act="gelu"), "act"), (dict(slope=-0.1), "slope"), (dict(slope=float("nan")), "slope"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(gamma=torch.ones(7)), "gamma"), (dict(beta=torch.ones(8).double()), "beta"),
    (dict(gamma=torch.ones(16)[::2]), "gamma"), (dict(x=torch.ones(2, 3, 8).double()), "fp32"), (dict(x=torch.ones(8)), r"\[N, ..., C\]"),
    (dict(x=torch.ones(2, 8, 3).transpose(1, 2)), "side by side"), (dict(x=torch.ones(2, 4, 6, 8)[:, :, ::2].transpose(1, 2)), "one stride apart"),
    (dict(x=torch.ones(1, 1, 8).expand(2, 3, 8)), "one stride apart"), (dict(), "on cpu"),
])
def test_group_norm_refusals(kw, match):
    kw = dict(dict(x=torch.ones(2, 3, 8), groups=2), **kw)
    with pytest.raises(ValueError, match=match):
        _ops().group_norm(kw.pop("x"), kw.pop("groups"), **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(dy=torch.ones(2, 3, 4)), "dy"), (dict(dy=torch.ones(2, 3, 8).half()), "dy"), (dict(mean=torch.ones(2, 3)), "rstd"), (dict(mean=torch.ones(3, 2)), "mean"),
    (dict(rstd=torch.ones(2, 2).double()), "rstd"), (dict(mean=torch.ones(2, 3), rstd=torch.ones(2, 3)), "divide"), (dict(act="relu6"), "act"), (dict(), "on cpu"),
])
def test_group_norm_bwd_refusals(kw, match):
    kw = dict(dict(dy=torch.ones(2, 3, 8), x=torch.ones(2, 3, 8), mean=torch.ones(2, 2), rstd=torch.ones(2, 2)), **kw)
    with pytest.raises(ValueError, match=match):
        _ops().group_norm_bwd(**kw)


def _lists(n=3, dtype=torch.float32):
    return [torch.ones(4, 5, dtype=dtype) for _ in range(n)]


def test_list_refusals():
    ops = _ops()
    step = lambda *a, **k: ops.adamw_step(*a, **dict(dict(step=1, lr=1e-3), **k))  # noqa: E731
    L = _lists
    with pytest.raises(ValueError, match="on cpu"):
        step(L(), L(), L(), L())
    with pytest.raises(ValueError, match="has 2 tensors, params has 3"):
        step(L(), L(2), L(), L())
    with pytest.raises(ValueError, match=r"exp_avgs\[1\] differs in shape or strides from params"):
        step(L(), L(), [torch.ones(4, 5), torch.ones(5, 4), torch.ones(4, 5)], L())
    with pytest.raises(ValueError, match=r"grads\[0\] differs in shape or strides"):
        step(L(1), [torch.ones(5, 4).t()], L(1), L(1))
    with pytest.raises(ValueError, match=r"params\[2\] has another type"):
        step(L(2) + L(1, torch.float16), L(), L(), L())
    with pytest.raises(ValueError, match="share memory"):
        x = L(1)
        step(x + x, L(2), L(2), L(2))
    with pytest.raises(ValueError, match="share memory"):                     # partly
        x = torch.ones(30)
        step([x[:20], x[10:]], [torch.ones(20), torch.ones(20)], [torch.ones(20), torch.ones(20)], [torch.ones(20), torch.ones(20)])
    with pytest.raises(ValueError, match="share memory"):                     # a gradient inside a written state
        x = L(1)
        step(L(1), x, x, L(1))
    with pytest.raises(ValueError, match="gaps or overlap"):
        step([torch.ones(4, 10)[:, ::2]], L(1), L(1), L(1))
    with pytest.raises(ValueError, match="gaps or overlap"):
        ops.clip_grad_norm_([torch.ones(1).expand(4)], 1.0)
    with pytest.raises(TypeError, match=r"grads\[1\] is not a tensor"):
        ops.grad_norm([torch.ones(3), None])
    with pytest.raises(TypeError, match="is a list of tensors"):
        ops.grad_norm(torch.ones(3))
    with pytest.raises(ValueError, match="no tensors"):
        ops.grad_norm([])
    with pytest.raises(ValueError, match="dense tensor"):
        ops.grad_norm([torch.ones(3).to_sparse()])
    with pytest.raises(ValueError, match="dense tensor"):
        ops.grad_norm([torch.ones(3, device="meta")])
    with pytest.raises(ValueError, match="share memory"):
        x = torch.ones(3)
        ops.clip_grad_norm_([x, x], 1.0)


def test_scale_lists_of_the_8bit_states_are_checked():
    ops = _ops()
    f8 = lambda n: [torch.zeros(n, dtype=torch.uint8).view(torch.float8_e4m3fn)]  # noqa: E731
    for scales in (torch.ones(2), torch.ones(4), torch.ones(6)[::2]):
        with pytest.raises(ValueError, match="exp_avg_scales.*one scale for each block"):
            ops.adamw8_step([torch.ones(513)], [torch.ones(513)], f8(513), [scales], f8(513), [torch.ones(3)], step=1, lr=1e-3)


def test_the_library_refuses_what_the_wrappers_would_not_send():
    from coarse3d_amd import _lib as L
    lib = L.lib()
    rec = (L.OptTensor * 1)()
    rec[0].n = 8
    d = L.AdamWDesc()
    assert lib.c3d_adamw_step(rec, 1, None, None) != 0
    d.state_bits, d.step, d.beta1, d.beta2 = 32, 1, 0.9, 0.999
    assert lib.c3d_adamw_step(rec, 1, ctypes.byref(d), None) != 0 and b"null pointer" in lib.c3d_last_error()
    for field, value in (("state_bits", 4), ("param_type", 3), ("grad_type", 2), ("has_master", 1), ("beta1", 1.0), ("beta2", -0.1), ("eps", -1.0), ("step", 0)):
        e = L.AdamWDesc.from_buffer_copy(d)
        setattr(e, field, value)
        assert lib.c3d_adamw_step(rec, 1, ctypes.byref(e), None) == 2, field
    rec[0].n = -1
    assert lib.c3d_adamw_step(rec, 1, ctypes.byref(d), None) == 2
    assert lib.c3d_grad_norm(rec, 1, 0, 1.0, None, 8, 8, None) == 2
    rec[0].n = 8
    rec[0].ptr[1] = 16
    assert lib.c3d_grad_norm(rec, 1, 3, 1.0, 8, 8, 8, None) == 2 and lib.c3d_grad_norm(rec, 1, 0, float("nan"), 8, 8, 8, None) == 2
    rec[0].n = 1 << 20
    assert lib.c3d_grad_norm(rec, 1, 0, 1.0, None, 8, 8, None) == 2 and lib.c3d_clip_grads(rec, 1, 0, 1.0, None, 8, 8, None) == 2
    gn = lambda **k: lib.c3d_group_norm(*dict(dict(x=16, ns=24, ps=8, N=2, HW=3, C=8, G=2, type=0, ga=None, be=None, eps=1e-5, act=1, slope=0.01, y=16,  # noqa: E731
                                                   mean=16, rstd=16, ws=16, s=None), **k).values())
    for k in (dict(G=3), dict(N=-1), dict(HW=-1), dict(type=5), dict(act=9), dict(slope=2.0), dict(eps=-1.0), dict(x=None), dict(ws=None, HW=100000, ns=800000), dict(ps=7), dict(ns=23)):
        assert gn(**k) == 2, k
    assert gn(N=0) == 0 and gn(HW=0) == 0


def test_negative_views_and_tiny_eps_are_refused():
    """A tensor whose memory holds the negative of its values, and an eps that the reciprocal would take for 0."""
    ops = _ops()
    neg = torch._neg_view(torch.ones(4, 5))
    with pytest.raises(ValueError, match=r"grads\[0\] is not a dense tensor"):
        ops.grad_norm([neg])
    with pytest.raises(ValueError, match="x is not a dense tensor"):
        ops.group_norm(torch._neg_view(torch.ones(2, 3, 8)), 2)
    for eps, match in ((1e-39, "2\\^-126"), (1e-60, "2\\^-126"), (float("nan"), "2\\^-126"), (-1e-8, "2\\^-126"), (0.0, "on cpu"), (2.0 ** -126, "on cpu")):
        with pytest.raises(ValueError, match=match):
            ops.adamw_step(_lists(), _lists(), _lists(), _lists(), step=1, lr=1e-3, eps=eps)


def test_gradients_are_collected_with_their_types():
    from coarse3d_amd import _lib as L
    ps = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(2, dtype=torch.bfloat16)), torch.nn.Parameter(torch.ones(1))]
    ps[0].grad, ps[1].grad = torch.ones(3), torch.ones(2, dtype=torch.bfloat16)
    grads, types = L.native().grads_of(ps)
    assert grads[0] is ps[0].grad and grads[1] is ps[1].grad and grads[2] is None
    assert len(types) == 3 and types[2] == 255 and len(set(types)) == 3
    assert L.native().grads_of([]) == ([], b"")
    with pytest.raises(TypeError):
        L.native().grads_of([1])


def test_optimiser_replans_when_its_parameters_change():
    """Parameters put in another's place are stepped (here: refused for being on the CPU) with states of their own; checkpoints with options
    that this optimiser lacks are refused."""
    from coarse3d_amd.optim import AdamW
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(2)]
    opt = AdamW(ps, lr=0.1)
    for p in ps:
        p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="on cpu"):
        opt.step()
    new = torch.nn.Parameter(torch.ones(5))
    new.grad = torch.ones(5)
    opt.param_groups[0]["params"][1] = new
    with pytest.raises(ValueError, match="on cpu"):
        opt.step()
    assert any(p is new for run in opt._plan[2] for p in run[3]) and opt.state[new]["exp_avg"].shape == (5,)
    sd = torch.optim.AdamW(ps, amsgrad=True).state_dict()
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(sd)
