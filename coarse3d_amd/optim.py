"""Optimisers: ``FlatAdamW`` (below), and ``AdamW`` / ``clip_grad_norm_`` over many tensors (their docstrings).

FlatAdamW: AdamW over ONE flat parameter / gradient / state buffer.

The reference builds ``torch.optim.AdamW(model.parameters(), lr)`` (tasks/weak_segmentation/trainer.py:146-151: one
parameter group, default betas / eps / weight decay on every tensor).  With one group the update is the same elementwise
formula on every parameter, so 192 tensors can be stepped as one: torch's own fused AdamW kernel (``torch._fused_adamw_``)
over single flat buffers is ONE launch instead of six multi-tensor launches of ~30 small tensors each (6 x 40 us -> ~20 us at
7.5 M parameters), and the host side of the step shrinks from ~5 ms to ~0.1 ms.  Same arithmetic, bit-identical update
(tests/test_gpu_step.py).

The parameters keep their identity (``p.data`` becomes a view of the flat buffer), ``param_groups`` lists them as
usual (learning-rate schedulers work unchanged), and the gradients are expected in the model's persistent flat gradient
buffer (``SalsaNextProto._bound_grad_views``); a gradient that arrived any other way is copied in first.

**Parameters without a gradient are skipped, as torch's AdamW skips them** (no weight decay, no step count, no moment
decay): the flat buffers are cut into *segments* -- maximal runs of parameters that have always been stepped together --
each with its own step counter, and one ``_fused_adamw_`` call steps the segments whose parameters carry a gradient.
With the reference's shipped ``contrast_warmup: 5`` (config_semantic_kitti.yaml:20) the projector has no gradient during
the first epochs: the buffer splits once into [backbone | projector], the backbone segment is stepped alone until the
embedding branch switches on.  A captured step (hipGraph) bakes the list of active segments in, which is why
``TrainStep`` keeps one graph per (shape, embedding branch on / off).

``state_dict()`` / ``load_state_dict()`` speak the checkpoint layout of ``torch.optim.AdamW(model.parameters())`` -- the
reference's optimiser (trainer.py:129, main.py:141,154): ``param_groups[0]["params"]`` indexes ALL parameters of the model
in ``model.parameters()`` order (197 for SalsaNextProto: the frozen ``prototypes`` is index 0, ``feat_norm.*`` /
``mask_norm.*`` are 193-196), and ``state`` holds entries for the parameters that have been stepped."""
import operator

import torch

from . import _lib, ops
from .ops import grad_norm


class FlatAdamW(torch.optim.Optimizer):
    graph_safe = True            # TrainStep(graph=True) may capture the update

    def __init__(self, named_params, grad_views, flat_grad, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 all_params=None):
        """named_params: (name, parameter) of the parameters that live in the flat buffers, in buffer order.
        all_params: every parameter of the model in ``model.parameters()`` order (the index space of checkpoints and of
        ``param_groups[0]["params"]``); default: the flat ones only."""
        named = list(named_params)
        params = [p for _, p in named]
        every = list(all_params) if all_params is not None else params
        pos = {id(p): i for i, p in enumerate(every)}
        if any(id(p) not in pos for p in params):
            raise ValueError("FlatAdamW: all_params must contain every flat parameter")
        super().__init__(every, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        total = sum(p.numel() for p in params)
        if flat_grad.numel() != total:
            raise ValueError("FlatAdamW: the flat gradient buffer does not match the parameters")
        dev = params[0].device
        self.flat_param = torch.empty(total, device=dev, dtype=torch.float32)
        self._offsets = [0]
        with torch.no_grad():
            for p in params:
                off = self._offsets[-1]
                view = self.flat_param[off:off + p.numel()].view_as(p)
                view.copy_(p.data)
                p.data = view                     # the Parameter object (and everything holding it) stays
                self._offsets.append(off + p.numel())
        self.flat_grad = flat_grad
        self.grad_views = [grad_views[n] for n, _ in named]
        self.exp_avg = torch.zeros_like(self.flat_param)
        self.exp_avg_sq = torch.zeros_like(self.flat_param)
        # segments [first flat parameter, one past the last) with their own step counters; one segment until some
        # parameters are stepped without the others
        self._segments = [[0, len(params), torch.zeros((), device=dev, dtype=torch.float32)]]
        # the learning rate as a device scalar: a captured step (TrainStep(graph=True)) must not bake a Python float in;
        # refreshed from param_groups[0]["lr"] (what schedulers write) by ``sync_lr`` outside the graph
        self.lr_t = torch.full((), float(lr), device=dev, dtype=torch.float32)
        self._lr_seen = float(lr)
        # False: the update takes the learning rate as a Python float (double precision inside the kernel, bit-identical
        # to torch.optim.AdamW(fused=True)); True (TrainStep(graph=True)): as the float32 device scalar above
        self.tensor_lr = False
        self._params = params
        self._index = [pos[id(p)] for p in params]       # flat parameter -> index in model.parameters()
        # bumped whenever the segment list (boundaries or step-counter tensors) is replaced: a captured step has the
        # old slices and counters baked in and must be dropped (TrainStep._graph_step compares it, like packs.generation)
        self.generation = 0

    @property
    def step_t(self):
        """Step counter of the first segment (the whole buffer while every parameter has always had a gradient)."""
        return self._segments[0][2]

    def zero_grad(self, set_to_none=True):
        if set_to_none:
            for p in self._params:
                p.grad = None
        else:
            self.flat_grad.zero_()

    def _split(self, active):
        """Cut the segments so that each one is entirely active or entirely inactive (a cut clones the step counter:
        both halves have the same history up to now).  Not during a capture: the segment list is part of what a
        graph bakes in, so the eager steps ahead of a capture have to run in the same configuration."""
        out = []
        for lo, hi, st in self._segments:
            start = lo
            for i in range(lo + 1, hi + 1):
                if i == hi or active[i] != active[start]:
                    out.append([start, i, st if start == lo else st.clone()])
                    start = i
        if len(out) != len(self._segments):
            if self.flat_param.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FlatAdamW: the set of parameters with a gradient changed inside a graph capture; run "
                                   "an eager step in this configuration first")
            self._segments = out
            self.generation += 1

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check_aliasing()
        active = []
        for p, v in zip(self._params, self.grad_views):
            g = p.grad
            active.append(g is not None)
            if g is not None and g.data_ptr() != v.data_ptr():   # came through autograd's AccumulateGrad, not the bound buffer
                v.copy_(g)
        self._split(active)
        segs = [s for s in self._segments if active[s[0]]]
        if not segs:
            return loss
        grp = self.param_groups[0]
        if not (self.flat_param.is_cuda and torch.cuda.is_current_stream_capturing()):
            self.sync_lr()
        o = self._offsets
        cut = lambda t: [t[o[lo]:o[hi]] for lo, hi, _ in segs]    # noqa: E731
        steps = [s[2] for s in segs]
        torch._foreach_add_(steps, 1)
        torch._fused_adamw_(cut(self.flat_param), cut(self.flat_grad), cut(self.exp_avg), cut(self.exp_avg_sq), [], steps,
                            amsgrad=False, lr=self.lr_t if self.tensor_lr else float(grp["lr"]), beta1=grp["betas"][0],
                            beta2=grp["betas"][1],
                            weight_decay=grp["weight_decay"], eps=grp["eps"], maximize=False, grad_scale=None, found_inf=None)
        return loss

    def sync_lr(self):
        """Copy param_groups[0]["lr"] into the device scalar the update reads (no-op while it is unchanged)."""
        lr = float(self.param_groups[0]["lr"])
        if lr != self._lr_seen:
            self.lr_t.fill_(lr)
            self._lr_seen = lr

    def _check_aliasing(self):
        """``p.data`` must still be the views of ``flat_param`` made in __init__: model.double() / .to(device) /
        load_state_dict(assign=True) rebind it, and the flat update would then move an orphaned buffer while the
        model silently stops training."""
        lo = self.flat_param.data_ptr()
        hi = lo + self.flat_param.numel() * 4
        for p in (self._params[0], self._params[-1]):
            if not (lo <= p.data_ptr() < hi) or p.dtype != torch.float32:
                raise RuntimeError("FlatAdamW: a parameter no longer lives in the flat buffer (dtype / device change or "
                                   "load_state_dict(assign=True) after the optimiser was built): rebuild the optimiser")

    def state_dict(self):
        """The layout of ``torch.optim.AdamW(model.parameters()).state_dict()`` -- what the reference writes into its
        checkpoints (tasks/weak_segmentation/main.py:141,154) and reads back with ``optimizer.load_state_dict``
        (trainer.py:129): ``param_groups[0]["params"] = range(number of model parameters)`` and per-parameter
        ``state[i] = {step, exp_avg, exp_avg_sq}`` for the parameters that have been stepped (parameters that never
        had a gradient -- the frozen bank and LayerNorms, the projector during the contrast warm-up -- have no entry,
        as in torch)."""
        groups = [dict({k: v for k, v in g.items() if k != "params"}, params=list(range(len(g["params"]))))
                  for g in self.param_groups]
        state = {}
        o = self._offsets
        for lo, hi, st in self._segments:
            if float(st) <= 0:
                continue
            for j in range(lo, hi):
                p = self._params[j]
                state[self._index[j]] = {"step": st.clone(), "exp_avg": self.exp_avg[o[j]:o[j + 1]].view_as(p).clone(),
                                         "exp_avg_sq": self.exp_avg_sq[o[j]:o[j + 1]].view_as(p).clone()}
        return {"state": state, "param_groups": groups}

    @torch.no_grad()
    def load_state_dict(self, sd):
        """Accepts ``torch.optim.AdamW(model.parameters())`` checkpoints (this class, torch, the reference), the
        trainable-parameters-only layout round 3 wrote (indices 0..191) and round 2's flat layout
        (``{"flat": True, step, exp_avg, exp_avg_sq}``).  Parameters without an entry start from zero moments and step
        0; runs of parameters with equal step counts become the segments of the flat update."""
        dev = self.flat_param.device
        if self.flat_param.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FlatAdamW.load_state_dict inside a graph capture")
        self.generation += 1                 # new step-counter tensors / segment boundaries: captured steps are stale
        if sd.get("flat"):
            self._segments = [[0, len(self._params), torch.zeros((), device=dev, dtype=torch.float32)]]
            self.step_t.copy_(sd["step"])
            self.exp_avg.copy_(sd["exp_avg"])
            self.exp_avg_sq.copy_(sd["exp_avg_sq"])
        else:
            if len(sd["param_groups"]) != 1:
                raise ValueError("FlatAdamW.load_state_dict: expected one parameter group")
            ids = list(sd["param_groups"][0]["params"])
            n_all = len(self.param_groups[0]["params"])
            if len(ids) == n_all:
                where = [ids[i] for i in self._index]                 # model.parameters() order
            elif len(ids) == len(self._params):
                where = ids                                          # the trainable parameters only (round 3)
            else:
                raise ValueError(f"FlatAdamW.load_state_dict: the checkpoint covers {len(ids)} parameters; this model has "
                                 f"{n_all} ({len(self._params)} trainable)")
            state = sd["state"]
            self.exp_avg.zero_()
            self.exp_avg_sq.zero_()
            steps = []
            o = self._offsets
            for j, key in enumerate(where):
                st = state.get(key)
                if st is None:
                    steps.append(0.0)
                    continue
                n = o[j + 1] - o[j]
                if st["exp_avg"].numel() != n:
                    raise ValueError(f"FlatAdamW.load_state_dict: state {key} does not fit its parameter")
                self.exp_avg[o[j]:o[j + 1]].copy_(st["exp_avg"].reshape(-1))
                self.exp_avg_sq[o[j]:o[j + 1]].copy_(st["exp_avg_sq"].reshape(-1))
                steps.append(float(st["step"]))
            segs, start = [], 0
            for j in range(1, len(steps) + 1):
                if j == len(steps) or steps[j] != steps[start]:
                    segs.append([start, j, torch.full((), steps[start], device=dev, dtype=torch.float32)])
                    start = j
            self._segments = segs
        for g, s in zip(self.param_groups, sd["param_groups"]):
            g.update({k: v for k, v in s.items() if k != "params"})


class _Cohort:
    """Parameters that have always been stepped together, and how often."""
    __slots__ = ("step", "step_t")

    def __init__(self, step=0, step_t=None):
        self.step, self.step_t = step, step_t


class AdamW(torch.optim.Optimizer):
    """AdamW over any list of parameters on the many-tensor kernels (``ops.adamw_step`` / ``ops.adamw8_step``): the formula, the
    argument names and -- with 32-bit states -- the checkpoint layout of ``torch.optim.AdamW``, parameter groups, schedulers
    and parameters without a gradient (skipped, as torch skips them) included.  Beside ``FlatAdamW``, which steps ONE flat buffer
    through torch's kernel, it takes parameters where they are and adds what training on one or two scans per GPU asks for:

    ``state_bits=8``: both moments in 8 bits (e4m3 times a power of two for every 256 elements, rounded stochastically from ``seed``
        and the step count): 2 bytes a parameter instead of 8, and 16 instead of 28 bytes moved a step.
    ``master_weights=True``: 16-bit parameters are stepped as fp32 copies in the state and written from them.
    ``max_grad_norm``: the gradients are clipped by their global norm on load -- one pass over them, no write; ``last_grad_norm``
        is that norm (a device scalar, before clipping).
    ``capturable=True``: step counts and learning rates live on the device (all parameters on one), for a captured step
        (``TrainStep(graph=True)``); ``sync_lr()`` copies changed learning rates, ``generation`` counts what makes a captured step
        stale.  As with every optimiser, the first steps of a configuration have to run outside the capture."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, master_weights=False,
                 max_grad_norm=None, capturable=False, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits is 8 or 32, got {state_bits}")
        if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"AdamW: lr, eps and weight_decay are not negative and betas in [0, 1); got {lr}, {eps}, {weight_decay}, {betas}")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"AdamW: max_grad_norm is not negative, got {max_grad_norm}")
        self.state_bits, self.master_weights, self.max_grad_norm = state_bits, master_weights, max_grad_norm
        self.capturable, self.seed = capturable, seed
        self.last_grad_norm = None
        self.generation = 0
        self._native = _lib.native()
        self._cohort_of = {}             # parameter -> _Cohort
        self._plan = None                # (each group's parameters, their gradients' types, launch lists) of the last step
        self._lr_t = {}                  # group index -> (value seen, device scalar)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    _OWN = ("state_bits", "master_weights", "max_grad_norm", "capturable", "seed", "last_grad_norm", "generation", "_cohort_of", "_lr_t")

    def __getstate__(self):
        return dict(super().__getstate__(), **{k: self.__dict__[k] for k in self._OWN})

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plan, self._native = None, _lib.native()

    @property
    def graph_safe(self):
        """Whether ``TrainStep(graph=True)`` may capture the update."""
        return self.capturable

    def add_param_group(self, group):
        super().add_param_group(group)
        self._plan = None

    # ------------------------------------------------------------------ state
    def _init_state(self, p):
        like = lambda dtype: torch.empty_like(p, dtype=dtype).zero_()  # noqa: E731
        st = self.state[p]
        if self.state_bits == 8:
            blocks = (p.numel() + ops.ADAMW8_BLOCK - 1) // ops.ADAMW8_BLOCK
            for name in ("exp_avg", "exp_avg_root"):
                st[name] = like(torch.uint8).view(torch.float8_e4m3fn)
                st[name + "_scale"] = torch.zeros(blocks, device=p.device, dtype=torch.float32)
        else:
            st["exp_avg"], st["exp_avg_sq"] = like(torch.float32), like(torch.float32)
        if self.master_weights and p.dtype != torch.float32:
            st["master"] = p.detach().float()

    _STATE = {32: ("exp_avg", "exp_avg_sq", None, None), 8: ("exp_avg", "exp_avg_root", "exp_avg_scale", "exp_avg_root_scale")}

    def _split_cohorts(self, params, grads):
        """Give every parameter with a gradient a cohort of parameters that all have one; new parameters get their state."""
        first, halves, capturing = None, {}, None
        for p, g in zip(params, grads):
            if g is None:
                continue
            if p not in self.state or not self.state[p]:
                capturing = torch.cuda.is_current_stream_capturing() if capturing is None and p.is_cuda else capturing
                if capturing:
                    raise RuntimeError("AdamW: a parameter is stepped for the first time inside a graph capture; run an eager step in "
                                       "this configuration first")
                if g.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                self._init_state(p)
                if first is None:
                    first = _Cohort(0, torch.zeros((), device=p.device, dtype=torch.float32) if self.capturable else None)
                    self.generation += 1
                self._cohort_of[p] = first
        # a cohort of which only some have a gradient: those get a counter of their own
        idle = {id(self._cohort_of[p]) for p, g in zip(params, grads) if g is None and p in self._cohort_of}
        if not idle:
            return
        for p, g in zip(params, grads):
            c = self._cohort_of.get(p)
            if g is not None and id(c) in idle:
                if id(c) not in halves:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: the set of parameters with a gradient changed inside a graph capture; run an eager "
                                           "step in this configuration first")
                    halves[id(c)] = _Cohort(c.step, c.step_t.clone() if c.step_t is not None else None)
                    self.generation += 1
                self._cohort_of[p] = halves[id(c)]

    def _launches(self, grads_by_group):
        """[(group index, cohort, parameter indices, params, [state lists], masters)] of parameters with a gradient: one entry for each
        group, step count, device and type."""
        runs = {}
        for gi, (group, grads) in enumerate(zip(self.param_groups, grads_by_group)):
            for i, (p, g) in enumerate(zip(group["params"], grads)):
                if g is not None:
                    master = "master" in self.state[p]
                    runs.setdefault((gi, id(self._cohort_of[p]), p.device, p.dtype, g.dtype, master), []).append(i)
        out = []
        for (gi, _, _, _, _, master), idx in runs.items():
            ps = [self.param_groups[gi]["params"][i] for i in idx]
            states = [None if name is None else [self.state[p][name] for p in ps] for name in self._STATE[self.state_bits]]
            out.append((gi, self._cohort_of[ps[0]], idx, ps, states, [self.state[p]["master"] for p in ps] if master else None))
        return out

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [g["params"] for g in self.param_groups]
        grads, types = zip(*map(self._native.grads_of, groups))
        plan = self._plan
        if plan is None or plan[1] != types or not all(all(map(operator.is_, a, b)) for a, b in zip(plan[0], groups)):
            self._split_cohorts([p for g in groups for p in g], [x for g in grads for x in g])
            plan = self._plan = ([list(g) for g in groups], types, self._launches(grads))
        launches = plan[2]
        if not launches:
            return loss
        capturing = launches[0][3][0].is_cuda and torch.cuda.is_current_stream_capturing()
        if self.capturable:
            if len({p.device for run in launches for p in run[3][:1]}) > 1:
                raise RuntimeError("AdamW(capturable=True): the parameters are on several devices")
            if not capturing:
                self.sync_lr()
        lists = [grads[gi] if len(idx) == len(grads[gi]) else [grads[gi][i] for i in idx] for gi, _, idx, _, _, _ in launches]
        scale = None
        if self.max_grad_norm is not None:
            scale = self._clip_factor(lists)
        for c in {id(run[1]): run[1] for run in launches}.values():
            c.step += 1
            if c.step_t is not None:
                c.step_t.add_(1.0)
        for (gi, cohort, _, ps, states, masters), gs in zip(launches, lists):
            group = self.param_groups[gi]
            more = dict(step=cohort.step_t if self.capturable else cohort.step, lr=self._lr_t[gi][1] if self.capturable else float(group["lr"]),
                        betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], grad_scale=scale, masters=masters)
            try:
                self._launch(gi, ps, gs, states, more)
            except ValueError:          # (refused before anything was launched) a gradient in another memory layout than its parameter
                if all(g.stride() == p.stride() for g, p in zip(gs, ps)):
                    raise
                self._launch(gi, ps, [torch.empty_like(p, dtype=g.dtype).copy_(g) for g, p in zip(gs, ps)], states, more)
        return loss

    def _launch(self, gi, params, grads, states, more):
        m, v, ms, vs = states
        if self.state_bits == 8:
            ops.adamw8_step(params, grads, m, ms, v, vs, seed=self.seed + gi, **more)
        else:
            ops.adamw_step(params, grads, m, v, **more)

    def _clip_factor(self, lists):
        by_type = {}
        for gs in lists:
            by_type.setdefault(gs[0].dtype, []).extend(gs)
        if len(by_type) == 1:
            self.last_grad_norm, scale = grad_norm(next(iter(by_type.values())), self.max_grad_norm)
            return scale
        norms = torch.stack([grad_norm(gs)[0] for gs in by_type.values()]).double()
        total = norms.square().sum().sqrt()
        self.last_grad_norm = total.float()
        return torch.clamp(self.max_grad_norm / (total + 1e-6), max=1.0).float()

    def sync_lr(self):
        """Copy learning rates that schedulers have changed into the device scalars of a capturable optimiser."""
        if not self.capturable:
            return
        for gi, group in enumerate(self.param_groups):
            lr = float(group["lr"])
            seen = self._lr_t.get(gi)
            if seen is None:
                if not group["params"]:
                    continue
                self._lr_t[gi] = (lr, torch.full((), lr, device=group["params"][0].device, dtype=torch.float32))
            elif seen[0] != lr:
                seen[1].fill_(lr)
                self._lr_t[gi] = (lr, seen[1])

    # ------------------------------------------------------------------ checkpoints
    def _step_of(self, p):
        c = self._cohort_of.get(p)
        return 0.0 if c is None else float(c.step_t) if c.step_t is not None else float(c.step)

    def state_dict(self):
        """torch's layout: ``state[i]`` of the i-th parameter over all groups, with its own ``step``; ``state_bits`` stands beside it."""
        groups, index, at = [], {}, 0
        for g in self.param_groups:
            groups.append(dict({k: v for k, v in g.items() if k != "params"}, params=list(range(at, at + len(g["params"])))))
            for p in g["params"]:
                index[id(p)] = at
                at += 1
        state = {index[id(p)]: dict({"step": torch.tensor(self._step_of(p))}, **{k: v.detach().clone() for k, v in st.items()})
                 for p, st in self.state.items() if st}
        return {"state": state, "param_groups": groups, "state_bits": self.state_bits}

    @torch.no_grad()
    def load_state_dict(self, sd):
        """Checkpoints of this class with the same ``state_bits``, and of ``torch.optim.AdamW`` with 32."""
        if len(sd["param_groups"]) != len(self.param_groups) or any(
                len(a["params"]) != len(b["params"]) for a, b in zip(sd["param_groups"], self.param_groups)):
            raise ValueError("AdamW.load_state_dict: the checkpoint's parameter groups differ from this optimiser's")
        if any(g.get("amsgrad") or g.get("maximize") for g in sd["param_groups"]):
            raise ValueError("AdamW.load_state_dict: the checkpoint is of an optimiser with amsgrad or maximize, which this one does not have")
        params = {}
        for a, b in zip(sd["param_groups"], self.param_groups):
            params.update(zip(a["params"], b["params"]))
        names = [n for n in self._STATE[self.state_bits] if n is not None]
        new = {}
        for key, st in sd["state"].items():
            p = params.get(key)
            if p is None or not set(names) <= set(st) or "step" not in st:
                raise ValueError(f"AdamW.load_state_dict: state {key} is not that of a parameter with {self.state_bits}-bit states")
            mine = {}
            for n in names + (["master"] if "master" in st else []):
                t = st[n]
                blocks = n.endswith("_scale")
                if (t.numel() != (p.numel() + ops.ADAMW8_BLOCK - 1) // ops.ADAMW8_BLOCK) if blocks else t.shape != p.shape:
                    raise ValueError(f"AdamW.load_state_dict: {n} of state {key} does not fit its parameter")
                if self.state_bits == 8 and not blocks and n != "master":
                    if t.dtype != torch.float8_e4m3fn:
                        raise ValueError(f"AdamW.load_state_dict: {n} of state {key} is {t.dtype}, not float8_e4m3fn")
                    # (codes belong to blocks of memory: the layout has to be the checkpoint's, or the parameter's where both are dense alike)
                    if t.stride() != p.stride():
                        raise ValueError(f"AdamW.load_state_dict: {n} of state {key} has another memory layout than its parameter")
                    mine[n] = torch.empty_like(p, dtype=torch.uint8).copy_(t.view(torch.uint8)).view(torch.float8_e4m3fn)
                elif blocks:
                    mine[n] = t.detach().to(device=p.device, dtype=torch.float32, copy=True).reshape(-1).contiguous()
                else:
                    mine[n] = torch.empty_like(p, dtype=torch.float32).copy_(t)
            if self.master_weights and p.dtype != torch.float32 and "master" not in mine:
                mine["master"] = p.detach().float()
            if not self.master_weights:
                mine.pop("master", None)
            new[p] = (mine, float(st["step"]))
        cohorts = {}
        self.state.clear()
        self._cohort_of.clear()
        for p, (mine, t) in new.items():
            self.state[p] = mine
            if (t, p.device) not in cohorts:
                cohorts[t, p.device] = _Cohort(int(t), torch.full((), t, device=p.device, dtype=torch.float32) if self.capturable else None)
            self._cohort_of[p] = cohorts[t, p.device]
        for g, s in zip(self.param_groups, sd["param_groups"]):
            g.update({k: tuple(v) if k == "betas" else v for k, v in s.items() if k in ("lr", "betas", "eps", "weight_decay", "initial_lr")})
        self._plan = None
        self.generation += 1


def clip_grad_norm_(parameters, max_norm):
    """``torch.nn.utils.clip_grad_norm_`` on the many-tensor kernels: scales the gradients of ``parameters`` in place such that their
    joint 2-norm is at most ``max_norm``; returns the norm they had, as a device scalar that nothing waits for."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    by_type = {}
    for p in params:
        if p.grad is not None:
            by_type.setdefault(p.grad.dtype, []).append(p.grad)
    if not by_type:
        return torch.zeros((), device=params[0].device if params else None)
    if len(by_type) == 1:
        return ops.clip_grad_norm_(next(iter(by_type.values())), max_norm)
    raise ValueError(f"clip_grad_norm_: the gradients have several types: {sorted(map(str, by_type))}")
