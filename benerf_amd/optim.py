"""`torch.optim.Adam` objects whose `step()` is ONE fused K8 launch (benerf_adam_step) over a flat parameter arena.

The reference builds five `torch.optim.Adam` (model/optimize.py:36-55) and its training loop calls `zero_grad()`, `step()` and
writes `param_group["lr"]` on them (train.py:196-200, 343-394); checkpoints store their `state_dict()` (train.py:443-455).
`FlatAdam` IS a `torch.optim.Adam` - same constructor, `param_groups`, `state`, `state_dict()` / `load_state_dict()` format
(per parameter: `step`, `exp_avg`, `exp_avg_sq`) - but

  * at its first `step()` its parameters are re-homed into one flat fp32 buffer (`ParamArena`: the `nn.Parameter`s keep names
    and shapes and alias it), next to flat gradient / exp_avg / exp_avg_sq buffers of the same layout;
  * the render nodes (engine.RenderPair / RenderRays) write the weight gradients straight into the arena's gradient buffer and
    hand autograd VIEWS of it, which `AccumulateGrad` adopts as `.grad` without a copy (the gradient is `None` after the
    reference's `zero_grad()`), so `p.grad` is a window on the arena;
  * `step()` checks those aliases (pointer comparisons, no device work), repairs what a caller replaced (a `.grad` that is
    somebody else's tensor is copied in; state loaded by `load_state_dict` is adopted) and updates every parameter of a group
    with one launch - torch's own multi-tensor Adam costs ~10 launches per optimiser and, under the reference's
    `torch.set_default_tensor_type("torch.cuda.FloatTensor")` (train.py:472), one `.item()` synchronisation PER PARAMETER and
    step, because its `step` counters are then created on the device (96 per iteration for the two NeRFs).

Arithmetic = torch's Adam with default betas / eps (benerf_adam_step is pinned by golden vector G10).  Options that change the
update rule (weight_decay, amsgrad, maximize) are refused: the reference never sets them.

`FusedAdamW` is the AdamW next to it (K9): any list of parameters where they live, decoupled decay, clipping by the global norm without
a synchronisation, moments in 32 or 8 bits, float32 master copies of half-precision parameters.
"""
import itertools
from operator import is_, itemgetter

import torch
from torch.optim.optimizer import _global_optimizer_post_hooks, _global_optimizer_pre_hooks

from . import kernels as K


class ParamArena:
    """Flat fp32 storage for a list of parameters: value, gradient, exp_avg, exp_avg_sq, all with one layout."""

    def __init__(self, params):
        params = list(params)
        dev = params[0].device
        self.device = dev
        self.params = params
        n = sum(p.numel() for p in params)
        self.p = torch.zeros(n, dtype=torch.float32, device=dev)
        self.g = torch.zeros(n, dtype=torch.float32, device=dev)
        self.m = torch.zeros(n, dtype=torch.float32, device=dev)
        self.v = torch.zeros(n, dtype=torch.float32, device=dev)
        self.slots = []                     # (offset, numel) per parameter, in order
        self.index = {id(p): i for i, p in enumerate(params)}
        o = 0
        for p in params:
            if p.dtype != torch.float32:
                raise TypeError("ParamArena: float32 parameters only")
            k = p.numel()
            self.slots.append((o, k))
            self.adopt(p, o, k)
            o += k
        self.base_p, self.base_g = self.p.data_ptr(), self.g.data_ptr()
        # which backward pass (torch._C._current_graph_task_id) last wrote the gradient slots starting at parameter i0: a second
        # render node of the SAME pass must add on top of the first one's result instead of overwriting it (engine._grad_targets)
        self.pass_ids = {}

    def adopt(self, p, o, k):
        """Move p's value into its slot and make p alias it (names, shapes, autograd identity unchanged)."""
        view = self.p[o:o + k].view(p.shape)
        view.copy_(p.detach())
        p.data = view
        p._benerf_slot = (self, o, k)

    def homed(self, i):
        p = self.params[i]
        o, k = self.slots[i]
        return p.data_ptr() == self.base_p + 4 * o and p.is_contiguous()

    def grad_view(self, i):
        """A FRESH view of parameter i's gradient slot (nobody else holds it: autograd may adopt it as `.grad`)."""
        o, k = self.slots[i]
        return self.g[o:o + k].view(self.params[i].shape)

    def grad_is_window(self, i):
        """True if parameter i's `.grad` is a window on its slot of the gradient buffer."""
        g = self.params[i].grad
        o, k = self.slots[i]
        return g is not None and g.data_ptr() == self.base_g + 4 * o and g.is_contiguous() and g.dtype == torch.float32


def arena_of(params):
    """(arena, [slot index of each parameter]) if all of `params` are homed members of ONE arena; else None."""
    first = getattr(params[0], "_benerf_slot", None)
    if first is None:
        return None
    arena = first[0]
    idx = []
    for p in params:
        slot = getattr(p, "_benerf_slot", None)
        if slot is None or slot[0] is not arena:
            return None
        i = arena.index.get(id(p))
        if i is None or not arena.homed(i):
            return None
        idx.append(i)
    return arena, idx


class FlatAdam(torch.optim.Adam):
    def __init__(self, params, lr=1e-3, **kw):
        super().__init__(params, lr=lr, **kw)
        # The arena is built - and the parameters re-homed into it - at the FIRST step(), not here: an optimiser that never steps
        # (engine.TrainStep keeps its own flat buffers and uses these objects only as checkpoint containers, export / import
        # _optimizer_state) must not move anybody's storage.  The first iteration of a loop therefore runs the generic path
        # (fresh gradient tensors, copied in), every later one the in-place path.
        self._arena = None
        self._index = {}
        self._state_seen = {}               # id(p) -> id(state dict) whose tensors are known to alias the arena

    # -- state: the reference's checkpoint format, backed by the arena -------------------------------------------------------
    def _adopt_state(self, p, i):
        """state[p] as torch's Adam keeps it, with exp_avg / exp_avg_sq as views of the arena; values set by load_state_dict or
        by anybody who assigned `state[p]` are copied in first."""
        a = self._arena
        o, k = a.slots[i]
        st = self.state.get(p)
        m_view, v_view = a.m[o:o + k].view(p.shape), a.v[o:o + k].view(p.shape)
        if not st:
            m_view.zero_()
            v_view.zero_()
            st = {"step": torch.tensor(0.0, dtype=torch.float32, device="cpu"), "exp_avg": m_view, "exp_avg_sq": v_view}
            self.state[p] = st
        else:
            if "exp_avg_scale" in st:           # FusedAdamW's 8-bit form
                st.update(convert_moments(st, 32))
                del st["exp_avg_scale"], st["exp_avg_sq_scale"]
            for key, view in (("exp_avg", m_view), ("exp_avg_sq", v_view)):
                cur = st.get(key)
                if cur is None:
                    view.zero_()
                elif cur.data_ptr() != view.data_ptr():
                    view.copy_(cur.to(device=view.device, dtype=torch.float32).reshape(view.shape))
                st[key] = view
            step = st.get("step", 0.0)
            step = float(step.item()) if torch.is_tensor(step) else float(step)     # a loaded device counter: one read, once
            st["step"] = torch.tensor(step, dtype=torch.float32, device="cpu")
        self._state_seen[id(p)] = id(st)
        return st

    def _live_state(self, p, i):
        st = self.state.get(p)
        if st and self._state_seen.get(id(p)) == id(st) and st["exp_avg"].data_ptr() == self._arena.m.data_ptr() + 4 * self._arena.slots[i][0]:
            return st
        return self._adopt_state(p, i)

    def state_dict(self):
        # every parameter that has been stepped carries live state already; nothing to flush
        return super().state_dict()

    def zero_grad(self, set_to_none=True):
        if self._arena is not None:
            self._arena.pass_ids.clear()
        return super().zero_grad(set_to_none=set_to_none)

    # -- the update ----------------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        a = self._arena
        if a is None:
            flat = [p for g in self.param_groups for p in g["params"]]
            if not flat:
                return loss
            a = self._arena = ParamArena(flat)
            self._index = a.index
        for group in self.param_groups:
            if group.get("weight_decay", 0) != 0 or group.get("amsgrad", False) or group.get("maximize", False):
                raise NotImplementedError("benerf_amd.optim.FlatAdam implements the reference's Adam (model/optimize.py:36-55): no "
                                          "weight_decay / amsgrad / maximize")
            beta1, beta2 = group["betas"]
            lr, eps = float(group["lr"]), float(group["eps"])
            run = None                      # [first offset, numel, t] of a run of consecutive slots updated by one launch
            steps = []
            for p in group["params"]:
                if p.grad is None:          # torch's Adam leaves such a parameter (and its counters) alone
                    run = self._flush(run, lr, beta1, beta2, eps)
                    continue
                i = self._index.get(id(p))
                if i is None:
                    raise NotImplementedError("FlatAdam: a parameter added after the first step() (add_param_group) has no slot in the arena")
                o, k = a.slots[i]
                if not a.grad_is_window(i):
                    a.g[o:o + k].copy_(p.grad.detach().to(torch.float32).reshape(-1))
                st = self._live_state(p, i)
                t = int(st["step"].item()) + 1          # a host tensor: the checkpointed counter is the only counter
                steps.append(st["step"])
                if not a.homed(i):
                    # somebody re-pointed p.data (e.g. engine.TrainStep took the graph over and owns the storage now): update the
                    # parameter where it lives, moments in this arena - never steal the storage back behind the other owner
                    run = self._flush(run, lr, beta1, beta2, eps)
                    if not p.data.is_contiguous():
                        raise RuntimeError("FlatAdam: a parameter outside the arena must be contiguous")
                    K.adam_step(p.data.view(-1), a.g[o:o + k], a.m[o:o + k], a.v[o:o + k], lr, t, beta1, beta2, eps)
                    continue
                if run is not None and run[0] + run[1] == o and run[2] == t:
                    run[1] += k
                else:
                    self._flush(run, lr, beta1, beta2, eps)
                    run = [o, k, t]
            self._flush(run, lr, beta1, beta2, eps)
            if steps:
                torch._foreach_add_(steps, 1.0)
        a.pass_ids.clear()
        return loss

    def _flush(self, run, lr, beta1, beta2, eps):
        if run is not None:
            a = self._arena
            o, k, t = run
            K.adam_step(a.p[o:o + k], a.g[o:o + k], a.m[o:o + k], a.v[o:o + k], lr, t, beta1, beta2, eps)
        return None


def encode_moment(x, root=False):
    """A float32 moment in 8 bits, to nearest: (float8_e4m3fn codes of x's shape, float32 scale of every 128 consecutive elements).  For
    a checkpoint of 32-bit moments; the step itself rounds stochastically (include/benerf_hip.h, K9).  Encode the ROOT of exp_avg_sq, with
    root=True: what is above 0 then becomes 2^-9 of its scale at least, as in the step - exp_avg has a scale of its own, and the next update must
    not be divided by eps alone."""
    n = x.numel()
    pad = torch.zeros(-(-n // K.ADAMW_BLOCK) * K.ADAMW_BLOCK, dtype=torch.float32, device=x.device)
    pad[:n] = x.detach().reshape(-1)
    rows = pad.view(-1, K.ADAMW_BLOCK)
    top = torch.where(rows.isfinite(), rows.abs(), 0.0).amax(1)
    exponent = (torch.frexp(top)[1] - 1).clamp_min(-100) - 7
    scale = ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)
    grid = rows / scale[:, None]
    if root:
        grid = torch.where(rows > 0, grid.clamp_min(2.0 ** -9), grid)
    code = torch.where(rows.isfinite(), grid, float("nan")).view(-1)[:n]
    return code.to(K.CODE_TYPE).view(x.shape), scale


def decode_moment(code, scale):
    """The float32 values that 8-bit codes and their scales stand for."""
    return (code.reshape(-1).to(torch.float32) * scale.repeat_interleave(K.ADAMW_BLOCK)[:code.numel()]).view(code.shape)


def zero_moments(params, bits):
    """Moments of a list of parameters at zero, in flat buffers (a tensor's slot at a multiple of 128 elements): the keyword arguments
    exp_avg, exp_avg_sq - and with 8 bits exp_avg_scale, exp_avg_sq_scale - of kernels.AdamWPlan."""
    B, out = K.ADAMW_BLOCK, {}
    blocks = [-(-p.numel() // B) for p in params]
    starts = list(itertools.accumulate(blocks, initial=0))
    for name in ("exp_avg", "exp_avg_sq"):
        flat = torch.zeros(starts[-1] * B, dtype=torch.uint8 if bits == 8 else torch.float32, device=params[0].device)
        if bits == 8:
            flat = flat.view(K.CODE_TYPE)
            scale = torch.zeros(starts[-1], dtype=torch.float32, device=params[0].device)
            out[name + "_scale"] = [scale[a:a + b] for a, b in zip(starts, blocks)]
        out[name] = [flat[a * B:a * B + p.numel()].view(p.shape) for a, p in zip(starts, params)]
    return out


def convert_moments(state, bits):
    """A parameter's saved moments in the form that `bits` asks for, as a new dict of the tensors zero_moments names."""
    coded = "exp_avg_scale" in state
    if not coded and state["exp_avg"].dtype == K.CODE_TYPE:
        raise ValueError("8-bit moments without their scales")
    if coded == (bits == 8):
        return {k: state[k] for k in ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if coded else ())}
    if coded:
        return {"exp_avg": decode_moment(state["exp_avg"], state["exp_avg_scale"]), "exp_avg_sq": decode_moment(state["exp_avg_sq"], state["exp_avg_sq_scale"]).square_()}
    out = {}
    out["exp_avg"], out["exp_avg_scale"] = encode_moment(state["exp_avg"].to(torch.float32))
    out["exp_avg_sq"], out["exp_avg_sq_scale"] = encode_moment(state["exp_avg_sq"].to(torch.float32).sqrt(), root=True)
    return out


def network_settings(args):
    """(state_bits or None for the reference's Adam, weight decay, max_norm) of the networks' optimiser: args.benerf_optimizer "adam"
    (default), "adamw" or "adamw8" (moments in 8 bits), args.benerf_weight_decay (0.01), args.benerf_max_grad_norm (None: no clipping)."""
    kind, most = getattr(args, "benerf_optimizer", "adam"), getattr(args, "benerf_max_grad_norm", None)
    if kind not in ("adam", "adamw", "adamw8"):
        raise ValueError("benerf_optimizer must be adam, adamw or adamw8, not %r" % (kind,))
    if kind == "adam":
        if most is not None or getattr(args, "benerf_weight_decay", 0):
            raise ValueError("benerf_max_grad_norm and benerf_weight_decay need benerf_optimizer adamw or adamw8")
        return None, 0.0, None
    return 8 if kind == "adamw8" else 32, float(getattr(args, "benerf_weight_decay", 1e-2)), most


class _Cohort:
    """Parameters of a group that have made the same steps: one counter (torch's `step`), shared by their state dicts."""

    def __init__(self, step, members):
        self.step, self.members = step, members


# checks of whole lists run through map(): a fifth off what a comprehension of method calls costs
_address, _numel, _device, _contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous


class _Group:
    """What a step needs of one parameter group, made once and again when something was replaced, dropped or moved."""
    MASTER = itemgetter("master")

    def __init__(self, params, plan, states, cohorts, on_device):
        self.params, self.plan, self.states, self.cohorts, self.on_device = params, plan, states, cohorts, on_device
        self.at = list(map(_address, params))
        self.kinds = itemgetter("exp_avg", "exp_avg_sq", "step", *(("exp_avg_scale", "exp_avg_sq_scale") if plan.state_bits == 8 else ()))
        self.with_master = [st for st, x in zip(states, plan.master or ()) if x is not None]
        self.look()

    def watched(self):
        """Every tensor of state that the plan or a counter stands for."""
        return itertools.chain(itertools.chain.from_iterable(map(self.kinds, self.states)), map(self.MASTER, self.with_master))

    def look(self):
        self.parts = list(self.watched())

    def holds(self, params):
        """Parameters, their addresses and their state are the ones that the plan was made for."""
        if len(params) != len(self.params) or not all(map(is_, params, self.params)) or list(map(_address, params)) != self.at:
            return False
        try:
            return all(map(is_, self.watched(), self.parts))
        except KeyError:            # a dropped one
            return False


def _hooks_or_profiler():
    return bool(_global_optimizer_pre_hooks or _global_optimizer_post_hooks or torch.autograd.profiler._is_profiler_enabled)


class FusedAdamW(torch.optim.AdamW):
    """torch.optim.AdamW (decoupled weight decay; same param_groups, state and state_dict) whose step() is one K9 launch per group.

    Parameters stay where they are: float32, bfloat16 or float16, contiguous, on one device.  A parameter without a gradient is left
    alone, with its moments and its counter; a parameter that has moved (`p.data = ...`) is followed, and so is a tensor of state that was
    assigned or dropped.
      state_bits  32: exp_avg, exp_avg_sq in float32, whatever the parameter's type.  8: exp_avg in float8_e4m3fn and exp_avg_sq as the
                  float8_e4m3fn codes of its ROOT, exp_avg_scale and exp_avg_sq_scale with a float32 for every 128 elements, rounded
                  stochastically with `seed` (16.1 instead of 28 bytes of traffic and 2.1 instead of 8 of memory per parameter).
                  load_state_dict takes either form (encode_moment / decode_moment).
      max_norm    None, or the global 2-norm over ALL groups to which gradients are clipped in the same step; a norm that is not finite
                  skips the step on the device.  After step(), grad_norm holds [norm, coefficient, skipped?, steps skipped so far].
      master      float32 copies (state["master"]) of half-precision parameters: read and updated instead of them, rounded into them.
                  They are made from the parameters at the first step: weights that are loaded later need theirs dropped
                  (`del opt.state[p]["master"]`), the next step makes them again.
      capturable  counters live on the device, a step can be captured (make one step before, outside; learning rates that change need
                  `lr` as a float32 tensor on the device).  With max_norm they live there too.  A captured step goes on with the state,
                  the counters and the set of gradients of its capture: load_state_dict, or a step outside with other gradients
                  missing, needs a new capture; a program that makes many of them with new optimisers calls kernels.release_captured()
                  between them.  Networks whose weights it changes are packed again at every forward pass, and must not be
                  replayed over between a forward pass and its backward.
      guard_range skip the step where the MLP's range guard says so, like FlatAdam.
    state[p]["step"] is ONE tensor for all parameters of a group that have made the same steps (state_dict gives each its own).
    amsgrad, maximize and differentiable are refused."""

    STATE_KEYS = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_norm=None, master=False,
                 capturable=False, seed=0, guard_range=True, **kw):
        if state_bits not in (8, 32):
            raise ValueError("FusedAdamW: moments have 8 or 32 bits, not %r" % (state_bits,))
        if max_norm is not None and not max_norm > 0:
            raise ValueError("FusedAdamW: max_norm must be positive, got %r" % (max_norm,))
        if kw.get("fused"):         # it would promise to undo a gradient scaler's factor
            raise NotImplementedError("FusedAdamW: fused=True is torch's own kernel; leave it out")
        self._settings = dict(state_bits=state_bits, max_norm=max_norm, master=bool(master), seed=int(seed), guard_range=bool(guard_range))
        self._plans, self._states = {}, []
        self.grad_norm = None
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=capturable, **kw)

    state_bits = property(lambda self: self._settings["state_bits"])
    max_norm = property(lambda self: self._settings["max_norm"])

    def __getstate__(self):
        return dict(super().__getstate__(), _settings=self._settings)

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans, self._states = {}, []
        self.grad_norm = None

    def state_dict(self):
        # every parameter gets a counter of its own: torch's AdamW, loading this, adds to each of them.  On the host, as torch keeps it.
        out = super().state_dict()
        on_device = {k for g in out["param_groups"] if g.get("capturable") for k in g["params"]}
        out["state"] = {k: dict(st, step=st["step"].clone() if k in on_device else st["step"].cpu().clone()) if torch.is_tensor(st.get("step")) else st
                        for k, st in out["state"].items()}
        return out

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # torch casts state to its parameter's type: moments, codes and master copies keep the one that they were saved in
        saved = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        mine = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for key, p in zip(saved, mine):
            st = state_dict["state"].get(key)
            if st:
                for name in self.STATE_KEYS:
                    if torch.is_tensor(st.get(name)):
                        self.state[p][name] = st[name].detach().to(device=p.device, copy=True)
        self._plans = {}

    # -- state --------------------------------------------------------------------------------------------------------------
    def _counts_on_device(self, group):
        return bool(group.get("capturable")) or self.max_norm is not None

    def _adopt(self, params):
        """state[p] of every parameter in the form this optimiser keeps: what fits stays where it is, another form is converted, what
        is missing starts at zero."""
        bits = self.state_bits
        fresh = []
        for p in params:
            st = self.state[p]
            if "exp_avg" not in st or "exp_avg_sq" not in st:
                fresh.append(p)
                continue
            for x in (st["exp_avg"], st["exp_avg_sq"]):
                if x.numel() != p.numel():
                    raise ValueError("FusedAdamW: a moment has %d elements, its parameter %d" % (x.numel(), p.numel()))
            if bits == 32:
                form = convert_moments(st, 32)
                st.pop("exp_avg_scale", None), st.pop("exp_avg_sq_scale", None)
            else:
                form = convert_moments(st, 8)
            for name, x in form.items():
                kind = K.CODE_TYPE if bits == 8 and not name.endswith("_scale") else torch.float32
                st[name] = x.to(device=p.device, dtype=kind).contiguous()
        if fresh:
            for name, ts in zero_moments(fresh, bits).items():
                for p, x in zip(fresh, ts):
                    self.state[p][name] = x
        for p in params:
            st = self.state[p]
            if not self._settings["master"]:
                st.pop("master", None)
            else:
                if p.dtype != torch.float32:
                    x = st.get("master")
                    st["master"] = p.detach().float() if x is None else x.to(device=p.device, dtype=torch.float32).contiguous()

    @torch.no_grad()
    def _make(self, group):
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: make one step outside before a step is captured")
        params = list(group["params"])
        self._adopt(params)
        states = [self.state[p] for p in params]
        scales = {}
        if self.state_bits == 8:
            scales = {name: [st[name] for st in states] for name in ("exp_avg_scale", "exp_avg_sq_scale")}
        if self._settings["master"] and any(p.dtype != torch.float32 for p in params):
            scales["master"] = [st.get("master") if p.dtype != torch.float32 else None for p, st in zip(params, states)]
        plan = K.AdamWPlan([p.data for p in params], [st["exp_avg"] for st in states], [st["exp_avg_sq"] for st in states], **scales)
        on_device = self._counts_on_device(group)
        device = plan.device if on_device else torch.device("cpu")
        if self.max_norm is not None and (self.grad_norm is None or self.grad_norm.device != plan.device):
            self.grad_norm = torch.zeros(4, dtype=torch.float32, device=plan.device)
        by_value = {}
        for k, st in enumerate(states):
            by_value.setdefault(float(st.get("step", 0.0)), []).append(k)
        cohorts = []
        for value, members in by_value.items():
            c = _Cohort(torch.tensor(value, dtype=torch.float32, device=device), members)
            for k in members:
                states[k]["step"] = c.step
            cohorts.append(c)
        return _Group(params, plan, states, cohorts, on_device)

    def _group(self, index, group):
        g = self._plans.get(index)
        if g is None or g.on_device != self._counts_on_device(group) or not g.holds(group["params"]):
            g = self._plans[index] = self._make(group)
            self._states = list(self.state.values())
        return g

    @staticmethod
    def _gradients(g):
        """The group's gradients, contiguous, and whether some are missing."""
        grads, sizes = [p.grad for p in g.params], g.plan.numels
        there = grads
        if any(map(is_, grads, itertools.repeat(None))):
            sizes, there = [n for n, x in zip(sizes, grads) if x is not None], [x for x in grads if x is not None]
        if list(map(_numel, there)) != sizes or not set(map(_device, there)) <= {g.plan.device.index}:     # p.data was replaced behind its gradient
            raise RuntimeError("FusedAdamW: a gradient has another size or device than its parameter")
        if not all(map(_contiguous, there)):
            if any(x.layout is not torch.strided for x in there):
                raise NotImplementedError("FusedAdamW: sparse gradients")
            grads = [x if x is None else x.detach().contiguous() for x in grads]
        return grads, len(there) < len(grads)

    # -- the update ----------------------------------------------------------------------------------------------------------
    def step(self, closure=None):
        # torch wraps step() of every optimiser with its hooks and a profiler range, at 10 us a call: only where there are any
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _hooks_or_profiler():
            return self._hooked_step(closure)
        return self._step(closure)

    step.hooked = True

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if len(self.state) != len(self._states) or not all(map(is_, self.state.values(), self._states)):
            self._plans = {}                # state[p] was assigned
        work, norms = [], []                # (group's place, group, plan and counters, cohort, its gradients)
        for index, group in enumerate(self.param_groups):
            if group["amsgrad"] or group["maximize"] or group["differentiable"]:
                raise NotImplementedError("FusedAdamW: amsgrad, maximize and differentiable are not built")
            if not group["params"]:
                continue
            g = self._group(index, group)
            grads, missing = self._gradients(g)
            if missing:
                if all(x is None for x in grads):
                    continue
                self._split(g, grads)
            whole = K.GradList.of_checked(grads, g.plan)
            norms.append(whole)
            for c in g.cohorts:
                if len(c.members) == len(grads):
                    work.append((index, group, g, c, whole))
                elif grads[c.members[0]] is not None:
                    mine = set(c.members)
                    work.append((index, group, g, c, K.GradList.of_checked([x if k in mine else None for k, x in enumerate(grads)], g.plan)))
        if not work:
            return loss
        guard, words = self._settings["guard_range"], None
        on_device = [c.step for _, _, g, c, _ in work if g.on_device]
        if self.max_norm is not None:
            words = K.grad_norm(norms[0] if len(norms) == 1 else norms, self.max_norm, out=self.grad_norm, counters=on_device[:64], guard_range=guard)
            on_device = on_device[64:]
        for s in on_device:
            K.adamw_count(s, norm=words, guard_range=guard)
        for index, group, g, c, part in work:
            host, lr = not g.on_device, group["lr"]
            t = int(c.step.item()) + 1 if host else c.step
            if torch.is_tensor(lr) and not lr.is_cuda:
                lr = float(lr)
            K.adamw_step(g.plan, part, lr, t, group["betas"], group["eps"], group["weight_decay"], norm=words,
                         seed=self._settings["seed"] + index * 0x9E3779B97F4A7C15, guard_range=guard)
            if host:
                c.step += 1.0
        return loss

    _hooked_step = torch.optim.Optimizer.profile_hook_step(_step)

    def _split(self, g, grads):
        """Cohorts in which only some have a gradient this time part: the others' counter stays."""
        for c in list(g.cohorts):
            have = [k for k in c.members if grads[k] is not None]
            if have and len(have) < len(c.members):
                if g.on_device and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("FusedAdamW: make one step with the same gradients missing outside before it is captured")
                c.members = [k for k in c.members if grads[k] is None]
                new = _Cohort(c.step.clone(), have)
                for k in have:
                    g.states[k]["step"] = new.step
                g.cohorts.append(new)
        g.look()
