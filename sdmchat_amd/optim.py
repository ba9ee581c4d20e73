"""The optimiser of a training step on the AdamW kernel (core.adamw): all tensors of a parameter group in a few launches, the
clip by the global norm as the gradients are read, moments in 32 or in 8 bits.  (The reference trains with torch's AdamW behind
clip_grad_norm_, experiments/track4/sdmllm/track4_sdmllm_train_one_arm.py:232.)
"""
import math

import torch

from . import core

# A call's seed is its group's plus this (from the square root of 3) times the place of its first parameter in the optimiser.  The
# library adds t times another odd number (from the golden ratio) before it hashes: of places under 2,341 apart two steps meet the
# same sum only 1.7 million steps apart (of places under 36,672, 110,000), so no two calls of a run round by the same bits.
_CALL = 3144134277


class AdamW(torch.optim.Optimizer):
    """AdamW on float32 or bfloat16 parameters of one or more GPUs.

        opt = AdamW(model.parameters(), lr=3e-4, weight_decay=0.1, max_norm=1.0, state_bits=8)
        loss.backward()
        opt.step()                # opt.norm: the gradients' norm before the clip, a float32 scalar on the GPU
        opt.zero_grad()

    max_norm: gradients are clipped to this norm over all parameter groups, which must be on one GPU then; the .grad tensors
    stay as they are (a norm that is NaN reaches every parameter, as a product with it does).  state_bits: 32, or 8
    (core.new_moments: 2.06 bytes a value instead of 8, in the order of the parameter's values in memory, which has to stay what
    it is); a parameter group may have its own, as its own lr, betas, eps and weight_decay.  capturable: the steps are counted on
    the GPU, so a graph may capture step() once it has run; lr may then be a float32 tensor of one element that a schedule
    writes.  seed: of the 8-bit moments' rounding.  bfloat16 parameters are rounded to nearest, so a change below half their last
    place is lost: keep float32 parameters and bfloat16 autocast where that matters.  Sparse gradients and parameters whose values
    are not dense in memory are refused."""

    norm = None   # of the last step's gradients
    _OPTIONS = {"lr", "betas", "eps", "weight_decay", "state_bits", "max_norm", "capturable", "seed"}   # of a parameter group

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_norm=None,
                 capturable=False, seed=0):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      max_norm=max_norm, capturable=capturable, seed=seed))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()   # a refused group is none of the optimiser's
            raise

    def _check_group(self, group):
        lr, betas = group["lr"], group["betas"]
        if torch.is_tensor(lr) and not group["capturable"]:
            raise ValueError("AdamW: an lr on the device needs capturable")
        if not torch.is_tensor(lr) and not (math.isfinite(lr) and lr >= 0.0):
            raise ValueError(f"AdamW: lr {lr} must be finite and not negative")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"AdamW: betas {betas} must be two numbers in [0, 1)")
        if not (math.isfinite(group["eps"]) and group["eps"] >= 0.0):
            raise ValueError(f"AdamW: eps {group['eps']} must be finite and not negative")
        if not (math.isfinite(group["weight_decay"]) and group["weight_decay"] >= 0.0):
            raise ValueError(f"AdamW: weight_decay {group['weight_decay']} must be finite and not negative")
        if group["state_bits"] not in (32, 8):
            raise ValueError(f"AdamW: state_bits {group['state_bits']} is not 32 or 8")
        if group["max_norm"] is not None and not group["max_norm"] > 0.0:
            raise ValueError(f"AdamW: max_norm {group['max_norm']} must be positive")
        if group["max_norm"] != self.defaults["max_norm"] or group["capturable"] != self.defaults["capturable"]:
            raise ValueError("AdamW: max_norm and capturable are the same for all parameter groups")
        for p in group["params"]:
            if p.dtype not in core._DT:
                raise ValueError(f"AdamW: a parameter of {p.dtype}, not float32 or bfloat16")

    def _start(self, p, bits, clock):
        st = self.state[p]
        st["step"] = clock
        if bits == 8:
            st["moments"] = core.new_moments(p)
        else:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, requires_grad=False)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, requires_grad=False)
        return st

    def _clocks(self, group, live, capturing):
        """The live parameters of a group by their step counts: [(count or its device tensor, [(param, state)])]."""
        clocks, out, fresh = {}, [], {}
        on_device = self.defaults["capturable"]
        for p in live:
            st = self.state.get(p)
            if not st:
                if capturing:
                    raise RuntimeError("AdamW.step: run a step before capturing one (its moments must not be the graph's)")
                if p.device not in fresh:
                    fresh[p.device] = torch.zeros((), dtype=torch.int64, device=p.device) if on_device else 0
                st = self._start(p, group["state_bits"], fresh[p.device])
            step = st["step"]
            key = id(step) if on_device else (step, p.device)
            if key not in clocks:
                clocks[key] = []
                out.append((step, clocks[key]))
            clocks[key].append((p, st))
        if on_device and len(live) < len(group["params"]):
            # parameters without a gradient in this step keep their count: those with one go on with a copy
            alive = set(map(id, live))
            stay = {id(self.state[p]["step"]) for p in group["params"] if id(p) not in alive and self.state.get(p)}
            for i, (step, members) in enumerate(out):
                if id(step) in stay:
                    if capturing:
                        raise RuntimeError("AdamW.step: a captured step must have the gradients that the step before it had")
                    out[i] = step.clone(), members
                    for _, st in members:
                        st["step"] = out[i][0]
        return out

    @torch.no_grad()
    def step(self, closure=None):
        """One step on every parameter that has a gradient; returns the closure's loss."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_current_stream_capturing() if torch.cuda.is_available() else False
        if capturing and not self.defaults["capturable"]:
            raise RuntimeError("AdamW.step: a graph would replay the same step; construct the optimiser with capturable=True")
        groups = [(group, [p for p in group["params"] if p.grad is not None]) for group in self.param_groups]
        max_norm, self.norm = self.defaults["max_norm"], None
        if max_norm is not None and any(live for _, live in groups):
            self.norm = core.grad_norm([p.grad for _, live in groups for p in live])
        before = 0   # parameters of the groups before
        for group, live in groups:
            for step, members in self._clocks(group, live, capturing):
                ps = [p for p, _ in members]
                if group["state_bits"] == 8:
                    moments = [[st["moments"] for _, st in members]]
                else:
                    moments = [[st["exp_avg"] for _, st in members], [st["exp_avg_sq"] for _, st in members]]
                on_device = torch.is_tensor(step)
                # a call's positions begin at 0: each has a seed of its own, whatever else takes part in the step
                place = before + next(i for i, p in enumerate(group["params"]) if p is ps[0])
                core.adamw(ps, [p.grad for p in ps], *moments, step=step if on_device else step + 1, lr=group["lr"],
                           betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], max_norm=max_norm,
                           norm=self.norm, seed=group["seed"] + _CALL * place)
                if not on_device:
                    for _, st in members:
                        st["step"] = step + 1
            before += len(group["params"])
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but for the moments' types, which stay what they are (float32, or the bytes of 8-bit moments), and an lr
        that is a tensor here: it stays, and takes the loaded value.  The moments and counts are new tensors: a graph that
        captured a step holds the old ones.  What is refused changes nothing."""
        mine, loaded = [g["lr"] for g in self.param_groups], {}

        def check(_, state_dict):   # after the hooks before
            loaded.update(self._loaded_state(state_dict))
            return dict(state_dict, state={})

        def fill(_):   # before the hooks after
            self.state.update(loaded)
            for group, lr in zip(self.param_groups, mine):
                if torch.is_tensor(lr):
                    lr.detach().fill_(float(group["lr"]))
                    group["lr"] = lr
                elif torch.is_tensor(group["lr"]) and group["params"]:
                    group["lr"] = group["lr"].to(group["params"][0].device)
        hooks = [self.register_load_state_dict_pre_hook(check), self.register_load_state_dict_post_hook(fill, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _loaded_state(self, state_dict):
        """The state that a state dict holds, {parameter: its own copies}; ValueError for what is not this optimiser's kind."""
        name, on_device = "AdamW.load_state_dict", self.defaults["capturable"]
        groups = state_dict["param_groups"]
        if any(not g.keys() >= self._OPTIONS for g in groups):
            raise ValueError(f"{name}: not the state of this optimiser")
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError(f"{name}: parameter groups of other sizes")
        if any(g["max_norm"] != self.defaults["max_norm"] or g["capturable"] != on_device for g in groups):
            raise ValueError(f"{name}: max_norm and capturable must be the optimiser's own")
        if any(torch.is_tensor(g["lr"]) and g["lr"].numel() != 1 for g in groups):
            raise ValueError(f"{name}: an lr of several values")
        found = [(i, group["state_bits"], p, state_dict["state"].get(key)) for i, (group, own) in enumerate(
            zip(groups, self.param_groups)) for key, p in zip(group["params"], own["params"])]
        for _, bits, p, st in found:
            if not st:
                continue
            want = {"moments": ((-(-p.numel() // core.MOMENT_BLOCK), core.MOMENT_BYTES), torch.uint8)} if bits == 8 else {
                "exp_avg": (tuple(p.shape), torch.float32), "exp_avg_sq": (tuple(p.shape), torch.float32)}
            if {k: (tuple(v.shape), v.dtype) if torch.is_tensor(v) else v for k, v in st.items() if k != "step"} != want:
                raise ValueError(f"{name}: the state of a parameter {tuple(p.shape)} is not {want}")
            step = st.get("step")
            if not (isinstance(step, int) or (torch.is_tensor(step) and step.numel() == 1)) or step < 0:
                raise ValueError(f"{name}: a parameter's step must be a whole number from 0 on, got {step}")
        state, clocks = {}, {}
        for i, _, p, st in found:
            if not st:
                continue
            count = int(st["step"])
            if on_device:
                at = (i, count, p.device)
                if at not in clocks:
                    clocks[at] = torch.full((), count, dtype=torch.int64, device=p.device)
                count = clocks[at]
            state[p] = {"step": count}
            for k, v in st.items():
                if k == "moments":
                    state[p][k] = v.detach().to(p.device, copy=True).contiguous()
                elif k != "step":
                    state[p][k] = torch.empty_like(p, dtype=torch.float32, requires_grad=False).copy_(v.detach())
        return state
