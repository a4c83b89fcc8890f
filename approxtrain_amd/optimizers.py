"""``AdamW`` over all of a model's tensors in a launch or two, moments in 32 bits or in 8 (the reference trains with
Keras's optimizers)."""
from itertools import repeat
from operator import is_not

import torch

from . import functors


class _Moments(functors.AdamWState):
    """Moments of parameters of one type that began to step together.  ``steps``: how many each has taken, one number
    while all have taken as many, else a list."""

    def __init__(self, params, state_bits):
        super().__init__(params, state_bits)
        self.steps = 0

    def update(self, grads, grad_scale, hyper):
        if type(self.steps) is int and all(map(is_not, grads, repeat(None))):
            functors.adamw_step(self, grads, self.steps + 1, *hyper, grad_scale)
            self.steps += 1
            return
        old = self.steps if type(self.steps) is list else [self.steps] * len(grads)
        steps = [n if g is None else n + 1 for n, g in zip(old, grads)]
        for number in sorted({n for n, g in zip(steps, grads) if g is not None}):  # (a call has one number for all its tensors)
            functors.adamw_step(self, [g if n == number else None for n, g in zip(steps, grads)], number, *hyper, grad_scale)
        self.steps = steps if len(set(steps)) > 1 else steps[0]


class AdamW(torch.optim.Optimizer):
    """AdamW with torch's vocabulary: ``p -= lr (m^ / (sqrt(v^) + eps) + weight_decay p)``.  The parameters of a group
    (contiguous, in device memory) are updated together, those of one type in one call of ``functors.adamw_step``; each
    goes by the number of steps that it has had a gradient for, and those that had other numbers than the rest take
    a call of their own.  A parameter that is frozen at the first step has no moments until it has a gradient.
    ``state_bits``: 32, or 8 for moments of a byte each.  A step that is captured into a graph keeps its number (the
    bias corrections) when it is replayed, and has to be preceded by one that is not."""

    _NOT_SAVED = ("params", "buckets", "outside")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def _buckets(self, group):
        """The moments of a group's parameters, by type and by when they joined."""
        if "buckets" not in group:
            group["buckets"], group["outside"], group["step"] = [], list(group["params"]), 0
            self._join(group, [p for p in group["params"] if p.requires_grad or p.grad is not None])
        elif group["outside"]:
            self._join(group, [p for p in group["outside"] if p.grad is not None])
        return group["buckets"]

    @staticmethod
    def _join(group, params):
        kinds = {}
        for p in params:
            kinds.setdefault(p.dtype, []).append(p)
        group["buckets"] += [_Moments(list_, group["state_bits"]) for list_ in kinds.values()]
        joined = {id(p) for p in params}
        group["outside"] = [p for p in group["outside"] if id(p) not in joined]

    def add_param_group(self, param_group):
        super().add_param_group({k: v for k, v in param_group.items() if k not in ("buckets", "outside", "step")})

    @torch.no_grad()
    def step(self, closure=None, grad_scale=None):
        """One update.  ``grad_scale``: a float32 tensor of one element that multiplies every gradient, or None."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            hyper = (group["lr"], *group["betas"], group["eps"], group["weight_decay"])
            for state in self._buckets(group):
                grads = [p.grad for p in state.params]
                state.update([g if g is None or g.is_contiguous() else g.contiguous() for g in grads], grad_scale, hyper)
                group["step"] = max(group["step"], state.steps if type(state.steps) is int else max(state.steps))
        return loss

    def state_dict(self):
        """Hyperparameters and moments of every group, with the parameters' places in it and their numbers of steps."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        groups = []
        for group in self.param_groups:
            place = {id(p): i for i, p in enumerate(group["params"])}
            moments = [{"params": [place[id(p)] for p in s.params], "steps": s.steps if type(s.steps) is int else list(s.steps), "sizes": list(s.sizes),
                        "m": s.m, "v": s.v, "m_scale": s.m_scale, "v_scale": s.v_scale} for s in self._buckets(group)]
            saved = {k: v for k, v in group.items() if k not in self._NOT_SAVED}
            groups.append({**saved, "moments": moments})
        state_dict = {"groups": groups}
        for hook in self._optimizer_state_dict_post_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        return state_dict

    def _places(self, group, saved):
        """Of each of the saved moments the parameters' places in the group, checked against it."""
        params = group["params"]
        if all("params" in m for m in saved["moments"]):
            places = [list(m["params"]) for m in saved["moments"]]
        else:  # (written before the places were: those that require gradients, by type)
            place = {id(p): i for i, p in enumerate(params)}
            places = [[place[id(p)] for p in s.params] for s in self._buckets(group)]
        every = [i for at in places for i in at]
        good = len(places) == len(saved["moments"]) and len(set(every)) == len(every) and all(0 <= i < len(params) for i in every)
        for at, m in zip(places, saved["moments"]):
            steps = m.get("steps", 0)
            good = good and [params[i].numel() for i in at] == list(m["sizes"]) and len({params[i].dtype for i in at}) == 1
            good = good and (type(steps) is int or len(steps) == len(at))
        if not good:
            raise ValueError("the saved state is of other parameters")
        return places

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        groups = state_dict["groups"]
        if len(groups) != len(self.param_groups):
            raise ValueError("the saved state has another number of parameter groups")
        if any(saved["state_bits"] != group["state_bits"] for group, saved in zip(self.param_groups, groups)):
            raise ValueError("the saved state's moments have another number of bits")
        all_places = [self._places(group, saved) for group, saved in zip(self.param_groups, groups)]
        for group, saved, places in zip(self.param_groups, groups, all_places):
            params = group["params"]
            lists = [[params[i] for i in at] for at in places]
            have = [[id(p) for p in s.params] for s in group.get("buckets", [])]
            if "buckets" not in group or have != [[id(p) for p in list_] for list_ in lists]:
                group["buckets"] = [_Moments(list_, group["state_bits"]) for list_ in lists]
                within = {id(p) for list_ in lists for p in list_}
                group["outside"] = [p for p in params if id(p) not in within]
            for s, moments in zip(group["buckets"], saved["moments"]):
                steps = moments.get("steps", saved["step"])
                s.steps = steps if type(steps) is int else list(steps)
                for k in ("m", "v", "m_scale", "v_scale"):
                    getattr(s, k).copy_(moments[k])
            group.update({k: v for k, v in saved.items() if k != "moments"})
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)
