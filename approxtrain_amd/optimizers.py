"""``AdamW`` over all of a model's tensors in a launch or two, moments in 32 bits or in 8 (the reference trains with
Keras's optimizers)."""
import torch

from . import functors


class AdamW(torch.optim.Optimizer):
    """AdamW with torch's vocabulary: ``p -= lr (m^ / (sqrt(v^) + eps) + weight_decay p)``.  The parameters of a group
    (contiguous, in device memory) are updated together, those of one type in one call of ``functors.adamw_step``.
    ``state_bits``: 32, or 8 for moments of a byte each.  A step that is captured into a graph keeps its number (the
    bias corrections) when it is replayed."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def _buckets(self, group):
        """A group's parameters by type, each list with its moments."""
        known = group.get("buckets")
        if known is None:
            kinds = {}
            for p in group["params"]:
                if p.requires_grad:
                    kinds.setdefault(p.dtype, []).append(p)
            known = group["buckets"] = [functors.AdamWState(list_, group["state_bits"]) for list_ in kinds.values()]
            group["step"] = 0
        return known

    def add_param_group(self, param_group):
        super().add_param_group({k: v for k, v in param_group.items() if k not in ("buckets", "step")})

    @torch.no_grad()
    def step(self, closure=None, grad_scale=None):
        """One update.  ``grad_scale``: a float32 tensor of one element that multiplies every gradient, or None."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            buckets = self._buckets(group)
            group["step"] += 1
            for state in buckets:
                grads = [p.grad if p.grad is None or p.grad.is_contiguous() else p.grad.contiguous() for p in state.params]
                functors.adamw_step(state, grads, group["step"], group["lr"], *group["betas"], group["eps"], group["weight_decay"], grad_scale)
        return loss

    def state_dict(self):
        """Hyperparameters, step numbers and moments of every group."""
        groups = []
        for group in self.param_groups:
            saved = {k: v for k, v in group.items() if k not in ("params", "buckets")}
            saved["moments"] = [{"sizes": list(s.sizes), "m": s.m, "v": s.v, "m_scale": s.m_scale, "v_scale": s.v_scale} for s in self._buckets(group)]
            saved["step"] = group["step"]
            groups.append(saved)
        return {"groups": groups}

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        groups = state_dict["groups"]
        if len(groups) != len(self.param_groups):
            raise ValueError("the saved state has another number of parameter groups")
        for group, saved in zip(self.param_groups, groups):
            if saved["state_bits"] != group["state_bits"]:
                raise ValueError("the saved state's moments have another number of bits")
            buckets = self._buckets(group)
            if [list(s.sizes) for s in buckets] != [list(m["sizes"]) for m in saved["moments"]]:
                raise ValueError("the saved state is of other parameters")
            for s, moments in zip(buckets, saved["moments"]):
                for k in ("m", "v", "m_scale", "v_scale"):
                    getattr(s, k).copy_(moments[k])
            group.update({k: v for k, v in saved.items() if k != "moments"})
