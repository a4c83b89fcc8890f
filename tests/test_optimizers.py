"""The optimizer class's host side: which parameters it steps, by which step number, what it saves.  The native calls are
replaced by the same formulas in 64 bits on host tensors."""
import copy
import pickle

import pytest
import torch

from approxtrain_amd import functors
from approxtrain_amd.optimizers import AdamW


class HostCalls:
    """Stands in for ``_native``: tensors on the host, moments of 32 bits."""

    class TensorList:
        def __init__(self, sizes, dtype, device):
            self.sizes = sizes
            self.cannot_be_copied = lambda: None  # (nor can the native one)

        def __reduce__(self):
            raise TypeError("cannot pickle 'TensorList' object")

        def check(self, tensors, name):
            assert [t.numel() for t in tensors] == self.sizes
            if len({t.dtype for t in tensors}) != 1:
                raise ValueError(f"{name} differ in type")

    @staticmethod
    def adamw_step(list_, params, grads, bits, m, v, m_scale, v_scale, step, lr, beta1, beta2, eps, decay, grad_scale):
        assert bits == 32 and len(grads) == len(params) == len(list_.sizes)
        at = 0
        for p, g in zip(params, grads):
            n = p.numel()
            if g is not None:
                ms, vs, g = m[at:at + n].double(), v[at:at + n].double(), g.reshape(-1).double() * (1.0 if grad_scale is None else float(grad_scale))
                ms, vs = beta1 * ms + (1 - beta1) * g, beta2 * vs + (1 - beta2) * g * g
                new = p.detach().reshape(-1).double() * (1 - lr * decay) - lr * (ms / (1 - beta1 ** step)) / ((vs / (1 - beta2 ** step)).sqrt() + eps)
                p.detach().copy_(new.reshape(p.shape)), m[at:at + n].copy_(ms), v[at:at + n].copy_(vs)
            at += -(-n // 256) * 256


@pytest.fixture(autouse=True)
def host_calls(monkeypatch):
    monkeypatch.setattr(functors, "_native", lambda: HostCalls)
    monkeypatch.setattr(functors, "_device_of", lambda t, name: 0)


SHAPES = [(3, 5), (7,), (300,), (2, 2)]
HYPER = dict(lr=1e-2, betas=(0.8, 0.9), eps=1e-6, weight_decay=0.1)


def pair(shapes=SHAPES, **kw):
    """The same parameters twice, under this optimizer and under torch's."""
    gen = torch.Generator().manual_seed(1)
    mine = [torch.nn.Parameter(torch.randn(s, generator=gen)) for s in shapes]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    return mine, theirs, AdamW(mine, **{**HYPER, **kw}), torch.optim.AdamW(theirs, foreach=False, **{**HYPER, **kw})


def step(mine, theirs, opt, other, seed, which):
    gen = torch.Generator().manual_seed(seed)
    for i, (p, q) in enumerate(zip(mine, theirs)):
        g = torch.randn(p.shape, generator=gen)
        p.grad, q.grad = (g.clone(), g.clone()) if i in which else (None, None)
    opt.step(), other.step()


def assert_same(mine, theirs):
    """Torch's own steps round every operation to 32 bits, a dozen of them, of values up to |p| + 10 lr; ours rounds once."""
    for i, (p, q) in enumerate(zip(mine, theirs)):
        assert bool(((p - q).abs() <= 40 * 2.0 ** -24 * (q.abs() + 0.1)).all()), i


def test_parameters_that_were_frozen_at_the_first_step_are_stepped_once_they_have_gradients():
    mine, theirs, opt, other = pair()
    for t in (mine, theirs):
        t[1].requires_grad_(False), t[3].requires_grad_(False)
    step(mine, theirs, opt, other, 1, {0, 2})
    opt.state_dict()
    assert_same(mine, theirs)
    for t in (mine, theirs):
        t[1].requires_grad_(True)
    step(mine, theirs, opt, other, 2, {0, 1, 2})
    assert_same(mine, theirs)
    for t in (mine, theirs):
        t[3].requires_grad_(True)
    step(mine, theirs, opt, other, 3, {0, 1, 2, 3})
    step(mine, theirs, opt, other, 4, {0, 1, 2, 3})
    assert_same(mine, theirs)


def test_a_gradient_that_comes_late_or_is_absent_now_and_then_counts_its_own_steps():
    """The corrections of a tensor's moments go by the steps that it has taken, not by its group's."""
    mine, theirs, opt, other = pair()
    for seed, which in enumerate(({0, 1}, {0, 1}, set(), {0}, {0, 2}, {0, 1, 2, 3}, {1, 2, 3}, {0, 1, 2, 3})):
        step(mine, theirs, opt, other, 10 + seed, which)
        assert_same(mine, theirs)
    assert opt.param_groups[0]["step"] == 6


def test_a_saved_state_goes_on_with_late_parameters_and_their_own_numbers():
    mine, theirs, opt, other = pair()
    for t in (mine, theirs):
        t[2].requires_grad_(False)
    step(mine, theirs, opt, other, 1, {0, 1, 3})
    step(mine, theirs, opt, other, 2, {0, 1, 2})
    saved = opt.state_dict()
    copies = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    resumed = AdamW(copies, lr=1.0)
    resumed.load_state_dict(saved)
    for seed, which in ((3, {0, 1, 2, 3}), (4, {1, 2})):
        gen = torch.Generator().manual_seed(seed)
        for i, p in enumerate(copies):
            g = torch.randn(p.shape, generator=gen)
            p.grad = g if i in which else None
        resumed.step()
        step(mine, theirs, opt, other, seed, which)
    for p, q in zip(mine, copies):
        assert torch.equal(p, q)
    assert_same(mine, theirs)


def test_states_saved_without_numbers_of_their_own_go_by_the_group_s():
    """As earlier versions wrote them: the moments of the parameters that require gradients, by type, and one step number."""
    mine, theirs, opt, other = pair()
    for seed in (1, 2, 3):
        step(mine, theirs, opt, other, seed, {0, 1, 2, 3})
    saved = opt.state_dict()
    for group in saved["groups"]:
        for moments in group["moments"]:
            for k in set(moments) - {"sizes", "m", "v", "m_scale", "v_scale"}:
                del moments[k]
    resumed = AdamW(mine)
    resumed.load_state_dict(saved)
    step(mine, theirs, resumed, other, 4, {0, 1, 2, 3})
    assert_same(mine, theirs)


def test_states_of_other_parameters_are_refused_and_change_nothing():
    mine, theirs, opt, other = pair()
    step(mine, theirs, opt, other, 1, {0, 1, 2, 3})
    saved = opt.state_dict()
    fewer, shapes, types = mine[:3], [torch.nn.Parameter(torch.zeros(s)) for s in ((3, 5), (8,), (300,), (2, 2))], mine[:3] + [mine[3].detach().bfloat16()]
    for params in (fewer, shapes, types):
        target = AdamW(params, lr=0.5)
        with pytest.raises(ValueError, match="other parameters"):
            target.load_state_dict(saved)
        assert target.param_groups[0]["lr"] == 0.5
    with pytest.raises(ValueError, match="parameter groups"):
        AdamW([{"params": mine[:2]}, {"params": mine[2:]}]).load_state_dict(saved)
    with pytest.raises(ValueError, match="bits"):
        AdamW(mine, state_bits=8).load_state_dict(saved)


def test_an_optimizer_that_has_stepped_can_be_copied_and_pickled():
    mine, theirs, opt, other = pair()
    step(mine, theirs, opt, other, 1, {0, 1, 2})
    for again in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt)), copy.deepcopy(opt)):
        params, (twin, reference) = again.param_groups[0]["params"], copy.deepcopy([theirs, other])
        assert params[0] is not mine[0] and again.param_groups[0]["buckets"][0].params[0] is params[0]
        for seed in (2, 3):
            step(params, twin, again, reference, seed, {0, 1, 2, 3})
        assert_same(params, twin)
    step(mine, theirs, opt, other, 4, {1, 3})
    assert_same(mine, theirs)


def test_registered_hooks_run_around_saving_and_loading():
    mine, theirs, opt, other = pair()
    step(mine, theirs, opt, other, 1, {0, 1, 2, 3})
    seen = []
    opt.register_state_dict_pre_hook(lambda o: seen.append(("saving", o is opt)))
    opt.register_state_dict_post_hook(lambda o, d: {**d, "note": 5})
    saved = opt.state_dict()
    assert saved["note"] == 5 and seen == [("saving", True)]
    target = AdamW(mine, lr=1.0)

    def unwrap(o, d):
        seen.append(d["note"])
        d["note"] = None  # (a hook may change what it is given: a shallow copy)
        return {"groups": d["groups"]}

    target.register_load_state_dict_pre_hook(unwrap)
    target.register_load_state_dict_post_hook(lambda o: seen.append(o.param_groups[0]["lr"]))
    target.load_state_dict(saved)
    assert seen == [("saving", True), 5, HYPER["lr"]] and saved["note"] == 5
