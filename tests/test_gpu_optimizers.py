"""The optimizer class on the device: parameters that join late or miss gradients, against each stepped by itself."""
import copy
import pickle

import pytest
import torch

from approxtrain_amd import functors
from approxtrain_amd.optimizers import AdamW

pytestmark = pytest.mark.gpu

SHAPES = [((30, 40), torch.float32), ((7,), torch.bfloat16), ((300,), torch.float32), ((5, 5), torch.bfloat16), ((257,), torch.float32)]


def parameters():
    gen = torch.Generator(device="cuda").manual_seed(3)
    return [torch.nn.Parameter(torch.randn(s, device="cuda", generator=gen).to(t)) for s, t in SHAPES]


@pytest.mark.parametrize("bits", [32, 8])
def test_late_and_missing_gradients(bits):
    params = parameters()
    alone = [p.detach().clone() for p in params]
    states, numbers = [functors.AdamWState([a], bits) for a in alone], [0] * len(alone)
    params[0].requires_grad_(False), params[3].requires_grad_(False)
    opt = AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for which in ({1, 2, 4}, {1, 4}, {0, 1, 2, 4}, {0, 1, 2, 3, 4}, {2}, {0, 1, 2, 3, 4}):
        for i, p in enumerate(params):
            p.grad = None
            if i in which:
                p.requires_grad_()
                p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)
                numbers[i] += 1
                functors.adamw_step(states[i], [p.grad], numbers[i], 1e-2, 0.9, 0.999, 1e-8, 0.1)
        opt.step()
        for i, (p, a) in enumerate(zip(params, alone)):
            assert torch.equal(p, a), i


def test_late_gradients_against_torch():
    """The first update of a parameter that joins after many steps is lr long, as a first update is."""
    params, theirs = parameters()[::2], parameters()[::2]
    opt, other = AdamW(params, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.1)
    gen = torch.Generator(device="cuda").manual_seed(5)
    for number in range(40):
        for i, (p, q) in enumerate(zip(params, theirs)):
            g = torch.randn(p.shape, device="cuda", generator=gen)
            p.grad, q.grad = (g, g.clone()) if i or number >= 30 else (None, None)
        opt.step(), other.step()
    for p, q in zip(params, theirs):
        # either side rounds p and the update a dozen times a step, updates of at most 10 lr
        assert bool(((p - q).abs() <= 40 * 24 * 2.0 ** -24 * (q.abs() + 0.1)).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copy_goes_on_as_its_original(bits):
    params = parameters()
    opt = AdamW(params, state_bits=bits)
    gen = torch.Generator(device="cuda").manual_seed(6)
    for p in params:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)
    opt.step()
    for make in (copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))):
        again = make(opt)
        theirs = again.param_groups[0]["params"]
        for p, q in zip(params, theirs):
            assert p is not q and torch.equal(p, q)
            p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)
            q.grad = p.grad.clone()
        opt.step(), again.step()
        for p, q in zip(params, theirs):
            assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_made_in_a_capture_are_refused(bits):
    """Their clearing would be part of the graph: every replay would step from moments of zero."""
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.ones(300, device="cuda")
    opt = AdamW([p], state_bits=bits)
    torch.cuda.synchronize()
    for call in (opt.step, lambda: functors.AdamWState([p], bits)):
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    torch.cuda.synchronize()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    twin = torch.ones(300, device="cuda")
    state = functors.AdamWState([twin], bits)
    functors.adamw_step(state, [p.grad], 1)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        functors.adamw_step(state, [p.grad], 2)
        assert torch.equal(p, twin)
