"""8-bit moments at the ends of the floats' range, as unused neurons and gradients before clipping have them: second moments
below 2^-96 and among the denormals, and blocks whose largest magnitude lies beyond 2^60 or below 2^-60."""
import numpy as np
import pytest
import torch

from approxtrain_amd import functors
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)
SIZES = [1, 257, 70001]


def gradients(seed, scale):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * torch.exp2(torch.randint(-8, 3, (n,), generator=gen).float()) * scale).cuda() for n in SIZES]


@pytest.mark.parametrize("scale", [1e-12, 1e-13, 1e-15, 1e-17, 1e-19, 3e-20, 1e-21, 1e-24, 1e18])
def test_codes_are_the_definition_s_at_any_magnitude(scale):
    params = [g * 0.1 / scale for g in gradients(1, scale)]
    state = functors.AdamWState(params, state_bits=8)
    for step in (1, 2, 3):
        grads = gradients(10 + step, scale)
        before = [t.cpu().numpy().copy() for t in (state.m, state.m_scale, state.v, state.v_scale)]
        old = [p.cpu().numpy().copy() for p in params]
        functors.adamw_step(state, grads, step, **HYPER)
        after = [t.cpu().numpy() for t in (state.m, state.m_scale, state.v, state.v_scale)]
        for p, g, o, s, n in zip(params, grads, old, state.starts, SIZES):
            e = s + -(-n // 256) * 256
            full = [np.concatenate([t, np.zeros(e - s - n, np.float32)]) for t in (o, g.cpu().numpy())]
            want = ref.adamw_8bit(*full, before[0][s:e], before[1][s // 256:e // 256], before[2][s:e], before[3][s // 256:e // 256], step, **HYPER)
            assert np.array_equal(after[0][s:e], want[1]) and np.array_equal(after[1][s // 256:e // 256], want[2])
            assert np.array_equal(after[2][s:e], want[3]) and np.array_equal(after[3][s // 256:e // 256], want[4])
            new = p.cpu().numpy()
            assert (np.abs(new - want[0][:n]) <= 4 * 2.0 ** -24 * (np.abs(new) + np.abs(new - o))).all()


def test_tiny_and_ordinary_blocks_side_by_side():
    """A block whose roots leave the fast path's range leaves its neighbours' results as they are."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    g = torch.randn(1024, device="cuda", generator=gen)
    mixed = g.clone()
    mixed[300:512] *= 1e-17
    states = [functors.AdamWState([torch.ones(1024, device="cuda")], 8) for _ in range(2)]
    for s, grad in zip(states, (g, mixed)):
        functors.adamw_step(s, [grad], 1, **HYPER)
    for k in ("m", "v"):
        a, b = (getattr(s, k) for s in states)
        assert torch.equal(a[:256], b[:256]) and torch.equal(a[512:], b[512:])


@pytest.mark.parametrize("bits,dtype,sizes", [(32, torch.float32, (10_500_001, 10_999_998)), (32, torch.bfloat16, (15_000_001, 14_999_998)),
                                              (8, torch.float32, (16_000_001, 18_000_002)), (8, torch.bfloat16, (20_000_001, 1, 40_000_002))])
def test_steps_past_the_cache_are_those_through_it(bits, dtype, sizes):
    """All of a step's tensors are more than 320 MB; each alone, and all but one without gradients, are less."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    whole = [torch.empty(n + 1, device="cuda", dtype=dtype).normal_(generator=gen) for n in sizes]
    params = [t[i % 2:i % 2 + n] for i, (t, n) in enumerate(zip(whole, sizes))]
    alone = [p.clone() for p in params]
    state, parts = functors.AdamWState(params, bits), functors.AdamWState(alone, bits)
    for step in (1, 2):
        grads = [torch.empty(n, device="cuda", dtype=dtype).normal_(generator=gen) for n in sizes]
        functors.adamw_step(state, grads, step)
        for i in range(len(sizes)):
            functors.adamw_step(parts, [g if j == i else None for j, g in enumerate(grads)], step)
    for p, q in zip(params, alone):
        assert torch.equal(p, q)
    assert torch.equal(state.m, parts.m) and torch.equal(state.v, parts.v)
    if bits == 8:
        assert torch.equal(state.m_scale, parts.m_scale) and torch.equal(state.v_scale, parts.v_scale)
