"""The AdamW step against its definition in 64 bits, and with 8-bit moments against the definition rounded to 32
bits step by step.  An update is a handful of roundings of 2^-24 each: m and v take at most three, their sums
staying within |m| + |g| and v + g^2; the quotient takes six more."""
import numpy as np
import pytest
import torch

from approxtrain_amd import functors
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)
SIZES = [1, 255, 256, 257, 0, 3, 4096, 4097, 5000, 70001]
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def tensors(sizes, dtype, seed, scale, shift=0):
    g = torch.Generator().manual_seed(seed)
    got = []
    for n in sizes:
        t = torch.empty(n + shift, dtype=dtype, device="cuda")[shift:]
        t.copy_(torch.randn(n, generator=g) * scale * torch.exp2(torch.randint(-8, 3, (n,), generator=g).float()))
        got.append(t)
    return got


def host64(t):
    return t.detach().double().cpu().numpy()


def assert_update(p, m, v, want, before, g, dtype):
    """p, m, v of one tensor against the float64 update of the float64 ``before`` = (p, m, v) by gradient g."""
    u = 2.0 ** -24
    assert (np.abs(m - want[1]) <= 4 * u * (np.abs(before[1]) + np.abs(g))).all()
    assert (np.abs(v - want[2]) <= 5 * u * (before[2] + g * g) + 1e-45).all()
    change = np.abs(want[0] - before[0])
    # relative to the change: m, v and the quotient; relative to p: its product and sum
    off = 32 * u * (change + np.abs(before[0])) + 32 * u * HYPER["lr"] * (np.abs(before[1]) + np.abs(g)) / (np.sqrt(want[2]) + 1e-12)
    if dtype != torch.float32:
        off = off + torch.finfo(dtype).eps / 2 * np.abs(want[0]) * 1.01 + torch.finfo(dtype).tiny
    assert (np.abs(p - want[0]) <= off).all()


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("gdtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_three_steps_with_32_bit_moments(dtype, gdtype, shift):
    params = tensors(SIZES, DTYPES[dtype], 1, 0.1, shift)
    state = functors.AdamWState(params)
    assert state.m.numel() % 256 == 0 and state.m.dtype == torch.float32
    for step in (1, 2, 3):
        grads = tensors(SIZES, DTYPES[gdtype], 10 + step, 0.01, shift)
        before = [(host64(p), host64(state.m[s:s + n]), host64(state.v[s:s + n])) for p, s, n in zip(params, state.starts, SIZES)]
        functors.adamw_step(state, grads, step, **HYPER)
        for p, g, b, s, n in zip(params, grads, before, state.starts, SIZES):
            if n:
                assert_update(host64(p), host64(state.m[s:s + n]), host64(state.v[s:s + n]), ref.adamw(b[0], host64(g), b[1], b[2], step, **HYPER), b,
                              host64(g), DTYPES[dtype])


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("clip", [None, 0.37])
def test_steps_with_8_bit_moments(clip, shift):
    params = tensors(SIZES, torch.float32, 2, 0.1, shift)
    state = functors.AdamWState(params, state_bits=8)
    scale = None if clip is None else torch.tensor([clip], device="cuda")
    u = 2.0 ** -24
    for step in (1, 2, 3, 4):
        grads = tensors(SIZES, torch.float32, 20 + step, 0.01, shift)
        before = [t.cpu().numpy().copy() for t in (state.m, state.m_scale, state.v, state.v_scale)]
        old = [p.cpu().numpy().copy() for p in params]
        functors.adamw_step(state, grads, step, grad_scale=scale, **HYPER)
        after = [t.cpu().numpy() for t in (state.m, state.m_scale, state.v, state.v_scale)]
        for p, g, o, s, n in zip(params, grads, old, state.starts, SIZES):
            if n == 0:
                continue
            e = s + -(-n // 256) * 256
            full = [np.concatenate([t, np.zeros(e - s - n, np.float32)]) for t in (o, g.cpu().numpy())]
            want = ref.adamw_8bit(*full, before[0][s:e], before[1][s // 256:e // 256], before[2][s:e], before[3][s // 256:e // 256], step,
                                  grad_scale=clip, **HYPER)
            assert np.array_equal(after[0][s:e], want[1]) and np.array_equal(after[1][s // 256:e // 256], want[2])
            assert np.array_equal(after[2][s:e], want[3]) and np.array_equal(after[3][s // 256:e // 256], want[4])
            new = p.cpu().numpy()
            assert (np.abs(new - want[0][:n]) <= 4 * u * (np.abs(new) + np.abs(new - o))).all()
    values, roots = state.first_moments().cpu().numpy(), state.second_roots().cpu().numpy()
    assert np.array_equal(values, ref.decode(after[0], after[1], False)) and np.array_equal(roots, ref.decode(after[2], after[3], True))


def test_all_codes_read_back():
    state = functors.AdamWState([torch.zeros(512, device="cuda")], state_bits=8)
    codes = torch.arange(512, device="cuda").to(torch.uint8)
    state.m.copy_(codes), state.v.copy_(codes)
    scales = torch.tensor([0.37, 3e-30], device="cuda")
    state.m_scale.copy_(scales), state.v_scale.copy_(scales)
    c, s = codes.cpu().numpy(), scales.cpu().numpy()
    assert np.array_equal(state.first_moments().cpu().numpy(), ref.decode(c, s, False))
    assert np.array_equal(state.second_roots().cpu().numpy(), ref.decode(c, s, True))


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_holds_and_missing_gradients(bits):
    """Two hundred and fifty tensors, every third without a gradient, as one by one."""
    sizes = [1 + (37 * i) % 900 for i in range(250)]
    params, grads = tensors(sizes, torch.float32, 3, 0.1), tensors(sizes, torch.float32, 4, 0.01)
    alone = [p.clone() for p in params]
    some = [None if i % 3 == 2 else g for i, g in enumerate(grads)]
    state = functors.AdamWState(params, bits)
    for step in (1, 2):
        functors.adamw_step(state, some, step, **HYPER)
    for i, (p, a, g) in enumerate(zip(params, alone, some)):
        if g is not None:
            one = functors.AdamWState([a], bits)
            for step in (1, 2):
                functors.adamw_step(one, [g], step, **HYPER)
            assert torch.equal(state.m[state.starts[i]:state.starts[i] + one.m.numel()], one.m), i
        assert torch.equal(p, a), i


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite_stay_in_their_block(bits):
    params = [torch.ones(1000, device="cuda")]
    state = functors.AdamWState(params, bits)
    g = torch.full((1000,), 0.1, device="cuda")
    g[300], g[301] = float("nan"), float("inf")
    functors.adamw_step(state, [g], 1, **HYPER)
    bad = ~torch.isfinite(params[0])
    assert bad[300] and bad[301] and int(bad.sum()) == 2
    moments = torch.isfinite(state.first_moments())
    reach = slice(256, 512) if bits == 8 else slice(300, 302)
    assert not moments[reach].any() and moments[:256].all() and moments[512:].all()


def test_zero_gradients_and_zero_moments():
    for bits in (32, 8):
        params = [torch.full((300,), 2.0, device="cuda")]
        state = functors.AdamWState(params, bits)
        functors.adamw_step(state, [torch.zeros(300, device="cuda")], 1, **HYPER)
        keep = np.float32(1 - HYPER["lr"] * HYPER["weight_decay"])
        assert torch.equal(params[0].cpu(), torch.full((300,), float(np.float32(2.0) * keep)))
        assert not state.first_moments().any() and not state.second_roots().any()


def test_autograd_notices_the_update():
    p = torch.ones(10, device="cuda", requires_grad=True)
    y = (p * p).sum()
    functors.adamw_step(functors.AdamWState([p]), [torch.ones(10, device="cuda")], 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    p, g = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    for bad in ([], [p.double()], [torch.zeros(4, 6, device="cuda").t()], [p, p.bfloat16()]):
        with pytest.raises((ValueError, TypeError)):
            functors.AdamWState(bad)
    with pytest.raises(ValueError, match="state_bits"):
        functors.AdamWState([p], 16)
    state = functors.AdamWState([p])
    for grads in ([g[:9]], [g.cpu()], [torch.zeros(20, device="cuda")[::2]], [g, g], []):
        with pytest.raises(ValueError):
            functors.adamw_step(state, grads, 1)
    with pytest.raises(TypeError, match="gradients"):
        functors.adamw_step(state, [g.double()], 1)
    with pytest.raises(ValueError, match="grad_scale"):
        functors.adamw_step(state, [g], 1, grad_scale=torch.ones(1))
    for hyper in (dict(step=0), dict(step=1, beta1=1.0), dict(step=1, beta2=-0.1), dict(step=1, eps=-1.0)):
        with pytest.raises(RuntimeError, match="adamw"):
            functors.adamw_step(state, [g], **hyper)
    functors.adamw_step(state, [None], 1)
    assert not p.any() and not state.m.any()


@pytest.mark.parametrize("bits,dtype,sizes", [(32, torch.float32, (15_000_001, 14_999_998)), (32, torch.bfloat16, (15_000_001, 14_999_998)),
                                              (8, torch.bfloat16, (60_000_001, 1, 60_000_002))])
def test_moments_larger_than_the_cache(bits, dtype, sizes):
    """More than 224 MB of moments: every tensor as it steps alone, on addresses that four elements do and do not share."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    whole = [torch.empty(n + 1, device="cuda", dtype=dtype).normal_(generator=gen) for n in sizes]
    params = [t[i % 2:i % 2 + n] for i, (t, n) in enumerate(zip(whole, sizes))]
    alone = [p.clone() for p in params]
    state, states = functors.AdamWState(params, bits), [functors.AdamWState([p], bits) for p in alone]
    for step in (1, 2):
        grads = [torch.empty(n, device="cuda", dtype=dtype).normal_(generator=gen) for n in sizes]
        functors.adamw_step(state, grads, step)
        for s, g in zip(states, grads):
            functors.adamw_step(s, [g], step)
    for p, q in zip(params, alone):
        assert torch.equal(p, q)
    assert torch.equal(state.m, torch.cat([s.m for s in states])) and torch.equal(state.v, torch.cat([s.v for s in states]))
    if bits == 8:
        assert torch.equal(state.m_scale, torch.cat([s.m_scale for s in states])) and torch.equal(state.v_scale, torch.cat([s.v_scale for s in states]))
