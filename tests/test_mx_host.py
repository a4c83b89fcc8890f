"""Refusals of the 4-bit products and of the optimizer's step that need no device: they come back before any
kernel could run."""
import ctypes as C

import pytest
import torch

from approxtrain_amd import functors, load_library, math_ops
from approxtrain_amd._lib import AdamWHyper

A = 1 << 20  # an address that is never read


def lib():
    return load_library()


def test_operand_sizes():
    size = lib().amsim_mxfp4_operand_workspace_bytes
    assert size(1, 1) == 1024 + 256 and size(16, 128) == 1024 + 256 and size(17, 129) == 2 * 2 * 1024 + 2 * 256
    assert size(65, 128) == 5 * 1024 + 2 * 256
    assert size(4096, 4096) == 4096 * 4096 * 17 // 32
    assert size(-1, 5) == size(5, -1) == size(1 << 31, 1) == size(1, 1 << 31) == size((1 << 31) - 1, (1 << 31) - 1) == 0


@pytest.mark.parametrize("args,status", [
    ((A, 3, 4, 4, 4, A, A, None), 1), ((A, -1, 4, 4, 4, A, A, None), 1), ((A, 0, 0, 4, 4, A, A, None), 1), ((A, 0, 4, 0, 4, A, A, None), 1),
    ((A, 0, 4, 4, 3, A, A, None), 1), ((None, 0, 4, 4, 4, A, A, None), 1), ((A, 0, 4, 4, 4, None, None, None), 1),
    ((A, 0, 4, 4, 4, A + 8, None, None), 1), ((A + 2, 0, 4, 4, 4, A, None, None), 1), ((A + 1, 1, 4, 4, 4, A, None, None), 1),
    ((A, 0, -4, 4, 4, A, A, None), 6), ((A, 0, 1 << 31, 4, 4, A, A, None), 6), ((A, 0, 1 << 30, 1 << 15, 1 << 15, A, A, None), 6)])
def test_quantize_refuses(args, status):
    assert lib().amsim_mxfp4_quantize(*args) == status


@pytest.mark.parametrize("args,status", [
    ((A, 4, 4, 5, A, None), 1), ((None, 4, 4, 0, A, None), 1), ((A, 4, 4, 0, None, None), 1), ((A, 0, 4, 0, A, None), 1), ((A, 4, 0, 0, A, None), 1),
    ((A + 4, 4, 4, 0, A, None), 1), ((A, 4, 4, 0, A + 4, None), 1), ((A, 4, 1 << 31, 0, A, None), 6)])
def test_dequantize_refuses(args, status):
    assert lib().amsim_mxfp4_dequantize(*args) == status


def matmul(a=A, b=A, m=4, n=4, k=4, bias=None, bias_dtype=0, act=0, out=A, out_dtype=0, ws=None, nbytes=0):
    return lib().amsim_mxfp4_matmul(a, b, m, n, k, bias, bias_dtype, act, out, out_dtype, ws, nbytes, None)


def linear(x=A, dtype=0, stride=4, w=A, m=4, n=4, k=4, bias=None, bias_dtype=0, act=0, out=A, ws=A, nbytes=1 << 30):
    return lib().amsim_mxfp4_linear(x, dtype, stride, w, m, n, k, bias, bias_dtype, act, out, ws, nbytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(a=None), 1), (dict(b=None), 1), (dict(out=None), 1), (dict(m=0), 1), (dict(n=0), 1), (dict(k=0), 1), (dict(out_dtype=3), 1),
    (dict(bias=A, bias_dtype=9), 1), (dict(act=2), 1), (dict(act=-1), 1), (dict(a=A + 4), 1), (dict(b=A + 8), 1), (dict(out=A + 4), 1),
    (dict(bias=A + 1), 1), (dict(bias=A + 1, bias_dtype=1), 1), (dict(m=-1), 6), (dict(n=1 << 31), 6), (dict(m=1 << 30, n=1 << 30), 6)])
def test_matmul_refuses(bad, status):
    assert matmul(**bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), 1), (dict(w=None), 1), (dict(out=None), 1), (dict(dtype=3), 1), (dict(stride=3), 1), (dict(x=A + 2), 1), (dict(x=A + 1, dtype=1), 1),
    (dict(w=A + 8), 1), (dict(m=0), 1), (dict(act=5), 1), (dict(k=1 << 31), 6)])
def test_linear_refuses(bad, status):
    assert linear(**bad) == status


def test_missing_workspaces_are_refused():
    need = lib().amsim_mxfp4_matmul_workspace_bytes(8, 8, 1 << 20)
    assert need > 0 and matmul(m=8, n=8, k=1 << 20) == 5 and matmul(m=8, n=8, k=1 << 20, ws=A + 16, nbytes=need) == 5
    assert matmul(m=8, n=8, k=1 << 20, ws=A, nbytes=need - 1) == 5
    assert lib().amsim_mxfp4_linear_workspace_bytes(4096, 64, 256) > 0
    assert linear(m=4096, n=64, k=256, stride=256, ws=None, nbytes=0) == 5


@pytest.mark.parametrize("bad", [dict(step=0), dict(beta1=1.0), dict(beta2=1.0), dict(beta1=-0.5), dict(eps=-1e-8), dict(beta2=float("nan"))])
def test_adamw_refuses_hyperparameters(bad):
    h = dict(step=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0)
    h.update(bad)
    one = (C.c_void_p * 1)(A)
    assert lib().amsim_adamw_step(1, one, one, (C.c_int64 * 1)(8), 0, 0, 32, A, A, None, None, C.byref(AdamWHyper(**h)), None, None) == 1


@pytest.mark.parametrize("bad,status", [
    (dict(p=None), 1), (dict(p=A + 2), 1), (dict(g=A + 1), 1), (dict(n=-1), 1), (dict(m=None), 1), (dict(m=A + 8), 1), (dict(bits=16), 1),
    (dict(bits=8), 1), (dict(pd=3), 1), (dict(gd=-1), 1), (dict(n=(1 << 35) + 1), 6), (dict(count=-1), 1), (dict(hyper=False), 1)])
def test_adamw_refuses(bad, status):
    v = dict(p=A, g=A, n=8, m=A, bits=32, pd=0, gd=0, count=1, hyper=True)
    v.update(bad)
    h = C.byref(AdamWHyper(1, 1e-3, 0.9, 0.999, 1e-8, 0.0)) if v["hyper"] else None
    rc = lib().amsim_adamw_step(v["count"], (C.c_void_p * 1)(v["p"]), (C.c_void_p * 1)(v["g"]), (C.c_int64 * 1)(v["n"]), v["pd"], v["gd"], v["bits"],
                                v["m"], A, None, None, h, None, None)
    assert rc == status


def test_adamw_of_nothing_launches_nothing():
    h = C.byref(AdamWHyper(1, 1e-3, 0.9, 0.999, 1e-8, 0.0))
    assert lib().amsim_adamw_step(0, None, None, None, 0, 0, 32, None, None, None, None, h, None, None) == 0
    assert lib().amsim_adamw_step(1, (C.c_void_p * 1)(None), (C.c_void_p * 1)(None), (C.c_int64 * 1)(0), 0, 0, 32, None, None, None, None, h, None, None) == 0
    assert lib().amsim_adamw_state_values(A, A, 0, 0, A, None) == 0
    assert lib().amsim_adamw_state_values(A, A, 1, 0, A + 4, None) == 1 and lib().amsim_adamw_state_values(A, A, -1, 0, A, None) == 1


def test_tensors_that_are_not_on_a_device_are_refused():
    x = torch.zeros(4, 4)
    for call in (lambda: functors.mxfp4_quantize(x), lambda: functors.mxfp4_quantize_both(x), lambda: math_ops.linearmx(x, x),
                 lambda: functors.AdamWState([x])):
        with pytest.raises(TypeError, match="device memory"):
            call()
    with pytest.raises(ValueError, match="axis"):
        functors.mxfp4_quantize(x, axis=3)
    with pytest.raises(TypeError, match="MXTensor"):
        functors.mxfp4_linear(x, x)
    with pytest.raises(ValueError, match="linearmx"):
        math_ops.linearmx(x, torch.zeros(5, 4))
    with pytest.raises(ValueError, match="no tensors"):
        functors.AdamWState([])


def test_calls_without_a_derivative_refuse_what_would_need_one():
    """They came back without a graph, and a branch behind them lost its gradient without a word."""
    x, b = torch.zeros(4, 4), torch.zeros(4)
    w = functors.MXTensor(torch.zeros(1280, dtype=torch.uint8), 4, 4)
    xg, bg = x.clone().requires_grad_(), b.clone().requires_grad_()
    calls = (lambda x, b: functors.mxfp4_linear(x, w, b), lambda x, b: functors.mxfp4_matmul(w, w, b))
    for call, args in ((calls[0], (xg, b)), (calls[0], (x, bg)), (calls[0], (xg * 2, None)), (calls[1], (None, bg))):
        with pytest.raises(RuntimeError, match="no gradient"):
            call(*args)
        with torch.no_grad(), pytest.raises(TypeError, match="device memory"):
            call(*args)
    with torch.autograd.forward_ad.dual_level():
        for call, args in ((calls[0], (torch.autograd.forward_ad.make_dual(x, x), None)), (calls[0], (x, torch.autograd.forward_ad.make_dual(b, b))),
                           (calls[1], (None, torch.autograd.forward_ad.make_dual(b, b)))):
            with pytest.raises(TypeError, match="forward-mode"):
                call(*args)


def test_bias_gradients_of_more_columns_than_a_launch_takes_are_refused():
    """Their sums take a workgroup of 1024 for 16 columns: the launch failed behind others that had been made."""
    n = 1 << 26
    need = lib().amsim_mxfp4_dense_grad_workspace_bytes(1, n, 1)
    assert need > 0
    assert lib().amsim_mxfp4_dense_grad(A, 0, n, None, None, None, 1, n, 1, None, None, 0, A, 0, A, need, None) == 6


@pytest.mark.parametrize("python,native", [("false", False), ("python3", True)])
def test_the_library_builds_where_torch_is_not(python, native):
    """From C it needs hipcc alone; the module for torch's tensors is built where torch is found."""
    import os
    import subprocess
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "approxtrain_amd", "csrc")
    run = subprocess.run(["make", "-n", "-B", f"PYTHON={python}"], cwd=folder, capture_output=True, text=True, check=True)
    assert "-o ../libamsim.so" in run.stdout and ("-o ../_native.so" in run.stdout) == native
