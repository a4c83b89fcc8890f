"""Refusals of the 8-bit products that need no device: they come back before any kernel could run."""
import ctypes as C

import pytest
import torch

from approxtrain_amd import functors, layers, load_library, math_ops

A = 1 << 20  # an address that is never read


def lib():
    return load_library()


def test_operand_sizes():
    size = lib().amsim_i8_operand_workspace_bytes
    assert size(1, 1) == 1024 + 4 and size(16, 64) == 1024 + 64 and size(17, 65) == 2 * 2 * 1024 + 68
    assert size(4096, 4096) == 4096 * 4096 + 4 * 4096
    assert size(1, 1 << 21) == (1 << 15) * 1024 + 4 and size(1, (1 << 21) + 1) == 0
    assert size(-1, 5) == size(5, -1) == size(0, 5) == size(5, 0) == size(1 << 31, 1) == 0
    kept = lib().amsim_i8_kept_workspace_bytes
    assert kept(17, 65) == 4 * 1024 + 4 * 65 and kept(0, 4) == 0 and kept(4, 1 << 22) == 0


def quantize(x=A, dtype=0, rows=4, cols=4, stride=4, by_rows=A, by_columns=A, ws=A, nbytes=1 << 20):
    return lib().amsim_i8_quantize(x, dtype, rows, cols, stride, by_rows, by_columns, ws, nbytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=3), 1), (dict(dtype=-1), 1), (dict(rows=0), 1), (dict(cols=0), 1), (dict(stride=3), 1), (dict(x=None), 1), (dict(by_rows=None, by_columns=None), 1),
    (dict(by_rows=A + 8), 1), (dict(by_columns=A + 4), 1), (dict(x=A + 2), 1), (dict(x=A + 1, dtype=1), 1), (dict(ws=None), 5), (dict(ws=A + 64), 5), (dict(nbytes=16), 5),
    (dict(rows=-4), 6), (dict(cols=1 << 31), 6), (dict(cols=(1 << 21) + 1, stride=1 << 22), 6), (dict(rows=(1 << 21) + 1), 6), (dict(rows=1 << 30, by_columns=None), 6)])
def test_quantize_refuses(bad, status):
    assert quantize(**bad) == status


@pytest.mark.parametrize("args,status", [
    ((A, 4, 4, 5, A, None), 1), ((None, 4, 4, 0, A, None), 1), ((A, 4, 4, 0, None, None), 1), ((A, 0, 4, 0, A, None), 1), ((A, 4, 0, 0, A, None), 1),
    ((A + 4, 4, 4, 0, A, None), 1), ((A, 4, 4, 0, A + 4, None), 1), ((A, 4, 1 << 22, 0, A, None), 6), ((A, 1 << 30, 64, 0, A, None), 6)])
def test_dequantize_refuses(args, status):
    assert lib().amsim_i8_dequantize(*args) == status


def matmul(a=A, b=A, m=4, n=4, k=4, bias=None, bias_dtype=0, act=0, out=A, out_dtype=0, ws=None, nbytes=0):
    return lib().amsim_i8_matmul(a, b, m, n, k, bias, bias_dtype, act, out, out_dtype, ws, nbytes, None)


def linear(x=A, dtype=0, stride=4, w=A, m=4, n=4, k=4, bias=None, bias_dtype=0, act=0, out=A, ws=A, nbytes=1 << 30):
    return lib().amsim_i8_linear(x, dtype, stride, w, m, n, k, bias, bias_dtype, act, out, ws, nbytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(a=None), 1), (dict(b=None), 1), (dict(out=None), 1), (dict(m=0), 1), (dict(n=0), 1), (dict(k=0), 1), (dict(out_dtype=3), 1),
    (dict(bias=A, bias_dtype=9), 1), (dict(act=2), 1), (dict(act=-1), 1), (dict(a=A + 4), 1), (dict(b=A + 8), 1), (dict(out=A + 4), 1),
    (dict(bias=A + 1), 1), (dict(m=-1), 6), (dict(n=1 << 31), 6), (dict(m=1 << 30, n=1 << 30), 6), (dict(k=1 << 22), 6), (dict(m=1000, n=1000, k=100000), 5)])
def test_matmul_refuses(bad, status):
    assert matmul(**bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), 1), (dict(w=None), 1), (dict(out=None), 1), (dict(dtype=3), 1), (dict(stride=3), 1), (dict(x=A + 2), 1), (dict(x=A + 1, dtype=1), 1),
    (dict(w=A + 8), 1), (dict(m=0), 1), (dict(act=5), 1), (dict(k=1 << 31), 6), (dict(m=100, ws=None), 5), (dict(m=100, ws=A + 16), 5), (dict(m=100, nbytes=100), 5)])
def test_linear_refuses(bad, status):
    assert linear(**bad) == status


def dense(x=A, dtype=0, stride=4, kernel=A, kdtype=0, kstride=4, m=4, n=4, k=4, bias=None, bdtype=0, act=0, out=A, xk=A, kk=A, ws=A, nbytes=1 << 30):
    return lib().amsim_i8_dense(x, dtype, stride, kernel, kdtype, kstride, m, n, k, bias, bdtype, act, out, xk, kk, ws, nbytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), 1), (dict(kernel=None), 1), (dict(out=None), 1), (dict(dtype=4), 1), (dict(kdtype=4), 1), (dict(stride=3), 1), (dict(kstride=3), 1), (dict(xk=A + 8), 1),
    (dict(kk=A + 8), 1), (dict(kernel=A + 2), 1), (dict(act=3), 1), (dict(m=0), 1), (dict(ws=None), 5), (dict(ws=A + 128), 5), (dict(nbytes=1000), 5),
    (dict(m=1 << 22), 6), (dict(n=1 << 22), 6)])
def test_dense_refuses(bad, status):
    assert dense(**bad) == status


def grad(g=A, dtype=0, stride=4, out=None, xk=A, kk=A, m=4, n=4, k=4, gx=A, gk=A, kdtype=0, gb=A, bdtype=0, ws=A, nbytes=1 << 30):
    return lib().amsim_i8_dense_grad(g, dtype, stride, out, xk, kk, m, n, k, gx, gk, kdtype, gb, bdtype, ws, nbytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(g=None), 1), (dict(xk=None), 1), (dict(kk=None), 1), (dict(dtype=3), 1), (dict(kdtype=3), 1), (dict(bdtype=3), 1), (dict(stride=3), 1), (dict(out=A + 2), 1),
    (dict(xk=A + 8), 1), (dict(kk=A + 8), 1), (dict(gx=A + 8), 1), (dict(gk=A + 8), 1), (dict(gb=A + 2), 1), (dict(m=0), 1), (dict(ws=None), 5), (dict(nbytes=1000), 5),
    (dict(m=1 << 22), 6), (dict(n=1 << 22), 6), (dict(k=1 << 31), 6)])
def test_dense_grad_refuses(bad, status):
    assert grad(**bad) == status


def test_nothing_asked_for_is_nothing_done():
    assert grad(gx=None, gk=None, gb=None) == 0


def test_plans():
    info = (C.c_int64 * 4)()
    f = lib().amsim_i8_plan
    f.argtypes = [C.c_int, C.c_void_p, C.c_void_p]
    assert f(0, (C.c_int64 * 3)(1, 1, 1), info) == 1 and f(1, None, info) == 1 and f(1, (C.c_int64 * 3)(1, 1, 1 << 22), info) == 6
    assert f(1, (C.c_int64 * 3)(64, 100, 16384), info) == 0 and list(info) == [0, 0, 0, 0]
    for m, n, k in ((1, 1, 1 << 21), (100, 100, 131073), (1 << 20, 3, 200000), (65, 1, 1)):
        assert f(1, (C.c_int64 * 3)(m, n, k), info) == 0 and info[2] * 131072 >= k


def test_host_tensors_and_others_are_refused():
    x, w = torch.ones(2, 4), functors.I8Tensor(torch.zeros(1028, dtype=torch.uint8), 1, 4)
    for call in (lambda: functors.int8_quantize(x), lambda: functors.int8_linear(x, w), lambda: functors.int8_dequantize(w), lambda: functors.int8_matmul(w, w),
                 lambda: math_ops.lineari8(x, torch.ones(4, 3)), lambda: layers.densei8(3, input_dim=4)(x), lambda: functors.int8_linear(x, x),
                 lambda: functors.int8_matmul(w, x), lambda: functors.int8_quantize(3), lambda: math_ops.lineari8(x, None)):
        with pytest.raises(TypeError):
            call()


def test_layer_arguments():
    with pytest.raises(ValueError):
        layers.densei8(0)
    with pytest.raises(ValueError):
        layers.densei8(4).pack()
    with pytest.raises(ValueError):
        layers.densei8(4, activation="nothing")
    with pytest.raises(TypeError):
        layers.densei8(4, mant_mul_lut="x")
