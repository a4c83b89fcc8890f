"""Every kind of tile, of split and of pair that the planner picks for the two products of an 8-bit backward pass, at extents that
fill none of them.  The plans are asserted, on the host too, so that a refit of the planner cannot take a kernel out of
these tests unseen.

The sums are exact and compared with those of whole numbers in 64 bits; a result has the sum's rounding to 32 bits and one for
each scale, one of 16 bits half a step more."""
import ctypes as C

import pytest
import torch

from approxtrain_amd import load_library, math_ops
from tests import rows_reference as ref

# (rows and columns of the tile, splits of x's gradient and of the kernel's; 0: one workgroup's waves share it), rows, units, width
PAIRS = [((64, 64, 1, 1), 67, 33, 66), ((64, 64, 1, 0), 65, 34, 33), ((64, 64, 0, 1), 33, 34, 67), ((64, 64, 1, 12), 2226, 32, 70), ((64, 64, 13, 1), 65, 2446, 68),
         ((64, 64, 13, 0), 66, 2307, 36), ((64, 64, 4, 2), 6211, 8327, 37), ((128, 128, 1, 1), 74, 67, 16597), ((128, 128, 0, 1), 35, 706, 8017),
         ((128, 128, 1, 16), 12746, 229, 201), ((128, 128, 8, 1), 193, 6513, 458), ((128, 128, 2, 4), 12459, 5332, 67), ((256, 128, 1, 1), 153, 193, 16153),
         ((256, 128, 0, 1), 39, 4700, 1431), ((256, 128, 1, 16), 10973, 68, 1167), ((256, 128, 8, 1), 193, 9734, 1505), ((256, 128, 2, 4), 20685, 13827, 133),
         ((256, 256, 1, 1), 801, 705, 6795), ((256, 256, 1, 4), 8631, 1832, 733), ((256, 256, 4, 1), 2027, 8201, 759), ((256, 256, 4, 2), 15241, 20114, 131)]


@pytest.mark.parametrize("want,m,n,k", PAIRS)
def test_plans_of_pairs(want, m, n, k):
    lib = load_library()
    lib.amsim_i8_plan.argtypes = [C.c_int, C.c_void_p, C.c_void_p]
    e, info = (C.c_int64 * 6)(m, k, n, k, n, m), (C.c_int64 * 4)()
    assert lib.amsim_i8_plan(2, C.addressof(e), C.addressof(info)) == 0
    assert tuple(info) == want


def close(got, product, name):
    half = ref.half_step(got.dtype) if got.dtype != torch.float32 else 0
    tol = ((3 * ref.U + half) * 1.01) * product.abs() + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - product).abs()
    assert (off <= tol).all(), f"{name}: worst {float((off / tol).max()):.3g} of the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kernel_dtype,relu", [("bfloat16", "float32", False), ("float32", "bfloat16", True)])
@pytest.mark.parametrize("want,m,n,k", PAIRS)
def test_gradients(want, m, n, k, dtype, kernel_dtype, relu):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = torch.randn((m, k), device="cuda", generator=g).to(getattr(torch, dtype)).requires_grad_()
    kernel = (torch.randn((k, n), device="cuda", generator=g) * k ** -0.5).to(getattr(torch, kernel_dtype)).requires_grad_()
    dy = (torch.randn((m, n), device="cuda", generator=g) * 0.01).to(x.dtype)
    out = math_ops.lineari8(x, kernel, activation="relu" if relu else None)
    dx, dw = torch.autograd.grad(out, [x, kernel], dy)
    (qx, sx), (qw, sw) = ref.int8(x.detach()), ref.int8(kernel.detach(), 0)
    given = dy.float()
    if relu:
        given = torch.where(out > 0, given, 0.0)
    qv, sv = ref.int8(given * sw.float())
    close(dx, torch.matmul(qv, qw.t().contiguous()) * sv, "dx")
    del qv
    qu, su = ref.int8(given * sx.float(), 0)
    close(dw, torch.matmul(qx.t().contiguous(), qu) * su, "dw")
