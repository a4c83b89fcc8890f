"""Training steps of more rows, or more units, than a sum of 8-bit products has terms: the gradient whose reduction fits is given
all the same, and the other is refused before anything is multiplied."""
import pytest
import torch

from approxtrain_amd import load_library, math_ops
from tests import rows_reference as ref

A = 1 << 20  # an address that is never read
MOST = 1 << 21


def grad(m, n, k, gx=A, gk=A, gb=A):
    return load_library().amsim_i8_dense_grad(A, 0, n, None, A, A, m, n, k, gx, gk, 0, gb, 0, A, 0, None)


def test_what_is_refused():
    need = load_library().amsim_i8_dense_grad_workspace_bytes
    assert need(MOST + 1, 4, 4) > 0 and need(4, MOST + 1, 4) > 0 and need(4, 4, MOST + 1) == 0
    # (6: out of range; 5: the workspace, which is none here)
    assert grad(MOST + 1, 4, 4) == 6 and grad(MOST + 1, 4, 4, gk=None) == 5 and grad(MOST + 1, 4, 4, gx=None, gk=None) == 5
    assert grad(4, MOST + 1, 4) == 6 and grad(4, MOST + 1, 4, gx=None) == 5 and grad(MOST, MOST, 4) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("relu", [False, True])
def test_more_rows_than_a_sum_has(relu):
    m, n, k = MOST + 5, 3, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((m, k), device="cuda", generator=g).requires_grad_()
    kernel, bias = torch.randn((k, n), device="cuda", generator=g), torch.randn(n, device="cuda", generator=g).requires_grad_()
    dy = torch.randn((m, n), device="cuda", generator=g)
    out = math_ops.lineari8(x, kernel, bias, "relu" if relu else None)
    dx, db = torch.autograd.grad(out, [x, bias], dy)
    given = torch.where(out > 0, dy, 0.0) if relu else dy
    qw, sw = ref.int8(kernel, 0)
    qv, sv = ref.int8(given * sw.float())
    want = torch.matmul(qv, qw.t().contiguous()) * sv
    assert ((dx.double() - want).abs() <= 3.03 * ref.U * want.abs() + 2.0 ** -149).all()
    exact, tol = given.double().sum(0), (m / 64 + 100) * ref.U * given.double().abs().sum(0)
    assert ((db.double() - exact).abs() <= tol).all()
    with pytest.raises(ValueError, match="out of the 8-bit products' range"):
        math_ops.lineari8(x, kernel.requires_grad_())


@pytest.mark.gpu
def test_more_units_than_a_sum_has():
    m, n, k = 3, MOST + 5, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    x, kernel = torch.randn((m, k), device="cuda", generator=g), torch.randn((k, n), device="cuda", generator=g).requires_grad_()
    dy = torch.randn((m, n), device="cuda", generator=g)
    dw, = torch.autograd.grad(math_ops.lineari8(x, kernel), [kernel], dy)
    qx, sx = ref.int8(x)
    qu, su = ref.int8(dy * sx.float(), 0)
    want = torch.matmul(qx.t().contiguous(), qu) * su
    assert ((dw.double() - want).abs() <= 3.03 * ref.U * want.abs() + 2.0 ** -149).all()
    with pytest.raises(ValueError, match="out of the 8-bit products' range"):
        math_ops.lineari8(x.requires_grad_(), kernel)
