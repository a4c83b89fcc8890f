"""Every byte that the 8-bit conversions, the products and the row kernels write, and none beside them: buffers of the caller's
with two fillings and guards around them, through the C ABI, against operands that are laid out on the host."""
import pytest
import torch

from approxtrain_amd import load_library
from approxtrain_amd._lib import check
from tests import rows_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}
GUARD = 4096


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(DTYPES[dtype])


class Buffer:
    """``n`` bytes on a 256-byte boundary, filled, with as much around them as no kernel may touch."""

    def __init__(self, n, fill):
        self.n, self.fill = n, fill
        self.all = torch.full((n + 2 * GUARD,), fill, dtype=torch.uint8, device="cuda")

    def ptr(self):
        return self.all.data_ptr() + GUARD

    def bytes(self):
        a = self.all.cpu()
        assert (a[:GUARD] == self.fill).all() and (a[GUARD + self.n:] == self.fill).all(), "written outside"
        return a[GUARD:GUARD + self.n]


def as_bytes(t):
    return t.contiguous().view(torch.uint8).reshape(-1)


def laid_out(q, scales):
    """Codes [rows, length] as the products take them (16 rows x 64 values in a piece, 16 values of a row together), zeros
    behind the ends, and the scales behind."""
    rows, length = q.shape
    r, s = -(-rows // 16), -(-length // 64)
    whole = torch.zeros(r * 16, s * 64, dtype=torch.int8)
    whole[:rows, :length] = q.to(torch.int8)
    pieces = whole.view(r, 16, s, 4, 16).permute(0, 2, 3, 1, 4)
    return torch.cat([as_bytes(pieces), as_bytes(scales.reshape(-1).float())])


# one launch and two, rows by themselves and by sixteen in every number of units, remainders of 16 rows and of 64 columns
SHAPES = [(1, 1), (15, 64), (16, 63), (17, 70), (33, 130), (70, 17), (129, 257), (256, 65), (300, 1000), (513, 65), (600, 436), (700, 400), (1025, 70), (1030, 600),
          (1041, 1100), (1030, 2100), (1030, 4200), (20, 1100), (20, 4200), (20, 8300), (2003, 33), (5000, 10)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_operands(rows, cols, dtype):
    lib = load_library()
    x = make((rows, cols), dtype, rows + cols)
    device = x.cuda()
    want = {True: laid_out(*ref.int8(x)), False: laid_out(*ref.int8(x.t()))}
    for fill in (0xa5, 0x5a):
        for directions in ((True, False), (False, True), (True, True)):
            out = [Buffer(lib.amsim_i8_operand_workspace_bytes(*e), fill) if wanted else None for wanted, e in zip(directions, ((rows, cols), (cols, rows)))]
            ws = Buffer(lib.amsim_i8_quantize_workspace_bytes(rows, cols), fill)
            check(lib.amsim_i8_quantize(device.data_ptr(), CODES[dtype], rows, cols, cols, *[b and b.ptr() for b in out], ws.ptr(), ws.n, None))
            torch.cuda.synchronize()
            ws.bytes()
            for b, w in zip(out, (want[True], want[False])):
                if b is not None:
                    assert torch.equal(b.bytes(), w)


STEPS = [(1, 1, 1), (1, 30, 70), (17, 33, 65), (64, 100, 100), (65, 16, 130), (128, 300, 784), (250, 10, 2100), (513, 70, 129), (700, 45, 400), (1030, 130, 600), (1041, 70, 1100),
         (1030, 20, 4200), (40, 50, 8300), (2003, 1003, 33)]


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype,kernel_dtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("m,n,k", STEPS)
def test_a_training_step(m, n, k, dtype, kernel_dtype, relu):
    """What is kept, byte by byte; results that do not depend on what lay in the workspaces and the results' places."""
    lib = load_library()
    x, kernel, bias, dy = make((m, k), dtype, 1), make((k, n), kernel_dtype, 2, 0.1), make((n,), "f32", 3), make((m, n), dtype, 4, 0.01)
    (qx, sx), (qw, sw) = ref.int8(x), ref.int8(kernel, 0)
    kept = laid_out(qx.t(), sx), laid_out(qw, sw)
    device = [t.cuda() for t in (x, kernel, bias, dy)]
    size, kernel_size = x.element_size(), kernel.element_size()
    seen = None
    for fill in (0xa5, 0x5a, 0xff):
        out, xk, kk = Buffer(m * n * size, fill), Buffer(lib.amsim_i8_kept_workspace_bytes(k, m), fill), Buffer(lib.amsim_i8_kept_workspace_bytes(k, n), fill)
        ws = Buffer(lib.amsim_i8_dense_workspace_bytes(m, n, k), fill)
        check(lib.amsim_i8_dense(device[0].data_ptr(), CODES[dtype], k, device[1].data_ptr(), CODES[kernel_dtype], n, m, n, k, device[2].data_ptr(), 0, int(relu),
                                 out.ptr(), xk.ptr(), kk.ptr(), ws.ptr(), ws.n, None))
        torch.cuda.synchronize()
        ws.bytes()
        assert torch.equal(xk.bytes(), kept[0]) and torch.equal(kk.bytes(), kept[1])
        results = [out.bytes()]
        for which in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
            gx, gk, gb = Buffer(m * k * size, fill), Buffer(k * n * kernel_size, fill), Buffer(4 * n, fill)
            ws = Buffer(lib.amsim_i8_dense_grad_workspace_bytes(m, n, k), fill)
            check(lib.amsim_i8_dense_grad(device[3].data_ptr(), CODES[dtype], n, out.ptr() if relu else None, xk.ptr(), kk.ptr(), m, n, k, gx.ptr() if which[0] else None,
                                          gk.ptr() if which[1] else None, CODES[kernel_dtype], gb.ptr() if which[2] else None, 0, ws.ptr(), ws.n, None))
            torch.cuda.synchronize()
            ws.bytes()
            for b, wanted in zip((gx, gk, gb), which):
                if wanted:
                    results.append(b.bytes())
                else:
                    assert (b.bytes() == fill).all()
        if seen is not None:
            assert all(torch.equal(a, b) for a, b in zip(seen, results))
        seen = results


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 17), (5, 128), (7, 130), (9, 700), (4, 1027), (3, 2050), (3, 5000), (2, 9001), (2, 16390), (70, 33)])
def test_rows_and_what_is_kept_of_them(rows, cols, dtype):
    lib = load_library()
    x = make((rows, cols), dtype, 5)
    q, s = ref.int8(x)
    pitch = -(-cols // 16) * 16
    codes = torch.zeros(rows, pitch, dtype=torch.int8)
    codes[:, :cols] = q.to(torch.int8)
    kept = torch.cat([as_bytes(codes), as_bytes(s.reshape(-1).float())])
    device, dy = x.cuda(), make((rows, cols), dtype, 6).cuda()
    seen = None
    for fill in (0xa5, 0x5a):
        results = []
        for kind in (2, 3):
            out, k8 = Buffer(rows * cols * x.element_size(), fill), Buffer(lib.amsim_kept8_workspace_bytes(rows, cols), fill)
            check(lib.amsim_activation(device.data_ptr(), CODES[dtype], rows, cols, cols, kind, out.ptr(), k8.ptr(), None))
            torch.cuda.synchronize()
            assert torch.equal(k8.bytes(), kept)
            grad = Buffer(out.n, fill)
            check(lib.amsim_activation_grad(dy.data_ptr(), CODES[dtype], rows, cols, cols, k8.ptr(), kind, grad.ptr(), None))
            torch.cuda.synchronize()
            results += [out.bytes(), grad.bytes()]
        out, stats, k8 = Buffer(rows * cols * x.element_size(), fill), Buffer(8 * rows, fill), Buffer(lib.amsim_kept8_workspace_bytes(rows, cols), fill)
        check(lib.amsim_layer_norm(device.data_ptr(), CODES[dtype], rows, cols, cols, None, None, 0, 1e-3, out.ptr(), stats.ptr(), k8.ptr(), None))
        torch.cuda.synchronize()
        assert torch.equal(k8.bytes(), kept)
        results += [out.bytes(), stats.bytes()]
        for x_ptr, kept_ptr in ((device.data_ptr(), None), (None, k8.ptr())):
            gx, gg, gb, ws = Buffer(out.n, fill), Buffer(4 * cols, fill), Buffer(4 * cols, fill), Buffer(lib.amsim_layer_norm_grad_workspace_bytes(rows, cols), fill)
            check(lib.amsim_layer_norm_grad(dy.data_ptr(), CODES[dtype], rows, cols, cols, x_ptr, cols, kept_ptr, stats.ptr(), None, 0, gx.ptr(), gg.ptr(), gb.ptr(),
                                            ws.ptr(), ws.n, None))
            torch.cuda.synchronize()
            ws.bytes()
            results += [b.bytes() for b in (gx, gg, gb)]
        if seen is not None:
            assert all(torch.equal(a, b) for a, b in zip(seen, results))
        seen = results
