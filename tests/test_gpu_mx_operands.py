"""Operands are their values alone: every byte is written, whatever the memory held before."""
import pytest
import torch

from approxtrain_amd import functors, load_library
from approxtrain_amd.layers import packed_densemx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 16), (17, 33), (33, 200), (48, 49), (64, 64), (100, 10), (130, 257), (300, 785)])
def test_bytes_do_not_depend_on_what_the_memory_held(rows, cols):
    lib = load_library()
    x = torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows))
    sizes = [lib.amsim_mxfp4_operand_workspace_bytes(rows, cols), lib.amsim_mxfp4_operand_workspace_bytes(cols, rows)]
    for by_rows, by_columns in ((True, False), (False, True), (True, True)):
        got = []
        for fill in (0, 255):
            buffers = [torch.full((n,), fill, dtype=torch.uint8, device="cuda") for n in sizes]
            functors.check(lib.amsim_mxfp4_quantize(x.data_ptr(), 0, rows, cols, cols, buffers[0].data_ptr() if by_rows else None,
                                                    buffers[1].data_ptr() if by_columns else None, torch.cuda.current_stream().cuda_stream))
            got.append([b for b, wanted in zip(buffers, (by_rows, by_columns)) if wanted])
        for a, b in zip(*got):
            assert torch.equal(a, b)
    r, c = functors.mxfp4_quantize_both(x)
    assert torch.equal(r.data, functors.mxfp4_quantize(x).data) and torch.equal(c.data, functors.mxfp4_quantize(x, axis=0).data)


def test_a_layer_packed_twice_is_saved_as_the_same_bytes():
    kernel = torch.randn(70, 33, device="cuda")
    saved = []
    for fill in (0, 255):
        junk = [torch.full((4096,), fill, dtype=torch.uint8, device="cuda") for _ in range(64)]
        del junk
        saved.append(packed_densemx(kernel).state_dict()["weights"])
    assert torch.equal(*saved)
