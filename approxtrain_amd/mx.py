"""Tensors in microscaled 4-bit floating point (MXFP4), as the operands of the library's 4-bit products."""
import torch

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class MXTensor:
    """``rows`` x ``length`` values, every 32 of them along the length in e2m1 with one power-of-two scale.
    ``data`` holds codes and scales in the order the matrix cores take them (opaque bytes; ``dequantize``
    reads them back).  Made by ``functors.mxfp4_quantize``."""

    __slots__ = ("data", "rows", "length")

    def __init__(self, data, rows, length):
        self.data, self.rows, self.length = data, rows, length

    @property
    def shape(self):
        return torch.Size((self.rows, self.length))

    @property
    def device(self):
        return self.data.device

    def nbytes(self):
        return self.data.numel()

    def dequantize(self, dtype=torch.float32):
        from . import functors
        return functors.mxfp4_dequantize(self, dtype)

    def __repr__(self):
        return f"MXTensor({self.rows} x {self.length}, device='{self.data.device}')"
