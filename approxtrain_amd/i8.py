"""Tensors in 8-bit integers with a scale for each row: the operands of the library's 8-bit products, and what a backward
pass keeps of its input."""
import torch


class I8Tensor:
    """``rows`` x ``length`` values as integers of at most 127 with one float32 scale for each row, its largest magnitude by
    127.  ``data`` holds codes and scales in the order the matrix cores take them (opaque bytes; ``dequantize``
    reads them back).  Made by ``functors.int8_quantize``."""

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
        return functors.int8_dequantize(self, dtype)

    def __repr__(self):
        return f"I8Tensor({self.rows} x {self.length}, device='{self.data.device}')"


class Kept8:
    """A tensor's values in 8 bits: of every row (its last axis) integers of at most 127 and one float32 scale, the row's
    largest magnitude by 127.  ``data`` are opaque bytes; ``values`` reads them back.  Made by ``functors.keep8``."""

    __slots__ = ("data", "shape", "dtype")

    def __init__(self, data, shape, dtype):
        self.data, self.shape, self.dtype = data, torch.Size(shape), dtype

    @property
    def device(self):
        return self.data.device

    def nbytes(self):
        return self.data.numel()

    def values(self, dtype=None):
        """The values that the bytes stand for, in ``dtype`` (None: the tensor's own)."""
        from . import functors
        return functors.kept8_values(self, dtype)

    def __repr__(self):
        return f"Kept8({tuple(self.shape)}, device='{self.data.device}')"
