"""Tensors in 8-bit integers with a scale for each row: what a backward pass keeps of its input."""
import torch


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
