"""Shared by the tests of the transformer-layer entry points: device tensors with
guard bytes on both sides, and the element types."""
import numpy as np
import torch

TYPES = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "f16": (2, torch.float16)}
GUARD = 512          # bytes before and after a guarded buffer
FILL = 0xA5


class Buf:
    """A device buffer between guards.  `shift`: elements by which its start is off
    the 256-byte boundary."""

    def __init__(self, shape, dtype, data=None, shift=0):
        n = int(np.prod(shape))
        size = torch.empty((), dtype=dtype).element_size()
        self.raw = torch.full((2 * GUARD + (n + shift) * size + 256,), FILL, dtype=torch.uint8,
                              device="cuda")
        self.lo, self.hi = GUARD + shift * size, GUARD + (shift + n) * size
        self.t = self.raw[self.lo:self.hi].view(dtype).view(shape)
        if data is not None:
            self.t.copy_(torch.as_tensor(data).to(dtype))

    @property
    def ptr(self):
        return self.raw.data_ptr() + self.lo

    def intact(self):
        return bool((self.raw[:self.lo] == FILL).all()) and bool((self.raw[self.hi:] == FILL).all())


def values(t):
    """float64 numpy values of a device tensor."""
    return t.double().cpu().numpy()


def half_step(t):
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[t]


def smallest(t):
    """Half the type's smallest step (its subnormals')."""
    return {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}[t]
