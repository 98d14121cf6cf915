"""Rows of f32 / f16 / bf16 values for the tests of the int8 lane and of scoring: bit patterns, strides, guard bytes."""
from __future__ import annotations

import numpy as np

from camelid_amd import binding as B
from camelid_amd.binding import DeviceBuffer

TYPES = {"f32": B.CML_F32, "f16": B.CML_F16, "bf16": B.CML_BF16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BITS = {"f32": np.uint32, "f16": np.uint16, "bf16": np.uint16}
GUARD = 0xA5


def to_bits(v: np.ndarray, t: str) -> np.ndarray:
    """f32 values rounded to the type, to nearest, ties to even."""
    v = np.ascontiguousarray(v, np.float32)
    if t == "f32":
        return v.view(np.uint32)
    if t == "f16":
        with np.errstate(over="ignore"):
            return v.astype(np.float16).view(np.uint16)
    u = v.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(v), np.uint16(0x7FC0), r)


def from_bits(b: np.ndarray, t: str) -> np.ndarray:
    """The values as f32."""
    if t == "f32":
        return b.view(np.float32)
    if t == "f16":
        return b.view(np.float16).astype(np.float32)
    return (b.astype(np.uint32) << 16).view(np.float32)


class Rows:
    """A [n, cols] operand on the device, `stride` elements from row to row, `offset` elements into its allocation, guard bytes everywhere else."""

    def __init__(self, bits: np.ndarray, stride: int | None = None, offset: int = 0):
        self.n, self.cols = bits.shape
        self.stride, self.offset, self.dtype = stride or self.cols, offset, bits.dtype
        flat = np.full((offset + self.n * self.stride + 8) * bits.itemsize, GUARD, np.uint8).view(bits.dtype)
        flat[offset:offset + self.n * self.stride].reshape(self.n, self.stride)[:, :self.cols] = bits
        self.flat = flat
        self.buf = DeviceBuffer.from_numpy(flat)
        self.ptr = self.buf.ptr + offset * bits.itemsize

    @classmethod
    def empty(cls, n: int, cols: int, dtype, stride: int | None = None, offset: int = 0) -> "Rows":
        return cls(np.full(n * cols * np.dtype(dtype).itemsize, GUARD, np.uint8).view(dtype).reshape(n, cols), stride, offset)

    def get(self) -> np.ndarray:
        """The rows, after a check that nothing around them was written."""
        flat = self.buf.to_numpy(self.dtype, self.flat.shape)
        body = flat[self.offset:self.offset + self.n * self.stride].reshape(self.n, self.stride)
        outside = np.concatenate([flat[:self.offset], flat[self.offset + self.n * self.stride:], body[:, self.cols:].reshape(-1)])
        assert np.all(np.ascontiguousarray(outside).view(np.uint8) == GUARD), "written outside the rows"
        return body[:, :self.cols].copy()
