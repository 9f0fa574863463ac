"""Matrices in blocks of small floating-point numbers: 4-bit operands of products and 8-bit records of activations.

A block is a run of neighbours along one axis of a matrix that share a scale:

    "mxfp4"   4-bit numbers (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6), blocks of 32, the scale a power of two
    "nvfp4"   4-bit numbers, blocks of 16, the scale an 8-bit number (E4M3) times one power of two per matrix
    "mxfp8"   8-bit numbers (E4M3, up to 448), blocks of 32, the scale a power of two

NervanaGPU.block_empty makes one, quantize fills it, dequantize reads it, block_dot multiplies, relu_mask masks
deltas by the sign of a recorded activation. The reference stores fp16 and nothing smaller
(nervanagpu/nervanagpu.py:469-520).
"""
import ctypes
import math

import numpy as np

from . import _lib

FORMATS = {"mxfp4": 0, "nvfp4": 1, "mxfp8": 2}      # the numbers of include/nervana_b200.h


class BlockTensor(object):
    """A (rows, cols) matrix in blocks along `axis` (1: along its rows, 0: down its columns).

    Products sum over the blocked axis, so the left operand of block_dot has axis 1 and the right one axis 0.
    `scale` (nvfp4 only) is the matrix's power of two, 2^-32 to 2^32: block scales hold max|block| / (6 * scale) in 8 bits,
    from 2^-9 to 448, so it should bring most blocks' max / 6 near 1. Numbers beyond 2688 * scale are limited to that,
    without a word; nothing here measures the matrix. `.T` is a view of the same memory with the other
    axis. codes and scales are uint8 tensors (the padding between rows stays zero) that a program may save and
    set again."""

    def __init__(self, backend, shape, format, axis=1, scale=1.0, name=None, codes=None, scales=None, desc=None):
        self.backend = backend
        self.name = name
        if desc is None:
            if format not in FORMATS:
                raise ValueError("block formats are %s, not %r" % (", ".join(sorted(FORMATS)), format))
            assert len(shape) == 2, "a matrix in blocks has two dimensions"
            assert axis in (0, 1), "blocks run along axis 0 or 1"
            shape = tuple(int(s) for s in shape)
            assert min(shape) > 0, "a matrix in blocks has at least one row and column"
            scale = float(scale)
            if format != "nvfp4":
                assert scale == 1.0, "only nvfp4 matrices have a scale"
            assert math.isfinite(scale) and scale > 0 and math.frexp(scale)[0] == 0.5, "the scale is a power of two"
            device = ctypes.c_int()
            _lib.check(backend.lib.ng_current_device(ctypes.byref(device)))
            desc = _lib.BlockDesc(FORMATS[format], axis, shape[0], shape[1], device.value, scale, None, None)
            sizes = ctypes.c_size_t(), ctypes.c_size_t()
            _lib.check(backend.lib.ng_block_bytes(ctypes.byref(desc), ctypes.byref(sizes[0]), ctypes.byref(sizes[1])))
            codes = backend.zeros((sizes[0].value,), dtype=np.uint8, name=name)
            scales = backend.zeros((sizes[1].value,), dtype=np.uint8, name=name)
            # (whatever stream fills it first: the zeros are there)
            _lib.check(backend.lib.ng_stream_sync(backend.stream))
            desc.codes, desc.scales = codes.ptr, scales.ptr
        self.shape, self.format, self.axis, self.scale = tuple(shape), format, axis, float(scale)
        self.codes, self.scales, self.desc = codes, scales, desc
        self._turned = None

    def __str__(self):
        return "BlockTensor(%s) name:%s shape:%s axis:%d scale:%g" % (self.format, self.name, self.shape, self.axis, self.scale)

    __repr__ = __str__

    @property
    def size(self):
        return self.shape[0] * self.shape[1]

    @property
    def nbytes(self):
        """Device memory that codes and scales take, padding included."""
        return self.codes.nbytes + self.scales.nbytes

    @property
    def T(self):
        if self._turned is None:       # (made once: it took 1 us of a weight gradient's 4.5 on the host)
            d = self.desc
            desc = _lib.BlockDesc(d.format, 1 - self.axis, self.shape[1], self.shape[0], d.device, d.scale, d.codes, d.scales)
            self._turned = BlockTensor(self.backend, self.shape[::-1], self.format, 1 - self.axis, self.scale, self.name,
                                       self.codes, self.scales, desc)
        return self._turned
