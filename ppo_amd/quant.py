"""QuantizedRows - a store of observation rows (hidden states) in 8 or 4 bits: quantised as they are written, read back by a
minibatch's indices.  A quarter (int4: an eighth) of the memory and of the gather's traffic of fp32 rows; formats and rounding
are defined in include/ppo_xp.h (ppo_xp_quantize_rows, ppo_xp_dequantize_rows).
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import EINVAL, PpoXpPanic

_call = _lib.bound                                # csrc/torchcall.cpp
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_GROUPS = (16, 32, 64, 128, 256, 512)

#: format -> (PPO_XP_Q_*, type of the codes)
FORMATS = {"int8": (1, torch.int8), "e4m3": (2, torch.float8_e4m3fn), "int4": (3, torch.uint8)}


def _panic(msg):
    raise PpoXpPanic(EINVAL, msg)


def _check(row_size, format, group, dtype=torch.float32):
    """What a store is made of, and the type its rows are read as."""
    if format not in FORMATS:
        _panic(f"QuantizedRows: format {format!r} is none of {sorted(FORMATS)}")
    if not 1 <= row_size <= 1 << 24:
        _panic(f"QuantizedRows: rows of {row_size} elements (1 .. 2^24 expected)")
    if group not in _GROUPS:
        _panic(f"QuantizedRows: group {group} is none of {list(_GROUPS)}")
    if dtype not in _DTYPES:
        _panic(f"QuantizedRows: rows are read as f32, bf16 or f16, not {dtype}")


class QuantizedRows:
    """`num_rows` rows of `row_size` elements; one f32 scale per `group` of them (16, 32, 64, 128, 256 or 512).

    codes  [num_rows, row_size] int8 / float8_e4m3fn, or [num_rows, ceil(row_size / 2)] uint8 with two 4-bit codes a byte
    scales [num_rows, ceil(row_size / group)] f32
    Like the buffer's streams the rows start out as zeros.  Calls run on torch's current stream and do not synchronise."""

    def __init__(self, num_rows: int, row_size: int, format: str = "int8", group: int = 64, device: int = 0):
        _check(row_size, format, group)
        if num_rows < 0:
            _panic(f"QuantizedRows: {num_rows} rows")
        dev = torch.device("cuda", int(device))
        nbytes = (row_size + 1) // 2 if format == "int4" else row_size
        codes = torch.zeros(num_rows, nbytes, dtype=torch.uint8, device=dev).view(FORMATS[format][1])
        self._init(codes, torch.zeros(num_rows, -(-row_size // group), device=dev), row_size, format, group)

    @classmethod
    def of(cls, codes, scales, row_size: int, format: str, group: int):
        """A store over tensors the caller owns (see the class for their shapes and types); rows may lie apart."""
        self = cls.__new__(cls)
        self._init(codes, scales, row_size, format, group)
        return self

    def _init(self, codes, scales, row_size, format, group):
        _check(row_size, format, group)
        kind, dtype = FORMATS[format]
        nbytes = (row_size + 1) // 2 if format == "int4" else row_size
        if not codes.is_cuda or codes.dtype is not dtype or codes.dim() != 2 or codes.shape[1] != nbytes or scales.dtype is not torch.float32 \
                or scales.device != codes.device or scales.shape != (codes.shape[0], -(-row_size // group)):
            _panic(f"QuantizedRows: codes [n, {nbytes}] {dtype} and scales [n, {-(-row_size // group)}] f32 on one GPU expected")
        for t in (codes, scales):
            if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
                _panic("QuantizedRows: rows of codes and scales must be contiguous and must not overlap")
        self.codes, self.scales, self.row_size, self.format, self.group = codes, scales, int(row_size), format, int(group)
        self._kind = kind

    def __len__(self):
        return self.codes.shape[0]

    def write(self, rows, at: int = 0):
        """Quantises `rows` [n, row_size] (f32, bf16, f16) into rows at .. at + n of the store."""
        _call.write(self.codes, self.scales, self.row_size, self._kind, self.group, rows, at)

    def read(self, index=None, dtype=torch.float32, out=None):
        """Rows index[j] (contiguous int32 / int64 CUDA tensor), a slice of rows, or all rows, as `dtype`."""
        if dtype not in _DTYPES:
            _panic("read: f32, bf16 or f16 expected")
        at = n = 0
        if index is None or isinstance(index, slice):
            at, end, step = (index or slice(None)).indices(len(self))
            if step != 1:
                _panic("read: a slice of consecutive rows expected")
            index, n = None, max(0, end - at)
        return _call.read(self.codes, self.scales, self.row_size, self._kind, self.group, index, at, n, _DTYPES[dtype], out)
