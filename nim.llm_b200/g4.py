"""4-bit weights with group scales: the arrays nls_g4_matmul takes, and the
settings records of nls_draw_batch.

`G4Weights` holds a rows x cols matrix as torch tensors in the library's
layout: q uint8 [rows, cols / 2] (column 2j in the low nibble of byte j,
column 2j + 1 in the high one), scales and optional mins [ceil(cols / group),
rows]; w = s * (q - 8), or s * q + m with mins. `g4_pack` brings values that a
quantiser already has into that layout; `g4_quantize` rounds a weight matrix
to it.
"""
from __future__ import annotations

from typing import Optional

import numpy as np

from ._abi import DRAW_PARAMS_DTYPE, G4WeightsStruct, NLS_DT


_DT_CODES: dict = {}   # torch dtype -> NLS_DT_*


def dt_code(dtype) -> int:
    """NLS_DT_* of a torch dtype."""
    code = _DT_CODES.get(dtype)
    if code is None:
        name = {"torch.float32": "f32", "torch.float16": "f16", "torch.bfloat16": "bf16"}.get(str(dtype))
        if name is None:
            raise TypeError(f"float32, float16 or bfloat16 expected, not {dtype}")
        code = _DT_CODES[dtype] = NLS_DT[name]
    return code


def _line(rows: int) -> int:
    """Values from one group's scales to the next: rows, to whole 8."""
    return -(-rows // 8) * 8


class G4Weights:
    """A rows x cols matrix of 4-bit values with group scales (nls_g4_weights).

    q: uint8 [rows, cols / 2], rows 16-byte aligned; scales, mins: one type,
    [ceil(cols / group), rows], lines a multiple of 8 values apart (a [:, :rows]
    view of a wider tensor). All on one CUDA device; the tensors are kept."""

    def __init__(self, q, scales, mins=None, group: int = 128):
        import torch
        if q.dtype != torch.uint8 or q.dim() != 2 or q.stride(1) != 1:
            raise ValueError("q must be a uint8 matrix with contiguous rows")
        rows, cols = q.shape
        cols *= 2
        group = int(group)
        if group not in (32, 64) and (group < 128 or group % 128):
            raise ValueError("group must be 32, 64 or a multiple of 128")
        if rows < 1 or cols < 32 or cols % 32:
            raise ValueError("at least one row, and columns in whole 32, are needed")
        if rows > 1 << 30 or cols > 1 << 24:
            raise ValueError("at most 2^30 rows and 2^24 columns")
        lines = -(-cols // group)
        s_ld = scales.stride(0) if lines > 1 else _line(rows)
        q_ld = q.stride(0) if rows > 1 else -(-cols // 32) * 16
        if q_ld % 16 or s_ld % 8 or s_ld < rows:
            raise ValueError("q's rows must be 16-byte multiples apart and the scales' lines multiples of 8 values")
        dtype, device = scales.dtype, q.device
        for name, t in (("scales", scales), ("mins", mins)):
            if t is None:
                continue
            if tuple(t.shape) != (lines, rows) or t.stride(1) != 1 or (lines > 1 and t.stride(0) != s_ld):
                raise ValueError(f"{name} must be [ceil(cols / group), rows] with contiguous lines, scales and mins "
                                 "with the same line stride")
            if t.device != device or t.dtype != dtype:
                raise ValueError(f"{name} must be on q's device and of the scales' type")
            # the library reads a line in whole 16-byte pieces: the last one too
            # needs the room behind its last value
            if rows % 8 and t.untyped_storage().nbytes() < \
                    (t.storage_offset() + (lines - 1) * s_ld + _line(rows)) * t.element_size():
                raise ValueError("the last line of scales needs room for rows rounded up to 8 values (g4_pack makes it)")
        qp, sp = q.data_ptr(), scales.data_ptr()
        mp = None if mins is None else mins.data_ptr()
        if (qp | sp | (mp or 0)) % 16:
            raise ValueError("q, scales and mins must be 16-byte aligned")
        self.q, self.scales, self.mins = q, scales, mins
        self.rows, self.cols, self.group = rows, cols, group
        self.device = device
        self.struct = G4WeightsStruct(qp, sp, mp, q_ld, s_ld, rows, cols, group, dt_code(dtype))

    def __repr__(self) -> str:
        return (f"G4Weights({self.rows} x {self.cols}, group={self.group}, {self.scales.dtype}"
                f"{', mins' if self.mins is not None else ''})")

    def dequantize(self):
        """The matrix as float32 [rows, cols]."""
        import torch
        q = torch.stack((self.q & 15, self.q >> 4), 2).reshape(self.rows, self.cols).float()
        wide = lambda t: t.t().float().repeat_interleave(self.group, 1)[:, :self.cols]  # noqa: E731
        if self.mins is None:
            return (q - 8.0) * wide(self.scales)
        return q * wide(self.scales) + wide(self.mins)


def g4_pack(values, scales, mins=None, group: int = 128) -> G4Weights:
    """G4Weights of quantised values: `values` integers 0..15 [rows, cols],
    `scales` and `mins` [rows, ceil(cols / group)] (one line per row, as
    quantisers keep them)."""
    import torch
    rows, cols = values.shape
    if cols % 32:
        raise ValueError("columns in whole 32 are needed")
    if int(values.min()) < 0 or int(values.max()) > 15:
        raise ValueError("4-bit values are 0..15")
    v = values.to(torch.uint8)
    q = torch.zeros((rows, -(-(cols // 2) // 16) * 16), dtype=torch.uint8, device=v.device)[:, :cols // 2]
    q.copy_(v[:, 0::2] | (v[:, 1::2] << 4))

    def lines(t):
        wide = torch.zeros((t.shape[1], _line(rows)), dtype=t.dtype, device=t.device)
        wide[:, :rows] = t.t()
        return wide[:, :rows]

    return G4Weights(q, lines(scales), None if mins is None else lines(mins), group=group)


def g4_quantize(weight, group: int = 128, symmetric: bool = True, dtype=None) -> G4Weights:
    """Round a weight matrix [rows, cols] (float tensor) to 4 bits: symmetric,
    s = the value of largest magnitude in the group / -8 and q = round(w / s)
    + 8 in 0..15 (so that value is held exactly at q = 0); otherwise
    s = (max - min) / 15, m = min. `dtype`: the type of scales and mins
    (default: the weight's)."""
    import torch
    rows, cols = weight.shape
    dtype = weight.dtype if dtype is None else dtype
    groups = -(-cols // group)
    w = torch.nn.functional.pad(weight.float(), (0, groups * group - cols))
    w = w.reshape(rows, groups, group)
    real = (torch.arange(groups * group, device=w.device) < cols).reshape(1, groups, group)
    if symmetric:
        top = w.gather(2, w.abs().argmax(2, keepdim=True))
        s = (top / -8.0).to(dtype)
        m = None
        q = torch.round(w / torch.where(s == 0, 1.0, s.float())) + 8.0
    else:
        lo = torch.where(real, w, float("inf")).amin(2, keepdim=True)
        hi = torch.where(real, w, float("-inf")).amax(2, keepdim=True)
        s, m = ((hi - lo) / 15.0).to(dtype), lo.to(dtype)
        q = torch.round((w - m.float()) / torch.where(s == 0, 1.0, s.float()))
    q = q.clamp(0, 15).reshape(rows, groups * group)[:, :cols]
    return g4_pack(q.to(torch.uint8), s[:, :, 0], None if m is None else m[:, :, 0], group=group)


def draw_params(rows: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> np.ndarray:
    """The nls_draw_params records of `rows` rows; each setting is one value or
    one per row. top_k 0, top_p 1 and min_p 0 are off; temperature 0 is greedy."""
    rec = np.zeros(rows, DRAW_PARAMS_DTYPE)
    rec["temperature"], rec["top_k"], rec["top_p"], rec["min_p"] = temperature, top_k, top_p, min_p
    return rec


def rows_of(t, device_index: Optional[int], what: str):
    """(pointer, values from row to row) of a 2-d tensor with contiguous rows
    on the engine's device (None: host memory)."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1) or (shape[0] > 1 and stride[0] < shape[1]):
        raise ValueError(f"{what}: a matrix with contiguous rows expected")
    if t.device.index != device_index:
        raise ValueError(f"{what} is on {t.device}, " + ("other arguments on the host" if device_index is None else
                                                          f"the engine on cuda:{device_index}"))
    return t.data_ptr(), (stride[0] if shape[0] > 1 else max(1, shape[1]))
