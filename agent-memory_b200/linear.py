"""Linear layers over 4-bit weights: the matrices around the Q4 attention.

``Q4Weight`` holds a matrix (or one per expert) in the cache's 4-bit format, the output of
``mx.quantize`` (group 64, 8 codes per 32-bit word, one scale and bias per group).  It keeps
the codes as they are and lays the scales and biases out once.  ``quantized_matmul`` is
``mx.quantized_matmul(x, w, scales, biases, transpose=True)``; ``quantized_swiglu`` is the
gated half of an MLP, ``silu(x G^T) * (x U^T)``, in one pass over both matrices.

Sums are fp32 and the result is rounded once to the activations' type.  A few tokens multiply
exact weights: scales and biases are held in fp16 under powers of two per weight row, which keeps
a scale from 2**-28 and a bias from 2**-24 of the row's largest scale on (or of 1/16 of its largest
bias, if that is larger).  For more tokens a weight is ``scale * code + bias`` rounded to fp16 (11
bits, or 2**-14 of that largest scale if that is more); in a gated float16 layer, where two such
errors would be 1.6 times the output's own rounding, it is the sum of two fp16 parts.  An
activation enters as fp16 under a power of two per token: only values below 2**-24 of their
token's largest lose bits (and keep 2**-35 of that).  A token with infinite or NaN activations gets
the infinities and NaN of the formula.  The weights are frozen: there is no backward pass.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import Q4WeightDesc, check
from .kernels import GROUP_SIZE, _check_params, _half_code, as_codes, _require_cuda

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
# With at most so many tokens and inputs one matrix, or a gated pair, needs no workspace.
FEW_TOKENS, FEW_GATED_TOKENS, FEW_INPUTS = 8, 4, 49152


class Q4Weight:
    """A 4-bit matrix [n_out, n_in] (codes [n_out, n_in/8]) or one per expert (codes
    [experts, n_out, n_in/8]), ready for the kernels.  ``scales`` and ``biases`` are
    [..., n_in/64] float16 or bfloat16, the type of the activations it multiplies.

    The codes are used in place (no copy when contiguous and 16-byte aligned); the scales and
    biases are packed into a buffer of the same size on the current stream."""

    __slots__ = ("codes", "params", "row_scale", "dtype", "device", "index", "n_out", "n_in",
                 "experts", "grouped", "desc", "ref")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                 group_size: int = 64, bits: int = 4):
        _check_params(group_size, bits)
        self.device = _require_cuda(codes, scales, biases)
        self.index = self.device.index
        codes = as_codes(codes).contiguous()
        if codes.dim() not in (2, 3):
            raise ValueError(f"codes must be [n_out, n_in/8] or [experts, n_out, n_in/8], got "
                             f"{tuple(codes.shape)}")
        if scales.dtype != biases.dtype:
            raise TypeError("scales and biases must share one dtype")
        self.dtype = scales.dtype
        self.n_out, self.n_in = codes.shape[-2], codes.shape[-1] * 8
        self.grouped = codes.dim() == 3
        self.experts = codes.shape[0] if self.grouped else 1
        if self.n_in == 0 or self.n_in % GROUP_SIZE or self.n_out == 0 or self.experts == 0:
            raise ValueError(f"a weight of {self.experts} x {self.n_out} x {self.n_in} needs n_in a "
                             f"positive multiple of {GROUP_SIZE} and no empty dimension")
        want = (*codes.shape[:-1], self.n_in // GROUP_SIZE)
        if tuple(scales.shape) != want or tuple(biases.shape) != want:
            raise ValueError(f"scales and biases must be {want}, got {tuple(scales.shape)} and "
                             f"{tuple(biases.shape)}")
        if codes.data_ptr() % 16:
            codes = codes.clone()
        self.codes = codes
        rows, groups = self.experts * self.n_out, self.n_in // GROUP_SIZE
        with torch.cuda.device(self.device):
            self.params = torch.empty(rows, (groups + 3) // 4 * 4, dtype=torch.int32, device=self.device)
            self.row_scale = torch.empty(rows, dtype=torch.float32, device=self.device)
            scales, biases = scales.contiguous(), biases.contiguous()
            check("am_q4_weight_pack", _lib.load().am_q4_weight_pack(
                scales.data_ptr(), biases.data_ptr(), _half_code(self.dtype), rows, self.n_in,
                self.params.data_ptr(), self.row_scale.data_ptr(), _raw_stream(self.index)))
        d = Q4WeightDesc()
        d.codes, d.params, d.row_scale = codes.data_ptr(), self.params.data_ptr(), self.row_scale.data_ptr()
        d.n_out, d.n_in, d.experts, d.dtype = self.n_out, self.n_in, self.experts, _half_code(self.dtype)
        self.desc = d
        self.ref = ctypes.byref(d)

    def __repr__(self) -> str:
        e = f"{self.experts} x " if self.grouped else ""
        return f"Q4Weight({e}{self.n_out} x {self.n_in}, {self.dtype}, {self.device})"


def _rows_of(x: torch.Tensor, w: Q4Weight) -> torch.Tensor:
    """x as rows [M, n_in] the kernels can read (a copy only where the strides need one)."""
    shape = x.shape
    if shape[-1] != w.n_in:
        raise ValueError(f"x has {shape[-1]} inputs, the weight {w.n_in}")
    if x.dtype is not w.dtype:
        raise TypeError(f"x must be {w.dtype} like the weight's scales, got {x.dtype}")
    if x.device != w.device:
        raise ValueError(f"x is on {x.device}, the weight on {w.device} (no CPU path)")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("4-bit linear layers have no backward pass: detach x or use no_grad")
    if len(shape) != 2:
        x = x.reshape(-1, w.n_in)
    stride = x.stride()
    if stride[1] != 1 or x.data_ptr() % 16 or (x.shape[0] > 1 and (stride[0] % 8 or stride[0] < w.n_in)):
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _row_stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _check_pair(w: Q4Weight, up: Q4Weight) -> None:
    if (up.n_out != w.n_out or up.n_in != w.n_in or up.experts != w.experts or up.dtype is not w.dtype
            or up.device != w.device):
        raise ValueError(f"the matrices of a gated layer must be alike, got {w} and {up}")


def _check_out(out: torch.Tensor, w: Q4Weight, shape) -> None:
    if (tuple(out.shape) != tuple(shape) or out.dtype is not w.dtype or out.device != w.device
            or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {w.dtype} tensor {tuple(shape)} on {w.device}")


def _check_apart(out: torch.Tensor, rows: torch.Tensor, what: str) -> None:
    """Refuses a contiguous `out` that shares memory with the rows a call reads: CTAs store outputs
    while others still read."""
    if out.numel() == 0 or rows.numel() == 0:
        return
    start, width = rows.data_ptr(), rows.shape[1] * rows.element_size()
    step = max(rows.stride(0) * rows.element_size(), width)
    lo = out.data_ptr()
    first = max((lo - width - start) // step + 1, 0)  # the first row that ends behind out's start
    if first < rows.shape[0] and start + first * step < lo + out.numel() * out.element_size():
        raise ValueError(f"out shares memory with {what}")


def _status_ptr(status, device):
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.device != device or status.numel() < 1:
        raise ValueError(f"status must be an int32 tensor on {device}")
    return status.data_ptr()


def _linear(x: torch.Tensor, w: Q4Weight, up: Q4Weight | None, out, status):
    if w.grouped:
        raise ValueError(f"{w} holds one matrix per expert: use expert_matmul / expert_swiglu")
    rows2 = _rows_of(x, w)
    if w.index != _current_device():
        with torch.cuda.device(w.device):
            return _linear_call(x, rows2, w, up, out, status)
    return _linear_call(x, rows2, w, up, out, status)


def _linear_call(x, rows2, w, up, out, status):
    rows = rows2.shape[0]
    if out is not None:
        _check_out(out, w, (*x.shape[:-1], w.n_out))
        _check_apart(out, rows2, "x")
    elif x.dim() == 2:
        out = torch.empty(rows, w.n_out, dtype=w.dtype, device=w.device)
    else:
        out = torch.empty(*x.shape[:-1], w.n_out, dtype=w.dtype, device=w.device)
    lib = _lib.load()
    up_ref = up.ref if up is not None else None
    need, ws = 0, None
    # (scratch of the call from the caching allocator, on the call's stream)
    if rows > (FEW_TOKENS if up is None else FEW_GATED_TOKENS) or w.n_in > FEW_INPUTS:
        need = int(lib.am_q4_linear_workspace_bytes(w.ref, up_ref, rows))
        ws = torch.empty(need, dtype=torch.uint8, device=w.device) if need else None
    rc = lib.am_q4_linear(w.ref, up_ref, rows2.data_ptr(), _row_stride(rows2), rows, out.data_ptr(),
                          w.n_out, ws.data_ptr() if need else None, need,
                          _status_ptr(status, w.device), _raw_stream(w.index))
    if rc:
        check("am_q4_linear", rc)
    return out


def quantized_matmul(x: torch.Tensor, weight: Q4Weight, *, out: torch.Tensor | None = None,
                     status: torch.Tensor | None = None):
    """x [..., n_in] times the weight's transpose -> [..., n_out] in x's type (see module
    docstring).  One token is a matrix-vector product; any number of tokens is accepted.  ``out``
    may not share memory with x.
    ``status``: optional int32 device word that gets AM_STATUS_TIMEOUT where a bounded wait of the
    tensor tiles ran out (rows of the output are then unwritten)."""
    return _linear(x, weight, None, out, status)


def quantized_swiglu(x: torch.Tensor, gate: Q4Weight, up: Q4Weight, *,
                     out: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """silu(x gate^T) * (x up^T) -> [..., n_out] in x's type, both products in one kernel and the
    gate's result never rounded in between.  ``status`` as in quantized_matmul."""
    _check_pair(gate, up)
    return _linear(x, gate, up, out, status)
