"""Mixture-of-experts layers over 4-bit weights: routing, grouped products, combination.

A layer of experts runs as::

    r = route_experts(logits, top_k)              # which experts, their weights, sorted rows
    h = expert_swiglu(x, gate, up, r)             # [tokens * top_k, inner], rows by expert
    y = expert_matmul(h, down, r)                 # [tokens * top_k, width], rows by expert
    out = combine_experts(y, r.weights, r.positions, residual=x)

Nothing of it comes back to the host: the experts' row counts stay on the device, and the
products read each expert that has rows once.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._lib import check
from .kernels import _half_code, dtype_code
from .linear import (Q4Weight, _check_apart, _check_out, _check_pair, _current_device, _raw_stream, _row_stride,
                     _rows_of, _status_ptr)

MAX_EXPERTS, MAX_TOP_K = 1024, 32


class ExpertRouting(NamedTuple):
    """Which experts each token goes to (int32 tensors but for the weights).

    experts, weights, positions: [tokens, top_k]; offsets: [n_experts + 1]; order: [tokens *
    top_k], the (token, slot) pairs ``t * top_k + j`` sorted by expert (stable).  Rows
    ``[offsets[e], offsets[e + 1])`` of a sorted tensor are expert e's, and pair (t, j) is row
    ``positions[t, j]``."""

    experts: torch.Tensor
    weights: torch.Tensor
    offsets: torch.Tensor
    order: torch.Tensor
    positions: torch.Tensor


def _int32(t: torch.Tensor, shape, device, what: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device:
        raise ValueError(f"{what} must be int32 {tuple(shape)} on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def route_experts(logits: torch.Tensor, top_k: int, *, normalize: bool = True) -> ExpertRouting:
    """Top-k routing of logits [tokens, n_experts] (float32, float16 or bfloat16).

    Per token the ``top_k`` largest logits in falling order, the lower index first among equal
    ones (NaN counts as -inf), with softmax weights over the chosen logits (``normalize``) or
    over all of them.  A token whose logits are all -inf has weights 0; infinite logits share
    the weight equally."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, n_experts], got {tuple(logits.shape)}")
    tokens, n_experts = logits.shape
    if not 1 <= top_k <= min(MAX_TOP_K, n_experts) or n_experts > MAX_EXPERTS:
        raise ValueError(f"top_k in 1..min({MAX_TOP_K}, n_experts) and n_experts <= {MAX_EXPERTS} "
                         f"required, got {top_k} of {n_experts}")
    dev = logits.device
    if not logits.is_cuda:
        raise ValueError("Q4 kernels run on CUDA tensors only (no CPU path)")
    if logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("route_experts has no backward pass: detach the logits or use no_grad")
    if logits.stride(1) != 1 or (tokens > 1 and logits.stride(0) < n_experts):
        logits = logits.contiguous()
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _route_call(logits, tokens, n_experts, top_k, normalize, dev)
    return _route_call(logits, tokens, n_experts, top_k, normalize, dev)


def _route_call(logits, tokens, n_experts, top_k, normalize, dev):
    pairs = tokens * top_k
    # one buffer: experts, positions, order, offsets
    buf = torch.empty(3 * pairs + n_experts + 1, dtype=torch.int32, device=dev)
    weights = torch.empty(tokens, top_k, dtype=torch.float32, device=dev)
    base = buf.data_ptr()
    rc = _lib.load().am_route_experts(
        logits.data_ptr(), dtype_code(logits.dtype), _row_stride(logits), tokens, n_experts, top_k,
        1 if normalize else 0, base, weights.data_ptr(), base + 12 * pairs, base + 8 * pairs,
        base + 4 * pairs, _raw_stream(dev.index))
    if rc:
        check("am_route_experts", rc)
    shape, strides = (tokens, top_k), (top_k, 1)
    return ExpertRouting(buf.as_strided(shape, strides, 0), weights,
                         buf.as_strided((n_experts + 1,), (1,), 3 * pairs),
                         buf.as_strided((pairs,), (1,), 2 * pairs),
                         buf.as_strided(shape, strides, pairs))


def _expert_linear(x, w: Q4Weight, up, routing: ExpertRouting, gather: bool, out, status):
    if not w.grouped:
        raise ValueError(f"{w} is one matrix: use quantized_matmul / quantized_swiglu")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, {w.n_in}], got {tuple(x.shape)}")
    x = _rows_of(x, w)
    rows = routing.order.shape[0]
    offsets = _int32(routing.offsets, (w.experts + 1,), w.device, "routing.offsets")
    order, top_k = None, 1
    if gather:
        order = _int32(routing.order, (rows,), w.device, "routing.order")
        top_k = routing.experts.shape[1]
        if x.shape[0] * top_k != rows:
            raise ValueError(f"x has {x.shape[0]} tokens, the routing {rows} rows of {top_k} each")
    elif x.shape[0] != rows:
        raise ValueError(f"x has {x.shape[0]} rows, the routing {rows}")
    if w.index != _current_device():
        with torch.cuda.device(w.device):
            return _expert_call(x, w, up, offsets, order, top_k, rows, out, status)
    return _expert_call(x, w, up, offsets, order, top_k, rows, out, status)


def _expert_call(x, w, up, offsets, order, top_k, rows, out, status):
    if out is not None:
        _check_out(out, w, (rows, w.n_out))
        _check_apart(out, x, "x")
    else:
        out = torch.empty(rows, w.n_out, dtype=w.dtype, device=w.device)
    lib = _lib.load()
    up_ref = up.ref if up is not None else None
    need = int(lib.am_q4_expert_linear_workspace_bytes(w.ref, up_ref, rows))
    ws = torch.empty(need, dtype=torch.uint8, device=w.device) if need else None
    rc = lib.am_q4_expert_linear(w.ref, up_ref, x.data_ptr(), _row_stride(x), x.shape[0],
                                 offsets.data_ptr(), order.data_ptr() if order is not None else None,
                                 top_k, rows, out.data_ptr(), w.n_out, ws.data_ptr() if need else None,
                                 need, _status_ptr(status, w.device), _raw_stream(w.index))
    if rc:
        check("am_q4_expert_linear", rc)
    return out


def expert_matmul(x: torch.Tensor, weight: Q4Weight, routing: ExpertRouting, *, gather: bool = False,
                  out: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """Row r of x [tokens * top_k, n_in], sorted by expert, times its expert's matrix (with
    ``gather`` x is [tokens, n_in] and each pair's row is fetched through ``routing.order``)
    -> [tokens * top_k, n_out] sorted by expert.  ``status``: optional int32 device word that
    gets AM_STATUS_* bits: for order entries outside x, and where a bounded wait of the tensor
    tiles ran out (rows of the output are then unwritten)."""
    return _expert_linear(x, weight, None, routing, gather, out, status)


def expert_swiglu(x: torch.Tensor, gate: Q4Weight, up: Q4Weight, routing: ExpertRouting, *,
                  gather: bool = True, out: torch.Tensor | None = None,
                  status: torch.Tensor | None = None):
    """silu(x gate_e^T) * (x up_e^T) for each (token, slot) pair's expert e, from x [tokens, n_in]
    -> [tokens * top_k, n_out] sorted by expert (``gather=False``: x holds the sorted rows)."""
    _check_pair(gate, up)
    return _expert_linear(x, gate, up, routing, gather, out, status)


def combine_experts(y: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, *,
                    residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    status: torch.Tensor | None = None):
    """out[t] = residual[t] + sum_j weights[t, j] * y[positions[t, j]]: y [rows, width] float16
    or bfloat16, weights float32 and positions int32 [tokens, top_k].  fp32 sums, rounded once.
    ``out`` may be the residual itself; it may not share memory with y."""
    if not y.is_cuda:
        raise ValueError("Q4 kernels run on CUDA tensors only (no CPU path)")
    if y.dim() != 2 or positions.dim() != 2:
        raise ValueError("y must be [rows, width] and positions [tokens, top_k]")
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad):
        raise RuntimeError("combine_experts has no backward pass: detach its inputs or use no_grad")
    dev, shape, width = y.device, positions.shape, y.shape[1]
    tokens, top_k = shape
    if top_k == 0:
        raise ValueError("positions must hold at least one slot a token")
    positions = _int32(positions, shape, dev, "positions")
    if weights.dtype is not torch.float32 or weights.shape != shape or weights.device != dev:
        raise ValueError(f"weights must be float32 {tuple(shape)} on {dev}")
    if not weights.is_contiguous():
        weights = weights.contiguous()
    code = _half_code(y.dtype)
    y = _dense_rows(y, width)
    res, res_stride = None, 0
    if residual is not None:
        if residual.shape != (tokens, width) or residual.dtype is not y.dtype or residual.device != dev:
            raise ValueError(f"residual must be {y.dtype} {(tokens, width)} on {dev}")
        residual = _dense_rows(residual, width)
        res, res_stride = residual.data_ptr(), _row_stride(residual)
    if out is None:
        out = torch.empty(tokens, width, dtype=y.dtype, device=dev)
    elif (out.shape != (tokens, width) or out.dtype is not y.dtype or out.device != dev
          or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {y.dtype} tensor {(tokens, width)} on {dev}")
    else:
        _check_apart(out, y, "y")
        if residual is not None and not (out.data_ptr() == res and res_stride == width):
            _check_apart(out, residual, "residual other than row by row")
    args = (y.data_ptr(), code, _row_stride(y), y.shape[0], weights.data_ptr(), positions.data_ptr(),
            res, res_stride, out.data_ptr(), width, tokens, top_k, width, _status_ptr(status, dev),
            _raw_stream(dev.index))
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            rc = _lib.load().am_combine_experts(*args)
    else:
        rc = _lib.load().am_combine_experts(*args)
    if rc:
        check("am_combine_experts", rc)
    return out


def _dense_rows(t: torch.Tensor, width: int) -> torch.Tensor:
    stride = t.stride()
    return t if stride[1] == 1 and (stride[0] >= width or t.shape[0] <= 1) else t.contiguous()
