"""Orthogonalised updates: `orthogonalize`, the momentum step `muon_step` around it, and `FusedMuon`, the optimizer of a model whose matrices
take that step and whose other parameters keep `FusedAdamW`'s (the reference steps all of them with AdamW, train.py:216-223).

A matrix's update is replaced by (nearly) the closest matrix with all singular values one: every direction that the gradient points to moves equally
far, whatever its scale. The products are Newton-Schulz steps, all matrices of a model in one launch each (csrc/orthogonal.hip)."""
from __future__ import annotations

import ctypes as C
import functools
import math
import typing as t

import torch

from . import lib as L

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # drive singular values to about 1 (0.7 to 1.2) within five steps from 0.003 on
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_STEPS = 32
MAX_SIDE, MAX_LENGTH, MAX_ELEMENTS = 1 << 15, 1 << 22, 1 << 31
_SIZES = f"matrices have at most {MAX_ELEMENTS} elements, {MAX_SIDE} rows or columns of the shorter side and {MAX_LENGTH} of the longer"


def _coefficients(coefficients, steps: int) -> t.Any:
    if not 0 <= int(steps) <= MAX_STEPS:
        raise ValueError(f"orthogonalize: 0 to {MAX_STEPS} steps, got {steps}")
    c = tuple(coefficients)
    if len(c) == 3 and all(isinstance(x, (int, float)) for x in c):
        c = (c,) * int(steps)
    if len(c) != steps or any(len(x) != 3 for x in c):
        raise ValueError(f"orthogonalize: coefficients are (a, b, c) or one such triple for each of the {steps} steps")
    return _floats(tuple(float(v) for x in c for v in x))


@functools.lru_cache(maxsize=32)
def _floats(values: t.Tuple[float, ...]):
    return (C.c_float * max(1, len(values)))(*values)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(shapes: t.Tuple[t.Tuple[int, int], ...]) -> int:
    n = len(shapes)
    for s in shapes:
        if min(s) > MAX_SIDE or max(s) > MAX_LENGTH or s[0] * s[1] > MAX_ELEMENTS:
            raise ValueError(f"orthogonalize: {_SIZES}, got {s}")
    return int(L.load().v1t_orthogonalize_ws_bytes((C.c_int * n)(*[r for r, _ in shapes]), (C.c_int * n)(*[c for _, c in shapes]), n))


def _workspace(shapes: t.Sequence[t.Tuple[int, int]], device) -> torch.Tensor:
    nbytes = _workspace_bytes(tuple(shapes))
    L.check(min(nbytes, 0), "orthogonalize")
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _refused(code: int, what: str) -> None:
    if code == -1:
        raise ValueError(f"{what}: coefficients under which the iteration's numbers grow to 128 or more (or are not finite), or a negative eps")
    L.check(code, what)


def orthogonalize(updates, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
    """Each update's Newton-Schulz iterate: X = U / (|U|_F + eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T (of the shorter side).

    updates: a matrix, a stack (count, rows, cols), or a list of matrices of any shapes; bf16 / fp16 / fp32, any strides, one device. Returns new contiguous
    tensors, laid out alike. coefficients: (a, b, c) or one triple per step. A matrix of zeros stays zero; NaN or infinity spoils its own matrix only. Not
    differentiable.

    Sums are fp32 whatever the type, operands are held to 22 bits at one exponent per matrix, the result is rounded once: the error is that of fp32 arithmetic
    relative to the matrix (2e-6 of its norm), not to each number - a row 1e-5 below the others keeps some 15 bits, 1e-7 below 9. The same call gives the
    same bits; beside other matrices, whose sizes decide how the products are cut, a matrix's last bits may be others."""
    one = isinstance(updates, torch.Tensor)
    if one and updates.dim() not in (2, 3):
        raise ValueError(f"orthogonalize: a matrix, a stack of matrices or a list of matrices, got shape {tuple(updates.shape)}")
    us = ([updates] if updates.dim() == 2 else list(updates)) if one else list(updates)
    co = _coefficients(coefficients, steps)
    if not 0.0 <= float(eps) < math.inf:
        raise ValueError(f"orthogonalize: eps must be non-negative and finite, got {eps}")
    for u in us:
        if not isinstance(u, torch.Tensor) or u.dim() != 2:
            raise ValueError("orthogonalize: every update is a matrix")
        if u.dtype not in _DTYPES or u.dtype != us[0].dtype:
            raise TypeError(f"orthogonalize: updates share one of {list(_DTYPES)}, got {sorted({str(x.dtype) for x in us})}")
        if u.numel() > MAX_ELEMENTS:  # a size could wrap in the C entry's 32 bits; `_workspace` checks the sides
            raise ValueError(f"orthogonalize: {_SIZES}, got {tuple(u.shape)}")
        if u.device != us[0].device:
            raise ValueError("orthogonalize: updates on several devices")
        if torch.is_grad_enabled() and u.requires_grad:
            raise RuntimeError("orthogonalize: not differentiable; call it under torch.no_grad() or on detached tensors")
    if L.dual_level():
        L.refuse_tangents("orthogonalize", us)
    if not us:
        return updates.clone() if one else []
    L.require_cuda(us[0], "orthogonalize")
    if one and updates.dim() == 3:
        out = torch.empty(updates.shape, dtype=updates.dtype, device=updates.device)
        outs: t.List[torch.Tensor] = list(out)
    else:
        outs = [torch.empty(u.shape, dtype=u.dtype, device=u.device) for u in us]
        out = outs[0] if one else outs
    _orthogonalize([(u.resolve_neg(), o) for u, o in zip(us, outs) if u.numel()], int(steps), co, float(eps))
    return out


def _orthogonalize(pairs, steps: int, co, eps: float) -> None:
    if not pairs:
        return
    u0 = pairs[0][0]
    if u0.get_device() != torch.cuda.current_device():
        with torch.cuda.device(u0.get_device()):
            return _orthogonalize(pairs, steps, co, eps)
    units = (L.Matrix * len(pairs))()
    for m, (u, o) in zip(units, pairs):
        m.in_, m.out = u.data_ptr(), o.data_ptr()
        m.row_stride, m.col_stride = u.stride()
        m.rows, m.cols = u.shape
    ws = _workspace([tuple(u.shape) for u, _ in pairs], u0.device)
    _refused(L.load().v1t_orthogonalize(units, len(pairs), _DTYPES[u0.dtype], steps, co, eps, ws.data_ptr(), ws.numel(), L.stream_of(u0.get_device())), "orthogonalize")


def muon_step(params: t.Sequence[torch.Tensor], grads: t.Sequence[torch.Tensor], moments: t.Sequence[torch.Tensor], *, lr, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.0, l1: float = 0.0, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
              zero_grad: bool = False) -> None:
    """One step over matrices, in place: g' = g + l1 sign(p); m <- momentum m + g'; U = g' + momentum m (or m, without Nesterov's look ahead);
    p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows / cols)) orthogonalize(U).

    fp32 tensors without gaps of the same shape per matrix; a parameter of more dimensions (a convolution's) is a matrix of its first dimension
    by all others. lr: a number, or one per matrix. zero_grad: the gradients are cleared. No two tensors of the call may share memory."""
    params, grads, moments = list(params), list(grads), list(moments)
    if not len(params) == len(grads) == len(moments):
        raise ValueError(f"muon_step: {len(params)} parameters, {len(grads)} gradients, {len(moments)} momenta")
    lrs = [float(x) for x in lr] if isinstance(lr, (list, tuple)) else [float(lr)] * len(params)
    if len(lrs) != len(params):
        raise ValueError(f"muon_step: {len(lrs)} learning rates for {len(params)} parameters")
    co = _coefficients(coefficients, steps)
    eps, momentum, weight_decay, l1 = float(eps), float(momentum), float(weight_decay), float(l1)
    if not 0.0 <= eps < math.inf or not all(map(math.isfinite, (momentum, weight_decay, l1, *lrs))):
        raise ValueError("muon_step: eps is non-negative, every coefficient is finite")
    rs, spans, device = [], [], params[0].get_device() if params else 0
    for p, g, m, a in zip(params, grads, moments, lrs):
        shape = p.shape
        if len(shape) < 2:
            raise ValueError(f"muon_step: a parameter of shape {tuple(shape)} is no matrix")
        if not p.dtype is g.dtype is m.dtype is torch.float32:
            raise TypeError(f"muon_step: fp32 tensors are needed, got {[x.dtype for x in (p, g, m)]}")
        if not (g.shape == shape == m.shape and p.is_contiguous() and g.is_contiguous() and m.is_contiguous() and p.get_device() == g.get_device() == m.get_device() == device):
            raise ValueError(f"muon_step: parameter, gradient and momentum are contiguous tensors of one shape on one device, got {[(tuple(x.shape), str(x.device)) for x in (p, g, m)]}")
        if p.is_neg() or g.is_neg() or m.is_neg():
            raise ValueError("muon_step: views that negate their memory (the imaginary part of a conjugate) cannot be updated in place; resolve_neg() copies them")
        size = p.numel()
        if size == 0:
            continue
        if size > MAX_ELEMENTS:
            raise ValueError(f"muon_step: {_SIZES}, got {tuple(shape)}")
        rows, at = shape[0], (p.data_ptr(), g.data_ptr(), m.data_ptr())
        cols = size // rows
        spans += [(x, x + 4 * size) for x in at]
        rs.append(L.MuonRange(*at, rows, cols, a * (rows / cols) ** 0.5 if rows > cols else a, 1.0 - a * weight_decay, l1, 0))
    spans.sort()
    end = 0
    for x, y in spans:
        if x < end:
            raise ValueError("muon_step: tensors of the call share memory")
        end = y
    if L.dual_level():
        L.refuse_tangents("muon_step", params + grads + moments)
    if not rs:
        return
    L.require_cuda(params[0], "muon_step")
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            muon_ranges(rs, momentum, nesterov, int(steps), co, eps, zero_grad, params[0].device)
    else:
        muon_ranges(rs, momentum, nesterov, int(steps), co, eps, zero_grad, params[0].device)
    touched = params + moments + (grads if zero_grad else [])
    torch.autograd.graph.increment_version([x for x in touched if not x.is_inference()])


def muon_ranges(rs: t.Sequence[L.MuonRange], momentum: float, nesterov: bool, steps: int, co, eps: float, zero_grad: bool, device) -> None:
    """`v1t_muon_step` over a table of matrices, on the current stream."""
    ws = _workspace([(r.rows, r.cols) for r in rs], device)
    _refused(L.load().v1t_muon_step((L.MuonRange * len(rs))(*rs), len(rs), momentum, int(bool(nesterov)), steps, co, eps, int(bool(zero_grad)), ws.data_ptr(),
                                    ws.numel(), L.stream()), "muon_step")
