"""Rotary positions with several axes - a patch's row and column, a frame's time - on the queries and keys of an attention.

The reference's cores add a table of positions to the tokens (a learned one, core/vit.py:101-106; sines, core/cct.py:17-27): its length is
the training grid's. A rotation of q and k by the position makes their product depend on the distance of two tokens alone, for any grid
and any clip length. `ViTCore` / `CCTCore` run it in every block (`args.rotary`); `rotary` is the same operator for a core of one's own."""
from __future__ import annotations

import ctypes as C
import functools
import typing as t

import torch

from . import lib as L

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_LAYOUTS = {"pairs": 0, "halves": 1}
MAX_PAIRS = 256
MAX_SIZE = 1 << 31  # the C entry's sizes have 32 bits


class _Turn(t.NamedTuple):
    sections: t.Tuple[int, ...]
    pairs: int
    base: float
    shared: int
    halves: int
    inverse: int
    array: t.Any  # sections, for the C entry


@functools.lru_cache(maxsize=64)  # checks and conversions of a call's plain arguments cost as much as its launch
def _turn(sections: t.Tuple[int, ...], base: float, layout: str, shared: bool, inverse: bool) -> _Turn:
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) < 1:
        raise ValueError(f"rotary: sections are 1 to 4 non-negative numbers of pairs, got {sections}")
    if sum(sections) > MAX_PAIRS:
        raise ValueError(f"rotary: {sum(sections)} pairs a head, at most {MAX_PAIRS} are supported")
    if layout not in _LAYOUTS:
        raise ValueError(f"rotary: layout is 'pairs' or 'halves', got {layout!r}")
    if not 0.0 < base < float("inf"):
        raise ValueError(f"rotary: base must be positive and finite, got {base}")
    return _Turn(sections, sum(sections), base, int(shared), _LAYOUTS[layout], int(inverse), (C.c_int * len(sections))(*sections))


def _back(turn: _Turn) -> _Turn:
    return _turn(turn.sections, turn.base, "halves" if turn.halves else "pairs", bool(turn.shared), not turn.inverse)


def _check(q: torch.Tensor, k: t.Optional[torch.Tensor], positions: torch.Tensor, turn: _Turn) -> None:
    for x in (q, k):
        if x is None:
            continue
        if x.dim() not in (3, 4):
            raise ValueError(f"rotary: q and k are (tokens, heads, features) or (batch, tokens, heads, features), got {tuple(x.shape)}")
        if x.dtype not in _DTYPES or x.dtype != q.dtype:
            raise TypeError(f"rotary: q and k share one of {list(_DTYPES)}, got {[y.dtype for y in (q, k) if y is not None]}")
        if 2 * turn.pairs > x.shape[-1]:
            raise ValueError(f"rotary: {turn.pairs} pairs need {2 * turn.pairs} features a head, got {x.shape[-1]}")
        if x.device != q.device or x.shape[:-2] != q.shape[:-2] or x.shape[-1] != q.shape[-1]:
            raise ValueError(f"rotary: q and k share device, batch, tokens and features, got {tuple(q.shape)} on {q.device} and {tuple(x.shape)} on {x.device}")
        if x.shape[-2] < 1:
            raise ValueError("rotary: no heads")
        if max(x.shape) >= MAX_SIZE:
            raise ValueError(f"rotary: batch, tokens, heads and features are less than {MAX_SIZE} each, got {tuple(x.shape)}")
    if positions.dtype not in _POSITION_TYPES:
        raise TypeError(f"rotary: positions are one of {list(_POSITION_TYPES)}, got {positions.dtype}")
    if positions.requires_grad:
        raise ValueError("rotary: no gradient with respect to positions")
    ok = (q.shape[-3], len(turn.sections))
    if positions.device != q.device or tuple(positions.shape) not in ((ok, (q.shape[0],) + ok) if q.dim() == 4 else (ok,)):
        raise ValueError(f"rotary: positions are (tokens, axes) = {ok} - or (batch, tokens, axes) - on {q.device}, got {tuple(positions.shape)} on {positions.device}")


def _launch(turn: _Turn, positions: torch.Tensor, pairs_of: t.Sequence[t.Tuple[torch.Tensor, torch.Tensor]]) -> None:
    """One launch over [(x, y), ...]; x and y have unit stride in their last dimension, y is x or `_like` it."""
    x0 = pairs_of[0][0]
    if x0.numel() == 0:
        return
    device = x0.get_device()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _launch(turn, positions, pairs_of)
    ops = []
    for x, y in pairs_of:
        shape, sx, sy = x.shape, x.stride(), y.stride()
        if len(shape) == 3:
            shape, sx, sy = (1, *shape), (0, *sx), (0, *sy)
        ops.append(L.RotaryOperand(x.data_ptr(), y.data_ptr(), *sx[:3], *sy[:3], shape[2], 0 if x is y else (shape[3] + 7) // 8 * 8))
    sp = positions.stride()
    L.check(L.load().v1t_rotary((L.RotaryOperand * len(ops))(*ops), len(ops), _DTYPES[x0.dtype], shape[0], shape[1], shape[3], turn.array, len(turn.sections), turn.base, turn.shared,
                                turn.halves, turn.inverse, positions.data_ptr(), _POSITION_TYPES[positions.dtype], sp[0] if len(sp) == 3 else 0, sp[-2], sp[-1],
                                L.stream_of(device)), "rotary")


def _like(x: torch.Tensor) -> torch.Tensor:
    """x's shape with room for a multiple of 8 features a head: what lies behind the last whole 8 is moved as one store, too. `.data`: a
    tensor of its own over the wider one's storage; autograd lets a view that a function returns not be changed in place."""
    shape, d = x.shape, x.shape[-1]
    if d % 8 == 0:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    return torch.empty((*shape[:-1], (d + 7) // 8 * 8), dtype=x.dtype, device=x.device).narrow(-1, 0, d).data


def _rows(x: torch.Tensor) -> torch.Tensor:
    if x.is_neg():  # the imaginary part of a conjugate view holds its numbers with the other sign
        x = x.resolve_neg()
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, turn: _Turn, positions: torch.Tensor, q: torch.Tensor, k: t.Optional[torch.Tensor]):
        ctx.set_materialize_grads(False)
        ctx.turn = turn
        ctx.save_for_backward(positions)
        xs = [_rows(x) for x in (q, k) if x is not None]
        ys = [_like(x) for x in xs]
        _launch(turn, positions, list(zip(xs, ys)))
        if k is not None and q.requires_grad != k.requires_grad:
            ctx.mark_non_differentiable(ys[q.requires_grad])
        return ys[0] if k is None else tuple(ys)

    @staticmethod
    def backward(ctx, *grads):
        """A rotation is orthogonal: the gradient turns back. Differentiable itself (a second derivative turns forward again)."""
        (positions,) = ctx.saved_tensors
        if L.dual_level():
            L.refuse_tangents("rotary", grads)
        back = _back(ctx.turn)
        out: t.List[t.Optional[torch.Tensor]] = [None, None]
        which = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[2 + i]]
        if not torch.is_grad_enabled():
            xs = [_rows(grads[i]) for i in which]
            ys = [_like(x) for x in xs]
            if which:
                _launch(back, positions, list(zip(xs, ys)))
            for i, y in zip(which, ys):
                out[i] = y
        elif len(which) == 2:
            out = list(_apply(back, positions, *grads))
        elif which:
            out[which[0]] = _apply(back, positions, grads[which[0]], None)
        return (None, None, *out)


def _apply(turn: _Turn, positions: torch.Tensor, q: torch.Tensor, k: t.Optional[torch.Tensor]):
    out = _RotaryFn.apply(turn, positions, q, k)
    for y in (out,) if k is None else out:
        if y.requires_grad:  # both results' node is one
            L.leaves_in_capture(y, "rotary")
            break
    return out


def rotary(q: torch.Tensor, positions: torch.Tensor, *, sections: t.Sequence[int], k: t.Optional[torch.Tensor] = None, base: float = 10000.0,
           layout: str = "pairs", shared: bool = False, inverse: bool = False):
    """q (and k) turned by their tokens' positions: new tensors; differentiable in q and k, any number of times, in reverse mode (forward mode is refused).
    Where 8 does not divide the number of features, the result has rows with room for the next multiple: it is not contiguous (`reshape`, not `view`, joins
    its heads).

    q: (batch, tokens, heads, features) or (tokens, heads, features), bf16 / fp16 / fp32, any strides; k: the same with its own number of heads.
    positions: (tokens, axes) for all sequences, or (batch, tokens, axes); int32, int64 or fp32, negative ones too. A token at 0 on every axis is
    left as it is (a class token).
    sections: pairs of features that each axis turns, in order; pair i of an axis with s pairs turns by position * base^(-i / s), or - `shared` - the
    P pairs of all axes share one ladder, pair j turns by position * base^(-j / P). layout: pair j is features (2j, 2j + 1), "pairs", or (j, P + j),
    "halves". Features behind the 2P turned ones are copied.
    Positions are read exactly up to 2^53. An angle is a number of turns in 64 bits, the product of the position and the rate: it is off by some 2^-52
    of itself - at the highest rate 4e-11 of a turn at position 10^6, 0.04 at 10^15 - and loses its whole turns there. What is left of it, its cosine and its
    sine are fp32, as are the products, which are rounded once to the tensor's type."""
    turn = _turn(tuple(map(int, sections)), float(base), str(layout), bool(shared), bool(inverse))  # plain values: the cache keeps none that can change
    _check(q, k, positions, turn)
    if L.dual_level():
        L.refuse_tangents("rotary", (q, k, positions))
    L.require_cuda(q, "rotary")
    if positions.is_neg():
        positions = positions.resolve_neg()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _apply(turn, positions, q, k)
    xs = [_rows(x) for x in (q, k) if x is not None]
    ys = [_like(x) for x in xs]
    _launch(turn, positions, list(zip(xs, ys)))
    return ys[0] if k is None else tuple(ys)


def _apart(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether no element of q is one of k: whole ranges apart, or - views of one packed projection - q's and k's heads beside each other in every token's
    row, or head by head in turn. (Neither overlaps itself.)"""
    if q.numel() == 0 or k.numel() == 0 or q.untyped_storage().data_ptr() != k.untyped_storage().data_ptr():
        return True

    def extent(x, dims):
        return 1 + sum((n - 1) * s for n, s in zip(x.shape[dims:], x.stride()[dims:]))

    a, b = q.storage_offset(), k.storage_offset()
    (lo, x), (hi, y) = ((a, q), (b, k)) if a <= b else ((b, k), (a, q))
    if lo + extent(x, 0) <= hi:
        return True
    # the blocks of the inner dimensions lie at multiples of the same outer strides, which count like digits; what is left of the distance sets y's behind x's
    for inner in (-2, -1):
        outer = []
        for n, m, s, t in zip(x.shape[:inner], y.shape[:inner], x.stride(), y.stride()):
            if n > 1 and m > 1 and s != t:
                break
            if max(n, m) > 1:
                outer.append((s if n > 1 else t, n, m))
        else:
            left, above = hi - lo, 1 << 62
            for s, n, m in sorted(outer, reverse=True):
                ahead, left = divmod(left, s)
                if max(n, m + ahead) * s > above:
                    break
                above = s
            else:
                if extent(x, inner) <= left and left + extent(y, inner) <= above:
                    return True
    return False


def rotary_(q: torch.Tensor, positions: torch.Tensor, *, sections: t.Sequence[int], k: t.Optional[torch.Tensor] = None, base: float = 10000.0,
            layout: str = "pairs", shared: bool = False, inverse: bool = False):
    """`rotary` in place, outside autograd (a new token's q and k, a projection's buffer): the same values, features behind the turned ones untouched.
    Positions lie in memory of their own."""
    turn = _turn(tuple(map(int, sections)), float(base), str(layout), bool(shared), bool(inverse))  # plain values: the cache keeps none that can change
    _check(q, k, positions, turn)
    xs = [x for x in (q, k) if x is not None]
    for x in xs:
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("rotary_: a tensor that requires grad cannot be turned in place; use rotary")
        if x.is_neg():
            raise ValueError("rotary_: a view that negates its memory (the imaginary part of a conjugate) cannot be turned in place; resolve_neg() copies it")
        if x.stride(-1) != 1 and x.shape[-1] > 1:
            raise ValueError(f"rotary_: unit stride in the last dimension is needed, got strides {x.stride()}")
        dims = sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1)
        if any(s < prev_s * prev_n for (prev_s, prev_n), (s, _) in zip(dims, dims[1:])) or any(s == 0 for s, _ in dims):
            raise ValueError(f"rotary_: elements of an expanded or overlapping view cannot be turned in place, got shape {tuple(x.shape)}, strides {x.stride()}")
    if k is not None and not _apart(q, k):
        raise ValueError("rotary_: q and k share elements")
    if L.dual_level():
        L.refuse_tangents("rotary_", (q, k, positions))
    L.require_cuda(q, "rotary_")
    _launch(turn, positions.resolve_neg(), [(x, x) for x in xs])
    for x in xs:
        if not x.is_inference():
            torch.autograd.graph.increment_version(x)
    return xs[0] if k is None else tuple(xs)
