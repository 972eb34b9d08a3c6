"""Operators on the rows of a table: rows looked up by ids and the gradient of the table, rows sorted by the partitions
(experts) that they chose, brought back with weights, and the gradients of that. They follow a search or an assignment
(whose ids and partitions go in as they come out) and precede an index (whose table they train); the reference has none.

Unlike the stages of the pipeline these calls are ordered on torch's current stream of the context's device and do not wait:
they can be captured into a graph. Rows are fp32, fp16 or bf16 (a table that is looked up may hold bytes), the last
dimension is contiguous, the rows of a matrix may lie any stride apart; ids are int32 tensors that hold uint32 patterns, -1
(0xffffffff) for none. Like the rest of the package they take torch for device memory only: no gradient is recorded,
the gradients are calls of their own.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .api import Context

_FLOATS = {torch.float32: 0, torch.float16: 2, torch.bfloat16: 3}   # GLIDE_ROW_*
_TYPES = {**_FLOATS, torch.uint8: 1}


class Dispatched(NamedTuple):
    """What ``dispatch_rows`` returns. d_sorted [rows * choices, dim]: the rows by partition; d_map [rows * choices]: the row at each
    place, -1 behind the last; d_position [rows, choices]: the place of each choice, -1 for none; d_segment_start
    [partitions + 1]: the first place of each partition, then the number of places taken. Ids have the type of d_choice."""
    d_sorted: torch.Tensor
    d_map: torch.Tensor
    d_position: torch.Tensor
    d_segment_start: torch.Tensor


# A call on a few rows takes about as long on the host as on the device, so the checks below ask each tensor for as little as they can.

def _on_device(ctx: Context, name: str, t: torch.Tensor):
    if not isinstance(t, torch.Tensor) or t.device != ctx.torch_device:
        raise TypeError(f"{name} must be a tensor on {ctx.torch_device}, got {t.device if isinstance(t, torch.Tensor) else type(t)}")


def _matrix(ctx: Context, name: str, t: torch.Tensor, types=_FLOATS) -> tuple[int, int, int]:
    """Address, type and stride between rows (in values) of a 2-D tensor."""
    if not isinstance(t, torch.Tensor) or t.device != ctx.torch_device:
        _on_device(ctx, name, t)
    kind = types.get(t.dtype)
    if kind is None:
        raise TypeError(f"{name} must be one of {', '.join(str(x) for x in types)}, got {t.dtype}")
    strides = t.stride()
    if len(strides) != 2:
        raise TypeError(f"{name} must have two dimensions, got {tuple(t.shape)}")
    if strides[1] != 1 and t.shape[1] > 1:
        raise TypeError(f"{name} must have contiguous rows, got strides {strides}")
    return t.data_ptr(), kind, strides[0]


def _whole(ctx: Context, name: str, t: torch.Tensor, dtype: torch.dtype, shape=None) -> int:
    """The address of a contiguous tensor of 4-byte values."""
    if not isinstance(t, torch.Tensor) or t.device != ctx.torch_device:
        _on_device(ctx, name, t)
    if t.dtype != dtype and not (dtype == torch.int32 and t.dtype == torch.uint32):
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous, got strides {t.stride()}")
    return t.data_ptr()


def _check_result(ctx: Context, out: torch.Tensor, shape, dtype: torch.dtype):
    _on_device(ctx, "out", out)
    if out.dtype != dtype or tuple(out.shape) != tuple(shape):
        raise ValueError(f"out must be {dtype} of shape {tuple(shape)}, got {out.dtype} of {tuple(out.shape)}")


def _flat(name: str, t: torch.Tensor, dim: int) -> torch.Tensor:
    """The rows of a tensor of any number of dimensions as a matrix over the same memory."""
    if t.dim() == 2:
        return t
    try:
        return t.view(-1, dim)
    except RuntimeError:
        raise TypeError(f"{name}: rows of shape {tuple(t.shape)} and strides {t.stride()} do not lie one stride apart") from None


# torch.cuda.current_stream(...).cuda_stream without the 2 us that its object takes, where this torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream(ctx: Context) -> int:
    return _raw_stream(ctx.device)


def lookup_rows(ctx: Context, d_table: torch.Tensor, d_ids: torch.Tensor, scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """scale * d_table[d_ids], rounded once, of shape d_ids.shape + (dim,); rows of zeros where an id is -1 or not a row of the
    table. d_ids: what a search returned, or tokens, in any shape. fp32 rows for a table of bytes."""
    table, kind, stride = _matrix(ctx, "d_table", d_table, _TYPES)
    n, dim = d_table.shape
    ids = _whole(ctx, "d_ids", d_ids, torch.int32)
    shape, dtype = d_ids.shape + (dim,), torch.float32 if kind == 1 else d_table.dtype
    if out is None:
        out = d_table.new_empty(shape, dtype=dtype) if kind == 1 else d_table.new_empty(shape)
        to, to_stride = out.data_ptr(), dim
    else:
        _check_result(ctx, out, shape, dtype)
        to, _, to_stride = _matrix(ctx, "out", _flat("out", out, dim))
    ctx.check(ctx.lib.glide_lookup_rows(ctx.handle, table, kind, n, dim, stride, ids, d_ids.numel(), scale, to, to_stride, _stream(ctx)))
    return out


def lookup_rows_grad(ctx: Context, d_grad: torch.Tensor, d_ids: torch.Tensor, num: int, scale: float = 1.0,
                     dtype: torch.dtype | None = None, out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """The gradient of ``lookup_rows`` with respect to its table of `num` rows, given that of its result (d_ids.shape + (dim,)).
    dtype: that of d_grad (default) or fp32. accumulate: it is added to `out`, whose other rows stay as they are."""
    _on_device(ctx, "d_grad", d_grad)
    if d_grad.shape[:-1] != d_ids.shape or d_grad.dim() < 1:
        raise ValueError(f"d_grad must have shape {tuple(d_ids.shape)} + (dim,), got {tuple(d_grad.shape)}")
    if accumulate and out is None:
        raise ValueError("accumulate needs the tensor to add to")
    dim = d_grad.shape[-1]
    ids = _whole(ctx, "d_ids", d_ids, torch.int32)
    count = d_ids.numel()
    grad, kind, stride = _matrix(ctx, "d_grad", _flat("d_grad", d_grad, dim))
    if out is None:
        out = d_grad.new_empty((num, dim), dtype=dtype)
    else:
        _check_result(ctx, out, (num, dim), dtype or out.dtype)
    to, to_kind, to_stride = _matrix(ctx, "out", out)
    need = ctx.lib.glide_lookup_rows_grad_workspace(num, dim, count)
    scratch = d_grad.new_empty(need, dtype=torch.uint8) if need else None   # few ids need none
    ctx.check(ctx.lib.glide_lookup_rows_grad(ctx.handle, grad, kind, stride, ids, count, scale, to, to_kind, num, dim, to_stride,
                                             1 if accumulate else 0, scratch.data_ptr() if need else None, need, _stream(ctx)))
    return out


def dispatch_rows(ctx: Context, d_rows: torch.Tensor, d_choice: torch.Tensor, partitions: int, out: torch.Tensor | None = None) -> Dispatched:
    """Rows sorted by the partitions that they chose: d_choice [rows, choices] holds up to 128 partitions for each row (the ids of
    ``bruteforce_knn(ctx, d_centroids, d_rows, k)``, or a router's), -1 for none. Pairs of a row and a choice are ordered by partition,
    then row, then choice. out: where the sorted rows go; rows behind the last place taken (d_segment_start[partitions]) are left as they
    were. Without `out` they are undefined, any bits: a product that takes in all rows, not partition by partition, wants
    out=torch.zeros(...). The gradient with respect to d_rows is ``dispatch_rows_grad``."""
    rows, kind, stride = _matrix(ctx, "d_rows", d_rows)
    count, dim = d_rows.shape
    choice = _whole(ctx, "d_choice", d_choice, torch.int32)
    if d_choice.dim() != 2 or d_choice.shape[0] != count:
        raise ValueError(f"d_choice must have shape ({count}, choices), got {tuple(d_choice.shape)}")
    choices = d_choice.shape[1]
    pairs = count * choices
    if out is None:
        out = d_rows.new_empty((pairs, dim))
    else:
        _check_result(ctx, out, (pairs, dim), d_rows.dtype)
    to, _, to_stride = _matrix(ctx, "out", out)
    # results of ids have the type that the choices have: int32, or uint32 like them
    d_map = d_choice.new_empty(pairs)
    d_position = d_choice.new_empty((count, choices))
    d_start = d_choice.new_empty(partitions + 1)
    need = ctx.lib.glide_dispatch_rows_workspace(count, choices, partitions)
    scratch = d_choice.new_empty(need, dtype=torch.uint8) if need else None
    ctx.check(ctx.lib.glide_dispatch_rows(ctx.handle, rows, kind, count, dim, stride, choice, choices, partitions, to, to_stride,
                                          d_position.data_ptr(), d_map.data_ptr(), d_start.data_ptr(),
                                          scratch.data_ptr() if need else None, need, _stream(ctx)))
    return Dispatched(out, d_map, d_position, d_start)


def combine_rows(ctx: Context, d_sorted: torch.Tensor, d_position: torch.Tensor, d_weights: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """The way back: for each row the sum over its choices of weight * d_sorted[position], in fp32, rounded once. d_position: from
    ``dispatch_rows``; a place of -1 takes no part. d_weights: fp32 [rows, choices], None for 1."""
    data, kind, stride = _matrix(ctx, "d_sorted", d_sorted)
    sorted_rows, dim = d_sorted.shape
    position = _whole(ctx, "d_position", d_position, torch.int32)
    if d_position.dim() != 2:
        raise ValueError(f"d_position must have shape (rows, choices), got {tuple(d_position.shape)}")
    count, choices = shape = d_position.shape
    weights = None if d_weights is None else _whole(ctx, "d_weights", d_weights, torch.float32, shape)
    if out is None:
        out = d_sorted.new_empty((count, dim))
    else:
        _check_result(ctx, out, (count, dim), d_sorted.dtype)
    to, _, to_stride = _matrix(ctx, "out", out)
    ctx.check(ctx.lib.glide_combine_rows(ctx.handle, data, kind, sorted_rows, dim, stride, position, count, choices, weights, to, to_stride,
                                         _stream(ctx)))
    return out


def dispatch_rows_grad(ctx: Context, d_grad_sorted: torch.Tensor, d_position: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of ``dispatch_rows`` with respect to its rows: for each row the sum of the gradients at its places."""
    return combine_rows(ctx, d_grad_sorted, d_position, None, out)


# Up to so many bytes of a new gradient are cleared whole, of more those rows that no position names, which takes three launches. us of
# the call with a result handed in, cleared whole, cleared by its marks: 33 MB 15, 28, 33; 66 MB 26, 47, 39; 102 MB of short rows 43,
# 59, 60; 131 MB 50, 89, 65; 537 MB 187, 329, 202.
_FEW_BYTES = 48 << 20


def combine_rows_grad(ctx: Context, d_grad: torch.Tensor, d_sorted: torch.Tensor, d_position: torch.Tensor,
                      d_weights: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """The gradients of ``combine_rows`` with respect to its sorted rows (weight * d_grad at each place, zeros for rows that no position
    names) and to its weights (the products of d_grad with the sorted rows, fp32, 0 for a place of -1). out: where the gradient of
    the sorted rows goes; rows of it that no position names are left as they were, which saves clearing it for every call.
    Places have to be distinct, as ``dispatch_rows`` makes them."""
    grad, kind, grad_stride = _matrix(ctx, "d_grad", d_grad)
    data, data_kind, stride = _matrix(ctx, "d_sorted", d_sorted)
    sorted_rows, dim = d_sorted.shape
    position = _whole(ctx, "d_position", d_position, torch.int32)
    if d_position.dim() != 2:
        raise ValueError(f"d_position must have shape (rows, choices), got {tuple(d_position.shape)}")
    count, choices = shape = d_position.shape
    if kind != data_kind or d_grad.shape != (count, dim):
        raise ValueError(f"d_grad must be {d_sorted.dtype} of shape {(count, dim)}, got {d_grad.dtype} of {tuple(d_grad.shape)}")
    weights = None if d_weights is None else _whole(ctx, "d_weights", d_weights, torch.float32, shape)
    clear = out is None and sorted_rows * dim * d_sorted.element_size() > _FEW_BYTES
    if out is None:
        out = d_sorted.new_empty((sorted_rows, dim)) if clear else d_sorted.new_zeros((sorted_rows, dim))
    else:
        _check_result(ctx, out, (sorted_rows, dim), d_sorted.dtype)
    to, _, to_stride = _matrix(ctx, "out", out)
    d_grad_weights = d_position.new_empty(shape, dtype=torch.float32)
    if clear:
        need = ctx.lib.glide_clear_rows_without_place_workspace(sorted_rows)
        scratch = d_position.new_empty(need, dtype=torch.uint8)
        ctx.check(ctx.lib.glide_clear_rows_without_place(ctx.handle, to, kind, sorted_rows, dim, to_stride, position, count * choices,
                                                         scratch.data_ptr(), need, _stream(ctx)))
    ctx.check(ctx.lib.glide_combine_rows_grad(ctx.handle, grad, kind, count, dim, grad_stride, data, sorted_rows, stride, position, choices,
                                              weights, to, to_stride, d_grad_weights.data_ptr(), _stream(ctx)))
    return out, d_grad_weights
