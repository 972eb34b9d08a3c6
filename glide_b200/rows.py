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

_TYPE = {torch.float32: 0, torch.uint8: 1, torch.float16: 2, torch.bfloat16: 3}


class Dispatched(NamedTuple):
    """What ``dispatch_rows`` returns. d_sorted [rows * choices, dim]: the rows by partition; d_map [rows * choices]: the row at each
    place, -1 behind the last; d_position [rows, choices]: the place of each choice, -1 for none; d_segment_start
    [partitions + 1]: the first place of each partition, then the number of places taken."""
    d_sorted: torch.Tensor
    d_map: torch.Tensor
    d_position: torch.Tensor
    d_segment_start: torch.Tensor


def _on_device(ctx: Context, name: str, t: torch.Tensor):
    if not isinstance(t, torch.Tensor) or t.device != ctx.torch_device:
        raise TypeError(f"{name} must be a tensor on {ctx.torch_device}, got {t.device if isinstance(t, torch.Tensor) else type(t)}")


def _type(name: str, t: torch.Tensor, types=(torch.float32, torch.float16, torch.bfloat16)) -> int:
    if t.dtype not in types:
        raise TypeError(f"{name} must be one of {', '.join(str(x) for x in types)}, got {t.dtype}")
    return _TYPE[t.dtype]


def _matrix(ctx: Context, name: str, t: torch.Tensor) -> int:
    """The stride of the rows of a 2-D tensor, in values."""
    _on_device(ctx, name, t)
    if t.dim() != 2:
        raise TypeError(f"{name} must have two dimensions, got {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise TypeError(f"{name} must have contiguous rows, got strides {t.stride()}")
    return t.stride(0)


def _whole(ctx: Context, name: str, t: torch.Tensor, dtype: torch.dtype, shape=None) -> int:
    """The address of a contiguous tensor of 4-byte values."""
    _on_device(ctx, name, t)
    if t.dtype != dtype and not (dtype == torch.int32 and t.dtype == torch.uint32):
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous, got strides {t.stride()}")
    return t.data_ptr()


def _result(ctx: Context, name: str, out: torch.Tensor | None, shape, dtype: torch.dtype) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=ctx.torch_device)
    _on_device(ctx, name, out)
    if out.dtype != dtype or tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}, got {out.dtype} of {tuple(out.shape)}")
    return out


def _flat(name: str, t: torch.Tensor, dim: int) -> torch.Tensor:
    """The rows of a tensor of any number of dimensions as a matrix over the same memory."""
    try:
        return t.view(-1, dim) if t.dim() != 2 else t
    except RuntimeError:
        raise TypeError(f"{name}: rows of shape {tuple(t.shape)} and strides {t.stride()} do not lie one stride apart") from None


def _stream(ctx: Context) -> int:
    return torch.cuda.current_stream(ctx.torch_device).cuda_stream


def lookup_rows(ctx: Context, d_table: torch.Tensor, d_ids: torch.Tensor, scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """scale * d_table[d_ids], rounded once, of shape d_ids.shape + (dim,); rows of zeros where an id is -1 or not a row of the
    table. d_ids: what a search returned, or tokens, in any shape. fp32 rows for a table of bytes."""
    stride = _matrix(ctx, "d_table", d_table)
    row_type = _type("d_table", d_table, tuple(_TYPE))
    n, dim = d_table.shape
    ids = _whole(ctx, "d_ids", d_ids, torch.int32)
    out = _result(ctx, "out", out, (*d_ids.shape, dim), torch.float32 if row_type == 1 else d_table.dtype)
    to = _flat("out", out, dim)
    ctx.check(ctx.lib.glide_lookup_rows(ctx.handle, d_table.data_ptr(), row_type, n, dim, stride, ids, d_ids.numel(), scale,
                                        to.data_ptr(), _matrix(ctx, "out", to), _stream(ctx)))
    return out


def lookup_rows_grad(ctx: Context, d_grad: torch.Tensor, d_ids: torch.Tensor, num: int, scale: float = 1.0,
                     dtype: torch.dtype | None = None, out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """The gradient of ``lookup_rows`` with respect to its table of `num` rows, given that of its result (d_ids.shape + (dim,)).
    dtype: that of d_grad (default) or fp32. accumulate: it is added to `out`, whose other rows stay as they are."""
    _on_device(ctx, "d_grad", d_grad)
    row_type = _type("d_grad", d_grad)
    if tuple(d_grad.shape[:-1]) != tuple(d_ids.shape) or d_grad.dim() < 1:
        raise ValueError(f"d_grad must have shape {tuple(d_ids.shape)} + (dim,), got {tuple(d_grad.shape)}")
    if accumulate and out is None:
        raise ValueError("accumulate needs the tensor to add to")
    dim = d_grad.shape[-1]
    ids = _whole(ctx, "d_ids", d_ids, torch.int32)
    count = d_ids.numel()
    rows = _flat("d_grad", d_grad, dim)
    stride = _matrix(ctx, "d_grad", rows)
    out = _result(ctx, "out", out, (num, dim), dtype or (d_grad.dtype if out is None else out.dtype))
    grad_type, out_stride = _type("out", out), _matrix(ctx, "out", out)
    need = ctx.lib.glide_lookup_rows_grad_workspace(num, dim, count)
    scratch = torch.empty(need, dtype=torch.uint8, device=ctx.torch_device)
    ctx.check(ctx.lib.glide_lookup_rows_grad(ctx.handle, rows.data_ptr(), row_type, stride, ids, count, scale, out.data_ptr(), grad_type, num,
                                             dim, out_stride, 1 if accumulate else 0, scratch.data_ptr(), need, _stream(ctx)))
    return out


def dispatch_rows(ctx: Context, d_rows: torch.Tensor, d_choice: torch.Tensor, partitions: int, out: torch.Tensor | None = None) -> Dispatched:
    """Rows sorted by the partitions that they chose: d_choice [rows, choices] holds up to 128 partitions for each row (the ids of
    ``bruteforce_knn(ctx, d_centroids, d_rows, k)``, or a router's), -1 for none. Pairs of a row and a choice are ordered by partition,
    then row, then choice. out: where the sorted rows go; rows behind the last place taken are left as they were. The gradient
    with respect to d_rows is ``dispatch_rows_grad``."""
    stride = _matrix(ctx, "d_rows", d_rows)
    row_type = _type("d_rows", d_rows)
    count, dim = d_rows.shape
    choice = _whole(ctx, "d_choice", d_choice, torch.int32)
    if d_choice.dim() != 2 or d_choice.shape[0] != count:
        raise ValueError(f"d_choice must have shape ({count}, choices), got {tuple(d_choice.shape)}")
    choices = d_choice.shape[1]
    d_sorted = _result(ctx, "out", out, (count * choices, dim), d_rows.dtype)
    sorted_stride = _matrix(ctx, "out", d_sorted)
    d_map = torch.empty(count * choices, dtype=torch.int32, device=ctx.torch_device)
    d_position = torch.empty((count, choices), dtype=torch.int32, device=ctx.torch_device)
    d_start = torch.empty(partitions + 1, dtype=torch.int32, device=ctx.torch_device)
    need = ctx.lib.glide_dispatch_rows_workspace(count, choices, partitions)
    scratch = torch.empty(need, dtype=torch.uint8, device=ctx.torch_device)
    ctx.check(ctx.lib.glide_dispatch_rows(ctx.handle, d_rows.data_ptr(), row_type, count, dim, stride, choice, choices, partitions,
                                          d_sorted.data_ptr(), sorted_stride, d_position.data_ptr(), d_map.data_ptr(), d_start.data_ptr(),
                                          scratch.data_ptr(), need, _stream(ctx)))
    return Dispatched(d_sorted, d_map, d_position, d_start)


def combine_rows(ctx: Context, d_sorted: torch.Tensor, d_position: torch.Tensor, d_weights: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """The way back: for each row the sum over its choices of weight * d_sorted[position], in fp32, rounded once. d_position: from
    ``dispatch_rows``; a place of -1 takes no part. d_weights: fp32 [rows, choices], None for 1."""
    stride = _matrix(ctx, "d_sorted", d_sorted)
    row_type = _type("d_sorted", d_sorted)
    sorted_rows, dim = d_sorted.shape
    position = _whole(ctx, "d_position", d_position, torch.int32)
    if d_position.dim() != 2:
        raise ValueError(f"d_position must have shape (rows, choices), got {tuple(d_position.shape)}")
    count, choices = d_position.shape
    weights = None if d_weights is None else _whole(ctx, "d_weights", d_weights, torch.float32, d_position.shape)
    out = _result(ctx, "out", out, (count, dim), d_sorted.dtype)
    ctx.check(ctx.lib.glide_combine_rows(ctx.handle, d_sorted.data_ptr(), row_type, sorted_rows, dim, stride, position, count, choices,
                                         weights, out.data_ptr(), _matrix(ctx, "out", out), _stream(ctx)))
    return out


def dispatch_rows_grad(ctx: Context, d_grad_sorted: torch.Tensor, d_position: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of ``dispatch_rows`` with respect to its rows: for each row the sum of the gradients at its places."""
    return combine_rows(ctx, d_grad_sorted, d_position, None, out)


def combine_rows_grad(ctx: Context, d_grad: torch.Tensor, d_sorted: torch.Tensor, d_position: torch.Tensor,
                      d_weights: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """The gradients of ``combine_rows`` with respect to its sorted rows (weight * d_grad at each place; rows that no position names
    are left as they were) and to its weights (the products of d_grad with the sorted rows, fp32, 0 for a place of -1).
    out: where the gradient of the sorted rows goes. Places have to be distinct, as ``dispatch_rows`` makes them."""
    grad_stride = _matrix(ctx, "d_grad", d_grad)
    stride = _matrix(ctx, "d_sorted", d_sorted)
    row_type = _type("d_sorted", d_sorted)
    sorted_rows, dim = d_sorted.shape
    position = _whole(ctx, "d_position", d_position, torch.int32)
    if d_position.dim() != 2:
        raise ValueError(f"d_position must have shape (rows, choices), got {tuple(d_position.shape)}")
    count, choices = d_position.shape
    if d_grad.dtype != d_sorted.dtype or tuple(d_grad.shape) != (count, dim):
        raise ValueError(f"d_grad must be {d_sorted.dtype} of shape {(count, dim)}, got {d_grad.dtype} of {tuple(d_grad.shape)}")
    weights = None if d_weights is None else _whole(ctx, "d_weights", d_weights, torch.float32, d_position.shape)
    out = _result(ctx, "out", out, (sorted_rows, dim), d_sorted.dtype)
    d_grad_weights = torch.empty((count, choices), dtype=torch.float32, device=ctx.torch_device)
    ctx.check(ctx.lib.glide_combine_rows_grad(ctx.handle, d_grad.data_ptr(), row_type, count, dim, grad_stride, d_sorted.data_ptr(),
                                              sorted_rows, stride, position, choices, weights, out.data_ptr(),
                                              _matrix(ctx, "out", out), d_grad_weights.data_ptr(), _stream(ctx)))
    return out, d_grad_weights
