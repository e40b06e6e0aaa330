"""Operators driven by integer ids next to the energy network (``include/ebr_tokens.h``): what a training step does with
tokens before the first layer, inside a sparse layer and after the last one.

* ``scaled_embedding(tokens, weight, scale)``: ``scale * weight[tokens]`` with one rounding, from the float32 master table
  or a 16-bit one. Its gradient is a sum over the tokens sorted by id: no atomics, the same bits each time.
* ``expert_route(expert_ids, experts)`` sorts a router's choices by expert; ``expert_dispatch(x, route)`` copies tokens to
  their experts' rows and ``expert_combine(rows, route, weights)`` adds the rows back, weighted. Differentiable to every
  order (the network's energy gradient is itself differentiated in training): the adjoints are the same kernels.
* ``topk_distill_loss(logits, teacher_ids, teacher_logits)``: the Kullback-Leibler divergence from a teacher that is given
  by its top logits, per row or reduced. A reduced loss makes its gradient in the forward pass, where the logits are at hand.

All run the kernels of ``libebr_attn.so`` on the current CUDA stream, in float32 arithmetic with fixed summation orders.
An id outside its range is a padding id everywhere: a zero row, no expert, no entry. CUDA only: a CPU tensor is an error.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ebr_b200 import _native

Tensor = torch.Tensor

_DTYPES = {
    torch.float32: _native.FLOAT32,
    torch.float16: _native.FLOAT16,
    torch.bfloat16: _native.BFLOAT16,
}
_IDS = {torch.int32: _native.INT32, torch.int64: _native.INT64}


# ---------------------------------------------------------------------------------------------------- plumbing

_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _require(t: Tensor, what: str, name: str, types: dict, device: Optional[torch.device] = None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs only on CUDA (sm_100a) tensors, got {name} on {t.device}; there is no CPU path")
    if t.dtype not in types:
        raise TypeError(f"{what}: unsupported dtype {t.dtype} of {name}")
    if device is not None and t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, the other tensors are on {device}")


def _has_tangent(*tensors: Optional[Tensor]) -> bool:
    """Whether one of them carries a forward-mode tangent, which no kernel here propagates: such a call goes through its
    autograd Function, which refuses it. A direct call would drop it, and a dropped tangent counts as zero. Asked for only
    inside a forward-mode level (``forward_ad._current_level >= 0``): elsewhere there are none, and a call is short."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _fine(t: Tensor, types: dict) -> bool:
    return t.is_cuda and t.dtype in types


def _call(what: str, device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` on ``device``'s current stream (the C ABI launches on the current device). The raw stream
    handle is asked for directly: a ``torch.cuda.Stream`` object costs as much host time as the launch."""
    index = device.index
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    if status:
        _native.check(status, what)


def _row_view(t: Tensor) -> Tuple[Tensor, int]:
    """(tensor, row stride) of ``t`` [..., C] seen as rows of C unit-stride elements; copies where no one stride leads
    through all its rows."""
    c = t.shape[-1]
    if t.is_contiguous():
        return t, c
    stride = _row_stride(t)
    return (t.contiguous(), c) if stride is None else (t, stride)


def _row_stride(t: Tensor) -> Optional[int]:
    """The stride between the rows of a tensor that is not contiguous, None where there is no single one."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        return None
    step, rows = None, 1  # the rows of the dimensions so far lie `step` apart
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != step * rows:
            return None
        rows *= size
    return t.shape[-1] if step is None else step


def _scratch(nbytes: int, like: Tensor) -> Optional[Tensor]:
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _as(t: Tensor, dtype: torch.dtype) -> Tensor:
    return t if t.dtype == dtype else t.to(dtype)


# ---------------------------------------------------------------------------------------------------- embedding


def _lookup(tokens: Tensor, weight: Tensor, scale: float, dtype: torch.dtype) -> Tensor:
    weight, stride = _row_view(weight)
    v, c = weight.shape
    out = weight.new_empty((*tokens.shape, c), dtype=dtype)
    _call("scaled_embedding", weight.device, _native.lib().ebr_scaled_embedding, _DTYPES[weight.dtype], _DTYPES[dtype],
          _IDS[tokens.dtype], tokens.numel(), v, c, scale, tokens.data_ptr(), weight.data_ptr(), stride,
          out.data_ptr())  # fmt: skip
    return out


def _lookup_grad(tokens: Tensor, g: Tensor, scale: float, rows: int, dtype: torch.dtype) -> Tensor:
    g, stride = _row_view(g)
    n, c = tokens.numel(), g.shape[-1]
    dw = g.new_empty((rows, c), dtype=dtype)
    lib = _native.lib()
    nbytes = lib.ebr_scaled_embedding_grad_scratch_bytes(n, rows, c)
    scratch = _scratch(nbytes, g)
    _call("scaled_embedding_grad", g.device, lib.ebr_scaled_embedding_grad, _DTYPES[g.dtype], _DTYPES[dtype],
          _IDS[tokens.dtype], n, rows, c, scale, tokens.data_ptr(), g.data_ptr(), stride, dw.data_ptr(), _ptr(scratch),
          nbytes)  # fmt: skip
    return dw


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight: Tensor, tokens: Tensor, scale: float, dtype: torch.dtype) -> Tensor:
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.rows, ctx.dtype = scale, weight.shape[0], weight.dtype
        return _lookup(tokens, weight, scale, dtype)

    @staticmethod
    def backward(ctx, g: Tensor):
        (tokens,) = ctx.saved_tensors
        if torch.is_grad_enabled() or forward_ad._current_level >= 0 and _has_tangent(g):
            return _EmbedGrad.apply(g, tokens, ctx.scale, ctx.rows, ctx.dtype), None, None, None
        return _lookup_grad(tokens, g, ctx.scale, ctx.rows, ctx.dtype), None, None, None


class _EmbedGrad(torch.autograd.Function):
    """The table's gradient as a function of the output's; linear, so its own backward is the lookup."""

    @staticmethod
    def forward(ctx, g: Tensor, tokens: Tensor, scale: float, rows: int, dtype: torch.dtype) -> Tensor:
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.dtype = scale, g.dtype
        return _lookup_grad(tokens, g, scale, rows, dtype)

    @staticmethod
    def backward(ctx, gg: Tensor):
        (tokens,) = ctx.saved_tensors
        return _Embed.apply(gg, tokens, ctx.scale, ctx.dtype), None, None, None, None


def scaled_embedding(tokens: Tensor, weight: Tensor, scale: float = 1.0, dtype: Optional[torch.dtype] = None) -> Tensor:
    """``round(scale * weight[tokens])``, ``[*tokens.shape, C]`` of ``dtype`` (default: ``weight``'s).

    ``tokens``: int32 or int64 of any shape; an id outside ``[0, V)`` gives a row of zeros and no gradient. ``weight``
    ``[V, C]``: float32, float16 or bfloat16. Differentiable in ``weight`` to every order; the gradient has its type and is
    summed in float32."""
    if not _fine(weight, _DTYPES) or not _fine(tokens, _IDS) or tokens.device != weight.device:
        _require(weight, "scaled_embedding", "weight", _DTYPES)
        _require(tokens, "scaled_embedding", "tokens", _IDS, weight.device)
    if weight.dim() != 2 or not weight.shape[0] or not weight.shape[1]:
        raise ValueError(f"scaled_embedding: weight must be [V, C], got {tuple(weight.shape)}")
    dtype = weight.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise TypeError(f"scaled_embedding: unsupported output dtype {dtype}")
    tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad or forward_ad._current_level >= 0 and _has_tangent(weight):
        return _Embed.apply(weight, tokens, float(scale), dtype)
    return _lookup(tokens, weight, float(scale), dtype)


# ---------------------------------------------------------------------------------------------------- experts


class ExpertRoute(NamedTuple):
    """Where each token's slots go (``expert_route``). ``row_of`` [*tokens, K]: the slot's row, -1 for a dropped one.
    ``slot_of`` [rows]: the row's slot (token * K + k), -1 for a row of no slot. ``offsets`` [experts + 1]: the first
    sorted position of each expert, counting every slot, so ``offsets[1:] - offsets[:-1]`` are the experts' loads; without
    a capacity, expert e's rows are ``offsets[e]`` to ``offsets[e + 1]``. All int32 on the device."""

    row_of: Tensor
    slot_of: Tensor
    offsets: Tensor
    experts: int
    capacity: Optional[int]

    @property
    def rows(self) -> int:
        return self.slot_of.shape[0]

    @property
    def top_k(self) -> int:
        return self.row_of.shape[-1]


def expert_route(expert_ids: Tensor, experts: int, capacity: Optional[int] = None) -> ExpertRoute:
    """Sort the slots of ``expert_ids`` [..., K] (int32 or int64) by expert, keeping their order within an expert.

    Without ``capacity`` the experts' rows follow one another (``[tokens * K, C]`` buffers, the tail zero where ids are
    invalid). With it, each expert owns ``capacity`` rows (``[experts * capacity, C]``, a batch for ``torch.bmm``), its
    later slots are dropped and its unused rows are zero; nothing on the host depends on the loads, so the layer can be
    captured in a CUDA graph. At most 1024 experts; an id outside ``[0, experts)`` is a dropped slot."""
    _require(expert_ids, "expert_route", "expert_ids", _IDS)
    if expert_ids.dim() < 1 or not expert_ids.shape[-1]:
        raise ValueError(f"expert_route: expert_ids must be [..., K], got {tuple(expert_ids.shape)}")
    if not 1 <= experts <= 1024:
        raise ValueError(f"expert_route: 1 to 1024 experts, got {experts}")
    if capacity is not None and capacity < 1:
        raise ValueError(f"expert_route: the capacity must be positive, got {capacity}")
    ids, dev = expert_ids.contiguous(), expert_ids.device
    k, slots = ids.shape[-1], ids.numel()
    rows = slots if capacity is None else experts * capacity
    row_of = ids.new_empty(ids.shape, dtype=torch.int32)
    slot_of = ids.new_empty(rows, dtype=torch.int32)
    offsets = ids.new_empty(experts + 1, dtype=torch.int32)
    lib = _native.lib()
    nbytes = lib.ebr_expert_route_scratch_bytes(slots // k, k, experts)
    scratch = _scratch(nbytes, ids)
    _call("expert_route", dev, lib.ebr_expert_route, _IDS[ids.dtype], slots // k, k, experts, capacity or 0,
          ids.data_ptr(), row_of.data_ptr(), slot_of.data_ptr(), offsets.data_ptr(), _ptr(scratch), nbytes)  # fmt: skip
    return ExpertRoute(row_of, slot_of, offsets, experts, capacity)


def _weight_args(weights: Optional[Tensor], x: Tensor):
    if weights is None:
        return None, _native.FLOAT32
    if weights.dtype != torch.float32 and weights.dtype != x.dtype:
        weights = weights.float()
    return weights if weights.is_contiguous() else weights.contiguous(), _DTYPES[weights.dtype]


def _scatter(x: Tensor, route: ExpertRoute, weights: Optional[Tensor], rows_in: Optional[Tensor], want_rows: bool,
             dots_dtype: Optional[torch.dtype] = None) -> Tuple[Optional[Tensor], Optional[Tensor]]:  # fmt: skip
    x, stride = _row_view(x)
    c, row_of, slot_of = x.shape[-1], route.row_of, route.slot_of
    k, rows = row_of.shape[-1], slot_of.shape[0]
    weights, code = _weight_args(weights, x)
    if weights is None and dots_dtype is not None:
        code = _DTYPES[dots_dtype]
    out = x.new_empty((rows, c)) if want_rows else None
    dots = None
    if rows_in is not None:
        rows_in = _as(rows_in, x.dtype).contiguous()
        dots = x.new_empty(row_of.shape, dtype=torch.float32 if code == _native.FLOAT32 else x.dtype)
    _call("expert_scatter", x.device, _native.lib().ebr_expert_scatter, _DTYPES[x.dtype], code, row_of.numel() // k, k, c,
          rows, x.data_ptr(), stride, row_of.data_ptr(), slot_of.data_ptr(), _ptr(weights), _ptr(rows_in), _ptr(out),
          _ptr(dots))  # fmt: skip
    return out, dots


def _combine(rows: Tensor, route: ExpertRoute, weights: Optional[Tensor]) -> Tensor:
    rows, stride = _row_view(rows)
    c, row_of = rows.shape[-1], route.row_of
    k = row_of.shape[-1]
    weights, code = _weight_args(weights, rows)
    y = rows.new_empty((*row_of.shape[:-1], c))
    _call("expert_combine", rows.device, _native.lib().ebr_expert_combine, _DTYPES[rows.dtype], code, row_of.numel() // k,
          k, c, rows.data_ptr(), stride, row_of.data_ptr(), _ptr(weights), y.data_ptr())  # fmt: skip
    return y


class _Dispatch(torch.autograd.Function):
    """rows[row_of[t, k]] = weights[t, k] * x[t] (weights None: ones). Its adjoints are the combine and the row dots."""

    @staticmethod
    def forward(ctx, x: Tensor, weights: Optional[Tensor], route: ExpertRoute) -> Tensor:
        ctx.route = route
        ctx.weighted = weights is not None
        if ctx.weighted:
            ctx.save_for_backward(x, weights)
        return _scatter(x, route, weights, None, True)[0]

    @staticmethod
    def backward(ctx, g: Tensor):
        route = ctx.route
        direct = not (torch.is_grad_enabled() or forward_ad._current_level >= 0 and _has_tangent(g))
        if direct and not ctx.weighted:
            return _combine(g, route, None), None, None
        x, weights = ctx.saved_tensors if ctx.weighted else (None, None)
        gx = _Combine.apply(g, weights, route) if ctx.needs_input_grad[0] else None
        gw = _RowDots.apply(x, g, route, weights.dtype) if ctx.weighted and ctx.needs_input_grad[1] else None
        return gx, gw, None


class _Combine(torch.autograd.Function):
    """y[t] = sum_k weights[t, k] * rows[row_of[t, k]] (weights None: ones)."""

    @staticmethod
    def forward(ctx, rows: Tensor, weights: Optional[Tensor], route: ExpertRoute) -> Tensor:
        ctx.route = route
        ctx.weighted = weights is not None
        if ctx.weighted:
            ctx.save_for_backward(rows, weights)
        return _combine(rows, route, weights)

    @staticmethod
    def backward(ctx, g: Tensor):
        route = ctx.route
        rows, weights = ctx.saved_tensors if ctx.weighted else (None, None)
        need_rows, need_weights = ctx.needs_input_grad[:2]
        direct = not (torch.is_grad_enabled() or forward_ad._current_level >= 0 and _has_tangent(g))
        if direct and need_rows and need_weights and ctx.weighted:
            grows, gw = _scatter(_as(g, rows.dtype), route, weights, rows, True)  # both in one pass over g and the rows
            return grows, _as(gw, weights.dtype), None
        grows = _Dispatch.apply(g, weights, route) if need_rows else None
        gw = _RowDots.apply(g, rows, route, weights.dtype) if ctx.weighted and need_weights else None
        return grows, gw, None


class _RowDots(torch.autograd.Function):
    """dots[t, k] = <x[t], rows[row_of[t, k]]>: the gradient of the weights, bilinear in x and the rows."""

    @staticmethod
    def forward(ctx, x: Tensor, rows: Tensor, route: ExpertRoute, dtype: torch.dtype) -> Tensor:
        ctx.route = route
        ctx.save_for_backward(x, rows)
        code = dtype if dtype in (torch.float32, x.dtype) else torch.float32
        return _scatter(x, route, None, rows, False, code)[1].to(dtype)

    @staticmethod
    def backward(ctx, g: Tensor):
        x, rows = ctx.saved_tensors
        gx = _Combine.apply(rows, g, ctx.route) if ctx.needs_input_grad[0] else None
        grows = _Dispatch.apply(x, g, ctx.route) if ctx.needs_input_grad[1] else None
        return gx, grows, None, None


def expert_dispatch(x: Tensor, route: ExpertRoute) -> Tensor:
    """Each token's vector in the rows of its experts: ``[rows, C]`` with ``rows[route.row_of[t, k]] = x[t]`` and zeros in
    rows of no slot. ``x`` [*tokens, C] in float32, float16 or bfloat16; differentiable to every order."""
    if not _fine(x, _DTYPES) or x.device != route.row_of.device:
        _require(x, "expert_dispatch", "x", _DTYPES, route.row_of.device)
    if x.dim() < 1 or x.shape[:-1] != route.row_of.shape[:-1] or not x.shape[-1]:
        raise ValueError(
            f"expert_dispatch: x must be [*{tuple(route.row_of.shape[:-1])}, C] for this route, got {tuple(x.shape)}"
        )
    if torch.is_grad_enabled() and x.requires_grad or forward_ad._current_level >= 0 and _has_tangent(x):
        return _Dispatch.apply(x, None, route)
    return _scatter(x, route, None, None, True)[0]


def expert_combine(rows: Tensor, route: ExpertRoute, weights: Optional[Tensor] = None) -> Tensor:
    """The experts' rows added back to their tokens: ``y[t] = sum_k weights[t, k] * rows[route.row_of[t, k]]`` (``weights``
    None: ones), ``[*tokens, C]``, dropped slots adding nothing. ``rows`` [rows, C] in float32, float16 or bfloat16;
    ``weights`` [*tokens, K] (float32 or the rows' type are read as they are). The sum is float32 with one rounding.
    Differentiable in both to every order."""
    if not _fine(rows, _DTYPES) or rows.device != route.row_of.device:
        _require(rows, "expert_combine", "rows", _DTYPES, route.row_of.device)
    if rows.dim() != 2 or rows.shape[0] != route.rows or not rows.shape[1]:
        raise ValueError(f"expert_combine: rows must be [{route.rows}, C] for this route, got {tuple(rows.shape)}")
    if weights is not None:
        if not _fine(weights, _DTYPES) or weights.device != rows.device:
            _require(weights, "expert_combine", "weights", _DTYPES, rows.device)
        if weights.shape != route.row_of.shape:
            raise ValueError(
                f"expert_combine: weights must be {tuple(route.row_of.shape)} for this route, got {tuple(weights.shape)}"
            )
    if (torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))
            or forward_ad._current_level >= 0 and _has_tangent(rows, weights)):  # fmt: skip
        return _Combine.apply(rows, weights, route)
    return _combine(rows, route, weights)


# ---------------------------------------------------------------------------------------------------- distillation


def _distill_args(view: Tensor, ids: Tensor, top: Tensor, tau: float, factor: float):
    """The leading arguments that both entry points share."""
    k = ids.shape[-1]
    return (_DTYPES[view.dtype], _IDS[ids.dtype], _DTYPES[top.dtype], ids.numel() // k, view.shape[-1], k, tau, factor)


def _distill(view: Tensor, stride: int, ids: Tensor, top: Tensor, tau: float, row_weight: Optional[Tensor], factor: float,
             total: bool, gradient: bool):  # fmt: skip
    """(losses, total or None, stats, gradient or None): ``ebr_topk_distill`` on a row view of the logits."""
    rows = ids.numel() // ids.shape[-1]
    losses = view.new_empty(ids.shape[:-1], dtype=torch.float32)
    stats = view.new_empty((rows, 2), dtype=torch.float32)
    total = view.new_empty((), dtype=torch.float32) if total else None
    grad, grad_stride = _distill_grad_buffer(view, stride) if gradient else (None, 0)
    _call("topk_distill_loss", view.device, _native.lib().ebr_topk_distill,
          *_distill_args(view, ids, top, tau, factor), view.data_ptr(), stride, ids.data_ptr(),
          top.data_ptr(), _ptr(row_weight), losses.data_ptr(), stats.data_ptr(), _ptr(total), _ptr(grad),
          grad_stride)  # fmt: skip
    return losses, total, stats, grad


def _distill_gradient(view: Tensor, ids: Tensor, top: Tensor, tau: float, row_weight: Optional[Tensor], factor: float,
                      stats: Tensor, upstream: Tensor, made: Optional[Tensor]) -> Tensor:  # fmt: skip
    """The gradient for ``upstream``, a scalar or one value per row: ``ebr_topk_distill_grad`` on the forward's row view.
    ``made``: the buffer that the forward filled for an upstream of 1."""
    view, stride = _row_view(view)
    if made is None:
        grad, grad_stride = _distill_grad_buffer(view, stride)
    else:
        grad, grad_stride = _row_view(made)
    if upstream.dtype != torch.float32:
        upstream = upstream.float()
    if upstream.dim() == 0 or not any(upstream.stride()):  # one value, or one value expanded over the rows
        per_row = 0
    else:
        upstream, per_row = upstream.contiguous(), 1
    _call("topk_distill_loss", view.device, _native.lib().ebr_topk_distill_grad,
          *_distill_args(view, ids, top, tau, factor), view.data_ptr(), stride, ids.data_ptr(),
          top.data_ptr(), _ptr(row_weight), stats.data_ptr(), upstream.data_ptr(), per_row, int(made is not None),
          grad.data_ptr(), grad_stride)  # fmt: skip
    return grad


def _distill_grad_buffer(view: Tensor, stride: int) -> Tuple[Tensor, int]:
    """The gradient's buffer and row stride: contiguous, or with the logits' row stride where they are a view of slightly
    longer rows (a padded vocabulary), so that both rows start at the same place of a 16-byte word."""
    v = view.shape[-1]
    if v < stride <= v + 256 and view.dim() > 1:
        strides, step = [1], stride
        for size in reversed(view.shape[:-1]):
            strides.append(step)
            step *= size
        return torch.empty_strided(view.shape, strides[::-1], device=view.device, dtype=view.dtype), stride
    return view.new_empty(view.shape), v


class _TopkDistill(torch.autograd.Function):
    """Rows' losses (``reduced`` false) or their sum times the factor. A reduced loss writes its gradient for an upstream of
    1 in the forward pass, where a row's logits have just been read; the backward hands it out, and a kernel that reads
    the real upstream on the device rewrites it from the logits only where that is not 1 (a loss scale, a mixed loss).
    A further backward through the same graph gets a gradient of its own."""

    @staticmethod
    def forward(ctx, logits, ids, top, tau, row_weight, factor, reduced):
        view, stride = _row_view(logits)  # saved as it is: a copy, where there has to be one, is made once
        losses, total, stats, ctx.made = _distill(view, stride, ids, top, tau, row_weight, factor, reduced, reduced)
        ctx.save_for_backward(view, ids, top, row_weight, stats)
        ctx.tau, ctx.factor = tau, factor
        return total if reduced else losses

    @staticmethod
    def backward(ctx, g: Tensor):
        if torch.is_grad_enabled():
            return _TopkDistill._backward_once(ctx, g)
        return _TopkDistill._backward(ctx, g)

    @staticmethod
    def _backward(ctx, g: Tensor):
        if forward_ad._current_level >= 0 and _has_tangent(g):
            raise NotImplementedError("topk_distill_loss has no forward-mode derivative")
        view, ids, top, row_weight, stats = ctx.saved_tensors
        made, ctx.made = ctx.made, None
        grad = _distill_gradient(view, ids, top, ctx.tau, row_weight, ctx.factor, stats, g, made)
        return grad, None, None, None, None, None, None

    _backward_once = staticmethod(once_differentiable(_backward.__func__))


def topk_distill_loss(logits: Tensor, teacher_ids: Tensor, teacher_logits: Tensor, temperature: float = 1.0, *,
                      row_weight: Optional[Tensor] = None, reduction: str = "mean") -> Tensor:  # fmt: skip
    """Distillation from a teacher given by its top logits: for each row, ``temperature**2`` times the Kullback-Leibler
    divergence of ``softmax(logits / temperature)`` from the softmax of the row's K teacher entries.

    ``logits`` [..., V] in float32, float16 or bfloat16; ``teacher_ids`` [..., K] int32 or int64, an id outside ``[0, V)``
    being no entry (a shorter list, a masked row); ``teacher_logits`` [..., K]; ``row_weight`` [...] multiplies the rows'
    losses. A row without entries, with entries of -inf alone, or of weight 0, has loss 0 and gradient 0 whatever its logits
    hold. ``reduction``: ``"none"`` (the rows' losses, float32), ``"sum"`` or ``"mean"`` (the sum over the number of rows).
    Differentiable once, in ``logits``; the teacher and the weights are constants. A reduced loss keeps a gradient of the
    logits' size from the forward to the backward pass. Logits whose rows do not lie one stride apart are copied, once: leave positions out by
    ``row_weight`` or padding ids rather than by a slice such as ``logits[:, :-1]``."""
    what = "topk_distill_loss"
    if not (_fine(logits, _DTYPES) and _fine(teacher_ids, _IDS) and _fine(teacher_logits, _DTYPES)
            and logits.device == teacher_ids.device == teacher_logits.device):  # fmt: skip
        _require(logits, what, "logits", _DTYPES)
        _require(teacher_ids, what, "teacher_ids", _IDS, logits.device)
        _require(teacher_logits, what, "teacher_logits", _DTYPES, logits.device)
    shape, entries = logits.shape, teacher_ids.shape
    if not shape or not entries or entries[:-1] != shape[:-1] or not shape[-1]:
        raise ValueError(f"{what}: logits [..., V] and teacher_ids [..., K] must have the same rows, got "
                         f"{tuple(shape)} and {tuple(entries)}")  # fmt: skip
    if teacher_logits.shape != entries or not 1 <= entries[-1] <= 1024:
        raise ValueError(f"{what}: teacher_logits must be shaped as teacher_ids with 1 to 1024 entries a row, got "
                         f"{tuple(teacher_logits.shape)} and {tuple(entries)}")  # fmt: skip
    if shape[-1] > 1 << 19:
        raise ValueError(f"{what}: a vocabulary of at most {1 << 19}, got {shape[-1]}")
    if not 2.0**-126 <= temperature <= 1e30:
        raise ValueError(f"{what}: the temperature must be between 1.2e-38 and 1e30, got {temperature}")
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"{what}: reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if teacher_logits.requires_grad or (row_weight is not None and row_weight.requires_grad):
        raise ValueError(f"{what}: the teacher and the row weights are constants; detach them")
    if row_weight is not None:
        _require(row_weight, what, "row_weight", _DTYPES, logits.device)
        if row_weight.shape != shape[:-1]:
            raise ValueError(f"{what}: row_weight must be {tuple(shape[:-1])}, got {tuple(row_weight.shape)}")
        row_weight = row_weight.to(torch.float32).contiguous()
    ids = teacher_ids if teacher_ids.is_contiguous() else teacher_ids.contiguous()
    top = teacher_logits if teacher_logits.is_contiguous() else teacher_logits.contiguous()
    rows = ids.numel() // entries[-1]
    factor = 1.0 / rows if reduction == "mean" and rows else 1.0
    reduced = reduction != "none"
    if (torch.is_grad_enabled() and logits.requires_grad
            or forward_ad._current_level >= 0 and _has_tangent(logits, top, row_weight)):  # fmt: skip
        return _TopkDistill.apply(logits, ids, top, float(temperature), row_weight, factor, reduced)
    losses, total, _, _ = _distill(*_row_view(logits), ids, top, float(temperature), row_weight, factor, reduced, False)
    return total if reduced else losses


__all__ = [
    "ExpertRoute",
    "expert_combine",
    "expert_dispatch",
    "expert_route",
    "scaled_embedding",
    "topk_distill_loss",
]
