"""A mixture of experts around the MXFP4 product: tokens sorted by expert, gathered, multiplied with
their expert's weight, and combined again with their weights.

    plan = xpu_kernels.expert_sort(ids, num_experts)            # ids [T, k]: each token's experts
    h = xpu_kernels.expert_linear_mxfp4(x, up, plan)            # [T, K] -> [T * k, N], sorted
    y = xpu_kernels.expert_linear_mxfp4(act(h), down, plan, sorted=True)
    out = xpu_kernels.expert_combine(y, weights, plan)          # [T, K]

A slot is a token's choice: slot ``t * k + j`` is choice ``j`` of token ``t``.  An id outside
``[0, num_experts)`` is no expert: its slot comes after all experts' rows, gives a zero row and adds
nothing.  Nothing here synchronises: the counts stay on the device, and buffers that depend on
them have the largest size they can need.
"""

from __future__ import annotations

import torch

from .int8._lib import _lib
from .mxfp4 import (
    MXFP4,
    _TYPES,
    _check_rotate,
    _empty,
    _launch,
    _quantize,
    _quantize_columns,
    _rotate,
    _rows,
    _type,
)


class ExpertPlan:
    """Where each slot goes (:func:`expert_sort`), int32 on the device.

    ``order`` [T * k]: the slot of each row; ``positions`` [T, k]: the row of each slot; ``offsets``
    [E + 1]: where each expert's rows begin, the last where the rows of no expert begin;
    ``scale_rows`` [T, k]: a slot's row among rows padded to whole 128-row tiles an expert (-1: no
    expert), ``tiles`` [E + 1]: where each expert's tiles begin.
    """

    __slots__ = ("order", "positions", "scale_rows", "offsets", "tiles", "num_experts", "tokens", "top",
                 "max_tiles")

    @property
    def rows(self):
        return self.tokens * self.top

    def __repr__(self):
        return f"ExpertPlan(tokens={self.tokens}, top={self.top}, experts={self.num_experts})"


def expert_sort(ids, num_experts):
    """``ids`` [T, k] or [T] (int32 or int64, on the GPU) -> :class:`ExpertPlan`: a stable sort of the
    slots by expert, in one or two launches."""
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if not ids.is_cuda:
        raise TypeError(f"ids must be a CUDA tensor, got {ids.device}")
    if ids.dim() not in (1, 2):
        raise ValueError(f"ids must be [T, k] or [T], got {tuple(ids.shape)}")
    if not 1 <= num_experts <= 1024:
        raise ValueError(f"num_experts must be 1 to 1024, got {num_experts}")
    ids = ids.contiguous()
    n, e = ids.numel(), num_experts
    plan = ExpertPlan()
    plan.num_experts, plan.tokens = e, ids.shape[0]
    plan.top = ids.shape[1] if ids.dim() == 2 else 1
    plan.max_tiles = n // 128 + min(e, n)
    lib = _lib()
    work = lib.xpuint8_expert_sort_workspace_bytes(n, e)
    if work < 0:
        raise ValueError(f"expert_sort: too many slots ({n})")
    buffer = torch.empty(3 * n + 2 * (e + 1) + work // 4, dtype=torch.int32, device=ids.device)
    order, positions, scale_rows, offsets, tiles, work = buffer.split([n, n, n, e + 1, e + 1, work // 4])
    plan.order, plan.offsets, plan.tiles = order, offsets, tiles
    plan.positions, plan.scale_rows = positions.view(plan.tokens, plan.top), scale_rows.view(plan.tokens, plan.top)
    if n:
        at = buffer.data_ptr()
        _launch(lib, "xpuint8_expert_sort_stream", ids.device, ids.data_ptr(), ids.element_size(), n, e,
                at, at + 4 * n, at + 8 * n, at + 12 * n, at + 12 * n + 4 * (e + 1),
                at + 12 * n + 8 * (e + 1))
    else:
        offsets.zero_()
        tiles.zero_()
    return plan


def _same_device(x, plan, what):
    if x.device != plan.order.device:
        raise ValueError(f"{what} is on {x.device} and the plan on {plan.order.device}")


def _gather(x, plan):
    t = _type(x, "x")
    x, ldx = _rows(x)
    out = torch.empty((plan.rows, x.shape[1]), dtype=x.dtype, device=x.device)
    if out.numel():
        _launch(_lib(), "xpuint8_expert_gather_stream", x.device, x.data_ptr(), t, ldx, out.data_ptr(),
                plan.positions.data_ptr(), plan.scale_rows.data_ptr(), plan.tokens, plan.top, x.shape[1])
    return out


def _combine(y, weights, plan):
    t = _type(y, "y")
    y, ldy = _rows(y)
    out = torch.empty((plan.tokens, y.shape[1]), dtype=y.dtype, device=y.device)
    if not plan.top:
        out.zero_()
    elif out.numel():
        _launch(_lib(), "xpuint8_expert_combine_stream", y.device, y.data_ptr(), t, ldy,
                None if weights is None else weights.data_ptr(), out.data_ptr(),
                plan.positions.data_ptr(), plan.scale_rows.data_ptr(), plan.tokens, plan.top, y.shape[1])
    return out


class _GatherFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _gather(x, plan)

    @staticmethod
    def backward(ctx, dy):
        return _combine(dy, None, ctx.plan), None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, plan):
        ctx.plan = plan
        ctx.save_for_backward(y, weights)
        return _combine(y, weights, plan)

    @staticmethod
    def backward(ctx, dy):
        y, weights = ctx.saved_tensors
        plan = ctx.plan
        dy, ld_dy = _rows(dy)
        y, ld_y = _rows(y)
        grad_y = torch.empty((plan.rows, y.shape[1]), dtype=y.dtype, device=y.device)
        grad_w = torch.empty((plan.tokens, plan.top), dtype=torch.float32, device=y.device)
        if grad_y.numel():
            _launch(_lib(), "xpuint8_expert_combine_grad_stream", y.device, dy.data_ptr(), _type(y, "y"),
                    ld_dy, y.data_ptr(), ld_y, weights.data_ptr(), grad_y.data_ptr(), grad_w.data_ptr(),
                    plan.positions.data_ptr(), plan.scale_rows.data_ptr(), plan.tokens, plan.top,
                    y.shape[1])
        else:
            grad_w.zero_()
        return grad_y, grad_w, None


def expert_gather(x, plan):
    """``x`` [T, W] -> its rows in the plan's order [T * k, W]; zero rows for slots of no expert.
    Differentiable: the gradient of a token is the sum of its rows'."""
    if x.dim() != 2 or x.shape[0] != plan.tokens:
        raise ValueError(f"x must be [{plan.tokens}, W], got {tuple(x.shape)}")
    _same_device(x, plan, "x")
    if x.requires_grad and torch.is_grad_enabled():
        return _GatherFn.apply(x, plan)
    return _gather(x, plan)


def expert_combine(y, weights, plan):
    """``y`` [T * k, W] in the plan's order and ``weights`` [T, k] -> [T, W]: each token's rows times
    its weights, summed in 32 bits.  Differentiable in both."""
    if y.dim() != 2 or y.shape[0] != plan.rows:
        raise ValueError(f"y must be [{plan.rows}, W], got {tuple(y.shape)}")
    if tuple(weights.shape) != (plan.tokens, plan.top) and weights.numel() != plan.rows:
        raise ValueError(f"weights must be [{plan.tokens}, {plan.top}], got {tuple(weights.shape)}")
    _same_device(y, plan, "y")
    _same_device(weights, plan, "weights")
    if not weights.is_floating_point():
        raise TypeError(f"weights must be floating point, got {weights.dtype}")
    if weights.dtype != torch.float32 or weights.dim() != 2 or not weights.is_contiguous():
        weights = weights.to(torch.float32).reshape(plan.tokens, plan.top).contiguous()
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad):
        return _CombineFn.apply(y, weights, plan)
    return _combine(y, weights, plan)


# ------------------------------------------------------------------------------ the experts' product

def _quantize_sorted(x, plan, rotate, in_order, keep=False):
    """(codes of the plan's rows, scales in padded tiles, x's rotated values): x holds tokens, or the
    plan's rows (in_order)."""
    t = _type(x, "x")
    x, ldx = _rows(x)
    k = x.shape[1]
    codes = torch.empty((plan.rows, (k + 31) // 32 * 16), dtype=torch.uint8, device=x.device)
    scales = torch.empty((plan.max_tiles, (k + 127) // 128, 32, 16), dtype=torch.uint8, device=x.device)
    rotated = torch.empty(x.shape, dtype=x.dtype, device=x.device) if keep and rotate else None
    _launch(_lib(), "xpuint8_mxfp4_quantize_sorted_stream", x.device, x.data_ptr(), t, ldx,
            codes.data_ptr(), scales.data_ptr(), None if rotated is None else rotated.data_ptr(),
            plan.order.data_ptr() if in_order else None, plan.positions.data_ptr(),
            plan.scale_rows.data_ptr(), x.shape[0], 1 if in_order else plan.top, k, 1 if rotate else 0)
    return codes, scales, (rotated if rotate else x)


def _quantize_sorted_columns(x, plan):
    """x's rows (in the plan's order) quantised along the rows, each expert's padded to whole tiles:
    codes [W, max_tiles * 64], scales."""
    t = _type(x, "x")
    x, ldx = _rows(x)
    w, tiles = x.shape[1], plan.max_tiles
    codes = torch.empty((w, tiles * 64), dtype=torch.uint8, device=x.device)
    scales = torch.empty(((w + 127) // 128, tiles, 32, 16), dtype=torch.uint8, device=x.device)
    _launch(_lib(), "xpuint8_mxfp4_quantize_columns_stream", x.device, x.data_ptr(), t, ldx,
            codes.data_ptr(), scales.data_ptr(), x.shape[0], w, 1, plan.offsets.data_ptr(),
            plan.tiles.data_ptr(), plan.num_experts, tiles)
    return codes, scales


def _expert_mm(codes, scales, w, plan, dtype):
    n, k = w.shape[1:]
    out = torch.empty((plan.rows, n), dtype=dtype, device=codes.device)
    if out.numel():
        _launch(_lib(), "xpuint8_mxfp4_expert_mm_stream", out.device, codes.data_ptr(), scales.data_ptr(),
                w.codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(), _TYPES[dtype],
                plan.offsets.data_ptr(), plan.tiles.data_ptr(), plan.rows, plan.max_tiles, n, k,
                plan.num_experts)
    return out


def _check_product(x, shape, plan, rotate, in_order):
    if len(shape) != 3 or shape[0] != plan.num_experts or x.dim() != 2 or x.shape[1] != shape[2]:
        raise ValueError(f"x {tuple(x.shape)} and the experts' weight {tuple(shape)} do not fit "
                         f"[.., K] and [{plan.num_experts}, N, K]")
    want = plan.rows if in_order else plan.tokens
    if x.shape[0] != want:
        raise ValueError(f"x must have {want} rows ({'the sorted rows' if in_order else 'the tokens'}), "
                         f"got {x.shape[0]}")
    if shape[2] == 0:
        raise ValueError("the experts' weight needs K of at least 1")
    _same_device(x, plan, "x")
    _check_rotate(shape[2], rotate)


def expert_linear_mxfp4(x, w, plan, *, rotate=True, sorted=False):
    """Each row of the plan times its expert's weight: [T * k, N] of x's type, in the plan's order.

    ``x`` [T, K] holds the tokens, each quantised once and taken to its rows; with ``sorted`` it holds
    the plan's rows [T * k, K].  ``w`` is the MXFP4 stack [E, N, K] of :func:`prepare_weight_mxfp4`.
    Rows of no expert are zero.
    """
    _check_product(x, w.shape, plan, rotate, sorted)
    _same_device(w, plan, "the weight")
    x = x.detach()
    if plan.rows == 0:
        return torch.empty((0, w.shape[1]), dtype=x.dtype, device=x.device)
    codes, scales, _ = _quantize_sorted(x, plan, rotate, sorted)
    return _expert_mm(codes, scales, w, plan, x.dtype)


class _ExpertLinearFn(torch.autograd.Function):
    """As the MXFP4 linear's, expert by expert: dx from dy and w along N, dw from dy and the rows of x
    along each expert's own rows."""

    @staticmethod
    def forward(ctx, x, w, plan, rotate, in_order):
        codes, scales, xr = _quantize_sorted(x, plan, rotate, in_order, keep=True)
        wq, wr = _quantize(w, rotate, keep=True)
        ctx.save_for_backward(xr, wr)
        ctx.plan, ctx.rotate, ctx.in_order = plan, rotate, in_order
        return _expert_mm(codes, scales, wq, plan, x.dtype)

    @staticmethod
    def backward(ctx, dy):
        xr, wr = ctx.saved_tensors
        plan = ctx.plan
        dx = dw = None
        dy = dy.contiguous()
        if ctx.needs_input_grad[0]:
            codes, scales, _ = _quantize_sorted(dy, plan, False, True)
            dx = _expert_mm(codes, scales, _quantize_columns(wr), plan, xr.dtype)
            if not ctx.in_order:
                dx = _combine(dx, None, plan)
            dx = _rotate(dx) if ctx.rotate else dx
        if ctx.needs_input_grad[1]:
            e, n, k = wr.shape
            a = _quantize_sorted_columns(dy, plan)
            b = _quantize_sorted_columns(xr if ctx.in_order else _gather(xr, plan), plan)
            dw = torch.empty((e, n, k), dtype=wr.dtype, device=wr.device)
            if dw.numel():
                _launch(_lib(), "xpuint8_mxfp4_expert_dw_stream", dw.device, a[0].data_ptr(),
                        a[1].data_ptr(), b[0].data_ptr(), b[1].data_ptr(), dw.data_ptr(),
                        _TYPES[dw.dtype], plan.tiles.data_ptr(), plan.max_tiles, n, k, e)
            dw = _rotate(dw) if ctx.rotate else dw
        return dx, dw, None, None, None


def mxfp4_expert_linear(x, w, plan, *, rotate=True, sorted=False):
    """:func:`expert_linear_mxfp4` with its gradients: ``w`` [E, N, K] stays in its own type (bf16,
    fp16, fp32) and is quantised on every call, as are the gradients' operands."""
    _check_product(x, w.shape, plan, rotate, sorted)
    _type(x, "x")
    _type(w, "w")
    _same_device(w, plan, "w")
    if plan.rows == 0:
        return x.reshape(0, x.shape[1]) @ w.sum(0).to(x.dtype).T
    return _ExpertLinearFn.apply(x, w, plan, rotate, sorted)


def expert_ffn_mxfp4(x, ids, weights, up, down, *, rotate=True):
    """The experts' SwiGLU network: ``x`` [T, K] -> [T, K].

    ``ids`` and ``weights`` [T, k] are the router's; ``up`` is the MXFP4 stack [E, 2 F, K] with rows
    ``[gate | up]``, ``down`` [E, K, F].
    """
    plan = expert_sort(ids, up.shape[0])
    gate, value = expert_linear_mxfp4(x, up, plan, rotate=rotate).chunk(2, dim=1)
    h = torch.nn.functional.silu(gate) * value
    return expert_combine(expert_linear_mxfp4(h, down, plan, rotate=rotate, sorted=True), weights, plan)
