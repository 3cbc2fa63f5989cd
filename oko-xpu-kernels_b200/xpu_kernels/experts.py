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

from . import mxfp4
from .mxfp4 import _check_rotate, _load, _type


class ExpertPlan:
    """Where each slot goes (:func:`expert_sort`), int32 on the device.

    ``order`` [T * k]: the slot of each row; ``positions`` [T, k]: the row of each slot; ``offsets``
    [E + 1]: where each expert's rows begin, the last where the rows of no expert begin;
    ``scale_rows`` [T, k]: a slot's row among rows padded to whole 128-row tiles an expert (-1: no
    expert), ``tiles`` [E + 1]: where each expert's tiles begin.  ``max_tiles`` bounds the tiles of any
    routing of these sizes.
    """

    __slots__ = ("num_experts", "tokens", "top", "rows", "max_tiles", "_buffer", "_index")

    # the arrays follow one another in one buffer and become tensors when asked for
    @property
    def order(self):
        return self._buffer[:self.rows]

    @property
    def positions(self):
        n = self.rows
        return self._buffer[n:2 * n].view(self.tokens, self.top)

    @property
    def scale_rows(self):
        n = self.rows
        return self._buffer[2 * n:3 * n].view(self.tokens, self.top)

    @property
    def offsets(self):
        return self._buffer[3 * self.rows:3 * self.rows + self.num_experts + 1]

    @property
    def tiles(self):
        at = 3 * self.rows + self.num_experts + 1
        return self._buffer[at:at + self.num_experts + 1]

    def __repr__(self):
        return f"ExpertPlan(tokens={self.tokens}, top={self.top}, experts={self.num_experts})"


def expert_sort(ids, num_experts):
    """``ids`` [T, k] or [T] (int32 or int64, on the GPU) -> :class:`ExpertPlan`: a stable sort of the
    slots by expert, in one or two launches."""
    size = ids.element_size()
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    index = ids.get_device()
    if index < 0:
        raise TypeError(f"ids must be a CUDA tensor, got {ids.device}")
    shape = ids.shape
    if len(shape) not in (1, 2):
        raise ValueError(f"ids must be [T, k] or [T], got {tuple(shape)}")
    if not 1 <= num_experts <= 1024:
        raise ValueError(f"num_experts must be 1 to 1024, got {num_experts}")
    if not ids.is_contiguous():
        ids = ids.contiguous()
    plan = ExpertPlan()
    plan.num_experts, plan.tokens, plan._index = num_experts, shape[0], index
    plan.top = shape[1] if len(shape) == 2 else 1
    n = plan.rows = plan.tokens * plan.top
    plan.max_tiles = n // 128 + min(num_experts, n)
    plan._buffer = (mxfp4._native or _load()).sort(ids, num_experts)
    return plan


def _same_device(index, plan, x, what):
    if index != plan._index:
        raise ValueError(f"{what} is on {x.device} and the plan on {plan._buffer.device}")


def expert_gather(x, plan):
    """``x`` [T, W] -> its rows in the plan's order [T * k, W]; zero rows for slots of no expert.
    Differentiable: the gradient of a token is the sum of its rows'."""
    if x.dim() != 2 or x.shape[0] != plan.tokens:
        raise ValueError(f"x must be [{plan.tokens}, W], got {tuple(x.shape)}")
    _same_device(x.get_device(), plan, x, "x")
    _type(x, "x")
    return (mxfp4._native or _load()).gather(x, plan._buffer, plan.tokens, plan.top, plan.num_experts)


def expert_combine(y, weights, plan):
    """``y`` [T * k, W] in the plan's order and ``weights`` [T, k] (or [T * k], a value a slot) -> [T, W]:
    each token's rows times its weights, summed in 32 bits.  Differentiable in both."""
    if y.dim() != 2 or y.shape[0] != plan.rows:
        raise ValueError(f"y must be [{plan.rows}, W], got {tuple(y.shape)}")
    shape = (plan.tokens, plan.top)
    if weights.shape != shape and weights.shape != (plan.rows,):
        raise ValueError(f"weights must be [{plan.tokens}, {plan.top}], got {tuple(weights.shape)}")
    _same_device(y.get_device(), plan, y, "y")
    _same_device(weights.get_device(), plan, weights, "weights")
    if not weights.is_floating_point():
        raise TypeError(f"weights must be floating point, got {weights.dtype}")
    if weights.dtype != torch.float32 or weights.shape != shape or not weights.is_contiguous():
        weights = weights.to(torch.float32).reshape(shape).contiguous()
    _type(y, "y")
    return (mxfp4._native or _load()).combine(y, weights, plan._buffer, plan.tokens, plan.top, plan.num_experts)


# ------------------------------------------------------------------------------ the experts' product

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
    _same_device(x.get_device(), plan, x, "x")
    if rotate and shape[2] % 256:
        _check_rotate(shape[2], rotate)


def expert_linear_mxfp4(x, w, plan, *, rotate=True, sorted=False):
    """Each row of the plan times its expert's weight: [T * k, N] of x's type, in the plan's order.

    ``x`` [T, K] holds the tokens, each quantised once and taken to its rows; with ``sorted`` it holds
    the plan's rows [T * k, K].  ``w`` is the MXFP4 stack [E, N, K] of :func:`prepare_weight_mxfp4`.
    Rows of no expert are zero.  For serving: a backward pass that reaches the result raises
    (:func:`mxfp4_expert_linear` has gradients).
    """
    _check_product(x, w.shape, plan, rotate, sorted)
    _type(x, "x")
    codes, scales = w._held
    if codes.get_device() != plan._index:
        raise ValueError(f"the weight is on {w.device} and the plan on {plan._buffer.device}")
    return (mxfp4._native or _load()).expert_linear(x, codes, scales, w.shape[1], plan._buffer, plan.tokens, plan.top,
                                                    plan.num_experts, rotate, sorted)


def mxfp4_expert_linear(x, w, plan, *, rotate=True, sorted=False):
    """:func:`expert_linear_mxfp4` with its gradients: ``w`` [E, N, K] stays in its own type (bf16,
    fp16, fp32) and is quantised on every call, as are the gradients' operands: as the linear's, expert by
    expert, dx from dy and w along N, dw from dy and the rows of x along each expert's own rows."""
    _check_product(x, w.shape, plan, rotate, sorted)
    _type(x, "x")
    _type(w, "w")
    _same_device(w.get_device(), plan, w, "w")
    if plan.rows == 0:
        return x[:0] @ w[0].to(x.dtype).T
    return (mxfp4._native or _load()).expert_train(x, w, plan._buffer, plan.tokens, plan.top, rotate, sorted)


def expert_ffn_mxfp4(x, ids, weights, up, down, *, rotate=True):
    """The experts' SwiGLU network: ``x`` [T, K] -> [T, K].

    ``ids`` and ``weights`` [T, k] are the router's; ``up`` is the MXFP4 stack [E, 2 F, K] with rows
    ``[gate | up]``, ``down`` [E, K, F].  For serving: ``weights`` may ask for a gradient, which
    :func:`expert_combine` gives, but a backward pass to ``x`` raises (:func:`expert_linear_mxfp4`).
    """
    plan = expert_sort(ids, up.shape[0])
    gate, value = expert_linear_mxfp4(x, up, plan, rotate=rotate).chunk(2, dim=1)
    h = torch.nn.functional.silu(gate) * value
    return expert_combine(expert_linear_mxfp4(h, down, plan, rotate=rotate, sorted=True), weights, plan)
