"""MXFP4: 4-bit operands in blocks of 32 with a power-of-two scale, their product, and the linears
built on them.

    w = xpu_kernels.prepare_weight_mxfp4(weight)         # once: rotated and quantised
    y = xpu_kernels.linear_mxfp4(x, w, bias)             # serving: bf16 / fp16 / fp32 in and out
    y = xpu_kernels.mxfp4_linear(x, weight, bias)        # training: both operands in 4 bits, gradients too

A block of 32 values v is held as ``code * 2^(e - 127)`` with ``e = max(floor(log2 max|v|) + 125, 0)``
and each code the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, above 6 to 6); a block
with a NaN or an infinity is NaN.  ``rotate=True`` puts the group-256 rotation of the int8 path in
front of both operands (K a multiple of 256), which spreads outlier channels over their group and
leaves the product unchanged.

The kernels run on torch's current stream; nothing here synchronises.
"""

from __future__ import annotations

import torch

from .int8._lib import _err, _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_raw_stream = torch._C._cuda_getCurrentRawStream


def _launch(lib, entry, device, *args):
    """One C entry on the current stream of `device`; raises what it reports."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = getattr(lib, entry)(_raw_stream(index), *args)
    else:
        with torch.cuda.device(index):
            rc = getattr(lib, entry)(_raw_stream(index), *args)
    if rc != 0:
        _err(lib, entry[len("xpuint8_"):-len("_stream")])


def _type(x, what):
    t = _TYPES.get(x.dtype)
    if t is None:
        raise TypeError(f"{what} must be bfloat16, float16 or float32, got {x.dtype}")
    if not x.is_cuda:
        raise TypeError(f"{what} must be a CUDA tensor, got {x.device}")
    return t


def _rows(x):
    """x [R, K] with unit column stride (a copy where it has none), and its row stride."""
    if x.stride(1) != 1 and x.shape[1] != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else x.shape[1])


def _check_rotate(k, rotate):
    if rotate and k % 256:
        raise ValueError(f"K={k} is not a multiple of the ConvRot group size (256)")


class MXFP4:
    """A matrix [R, K] (or a stack [E, R, K]) in MXFP4.

    ``codes`` uint8 ``[.., R, ceil(K / 32) * 16]``: two codes to a byte, the earlier in the low half;
    ``scales`` uint8 ``[.., ceil(R / 128), ceil(K / 128), 32, 16]``: the exponent of row ``32 j + l`` of a
    128-row tile and its block ``b`` (of four) at ``[l, 4 j + b]``.  Both contiguous and 16-byte
    aligned, so they can be saved and loaded as they are.
    """

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes, scales, shape):
        shape = tuple(int(n) for n in shape)
        if len(shape) not in (2, 3):
            raise ValueError(f"an MXFP4 matrix has the shape [R, K] or [E, R, K], got {shape}")
        r, k = shape[-2:]
        lead = shape[:-2]
        want_codes = (*lead, r, (k + 31) // 32 * 16)
        want_scales = (*lead, (r + 127) // 128, (k + 127) // 128, 32, 16)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
        if tuple(codes.shape) != want_codes or tuple(scales.shape) != want_scales:
            raise ValueError(f"an MXFP4 matrix {shape} has codes {want_codes} and scales {want_scales}, "
                             f"got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"codes are on {codes.device} and scales on {scales.device}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        self.codes, self.scales, self.shape = codes, scales, shape

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return f"MXFP4({self.shape}, device={self.device})"


def _empty(shape, device):
    *lead, r, k = shape
    q = MXFP4.__new__(MXFP4)
    q.codes = torch.empty((*lead, r, (k + 31) // 32 * 16), dtype=torch.uint8, device=device)
    q.scales = torch.empty((*lead, (r + 127) // 128, (k + 127) // 128, 32, 16), dtype=torch.uint8,
                           device=device)
    q.shape = tuple(shape)
    return q


def _quantize(x, rotate=False, keep=False):
    """(MXFP4 of x [R, K] or [E, R, K], the rotated values where `keep` asks for them)."""
    t = _type(x, "x")
    k = x.shape[-1]
    if x.dim() == 2:
        x, ldx = _rows(x)
        each = x.shape[0]
    else:
        x, ldx, each = x.contiguous(), k, x.shape[-2]
    q = _empty(x.shape, x.device)
    rotated = torch.empty(x.shape, dtype=x.dtype, device=x.device) if keep and rotate else None
    rows = x.numel() // k if k else 0
    if rows:
        _launch(_lib(), "xpuint8_mxfp4_quantize_stream", x.device, x.data_ptr(), t, ldx,
                q.codes.data_ptr(), q.scales.data_ptr(), rotated.data_ptr() if keep and rotate else None,
                rows, k, each, 1 if rotate else 0)
    return q, (rotated if rotate else x)


def _quantize_columns(x):
    """MXFP4 of x's transpose: [R, C] -> [C, R], [E, R, C] -> [E, C, R]."""
    t = _type(x, "x")
    rows, cols = x.shape[-2:]
    if x.dim() == 2:
        x, ldx = _rows(x)
        matrices, shape = 1, (cols, rows)
    else:
        x, ldx, matrices = x.contiguous(), cols, x.shape[0]
        shape = (matrices, cols, rows)
    q = _empty(shape, x.device)
    if x.numel():
        _launch(_lib(), "xpuint8_mxfp4_quantize_columns_stream", x.device, x.data_ptr(), t, ldx,
                q.codes.data_ptr(), q.scales.data_ptr(), rows, cols, matrices, None, None, 0, 0)
    return q


def _rotate(x):
    """The rotation alone, of x's type, along the last axis."""
    x = x.contiguous()
    out = torch.empty_like(x)
    k = x.shape[-1]
    if x.numel():
        rows = x.numel() // k
        _launch(_lib(), "xpuint8_mxfp4_quantize_stream", x.device, x.data_ptr(), _type(x, "x"), k, None,
                None, out.data_ptr(), rows, k, rows, 1)
    return out


def quantize_mxfp4(x, *, rotate=False, transpose=False):
    """``x`` [R, K] or a stack [E, R, K] (bf16, fp16, fp32; any K) -> :class:`MXFP4` along K.

    ``rotate`` puts the group-256 rotation in front (K a multiple of 256), its result rounded to x's
    type.  ``transpose`` gives the MXFP4 of ``x``'s transpose instead, blocks along R.
    """
    if x.dim() not in (2, 3):
        raise ValueError(f"x must be [R, K] or [E, R, K], got {tuple(x.shape)}")
    if transpose:
        if rotate:
            raise ValueError("rotate goes along K: transpose quantises along the other axis")
        return _quantize_columns(x)
    _check_rotate(x.shape[-1], rotate)
    return _quantize(x, rotate)[0]


def dequantize_mxfp4(q, dtype=torch.bfloat16):
    """The values that ``q`` stands for (rotated ones where it was quantised with ``rotate``)."""
    t = _TYPES.get(dtype)
    if t is None:
        raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    if out.numel():
        r, k = q.shape[-2:]
        _launch(_lib(), "xpuint8_mxfp4_dequantize_stream", out.device, q.codes.data_ptr(),
                q.scales.data_ptr(), out.data_ptr(), t, out.numel() // k, k, r)
    return out


def prepare_weight_mxfp4(w, rotate=True):
    """A weight [N, K] (or the experts' [E, N, K]) for :func:`linear_mxfp4`: rotated and quantised."""
    return quantize_mxfp4(w.detach(), rotate=rotate)


def _bias(bias, n, device):
    if bias is None:
        return None
    if bias.numel() != n:
        raise ValueError(f"bias has {bias.numel()} values; expected N={n}")
    b = bias.detach().reshape(-1).to(device=device, dtype=torch.float32).contiguous()
    return b.clone() if b.data_ptr() % 16 else b


def _mm(a, b, bias, dtype):
    m, n, k = a.shape[0], b.shape[0], a.shape[1]
    out = torch.empty((m, n), dtype=dtype, device=a.codes.device)
    if m and n:
        _launch(_lib(), "xpuint8_mxfp4_mm_stream", out.device, a.codes.data_ptr(), a.scales.data_ptr(),
                b.codes.data_ptr(), b.scales.data_ptr(), None if bias is None else bias.data_ptr(),
                out.data_ptr(), _TYPES[dtype], n, m, n, k)
    return out


def mxfp4_mm(a, b, bias=None, dtype=torch.bfloat16):
    """``a @ b.T (+ bias)`` of two MXFP4 matrices [M, K] and [N, K]: summed in 32 bits, rounded once."""
    if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"mxfp4_mm takes [M, K] and [N, K], got {a.shape} and {b.shape}")
    if a.shape[1] == 0:
        raise ValueError("mxfp4_mm needs K of at least 1")
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    if a.device != b.device:
        raise ValueError(f"a is on {a.device} and b on {b.device}")
    return _mm(a, b, _bias(bias, b.shape[0], a.device), dtype)


def linear_mxfp4(x, w, bias=None, *, rotate=True):
    """The MXFP4 linear: ``x`` [.., K] (bf16, fp16, fp32) -> [.., N] of x's type.

    ``w`` is the :class:`MXFP4` weight [N, K] of :func:`prepare_weight_mxfp4`, ``rotate`` what it was
    prepared with.  ``bias`` is added in 32 bits before the one rounding.
    """
    if len(w.shape) != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x has {x.shape[-1]} columns and the weight is {w.shape}")
    if x.device != w.codes.device:
        raise ValueError(f"x is on {x.device} and the weight on {w.device}")
    n, k = w.shape
    _check_rotate(k, rotate)
    x2 = x.detach().reshape(-1, k)
    q, _ = _quantize(x2, rotate)
    out = _mm(q, w, _bias(bias, n, x.device), x.dtype)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)


class _Mxfp4LinearFn(torch.autograd.Function):
    """y = Q(x) Q(w)^T with both operands quantised along K; the gradients' products quantise their
    operands along their own contractions, dy and w along N for dx, dy and x along the rows for dw
    (straight through the roundings)."""

    @staticmethod
    def forward(ctx, x, w, bias, rotate):
        k = x.shape[-1]
        xq, xr = _quantize(x.reshape(-1, k), rotate, keep=True)
        wq, wr = _quantize(w, rotate, keep=True)
        ctx.save_for_backward(xr, wr)
        ctx.rotate, ctx.shape = rotate, x.shape
        ctx.bias_type = None if bias is None else bias.dtype
        return _mm(xq, wq, _bias(bias, w.shape[0], x.device), x.dtype).reshape(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dy):
        xr, wr = ctx.saved_tensors
        dy = dy.reshape(-1, dy.shape[-1])
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = _mm(_quantize(dy)[0], _quantize_columns(wr), None, xr.dtype)
            dx = (_rotate(dx) if ctx.rotate else dx).reshape(ctx.shape)
        if ctx.needs_input_grad[1]:
            if dy.shape[0]:
                dw = _mm(_quantize_columns(dy), _quantize_columns(xr), None, wr.dtype)
                dw = _rotate(dw) if ctx.rotate else dw
            else:
                dw = torch.zeros_like(wr)
        if ctx.needs_input_grad[2]:
            db = dy.sum(dim=0, dtype=torch.float32).to(ctx.bias_type)
        return dx, dw, db, None


def mxfp4_linear(x, w, bias=None, *, rotate=True):
    """The MXFP4 linear with its gradients: ``x`` [.., K], ``w`` [N, K] (bf16, fp16, fp32), both
    quantised on every call; ``dx`` and ``dw`` are MXFP4 products too, ``dbias`` is a sum."""
    if w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x has {x.shape[-1]} columns and the weight is {tuple(w.shape)}")
    _type(x, "x")
    _type(w, "w")
    if x.device != w.device:
        raise ValueError(f"x is on {x.device} and the weight on {w.device}")
    _check_rotate(w.shape[1], rotate)
    return _Mxfp4LinearFn.apply(x, w, bias, rotate)


class Mxfp4Linear(torch.nn.Module):
    """``nn.Linear`` for serving with a prepared MXFP4 weight."""

    def __init__(self, w, bias=None, *, rotate=True):
        super().__init__()
        if not isinstance(w, MXFP4) or len(w.shape) != 2:
            raise TypeError("Mxfp4Linear takes the MXFP4 weight of prepare_weight_mxfp4")
        _check_rotate(w.shape[1], rotate)
        self.register_buffer("codes", w.codes)
        self.register_buffer("scales", w.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32))
        self.shape, self.rotate = w.shape, rotate

    @classmethod
    def from_linear(cls, mod, *, rotate=True):
        return cls(prepare_weight_mxfp4(mod.weight, rotate), getattr(mod, "bias", None), rotate=rotate)

    def forward(self, x):
        return linear_mxfp4(x, MXFP4(self.codes, self.scales, self.shape), self.bias, rotate=self.rotate)

    def extra_repr(self):
        return f"in_features={self.shape[1]}, out_features={self.shape[0]}, bias={self.bias is not None}"


class TrainableMxfp4Linear(torch.nn.Module):
    """A linear whose parameter stays in its own type and is quantised to MXFP4 on every call."""

    def __init__(self, weight, bias=None, *, rotate=True):
        super().__init__()
        if weight.dtype not in _TYPES or weight.dim() != 2:
            raise TypeError(f"the weight must be a bfloat16, float16 or float32 [N, K], got {weight.dtype} "
                            f"{tuple(weight.shape)}")
        _check_rotate(weight.shape[1], rotate)
        self.weight = torch.nn.Parameter(weight.detach())
        self.bias = None if bias is None else torch.nn.Parameter(bias.detach())
        self.rotate = rotate

    @classmethod
    def from_linear(cls, mod, *, rotate=True):
        return cls(mod.weight, getattr(mod, "bias", None), rotate=rotate)

    def forward(self, x):
        return mxfp4_linear(x, self.weight, self.bias, rotate=self.rotate)

    def extra_repr(self):
        return f"{tuple(self.weight.shape)}, bias={self.bias is not None}"
