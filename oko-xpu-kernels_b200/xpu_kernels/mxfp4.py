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

import ctypes

import torch

from .int8._lib import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_native = None


def _load():
    """The torch binding over the loaded library (csrc/binding.cpp)."""
    global _native
    lib = _lib()
    try:
        from . import _native as module
    except ImportError as exc:
        raise RuntimeError(f"the torch binding is not usable ({exc}); build it with `make -C oko-xpu-kernels_b200/csrc` "
                           "or __graft_entry__.build()") from exc
    module.bind({name: ctypes.cast(getattr(lib, "xpuint8_" + name), ctypes.c_void_p).value for name in module.names()})
    _native = module
    return module


def _type(x, what):
    """x's type for the C entries; raises where there is none or x is not on a GPU."""
    t = _TYPES.get(x.dtype)
    if t is None:
        raise TypeError(f"{what} must be bfloat16, float16 or float32, got {x.dtype}")
    if not x.is_cuda:
        raise TypeError(f"{what} must be a CUDA tensor, got {x.device}")
    return t


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

    __slots__ = ("shape", "_codes", "_scales", "_buffer", "_at")

    def __init__(self, codes, scales, shape):
        if len(shape) == 2:
            r, k = shape
            want_codes, want_scales = (r, (k + 31) // 32 * 16), ((r + 127) // 128, (k + 127) // 128, 32, 16)
        elif len(shape) == 3:
            n, r, k = shape
            want_codes = (n, r, (k + 31) // 32 * 16)
            want_scales = (n, (r + 127) // 128, (k + 127) // 128, 32, 16)
        else:
            raise ValueError(f"an MXFP4 matrix has the shape [R, K] or [E, R, K], got {tuple(shape)}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
        if codes.shape != want_codes or scales.shape != want_scales:
            raise ValueError(f"an MXFP4 matrix {tuple(shape)} has codes {want_codes} and scales {want_scales}, "
                             f"got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.get_device() != scales.get_device():
            raise ValueError(f"codes are on {codes.device} and scales on {scales.device}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        self.shape = tuple(shape)
        self._codes, self._scales, self._buffer, self._at = codes, scales, None, 0

    @classmethod
    def _of(cls, buffer, shape):
        """The matrix whose codes and then scales are in `buffer`; they become tensors when asked for."""
        r, k = shape[-2:]
        n = shape[0] if len(shape) == 3 else 1
        q = cls.__new__(cls)
        q.shape, q._buffer, q._codes, q._scales = tuple(shape), buffer, None, None
        q._at = (n * r * ((k + 31) // 32 * 16) + 255) // 256 * 256
        return q

    # What the binding takes: the codes and the scales, or, before either became a tensor, the buffer and
    # where its scales begin.  Addresses are taken at the call alone.
    @property
    def _held(self):
        if self._codes is None and self._scales is None:
            return self._buffer, self._at
        return self.codes, self.scales

    @property
    def _index(self):
        return self._held[0].get_device()

    @property
    def codes(self):
        if self._codes is None:
            *lead, r, k = self.shape
            row = (k + 31) // 32 * 16
            self._codes = self._buffer[:(lead[0] if lead else 1) * r * row].view(*lead, r, row)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            *lead, r, k = self.shape
            self._scales = self._buffer[self._at:].view(*lead, (r + 127) // 128, (k + 127) // 128, 32, 16)
        return self._scales

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return f"MXFP4({self.shape}, device={self.device})"


def quantize_mxfp4(x, *, rotate=False, transpose=False):
    """``x`` [R, K] or a stack [E, R, K] (bf16, fp16, fp32; any K) -> :class:`MXFP4` along K.

    ``rotate`` puts the group-256 rotation in front (K a multiple of 256), its result rounded to x's
    type.  ``transpose`` gives the MXFP4 of ``x``'s transpose instead, blocks along R.
    """
    shape = x.shape
    if len(shape) not in (2, 3):
        raise ValueError(f"x must be [R, K] or [E, R, K], got {tuple(shape)}")
    if transpose and rotate:
        raise ValueError("rotate goes along K: transpose quantises along the other axis")
    if rotate and shape[-1] % 256:
        _check_rotate(shape[-1], rotate)
    _type(x, "x")
    buffer = (_native or _load()).quantize(x.detach() if x.requires_grad else x, rotate, transpose)
    return MXFP4._of(buffer, (*shape[:-2], shape[-1], shape[-2]) if transpose else shape)


def dequantize_mxfp4(q, dtype=torch.bfloat16):
    """The values that ``q`` stands for (rotated ones where it was quantised with ``rotate``)."""
    t = _TYPES.get(dtype)
    if t is None:
        raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    if q._index < 0:
        raise TypeError(f"q must be on a CUDA device, got {q.device}")
    return (_native or _load()).dequantize(*q._held, t, q.shape)


def prepare_weight_mxfp4(w, rotate=True):
    """A weight [N, K] (or the experts' [E, N, K]) for :func:`linear_mxfp4`: rotated and quantised."""
    return quantize_mxfp4(w.detach(), rotate=rotate)


def _check_bias(bias, n):
    if bias is not None and bias.numel() != n:
        raise ValueError(f"bias has {bias.numel()} values; expected N={n}")


def mxfp4_mm(a, b, bias=None, dtype=torch.bfloat16):
    """``a @ b.T (+ bias)`` of two MXFP4 matrices [M, K] and [N, K]: summed in 32 bits, rounded once."""
    if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"mxfp4_mm takes [M, K] and [N, K], got {a.shape} and {b.shape}")
    (m, k), n = a.shape, b.shape[0]
    if k == 0:
        raise ValueError("mxfp4_mm needs K of at least 1")
    t = _TYPES.get(dtype)
    if t is None:
        raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    index = a._index
    if index != b._index:
        raise ValueError(f"a is on {a.device} and b on {b.device}")
    if index < 0:
        raise TypeError(f"a and b must be on a CUDA device, got {a.device}")
    _check_bias(bias, n)
    return (_native or _load()).mm(*a._held, *b._held, bias, t, m, n, k)


def linear_mxfp4(x, w, bias=None, *, rotate=True):
    """The MXFP4 linear: ``x`` [.., K] (bf16, fp16, fp32) -> [.., N] of x's type.

    ``w`` is the :class:`MXFP4` weight [N, K] of :func:`prepare_weight_mxfp4`, ``rotate`` what it was
    prepared with.  ``bias`` is added in 32 bits before the one rounding.  For serving: a backward pass
    that reaches the result raises (:func:`mxfp4_linear` has gradients).
    """
    shape = x.shape
    if len(w.shape) != 2 or shape[-1] != w.shape[1]:
        raise ValueError(f"x has {shape[-1]} columns and the weight is {w.shape}")
    codes, scales = w._held
    if x.get_device() != codes.get_device():
        raise ValueError(f"x is on {x.device} and the weight on {w.device}")
    n, k = w.shape
    if rotate and k % 256:
        _check_rotate(k, rotate)
    _type(x, "x")
    if bias is not None:
        _check_bias(bias, n)
    return (_native or _load()).linear(x, codes, scales, n, bias, rotate)


def mxfp4_linear(x, w, bias=None, *, rotate=True):
    """The MXFP4 linear with its gradients: ``x`` [.., K], ``w`` [N, K] (bf16, fp16, fp32), both
    quantised on every call; ``dx`` and ``dw`` are MXFP4 products too, ``dbias`` is a sum.

    y = Q(x) Q(w)^T with both operands quantised along K.  The gradients' products quantise their
    operands along their own contractions, dy and w along N for dx, dy and x along the rows for dw
    (straight through the roundings).  What is kept between the two is in 4 bits: x and w along those
    axes, where their gradient is wanted.
    """
    if w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x has {x.shape[-1]} columns and the weight is {tuple(w.shape)}")
    _type(x, "x")
    _type(w, "w")
    if x.get_device() != w.get_device():
        raise ValueError(f"x is on {x.device} and the weight on {w.device}")
    if w.shape[1] == 0:
        raise ValueError("mxfp4_linear needs K of at least 1")
    _check_rotate(w.shape[1], rotate)
    _check_bias(bias, w.shape[0])
    return (_native or _load()).train(x, w, bias, rotate)


class Mxfp4Linear(torch.nn.Module):
    """``nn.Linear`` for serving with a prepared MXFP4 weight (:func:`linear_mxfp4`: no gradients)."""

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
