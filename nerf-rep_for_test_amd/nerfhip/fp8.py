"""8-bit block-scaled products (csrc/fp8_ops.hip): e4m3 values with one
power-of-two scale for 1 x 128 of the activations and 128 x 128 of the weights.

``linear`` is ``nerf_linear_fm``'s kind of layer (y = x W^T + bias, ReLU) for
row-major activations in 32 or 16 bits and weights that were rounded to 8 bits
once (``quantize_weight``). It is an inference operator: activations are rounded
inside of it and it has no gradient.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from ._lib import NerfHipError, enqueue, ptr

BLOCK = 128
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # NERF_F32 ..


class _Fp8Linear(ctypes.Structure):
    """NerfFp8Linear (include/nerfhip.h)."""
    _fields_ = [("x", ctypes.c_void_p), ("ldx", ctypes.c_int64), ("x_rows", ctypes.c_int64),
                ("order", ctypes.c_void_p), ("x_type", ctypes.c_int), ("out_type", ctypes.c_int),
                ("slots", ctypes.c_int), ("E", ctypes.c_int), ("relu", ctypes.c_int),
                ("M", ctypes.c_int64), ("N", ctypes.c_int64), ("K", ctypes.c_int64),
                ("wq", ctypes.c_void_p), ("ws", ctypes.c_void_p), ("offsets", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("out", ctypes.c_void_p), ("ldo", ctypes.c_int64)]


def _blocks(n):
    return -(-n // BLOCK)


class Fp8Weight:
    """Weights in 8 bits: ``q`` float8_e4m3fn [N, Kp] or [E, N, Kp] with Kp = ``k``
    rounded up to 128 (zeros behind ``k``), ``scale`` [.., ceil(N / 128), Kp / 128] as
    E8M0 bytes (uint8 or float8_e8m0fnu: byte b stands for 2^(b - 127))."""

    __slots__ = ("q", "scale", "k")

    def __init__(self, q, scale, k):
        k = int(k)
        if q.dtype != torch.float8_e4m3fn or q.dim() not in (2, 3):
            raise ValueError("Fp8Weight: q must be float8_e4m3fn [N, Kp] or [E, N, Kp]")
        if k < 1 or q.numel() == 0 or q.shape[-1] != _blocks(k) * BLOCK:
            raise ValueError(f"Fp8Weight: q's rows must be k = {k} rounded up to {BLOCK} values long")
        if scale.dtype not in (torch.uint8, torch.float8_e8m0fnu):
            raise ValueError("Fp8Weight: scale must hold E8M0 bytes (uint8 or float8_e8m0fnu)")
        want = (*q.shape[:-2], _blocks(q.shape[-2]), q.shape[-1] // BLOCK)
        if tuple(scale.shape) != want:
            raise ValueError(f"Fp8Weight: scale must be {list(want)}, got {list(scale.shape)}")
        if not q.is_contiguous() or not scale.is_contiguous() or q.device != scale.device:
            raise ValueError("Fp8Weight: q and scale must be contiguous, on one device")
        self.q, self.scale, self.k = q, scale, k

    @property
    def shape(self):
        return (*self.q.shape[:-1], self.k)

    def dequantize(self):
        """The float32 values that the 8 bits stand for."""
        s = self.scale.view(torch.uint8).int() - 127
        s = s.repeat_interleave(BLOCK, -2)[..., :self.q.shape[-2], :].repeat_interleave(BLOCK, -1)
        w = torch.ldexp(self.q.float(), s)
        return torch.where(s == 128, torch.full_like(w, float("nan")), w)[..., :self.k]


def quantize_weight(w):
    """Weights [N, K] or a stack [E, N, K] (float32, bfloat16 or float16) as ``Fp8Weight``."""
    if w.dim() not in (2, 3) or w.dtype not in TYPES or w.numel() == 0:
        raise ValueError("quantize_weight: weights must be [N, K] or [E, N, K] float32, bfloat16 or float16")
    _lib.require_gpu(w)
    w = w.detach()
    if w.stride(-1) != 1:
        w = w.contiguous()
    E, (N, K) = (w.shape[0] if w.dim() == 3 else 1), w.shape[-2:]
    q = torch.empty((*w.shape[:-1], _blocks(K) * BLOCK), device=w.device, dtype=torch.float8_e4m3fn)
    scale = torch.empty((*w.shape[:-2], _blocks(N), _blocks(K)), device=w.device, dtype=torch.uint8)
    enqueue("nerf_fp8_quantize_weight", w, ptr(w), TYPES[w.dtype], w.stride(0) if w.dim() == 3 else 0, w.stride(-2),
            E, N, K, ptr(q), ptr(scale))
    return Fp8Weight(q, scale, K)


def refuse_dual(who, *tensors):
    """The kernels would drop a dual number's tangent."""
    for t in tensors:
        if t is not None and unpack_dual(t).tangent is not None:
            raise NerfHipError(f"{who} has no forward-mode derivative: unpack its dual inputs first")


def launch(x, weight, M, order, slots, offsets, bias, relu, out_dtype, who):
    """The checked launch that ``linear`` and ``experts.expert_linear`` share: x [rows, K] ->
    [M, N]."""
    if x.dtype not in TYPES or x.dim() != 2:
        raise ValueError(f"{who}: activations must be float32, bfloat16 or float16")
    K, N = weight.k, weight.q.shape[-2]
    if x.shape[1] != K:
        raise ValueError(f"{who}: activations have {x.shape[1]} columns, the weights {K}")
    refuse_dual(who, x, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise NerfHipError(f"{who} has no gradient: detach its inputs or run it under torch.no_grad()")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in TYPES:
        raise ValueError(f"{who}: out_dtype must be float32, bfloat16 or float16")
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != tuple(weight.q.shape[:-1]):
            raise ValueError(f"{who}: bias must be float32 {list(weight.q.shape[:-1])}")
        bias = bias.contiguous()
    for t in (weight.q, bias, order, offsets):
        if t is not None and t.device != x.device:
            raise ValueError(f"{who}: all tensors must be on {x.device}")
    _lib.require_gpu(x)
    if x.stride(1) != 1 and K > 1 or x.stride(0) < 0:
        x = x.contiguous()
    out = torch.empty((M, N), device=x.device, dtype=out_dtype)
    if M == 0:
        return out
    E = weight.q.shape[0] if weight.q.dim() == 3 else 1
    d = _Fp8Linear(ptr(x), x.stride(0), x.shape[0], ptr(order), TYPES[x.dtype], TYPES[out_dtype], slots, E,
                   int(relu), M, N, K, ptr(weight.q), ptr(weight.scale), ptr(offsets), ptr(bias), ptr(out), N)
    need = _lib.lib().nerf_fp8_linear_workspace(M, N, K, E, int(offsets is not None))
    ws = torch.empty((need,), device=x.device, dtype=torch.uint8) if need else None
    enqueue("nerf_fp8_linear", x, ctypes.addressof(d), ptr(ws), need)
    return out


def linear(x, weight, bias=None, relu=False, out_dtype=None):
    """y [.., N] = x [.., K] W^T (+ bias [N] float32, ReLU) with the activations rounded to
    8-bit blocks of 128; sums in float32, y in ``out_dtype`` (default: x's type). float32 results have
    exact products, 16-bit ones the 8-bit matrix instruction's: 8 neighbouring products are added with 13 bits
    below the largest, 1e-5 of a result's norm for values of usual spread and 7 * 2^-13 of the largest product at
    most (1.75 half steps of float16, less than bfloat16's; ``out_dtype=torch.float32`` has none of it). A block with a value that is not finite makes its row's outputs NaN. K up to 2^23."""
    if not isinstance(weight, Fp8Weight) or weight.q.dim() != 2:
        raise ValueError("linear: weight must be an Fp8Weight of one matrix")
    if weight.k > 1 << 23:
        raise ValueError("linear: K up to 2^23")
    if x.dim() < 1 or x.shape[-1] != weight.k:
        raise ValueError(f"linear: activations must be [.., {weight.k}]")
    flat = x.reshape(-1, x.shape[-1])
    y = launch(flat, weight, flat.shape[0], None, 1, None, bias, relu, out_dtype, "linear")
    return y.view(*x.shape[:-1], y.shape[1])
