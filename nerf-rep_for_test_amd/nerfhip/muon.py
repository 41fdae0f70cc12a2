"""Muon: matrices' updates orthogonalised by Newton-Schulz products
(csrc/muon_ops.hip), beside nerfhip.adam's Adam.

``orthogonalize`` is the operator alone, ``muon_update`` one step of momentum,
orthogonalisation, weight decay and step for a list of matrices (17 launches for
all of them, at most 32 a set), ``HipMuon`` the optimizer that
the trainer takes: matrices of hidden layers by Muon, everything else by Adam.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import enqueue, ptr
from .adam import HipAdam
from .fp8 import TYPES

STEPS, EPS = 5, 1e-7


class _Group(ctypes.Structure):
    """NerfMuonGroup (include/nerfhip.h)."""
    _fields_ = [("out", ctypes.c_void_p), ("g", ctypes.c_void_p), ("momentum", ctypes.c_void_p),
                ("m", ctypes.c_int64), ("n", ctypes.c_int64), ("count", ctypes.c_int64),
                ("out_stride", ctypes.c_int64), ("g_stride", ctypes.c_int64)]


class _Options(ctypes.Structure):
    """NerfMuonOptions (include/nerfhip.h)."""
    _fields_ = [("type", ctypes.c_int), ("update", ctypes.c_int), ("nesterov", ctypes.c_int),
                ("steps", ctypes.c_int), ("lr", ctypes.c_float), ("momentum", ctypes.c_float),
                ("weight_decay", ctypes.c_float), ("eps", ctypes.c_float), ("clip", ctypes.c_float),
                ("lr_device", ctypes.c_void_p)]


def _run(groups, options, like):
    arr = (_Group * len(groups))(*groups)
    need = _lib.lib().nerf_muon_workspace(ctypes.addressof(arr), len(groups))
    ws = torch.empty((need,), device=like.device, dtype=torch.uint8)
    enqueue("nerf_muon", like, ctypes.addressof(arr), len(groups), ctypes.addressof(options), ptr(ws), need)


def _check_steps(steps):
    if int(steps) != steps or not 1 <= steps <= 100:
        raise ValueError("muon: steps must be a whole number from 1 to 100")
    return int(steps)


def _is_eps(eps):
    """Positive and finite as the 32-bit number that the kernels take."""
    return 0.0 < ctypes.c_float(eps).value < float("inf")


@torch.no_grad()
def orthogonalize(g, steps=STEPS, eps=EPS):
    """Newton-Schulz orthogonalisation of a matrix [m, n] or a stack [.., m, n] (float32, bfloat16, float16;
    result in the same type): X = g / (|g| + eps), then ``steps`` times X = a X + (b A + c A A) X with
    A = X X^T, (a, b, c) = (3.4445, -4.7750, 2.0315); singular values end near 1 where |g| is not far below eps.
    Sums, norms and products hold float32 accuracy whatever the type and |g|. A matrix with a value that is not finite becomes NaN. No gradient."""
    if g.dim() < 2 or g.dtype not in TYPES:
        raise ValueError("orthogonalize: g must be [.., m, n] float32, bfloat16 or float16")
    steps = _check_steps(steps)
    if not _is_eps(eps):
        raise ValueError("orthogonalize: eps must be a positive 32-bit number")
    m, n = g.shape[-2:]
    if max(m, n) > 1 << 20:
        raise ValueError("orthogonalize: sides up to 2^20")
    _lib.require_gpu(g)
    g = g.contiguous()
    out = torch.empty_like(g)
    if out.numel() == 0:
        return out
    o = _Options(TYPES[g.dtype], 0, 0, steps, 0.0, 0.0, 0.0, float(eps), -1.0, None)
    _run([_Group(ptr(out), ptr(g), None, m, n, out.numel() // (m * n), m * n, m * n)], o, g)
    return out


def _float32_matrix(t, shape, what):
    if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise ValueError(f"muon_update: {what} must be contiguous float32 matrices of their parameter's shape")


def _refuse_shared(spans):
    """Memory (start, end, whether it is written): what is written may not be another's, too."""
    spans.sort()
    if all(a[1] <= b[0] for a, b in zip(spans, spans[1:])):
        return
    any_end = written_end = 0
    for start, end, write in spans:
        if start < (any_end if write else written_end):
            raise ValueError("muon_update: a matrix or momentum shares memory with another one or with a gradient")
        any_end = max(any_end, end)
        if write:
            written_end = max(written_end, end)


@torch.no_grad()
def muon_update(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=STEPS, eps=EPS,
                clip=None):
    """One Muon step for a list of matrices, in place (params and momenta):
    buf = momentum * buf + g; u = g + momentum * buf (``nesterov``; else buf);
    p = p * (1 - lr * weight_decay) - lr * sqrt(max(1, m / n)) * orthogonalize(u).
    ``lr``: a number, or one float32 on the device (then the step can be captured and replayed with another
    one). ``clip``: gradients clamped to [-clip, clip] on their way in (the gradients themselves stay). No two
    of params and momenta may share memory, nor a gradient with them."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError("muon_update: params, grads and momenta must be lists of one length")
    steps = _check_steps(steps)
    if not 0.0 <= momentum < 1.0 or not _is_eps(eps) or not 0.0 <= weight_decay < float("inf"):
        raise ValueError("muon_update: momentum must be in [0, 1), eps positive, weight_decay >= 0")
    if clip is not None and not clip >= 0:
        raise ValueError("muon_update: clip must be None or >= 0")
    spans, groups = [], []
    for p, g, b in zip(params, grads, momenta):
        _float32_matrix(p, None, "params")
        _float32_matrix(g, p.shape, "grads")
        _float32_matrix(b, p.shape, "momenta")
        if p.device != params[0].device or g.device != p.device or b.device != p.device:
            raise ValueError("muon_update: all tensors must be on one device")
        if max(p.shape) > 1 << 20:
            raise ValueError("muon_update: sides up to 2^20")
        if p.numel() == 0:
            continue
        size, at_p, at_g, at_b = 4 * p.numel(), ptr(p), ptr(g), ptr(b)
        spans += (at_p, at_p + size, True), (at_b, at_b + size, True), (at_g, at_g + size, False)
        groups.append(_Group(at_p, at_g, at_b, *p.shape, 1, 0, 0))
    _refuse_shared(spans)
    dev_lr = torch.is_tensor(lr)
    if dev_lr and (lr.dtype != torch.float32 or lr.numel() != 1 or (params and lr.device != params[0].device)):
        raise ValueError("muon_update: a tensor lr must be one float32 on the parameters' device")
    if not groups:
        return
    _lib.require_gpu(params[0])
    o = _Options(0, 1, int(bool(nesterov)), steps, 0.0 if dev_lr else float(lr), float(momentum), float(weight_decay),
                 float(eps), -1.0 if clip is None else float(clip), ptr(lr) if dev_lr else None)
    _run(groups, o, params[0])
    _lib.written(*params, *momenta)


def is_hidden_matrix(p):
    """What HipMuon orthogonalises: matrices with 16 rows and columns at least (a network's hidden
    layers; its density and colour heads have 1 and 3 rows)."""
    return p.dim() == 2 and min(p.shape) >= 16


class HipMuon(torch.optim.Optimizer):
    """Muon for the matrices that ``is_hidden_matrix`` names, HipAdam (same ``lr``, ``betas``, ``adam_eps``)
    for every other parameter; gradients clamped to [-``clip``, clip] on their way in (None: not). Matrices
    move by ``lr * muon_ratio`` times an orthogonal matrix: with Adam's usual 5e-4 and the ratio 40 by 0.02.
    ``weight_decay`` is theirs alone.

    Group 0 holds the matrices (state: ``momentum_buffer``), group 1 the rest (HipAdam's state). lr is a
    device tensor in both (fill it to change it; the step then stays one captured graph). float32 contiguous
    parameters on one ROCm device; every parameter needs a gradient at every step, as with HipAdam."""

    def __init__(self, params, lr=5e-4, muon_ratio=40.0, momentum=0.95, nesterov=True, weight_decay=0.0, steps=STEPS,
                 betas=(0.9, 0.999), adam_eps=1e-8, clip=None):
        params = list(params)
        if any(isinstance(p, dict) for p in params):
            raise ValueError("HipMuon takes parameters, not groups: it makes its own two")
        matrices = [p for p in params if is_hidden_matrix(p)]
        rest = [p for p in params if not is_hidden_matrix(p)]
        if not matrices:
            raise ValueError("HipMuon: no matrix with 16 rows and columns among the parameters")
        if not muon_ratio > 0:
            raise ValueError("HipMuon: muon_ratio must be positive")
        if clip is not None and not clip >= 0:
            raise ValueError("HipMuon: clip must be None (no clipping) or >= 0")
        dev = matrices[0].device
        if dev.type != "cuda":
            raise _lib.NerfHipError("HipMuon needs a ROCm GPU device (no CPU fallback)")
        self.adam = HipAdam(rest, lr=lr, betas=betas, eps=adam_eps, clip=clip) if rest else None
        self.muon_ratio, self.clip = float(muon_ratio), clip
        self._lr = torch.zeros((), device=dev, dtype=torch.float32)
        super().__init__([{"params": matrices}],
                         dict(lr=torch.tensor(lr, device=dev, dtype=torch.float32), momentum=float(momentum),
                              nesterov=bool(nesterov), weight_decay=float(weight_decay), steps=_check_steps(steps)))
        if self.adam is not None:
            self.param_groups.append(self.adam.param_groups[0])
            self._share()

    def _share(self):
        """One state and one group object for both optimizers."""
        if self.adam is not None:
            self.adam.state = self.state
            self.adam.param_groups = [self.param_groups[1]]

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        self._share()

    @torch.no_grad()
    def step(self, closure=None):
        if closure is not None:
            raise ValueError("HipMuon.step takes no closure")
        if len(self.param_groups) != (1 if self.adam is None else 2):
            raise ValueError("HipMuon keeps its own two parameter groups: none can be added")
        g = self.param_groups[0]
        missing = [p for h in self.param_groups for p in h["params"] if p.grad is None]
        every = sum(len(h["params"]) for h in self.param_groups)
        if missing:
            if len(missing) == every:
                return None
            raise ValueError(f"HipMuon: {len(missing)} of {every} parameters have no gradient")
        lr = g["lr"]
        if not torch.is_tensor(lr) or lr.device != self._lr.device or lr.dtype != torch.float32:
            # a float set by someone else, or a tensor of a state dict loaded to another device
            lr = g["lr"] = torch.tensor(float(lr), device=self._lr.device, dtype=torch.float32)
        buffers = []
        for p in g["params"]:
            st = self.state[p]
            if "momentum_buffer" not in st:
                st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            buffers.append(st["momentum_buffer"])
        torch.mul(lr, self.muon_ratio, out=self._lr)
        muon_update(g["params"], [p.grad for p in g["params"]], buffers, self._lr, momentum=g["momentum"],
                    nesterov=g["nesterov"], weight_decay=g["weight_decay"], steps=g["steps"], clip=self.clip)
        if self.adam is not None:
            self.adam.step()
        return None
