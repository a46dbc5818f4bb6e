"""Orthogonalised matrices by Newton-Schulz products and the optimizer step built on them (``csrc/newton_schulz_sm100.cu``).

The contract of the calls is at :func:`kareus_b200.kernels.orthogonalize` and :func:`kareus_b200.kernels.muon_step`."""
from __future__ import annotations

import functools
import math

import torch

import kareus_b200.kernels as _entry

from . import ref
from .cuda import KernelError, _check, _count, _no_recording, _stream, lib, require_current_device, status_word

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@functools.lru_cache(maxsize=64)
def fp16_scales(steps: int, coefficients: tuple) -> tuple:
    """Powers of two under which what the steps hold in fp16 fits: one (at most 2^14) for X, G = X Xt and P = b G + c G G, one for
    products of up to three consecutive a I + P.  Entries are at most the largest singular value; those of X start at 1 or below, and
    the range that a step can reach is sampled."""
    a, b, c = coefficients
    bound, worst, worst_q = 1.0, 1.0, 1.0
    for k in range(steps):
        s = torch.linspace(0.0, bound * 1.01, 8193, dtype=torch.float64, device="cpu")       # 1 %: what rounding adds
        t, prod = s * s, 1.0
        for j in range(min(3, steps - k)):
            q = a + b * t + c * t * t
            if j == 0:
                worst = max(worst, t.max().item(), (q - a).abs().max().item())
                bound = (s * q).abs().max().item()
                worst = max(worst, bound)
            prod = prod * q
            t = t * q * q
            worst_q = max(worst_q, prod.abs().max().item())
        if not worst < 1e3 or not worst_q < 3e4:
            raise KernelError(f"Newton-Schulz coefficients {coefficients} let the iterates grow without bound")
    return tuple(2.0 ** min(14, math.floor(math.log2(65000.0 / w))) for w in (worst, worst_q))


def _parameters(steps, coefficients, eps):
    steps, coefficients, eps = int(steps), tuple(float(v) for v in coefficients), float(eps)
    # squares are summed in fp32: of entries below 1e-19, whose squares it does not hold, the norm counts for nothing beside such an eps
    if steps < 1 or len(coefficients) != 3 or not all(math.isfinite(v) for v in coefficients) or not 1e-12 <= eps < math.inf:
        raise KernelError(f"Newton-Schulz: at least one step, three finite coefficients and a finite eps >= 1e-12, got {steps}, "
                          f"{coefficients}, {eps}")
    return steps, coefficients, eps


def _workspace(batch, m, n, device):
    size = lib().kb_newton_schulz_bytes(batch, m, n)
    if size < 0:
        raise KernelError(f"Newton-Schulz: {batch} matrices of {m} x {n} are too many or too large")
    return torch.empty(size, dtype=torch.uint8, device=device)


def orthogonalize(x, steps, coefficients, eps):
    steps, coefficients, eps = _parameters(steps, coefficients, eps)
    if _entry._OPS is not None and x.is_cuda:
        r = _entry._OPS.orthogonalize(x, *coefficients, steps, eps, *fp16_scales(steps, coefficients))
        if r is not None:
            return r
    if x.dim() < 2 or not x.is_floating_point():
        raise KernelError(f"orthogonalize takes matrices of floating-point numbers, got {x.dtype} of shape {tuple(x.shape)}")
    if not (x.is_cuda and x.dtype in (torch.bfloat16, torch.float32)):
        return ref.orthogonalize(x, steps, coefficients, eps)
    require_current_device("orthogonalize", x)
    scales = fp16_scales(steps, coefficients)
    status_word(x.device)                     # the native call takes over from the next one on
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    if not x.numel():
        return out
    if not x.is_contiguous():
        _no_recording("making the matrices of a Newton-Schulz iteration contiguous")
        x = x.contiguous()
    m, n = x.shape[-2:]
    batch = x.numel() // (m * n)
    work = _workspace(batch, m, n, x.device)
    _check(lib().kb_newton_schulz(x.data_ptr(), 1 if x.dtype == torch.bfloat16 else 0, batch, m, n, *coefficients, steps, eps, *scales,
                                  out.data_ptr(), work.data_ptr(), status_word(x.device).data_ptr(), _stream()),
           f"orthogonalize {batch} x {m} x {n}")
    _count(lib().kb_newton_schulz_launches(batch, m, n, steps))
    return out


def muon_step(p, g, m, master, lr, momentum, weight_decay, scale, nesterov, steps, coefficients, eps, grad_scale_tensor):
    steps, coefficients, eps = _parameters(steps, coefficients, eps)
    if g.dim() != 2 or any(t.shape != g.shape for t in (p, m, master)):
        raise KernelError("muon_step takes one matrix: weight, gradient, momentum and master of one shape, got "
                          + ", ".join(str(tuple(t.shape)) for t in (p, g, m, master)))
    if any(t.device != g.device for t in (p, m, master)):
        raise KernelError(f"muon_step: tensors on several devices: {[str(t.device) for t in (p, g, m, master)]}")
    if scale is None:
        scale = 0.2 * math.sqrt(max(g.shape))
    if not (g.is_cuda and p.dtype == torch.bfloat16):
        gs = 1.0 if grad_scale_tensor is None else grad_scale_tensor.to(g.dtype)
        return ref.muon_step(p, g, m, master, lr, momentum, weight_decay, scale, nesterov, steps, coefficients, eps, gs)
    require_current_device("muon_step", g)
    if any(t.dtype != torch.float32 for t in (g, m, master)) or not all(t.is_contiguous() for t in (p, g, m, master)):
        raise KernelError("muon_step: gradient, momentum and master have to be fp32, all tensors contiguous")
    if grad_scale_tensor is not None and (grad_scale_tensor.dtype != torch.float32 or grad_scale_tensor.numel() != 1
                                          or grad_scale_tensor.device != g.device):
        raise KernelError("muon_step: the gradient's factor is one fp32 value on the gradient's device")
    o = torch.empty(g.shape, dtype=torch.bfloat16, device=g.device)
    if not g.numel():
        return o
    rows, cols = g.shape
    work = _workspace(1, rows, cols, g.device)
    _check(lib().kb_muon_step(g.data_ptr(), m.data_ptr(), master.data_ptr(), p.data_ptr(), o.data_ptr(), rows, cols, float(momentum),
                              1 if nesterov else 0, 1.0 - lr * weight_decay, lr * scale,
                              0 if grad_scale_tensor is None else grad_scale_tensor.data_ptr(), *coefficients, steps, eps,
                              *fp16_scales(steps, coefficients), work.data_ptr(), status_word(g.device).data_ptr(), _stream()),
           f"muon_step {rows} x {cols}")
    fused = lib().kb_muon_fuses(master.data_ptr(), p.data_ptr(), cols)
    _count(lib().kb_newton_schulz_launches(1, rows, cols, steps) + (0 if fused else 1))
    return o
