"""Weight updates by orthogonalised momentum, for the primitives' layers and the feature decoder's.

The step that follows primitive_gemm.grouped_weight_gradients: the gradient's running mean is taken to the nearest matrix with
singular values of about one by a Newton-Schulz iteration, matrix by matrix, and subtracted from the weights.  The rule and its coefficients are
those of K. Jordan and others, "Muon: An optimizer for hidden layers in neural networks" (2024).  Works on stacks of
matrices ([N, 32, 72], [N, 32, 32] and [N, 4, 32] of a scene) and on single ones; biases and other vectors are left to the caller's
own rule.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd.graph import increment_version

from . import _lib as L
from .engine import _on, _refuse_tangents, _stream_ptr

COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # (a, b, c): five steps take singular values from 0.01 .. 1 to 0.7 .. 1.2
_TYPES = {torch.float32: L.PRECISION_F32, torch.float16: L.PRECISION_F16, torch.bfloat16: L.PRECISION_BF16}


def _shape(name, t):
    """(matrices, rows, columns) of a matrix or a stack."""
    if t.ndim not in (2, 3):
        raise ValueError(f"{name} must be a matrix [rows, columns] or a stack of them [N, rows, columns], got {tuple(t.shape)}")
    n, rows, cols = (1, *t.shape) if t.ndim == 2 else t.shape
    if rows < 1 or cols < 1 or min(rows, cols) > L.MUON_MAX_SMALL or max(rows, cols) > L.MUON_MAX_LARGE:
        raise ValueError(f"{name}: matrices may have 1..{L.MUON_MAX_SMALL} rows or columns on the shorter side and at most "
                         f"{L.MUON_MAX_LARGE} on the longer, got {tuple(t.shape)}")
    return int(n), int(rows), int(cols)


def _check_tensors(tensors):
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda or not t.is_contiguous() or t.device != dev:
            raise ValueError("all inputs must be contiguous tensors on one CUDA device")
    return dev


def _answer(shapes, check):
    """A word for the answer of kernels that wait on the device, or None."""
    if not check or not any(L.load().mlpsp_orthogonalize_stack_waits(*shape) for shape in shapes):
        return None
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("matrices of these sizes and this number wait for the kernel's answer: pass check=False inside a graph capture")
    return C.c_int32(0)


def _read(answer, what):
    if answer is not None and answer.value:
        raise RuntimeError(f"{what}: a device-side wait gave up; results are invalid")


def _written(rc, what, tensors):
    """In-place writes count as such: scenes packed from the old weights are packed anew, autograd sees saved tensors change.  Also those of the
    launches before one that failed, if the library's call did (rc)."""
    if rc in (0, L.E_CUDA):
        increment_version([t for t in tensors if not t.is_inference()])
    L.check(rc, what)


def _coefficients(coefficients, steps, eps):
    if not isinstance(steps, int) or isinstance(steps, bool) or not 1 <= steps <= 32:
        raise ValueError("steps must be an integer from 1 to 32")
    if not 1e-15 <= float(eps) <= 1.0:
        raise ValueError("eps must be within [1e-15, 1]")
    a, b, c = (float(v) for v in coefficients)
    return steps, a, b, c, float(eps)


@torch.no_grad()
def orthogonalize(update: torch.Tensor, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7, out: torch.Tensor | None = None,
                  check: bool = True) -> torch.Tensor:
    """Newton-Schulz iteration of a matrix or of every matrix of a stack: X = U / max(|U|_F, eps), then `steps` times
    X <- a X + (b A + c A^2) X with A = X X^T.

    update: float32, float16 or bfloat16, [rows, columns] or [N, rows, columns], contiguous; out (update itself, or a tensor
    apart from it) receives the result in update's type.  The iteration has FP32 accuracy whatever the type.  A matrix of zeros stays
    zero; one that holds an infinity or a NaN becomes NaN and touches no other.  Coefficients under which singular values leave
    [0, 4] are refused.  There is no gradient: the result does not require grad, and inputs with forward-mode tangents are refused.

    Large matrices (more than 64 rows on the shorter side, or more than 512, with 33 to 64 rows 256, on the longer) may go to a kernel
    with bounded waits, for whose answer the call waits (RuntimeError if one gave up) unless check is False, where only NaN in the
    result shows it; their number decides on the kernel and on the CTAs that share a matrix, which shows in the last bits."""
    _refuse_tangents("orthogonalize", (update, out))
    n, rows, cols = _shape("update", update)
    if update.dtype not in _TYPES:
        raise ValueError("update must be float32, float16 or bfloat16")
    args = _coefficients(coefficients, steps, eps)
    if out is None:
        out = torch.empty_like(update, memory_format=torch.contiguous_format)
    elif out.shape != update.shape or out.dtype != update.dtype:
        raise ValueError("out must have the shape and type of update")
    elif 0 < abs(out.data_ptr() - update.data_ptr()) < update.numel() * update.element_size():
        raise ValueError("out must be update or lie apart from it")
    dev = _check_tensors([update, out])
    with _on(dev):
        answer = _answer([(n, rows, cols)], check)
        rc = L.load().mlpsp_orthogonalize(L.ptr(update), _TYPES[update.dtype], n, rows, cols, *args, L.ptr(out),
                                          None if answer is None else C.byref(answer), _stream_ptr(dev))
    _written(rc, "mlpsp_orthogonalize", [out])
    _read(answer, "orthogonalize")
    return out


@torch.no_grad()
def muon_step(weights, grads, momenta, *, lr: float, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
              steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7, active: torch.Tensor | None = None, check: bool = True) -> None:
    """One optimizer step, in place, on one weight tensor or a list of them, each a matrix or a stack:

        m <- m + (1 - momentum) (g - m),   U = g + momentum (m - g) (nesterov) or m
        w <- (1 - lr weight_decay) w - lr sqrt(max(1, rows / columns)) orthogonalize(U)

    weights and momenta are float32 (momenta start at zero), grads float32, float16 or bfloat16, all contiguous and of one shape
    per entry.  active: bool [N], for stacks of N matrices only: primitives whose entry is False (no record reached them,
    csr.offsets[1:] == csr.offsets[:-1]) keep weights and momenta; their gradients are not read.  The orthogonalised update does not
    shrink with the gradient, so a primitive that is not left out moves by lr however little it was seen; a zero gradient and
    zero momentum leave its direction at zero.  A gradient that is not finite makes its own matrix NaN: check gradients first, as
    grouped_weight_gradients does.  check: as in orthogonalize; without it a wait that gave up shows as NaN in the weights."""
    lists = [[t] if torch.is_tensor(t) else list(t) for t in (weights, grads, momenta)]
    if not lists[0] or len({len(k) for k in lists}) != 1:
        raise ValueError("weights, grads and momenta must be as many, at least one")
    _refuse_tangents("muon_step", (t for k in lists for t in k))
    shapes = [_shape("weights", w) for w in lists[0]]
    for w, g, m in zip(*lists):
        if w.dtype != torch.float32 or m.dtype != torch.float32:
            raise ValueError("weights and momenta must be FP32")
        if g.dtype not in _TYPES:
            raise ValueError("grads must be float32, float16 or bfloat16")
        if g.shape != w.shape or m.shape != w.shape:
            raise ValueError("a weight, its gradient and its momentum must have one shape")
    dev = _check_tensors([t for k in lists for t in k] + ([] if active is None else [active]))
    if active is not None and (active.dtype != torch.bool or active.ndim != 1
                               or any(w.ndim != 3 or w.shape[0] != active.numel() for w in lists[0])):
        raise ValueError("active must be bool [N], and every weight a stack of N matrices")
    args = _coefficients(coefficients, steps, eps)
    lr, momentum, weight_decay = float(lr), float(momentum), float(weight_decay)
    if not (0.0 <= lr < 1e30 and 0.0 <= weight_decay < 1e30 and 0.0 <= momentum < 1.0):
        raise ValueError("lr and weight_decay must be finite and not negative, momentum within [0, 1)")
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), k != 1) for k in range(3) for t in lists[k] if t.numel())
    reached = [0, 0]        # where the arrays so far end: any of them, written ones
    for first, end, written in spans:
        if first < reached[0 if written else 1]:
            raise ValueError("weights and momenta must not overlap each other or a gradient")
        reached[0] = max(reached[0], end)
        reached[1] = max(reached[1], end if written else 0)
    lib = L.load()
    with _on(dev):
        answer = _answer(shapes, check)
        tensors = (L.MuonTensor * len(shapes))(*(
            (L.ptr(w), L.ptr(g), L.ptr(m), n, rows, cols, math.sqrt(max(1.0, rows / cols)), _TYPES[g.dtype], 0)
            for w, g, m, (n, rows, cols) in zip(*lists, shapes)))
        rc = lib.mlpsp_muon_step(tensors, len(shapes), L.ptr(active), lr, momentum, int(bool(nesterov)), weight_decay, *args,
                                 None if answer is None else C.byref(answer), _stream_ptr(dev))
    _written(rc, "mlpsp_muon_step", lists[0] + lists[2])
    _read(answer, "muon_step")
