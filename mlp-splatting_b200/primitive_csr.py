"""Primitive-major record grouping, same surface as scannet/primitive_csr.py:14-29.

`group_records` returns the same `PrimitiveCSR` fields; the stable grouping runs as a device-wide
radix sort inside libmlpsp_b200.so instead of torch.argsort/bincount/cumsum.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib as L
from .engine import _on, _refuse_tangents, _stream_ptr


@dataclass
class PrimitiveCSR:
    offsets: torch.Tensor
    record_indices: torch.Tensor
    x6: torch.Tensor
    grad4: torch.Tensor
    relu_masks: torch.Tensor | None = None


def _group(primitive_ids, num_primitives, x6=None, grad4=None, relu_masks=None):
    lib = L.load()
    if not primitive_ids.is_cuda:
        raise RuntimeError("group_records runs on a CUDA device; there is no CPU path")
    ids = primitive_ids.to(torch.int32).contiguous()
    dev = ids.device
    R, n = int(ids.numel()), int(num_primitives)
    offsets = torch.empty(n + 1, device=dev, dtype=torch.int64)
    order = torch.empty(R, device=dev, dtype=torch.int64)
    outs = [None if t is None else torch.empty_like(t) for t in (x6, grad4, relu_masks)]
    nbytes = int(lib.mlpsp_group_records_scratch_bytes(R, n))
    scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    with _on(dev):
        st = _stream_ptr(dev)
        L.check(lib.mlpsp_group_rows(L.ptr(ids), R, n, L.ptr(x6), L.ptr(grad4), L.ptr(relu_masks), L.ptr(offsets), L.ptr(order),
                                     *(L.ptr(t) for t in outs), L.ptr(scratch), nbytes, st), "mlpsp_group_rows")
    return offsets, order, outs


def group_order(primitive_ids: torch.Tensor, num_primitives: int):
    """(offsets int64 [N+1], order int64 [R]): records grouped by primitive, record order kept inside a group."""
    return _group(primitive_ids, num_primitives)[:2]


def group_records(primitive_ids, x6, grad4, num_primitives: int, relu_masks=None) -> PrimitiveCSR:
    """Group records by primitive, preserving pixel order inside each group."""
    rows = [t for t in (x6, grad4, relu_masks) if t is not None]
    R = int(primitive_ids.numel())
    if (primitive_ids.is_cuda and all(t.is_contiguous() and t.device == primitive_ids.device for t in rows)
            and x6.dtype == torch.float32 and tuple(x6.shape) == (R, 6) and x6.data_ptr() % 8 == 0
            and grad4.dtype == torch.float32 and tuple(grad4.shape) == (R, 4) and grad4.data_ptr() % 16 == 0
            and (relu_masks is None or (relu_masks.dtype == torch.int32 and tuple(relu_masks.shape) == (R, 2)
                                        and relu_masks.data_ptr() % 8 == 0))
            and not any(t.requires_grad for t in rows)):
        # the record layout of the path: the sort's last kernel moves the rows as well
        offsets, order, outs = _group(primitive_ids, num_primitives, x6, grad4, relu_masks)
        return PrimitiveCSR(offsets, order, *outs)
    offsets, order = group_order(primitive_ids, num_primitives)
    return PrimitiveCSR(offsets, order, x6[order], grad4[order],
                        None if relu_masks is None else relu_masks[order])


@torch.no_grad()
def primitive_records_reverse(ids, offsets, x6, raw, log_scales, quats, grad_rgb, grad_t):
    """Reverse compositing over saved records, the extension entry of the same name in the reference
    (scannet/cuda/primitive_records.cuh:51-74): returns [d4 (R,4), grad_positions (N,3), grad_log_scales (N,3),
    grad_quats (N,4)].  ids int32 [R]; offsets int64 [pixels+1]; x6 [R,6]; raw [R,8]; float32 CUDA tensors."""
    for t in (ids, offsets, x6, raw, log_scales, quats, grad_rgb, grad_t):
        if not (t.is_cuda and t.is_contiguous() and t.device == ids.device):
            raise ValueError("all inputs must be contiguous tensors on one CUDA device")
    if ids.dtype != torch.int32 or offsets.dtype != torch.int64:
        raise ValueError("ids must be int32 and offsets int64")
    if any(t.dtype != torch.float32 for t in (x6, raw, log_scales, quats, grad_rgb, grad_t)):
        raise ValueError("records, geometry and adjoints must be FP32")
    total, pixels, n = int(ids.numel()), int(grad_rgb.shape[0]), int(log_scales.shape[0])
    if offsets.ndim != 1 or offsets.numel() != pixels + 1 or x6.shape != (total, 6) or raw.shape != (total, 8):
        raise ValueError("record tensors do not match the pixel offsets")
    if quats.shape != (n, 4) or log_scales.shape != (n, 3) or grad_rgb.shape != (pixels, 3) or grad_t.numel() != pixels:
        raise ValueError("geometry or adjoint shapes do not match")
    lib = L.load()
    dev = ids.device
    d4 = torch.empty((total, 4), device=dev, dtype=torch.float32)
    gp = torch.empty((n, 3), device=dev, dtype=torch.float32)
    gs = torch.empty((n, 3), device=dev, dtype=torch.float32)
    gq = torch.empty((n, 4), device=dev, dtype=torch.float32)
    nbytes = int(lib.mlpsp_records_reverse_scratch_bytes(total, n))
    scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    found = C.c_int32(0)
    with _on(dev):
        st = _stream_ptr(dev)
        L.check(lib.mlpsp_records_reverse_checked(
            L.ptr(ids), L.ptr(offsets), L.ptr(x6), L.ptr(raw), L.ptr(log_scales), L.ptr(quats), L.ptr(grad_rgb), L.ptr(grad_t),
            pixels, total, n, L.ptr(d4), L.ptr(gp), L.ptr(gs), L.ptr(gq), L.ptr(scratch), nbytes, C.byref(found), st),
            "mlpsp_records_reverse")
    if found.value & L.REVERSE_BAD_OFFSETS:
        raise ValueError("pixel offsets must start at zero, end at the record count and be monotone")
    if found.value & L.REVERSE_BAD_IDS:
        raise ValueError("record primitive ids out of range")
    return [d4, gp, gs, gq]


# ---- rows of pixels to the primitives that their records name, and back ----
_ROW_TYPES = {torch.float32: L.PRECISION_F32, torch.float16: L.PRECISION_F16, torch.bfloat16: L.PRECISION_BF16}


@dataclass(frozen=True)
class RecordRoute:
    """Where the records of `pixels` pixels lie once they are grouped by primitive.

    offsets      int64 [N+1]: the records of primitive i take the places offsets[i] .. offsets[i+1]-1, as in a PrimitiveCSR
    slots        int32 [R], a permutation: the place of every record; places at offsets[N] and behind are those of dropped
                 records (primitive id outside [0, N))
    fan          records per pixel, or 0 with pixel_offsets int64 [pixels+1]: first record of every pixel, then R
    Kernels never follow slots or offsets out of the tensors they index."""

    offsets: torch.Tensor
    slots: torch.Tensor
    pixels: int
    fan: int
    pixel_offsets: torch.Tensor | None = None

    @property
    def records(self):
        return int(self.slots.numel())


def _check_route(route, rows, other=None, weights=None):
    """The calls of a small model are a dozen microseconds of host time, so these checks are written out."""
    if not isinstance(route, RecordRoute):
        raise TypeError("route must be a RecordRoute, as route_records returns it")
    slots, offsets, first = route.slots, route.offsets, route.pixel_offsets
    dev = slots.get_device()
    if (dev < 0 or offsets.get_device() != dev or rows.get_device() != dev or not slots.is_contiguous() or not offsets.is_contiguous()
            or not rows.is_contiguous() or (first is not None and (first.get_device() != dev or not first.is_contiguous()))
            or (other is not None and (other.get_device() != dev or not other.is_contiguous()))
            or (weights is not None and (weights.get_device() != dev or not weights.is_contiguous()))):
        raise ValueError("all inputs must be contiguous tensors on one CUDA device")
    if slots.dtype != torch.int32 or offsets.dtype != torch.int64 or offsets.numel() < 1:
        raise ValueError("slots must be int32 and offsets int64 with the initial zero")
    if first is None:
        if route.pixels < 0 or route.fan < 0 or route.pixels * route.fan != slots.numel():
            raise ValueError("the record count must be pixels x fan")
    elif first.dtype != torch.int64 or first.ndim != 1 or first.numel() != route.pixels + 1:
        raise ValueError("pixel offsets must be int64 with one entry more than pixels")
    if weights is not None and (weights.dtype != torch.float32 or weights.numel() != slots.numel()):
        raise ValueError("weights must be float32, one for every record")
    return dev


def _check_rows(name, rows, count):
    if rows.dtype not in _ROW_TYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    if rows.ndim != 2 or rows.shape[0] != count or not 1 <= rows.shape[1] <= L.ROUTE_MAX_DIM:
        raise ValueError(f"{name} must have shape ({count}, 1..{L.ROUTE_MAX_DIM}), got {tuple(rows.shape)}")


def _call(name, dev, *args):
    """A row call of the library on device `dev`, whose last argument is the stream."""
    fn = getattr(L.load(), name)
    if torch.cuda.current_device() == dev:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        L.check(rc, name)


def _route_args(route):
    """(pixels, fan, pixel_offsets, slots, records, kept) of the C calls."""
    first, offsets, slots = route.pixel_offsets, route.offsets, route.slots
    return (route.pixels, route.fan if first is None else 0, None if first is None else first.data_ptr(), slots.data_ptr(), slots.numel(),
            offsets.data_ptr() + 8 * (offsets.numel() - 1))


def route_records(primitive_ids: torch.Tensor, num_primitives: int, pixel_offsets: torch.Tensor | None = None, *,
                  check: bool = True) -> RecordRoute:
    """The places of a frame's records among the records grouped by primitive (a stable grouping, as group_records).

    primitive_ids: int32 or int64 [pixels, fan], fan primitives for every pixel, or [R] with pixel_offsets int64
    [pixels+1] (the lists of render_tiles_training_records).  An id outside [0, num_primitives), -1 by convention, drops its
    record.  With pixel_offsets the call waits for their check (ValueError) unless check is False."""
    first = pixel_offsets
    if not primitive_ids.is_cuda:
        raise RuntimeError("route_records runs on a CUDA device; there is no CPU path")
    if primitive_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("primitive ids must be int32 or int64")
    if first is None:
        if primitive_ids.ndim != 2:
            raise ValueError("primitive_ids must be [pixels, fan], or [records] with pixel_offsets")
        pixels, fan = (int(d) for d in primitive_ids.shape)
    else:
        if primitive_ids.ndim != 1:
            raise ValueError("primitive_ids must be [records] when pixel_offsets is given")
        if first.ndim != 1 or first.dtype != torch.int64 or first.numel() < 1 or not first.is_contiguous() \
                or first.device != primitive_ids.device:
            raise ValueError("pixel offsets must be contiguous int64 with the initial zero, on the ids' device")
        pixels, fan = int(first.numel()) - 1, 0
    n, R = int(num_primitives), int(primitive_ids.numel())
    if not 0 <= n < 2 ** 31 - 1 or pixels >= 2 ** 31 or R >= 2 ** 31:
        raise ValueError("primitives, pixels and records must be below 2^31")
    if primitive_ids.dtype == torch.int64:      # ids beyond 32 bits are out of range, not wrapped into it
        primitive_ids = primitive_ids.clamp(-1, n).to(torch.int32)
    lib, dev = L.load(), primitive_ids.device
    ids = primitive_ids.contiguous()
    if first is not None and check:
        with _on(dev):      # the stream that the call is for
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("route_records waits for the check of pixel_offsets: pass check=False inside a graph capture")
    offsets = torch.empty(n + 1, device=dev, dtype=torch.int64)
    slots = torch.empty(R, device=dev, dtype=torch.int32)
    nbytes = int(lib.mlpsp_route_records_scratch_bytes(R, n))
    scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
    found = C.c_int32(0)
    _call("mlpsp_route_records", ids.get_device(), ids.data_ptr(), R, n, L.ptr(first), pixels, offsets.data_ptr(), slots.data_ptr(),
          L.ptr(scratch), nbytes, C.byref(found) if first is not None and check else None)
    if found.value & L.ROUTE_BAD_OFFSETS:
        raise ValueError("pixel offsets must start at zero, end at the record count and be monotone")
    return RecordRoute(offsets, slots, pixels, fan, first)


def _dispatch(x, route):
    dev = _check_route(route, x)
    _check_rows("x", x, route.pixels)
    out = x.new_empty((route.slots.numel(), x.shape[1]))
    _call("mlpsp_dispatch_rows", dev, x.data_ptr(), _ROW_TYPES[x.dtype], x.shape[1], *_route_args(route), out.data_ptr())
    return out


def _combine(y, route, weights, name="y"):
    dev = _check_route(route, y, None, weights)
    _check_rows(name, y, route.slots.numel())
    out = y.new_empty((route.pixels, y.shape[1]))
    _call("mlpsp_combine_rows", dev, y.data_ptr(), _ROW_TYPES[y.dtype], y.shape[1], None if weights is None else weights.data_ptr(),
          *_route_args(route), out.data_ptr())
    return out


def _combine_gradients(grad_out, y, route, weights, want_y, weights_shape):
    """y may be None without weights_shape (the gradient of y does not read it), weights None for ones or without want_y."""
    dev = _check_route(route, grad_out, y, weights)
    _check_rows("grad_out", grad_out, route.pixels)
    if y is not None:
        _check_rows("y", y, route.slots.numel())
        if y.dtype != grad_out.dtype or y.shape[1] != grad_out.shape[1]:
            raise ValueError("grad_out and y must have one element type and row length")
    dim = grad_out.shape[1]
    grad_y = grad_out.new_empty((route.slots.numel(), dim)) if want_y else None
    grad_weights = None if weights_shape is None else grad_out.new_empty(weights_shape, dtype=torch.float32)
    if want_y or weights_shape is not None:
        _call("mlpsp_combine_rows_gradients", dev, grad_out.data_ptr(), L.ptr(y), _ROW_TYPES[grad_out.dtype], dim, L.ptr(weights),
              *_route_args(route), L.ptr(grad_y), L.ptr(grad_weights))
    return grad_y, grad_weights


def _saved_route(ctx, offsets, slots, first):
    return RecordRoute(offsets, slots, ctx.pixels, ctx.fan, first)


class _DispatchRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, route):
        ctx.save_for_backward(route.offsets, route.slots, route.pixel_offsets)
        ctx.pixels, ctx.fan = route.pixels, route.fan
        return _dispatch(x, route)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _combine(grad.contiguous(), _saved_route(ctx, *ctx.saved_tensors), None, "grad_rows"), None


class _CombineRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, route, weights):
        ctx.weights_shape = weights.shape if weights is not None and ctx.needs_input_grad[2] else None
        ctx.save_for_backward(None if ctx.weights_shape is None else y, weights if ctx.needs_input_grad[0] else None, route.offsets, route.slots,
                              route.pixel_offsets)
        ctx.pixels, ctx.fan = route.pixels, route.fan
        return _combine(y, route, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, weights, *where = ctx.saved_tensors
        grad_y, grad_weights = _combine_gradients(grad.contiguous(), y, _saved_route(ctx, *where), weights, ctx.needs_input_grad[0],
                                                  ctx.weights_shape if ctx.needs_input_grad[2] else None)
        return grad_y, None, grad_weights


def dispatch_rows(x: torch.Tensor, route: RecordRoute) -> torch.Tensor:
    """Every pixel's row to its records, grouped by primitive: out[route.slots[r]] = x[pixel of r]; the rows of dropped
    records, from route.offsets[N] on, are zero.  x [pixels, D] float32, float16 or bfloat16, contiguous; out [records, D].
    Differentiable in x (reverse mode, once); dispatch_rows_gradient is the gradient without autograd."""
    _refuse_tangents("dispatch_rows", (x,))
    if torch.is_grad_enabled() and x.requires_grad:
        return _DispatchRows.apply(x, route)
    return _dispatch(x, route)


@torch.no_grad()
def dispatch_rows_gradient(grad_rows: torch.Tensor, route: RecordRoute) -> torch.Tensor:
    """Gradient of dispatch_rows with respect to x [pixels, D]: the sums of every pixel's records' rows of grad_rows [records, D],
    in FP32 in the order of the records, rounded once; rows of dropped records are not read."""
    _refuse_tangents("dispatch_rows_gradient", (grad_rows,))
    return _combine(grad_rows, route, None, "grad_rows")


def combine_rows(y: torch.Tensor, route: RecordRoute, weights: torch.Tensor | None = None) -> torch.Tensor:
    """The records' rows back to their pixels: out[p] = sum of weights[r] * y[route.slots[r]] over the records r of p (ones
    without weights), in FP32 in the order of the records, rounded once to y's type.  y [records, D] grouped by primitive,
    float32, float16 or bfloat16, contiguous; weights float32, one per record in record order ([pixels, fan] or [records]).  Rows
    of dropped records are not read; a pixel without records gets zeros.  A pixel's records are visited one behind the other: lists of
    hundreds are what it is made for, 100,000 records of one pixel take 7 ms.  Differentiable in y and weights
    (reverse mode, once); combine_rows_gradients gives both gradients without autograd."""
    _refuse_tangents("combine_rows", (y, weights))
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        return _CombineRows.apply(y, route, weights)
    return _combine(y, route, weights)


@torch.no_grad()
def combine_rows_gradients(grad_out: torch.Tensor, y: torch.Tensor, route: RecordRoute, weights: torch.Tensor | None = None):
    """(gradient of combine_rows with respect to y [records, D], with respect to weights in their shape, or None without
    weights) from grad_out [pixels, D].  Zero for dropped records."""
    _refuse_tangents("combine_rows_gradients", (grad_out, y, weights))
    return _combine_gradients(grad_out, y, route, weights, True, None if weights is None else weights.shape)
