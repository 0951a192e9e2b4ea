"""Layers that follow the tree: what a model does with the responsibilities of the VI step.

    leaf, weight = top_leaves(phi, k, num_leaves=L)       # the k likeliest leaves of every frame
    plan = sort_by_leaf(leaf, L)                          # (frame, choice) slots in leaf order
    rows = dispatch(x, plan)                              # the frames' rows in that order
    rows = dense(rows, W, b, activation="gelu", offsets=plan.offsets)     # W[g], b[g]: every leaf its own
    y    = combine(rows, plan, weight)                    # back, weighted

    h    = dense(x, W, b, activation="softsign", residual=r)              # one weight for all rows

`dense` with one weight is the reference's dense layer (/root/reference/src/layers.py:76-114) with what stands around
it in its encoder and decoder (/root/reference/src/model.py:70-94); the rest has no counterpart there.

Tensors are fp32, bf16 or fp16 on one GPU (responsibilities and weights of leaves fp32); everything is differentiable
once through torch.autograd, runs on the tensors' device and its current stream, allocates through torch and waits for
nothing, so it can be captured into a HIP graph (after one call outside a capture).  No CPU fallback.  A leaf number
outside [0, L) -- `top_leaves` gives -1 -- means "no leaf": such a slot takes part in nothing."""
from __future__ import annotations

import ctypes as C
import functools
import threading

import torch

from . import _lib
from ._lib import lib, check

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # BNPVI_F32, BNPVI_BF16, BNPVI_F16
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "softsign": 2, "tanh": 3, "silu": 4, "gelu": 5}
_MAX_PITCH = 1 << 22                                                      # bytes between rows that are multiplied

_contexts = {}
_contexts_lock = threading.Lock()


def _ctx(device):
    """The library's context of a device; made once, kept until the process ends."""
    c = _contexts.get(device.index)
    if c is None:
        with _contexts_lock:
            c = _contexts.get(device.index)
            if c is None:
                h = C.c_void_p()
                with torch.cuda.device(device):
                    check(lib.bnpvi_ctx_create(device.index, C.byref(h)), "bnpvi_ctx_create")
                c = _contexts[device.index] = h
    return c


try:                                                  # the handle alone: a Stream object costs 2 us a call
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def _stream(device):
    return _raw_stream(device.index)


def _on_gpu(what, **tensors):
    """All given tensors on one GPU; returns it."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s: %s must be a torch tensor, not %s" % (what, name, type(t).__name__))
        if not t.is_cuda:
            raise RuntimeError("%s: %s is on %s; a ROCm GPU is needed and there is no CPU fallback" % (what, name, t.device))
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError("%s: %s is on %s, other tensors on %s" % (what, name, t.device, device))
    return device


def _element_type(what, dtype, **tensors):
    if dtype not in _TYPES:
        raise TypeError("%s: %s is not supported (float32, bfloat16, float16)" % (what, dtype))
    for name, t in tensors.items():
        if t is not None and t.dtype != dtype:
            raise TypeError("%s: %s is %s, not %s" % (what, name, t.dtype, dtype))
    return _TYPES[dtype]


def _rows(t):
    """`t` (2-D) with contiguous rows at a pitch the kernels take: itself where it is so already."""
    n, w = t.shape
    if n == 0 or w == 0:
        return t
    if (w == 1 or t.stride(1) == 1) and (n == 1 or w <= t.stride(0)) and t.stride(0) * t.element_size() <= _MAX_PITCH:
        return t
    return t.contiguous()


def _pitch(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------ top leaves
def _top_forward(phi, L, k, renormalize, want_total):
    N = phi.shape[0]
    leaf = phi.new_empty((N, k), dtype=torch.int32)
    weight = phi.new_empty((N, k))
    total = phi.new_empty((N,)) if want_total else None
    check(lib.bnpvi_top_leaves(_ctx(phi.device), phi.data_ptr(), _pitch(phi), N, L, k, int(renormalize), leaf.data_ptr(),
                               weight.data_ptr(), _ptr(total), _stream(phi.device)), "bnpvi_top_leaves")
    return leaf, weight, total


class _TopLeaves(torch.autograd.Function):
    @staticmethod
    def forward(ctx, phi, L, k, renormalize):
        rows = _rows(phi)
        leaf, weight, total = _top_forward(rows, L, k, renormalize, renormalize)
        ctx.mark_non_differentiable(leaf)
        ctx.sizes = (phi.shape, L, k, renormalize)
        ctx.save_for_backward(leaf, weight, total)
        return leaf, weight

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _dleaf, dweight):
        leaf, weight, total = ctx.saved_tensors
        shape, L, k, renormalize = ctx.sizes
        dweight = dweight.contiguous()
        dphi = weight.new_empty(shape)
        check(lib.bnpvi_top_leaves_backward(_ctx(leaf.device), leaf.data_ptr(), weight.data_ptr(), _ptr(total),
                                            dweight.data_ptr(), shape[0], L, k, int(renormalize), dphi.data_ptr(),
                                            shape[1], shape[1], _stream(leaf.device)), "bnpvi_top_leaves_backward")
        return dphi, None, None, None


def top_leaves(phi, k, num_leaves=None, renormalize=True):
    """The `k` likeliest leaves of every frame.

    phi: (N, >= L) float32 responsibilities, leaves in the first L = `num_leaves` columns (default: all), as
    `DeviceVI.phi` holds them.  Returns (leaf (N, k) int32, weight (N, k) float32), likeliest first, ties to the lowest
    leaf.  Only finite positive entries are taken: where a frame has fewer than k, leaf is -1 and weight 0.  With
    `renormalize` the weights of a frame sum to 1 (0 for a frame without any leaf).  The gradient flows from the
    weights to the chosen entries of phi; the choice itself has none.  1 <= k <= min(8, L)."""
    _on_gpu("top_leaves", phi=phi)
    if phi.dim() != 2 or phi.dtype != torch.float32:
        raise ValueError("top_leaves: phi must be a 2-D float32 tensor, got %s of %s" % (tuple(phi.shape), phi.dtype))
    L = phi.shape[1] if num_leaves is None else int(num_leaves)
    k = int(k)
    if not 1 <= L <= phi.shape[1]:
        raise ValueError("top_leaves: num_leaves=%d for phi with %d columns" % (L, phi.shape[1]))
    most = min(lib.bnpvi_top_leaves_max(), L)
    if not 1 <= k <= most:
        raise ValueError("top_leaves: k=%d (1 .. %d for %d leaves)" % (k, most, L))
    if phi.requires_grad and torch.is_grad_enabled():
        return _TopLeaves.apply(phi, L, k, bool(renormalize))
    return _top_forward(_rows(phi), L, k, bool(renormalize), False)[:2]


# ------------------------------------------------------------------------------------------------ sort, dispatch, combine
class LeafPlan(object):
    """The (frame, choice) slots of N frames with k choices each, in leaf order; slot = frame * k + choice.

    place   (N, k) int32  place of each slot in leaf order
    order   (N * k,) int32  slot at each place
    offsets (L + 1,) int32  first place of each leaf; from offsets[L] on lie the slots without a leaf"""

    __slots__ = ("place", "order", "offsets", "num_leaves")

    def __init__(self, place, order, offsets, num_leaves):
        self.place, self.order, self.offsets, self.num_leaves = place, order, offsets, num_leaves

    @property
    def num_frames(self):
        return self.place.shape[0]

    @property
    def choices(self):
        return self.place.shape[1]


@functools.lru_cache(maxsize=1024)
def _sort_workspace(M, L):
    return lib.bnpvi_leaf_sort_workspace(M, L)


def sort_by_leaf(leaf, num_leaves):
    """Stable sort of the slots by leaf: LeafPlan.  leaf: (N,) or (N, k) int32 / int64; N k < 2^31, num_leaves <= 16384."""
    device = _on_gpu("sort_by_leaf", leaf=leaf)
    if leaf.dim() not in (1, 2) or leaf.dtype not in (torch.int32, torch.int64):
        raise ValueError("sort_by_leaf: leaf must be a (N,) or (N, k) int32 or int64 tensor, got %s of %s"
                         % (tuple(leaf.shape), leaf.dtype))
    if leaf.dim() == 1:
        leaf = leaf[:, None]
    N, k = leaf.shape
    L, M = int(num_leaves), N * k
    if k < 1:
        raise ValueError("sort_by_leaf: no choices (shape %s)" % (tuple(leaf.shape),))
    if not 1 <= L <= lib.bnpvi_leaf_sort_max_leaves():
        raise ValueError("sort_by_leaf: num_leaves=%d (1 .. %d)" % (L, lib.bnpvi_leaf_sort_max_leaves()))
    if M >= 1 << 31:
        raise ValueError("sort_by_leaf: %d slots (below 2^31)" % M)
    if leaf.dtype == torch.int64:
        leaf = leaf.clamp(-1, L).to(torch.int32)
    leaf = leaf.contiguous()
    place = leaf.new_empty((N, k))
    order = leaf.new_empty((M,))
    offsets = leaf.new_empty((L + 1,))
    need = _sort_workspace(M, L)
    work = leaf.new_empty((need,), dtype=torch.uint8) if need else None
    check(lib.bnpvi_leaf_sort(_ctx(device), leaf.data_ptr(), M, L, place.data_ptr(), order.data_ptr(), offsets.data_ptr(),
                              _ptr(work), need, _stream(device)), "bnpvi_leaf_sort")
    return LeafPlan(place, order, offsets, L)


def _to_leaves(x, place, offsets):
    x = _rows(x)
    (N, k), D = place.shape, x.shape[1]
    xs = x.new_empty((N * k, D))
    if D:
        check(lib.bnpvi_rows_to_leaves(_ctx(x.device), _TYPES[x.dtype], x.data_ptr(), _pitch(x), N, k, D, place.data_ptr(),
                                       offsets.data_ptr(), offsets.shape[0] - 1, xs.data_ptr(), D, _stream(x.device)),
              "bnpvi_rows_to_leaves")
    return xs


def _from_leaves(ys, place, offsets, weight):
    ys = _rows(ys)
    (N, k), D = place.shape, ys.shape[1]
    y = ys.new_empty((N, D))
    if D:
        check(lib.bnpvi_rows_from_leaves(_ctx(ys.device), _TYPES[ys.dtype], ys.data_ptr(), _pitch(ys), place.data_ptr(),
                                         _ptr(weight), offsets.data_ptr(), offsets.shape[0] - 1, N, k, D, y.data_ptr(), D,
                                         _stream(ys.device)), "bnpvi_rows_from_leaves")
    return y


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, place, offsets):
        ctx.save_for_backward(place, offsets)
        return _to_leaves(x, place, offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxs):
        place, offsets = ctx.saved_tensors
        return _from_leaves(dxs, place, offsets, None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weight, place, offsets):
        ctx.save_for_backward(ys if weight is not None else None, weight, place, offsets)
        return _from_leaves(ys, place, offsets, weight)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ys, weight, place, offsets = ctx.saved_tensors
        if weight is None:
            return _to_leaves(dy, place, offsets), None, None, None
        dy, ys = _rows(dy), _rows(ys)
        (N, k), D = place.shape, ys.shape[1]
        dys = ys.new_empty((N * k, D)) if ctx.needs_input_grad[0] else None
        dweight = weight.new_empty((N, k)) if ctx.needs_input_grad[1] else None
        if D:
            check(lib.bnpvi_rows_from_leaves_backward(
                _ctx(ys.device), _TYPES[ys.dtype], dy.data_ptr(), _pitch(dy), ys.data_ptr(), _pitch(ys), place.data_ptr(),
                weight.data_ptr(), offsets.data_ptr(), offsets.shape[0] - 1, N, k, D, _ptr(dys), D, _ptr(dweight),
                _stream(ys.device)), "bnpvi_rows_from_leaves_backward")
        elif dweight is not None:
            dweight.zero_()
        return dys, dweight, None, None


def _check_plan(what, plan, **tensors):
    if not isinstance(plan, LeafPlan):
        raise TypeError("%s: plan must be a LeafPlan (sort_by_leaf), not %s" % (what, type(plan).__name__))
    return _on_gpu(what, **dict(tensors, place=plan.place, offsets=plan.offsets))


def dispatch(x, plan):
    """The frames' rows in leaf order: (N k, D) with row place[n, j] = x[n] for every slot with a leaf, and zeros from row
    offsets[L] on.  x: (N, D)."""
    _check_plan("dispatch", plan, x=x)
    _element_type("dispatch", x.dtype)
    if x.dim() != 2 or x.shape[0] != plan.num_frames:
        raise ValueError("dispatch: x has shape %s, the plan %d frames" % (tuple(x.shape), plan.num_frames))
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, plan.place, plan.offsets)
    return _to_leaves(x, plan.place, plan.offsets)


def combine(rows, plan, weight=None):
    """Back to frames: y[n] = sum_j weight[n, j] rows[place[n, j]] over the slots with a leaf (0 for a frame without any),
    summed in fp32 in the order of j.  rows: (N k, D), weight: (N, k) float32 or None (all 1)."""
    _check_plan("combine", plan, rows=rows, weight=weight)
    _element_type("combine", rows.dtype)
    N, k = plan.place.shape
    if rows.dim() != 2 or rows.shape[0] != N * k:
        raise ValueError("combine: rows has shape %s, the plan %d slots" % (tuple(rows.shape), N * k))
    if weight is not None:
        if tuple(weight.shape) != (N, k) or weight.dtype != torch.float32:
            raise ValueError("combine: weight must be (%d, %d) float32, got %s of %s"
                             % (N, k, tuple(weight.shape), weight.dtype))
        weight = weight.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (weight is not None and weight.requires_grad)):
        return _Combine.apply(rows, weight, plan.place, plan.offsets)
    return _from_leaves(rows, plan.place, plan.offsets, weight)


# ------------------------------------------------------------------------------------------------ dense
@functools.lru_cache(maxsize=4096)
def _dense_workspace(dtype, M, K, n, G, backward):
    return lib.bnpvi_dense_workspace(dtype, M, K, n, G, backward)


def _weights(w):
    """A weight (n, K) or (G, n, K) with contiguous rows, and its pitches (row, group)."""
    def fits(t):
        n, K = t.shape[-2:]
        return (K == 1 or t.stride(-1) == 1) and (n == 1 or K <= t.stride(-2)) and t.stride(-2) * t.element_size() <= _MAX_PITCH
    if not fits(w):
        w = w.contiguous()
    ldw = w.stride(-2) if w.shape[-2] > 1 else w.shape[-1]
    return w, ldw, w.stride(0) if w.dim() == 3 and w.shape[0] > 1 else 0


def _dense_forward(x, w, bias, act, residual, offsets, want_dact):
    T = _TYPES[x.dtype]
    (M, K), n = x.shape, w.shape[-2]
    G = w.shape[0] if w.dim() == 3 else 0
    x = _rows(x)
    w, ldw, wg = _weights(w)
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows(residual)
    y = x.new_empty((M, n))
    dact = None
    if want_dact and act:
        dact = x.new_empty((M, n), dtype=torch.float16 if x.dtype == torch.bfloat16 else torch.float32)
    need = _dense_workspace(T, M, K, n, G, 0)
    work = x.new_empty((need,), dtype=torch.uint8) if need else None
    check(lib.bnpvi_dense(_ctx(x.device), T, x.data_ptr(), _pitch(x), w.data_ptr(), ldw, wg, _ptr(bias), n if G > 1 else 0,
                          act, _ptr(residual), 0 if residual is None else _pitch(residual), _ptr(offsets), G, M, K, n,
                          y.data_ptr(), n, _ptr(dact), n, _ptr(work), need, _stream(x.device)), "bnpvi_dense")
    return y, dact


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, offsets, act):
        y, dact = _dense_forward(x, w, bias, act, residual, offsets, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, w, offsets, dact)
        ctx.bias_shape = None if bias is None else bias.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, offsets, dact = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        (M, K), n = x.shape, w.shape[-2]
        G = w.shape[0] if w.dim() == 3 else 0
        T = _TYPES[x.dtype]
        dy = _rows(dy)
        dx = x.new_empty((M, K)) if need_x else None
        dw = x.new_empty(w.shape) if need_w else None
        db = x.new_empty(ctx.bias_shape) if need_b else None
        dres = None
        if need_r:
            dres = x.new_empty((M, n)) if G else dy
        x = _rows(x)
        w, ldw, wg = _weights(w)
        own_dres = dres if G else None
        if need_x or need_w or need_b or own_dres is not None:
            need = _dense_workspace(T, M, K, n, G, 1)
            work = x.new_empty((need,), dtype=torch.uint8) if need else None
            check(lib.bnpvi_dense_backward(_ctx(x.device), T, dy.data_ptr(), _pitch(dy), _ptr(dact), n, x.data_ptr(),
                                           _pitch(x), w.data_ptr(), ldw, wg, _ptr(offsets), G, M, K, n, _ptr(dx), K,
                                           _ptr(dw), _ptr(db), _ptr(own_dres), n, _ptr(work), need, _stream(x.device)),
                  "bnpvi_dense_backward")
        return dx, dw, db, dres, None, None


def dense(x, weight, bias=None, activation=None, residual=None, offsets=None):
    """y = residual + act(x weight^T + bias).

    weight (n, K), bias (n,): one weight for all rows; x (..., K), residual (..., n).
    weight (G, n, K), bias (G, n) and offsets (G + 1,) int32 (`LeafPlan.offsets`): rows offsets[g] .. offsets[g + 1] - 1
    of x (M, K) use weight[g] and bias[g]; rows of no group give 0, take no part in any gradient, and what x and residual
    hold there is not looked at.
    activation: None, "relu", "softsign", "tanh", "silu", "gelu" (with the normal distribution function).
    Sums in fp32, one rounding of y; for the backward pass act'(z) is kept beside y where there is an activation."""
    device = _on_gpu("dense", x=x, weight=weight, bias=bias, residual=residual, offsets=offsets)
    if activation not in ACTIVATIONS:
        raise ValueError("dense: activation %r unknown (%s)" % (activation, ", ".join(str(a) for a in ACTIVATIONS)))
    _element_type("dense", x.dtype, weight=weight, bias=bias, residual=residual)
    if weight.dim() not in (2, 3) or (weight.dim() == 3) != (offsets is not None):
        raise ValueError("dense: weight is (n, K), or (G, n, K) together with offsets; got %s and %s offsets"
                         % (tuple(weight.shape), "no" if offsets is None else "some"))
    n, K = weight.shape[-2:]
    if n < 1 or K < 1 or n > 1 << 20 or K > 1 << 20:
        raise ValueError("dense: weight has shape %s (1 <= n, K <= 2^20)" % (tuple(weight.shape),))
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError("dense: x has shape %s, weight %s" % (tuple(x.shape), tuple(weight.shape)))
    shape = tuple(x.shape[:-1]) + (n,)
    if weight.dim() == 3:
        G = weight.shape[0]
        if x.dim() != 2:
            raise ValueError("dense: with offsets x is (M, K), got %s" % (tuple(x.shape),))
        if not 1 <= G <= lib.bnpvi_leaf_sort_max_leaves():
            raise ValueError("dense: %d groups (1 .. %d)" % (G, lib.bnpvi_leaf_sort_max_leaves()))
        if tuple(offsets.shape) != (G + 1,) or offsets.dtype != torch.int32:
            raise ValueError("dense: offsets must be (%d,) int32, got %s of %s" % (G + 1, tuple(offsets.shape), offsets.dtype))
        offsets = offsets.contiguous()
    if bias is not None and tuple(bias.shape) != tuple(weight.shape[:-1]):
        raise ValueError("dense: bias has shape %s, weight %s" % (tuple(bias.shape), tuple(weight.shape)))
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError("dense: residual has shape %s, the result %s" % (tuple(residual.shape), shape))
    if x.dim() != 2:
        x = x.reshape(-1, K)
        residual = None if residual is None else residual.reshape(-1, n)
    if x.shape[0] >= 1 << 31:
        raise ValueError("dense: %d rows (below 2^31)" % x.shape[0])
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        y = _Dense.apply(x, weight, bias, residual, offsets, act)
    else:
        y, _ = _dense_forward(x, weight, bias, act, residual, offsets, False)
    return y if len(shape) == 2 else y.reshape(shape)
