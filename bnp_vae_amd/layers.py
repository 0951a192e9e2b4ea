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
once through torch.autograd (backward: forward-mode tangents are refused, and so are recorders of torch calls such as
torch.jit.trace), runs on the tensors' device and its current stream, allocates through torch and waits for nothing, so it
can be captured into a HIP graph (after one call outside a capture).  A backward pass is captured with leaves of its own or
after every result of an eager pass over the same leaves is gone: torch ties a leaf's gradient node to the stream of its
first use.  No CPU fallback.

A leaf number outside [0, L) -- `top_leaves` gives -1 -- means "no leaf": such a slot takes part in nothing."""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _lib
from ._lib import lib, check

try:
    from . import _torch_layers as _ext
except ImportError as e:
    raise ImportError("bnp_vae_amd/_torch_layers.so does not load (%s): build it with make -C bnp_vae_amd/csrc; there is no "
                      "fallback" % e)
_ext.bind(_lib.LIB_PATH)

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "softsign": 2, "tanh": 3, "silu": 4, "gelu": 5}
_TOP_MAX = lib.bnpvi_top_leaves_max()
_MAX_LEAVES = lib.bnpvi_leaf_sort_max_leaves()

_contexts = {}
_contexts_lock = threading.Lock()


def _ctx(device):
    """The address of the library's context of a device; made once, kept until the process ends."""
    c = _contexts.get(device.index)
    if c is None:
        with _contexts_lock:
            c = _contexts.get(device.index)
            if c is None:
                h = C.c_void_p()
                with torch.cuda.device(device):
                    check(lib.bnpvi_ctx_create(device.index, C.byref(h)), "bnpvi_ctx_create")
                c = _contexts[device.index] = h.value
    return c


def _on_gpu(what, **tensors):
    """All given tensors on one GPU; returns it."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s: %s must be a torch tensor, not %s" % (what, name, type(t).__name__))
        if t.layout is not torch.strided or t.is_neg():
            raise TypeError("%s: %s must be a dense tensor whose memory holds its values (not sparse, not a negated view)" % (what, name))
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


# ------------------------------------------------------------------------------------------------ top leaves
def top_leaves(phi, k, num_leaves=None, renormalize=True):
    """The `k` likeliest leaves of every frame.

    phi: (N, >= L) float32 responsibilities, leaves in the first L = `num_leaves` columns (default: all), as
    `DeviceVI.phi` holds them.  Returns (leaf (N, k) int32, weight (N, k) float32), likeliest first, ties to the lowest
    leaf.  Only finite positive entries are taken: where a frame has fewer than k, leaf is -1 and weight 0.  With
    `renormalize` the weights of a frame sum to 1 (0 for a frame without any leaf).  The gradient flows from the
    weights to the chosen entries of phi; the choice itself has none.  1 <= k <= min(8, L)."""
    device = _on_gpu("top_leaves", phi=phi)
    if phi.dim() != 2 or phi.dtype != torch.float32:
        raise ValueError("top_leaves: phi must be a 2-D float32 tensor, got %s of %s" % (tuple(phi.shape), phi.dtype))
    L = phi.shape[1] if num_leaves is None else int(num_leaves)
    k = int(k)
    if not 1 <= L <= phi.shape[1]:
        raise ValueError("top_leaves: num_leaves=%d for phi with %d columns" % (L, phi.shape[1]))
    most = min(_TOP_MAX, L)
    if not 1 <= k <= most:
        raise ValueError("top_leaves: k=%d (1 .. %d for %d leaves)" % (k, most, L))
    return _ext.top_leaves(phi, L, k, bool(renormalize), _ctx(device))


# ------------------------------------------------------------------------------------------------ sort, dispatch, combine
class LeafPlan(object):
    """The (frame, choice) slots of N frames with k choices each, in leaf order; slot = frame * k + choice.

    place   (N, k) int32  place of each slot in leaf order
    order   (N * k,) int32  slot at each place
    offsets (L + 1,) int32  first place of each leaf; from offsets[L] on lie the slots without a leaf

    sort_by_leaf makes it.  One put together by hand has to be such a sort: rows whose place lies outside are left out, and
    places that repeat leave other rows unwritten.  Its tensors are checked here, once, and stay the plan's: another sort is
    another plan."""

    __slots__ = ("_place", "_order", "_offsets", "_num_leaves")

    def __init__(self, place, order, offsets, num_leaves):
        for name, t in (("place", place), ("order", order), ("offsets", offsets)):
            if not isinstance(t, torch.Tensor):
                raise TypeError("LeafPlan: %s must be a torch tensor, not %s" % (name, type(t).__name__))
        if place.dim() != 2 or place.dtype != torch.int32 or not place.is_contiguous():
            raise ValueError("LeafPlan: place must be a contiguous (N, k) int32 tensor")
        if tuple(order.shape) != (place.numel(),) or order.dtype != torch.int32 or not order.is_contiguous():
            raise ValueError("LeafPlan: order must be a contiguous (%d,) int32 tensor" % place.numel())
        if tuple(offsets.shape) != (num_leaves + 1,) or offsets.dtype != torch.int32 or not offsets.is_contiguous():
            raise ValueError("LeafPlan: offsets must be a contiguous (%d,) int32 tensor" % (num_leaves + 1))
        if not place.device == order.device == offsets.device:
            raise ValueError("LeafPlan: place is on %s, order on %s, offsets on %s" % (place.device, order.device, offsets.device))
        self._place, self._order, self._offsets, self._num_leaves = place, order, offsets, num_leaves

    @property
    def place(self):
        return self._place

    @property
    def order(self):
        return self._order

    @property
    def offsets(self):
        return self._offsets

    @property
    def num_leaves(self):
        return self._num_leaves

    @property
    def num_frames(self):
        return self._place.shape[0]

    @property
    def choices(self):
        return self._place.shape[1]


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
    if not 1 <= L <= _MAX_LEAVES:
        raise ValueError("sort_by_leaf: num_leaves=%d (1 .. %d)" % (L, _MAX_LEAVES))
    if M >= 1 << 31:
        raise ValueError("sort_by_leaf: %d slots (below 2^31)" % M)
    if leaf.dtype == torch.int64:
        leaf = leaf.clamp(-1, L).to(torch.int32)
    return LeafPlan(*_ext.sort_by_leaf(leaf, L, _ctx(device)), L)


def _check_plan(what, plan, **tensors):
    if not isinstance(plan, LeafPlan):
        raise TypeError("%s: plan must be a LeafPlan (sort_by_leaf), not %s" % (what, type(plan).__name__))
    device = _on_gpu(what, **tensors)
    if plan.place.device != device:
        raise ValueError("%s: the plan is on %s, other tensors on %s" % (what, plan.place.device, device))
    return device


def dispatch(x, plan):
    """The frames' rows in leaf order: (N k, D) with row place[n, j] = x[n] for every slot with a leaf, and zeros from row
    offsets[L] on.  x: (N, D)."""
    device = _check_plan("dispatch", plan, x=x)
    _element_type("dispatch", x.dtype)
    if x.dim() != 2 or x.shape[0] != plan.num_frames:
        raise ValueError("dispatch: x has shape %s, the plan %d frames" % (tuple(x.shape), plan.num_frames))
    return _ext.dispatch(x, plan.place, plan.offsets, _ctx(device))


def combine(rows, plan, weight=None):
    """Back to frames: y[n] = sum_j weight[n, j] rows[place[n, j]] over the slots with a leaf (0 for a frame without any),
    summed in fp32 in the order of j.  rows: (N k, D), weight: (N, k) float32 or None (all 1)."""
    device = _check_plan("combine", plan, rows=rows, weight=weight)
    _element_type("combine", rows.dtype)
    N, k = plan.place.shape
    if rows.dim() != 2 or rows.shape[0] != N * k:
        raise ValueError("combine: rows has shape %s, the plan %d slots" % (tuple(rows.shape), N * k))
    if weight is not None:
        if tuple(weight.shape) != (N, k) or weight.dtype != torch.float32:
            raise ValueError("combine: weight must be (%d, %d) float32, got %s of %s"
                             % (N, k, tuple(weight.shape), weight.dtype))
    return _ext.combine(rows, plan.place, plan.offsets, weight, _ctx(device))


# ------------------------------------------------------------------------------------------------ dense
def dense(x, weight, bias=None, activation=None, residual=None, offsets=None):
    """y = residual + act(x weight^T + bias).

    weight (n, K), bias (n,): one weight for all rows; x (..., K), residual (..., n).
    weight (G, n, K), bias (G, n) and offsets (G + 1,) int32 (`LeafPlan.offsets`): rows offsets[g] .. offsets[g + 1] - 1
    of x (M, K) use weight[g] and bias[g]; rows of no group give 0, take no part in any gradient, and what x and residual
    hold there is not looked at.
    activation: None, "relu", "softsign", "tanh", "silu", "gelu" (with the normal distribution function).
    Sums in fp32, one rounding of y and of each gradient; for the backward pass act'(z) is kept in fp32 beside y where there
    is an activation."""
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
        if not 1 <= G <= _MAX_LEAVES:
            raise ValueError("dense: %d groups (1 .. %d)" % (G, _MAX_LEAVES))
        if tuple(offsets.shape) != (G + 1,) or offsets.dtype != torch.int32:
            raise ValueError("dense: offsets must be (%d,) int32, got %s of %s" % (G + 1, tuple(offsets.shape), offsets.dtype))
    if bias is not None and tuple(bias.shape) != tuple(weight.shape[:-1]):
        raise ValueError("dense: bias has shape %s, weight %s" % (tuple(bias.shape), tuple(weight.shape)))
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError("dense: residual has shape %s, the result %s" % (tuple(residual.shape), shape))
    if x.dim() != 2:
        x = x.reshape(-1, K)
        residual = None if residual is None else residual.reshape(-1, n)
    if x.shape[0] >= 1 << 31:
        raise ValueError("dense: %d rows (below 2^31)" % x.shape[0])
    y = _ext.dense(x, weight, bias, residual, offsets, ACTIVATIONS[activation], _ctx(device))
    return y if len(shape) == 2 else y.reshape(shape)
