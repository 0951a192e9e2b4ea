"""Refusals of the layer operators that need no GPU: the Python checks in front of the library, and the library's own
checks of sizes, which come before any device call."""
import ctypes as C

import pytest
import torch

from bnp_vae_amd import _lib, layers


def test_cpu_tensors_are_refused():
    t = torch.zeros((4, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layers.top_leaves(t, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layers.sort_by_leaf(torch.zeros(4, dtype=torch.int32), 3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layers.dense(t, torch.zeros((3, 8)))
    plan = layers.LeafPlan(torch.zeros((4, 1), dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                           torch.zeros(4, dtype=torch.int32), 3)
    for call in (layers.dispatch, layers.combine):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call(t, plan)
        with pytest.raises(TypeError, match="LeafPlan"):
            call(t, None)
    with pytest.raises(TypeError, match="torch tensor"):
        layers.top_leaves([[0.5, 0.5]], 1)


def _fails(rc, text):
    assert rc == 1
    assert text in _lib.lib.bnpvi_last_error().decode(), _lib.lib.bnpvi_last_error()


class _Ctx(object):
    """A stand-in for a context (its memory is never looked at before the sizes are)."""

    def __init__(self):
        self.mem = C.create_string_buffer(4096)
        self.p = C.c_void_p(C.addressof(self.mem))


def test_library_refuses_sizes():
    lib, c, one = _lib.lib, _Ctx(), C.c_void_p(256)
    _fails(lib.bnpvi_top_leaves(None, one, 4, 1, 4, 1, 1, one, one, None, None), "ctx")
    _fails(lib.bnpvi_top_leaves(c.p, one, 3, 1, 4, 1, 1, one, one, None, None), "at least L")
    _fails(lib.bnpvi_top_leaves(c.p, one, 4, 1, 4, 5, 1, one, one, None, None), "k=5")
    _fails(lib.bnpvi_top_leaves(c.p, one, 64, 1, 64, 9, 1, one, one, None, None), "k=9")
    _fails(lib.bnpvi_top_leaves(c.p, one, 64, 1 << 33, 64, 1, 1, one, one, None, None), "N=")
    _fails(lib.bnpvi_top_leaves(c.p, None, 64, 1, 64, 1, 1, one, one, None, None), "NULL")
    _fails(lib.bnpvi_top_leaves_backward(c.p, one, one, None, one, 1, 4, 1, 1, one, 4, 4, None), "NULL")
    _fails(lib.bnpvi_top_leaves_backward(c.p, one, one, one, one, 1, 4, 1, 1, one, 4, 3, None), "cols=3")
    most = lib.bnpvi_leaf_sort_max_leaves()
    assert most >= 7776
    _fails(lib.bnpvi_leaf_sort(c.p, one, 10, most + 1, one, one, one, one, 1 << 40, None), "L=")
    _fails(lib.bnpvi_leaf_sort(c.p, one, 1 << 31, 4, one, one, one, one, 1 << 40, None), "slots")
    need = lib.bnpvi_leaf_sort_workspace(100000, 64)
    assert need > 0 and lib.bnpvi_leaf_sort_workspace(100, 64) == 0
    assert lib.bnpvi_leaf_sort_workspace(-1, 64) == -1 and lib.bnpvi_leaf_sort_workspace(5, 0) == -1
    _fails(lib.bnpvi_leaf_sort(c.p, one, 100000, 64, one, one, one, one, need - 1, None), "workspace")
    _fails(lib.bnpvi_leaf_sort(c.p, one, 100000, 64, one, one, one, None, need, None), "workspace")
    _fails(lib.bnpvi_rows_to_leaves(c.p, 3, one, 8, 4, 1, 8, one, one, 4, one, 8, None), "dtype")
    _fails(lib.bnpvi_rows_to_leaves(c.p, 0, one, 7, 4, 1, 8, one, one, 4, one, 8, None), "pitch")
    _fails(lib.bnpvi_rows_to_leaves(c.p, 0, one, 8, 1 << 30, 2, 8, one, one, 4, one, 8, None), "2^31")
    _fails(lib.bnpvi_rows_from_leaves(c.p, 0, one, 8, one, None, None, 4, 4, 1, 8, one, 8, None), "NULL")
    _fails(lib.bnpvi_rows_from_leaves(c.p, 0, one, 8, one, None, one, 4, 4, 0, 8, one, 8, None), "k=0")
    _fails(lib.bnpvi_rows_from_leaves_backward(c.p, 0, one, 8, one, 8, one, None, one, 4, 4, 1, 8, one, 8, one, None), "NULL")


def test_library_refuses_dense():
    lib, c, one = _lib.lib, _Ctx(), C.c_void_p(256)

    def dense(dtype=0, ldx=8, ldw=8, act=0, offsets=None, G=0, M=4, K=8, n=6, y=one, ldy=6, dact=None, work=one, size=1 << 40):
        return lib.bnpvi_dense(c.p, dtype, one, ldx, one, ldw, 0, None, 0, act, None, 0, offsets, G, M, K, n, y, ldy, dact, 5,
                               work, size, None)
    _fails(dense(dtype=7), "dtype")
    _fails(dense(act=6), "activation")
    _fails(dense(ldx=7), "pitches")
    _fails(dense(ldx=1 << 21), "pitches")
    _fails(dense(G=2), "offsets")
    _fails(dense(offsets=one), "offsets")
    _fails(dense(G=20000, offsets=one), "G=")
    _fails(dense(K=0), "K=0")
    _fails(dense(n=(1 << 20) + 1), "n=")
    _fails(dense(M=1 << 31), "M=")
    _fails(dense(ldy=5), "pitch of y")
    _fails(dense(dact=one), "pitch of y")
    _fails(dense(y=None), "NULL")
    need = lib.bnpvi_dense_workspace(1, 4096, 4096, 64, 9, 0)
    assert need > 0
    _fails(dense(dtype=1, ldx=4096, ldw=4096, K=4096, n=64, ldy=64, M=4096, G=9, offsets=one, size=need - 1), "workspace")
    _fails(dense(dtype=1, ldx=4096, ldw=4096, K=4096, n=64, ldy=64, M=4096, G=9, offsets=one, work=C.c_void_p(8)), "workspace")
    assert lib.bnpvi_dense_workspace(5, 1, 1, 1, 0, 0) == -1 and lib.bnpvi_dense_workspace(0, 1, 0, 1, 0, 1) == -1

    def backward(lddy=6, dx=one, work=one, size=1 << 40, dy=one):
        return lib.bnpvi_dense_backward(c.p, 0, dy, lddy, None, 0, one, 8, one, 8, 0, None, 0, 4, 8, 6, dx, 8, one, one, None, 0,
                                        work, size, None)
    _fails(backward(lddy=5), "pitch")
    _fails(backward(size=0), "workspace")
    _fails(backward(dy=None), "NULL")


def test_views_whose_memory_is_not_their_value_are_refused():
    negated = torch.zeros((4, 8), dtype=torch.complex64).conj().imag
    assert negated.is_neg()
    for t in (negated, torch.eye(4).to_sparse()):
        with pytest.raises(TypeError, match="dense tensor"):
            layers.top_leaves(t, 1)
        with pytest.raises(TypeError, match="dense tensor"):
            layers.dense(t, torch.zeros((3, 8)))


def test_plans_of_other_shapes_and_types_are_refused():
    i = dict(dtype=torch.int32)
    place, order, offsets = torch.zeros((4, 2), **i), torch.zeros(8, **i), torch.zeros(4, **i)
    plan = layers.LeafPlan(place, order, offsets, 3)
    assert plan.num_frames == 4 and plan.choices == 2
    for p, o, L in ((place.long(), offsets, 3), (place[0], offsets, 3), (place.t(), offsets, 3), (place, offsets, 4),
                    (place, offsets.long(), 3), (place, torch.zeros(8, **i)[::2], 3)):
        with pytest.raises(ValueError, match="LeafPlan"):
            layers.LeafPlan(p, order, o, L)


@pytest.mark.parametrize("L", [1, 64, 2407, 2408, 7776, 16384])
@pytest.mark.parametrize("M", [0, 1, 2047, 2048, 2049, 4096, 8191, 8192, 8193])
def test_a_sort_without_workspace_has_its_counters_in_the_lds(M, L):
    """One workgroup sorts alone where 16 waves' counters of L + 1 bins, the bins' firsts and 16 sums fit 160 KB; everywhere
    else the call needs a workspace for the chunks' counters, however many slots there are."""
    alone = M <= 8192 and 4 * (17 * (L + 1) + 16) <= 160 * 1024
    need = _lib.lib.bnpvi_leaf_sort_workspace(M, L)
    assert need == 0 if alone else need >= 8 * (L + 1)
    if not alone:
        c, one = _Ctx(), C.c_void_p(256)
        _fails(_lib.lib.bnpvi_leaf_sort(c.p, one, M, L, one, one, one, None, 0, None), "workspace")


def test_dual_tensors_are_refused():
    """Forward-mode differentiation: a result without its tangent would be a wrong derivative (here below the checks that
    refuse CPU tensors)."""
    import torch.autograd.forward_ad as fwd
    t, plain = torch.rand((4, 8)), torch.rand((4, 8))
    place, offsets = torch.zeros((4, 1), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with fwd.dual_level():
        dual = fwd.make_dual(t, torch.ones_like(t))
        one = fwd.make_dual(torch.ones(4, 1), torch.ones(4, 1))
        for call in (lambda: layers._ext.top_leaves(dual, 8, 2, True, 0),
                     lambda: layers._ext.dispatch(dual, place, offsets, 0),
                     lambda: layers._ext.combine(dual, place, offsets, None, 0),
                     lambda: layers._ext.combine(plain, place, offsets, one, 0),
                     lambda: layers._ext.dense(dual, plain, None, None, None, 0, 0),
                     lambda: layers._ext.dense(plain, dual, None, None, None, 0, 0),
                     lambda: layers._ext.dense(plain, plain, one[:, 0], None, None, 0, 0),
                     lambda: layers._ext.dense(plain, plain[:, :], None, dual[:, :4], None, 0, 0)):
            with pytest.raises(_lib.BnpviError, match="forward-mode"):
                call()


def test_recorders_of_torch_calls_are_refused():
    """torch.jit.trace and make_fx would record the allocation of the result without its kernel (here below the checks
    that refuse CPU tensors)."""
    from torch.fx.experimental.proxy_tensor import make_fx
    t, leaf = torch.rand((4, 8)), torch.zeros((4, 1), dtype=torch.int32)
    offsets = torch.zeros(4, dtype=torch.int32)
    for call in (lambda x: layers._ext.top_leaves(x, 8, 2, True, 0)[1], lambda x: layers._ext.dispatch(x, leaf, offsets, 0),
                 lambda x: layers._ext.combine(x, leaf, offsets, None, 0), lambda x: layers._ext.dense(x, x, None, None, None, 0, 0),
                 lambda x: layers._ext.sort_by_leaf(leaf, 3, 0)[0] + x[0, 0]):
        with pytest.raises(_lib.BnpviError, match="traced"):
            torch.jit.trace(call, (t,))
        with pytest.raises(_lib.BnpviError, match="traced"):
            make_fx(call)(t)


X_OFF, W_OFF, DY_OFF, DACT, DX, DW, DB, DRES, STEP = (1 << i for i in range(1, 10))


def _need(dtype, M, K, n, G, *bits):
    return _lib.lib.bnpvi_dense_workspace_for(dtype, M, K, n, G, sum(bits))


def test_a_dense_call_needs_no_copy_of_what_lies():
    """65536 x 4096 -> 256 in bf16 whose operands lie on 16 bytes: no copy of x, no dz where it is dy.  Split sums take at
    most 64 partial results of dW; every part is rounded up to 256 bytes."""
    M, K, n, e = 65536, 4096, 256, 2
    dw_parts, db_parts = 64 * n * K * 4, 2 * (M // 128) * n * 4
    asked = (1, DX, DW, DB)
    assert _need(1, M, K, n, 0) == 0
    assert _need(1, M, K, n, 0, *asked) <= dw_parts + db_parts + 4096
    assert _need(1, M, K, n, 0, DACT, *asked) <= dw_parts + db_parts + 2 * M * n * e + 4096
    assert M * K * e > dw_parts + db_parts + 2 * M * n * e                    # the copy of x alone is more
    assert _need(1, M, K, n, 0, X_OFF, *asked) >= M * K * e                   # where x is off 16 bytes its copy pays
    assert _need(0, 16385, 64, 4096, 0, *asked) < 16385 * 4096 * 4            # dz is dy
    assert _need(1, 32768, 1024, 1024, 0) == 0 and _need(1, 32768, 1024, 1024, 0, X_OFF) == 32768 * 1024 * e
    assert _need(1, M, K, n, 0, DACT, STEP, *asked) <= dw_parts + db_parts + M * n * e + 4096      # relu: dz in one part
    assert _need(1, M, K, n, 0, 1, DACT, DB) <= db_parts + 4096               # the bias alone: no dz either
    assert _need(5, 1, 1, 1, 0) == -1 and _need(0, 1, 0, 1, 0, 1) == -1


def test_the_workspace_of_all_calls_is_enough_for_each():
    import random
    rng = random.Random(3)
    for _ in range(150):
        dtype, G = rng.randrange(3), rng.choice([0, 0, 1, 5, 64])
        M, K, n = (int(2 ** rng.uniform(0, t)) for t in (16, 12, 12))
        most = [_lib.lib.bnpvi_dense_workspace(dtype, M, K, n, G, b) for b in (0, 1)]
        for call in range(1024):
            assert _need(dtype, M, K, n, G, call) <= most[call & 1], (dtype, M, K, n, G, call)


def test_a_plan_keeps_the_tensors_it_was_checked_with():
    import copy
    i = dict(dtype=torch.int32)
    plan = layers.LeafPlan(torch.zeros((4, 2), **i), torch.arange(8, **i), torch.tensor([0, 8, 8, 8], **i), 3)
    for name, value in (("place", torch.zeros((4, 2), **i)), ("order", torch.zeros(8, **i)), ("offsets", torch.zeros(1, **i)),
                        ("num_leaves", 9)):
        with pytest.raises(AttributeError):
            setattr(plan, name, value)
    again = copy.deepcopy(plan)
    assert torch.equal(again.order, plan.order) and again.order is not plan.order and again.num_leaves == 3


def test_orders_of_other_shapes_types_and_devices_are_refused():
    i = dict(dtype=torch.int32)
    place, order, offsets = torch.zeros((4, 2), **i), torch.zeros(8, **i), torch.zeros(4, **i)
    for o in (order[:7], order.long(), order[None], torch.zeros(16, **i)[::2], order.to("meta")):
        with pytest.raises(ValueError, match="LeafPlan"):
            layers.LeafPlan(place, o, offsets, 3)
    for o in (None, [0] * 8):
        with pytest.raises(TypeError, match="order"):
            layers.LeafPlan(place, o, offsets, 3)


def test_a_backward_call_names_a_known_activation():
    c, one = _Ctx(), C.c_void_p(256)
    for activation in (-2, 6):
        _fails(_lib.lib.bnpvi_dense_backward_act(c.p, 0, activation, one, 6, one, 6, one, 8, one, 8, 0, None, 0, 4, 8, 6, one, 8, one, one,
                                                 None, 0, one, 1 << 40, None), "activation")
    _fails(_lib.lib.bnpvi_dense_backward_act(c.p, 0, 1, one, 6, one, 6, one, 8, one, 8, 0, None, 0, 4, 8, 6, one, 8, one, one,
                                             None, 0, one, 0, None), "workspace")
