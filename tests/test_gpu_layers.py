"""Layers that follow the tree on the GPU, against plain restatements in 64 bits on the CPU.

Tolerances.  u = half a step of the element type (bf16 2^-8, fp16 2^-11, fp32 2^-24).  A sum of m products in fp32 is
off by at most (m + 16) 2^-23 of the sum of the products' magnitudes (two half steps an addition, whatever its order and
whatever the matrix unit does with its last bit); activations are good to 16 half steps of fp32 beside 1 and have slopes
of at most 1.13 and second derivatives of at most 2; a result is rounded once.  Every bound below is built of these."""
import math
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # smallest steps
ACTS = [None, "relu", "softsign", "tanh", "silu", "gelu"]


@pytest.fixture(scope="module")
def layers():
    from bnp_vae_amd import layers as module
    return module


def gpu(t):
    return t.to("cuda")


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def within(got, want, bound, what=""):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d values off, worst %g where %g is allowed (value %g)" % (
        what, int(bad.sum()), bad.numel(), float((off - bound)[bad].max() if bad.any() else 0),
        float(torch.as_tensor(bound).expand(want.shape)[bad][0]), float(want[bad][0]))


# ------------------------------------------------------------------------------------------------ top leaves
def top_reference(phi, L, k, renorm):
    p = phi[:, :L].double().numpy()
    N = p.shape[0]
    leaf = np.full((N, k), -1, np.int32)
    w = np.zeros((N, k))
    for r in range(N):
        ok = np.nonzero((p[r] > 0) & np.isfinite(p[r]))[0]
        best = ok[np.lexsort((ok, -p[r][ok]))][:k]
        leaf[r, :len(best)] = best
        w[r, :len(best)] = p[r][best]
        if renorm and len(best):
            w[r] /= w[r].sum()
    return torch.from_numpy(leaf), torch.from_numpy(w)


def phi_rows(N, cols, seed):
    g = torch.Generator().manual_seed(seed)
    phi = torch.softmax(torch.randn((N, cols), generator=g) * 20, 1)
    if N > 8 and cols > 3:
        phi[1] = 0.0                                  # no leaf at all
        phi[2] = 0.125                                # all tied
        phi[3, 1:] = -1.0                             # one positive entry
        phi[4] = float("nan")
        phi[5, 0] = float("inf")
        phi[6, 2] = float("nan")
        phi[7] = 2.0 ** -140                          # denormal responsibilities
    return phi


@pytest.mark.parametrize("N,L,cols,k,renorm", [
    (1, 1, 1, 1, True), (1, 64, 64, 2, True), (9, 5, 32, 5, False), (33, 25, 32, 3, True), (257, 32, 32, 8, True),
    (100, 33, 64, 2, False), (70, 64, 64, 1, True), (70, 61, 61, 4, True), (50, 128, 128, 8, True), (50, 129, 160, 7, False),
    (20, 512, 512, 4, True), (9, 7776, 7776, 8, True), (9, 7775, 7777, 3, True), (0, 64, 64, 2, True), (5001, 64, 64, 2, True)])
def test_top_leaves(layers, N, L, cols, k, renorm):
    phi = phi_rows(N, cols, N + L)
    leaf, weight = layers.top_leaves(gpu(phi), k, num_leaves=L, renormalize=renorm)
    want_leaf, want_weight = top_reference(phi, L, k, renorm)
    assert leaf.dtype == torch.int32 and torch.equal(leaf.cpu(), want_leaf)
    within(weight, want_weight, 2 ** -23 * want_weight + 2.0 ** -149, "weight")      # one rounding of an fp64 quotient
    # the gradient: with the values given to the formula in 64 bits
    x = gpu(phi).requires_grad_(True)
    leaf2, w = layers.top_leaves(x, k, num_leaves=L, renormalize=renorm)
    assert not leaf2.requires_grad and torch.equal(leaf2.cpu(), want_leaf)
    dw = rand((N, k), torch.float32, 5)
    got, = torch.autograd.grad(w, x, gpu(dw))
    want = torch.zeros((N, cols), dtype=torch.float64)
    bound = torch.zeros((N, cols), dtype=torch.float64)
    p64 = torch.where((phi > 0) & torch.isfinite(phi), phi, 0.0).double()
    for r in range(N):
        on = want_leaf[r] >= 0
        cols_r = want_leaf[r][on].long()
        d = dw[r][on].double()
        if renorm and on.any():
            s = p64[r][cols_r].sum()
            dot = (d * want_weight[r][on]).sum()
            # dot from weights rounded to fp32, the sum rounded to fp32 (absolute 2^-150 where it is denormal)
            off = 2.0 ** -22 * (d.abs() + (d * want_weight[r][on]).abs().sum()) + (d - dot).abs() * (2.0 ** -149 / s)
            want[r, cols_r], bound[r, cols_r] = (d - dot) / s, off / s
        else:
            want[r, cols_r] = d
    finite = want.abs() < 3e38                       # 1 / 2^-138 passes fp32's range
    within(torch.where(finite, got.cpu().double(), 0.0), torch.where(finite, want, 0.0),
           torch.where(finite, bound + 2.0 ** -24 * want.abs(), 0.0), "dphi")


def test_top_leaves_of_views(layers):
    """Rows that start off 16 bytes, a pitch wider than the row, a transposed matrix."""
    big = phi_rows(40, 70, 3)
    for view in (lambda t: t[:, 1:66], lambda t: t[:, :64], lambda t: t[::2, 4:], lambda t: t.t()):
        v = view(big)
        leaf, weight = layers.top_leaves(view(gpu(big)), 3)
        want_leaf, want_weight = top_reference(v, v.shape[1], 3, True)
        assert torch.equal(leaf.cpu(), want_leaf)
        within(weight, want_weight, 2 ** -23 * want_weight + 2.0 ** -149)


def test_top_leaves_gradient_against_differences(layers):
    """d/dphi of sum(c w) by central differences: step h on an entry of size p bends the quotient by O((h/S)^2)."""
    phi = torch.rand((6, 12), generator=torch.Generator().manual_seed(1)) + 0.2
    phi = phi * (1 + 0.05 * torch.arange(12))        # no two entries closer than the step can reverse matter below
    c = rand((6, 3), torch.float32, 2)
    x = gpu(phi).requires_grad_(True)
    leaf, w = layers.top_leaves(x, 3)
    got, = torch.autograd.grad(w, x, gpu(c))
    h = 2.0 ** -9
    def value(p):
        p = p.double()
        picked = torch.gather(p, 1, leaf.cpu().long())      # the choice itself is held
        return (c.double() * picked / picked.sum(1, keepdim=True)).sum()
    for r in range(6):
        for j in range(12):
            up, down = phi.clone().double(), phi.clone().double()
            up[r, j] += h
            down[r, j] -= h
            slope = float(value(up) - value(down)) / (2 * h)
            # third derivative of a quotient of sums of at least 0.6: at most 6 |c| / S^3
            assert abs(slope - float(got[r, j])) <= 6 * float(c.abs().sum()) / 0.6 ** 3 * h * h / 6 + 1e-6


# ------------------------------------------------------------------------------------------------ sort, dispatch, combine
def sort_reference(leaf, L):
    flat = leaf.reshape(-1).to(torch.int64)
    key = torch.where((flat >= 0) & (flat < L), flat, L)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel())
    counts = torch.bincount(key, minlength=L + 1)
    return place, order, torch.cumsum(counts, 0) - counts


@pytest.mark.parametrize("M,L", [(0, 3), (1, 1), (63, 2), (64, 64), (65, 7), (1000, 25), (1024, 64), (1025, 64), (8192, 512),
                                 (8193, 512), (50000, 64), (5000, 7776), (20000, 7776), (300001, 7776), (9000, 16384), (200, 16384),
                                 (300007, 3), (2100001, 100)])
@pytest.mark.parametrize("kind", ["spread", "one", "none"])
def test_sort_by_leaf(layers, M, L, kind):
    g = torch.Generator().manual_seed(M + L)
    leaf = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32)
    if kind == "one":
        leaf.fill_(L - 1)
    elif kind == "none":
        leaf.fill_(-1)
    elif M > 10:
        leaf[3], leaf[5], leaf[7] = L, 2 ** 31 - 1, -2 ** 31           # no leaf either
    plan = layers.sort_by_leaf(gpu(leaf), L)
    place, order, offsets = sort_reference(leaf, L)
    assert torch.equal(plan.offsets.cpu().long(), offsets)
    assert torch.equal(plan.order.cpu().long(), order)
    assert torch.equal(plan.place.cpu().long().reshape(-1), place)
    assert plan.num_frames == M and plan.choices == 1 and plan.num_leaves == L


def test_sort_by_leaf_of_int64_and_strided(layers):
    leaf = torch.randint(0, 9, (77, 6), generator=torch.Generator().manual_seed(0))
    leaf[4, 2] = 2 ** 40
    leaf[5, 4] = -2 ** 40
    plan = layers.sort_by_leaf(gpu(leaf)[:, ::2], 9)
    place, order, offsets = sort_reference(leaf[:, ::2], 9)
    assert torch.equal(plan.order.cpu().long(), order) and torch.equal(plan.offsets.cpu().long(), offsets)
    assert torch.equal(plan.place.cpu().long().reshape(-1), place)


def exchange_reference(x, ys, leaf, w, L):
    place, order, offsets = sort_reference(leaf, L)
    N, k = leaf.shape
    kept = int(offsets[L])
    place = place.view(N, k)
    on = (place < kept)[:, :, None]
    xs = torch.where(torch.arange(N * k)[:, None] < kept, x.double()[order // k], 0.0)
    rows = torch.where(on, ys.double()[place], 0.0)
    wk = torch.where(on, (torch.ones((N, k)) if w is None else w).double()[:, :, None], 0.0)
    return xs, (wk * rows).sum(1), rows, wk, place, order, kept


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("N,k,D,L", [(1, 1, 1, 1), (5, 2, 3, 4), (64, 1, 32, 25), (33, 3, 100, 7), (130, 2, 256, 64), (17, 4, 257, 5),
                                     (9, 2, 1030, 3), (1000, 8, 6, 600), (0, 2, 8, 3),
                                     (5000, 2, 37, 9), (4099, 3, 9, 40), (700, 2, 2, 3), (700, 2, 5, 3), (3000, 1, 7, 70), (2000, 5, 15, 7000)])
def test_dispatch_and_combine(layers, dtype, N, k, D, L):
    T = TYPES[dtype]
    x, ys = rand((N, D), T, 1), rand((N * k, D), T, 2)
    leaf = torch.randint(-1, L, (N, k), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    w = torch.rand((N, k), generator=torch.Generator().manual_seed(4)) + 0.1
    plan = layers.sort_by_leaf(gpu(leaf), L)
    kept = int(sort_reference(leaf, L)[2][L])
    ys[kept:] = float("nan")                          # rows of no leaf take part in nothing
    X, Y, W = (gpu(t).requires_grad_(True) for t in (x, ys, w))
    xs, y = layers.dispatch(X, plan), layers.combine(Y, plan, W)
    y1 = layers.combine(Y, plan)
    want_xs, want_y, rows, wk, place, order, kept = exchange_reference(x, ys, leaf, w, L)
    assert torch.equal(xs.detach().cpu().double(), want_xs)
    mag = (wk * rows).abs().sum(1)
    within(y, want_y, HALF[T] * want_y.abs() + TINY[T] + (k + 16) * 2.0 ** -23 * mag, "y")
    want1 = rows.sum(1)
    within(y1, want1, HALF[T] * want1.abs() + TINY[T] + (k + 16) * 2.0 ** -23 * rows.abs().sum(1), "y, weight 1")
    dxs, dy = rand((N * k, D), T, 5), rand((N, D), T, 6)
    dxs[kept:] = float("nan")
    dx, dys, dw = torch.autograd.grad([xs, y], [X, Y, W], [gpu(dxs), gpu(dy)])
    back = torch.where((place < kept)[:, :, None], dxs.double()[place], 0.0)
    within(dx, back.sum(1), HALF[T] * back.sum(1).abs() + TINY[T] + (k + 16) * 2.0 ** -23 * back.abs().sum(1), "dx")
    want = torch.zeros((N * k, D), dtype=torch.float64)
    want[place.reshape(-1)] = (wk * dy.double()[:, None]).reshape(N * k, D)
    within(dys, want, (HALF[T] + 2.0 ** -24) * want.abs() + TINY[T], "dys")
    prod = rows * dy.double()[:, None]
    within(dw, prod.sum(2), (D + 16) * 2.0 ** -23 * prod.abs().sum(2) + 2.0 ** -149, "dweight")
    d1, = torch.autograd.grad(y1, Y, gpu(dy))
    want[place.reshape(-1)] = ((place < kept)[:, :, None] * dy.double()[:, None]).reshape(N * k, D)
    assert torch.equal(d1.cpu().double(), want)


def test_dispatch_and_combine_of_views(layers):
    """Rows at a wider pitch and off 16 bytes, an expanded gradient, one slot's weight frozen."""
    leaf = torch.randint(-1, 4, (50, 2), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    plan = layers.sort_by_leaf(gpu(leaf), 4)
    big, bigs = rand((50, 41), torch.bfloat16, 1), rand((100, 41), torch.bfloat16, 2)
    w = torch.rand((50, 4), generator=torch.Generator().manual_seed(4))
    X, Y = gpu(big)[:, 1:34].requires_grad_(True), gpu(bigs)[:, 3:36].requires_grad_(True)
    xs, y = layers.dispatch(X, plan), layers.combine(Y, plan, gpu(w)[:, 1:3])
    want_xs, want_y, rows, wk, place, _order, kept = exchange_reference(big[:, 1:34], bigs[:, 3:36], leaf, w[:, 1:3], 4)
    assert torch.equal(xs.detach().cpu().double(), want_xs)
    within(y, want_y, 2.0 ** -8 * want_y.abs() + 18 * 2.0 ** -23 * (wk * rows).abs().sum(1) + 2.0 ** -133)
    dx, dys = torch.autograd.grad(xs.sum() + y.sum(), [X, Y])
    assert torch.equal(dx.cpu().double(), (place < kept).sum(1).double()[:, None].expand(50, 33))
    want = torch.zeros((100, 33), dtype=torch.float64)
    want[place.reshape(-1)] = wk.expand(50, 2, 33).reshape(100, 33)
    within(dys, want, 2.0 ** -8 * want.abs())


# ------------------------------------------------------------------------------------------------ dense
def act64(name, z):
    if name == "relu":
        return torch.relu(z), (z > 0).double()
    if name == "softsign":
        q = 1 / (1 + z.abs())
        return z * q, q * q
    if name == "tanh":
        return torch.tanh(z), 1 / torch.cosh(z) ** 2
    if name == "silu":
        q = torch.sigmoid(z)
        return z * q, q + z * q * (1 - q)
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def dense_reference(x, w, b, act, r, bounds, dy):
    """Values and the bounds of their errors; w (G, n, K), bounds the groups' rows."""
    T, M, (G, n, K) = x.dtype, x.shape[0], w.shape
    u, t = HALF[T], TINY[T]
    out = {}
    for name, shape in (("y", (M, n)), ("dx", (M, K)), ("dw", (G, n, K)), ("db", (G, n)), ("dr", (M, n))):
        out[name] = [torch.zeros(shape, dtype=torch.float64), torch.zeros(shape, dtype=torch.float64)]
    for g in range(G):
        lo, hi = bounds[g], bounds[g + 1]
        rows = slice(lo, hi)
        xg, wg, m = x[rows].double(), w[g].double(), hi - lo
        bg = torch.zeros(n, dtype=torch.float64) if b is None else b[g].double()
        rg = torch.zeros((m, n), dtype=torch.float64) if r is None else r[rows].double()
        z = xg @ wg.t() + bg
        zoff = (K + 16) * 2.0 ** -23 * (xg.abs() @ wg.abs().t() + bg.abs())
        a, d = act64(act, z)
        y = a + rg
        out["y"][0][rows] = y
        out["y"][1][rows] = u * y.abs() + t + 1.13 * zoff + 16 * 2.0 ** -24 * (1 + a.abs() + rg.abs()) * (act is not None) \
            + 2.0 ** -23 * (a.abs() + rg.abs())
        gy = dy[rows].double()
        dz = gy * d
        doff = 2 * zoff + 16 * 2.0 ** -24 if act is not None else torch.zeros_like(z)
        if act == "relu":
            doff = (z.abs() <= zoff).double()
        if act is not None and T is torch.bfloat16:
            doff = doff + 2.0 ** -11 * d.abs() + 2.0 ** -25
        raw = gy.abs() * doff + 2.0 ** -23 * dz.abs() * (act is not None)          # of dz before its rounding
        zz = raw + (u * (dz.abs() + raw) + t) * (act is not None)
        full = dz.abs() + zz
        dx = dz @ wg
        out["dx"][0][rows] = dx
        off = zz @ wg.abs() + (n + 16) * 2.0 ** -23 * (full @ wg.abs())
        out["dx"][1][rows] = off + u * (dx.abs() + off) + t
        dw = dz.t() @ xg
        off = zz.t() @ xg.abs() + (m + 16) * 2.0 ** -23 * (full.t() @ xg.abs())
        out["dw"][0][g], out["dw"][1][g] = dw, off + u * (dw.abs() + off) + t
        db = dz.sum(0)
        off = raw.sum(0) + (m + 16) * 2.0 ** -23 * (dz.abs() + raw).sum(0)
        out["db"][0][g], out["db"][1][g] = db, off + u * (db.abs() + off) + t
        out["dr"][0][rows] = gy
    return out


def check_dense(layers, M, K, n, T, act, bias, residual, sizes=None, seed=0, view=None, poison=True, head=0):
    """One forward and backward; sizes: rows of each group (None: one weight for all)."""
    G = 1 if sizes is None else len(sizes)
    x, w = rand((M, K), T, seed), rand((G, n, K), T, seed + 1, 1 / math.sqrt(K))
    b = rand((G, n), T, seed + 2, 0.5) if bias else None
    r = rand((M, n), T, seed + 3) if residual else None
    dy = rand((M, n), T, seed + 4)
    bounds = [0, M] if sizes is None else list(head + np.concatenate([[0], np.cumsum(sizes)]))
    bounds = [int(v) for v in bounds]
    if poison and sizes is not None:
        for t in (x, dy) + (() if r is None else (r,)):
            t[bounds[-1]:] = float("nan")
            t[:head] = float("inf")
    want = dense_reference(x, w, b, act, r, bounds, dy)
    put = view or gpu
    X = put(x).requires_grad_(True)
    W = put(w if sizes is not None else w[0]).requires_grad_(True)
    B = None if b is None else gpu(b if sizes is not None else b[0]).requires_grad_(True)
    R = None if r is None else put(r).requires_grad_(True)
    off = None if sizes is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    y = layers.dense(X, W, B, activation=act, residual=R, offsets=off)
    with torch.no_grad():
        assert torch.equal(layers.dense(X, W, B, activation=act, residual=R, offsets=off), y.detach())
    within(y, *want["y"], "y")
    names = [m for m, t in (("dx", X), ("dw", W), ("db", B), ("dr", R)) if t is not None]
    leaves = [t for t in (X, W, B, R) if t is not None]
    for name, got in zip(names, torch.autograd.grad(y, leaves, put(dy))):
        value, bound = want[name]
        if sizes is None and name in ("dw", "db"):
            value, bound = value[0], bound[0]
        within(got, value, bound, name)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("M,K,n", [(1, 1, 1), (1, 64, 32), (2, 8, 8), (5, 40, 7), (31, 24, 33), (33, 72, 64), (128, 64, 128),
                                   (129, 128, 136), (127, 65, 129), (300, 100, 40), (70, 250, 130), (257, 520, 30)])
def test_dense_sizes(layers, dtype, M, K, n):
    check_dense(layers, M, K, n, TYPES[dtype], "softsign", True, True, seed=M + K + n)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("act", ACTS)
def test_dense_activations(layers, dtype, act):
    check_dense(layers, 150, 48, 72, TYPES[dtype], act, True, False, seed=9)
    check_dense(layers, 37, 48, 72, TYPES[dtype], act, False, True, seed=19)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("M,K,n", [(1, 4096, 32), (8, 4096, 256), (40, 2048, 48), (500, 1000, 64), (2500, 64, 512), (4000, 160, 264),
                                   (3, 1000, 2050), (4, 1031, 9), (5, 700, 2500), (6, 33, 5), (7, 4096, 40), (8, 2050, 70), (8, 4096, 4100), (9, 1000, 40)])
def test_dense_long_sums_and_many_tiles(layers, dtype, M, K, n):
    check_dense(layers, M, K, n, TYPES[dtype], "gelu", True, True, seed=M)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("sizes,tail,head", [([3], 0, 0), ([0, 5, 0, 1, 70, 0], 4, 0), ([130, 1, 129, 33], 0, 0), ([0, 0, 0], 6, 0),
                                             ([64, 64], 64, 0), ([1] * 40, 0, 0), ([200, 300, 0, 250], 9, 3), ([7, 0, 12], 0, 5)])
@pytest.mark.parametrize("K,n", [(64, 128), (50, 31)])
def test_dense_per_leaf(layers, dtype, sizes, tail, head, K, n):
    check_dense(layers, head + sum(sizes) + tail, K, n, TYPES[dtype], "silu", True, True, sizes=sizes, seed=sum(sizes), head=head)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_dense_of_views(layers, dtype):
    """Wider pitches, rows off 16 bytes, transposed operands."""
    def wide(t):
        big = torch.full(tuple(t.shape[:-1]) + (t.shape[-1] + 11,), float("nan"), dtype=t.dtype, device="cuda")
        big[..., 8:8 + t.shape[-1]] = gpu(t)
        return big[..., 8:8 + t.shape[-1]].detach()
    def off(t):
        big = torch.full(tuple(t.shape[:-1]) + (t.shape[-1] + 16,), float("nan"), dtype=t.dtype, device="cuda")
        big[..., 3:3 + t.shape[-1]] = gpu(t)
        return big[..., 3:3 + t.shape[-1]].detach()
    def turned(t):
        return gpu(t.transpose(-1, -2).contiguous()).transpose(-1, -2)
    for view in (wide, off, turned):
        check_dense(layers, 140, 56, 136, TYPES[dtype], "tanh", True, True, seed=3, view=view)
        check_dense(layers, 140, 56, 136, TYPES[dtype], None, True, True, sizes=[60, 0, 70], seed=3, view=view)


def test_dense_shapes_around_a_row(layers):
    x, w, b = rand((3, 5, 24), torch.float32, 1), rand((16, 24), torch.float32, 2), rand((16,), torch.float32, 3)
    r = rand((3, 5, 16), torch.float32, 4)
    y = layers.dense(gpu(x), gpu(w), gpu(b), "relu", gpu(r))
    flat = layers.dense(gpu(x).reshape(15, 24), gpu(w), gpu(b), "relu", gpu(r).reshape(15, 16))
    assert y.shape == (3, 5, 16) and torch.equal(y.reshape(15, 16), flat)
    one = layers.dense(gpu(x)[0, 0], gpu(w), gpu(b))
    assert one.shape == (16,)
    empty = layers.dense(gpu(x)[:0], gpu(w).requires_grad_(True), gpu(b))
    assert empty.shape == (0, 5, 16)


@pytest.mark.parametrize("sizes", [None, [9, 0, 20]])
@pytest.mark.parametrize("have", ["", "b", "r", "br"])
def test_dense_gradients_of_some_inputs(layers, have, sizes):
    """Each input alone, and asked for alone of a pass that could give all: the bits of the pass that gives all."""
    M, K, n = 33, 40, 24
    shape = (n,) if sizes is None else (3, n)
    t = {"x": gpu(rand((M, K), torch.bfloat16, 1)), "w": gpu(rand(shape + (K,), torch.bfloat16, 2, 0.2))}
    if "b" in have:
        t["b"] = gpu(rand(shape, torch.bfloat16, 3))
    if "r" in have:
        t["r"] = gpu(rand((M, n), torch.bfloat16, 4))
    off = None if sizes is None else torch.tensor([0, 9, 9, 29], dtype=torch.int32, device="cuda")
    dy = gpu(rand((M, n), torch.bfloat16, 5))

    def run(names):
        leaves = {a: v.clone().requires_grad_(a in names) for a, v in t.items()}
        return leaves, layers.dense(leaves["x"], leaves["w"], leaves.get("b"), "tanh", leaves.get("r"), off)
    leaves, y = run(set(t))
    want = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)))
    for name in t:
        got, = torch.autograd.grad(y, [leaves[name]], dy, retain_graph=True)
        assert torch.equal(got, want[name]), name
        alone, out = run({name})
        got, = torch.autograd.grad(out, [alone[name]], dy)
        assert torch.equal(got, want[name]) and torch.equal(out, y), name


def test_combine_gradients_of_some_inputs(layers):
    plan = layers.sort_by_leaf(torch.randint(-1, 5, (50, 2), device="cuda", generator=torch.Generator("cuda").manual_seed(1)), 5)
    rows, w = gpu(rand((100, 36), torch.float32, 1)), gpu(rand((50, 2), torch.float32, 2))
    dy = gpu(rand((50, 36), torch.float32, 3))
    both = [rows.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    want = torch.autograd.grad(layers.combine(both[0], plan, both[1]), both, dy)
    a = rows.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(layers.combine(a, plan, w), [a], dy)[0], want[0])
    b = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(layers.combine(rows, plan, b), [b], dy)[0], want[1])


def test_a_second_differentiation_is_an_error(layers):
    x = gpu(rand((6, 8), torch.float32, 1)).requires_grad_(True)
    w = gpu(rand((5, 8), torch.float32, 2)).requires_grad_(True)
    plan = layers.sort_by_leaf(torch.zeros(6, dtype=torch.int32, device="cuda"), 1)
    phi = torch.rand((6, 4), device="cuda").requires_grad_(True)
    passes = [(layers.dense(x, w, activation="tanh"), x), (layers.dispatch(x, plan), x), (layers.combine(x, plan), x),
              (layers.combine(x, plan, torch.ones((6, 1), device="cuda")), x), (layers.top_leaves(phi, 2)[1], phi)]
    for out, leaf in passes:
        d, = torch.autograd.grad((out * out).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(d.sum() + leaf.sum(), leaf)


def test_an_input_changed_before_the_backward_pass_is_an_error(layers):
    x = gpu(rand((6, 8), torch.float32, 1))
    w = gpu(rand((5, 8), torch.float32, 2)).requires_grad_(True)
    y = layers.dense(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("G", [0, 3])
def test_dense_without_rows(layers, G):
    w = gpu(rand((G, 8, 16) if G else (8, 16), torch.float32, 1)).requires_grad_(True)
    b = gpu(rand((G, 8) if G else (8,), torch.float32, 2)).requires_grad_(True)
    x = torch.empty((0, 16), device="cuda", requires_grad=True)
    off = torch.zeros(G + 1, dtype=torch.int32, device="cuda") if G else None
    y = layers.dense(x, w, b, activation="gelu", offsets=off)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty((0, 8), device="cuda"))
    assert y.shape == (0, 8) and dx.shape == (0, 16)
    assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


def test_dense_gradient_against_differences(layers):
    """Central differences of sum(c y) in x, W, b: h^2 / 6 times a third derivative (at most 6 |W|^3 |c| for softsign),
    and the fp64 reference gives the values themselves, so nothing else enters."""
    x, w, b = (rand(s, torch.float32, i, 0.5) for i, s in enumerate([(4, 6), (5, 6), (5,)]))
    c = rand((4, 5), torch.float32, 7)
    X, W, B = (gpu(t).requires_grad_(True) for t in (x, w, b))
    y = layers.dense(X, W, B, activation="softsign")
    grads = torch.autograd.grad(y, [X, W, B], gpu(c))
    h = 2.0 ** -10
    base = [t.double() for t in (x, w, b)]
    def value(v):
        z = v[0] @ v[1].t() + v[2]
        return float((c.double() * z / (1 + z.abs())).sum())
    most = max(float(t.abs().max()) for t in base + [torch.ones(1)])
    for i, g in enumerate(grads):
        for j in range(base[i].numel()):
            up, down = [t.clone() for t in base], [t.clone() for t in base]
            up[i].view(-1)[j] += h
            down[i].view(-1)[j] -= h
            slope = (value(up) - value(down)) / (2 * h)
            # softsign's second derivative jumps by 4 at 0, where a difference is off by up to h |x|^2 |c| / 2 x 4
            allowed = float(c.abs().sum()) * most ** 3 * (h * h + 2 * h)
            assert abs(slope - float(g.view(-1)[j].cpu())) <= allowed


def test_dense_with_infinities(layers):
    """Rows with an infinity or NaN spoil themselves alone; activations at infinity have their limits."""
    for T in TYPES.values():
        x = torch.zeros((5, 16), dtype=T)
        x[0, 3], x[1, 4], x[2, 5], x[3, 0] = float("inf"), -float("inf"), float("nan"), 1.0
        w = torch.ones((8, 16), dtype=T)
        for act, at in ((None, [math.inf, -math.inf]), ("relu", [math.inf, 0.0]), ("softsign", [1.0, -1.0]), ("tanh", [1.0, -1.0]),
                        ("silu", [math.inf, 0.0]), ("gelu", [math.inf, 0.0])):
            y = layers.dense(gpu(x), gpu(w), activation=act).cpu().double()
            assert torch.equal(y[0], torch.full((8,), at[0], dtype=torch.float64)), (T, act, y[0])
            assert torch.equal(y[1], torch.full((8,), at[1], dtype=torch.float64)), (T, act, y[1])
            assert torch.isnan(y[2]).all() and torch.isfinite(y[3:]).all() and (y[4] == 0).all()


# ------------------------------------------------------------------------------------------------ a run of them together
def block(layers, phi, x, W1, b1, W2, b2, L, k):
    """Every frame through the layers of its k likeliest leaves, beside its own value."""
    leaf, weight = layers.top_leaves(phi, k, num_leaves=L)
    plan = layers.sort_by_leaf(leaf, L)
    h = layers.dense(layers.dispatch(x, plan), W1, b1, activation="gelu", offsets=plan.offsets)
    return x + layers.combine(layers.dense(h, W2, b2, offsets=plan.offsets), plan, weight)


def block_inputs(N, D, H, L, cols, seed=0):
    phi = phi_rows(N, cols, seed)
    phi = torch.nan_to_num(phi, nan=0.0, posinf=0.0)
    return [phi, rand((N, D), torch.float32, seed + 1), rand((L, H, D), torch.float32, seed + 2, 0.3), rand((L, H), torch.float32, seed + 3),
            rand((L, D, H), torch.float32, seed + 4, 0.3), rand((L, D), torch.float32, seed + 5)]


def test_layers_together(layers):
    N, D, H, L, k = 90, 24, 40, 9, 2
    phi, x, W1, b1, W2, b2 = inputs = block_inputs(N, D, H, L, 32)
    on = [gpu(t).requires_grad_(True) for t in inputs]
    y = block(layers, *on, L, k)
    dy = rand((N, D), torch.float32, 11)
    got = torch.autograd.grad(y, on, gpu(dy))
    leaf, _ = top_reference(phi, L, k, True)
    v = [t.double().requires_grad_(True) for t in inputs]
    out = []
    for r in range(N):
        s, parts = 0.0, []
        for j in range(k):
            l = int(leaf[r, j])
            if l < 0:
                continue
            h = v[2][l] @ v[1][r] + v[3][l]
            h = h * 0.5 * torch.erfc(-h / math.sqrt(2))
            parts.append(v[0][r, l] * (v[4][l] @ h + v[5][l]))
            s = s + v[0][r, l]
        out.append(v[1][r] + (sum(parts) / s if parts else 0.0))
    ref = torch.stack(out)
    want = torch.autograd.grad(ref, v, dy.double())
    # three fp32 sums of at most 56 terms in a row on values of order 1: 1e-4 of the largest value is 10 times their bound;
    # the gradient of phi is divided by a row's sum of responsibilities
    within(y, ref.detach(), 1e-4 * float(ref.abs().max()))
    for g, t, name in zip(got, want, ["dphi", "dx", "dW1", "db1", "dW2", "db2"]):
        if name == "dphi":
            total = torch.where(leaf >= 0, torch.gather(phi.double(), 1, leaf.clamp(min=0).long()), 0.0).sum(1, keepdim=True)
            scale = torch.where(total > 0, 1e-4 * float(ref.abs().max()) * dy.abs().sum(1, keepdim=True).double() / total, 0.0)
            finite = t.abs() < 3e38
            within(torch.where(finite, g.cpu().double(), 0.0), torch.where(finite, t, 0.0), torch.where(finite, scale, 0.0), name)
        else:
            within(g, t, 1e-4 * float(t.abs().max()), name)


def test_layers_in_a_graph(layers):
    """Forward and backward captured, replayed on new inputs between eager work; every replay equals the eager result."""
    N, D, H, L, k = 700, 64, 96, 25, 2
    static = [gpu(t).requires_grad_(i != 0) for i, t in enumerate(block_inputs(N, D, H, L, 32))]
    dy = gpu(rand((N, D), torch.float32, 3))
    def step(v):
        y = block(layers, *v, L, k)
        return [y] + list(torch.autograd.grad(y, v[1:], dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for turn in range(4):
        new = [gpu(t) for t in block_inputs(N, D, H, L, 32, seed=20 + turn)]
        with torch.no_grad():
            for s, t in zip(static, new):
                s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = step([t.requires_grad_(i != 0) for i, t in enumerate(new)])
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_two_graphs_of_one_pool(layers):
    """Two captured steps that share a memory pool, replayed in turn with eager work between: every replay equals eager."""
    N, D, H, L, k = 900, 64, 80, 30, 2
    dy = gpu(rand((N, D), torch.bfloat16, 3))
    w = [gpu(rand((L, H, D), torch.bfloat16, 5, 0.1)).requires_grad_(True), gpu(rand((L, D, H), torch.bfloat16, 6, 0.1)).requires_grad_(True)]
    def step(x, leaf):
        plan = layers.sort_by_leaf(leaf, L)
        y = layers.dense(layers.dispatch(x, plan), w[0], None, "gelu", offsets=plan.offsets)
        y = layers.combine(layers.dense(y, w[1], offsets=plan.offsets), plan)
        return [y.detach()] + list(torch.autograd.grad(y, w, dy))
    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        return gpu(rand((N, D), torch.bfloat16, seed)), gpu(torch.randint(-1, L, (N, k), generator=g, dtype=torch.int32))
    static = [inputs(1), inputs(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if i else None):
            outs.append(step(*static[i]))
    for turn in range(4):
        for i in (0, 1):
            new = inputs(10 + 2 * turn + i)
            for s, t in zip(static[i], new):
                s.copy_(t)
            graphs[i].replay()
            got = [t.clone() for t in outs[i]]
            torch.cuda.synchronize()
            for a, b in zip(got, step(*new)):
                assert torch.equal(a, b)


def test_gradients_and_biases_in_other_layouts(layers):
    """The gradient that arrives transposed or expanded, a bias that is one value or every second of a row: the bits of
    contiguous ones."""
    x, w = gpu(rand((60, 40), torch.float16, 1)).requires_grad_(True), gpu(rand((24, 40), torch.float16, 2)).requires_grad_(True)
    wide, one = gpu(rand((48,), torch.float16, 3)), gpu(rand((1,), torch.float16, 4))
    for b in (wide[::2], one.expand(24)):
        y, same = layers.dense(x, w, b, "silu"), layers.dense(x, w, b.contiguous(), "silu")
        assert torch.equal(y, same)
        for dy in (gpu(rand((24, 60), torch.float16, 5)).t(), one.expand(60, 24), gpu(rand((60, 48), torch.float16, 6))[:, ::2]):
            for p, q in zip(torch.autograd.grad(y, [x, w], dy, retain_graph=True),
                            torch.autograd.grad(same, [x, w], dy.contiguous(), retain_graph=True)):
                assert torch.equal(p, q)
    plan = layers.sort_by_leaf(gpu(torch.arange(60, dtype=torch.int32) % 7)[:, None].expand(60, 2), 7)
    rows, weight = gpu(rand((120, 40), torch.float16, 7)).requires_grad_(True), gpu(rand((2, 60), torch.float32, 8)).t().requires_grad_(True)
    y, flat = layers.combine(rows, plan, weight), weight.detach().contiguous().requires_grad_(True)
    same = layers.combine(rows, plan, flat)
    assert torch.equal(y, same)
    dy = gpu(rand((40, 60), torch.float16, 9)).t()
    for p, q in zip(torch.autograd.grad(y, [rows, weight], dy), torch.autograd.grad(same, [rows, flat], dy.contiguous())):
        assert torch.equal(p, q)


def test_layers_on_another_stream_and_in_threads(layers):
    """Two threads, each on a stream of its own, give the bits of one alone."""
    N, D, H, L, k = 3000, 64, 64, 64, 2
    inputs = [[gpu(t).requires_grad_(True) for t in block_inputs(N, D, H, L, 64, seed=s)] for s in (1, 2)]
    dy = gpu(rand((N, D), torch.float32, 3))
    def step(v):
        y = block(layers, *v, L, k)
        return [y] + list(torch.autograd.grad(y, v, dy))
    want = [step(v) for v in inputs]
    torch.cuda.synchronize()
    got, failed = [None, None], []
    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = step(inputs[i])
            s.synchronize()
        except Exception as e:                                   # noqa: BLE001 - reported by the main thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_same_bits_every_time(layers):
    for T in TYPES.values():
        x, w = gpu(rand((5000, 256), T, 1)).requires_grad_(True), gpu(rand((96, 256), T, 2)).requires_grad_(True)
        b, dy = gpu(rand((96,), T, 3)).requires_grad_(True), gpu(rand((5000, 96), T, 4))
        first = None
        for _ in range(10):
            y = layers.dense(x, w, b, activation="silu")
            now = [y] + list(torch.autograd.grad(y, [x, w, b], dy))
            first = first or now
            for p, q in zip(first, now):
                assert torch.equal(p, q)


# ------------------------------------------------------------------------------------------------ unequal leaves, large arrays
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("sizes,K,n", [([4100, 3, 0, 900, 997], 64, 136), ([0, 9000], 136, 64), ([2600, 2600, 2600], 40, 40)])
def test_dense_long_leaves_are_summed_in_pieces(layers, dtype, sizes, K, n):
    check_dense(layers, sum(sizes) + 7, K, n, TYPES[dtype], None, True, False, sizes=sizes, seed=5)
    check_dense(layers, sum(sizes) + 7, K, n, TYPES[dtype], "relu", True, True, sizes=sizes, seed=6)


@pytest.mark.parametrize("act", [None, "tanh"])
def test_dense_many_leaves(layers, act):
    g = torch.Generator().manual_seed(8)
    sizes = [int(v) for v in torch.randint(0, 5, (700,), generator=g)]
    check_dense(layers, sum(sizes) + 2, 32, 24, torch.bfloat16, act, True, True, sizes=sizes, seed=2)


def test_dense_past_32_bits(layers):
    """4.5 GB of x: the last rows, and a gradient summed over all of them."""
    M, K, n, T = 1100003, 2048, 32, torch.bfloat16
    torch.manual_seed(0)
    x = torch.randn((M, K), device="cuda", dtype=T)
    w = (torch.randn((n, K), device="cuda") / 45).to(T).requires_grad_(True)
    dy = torch.randn((M, n), device="cuda", dtype=T)
    x.requires_grad_(True)
    y = layers.dense(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    x, w = x.detach(), w.detach()
    for rows in (slice(0, 300), slice(M - 300, M)):
        a, b = x[rows].cpu().double(), w.cpu().double()
        z = a @ b.t()
        within(y[rows], z, 2.0 ** -8 * z.abs() + (K + 16) * 2.0 ** -23 * (a.abs() @ b.abs().t()), "y")
        d = dy[rows].cpu().double()
        want = d @ b
        within(dx[rows], want, 2.0 ** -8 * want.abs() + (n + 16) * 2.0 ** -23 * (d.abs() @ b.abs()), "dx")
    want, size = torch.zeros((n, K), dtype=torch.float64, device="cuda"), torch.zeros((n, K), dtype=torch.float64, device="cuda")
    for lo in range(0, M, 100000):
        d, a = dy[lo:lo + 100000].double().t().contiguous(), x[lo:lo + 100000].double()
        want += d @ a
        size += d.abs() @ a.abs()
    # parts of the sum, each with its own fp32 error: together no more than a sum of M terms has; its random walk is
    # bounded by a thousand steps here, as the parts are added up in at most that many partial sums of 1100 terms
    within(dw, want.cpu(), (2.0 ** -8 * want.abs() + M * 2.0 ** -23 * size).cpu(), "dw")
    rel = float((dw.double() - want).norm() / want.norm())
    assert rel < 2.0 ** -8, rel


def test_dispatch_and_combine_past_32_bits(layers):
    N, D = 600007, 4096
    x = torch.randn((N, D), device="cuda", dtype=torch.bfloat16)
    leaf = torch.randint(-1, 30, (N, 1), device="cuda", dtype=torch.int32)
    plan = layers.sort_by_leaf(leaf, 30)
    xs = layers.dispatch(x, plan)
    kept = int(plan.offsets[30])
    for lo in range(0, N, 100000):
        hi = min(N, lo + 100000)
        rows = x[plan.order[lo:hi].long()]
        rows[max(0, kept - lo):] = 0
        assert torch.equal(xs[lo:hi], rows)
    back = layers.combine(xs, plan)
    on = (leaf >= 0)
    for lo in range(0, N, 100000):
        assert torch.equal(back[lo:lo + 100000], torch.where(on[lo:lo + 100000], x[lo:lo + 100000], 0))


def test_another_device(layers):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU visible")
    x, w = rand((70, 40), torch.float32, 1), rand((24, 40), torch.float32, 2)
    here = layers.dense(gpu(x), gpu(w), activation="gelu")
    there = layers.dense(x.to("cuda:1"), w.to("cuda:1"), activation="gelu")
    assert torch.cuda.current_device() == 0 and torch.equal(here.cpu(), there.cpu())


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(layers):
    f = torch.zeros((6, 8), device="cuda")
    leaf = torch.zeros((6, 2), dtype=torch.int32, device="cuda")
    plan = layers.sort_by_leaf(leaf, 3)
    w, b = torch.zeros((5, 8), device="cuda"), torch.zeros((5,), device="cuda")
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    for call, error in [
            (lambda: layers.top_leaves(f, 0), ValueError), (lambda: layers.top_leaves(f, 9), ValueError),
            (lambda: layers.top_leaves(f, 3, num_leaves=2), ValueError), (lambda: layers.top_leaves(f, 1, num_leaves=9), ValueError),
            (lambda: layers.top_leaves(f.half(), 1), ValueError), (lambda: layers.top_leaves(f[0], 1), ValueError),
            (lambda: layers.sort_by_leaf(f, 3), ValueError), (lambda: layers.sort_by_leaf(leaf, 0), ValueError),
            (lambda: layers.sort_by_leaf(leaf, 16385), ValueError), (lambda: layers.sort_by_leaf(leaf[:, :0], 3), ValueError),
            (lambda: layers.dispatch(f[:5], plan), ValueError), (lambda: layers.dispatch(f.double(), plan), TypeError),
            (lambda: layers.combine(f, plan), ValueError),
            (lambda: layers.combine(torch.zeros((12, 8), device="cuda"), plan, torch.zeros((6, 1), device="cuda")), ValueError),
            (lambda: layers.combine(torch.zeros((12, 8), device="cuda"), plan, torch.zeros((6, 2), device="cuda").half()), ValueError),
            (lambda: layers.dense(f, w, activation="swish"), ValueError), (lambda: layers.dense(f.double(), w.double()), TypeError),
            (lambda: layers.dense(f, w.half()), TypeError), (lambda: layers.dense(f[:, :7], w), ValueError),
            (lambda: layers.dense(f, w, b[:4]), ValueError), (lambda: layers.dense(f, w, residual=f), ValueError),
            (lambda: layers.dense(f, w[None]), ValueError), (lambda: layers.dense(f, w, offsets=off), ValueError),
            (lambda: layers.dense(f, w.expand(3, 5, 8), offsets=off), ValueError),
            (lambda: layers.dense(f, w.expand(2, 5, 8), offsets=off.long()), ValueError),
            (lambda: layers.dense(f[None], w.expand(2, 5, 8), offsets=off), ValueError),
            (lambda: layers.dense(f, w.cpu()), RuntimeError)]:
        with pytest.raises(error):
            call()
    y = layers.dense(f.requires_grad_(True), w)
    d, = torch.autograd.grad(y.sum(), f, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()                            # differentiable once


def test_one_weight_for_all_leaves(layers):
    """A weight expanded over the leaves (no copy): its gradient is the sum of theirs."""
    x, w = gpu(rand((200, 32), torch.float32, 1)), gpu(rand((48, 32), torch.float32, 2)).requires_grad_(True)
    off = torch.tensor([0, 60, 60, 200], dtype=torch.int32, device="cuda")
    dy = gpu(rand((200, 48), torch.float32, 3))
    y = layers.dense(x, w.expand(3, 48, 32), offsets=off)
    y1 = layers.dense(x, w)
    a, = torch.autograd.grad(y, w, dy)
    b, = torch.autograd.grad(y1, w, dy)
    within(y, y1.detach().cpu().double(), 2 * 48 * 2.0 ** -23 * (x.abs() @ w.detach().abs().t()).cpu().double())
    within(a, b.cpu().double(), 2 * 220 * 2.0 ** -23 * (dy.abs().t() @ x.abs()).cpu().double())


# ------------------------------------------------------------------------------------------------ the framework's own paths
def fitted(D=16, N=1200, seed=3):
    from bnp_vae_amd import VarInf
    from oracle.vi_oracle import gaussian_mixture, make_latent_dict
    np.random.seed(seed)
    vi = VarInf(latent_code_size=D, stdev_thr=1e9)
    vi.update_variational_parameters(make_latent_dict(gaussian_mixture(N, D, 30, seed=seed, spread=4.0), [100, 57]))
    return vi


def test_leaf_routes_of_a_fitted_tree(layers):
    vi = fitted()
    leaf, weight, plan = vi.leaf_routes(3)
    leaves = vi._dfs_leaves()
    phi = torch.from_numpy(np.concatenate([l.phi for l in leaves], 1).astype(np.float32))
    want_leaf, want_weight = top_reference(phi, phi.shape[1], 3, True)
    assert torch.equal(leaf.cpu(), want_leaf)
    within(weight, want_weight, 2 ** -23 * want_weight + 2.0 ** -149)
    place, order, offsets = sort_reference(want_leaf, len(leaves))
    assert torch.equal(plan.order.cpu().long(), order) and torch.equal(plan.offsets.cpu().long(), offsets)
    # an expected path mean per frame: the leaves' means, weighted
    alpha = torch.from_numpy(np.asarray([l.alpha for l in leaves], dtype=np.float32))
    rows = gpu(alpha)[torch.where(leaf >= 0, leaf, 0).long().reshape(-1)][plan.order.long()]
    mean = layers.combine(rows.contiguous(), plan, weight)
    picked = torch.where(want_leaf >= 0, want_leaf, 0).long()
    terms = want_weight[:, :, None] * alpha.double()[picked]
    within(mean, terms.sum(1), 20 * 2.0 ** -23 * terms.abs().sum(1) + 1e-30)


def test_leaf_routes_needs_latents():
    from bnp_vae_amd import VarInf
    with pytest.raises(RuntimeError, match="no latent codes"):
        VarInf(latent_code_size=4).leaf_routes(1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_hierarchy_from_features(layers, dtype, monkeypatch):
    """nearest_leaf, closest_frames and class_vote with an encoder give what they give for that encoder's latents."""
    from bnp_vae_amd import hierarchy
    vi = fitted()
    nodes = vi.get_nodes_list(vi.root, [])
    F, D, T = 40, 16, TYPES[dtype]
    x = rand((500, F), torch.float32, 1)
    enc = [(gpu(rand((64, F), T, 2, 0.3)), gpu(rand((64,), T, 3)), "relu"), (gpu(rand((D, 64), T, 4, 0.8)), None, "softsign")]
    with torch.no_grad():
        z = layers.dense(layers.dense(gpu(x).to(T), *enc[0]), *enc[1]).float()
    h = torch.relu(x.to(T).double() @ enc[0][0].cpu().double().t() + enc[0][1].cpu().double())
    t = h @ enc[1][0].cpu().double().t()
    # the hidden layer is rounded to T, and so is z; softsign has slopes of at most 1
    within(z, t / (1 + t.abs()), 2 * HALF[T] * (h.abs() @ enc[1][0].cpu().double().abs().t() + 1) + 1e-5)
    monkeypatch.setattr(hierarchy, "ENCODE_ROWS", 128)
    for feats in (x, x.numpy(), gpu(x)):
        assert np.array_equal(hierarchy.nearest_leaf(nodes, feats, encoder=enc), hierarchy.nearest_leaf(nodes, z))
    a, top_a = hierarchy.closest_frames(nodes, x, 4, encoder=enc)
    b, top_b = hierarchy.closest_frames(nodes, z, 4)
    assert np.array_equal(a, b) and top_a == top_b
    labels = np.arange(500) % 3
    p, q = hierarchy.class_vote(nodes, x, labels, x[:50], 0.5, encoder=enc), hierarchy.class_vote(nodes, z, labels, z[:50], 0.5)
    assert np.array_equal(p[0], q[0]) and np.array_equal(p[1], q[1])
    with pytest.raises(ValueError, match="encoder"):
        hierarchy.nearest_leaf(nodes, x, encoder=[])


# ------------------------------------------------------------------------------------------------ sorts of one chunk over many leaves
@pytest.mark.parametrize("M", [2047, 2048, 2049])
@pytest.mark.parametrize("L", [2407, 2408, 7776, 16384])
def test_sort_of_a_chunk_over_many_leaves(layers, M, L):
    """As many slots as a chunk holds, where the counters of a single workgroup just fit the LDS and where they do not."""
    leaf = torch.randint(-1, L, (M,), generator=torch.Generator().manual_seed(M + L), dtype=torch.int32)
    leaf[5], leaf[-1] = L, L - 1
    plan = layers.sort_by_leaf(gpu(leaf), L)
    place, order, offsets = sort_reference(leaf, L)
    assert torch.equal(plan.offsets.cpu().long(), offsets)
    assert torch.equal(plan.order.cpu().long(), order)
    assert torch.equal(plan.place.cpu().long().reshape(-1), place)


@pytest.mark.parametrize("N,k", [(2048, 1), (1024, 2), (512, 4), (256, 8)])
def test_exchange_of_2048_slots_over_the_largest_tree(layers, N, k):
    L = 7776
    leaf = torch.randint(-1, L, (N, k), generator=torch.Generator().manual_seed(N), dtype=torch.int32)
    x = rand((N, 12), torch.float32, 1)
    plan = layers.sort_by_leaf(gpu(leaf), L)
    xs = layers.dispatch(gpu(x), plan)
    ys = rand((N * k, 12), torch.float32, 2)
    want_xs, want_y, rows, _wk, _place, _order, _kept = exchange_reference(x, ys, leaf, None, L)
    assert torch.equal(xs.cpu().double(), want_xs)
    within(layers.combine(gpu(ys), plan), want_y, 2.0 ** -24 * want_y.abs() + (k + 16) * 2.0 ** -23 * rows.abs().sum(1))


def test_closest_frames_of_2048_frames_below_a_wide_tree(layers):
    """Frames are brought into leaf order with the framework's own sort: on 2048 frames over 2500 leaves they lie as
    torch.sort puts them."""
    from bnp_vae_amd import hierarchy
    assign = torch.randint(0, 2500, (2048,), device="cuda", generator=torch.Generator("cuda").manual_seed(3), dtype=torch.int32)
    node = torch.randint(-1, 3000, (2048, 3), device="cuda", generator=torch.Generator("cuda").manual_seed(4), dtype=torch.int32)
    dist = torch.rand((2048, 3), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    rows, node_s, dist_s = hierarchy._by_leaf(assign, 2500, node, dist)
    want = torch.sort(assign.long(), stable=True).indices
    assert torch.equal(rows, want) and torch.equal(node_s, node[want]) and torch.equal(dist_s, dist[want])


# ------------------------------------------------------------------------------------------------ other ways to differentiate or record
def test_forward_mode_is_an_error(layers):
    import torch.autograd.forward_ad as fwd
    x, w, phi = gpu(rand((6, 8), torch.float32, 1)), gpu(rand((5, 8), torch.float32, 2)), torch.rand((6, 4), device="cuda")
    b, r, one = gpu(rand((5,), torch.float32, 3)), gpu(rand((6, 5), torch.float32, 4)), torch.ones((6, 1), device="cuda")
    plan = layers.sort_by_leaf(torch.zeros(6, dtype=torch.int32, device="cuda"), 1)
    calls = [(lambda t: layers.dense(t, w), x), (lambda t: layers.dense(x, t), w), (lambda t: layers.dense(x, w, t), b),
             (lambda t: layers.dense(x, w, None, "tanh", t), r), (lambda t: layers.dispatch(t, plan), x),
             (lambda t: layers.combine(t, plan), x), (lambda t: layers.combine(x, plan, t), one), (lambda t: layers.top_leaves(t, 2), phi)]
    for call, t in calls:
        for leaf in (t, t.clone().requires_grad_(True)):
            with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                call(fwd.make_dual(leaf, torch.ones_like(leaf)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
    with fwd.dual_level():                            # beside dual tensors the plain ones go their way
        fwd.make_dual(x.clone(), x)
        assert torch.equal(layers.dense(x, w), layers.dense(x.clone(), w))


def test_tracing_is_an_error(layers):
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, phi = gpu(rand((6, 8), torch.float32, 1)), gpu(rand((5, 8), torch.float32, 2)), torch.rand((6, 4), device="cuda")
    leaf = torch.zeros(6, dtype=torch.int32, device="cuda")
    plan = layers.sort_by_leaf(leaf, 1)
    for call, t in ((lambda t: layers.dense(t, w, activation="gelu"), x), (lambda t: layers.dispatch(t, plan), x),
                    (lambda t: layers.combine(t, plan), x), (lambda t: layers.top_leaves(t, 2)[1], phi),
                    (lambda t: layers.sort_by_leaf(t, 1).place, leaf)):
        want = call(t)
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (t,))
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(call)(t)
        assert torch.equal(call(t), want)


def test_functional_transforms_are_errors(layers):
    x, w = gpu(rand((3, 6, 8), torch.float32, 1)), gpu(rand((5, 8), torch.float32, 2))
    for call in (lambda: torch.func.vmap(lambda t: layers.dense(t, w))(x),
                 lambda: torch.func.grad(lambda t: layers.dense(t, w).sum())(x),
                 lambda: torch.func.vmap(lambda t: layers.top_leaves(t, 2)[1])(x)):
        with pytest.raises(RuntimeError):
            call()


# ------------------------------------------------------------------------------------------------ memory of a call
@pytest.mark.parametrize("dtype,act,shift", [("bf16", "softsign", 0), ("bf16", None, 0), ("f32", None, 0), ("f32", "gelu", 0), ("bf16", "gelu", 1)])
def test_memory_of_a_dense_pass(layers, dtype, act, shift):
    """What a pass allocates: its results, act'(z) in fp32, dz in two parts (bf16) or one, 8 MB for maps and partial sums
    of the bias, at most 64 partial results of dW -- and copies of x, W and dy only where they are off 16 bytes."""
    M, K, n, T = 131072, 512, 512, TYPES[dtype]
    e = T.itemsize
    def put(shape, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        return torch.randn(shape[:-1] + (shape[-1] + 8,), generator=g, device="cuda").to(T)[..., shift:shift + shape[-1]].detach()
    x, w, dy = put((M, K), 1).requires_grad_(True), put((n, K), 2).requires_grad_(True), put((M, n), 3)
    layers.dense(x[:100], w[:], activation=act).sum().backward()
    x.grad = w.grad = None
    copies = M * K * e + n * K * e if shift else 0
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    y = layers.dense(x, w, activation=act)
    kept = M * n * e + (M * n * 4 if act else 0)
    assert torch.cuda.memory_allocated() - start <= kept + (1 << 20)
    assert torch.cuda.max_memory_allocated() - start <= kept + copies + (8 << 20)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    dz = M * n * (4 if e == 2 else e) if act else M * n * e if shift else 0
    most = kept + M * K * e + n * K * e + dz + 64 * n * K * 4 + copies + (8 << 20)
    assert torch.cuda.max_memory_allocated() - start <= most


def test_class_vote_with_an_encoder_that_is_an_iterator(layers):
    """The layers are needed for the training and for the test frames."""
    from bnp_vae_amd import hierarchy
    vi = fitted()
    nodes = vi.get_nodes_list(vi.root, [])
    x, labels = rand((300, 40), torch.float32, 1), np.arange(300) % 3
    enc = [(gpu(rand((16, 40), torch.float32, 2, 0.3)), gpu(rand((16,), torch.float32, 3)), "softsign")]
    want = hierarchy.class_vote(nodes, x, labels, x[:50], 0.5, encoder=enc)
    got = hierarchy.class_vote(nodes, x, labels, x[:50], 0.5, encoder=iter(enc))
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_frames_without_a_nearest_leaf_keep_their_place(layers, monkeypatch):
    """A frame whose latents are NaN has no nearest leaf (its index is 2^31 - 1): its rows move with it, behind all leaves, as
    torch.sort puts them."""
    from bnp_vae_amd import hierarchy
    assign = torch.randint(0, 40, (500,), device="cuda", generator=torch.Generator("cuda").manual_seed(3), dtype=torch.int32)
    assign[[7, 90, 300]] = 2 ** 31 - 1
    node = torch.randint(0, 60, (500, 3), device="cuda", generator=torch.Generator("cuda").manual_seed(4), dtype=torch.int32)
    dist = torch.rand((500, 3), device="cuda", dtype=torch.float64)
    got, want = hierarchy._by_leaf(assign, 40, node, dist), torch.sort(assign.long(), stable=True).indices
    assert torch.equal(got[0], want) and torch.equal(got[1], node[want]) and torch.equal(got[2], dist[want])
    vi = fitted()
    nodes = vi.get_nodes_list(vi.root, [])
    z = rand((400, 16), torch.float32, 9, 4.0)
    z[[11, 200, 399]] = float("nan")
    path, top = hierarchy.closest_frames(nodes, z, 4)
    def by_torch(assign, L, *tables):
        rows = torch.sort(assign.to(torch.int64), stable=True).indices
        return [rows] + [t[rows] for t in tables]
    monkeypatch.setattr(hierarchy, "_by_leaf", by_torch)
    want_path, want_top = hierarchy.closest_frames(nodes, z, 4)
    assert np.array_equal(path, want_path) and top == want_top


def test_gradients_that_arrive_as_negated_views(layers):
    """Re(conj(i t) k) = t Im(k): the gradient of t is the imaginary part of a conjugate, whose memory has the other sign.
    Where it has a row's layout already, no copy makes it plain."""
    x, w = gpu(rand((7, 8), torch.float32, 1)).requires_grad_(True), gpu(rand((1, 8), torch.float32, 2)).requires_grad_(True)
    phi, rows = torch.rand((1, 4), device="cuda").requires_grad_(True), gpu(rand((7, 1), torch.float32, 3)).requires_grad_(True)
    plan, c = layers.sort_by_leaf(torch.arange(7, dtype=torch.int32, device="cuda"), 7), torch.complex(*(gpu(rand((7, 1), torch.float32, s)) for s in (4, 5)))
    one = torch.rand((7, 1), device="cuda")
    seen = []
    def conjugate(t):
        t.register_hook(lambda g: seen.append(g.is_neg()))
        return torch.complex(torch.zeros_like(t), t).conj()
    for call, leaves, k in ((lambda: layers.dense(x, w, activation="tanh"), [x, w], c), (lambda: layers.dense(x, w), [x, w], c),
                            (lambda: layers.top_leaves(phi, 1, renormalize=False)[1], [phi], c[:1]),
                            (lambda: layers.dispatch(rows, plan), [rows], c), (lambda: layers.combine(rows, plan), [rows], c),
                            (lambda: layers.combine(rows, plan, one), [rows], c)):
        got = torch.autograd.grad((conjugate(call()) * k).real.sum(), leaves)
        want = torch.autograd.grad((call() * k.imag).sum(), leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(seen)


def test_tensors_without_memory_are_errors(layers):
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w = gpu(rand((6, 8), torch.float32, 1)), gpu(rand((5, 8), torch.float32, 2))
    leaf = torch.zeros(6, dtype=torch.int32, device="cuda")
    plan = layers.sort_by_leaf(leaf, 1)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fx, fw, fleaf = (mode.from_tensor(t) for t in (x, w, leaf))
        for call in (lambda: layers.dense(fx, fw), lambda: layers.dense(x, w), lambda: layers.dispatch(fx, plan), lambda: layers.combine(fx, plan),
                     lambda: layers.top_leaves(fx, 2), lambda: layers.sort_by_leaf(fleaf, 1)):
            with pytest.raises(RuntimeError):
                call()
