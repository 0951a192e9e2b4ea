"""How exact the 16-bit layers are where 16 bits could cost more than the one rounding of each result, against the
formulas in 64 bits.

u = half a step of the element type (bf16 2^-8, fp16 2^-11), relative to a value.  Activations and their derivatives are
computed in fp32 with the hardware's exp2 and reciprocal: an argument of exp2 of magnitude A is off by 2^-24 A times two
roundings, so a derivative that is 2^-A is off by at most 2^-23 A + 2^-20 of itself, below 2^-15 for all A up to 150."""
import math

import pytest
import torch

from test_gpu_layers import HALF, TINY, TYPES, act64, gpu, rand, within

pytestmark = pytest.mark.gpu

# dz = dy act'(z) is held in two 16-bit parts: off by 2^-16 of itself in bf16 and 2^-22 in fp16, and where the second part
# is as small as the type's smallest step by half of that.
PARTS = {torch.bfloat16: (2.0 ** -16, 2.0 ** -134), torch.float16: (2.0 ** -22, 2.0 ** -25)}


@pytest.fixture(scope="module")
def layers():
    from bnp_vae_amd import layers as module
    return module


# ------------------------------------------------------------------------------------------------ derivatives far out
@pytest.mark.parametrize("act,most", [("softsign", 3e4), ("tanh", 40.0), ("silu", 80.0)])
@pytest.mark.parametrize("M", [8, 96])
def test_small_derivatives_keep_their_bits(layers, act, most, M):
    """bf16 holds the derivative far from 0 (softsign' is 1e-8 at 1e4), so the gradient has it too: relative to itself,
    not to 1.  z = x[:, 0] exactly, dx[:, 0] = dy act'(z), rounded to 16 bits where it is dz and where it is dx."""
    T = torch.bfloat16
    z = (torch.linspace(1.0, math.log2(most), M) ** 2 / math.log2(most)).exp2().to(T)
    z[::2] = -z[::2]
    if act == "silu":
        z = -z.abs()                              # towards + infinity its derivative is 1
    x = torch.zeros((M, 16), dtype=T)
    x[:, 0] = z
    w = torch.zeros((8, 16), dtype=T)
    w[0, 0] = 1
    X = gpu(x).requires_grad_(True)
    y = layers.dense(X, gpu(w), activation=act)
    dy = torch.zeros((M, 8), dtype=T)
    dy[:, 0] = rand((M,), T, 3)
    dx, = torch.autograd.grad(y, X, gpu(dy))
    want = dy[:, 0].double() * act64(act, z.double())[1]
    within(dx[:, 0], want, (2 * 2.0 ** -8 + 2.0 ** -14) * want.abs() + TINY[T])


@pytest.mark.parametrize("dtype,most", [("bf16", 13.0), ("f16", 5.5)])
@pytest.mark.parametrize("M", [8, 160])
def test_the_tail_of_gelu(layers, dtype, most, M):
    """gelu(z) and its derivative for negative z, relative to themselves: one rounding, and 2^-14 for the distribution
    function (2^-20) and exp2 (2^-15).  A result below the type's normal range is off by half of
    its smallest step."""
    T = TYPES[dtype]
    z = -torch.linspace(0.25, most, M).to(T)
    x, w = torch.zeros((M, 16), dtype=T), torch.zeros((8, 16), dtype=T)
    x[:, 0], w[0, 0] = z, 1
    X = gpu(x).requires_grad_(True)
    y = layers.dense(X, gpu(w), activation="gelu")
    dy = torch.zeros((M, 8), dtype=T)
    dy[:, 0] = 1
    dx, = torch.autograd.grad(y, X, gpu(dy))
    value, slope = act64("gelu", z.double())
    within(y[:, 0], value, (HALF[T] + 2.0 ** -14) * value.abs() + TINY[T] / 2, "y")
    # the slope passes 0 at z = -0.75: relative to its two terms there
    terms = 0.5 * torch.erfc(-z.double() / math.sqrt(2)) + z.double().abs() * torch.exp(-z.double() ** 2 / 2) / math.sqrt(2 * math.pi)
    within(dx[:, 0], slope, HALF[T] * slope.abs() + 2.0 ** -14 * terms + PARTS[T][0] * slope.abs() + TINY[T] / 2, "dx")


# ------------------------------------------------------------------------------------------------ dz in 16 bits


def quarters(shape, seed):
    """Multiples of 1/4 between -1 and 1: sums of their products are exact in fp32, so z is too."""
    return torch.randint(-4, 5, shape, generator=torch.Generator().manual_seed(seed)).double() / 4


def gradients(x, w, b, act, dy, bounds):
    """dx, dw, db in 64 bits and the bounds of their errors where z is exact; w (G, n, K)."""
    T, (M, K), (G, n, _) = dy.dtype, x.shape, w.shape
    u, t, (part, least) = HALF[T], TINY[T], PARTS[T]
    out = {k: [torch.zeros(s, dtype=torch.float64) for _ in range(2)] for k, s in (("dx", (M, K)), ("dw", (G, n, K)), ("db", (G, n)))}
    for g in range(G):
        rows = slice(bounds[g], bounds[g + 1])
        m, xg, wg, dyg = bounds[g + 1] - bounds[g], x[rows].double(), w[g].double(), dy[rows].double()
        dz = dyg * act64(act, xg @ wg.t() + b[g].double())[1]
        raw = 16 * 2.0 ** -24 * dyg.abs() + 2.0 ** -23 * dz.abs()
        off = raw + part * (dz.abs() + raw) + least
        for name, at, value, e, size, terms in (
                ("dx", rows, dz @ wg, off @ wg.abs(), (dz.abs() + off) @ wg.abs(), n),
                ("dw", g, dz.t() @ xg, off.t() @ xg.abs(), (dz.abs() + off).t() @ xg.abs(), m),
                ("db", g, dz.sum(0), raw.sum(0), (dz.abs() + raw).sum(0), m)):
            e = e + (2 * terms + 16) * 2.0 ** -23 * size          # both parts are added up
            out[name][0][at], out[name][1][at] = value, e + u * (value.abs() + e) + t
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["softsign", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("M,K,n,sizes", [(40, 24, 40, None), (33, 25, 37, None), (150, 24, 24, None), (130, 200, 33, None), (9, 70, 130, None),
                                         (90, 24, 40, [30, 0, 41, 3]), (70, 25, 31, [1, 33, 30])])
def test_gradients_are_rounded_once(layers, dtype, act, M, K, n, sizes):
    T = TYPES[dtype]
    G = 1 if sizes is None else len(sizes)
    bounds = [0, M] if sizes is None else [sum(sizes[:g]) for g in range(G + 1)]
    thin = 1 if K < 100 else 1 / 4                    # z of a few units
    x, w, b = quarters((M, K), 1).to(T), (quarters((G, n, K), 2) * thin).to(T), quarters((G, n), 3).to(T)
    dy = rand((M, n), T, 4)
    want = gradients(x, w, b, act, dy, bounds)
    leaves = [gpu(t).requires_grad_(True) for t in (x, w if sizes else w[0], b if sizes else b[0])]
    off = None if sizes is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    y = layers.dense(*leaves, activation=act, offsets=off)
    for name, got in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, gpu(dy))):
        value, bound = want[name]
        if sizes is None and name != "dx":
            value, bound = value[0], bound[0]
        within(got, value, bound, name)


def test_a_gradient_behind_the_largest_fp16_value(layers):
    """gelu' reaches 1.13, so dz can pass 65504 where dy does not: dx and dW are finite where their own sums are."""
    T = torch.float16
    for M in (4, 40):
        x, w = torch.zeros((M, 16), dtype=T), torch.zeros((8, 16), dtype=T)
        x[:, 0], x[:, 2], w[0, 0], w[0, 1] = 1.5, 2.0 ** -9, 1.0, 0.0625          # z = 1.5
        dy = torch.zeros((M, 8), dtype=T)
        dy[:, 0] = torch.tensor([60000.0, -64000.0]).repeat(M // 2)
        dy[0, 0] = 65504
        X, W = gpu(x).requires_grad_(True), gpu(w).requires_grad_(True)
        dx, dw = torch.autograd.grad(layers.dense(X, W, activation="gelu"), [X, W], gpu(dy))
        dz = dy[:, 0].double() * act64("gelu", torch.tensor(1.5, dtype=torch.float64))[1]
        assert float(dz.abs().max()) > 65504
        within(dx[:, 1], dz / 16, (2.0 ** -11 + 2.0 ** -18) * dz.abs() / 16)
        total = float(dz.sum()) * 2.0 ** -9
        within(dw[0, 2], torch.tensor(total, dtype=torch.float64), 2.0 ** -11 * abs(total) + 2.0 ** -18 * float(dz.abs().sum()) * 2.0 ** -9)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_infinities_in_a_gradient(layers, dtype):
    """An infinity or NaN of dy reaches dx and dW as the formula has it: infinite, not NaN, where one infinity is added up."""
    T = TYPES[dtype]
    x, w = torch.ones((40, 16), dtype=T), torch.full((8, 16), 2.0 ** -4, dtype=T)
    dy = torch.zeros((40, 8), dtype=T)
    dy[3, 2], dy[5, 1], dy[6, 0] = float("inf"), -float("inf"), float("nan")
    X, W = gpu(x).requires_grad_(True), gpu(w).requires_grad_(True)
    dx, dw = (t.cpu() for t in torch.autograd.grad(layers.dense(X, W, activation="silu"), [X, W], gpu(dy)))
    assert (dx[3] == float("inf")).all() and (dx[5] == -float("inf")).all() and torch.isnan(dx[6]).all()
    assert (dw[2] == float("inf")).all() and (dw[1] == -float("inf")).all() and torch.isnan(dw[0]).all()
    dx[[3, 5, 6]], dw[:3] = 0, 0
    assert (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,K,n,sizes", [(5000, 1032, 520, None), (3001, 600, 777, None), (20000, 512, 264, [3000, 0, 9000, 1, 7900]),
                                         (2000, 130, 300, [7] * 200), (40000, 1024, 1024, None), (3000, 2048, 4096, None),
                                         (60000, 512, 768, [30000, 0, 17, 9000, 20950]), (84650, 86, 41, [8465] * 10),
                                         (5122, 1574, 89, [197] * 26)])
def test_large_gradients_are_as_near_as_one_rounding(layers, dtype, M, K, n, sizes):
    """Every element is off by what rounding the exact value would cost plus at most twice the error in front of the
    rounding, and that is below 2^-15 of a value's size (z and the sums in fp32, dz in two parts), a fortieth of bf16's
    0.0017.  fp16's own rounding is eight times finer, and so is its dz."""
    T = TYPES[dtype]
    G = 1 if sizes is None else len(sizes)
    bounds = [0, M] if sizes is None else [sum(sizes[:g]) for g in range(G + 1)]
    x, w, b = rand((M, K), T, 1), rand((G, n, K), T, 2, 1 / math.sqrt(K)), rand((G, n), T, 3)
    dy = rand((M, n), T, 4)
    leaves = [gpu(t).requires_grad_(True) for t in (x, w if sizes else w[0], b if sizes else b[0])]
    off = None if sizes is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    got = torch.autograd.grad(layers.dense(*leaves, activation="silu", offsets=off), leaves, gpu(dy))
    x, w, b, dy = (gpu(t).double() for t in (x, w, b, dy))
    want = [torch.zeros_like(t, dtype=torch.float64) for t in (x, w, b)]
    for g in range(G):
        rows = slice(bounds[g], bounds[g + 1])
        q = torch.sigmoid(x[rows] @ w[g].t() + b[g])
        z = x[rows] @ w[g].t() + b[g]
        dz = dy[rows] * (q + z * q * (1 - q))
        want[0][rows], want[1][g], want[2][g] = dz @ w[g], dz.t() @ x[rows], dz.sum(0)
    for name, a, e in zip(("dx", "dw", "db"), got, want):
        e = e.reshape(a.shape)
        best, off_by = float((e.to(T).double() - e).norm()), float((a.double() - e).norm())
        assert off_by <= 1.05 * best + 2.0 ** -24 * float(e.norm()), (name, off_by / best)
