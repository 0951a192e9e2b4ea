"""The dense product where every sum is a whole number that fp32 holds: nothing is rounded but the result, so values and
gradients have to have the bits of the exact ones, rounded once -- in every tile, with every way of loading, in split sums,
over workgroups that take many tiles, and in leaves of any length.  A row left out, taken twice or read too early shows."""
import math

import numpy as np
import pytest
import torch

from test_gpu_layers import HALF, TINY, TYPES, act64, gpu, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from bnp_vae_amd import layers as module
    return module


def whole(shape, most, T, seed, shift=0, pad=0):
    """Whole numbers between -most and most, in rows that start `shift` elements behind the first of a pitch `pad` wider."""
    g = torch.Generator("cuda").manual_seed(seed)
    t = torch.randint(-most, most + 1, shape[:-1] + (shape[-1] + pad,), generator=g, device="cuda").to(T)
    return t[..., shift:shift + shape[-1]].detach()


def check_exact(layers, M, K, n, T, act, bias=True, residual=True, sizes=None, shift=0, pad=0, head=0, seed=1):
    G = 0 if sizes is None else len(sizes)
    lead = (G,) if G else ()
    x, w = whole((M, K), 2, T, seed, shift, pad).requires_grad_(True), whole(lead + (n, K), 2, T, seed + 1, shift, pad).requires_grad_(True)
    b = whole(lead + (n,), 8, T, seed + 2).requires_grad_(True) if bias else None
    r = whole((M, n), 64, T, seed + 3, shift, pad).requires_grad_(True) if residual else None
    dy = whole((M, n), 2, T, seed + 4, shift, pad)
    bounds = [0, M] if sizes is None else [int(v) for v in head + np.concatenate([[0], np.cumsum(sizes)])]
    off = None if sizes is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    y = layers.dense(x, w, b, activation=act, residual=r, offsets=off)
    leaves = [t for t in (x, w, b, r) if t is not None]
    got = dict(zip([m for m, t in (("dx", x), ("dw", w), ("db", b), ("dr", r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    got["y"] = y.detach()
    with torch.no_grad():
        want = {"y": torch.zeros((M, n), dtype=T, device="cuda"), "dx": torch.zeros((M, K), dtype=T, device="cuda"),
                "dr": torch.zeros((M, n), dtype=T, device="cuda"), "dw": torch.zeros(w.shape, dtype=T, device="cuda"),
                "db": torch.zeros(w.shape[:-1], dtype=T, device="cuda")}
        for g in range(len(bounds) - 1):
            rows = slice(bounds[g], bounds[g + 1])
            at = g if G else slice(None)
            z = x[rows].double() @ (w[g] if G else w).double().t().contiguous()
            if bias:
                z += (b[g] if G else b).double()
            dz = dy[rows].double() * (z > 0 if act == "relu" else 1)
            z = z.clamp(min=0) if act == "relu" else z
            if residual:
                z += r[rows].double()
            want["y"][rows], want["dr"][rows] = z.to(T), dy[rows]
            want["dx"][rows] = (dz @ (w[g] if G else w).double()).to(T)
            dw, db = dz.t().contiguous() @ x[rows].double(), dz.sum(0)
            assert float(dw.abs().max() if dw.numel() else 0) < 2 ** 24 and float(db.abs().max()) < 2 ** 24
            want["dw"][at], want["db"][at] = dw.to(T), db.to(T)
    for name, value in got.items():
        assert torch.equal(value, want[name]), "%s: %d of %d values off" % (name, int((value != want[name]).sum()), value.numel())


SHAPES = [
    (40000, 1024, 1024), (20000, 4096, 256), (9000, 512, 4104), (33000, 200, 264), (16384, 512, 512), (5000, 264, 520),     # tiles of 256, 128, 64
    (300, 8192, 512), (31, 4096, 2048), (513, 70000, 40),                                 # few rows, long sums in parts
    (70000, 64, 32), (90000, 24, 64), (50000, 1024, 32),                                  # narrow on either side
    (5, 4096, 3000), (8, 1031, 77), (1, 4096, 32),                                        # products with vectors
    (7000, 2001, 601), (32768, 1023, 1021), (600, 37, 41), (70000, 63, 31), (70000, 31, 63),     # rows off 16 bytes, copied and not
    (68278, 367, 254), (6141, 1067, 536), (20919, 1916, 5)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("M,K,n", SHAPES)
def test_dense_is_exact(layers, dtype, act, M, K, n):
    check_exact(layers, M, K, n, TYPES[dtype], act)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_dense_without_some_inputs_is_exact(layers, dtype, bias, residual):
    for act in (None, "relu"):
        check_exact(layers, 30000, 768, 512, TYPES[dtype], act, bias, residual)
        check_exact(layers, 30000, 256, 512, TYPES[dtype], act, bias, residual, sizes=[9000, 0, 12000, 8999])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("shift,pad", [(0, 8), (8, 24), (1, 3), (3, 16)])
def test_dense_of_views_is_exact(layers, dtype, act, shift, pad):
    check_exact(layers, 12000, 600, 520, TYPES[dtype], act, shift=shift, pad=pad)
    check_exact(layers, 12000, 333, 264, TYPES[dtype], act, shift=shift, pad=pad, sizes=[100, 7000, 0, 1, 4800])
    check_exact(layers, 200, 40, 48, TYPES[dtype], act, shift=shift, pad=pad, sizes=[60, 0, 129])


def some_sizes(count, total, seed, least=0):
    share = np.random.default_rng(seed).gamma(0.5, size=count)
    return [least + int(v) for v in share / share.sum() * (total - count * least)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("sizes,K,n", [
    ([40000, 0, 9000, 1, 10990], 512, 512), (some_sizes(64, 60000, 1), 512, 512), (some_sizes(12, 60000, 2), 1024, 256),
    ([200] * 256, 512, 512), (some_sizes(500, 20000, 3), 200, 136), (some_sizes(3000, 15000, 4), 64, 96), ([6] * 512, 250, 130),
    (some_sizes(5, 20000, 5), 301, 203), (some_sizes(8, 50000, 6), 32, 520), (some_sizes(8, 50000, 7), 520, 24), ([1] * 700, 40, 33),
    (some_sizes(200, 6000, 8), 257, 259), (some_sizes(3, 30000, 9), 31, 63),
    (some_sizes(26, 5052, 10), 1574, 89), (some_sizes(108, 200, 11), 472, 237), (some_sizes(162, 300, 12), 939, 1114), (some_sizes(10, 84653, 13), 86, 41)])
def test_dense_per_leaf_is_exact(layers, dtype, act, sizes, K, n):
    check_exact(layers, sum(sizes) + 77 + 5, K, n, TYPES[dtype], act, sizes=sizes, head=5)


def test_dense_past_32_bits_is_exact(layers):
    """4.5 GB of x: all of y and dW, and dx of 8 GB, from whole numbers."""
    check_exact(layers, 1100003, 2048, 32, torch.bfloat16, None, residual=False)
    check_exact(layers, 1100003, 2048, 32, torch.bfloat16, "relu", residual=False, sizes=[5, 600000, 0, 499998])


# ------------------------------------------------------------------------------------------------ the smallest values
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M", [1, 4, 8, 40, 700])
def test_subnormal_operands_count(layers, dtype, M):
    """x, and then dy, below the type's normal range: multiples of its smallest step, which large weights bring back.  The
    sums are exact, so a flushed operand shows whole."""
    T = TYPES[dtype]
    step, up = TINY[T], 2.0 ** (10 if T is torch.float16 else 120)
    K, n = 64, 48
    x = (whole((M, K), 40, torch.float64, 1) * step).to(T)
    w = (whole((n, K), 3, torch.float64, 2) * up).to(T)
    assert float(x.abs().max()) < 64 * step and float(x.double().abs().max()) > 0
    z = x.double() @ w.double().t().contiguous()
    y = layers.dense(x, w)
    assert torch.equal(y, z.to(T))
    X, W = x.requires_grad_(True), w.requires_grad_(True)
    B = torch.zeros(n, dtype=T, device="cuda", requires_grad=True)
    dy = (whole((M, n), 40, torch.float64, 3) * step).to(T)
    for act in (None, "relu"):
        # with an activation z has to be finite, so one of its factors is of order 1, and dW below the normal range too
        x1 = (whole((M, K), 3, torch.float64, 4) * (1 if act else up)).to(T).requires_grad_(True)
        y = layers.dense(x1, W, B, activation=act)
        dx, dw, db = torch.autograd.grad(y, [x1, W, B], dy)
        with torch.no_grad():
            dz = dy.double() * ((x1.double() @ W.double().t().contiguous()) > 0 if act else 1)
            assert torch.equal(dx, (dz @ W.double()).to(T)), act
            assert torch.equal(dw, (dz.t().contiguous() @ x1.double()).to(T)), act
            assert torch.equal(db, dz.sum(0).to(T)), act
    with torch.no_grad():
        small = (whole((M, K), 40, torch.float64, 5) * 2.0 ** -142).float()          # fp32's own
        assert torch.equal(layers.dense(small, w.double().sign().float() * 2.0 ** 100), (small.double() @ (w.double().sign() * 2.0 ** 100).t().contiguous()).float())


# ------------------------------------------------------------------------------------------------ differences
@pytest.mark.parametrize("act", ["softsign", "tanh", "silu", "gelu"])
def test_dense_gradients_against_differences(layers, act):
    """Central differences of sum(c y) in 64 bits in every entry of x, W and b: off by h^2 / 6 times the third derivative
    along the entry, which is |c| |d|^3 times at most 6 (softsign; its kink at 0 is kept out: |z| > 0.5), with d the entry's
    factor in z; the kernel's gradient by its fp32 sums and activations."""
    x, w = rand((4, 6), torch.float32, 1, 0.3).clamp(-0.7, 0.7), rand((5, 6), torch.float32, 2, 0.3).clamp(-0.7, 0.7)
    b, c = torch.tensor([4.0, -4.0, 3.9, -3.6, 3.5]), rand((4, 5), torch.float32, 7)
    v = [t.double() for t in (x, w, b)]
    z = v[0] @ v[1].t() + v[2]
    assert float(z.abs().min()) > 0.5
    X, W, B = (gpu(t).requires_grad_(True) for t in (x, w, b))
    grads = torch.autograd.grad(layers.dense(X, W, B, activation=act), [X, W, B], gpu(c))
    h = 2.0 ** -10
    def value(p):
        return float((c.double() * act64(act, p[0] @ p[1].t() + p[2])[0]).sum())
    for i, g in enumerate(grads):
        for j in range(v[i].numel()):
            up, down = [t.clone() for t in v], [t.clone() for t in v]
            up[i].view(-1)[j] += h
            down[i].view(-1)[j] -= h
            slope = (value(up) - value(down)) / (2 * h)
            if i == 0:
                reach, row = v[1][:, j % 6].abs(), c[j // 6].double().abs()
            elif i == 1:
                reach, row = v[0][:, j % 6].abs(), c[:, j // 6].double().abs()
            else:
                reach, row = torch.ones(4, dtype=torch.float64), c[:, j].double().abs()
            # act' to 16 half steps beside 1 and 2 |act''| <= 4 times z's own error, sums of at most 6 terms
            kernel = float((row * reach).sum()) * (16 * 2.0 ** -24 + 4 * 22 * 2.0 ** -23 * 8 + 22 * 2.0 ** -23)
            assert abs(slope - float(g.view(-1)[j].cpu())) <= float((row * reach ** 3).sum()) * h * h + kernel


# ------------------------------------------------------------------------------------------------ the C entry points
def backward(layers, activation, dtype, dy, dact, x, w, offsets, G):
    """bnpvi_dense_backward, or with an activation bnpvi_dense_backward_act: dx, dw, db."""
    import ctypes as C
    lib, p = layers.lib, lambda t: None if t is None else C.c_void_p(t.data_ptr())
    (M, K), n = x.shape, w.shape[-2]
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(w.shape[:-1], dtype=x.dtype, device="cuda")
    need = lib.bnpvi_dense_workspace(dtype, M, K, n, G, 1)
    work = torch.full((need,), 0x7f, dtype=torch.uint8, device="cuda")
    args = [p(dy), n, p(dact), n, p(x), K, p(w), K, n * K, p(offsets), G, M, K, n, p(dx), K, p(dw), p(db), None, 0, p(work), need,
            C.c_void_p(torch.cuda.current_stream().cuda_stream)]
    ctx = C.c_void_p(layers._ctx(x.device))
    if activation is None:
        rc = lib.bnpvi_dense_backward(ctx, dtype, *args)
    else:
        rc = lib.bnpvi_dense_backward_act(ctx, dtype, activation, *args)
    assert rc == 0, lib.bnpvi_last_error()
    return dx, dw, db


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,K,n,sizes", [
    (40000, 1024, 1024, None), (20000, 4096, 256, None), (16384, 512, 512, None), (5000, 264, 520, None), (300, 2048, 512, None),
    (40, 24, 33, None), (70000, 64, 32, None), (7000, 1001, 601, None), (600, 37, 41, None), (31, 1024, 70, None),
    (60000, 512, 512, [40000, 0, 9000, 1, 10990]), (60000, 512, 512, some_sizes(64, 60000, 1)), (51200, 512, 512, [200] * 256),
    (15000, 64, 96, some_sizes(3000, 15000, 4)), (20000, 301, 203, some_sizes(5, 20000, 5)), (5052, 1574, 89, some_sizes(26, 5052, 10)),
    (20000, 86, 41, some_sizes(10, 20000, 13))])
def test_both_parts_of_dz_are_exact(layers, dtype, M, K, n, sizes):
    """act'(z) given as multiples of 2^-8 up to 16, so that dz needs 12 bits: two parts hold it, one does not; all sums are
    below 2^24 of these steps.  What a forward pass would give is no matter here."""
    T, code = TYPES[dtype], {"bf16": 1, "f16": 2}[dtype]
    lead = (len(sizes),) if sizes else ()
    x, w, dy = whole((M, K), 1, T, 1), whole(lead + (n, K), 1, T, 2), whole((M, n), 2, T, 3)
    x, w = x * (whole((M, K), 3, T, 4) == 0), w * (whole(lead + (n, K), 3, T, 5) == 0)          # mostly zeros: shorter sums
    dact = whole((M, n), 4095, torch.float32, 6) / 256
    bounds = [0, M] if sizes is None else [int(v) for v in np.concatenate([[0], np.cumsum(sizes)])]
    off = torch.tensor(bounds, dtype=torch.int32, device="cuda") if sizes else None
    dx, dw, db = backward(layers, None, code, dy, dact, x, w, off, len(sizes or ()))
    dz = dy.double() * dact.double()
    assert float((dz.to(T).double() != dz).double().mean()) > 0.01
    for g in range(len(bounds) - 1):
        rows, at = slice(bounds[g], bounds[g + 1]), g if sizes else slice(None)
        for name, got, want in (("dx", dx[rows], dz[rows] @ w[at].double()), ("dw", dw[at], dz[rows].t().contiguous() @ x[rows].double()),
                                ("db", db[at], dz[rows].sum(0))):
            assert float(want.abs().max() if want.numel() else 0) < 2 ** 16, name
            assert torch.equal(got, want.to(T)), (name, g, int((got != want.to(T)).sum()))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("sizes", [None, [70, 0, 400, 29]])
def test_a_named_activation_changes_no_bit(layers, dtype, sizes):
    """relu's dz has the bits of dy, with and without a second part; other activations go the same way named or not."""
    T = (torch.float32, torch.bfloat16, torch.float16)[dtype]
    M, K, n, G = 500, 72, 136, len(sizes or ())
    lead = (G,) if G else ()
    x, w, dy = whole((M, K), 2, T, 1), whole(lead + (n, K), 2, T, 2), whole((M, n), 2, T, 3)
    off = None if sizes is None else torch.tensor([0] + [int(v) for v in np.cumsum(sizes)], dtype=torch.int32, device="cuda")
    for activation, dact in ((1, whole((M, n), 1, torch.float32, 4).abs()), (5, torch.rand((M, n), device="cuda")), (-1, None)):
        for a, b in zip(backward(layers, None, dtype, dy, dact, x, w, off, G), backward(layers, activation, dtype, dy, dact, x, w, off, G)):
            rows = slice(0, sum(sizes)) if sizes and a.shape[0] == M else slice(None)
            assert torch.equal(a[rows], b[rows])
