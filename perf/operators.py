"""Cases of the layer operators that follow the tree: the leaves that matter for a frame (`top`), rows sorted by
leaf and back with their weights (`exchange`), and the dense product with bias, activation and residual, with one
weight for all rows or one per leaf (`dense`).

`run` computes a case in elementary torch operations in 32 bits, or, where `own` is set, through
`bnp_vae_amd.layers`.  `exact` computes the same from the definitions in 64 bits."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEVICE = "cuda"


def _layers():
    from bnp_vae_amd import layers
    return layers


# ------------------------------------------------------------------------------------------------ cases
def _top(N, L, k, train, renorm=True):
    return {"op": "top", "N": N, "L": L, "k": k, "train": train, "renorm": renorm}


def _exchange(N, D, L, k, dtype, train):
    return {"op": "exchange", "N": N, "D": D, "L": L, "k": k, "dtype": dtype, "train": train}


def _dense(M, K, n, dtype, act, train, bias=True, residual=False, G=0):
    return {"op": "dense", "M": M, "K": K, "n": n, "dtype": dtype, "act": act, "train": train, "bias": bias,
            "residual": residual, "G": G}


def listed():
    return [
        # one frame asked for its two likeliest leaves while a prediction is served: latency
        dict(_top(1, 64, 2, False), name="top, one frame"),
        # every frame of a one-million-frame training set, the tree of 8 x 8 leaves, weights learnt through
        dict(_top(1000000, 64, 2, True), name="top, 1M frames, 64 leaves"),
        # an evaluation pass over a tree of 512 leaves
        dict(_top(150001, 512, 4, False), name="top, 150k frames, 512 leaves"),
        # a training minibatch of latents on the 5 x 5 tree: latency of the five calls
        dict(_exchange(500, 32, 25, 1, "f32", True), name="exchange, minibatch of 500"),
        # activations of a large training batch, two leaves a frame
        dict(_exchange(262144, 256, 64, 2, "bf16", True), name="exchange, 262k x 256 bf16"),
        # an evaluation pass over the largest tree (6^5 leaves) with rows of an odd width
        dict(_exchange(300001, 100, 7776, 3, "f32", False), name="exchange, 300k x 100, 7776 leaves"),
        # one frame's fc features to its latent code: latency
        dict(_dense(1, 4096, 32, "f32", "softsign", False), name="dense, one frame 4096 to 32"),
        # training the encoder on a large batch of fc features
        dict(_dense(65536, 4096, 256, "bf16", "softsign", True), name="dense, encoder 4096 to 256 bf16"),
        # training the decoder in the latents' own type, an odd batch
        dict(_dense(16385, 64, 4096, "f32", "none", True), name="dense, decoder 64 to 4096 f32"),
        # a hidden block with its skip connection
        dict(_dense(32768, 1024, 1024, "bf16", "gelu", True, residual=True), name="dense, residual block bf16"),
        # every leaf's own layer on the frames sorted to it, in training
        dict(_dense(131072, 512, 512, "bf16", "silu", True, G=64), name="dense, 64 leaves bf16"),
        # a served batch over 512 leaves, few rows each, odd sizes
        dict(_dense(3000, 250, 130, "f16", "relu", False, residual=True, G=512), name="dense, 512 leaves f16"),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of its range; about half of them odd."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["top", "exchange", "dense", "dense", "leaves"])
    if op == "top":
        L = _spread(rng, 2, 7776)
        N = _spread(rng, 1, max(1, min(1000000, 64000000 // max(L, 64))))
        return _top(N, L, rng.randint(1, min(8, L)), rng.random() < 0.5, rng.random() < 0.7)
    if op == "exchange":
        dtype, k = rng.choice(["f32", "bf16", "f16"]), rng.randint(1, 4)
        D = _spread(rng, 1, 1024)
        N = _spread(rng, 4, max(4, min(262144, 64000000 // (D * k))))
        return _exchange(N, D, _spread(rng, 1, 7776), k, dtype, rng.random() < 0.5)
    dtype = rng.choice(["f32", "bf16", "f16"])
    act = rng.choice(["none", "relu", "softsign", "tanh", "silu", "gelu"])
    K, n = _spread(rng, 8, 4096), _spread(rng, 8, 4096)
    train, bias, residual = rng.random() < 0.5, rng.random() < 0.8, rng.random() < 0.5
    if op == "dense":
        M = _spread(rng, 1, max(1, min(65536, int(3.0e10 / (K * n)), int(1.0e8 / max(K, n)))))
        return _dense(M, K, n, dtype, act, train, bias, residual)
    K, n = min(K, 1024), min(n, 1024)
    G = _spread(rng, 2, max(2, min(512, int(3.0e7 / (K * n)))))
    M = _spread(rng, 4, max(4, min(65536, int(1.0e10 / (K * n)), int(2.0e7 / max(K, n)))))
    return _dense(M, K, n, dtype, act, train, bias, residual, G)


def _padded(L):
    return (L + 31) // 32 * 32


def work(case):
    if case["op"] == "top":
        N, L, k = case["N"], case["L"], case["k"]
        b = 4.0 * N * L + 8.0 * N * k
        if case["train"]:
            b += 4.0 * N * k + 4.0 * N * _padded(L)
        return {"bytes": b, "flops": 1.0 * N * L}
    if case["op"] == "exchange":
        N, D, L, k = case["N"], case["D"], case["L"], case["k"]
        e, M = TYPES[case["dtype"]].itemsize, N * k
        b = 12.0 * M + 4.0 * (L + 1) + e * D * (2.0 * N + 2.0 * M) + 4.0 * M
        f = 2.0 * M * D
        if case["train"]:
            b += e * D * (2.0 * N + 2.0 * M) + 4.0 * M
            f += 4.0 * M * D
        return {"bytes": b, "flops": f}
    M, K, n, G = case["M"], case["K"], case["n"], max(1, case["G"])
    e = TYPES[case["dtype"]].itemsize
    b = e * (1.0 * M * K + G * n * K + M * n * (1 + case["residual"]) + G * n * case["bias"])
    f = 2.0 * M * n * K
    if case["train"]:
        b += e * (1.0 * M * n + M * K + G * n * K + G * n * case["bias"])
        f *= 3
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------ inputs
def _shares(L, g):
    """Shares of the leaves of a learnt tree: unequal, none of them a single one's."""
    return torch.softmax(0.7 * torch.randn(L, generator=g, device=DEVICE), 0)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    s = dict(case)
    if case["op"] == "top":
        N, L, k = case["N"], case["L"], case["k"]
        # responsibilities: a softmax over the leaves, many of them so far away that they underflow to 0; the columns
        # behind the last leaf hold 0, as an E-step leaves them
        phi = torch.zeros((N, _padded(L)), device=DEVICE)
        phi[:, :L] = torch.softmax(normal(N, L).mul_(20.0), 1)
        s["phi"] = phi.requires_grad_(case["train"])
        if case["train"]:
            s["dweight"] = normal(N, k)
        return s
    T = TYPES[case["dtype"]]
    if case["op"] == "exchange":
        N, D, L, k = case["N"], case["D"], case["L"], case["k"]
        # leaves by their shares; a few frames have fewer than k leaves
        leaf = torch.multinomial(_shares(L, g), N * k, replacement=True, generator=g).view(N, k).to(torch.int32)
        leaf[torch.rand((N, k), generator=g, device=DEVICE) < 0.03] = -1
        weight = torch.rand((N, k), generator=g, device=DEVICE) + 0.05
        s["leaf"] = leaf
        s["weight"] = (weight / weight.sum(1, keepdim=True)).requires_grad_(case["train"])
        s["x"] = normal(N, D).to(T).requires_grad_(case["train"])
        s["ys"] = normal(N * k, D).to(T).requires_grad_(case["train"])
        if case["train"]:
            s["dy"] = normal(N, D).to(T)
            s["dxs"] = normal(N * k, D).to(T)
        return s
    M, K, n, G = case["M"], case["K"], case["n"], case["G"]
    lead = (G,) if G else ()
    s["x"] = normal(M, K).to(T).requires_grad_(case["train"])
    s["w"] = (normal(*lead, n, K) / math.sqrt(K)).to(T).requires_grad_(case["train"])
    s["b"] = normal(*lead, n).mul_(0.5).to(T).requires_grad_(case["train"]) if case["bias"] else None
    s["r"] = normal(M, n).to(T).requires_grad_(case["train"]) if case["residual"] else None
    s["dy"] = normal(M, n).to(T) if case["train"] else None
    s["offsets"] = None
    if G:
        # rows per leaf by the shares; the last few rows of the batch belong to no leaf
        leaf = torch.multinomial(_shares(G, g), M, replacement=True, generator=g)
        leaf = leaf[torch.rand(M, generator=g, device=DEVICE) > 0.02]
        counts = torch.bincount(leaf, minlength=G)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"] = max(1, int(counts.max()))
    return s


# ------------------------------------------------------------------------------------------------ the passes
def run(s):
    if own:
        return {"top": _own_top, "exchange": _own_exchange, "dense": _own_dense}[s["op"]](s)
    with torch.no_grad():
        return {"top": _plain_top, "exchange": _plain_exchange, "dense": _plain_dense}[s["op"]](s)


def _own_top(s):
    leaf, weight = _layers().top_leaves(s["phi"], s["k"], num_leaves=s["L"], renormalize=s["renorm"])
    out = {"leaf": leaf, "weight": weight}
    if s["train"]:
        out["dphi"], = torch.autograd.grad(weight, s["phi"], s["dweight"])
    return out


def _plain_top(s):
    phi, L, k = s["phi"], s["L"], s["k"]
    p = phi[:, :L]
    p = torch.where((p > 0) & (p < math.inf), p, 0.0)
    column = torch.arange(L, device=p.device)
    leaf, weight = [], []
    for _ in range(k):
        m = p.max(1, keepdim=True).values
        at = torch.where(p == m, column, L).min(1, keepdim=True).values
        weight.append(m)
        leaf.append(torch.where(m > 0, at, -1))
        p = p.scatter(1, at, 0.0)
    leaf, weight = torch.cat(leaf, 1), torch.cat(weight, 1)
    total = weight.sum(1, keepdim=True)
    if s["renorm"]:
        weight = torch.where(total > 0, weight / total, 0.0)
    out = {"leaf": leaf.to(torch.int32), "weight": weight}
    if s["train"]:
        d = s["dweight"]
        if s["renorm"]:
            d = torch.where(total > 0, (d - (d * weight).sum(1, keepdim=True)) / total, 0.0)
        d = torch.where(leaf >= 0, d, 0.0)
        out["dphi"] = torch.zeros_like(phi).scatter_add_(1, leaf.clamp(min=0), d)
    return out


def _own_exchange(s):
    layers = _layers()
    plan = layers.sort_by_leaf(s["leaf"], s["L"])
    xs = layers.dispatch(s["x"], plan)
    y = layers.combine(s["ys"], plan, s["weight"])
    out = {"place": plan.place, "order": plan.order, "offsets": plan.offsets, "xs": xs, "y": y}
    if s["train"]:
        out["dx"], out["dys"], out["dweight"] = torch.autograd.grad(
            [xs, y], [s["x"], s["ys"], s["weight"]], [s["dxs"], s["dy"]])
    return out


def _plain_exchange(s):
    leaf, x, ys, w = s["leaf"], s["x"].float(), s["ys"].float(), s["weight"]
    N, k, L, T = s["N"], s["k"], s["L"], s["x"].dtype
    key = leaf.reshape(-1).to(torch.int64)
    kept = (key >= 0) & (key < L)
    key = torch.where(kept, key, L)
    by_leaf = torch.sort(key, stable=True)
    order = by_leaf.indices
    place = torch.empty_like(order)
    place[order] = torch.arange(N * k, device=order.device)
    offsets = torch.searchsorted(by_leaf.values, torch.arange(L + 1, device=order.device))
    real = (by_leaf.values < L)[:, None]
    xs = torch.where(real, x[order // k], 0.0)
    wk = torch.where(kept.view(N, k), w, 0.0)[:, :, None]
    rows = torch.where(kept.view(N, k, 1), ys[place].view(N, k, -1), 0.0)
    y = (wk * rows).sum(1)
    out = {"place": place.to(torch.int32).view(N, k), "order": order.to(torch.int32),
           "offsets": offsets.to(torch.int32), "xs": xs.to(T), "y": y.to(T)}
    if s["train"]:
        dy, dxs = s["dy"].float(), s["dxs"].float()
        out["dx"] = torch.where(kept.view(N, k, 1), dxs[place].view(N, k, -1), 0.0).sum(1).to(T)
        out["dys"] = torch.where(real, (dy[:, None] * wk).view(N * k, -1)[order], 0.0).to(T)
        out["dweight"] = (rows * dy[:, None]).sum(2)
    return out


def _own_dense(s):
    act = None if s["act"] == "none" else s["act"]
    y = _layers().dense(s["x"], s["w"], s["b"], activation=act, residual=s["r"], offsets=s["offsets"])
    out = {"y": y}
    if s["train"]:
        names = [m for m in ("x", "w", "b", "r") if s[m] is not None]
        out.update(zip(["d" + m for m in names], torch.autograd.grad(y, [s[m] for m in names], s["dy"])))
    return out


def _act(name, z):
    """act(z) and its derivative."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "softsign":
        q = 1 / (1 + z.abs())
        return z * q, q * q
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if name == "silu":
        q = torch.sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _plain_dense(s):
    x, w, T = s["x"].float(), s["w"].float(), s["x"].dtype
    M, G = s["M"], s["G"]
    if not G:
        z = x @ w.t()
        if s["b"] is not None:
            z = z + s["b"].float()
        a, d = _act(s["act"], z)
        out = {"y": (a if s["r"] is None else a + s["r"].float()).to(T)}
        if s["train"]:
            dz = s["dy"].float() * d
            out["dx"], out["dw"] = (dz @ w).to(T), (dz.t() @ x).to(T)
            if s["b"] is not None:
                out["db"] = dz.sum(0).to(T)
            if s["r"] is not None:
                out["dr"] = s["dy"]
        return out
    # one batch entry per leaf, as many rows as the fullest has; rows of no leaf go to a row behind them all
    row = torch.arange(M, device=x.device)
    off = s["offsets"].to(torch.int64)
    g = torch.searchsorted(off[1:], row, right=True)
    mine = (row < off[-1])[:, None]
    gc = g.clamp(max=G - 1)
    slot = torch.where(mine[:, 0], gc * s["most"] + row - off[gc], G * s["most"])

    def to_leaves(v):
        full = v.new_zeros((G * s["most"] + 1, v.shape[1]))
        full[slot] = torch.where(mine, v, 0.0)
        return full[:-1].view(G, s["most"], v.shape[1])

    def back(v):
        flat = v.reshape(G * s["most"], v.shape[2])
        return torch.where(mine, flat[slot.clamp(max=G * s["most"] - 1)], 0.0)

    xg = to_leaves(x)
    z = torch.bmm(xg, w.transpose(1, 2).contiguous())
    if s["b"] is not None:
        z = z + s["b"].float()[:, None]
    z = back(z)
    a, d = _act(s["act"], z)
    y = a if s["r"] is None else a + s["r"].float()
    out = {"y": torch.where(mine, y, 0.0).to(T)}
    if s["train"]:
        dz = torch.where(mine, s["dy"].float() * d, 0.0)
        dzg = to_leaves(dz)
        out["dx"] = back(torch.bmm(dzg, w)).to(T)
        out["dw"] = torch.bmm(dzg.transpose(1, 2).contiguous(), xg).to(T)
        if s["b"] is not None:
            out["db"] = dzg.sum(1).to(T)
        if s["r"] is not None:
            out["dr"] = torch.where(mine, s["dy"], 0.0)
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"top": _exact_top, "exchange": _exact_exchange, "dense": _exact_dense}[case["op"]](s)


def _exact_top(s):
    L, k, N = s["L"], s["k"], s["N"]
    phi = s["phi"].detach()[:, :L].double()
    by_size = torch.sort(phi, dim=1, descending=True, stable=True)
    leaf = torch.where(by_size.values[:, :k] > 0, by_size.indices[:, :k], -1)
    p = phi.requires_grad_(True)
    picked = torch.where(leaf >= 0, torch.gather(p, 1, leaf.clamp(min=0)), 0.0)
    weight = picked / picked.sum(1, keepdim=True) if s["renorm"] else picked
    out = {"leaf": leaf.to(torch.int32), "weight": weight.detach()}
    if s["train"]:
        d, = torch.autograd.grad(weight, p, s["dweight"].double())
        out["dphi"] = torch.cat([d, d.new_zeros((N, _padded(L) - L))], 1)
    return out


def _exact_exchange(s):
    N, D, L, k = s["N"], s["D"], s["L"], s["k"]
    flat = s["leaf"].reshape(-1).cpu()
    key = torch.where((flat >= 0) & (flat < L), flat, L).tolist()
    order = torch.tensor(sorted(range(N * k), key=key.__getitem__), dtype=torch.int64)
    sizes = torch.bincount(torch.tensor(key), minlength=L + 1)
    offsets = torch.cumsum(sizes, 0) - sizes
    kept = int(offsets[L])
    place = torch.zeros(N * k, dtype=torch.int64).index_copy(0, order, torch.arange(N * k))
    head = order[:kept].to(DEVICE)
    frame = head // k
    x, ys, w = (s[m].detach().double().requires_grad_(True) for m in ("x", "ys", "weight"))
    xs = torch.cat([x[frame], x.new_zeros((N * k - kept, D))])
    y = x.new_zeros((N, D)).index_add(0, frame, ys[:kept] * w.reshape(-1)[head][:, None])
    out = {"place": place.view(N, k).to(torch.int32), "order": order.to(torch.int32),
           "offsets": offsets.to(torch.int32), "xs": xs.detach(), "y": y.detach()}
    if s["train"]:
        out["dx"], out["dys"], out["dweight"] = torch.autograd.grad(
            [xs, y], [x, ys, w], [s["dxs"].double(), s["dy"].double()])
    return out


def _exact_act(name, z):
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return {"none": lambda v: v, "relu": torch.relu, "tanh": torch.tanh,
            "softsign": lambda v: v / (v.abs() + 1), "silu": lambda v: v / (1 + torch.exp(-v))}[name](z)


def _exact_dense(s):
    M, n, G = s["M"], s["n"], s["G"]
    x, w, b, r = (None if s[m] is None else s[m].detach().double().requires_grad_(True) for m in ("x", "w", "b", "r"))
    bounds = s["offsets"].tolist() if G else [0, M]
    parts = []
    for g in range(max(1, G)):
        lo, hi = bounds[g], bounds[g + 1]
        z = torch.mm(x[lo:hi], (w[g] if G else w).t())
        if b is not None:
            z = z + (b[g] if G else b)
        a = _exact_act(s["act"], z)
        parts.append(a if r is None else a + r[lo:hi])
    y = torch.cat(parts + [x.new_zeros((M - bounds[-1], n))])
    out = {"y": y.detach()}
    if s["train"]:
        names = [m for m, v in (("x", x), ("w", w), ("b", b), ("r", r)) if v is not None]
        wanted = [v for v in (x, w, b, r) if v is not None]
        out.update(zip(["d" + m for m in names], torch.autograd.grad(y, wanted, s["dy"].double())))
    return out
