"""Measured calls of the dense routed operators and of the adapters beside the projections.

Kinds, each forward alone (serving) or with its gradients (training):

- ``experts``: ``gather_mm``, the product of routed rows with dense expert weights, for layers whose experts stay
  unquantised: ``out[t, j] = W[idx[t, j]] . x[t]``;
- ``adapters``: ``gather_lora``, low-rank adapters of many requests added to a shared projection's rows:
  ``out[r] = base[r] + s[a] (x[r] A[a]^T) B[a]^T`` with ``a = idx[r]`` (-1: no adapter);
- ``combine``: ``route_combine``, the weighted sum of a token's routed rows.

Sizes are those of this package's layers (384 experts top-6 of 4096 -> 2048, 128 top-8 of 7168 -> 2048, ...) and
generic ones. Activations are N(0, 1), weights keep their products near 1, routes are distinct per token.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # batch-1 decode through one dense projection of the 384-expert layer: latency and six experts' weights
        _experts("experts_token_1", 1, 384, 6, 4096, 2048, "float16"),
        # a speculative-verify window
        _experts("experts_verify_8", 8, 256, 6, 4096, 2048, "bfloat16"),
        # a short prompt of an odd length through wide experts, about 20 rows each
        _experts("experts_ragged_333", 333, 128, 8, 7168, 2048, "bfloat16"),
        # a prompt through many experts of skewed popularity: from none to hundreds of rows each
        _experts("experts_prefill_2048", 2048, 384, 6, 4096, 2048, "float16", routing="zipf"),
        # a large prefill batch through few experts: the largest product
        _experts("experts_prefill_8192", 8192, 32, 8, 4096, 2048, "bfloat16"),
        # a training step of one projection: output, gradients of the rows and of every expert
        _experts("experts_train_4096", 4096, 64, 8, 2048, 768, "bfloat16", train=True),
        # one request's token: the smallest call, all latency
        _adapters("adapters_row_1", 1, 32, 16, 4096, 4096, "float16"),
        # a decode batch, each row a request with an adapter of its own
        _adapters("adapters_batch_64", 64, 96, 64, 4096, 2048, "bfloat16"),
        # prompts of many requests in one batch, ragged, an odd number of rows
        _adapters("adapters_prefill_4093", 4093, 16, 32, 4096, 4096, "bfloat16"),
        # a training step of eight adapters together
        _adapters("adapters_train_2048", 2048, 8, 16, 4096, 2048, "bfloat16", train=True),
        # the end of an unquantised expert layer: a prompt's routed rows summed per token
        _combine("combine_2048", 2048, 6, 4096, "bfloat16"),
        # the same with the gradients of the rows and of the routing weights, an odd number of tokens
        _combine("combine_train_1021", 1021, 8, 4096, "bfloat16", train=True),
    ]


def _experts(name, tokens, experts, top_k, in_dims, out_dims, dtype, routing="normal", train=False):
    return {"name": name, "kind": "experts", "tokens": tokens, "experts": experts, "top_k": top_k, "in_dims": in_dims,
            "out_dims": out_dims, "dtype": dtype, "routing": routing, "train": train}


def _adapters(name, rows, adapters, rank, in_dims, out_dims, dtype, top_k=0, train=False):
    return {"name": name, "kind": "adapters", "rows": rows, "adapters": adapters, "rank": rank, "in_dims": in_dims,
            "out_dims": out_dims, "dtype": dtype, "top_k": top_k, "train": train}


def _combine(name, tokens, top_k, hidden, dtype, train=False):
    return {"name": name, "kind": "combine", "tokens": tokens, "top_k": top_k, "hidden": hidden, "dtype": dtype,
            "train": train}


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["experts", "experts", "experts", "adapters", "adapters", "adapters", "combine"])
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    train = rng.random() < 0.4
    if kind == "combine":
        return _unnamed(_combine("", _log(rng, 1, 2048), rng.randint(1, 8), 4 * rng.randint(64, 1024), dtype, train))
    if kind == "adapters":
        in_dims, out_dims = 8 * rng.randint(64, 512), rng.choice([8 * rng.randint(64, 512), rng.randint(500, 4096)])
        routed = rng.random() < 0.25
        # routed: one adapter per (request's adapter, expert)
        adapters = rng.randint(2, 8) * 16 if routed else _log(rng, 1, 96)
        rank = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 128)])
        rows = _log(rng, 1, 512 if routed or dtype == "float32" else 4096)
        return _unnamed(_adapters("", rows, adapters, min(rank, 8192 // adapters), in_dims, out_dims, dtype,
                                  top_k=rng.randint(2, 8) if routed else 0, train=train))
    in_dims, out_dims = rng.choice([(4096, 2048), (2048, 4096), (4096, 1536), (2880, 1440), (7168, 2048),
                                    (8 * rng.randint(64, 512), rng.randint(200, 2048))])
    top_k = rng.randint(1, 8)
    most = (2.0e9 if not train else 4.0e8) / (2 if dtype == "float32" else 1)  # weight values
    experts = _log(rng, top_k, max(top_k, min(384, int(most / (in_dims * out_dims)))))
    flops = 4e11 if dtype != "float32" else 4e10
    tokens = _log(rng, 1, max(1, min(8192, int(flops / (2 * top_k * in_dims * out_dims * (3 if train else 1))))))
    return _unnamed(_experts("", tokens, experts, top_k, in_dims, out_dims, dtype,
                             routing=rng.choice(["normal", "zipf"]), train=train))


def _unnamed(case):
    del case["name"]
    return case


# --------------------------------------------------------------------------- inputs


class _Inputs:
    """Seeded device tensors."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return torch.empty(shape, device=self.dev, dtype=dtype).normal_(0.0, std, generator=self.g)

    def uniform(self, *shape):
        return torch.rand(shape, device=self.dev, generator=self.g)

    def whole(self, hi, *shape):
        return torch.randint(0, hi, shape, device=self.dev, generator=self.g)

    def routes(self, tokens, experts, top_k, routing):
        """Distinct experts per token: by popularity (Zipf 1.1 over a random order) or evenly."""
        score = -torch.log(-torch.log(self.uniform(tokens, experts).clamp(1e-7, 1 - 1e-7)))
        if routing == "zipf":
            rank = torch.argsort(self.uniform(experts)).float() + 1
            score = score - 1.1 * torch.log(rank)
        return torch.topk(score, top_k, dim=1).indices.to(torch.int32)


def prepare(case, seed):
    g, dtype, train = _Inputs(seed), _DTYPES[case["dtype"]], case["train"]
    s = {"kind": case["kind"], "train": train}
    if case["kind"] == "experts":
        T, E, k, K, N = (case[n] for n in ("tokens", "experts", "top_k", "in_dims", "out_dims"))
        s["idx"] = g.routes(T, E, k, case["routing"])
        s["x"] = g.normal(T, K, dtype=dtype)
        s["w"] = g.normal(E, N, K, dtype=dtype, std=K ** -0.5)
        if train:
            s["dy"] = g.normal(T, k, N, dtype=dtype)
        grads = ("x", "w")
    elif case["kind"] == "adapters":
        T, n, r, K, N, k = (case[m] for m in ("rows", "adapters", "rank", "in_dims", "out_dims", "top_k"))
        s["x"] = g.normal(T, K, dtype=dtype)
        s["a"] = g.normal(n, r, K, dtype=dtype, std=K ** -0.5)
        s["b"] = g.normal(n, N, r, dtype=dtype, std=r ** -0.5)
        s["scale"] = g.uniform(n) + 0.5
        if k:  # (adapter of the request, expert of the route), 16 experts
            s["idx"] = (16 * g.whole(n // 16, T, 1) + g.routes(T, 16, k, "normal")).to(torch.int32)
            rows = (T, k)
        else:  # up to 256 rows: a request each; more: ragged runs of rows, about 100 each
            req = torch.arange(T, device=g.dev) if T <= 256 else torch.cumsum((g.uniform(T) < 0.01).long(), 0)
            of = g.whole(n, T)
            of = torch.where(g.uniform(T) < 0.125, -1, of)  # one request in eight has no adapter
            s["idx"] = of[req].to(torch.int32)
            rows = (T,)
        s["base"] = g.normal(*rows, N, dtype=dtype)
        if train:
            s["dy"] = g.normal(*rows, N, dtype=dtype)
        grads = ("x", "a", "b")
    else:
        T, k, H = case["tokens"], case["top_k"], case["hidden"]
        s["y"] = g.normal(T, k, H, dtype=dtype)
        s["w"] = torch.softmax(g.normal(T, k), dim=1)
        if train:
            s["dy"] = g.normal(T, H)
        grads = ("y", "w")
    if train:
        for name in grads:
            s[name].requires_grad_(True)
    return s


# --------------------------------------------------------------------------- one pass


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["kind"] == "experts":
            return _plain_experts(state)
        if state["kind"] == "adapters":
            return _plain_adapters(state)
        return _plain_combine(state)


def _run_own(s):
    import keep_amd

    if s["kind"] == "experts":
        out = keep_amd.gather_mm(s["x"], s["w"], s["idx"])
        if not s["train"]:
            return {"out": out}
        dx, dw = torch.autograd.grad(out, (s["x"], s["w"]), s["dy"])
        return {"out": out, "dx": dx, "dw": dw}
    if s["kind"] == "adapters":
        out = keep_amd.gather_lora(s["x"], s["a"], s["b"], s["idx"], base=s["base"], scales=s["scale"])
        if not s["train"]:
            return {"out": out}
        dx, da, db = torch.autograd.grad(out, (s["x"], s["a"], s["b"]), s["dy"])
        return {"out": out, "dx": dx, "da": da, "db": db}
    out = keep_amd.route_combine(s["y"], s["w"])
    if not s["train"]:
        return {"out": out}
    dy, dw = torch.autograd.grad(out, (s["y"], s["w"]), s["dy"])
    return {"out": out, "dy": dy, "dw": dw}


def _plain_experts(s):
    """Routes sorted by expert and laid out in tiles of one expert each (as many as the sizes can need, so that the
    host waits for no count), one batched product over the tiles."""
    x, w, idx = s["x"], s["w"], s["idx"]
    (T, K), (E, N, _), k = x.shape, w.shape, idx.shape[1]
    flat, R = idx.reshape(-1).long(), idx.numel()
    if R <= 64:  # every route a tile
        tile_expert, slot, row, tile = flat, torch.arange(R, device=x.device), torch.arange(R, device=x.device), 1
    else:
        tile = 1 << max(4, (R // E).bit_length())
        row = torch.argsort(flat, stable=True)
        counts = (flat[:, None] == torch.arange(E, device=x.device)).sum(0)
        ends = torch.cumsum((counts + tile - 1) // tile, 0)
        n_tiles = R // tile + min(E, R)
        tile_expert = torch.searchsorted(ends, torch.arange(n_tiles, device=x.device), right=True).clamp(max=E - 1)
        e = flat[row]
        first = torch.cumsum(counts, 0) - counts
        slot = (ends - (counts + tile - 1) // tile)[e] * tile + torch.arange(R, device=x.device) - first[e]
    n_tiles = tile_expert.numel()
    wt = w[tile_expert].float()
    xs = torch.zeros((n_tiles * tile, K), device=x.device)
    xs[slot] = x[row // k].float()
    xs = xs.view(n_tiles, tile, K)
    out = torch.empty((R, N), device=x.device)
    out[row] = torch.bmm(xs, wt.transpose(1, 2)).view(-1, N)[slot]
    out = out.view(T, k, N).to(x.dtype)
    if not s["train"]:
        return {"out": out}
    dys = torch.zeros((n_tiles * tile, N), device=x.device)
    dys[slot] = s["dy"].reshape(R, N)[row].float()
    dys = dys.view(n_tiles, tile, N)
    dx = torch.empty((R, K), device=x.device)
    dx[row] = torch.bmm(dys, wt).view(-1, K)[slot]
    del wt
    part = torch.bmm(dys.transpose(1, 2), xs)  # each tile's share of its expert's gradient
    of = (tile_expert == torch.arange(E, device=x.device)[:, None]).float()
    dw = torch.mm(of, part.view(n_tiles, N * K)).view(E, N, K)
    return {"out": out, "dx": dx.view(T, k, K).sum(1).to(x.dtype), "dw": dw.to(w.dtype)}


def _plain_adapters(s):
    """Every adapter for every row in two large products; a row keeps its own adapter's block of the first."""
    x, a, b, idx, scale = s["x"], s["a"], s["b"], s["idx"], s["scale"]
    (T, K), (n, r, _), N = x.shape, a.shape, b.shape[1]
    flat = idx.reshape(-1)
    k = flat.numel() // T
    mask = (flat[:, None] == torch.arange(n, device=x.device)).float()
    xf, af = x.float(), a.float().reshape(n * r, K)
    bf = b.float().transpose(0, 1).reshape(N, n * r)
    t = torch.mm(xf, af.t()).view(T, 1, n, r).expand(T, k, n, r).reshape(T * k, n, r) * mask[:, :, None]
    ts = (t * scale[:, None]).view(T * k, n * r)
    out = (s["base"].float() + torch.mm(ts, bf.t()).view(s["base"].shape)).to(x.dtype)
    if not s["train"]:
        return {"out": out}
    dy = s["dy"].reshape(T * k, N).float()
    dt = (torch.mm(dy, bf).view(T * k, n, r) * (mask * scale)[:, :, None]).view(T, k, n * r)
    db = torch.mm(ts.t(), dy).view(n, r, N).transpose(1, 2)
    dt = dt.sum(1)  # a row's routes
    dx = torch.mm(dt, af)
    da = torch.mm(dt.t(), xf).view(n, r, K)
    return {"out": out, "dx": dx.to(x.dtype), "da": da.to(a.dtype), "db": db.to(b.dtype)}


def _plain_combine(s):
    y, w = s["y"].float(), s["w"]
    out = (y * w[:, :, None]).sum(1)
    if not s["train"]:
        return {"out": out}
    dy = s["dy"]
    return {"out": out, "dy": (w[:, :, None] * dy[:, None]).to(s["y"].dtype), "dw": (y * dy[:, None]).sum(2)}


# --------------------------------------------------------------------------- what a pass needs


def _experts_hit(case):
    """How many experts some route names, by expectation (routes taken as independent)."""
    E, routes = case["experts"], case["tokens"] * case["top_k"]
    if case["routing"] == "normal":
        return E * (1 - (1 - case["top_k"] / E) ** case["tokens"])
    p = [(i + 1) ** -1.1 for i in range(E)]
    total = sum(p)
    return sum(1 - (1 - min(v / total, 0.5)) ** routes for v in p)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    train = case["train"]
    if case["kind"] == "experts":
        T, k, K, N = (case[n] for n in ("tokens", "top_k", "in_dims", "out_dims"))
        hit = _experts_hit(case)
        weights, x, y = hit * N * K * size, T * K * size, T * k * N * size
        if not train:
            return {"bytes": weights + x + y + 4 * T * k, "flops": 2 * T * k * K * N}
        # weights, x and dy in; out, dx and every expert's gradient out
        return {"bytes": weights + 2 * x + 2 * y + case["experts"] * N * K * size + 4 * T * k,
                "flops": 6 * T * k * K * N}
    if case["kind"] == "adapters":
        T, n, r, K, N = (case[m] for m in ("rows", "adapters", "rank", "in_dims", "out_dims"))
        routes = T * max(1, case["top_k"])
        requests = routes if T <= 256 or case["top_k"] else 1 + T / 100
        hit = n * (1 - (1 - 1 / n) ** (requests if case["top_k"] else 7 / 8 * requests)) if n > 1 else 1
        weights, x, y = hit * r * (K + N) * size, T * K * size, routes * N * size
        if not train:
            return {"bytes": weights + x + 2 * y + 4 * routes, "flops": 2 * routes * r * (K + N)}
        # A, B, x, base and dy in; out, dx and both gradients out
        return {"bytes": weights + n * r * (K + N) * size + 2 * x + 3 * y + 4 * routes,
                "flops": 6 * routes * r * (K + N)}
    T, k, H = case["tokens"], case["top_k"], case["hidden"]
    y = T * k * H * size
    if not train:
        return {"bytes": y + 4 * T * k + 4 * T * H, "flops": 2 * T * k * H}
    return {"bytes": 2 * y + 8 * T * k + 8 * T * H, "flops": 5 * T * k * H}


# --------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    train = case["train"]
    if case["kind"] == "combine":
        y, w = s["y"].double(), s["w"].double()
        got = {"out": torch.einsum("tkh,tk->th", y, w)}
        if train:
            dy = s["dy"].double()
            got["dy"] = torch.einsum("tk,th->tkh", w, dy)
            got["dw"] = torch.einsum("tkh,th->tk", y, dy)
        return got
    x = s["x"].double()
    idx = s["idx"] if s["idx"].ndim == 2 else s["idx"][:, None]
    T, k = idx.shape
    token, expert = torch.arange(T, device=x.device).repeat_interleave(k), idx.reshape(-1)
    if case["kind"] == "experts":
        w = s["w"]
        E, N, K = w.shape
        out = torch.zeros((T * k, N), dtype=torch.float64, device=x.device)
        dx = torch.zeros_like(x) if train else None
        dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device) if train else None
        for e in torch.unique(expert).tolist():
            at = (expert == e).nonzero()[:, 0]
            we, xe = w[e].double(), x[token[at]]
            out[at] = xe @ we.t()
            if train:
                dye = s["dy"].reshape(T * k, N)[at].double()
                dx.index_add_(0, token[at], dye @ we)
                dw[e] = dye.t() @ xe
        got = {"out": out.view(T, k, N)}
        return {**got, "dx": dx, "dw": dw} if train else got
    a, b, scale = s["a"].double(), s["b"].double(), s["scale"].double()
    out = s["base"].double().reshape(T * k, -1).clone()
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for e in torch.unique(expert).tolist():
        if e < 0:
            continue
        at = (expert == e).nonzero()[:, 0]
        xe = x[token[at]]
        te = xe @ a[e].t()
        out[at] += scale[e] * (te @ b[e].t())
        if train:
            dye = scale[e] * s["dy"].reshape(T * k, -1)[at].double()
            dte = dye @ b[e]
            dx.index_add_(0, token[at], dte @ a[e])
            da[e] = dte.t() @ xe
            db[e] = dye.t() @ te
    got = {"out": out.view(s["base"].shape)}
    return {**got, "dx": dx, "da": da, "db": db} if train else got
