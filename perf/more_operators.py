"""Measured calls of the steps around the routed experts: norm, expert choice and the dense projections.

Kinds, each forward alone (serving) or with its gradients (training):

- ``norm``: ``rmsnorm``, the residual's addition and the root-mean-square norm in front of the router and the experts:
  ``h = residual + x``, ``y = h / sqrt(mean(h^2) + eps) * weight``; serving also as ``rmsnorm_quant``, ``y`` in 8 bits
  (e4m3) with a scale per 128 values;
- ``route``: ``route_experts``, the choice of each token's experts from the router's logits: scores, a bias that balances
  the choice, groups of experts, the top k, weights that add up to one;
- ``linear``: ``linear``, a dense projection with its epilogue, ``residual + act(x W^T + bias)`` (the router's own
  product, a shared expert's); serving also as ``linear_q8``, operands in 8 bits with scales per 128 values of a row of
  ``x`` and per 128 x 128 of ``W``.

Sizes are those of this package's layers (hidden 2048 to 7168, 64 to 384 experts, intermediate 1440 to 2048) and generic
ones. Activations are N(0, 1), weights keep their products near 1.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_BLOCK = 128  # values of a row that share a scale
_EPS = 1e-6


def listed():
    return [
        # one token of a decode step between attention and the experts: the smallest call, all latency
        _norm("norm_token_1", 1, 7168, "bfloat16", "bfloat16"),
        # a prompt's rows as the 8-bit products take them, and the residual stream
        _norm("norm_quant_2048", 2048, 4096, "bfloat16", "bfloat16", quant=True),
        # an odd number of rows of a width that is no power of two, the residual stream kept in float32
        _norm("norm_ragged_333", 333, 2880, "float16", "float32"),
        # a training step's norm: rows, residual stream, their gradients and the weight's
        _norm("norm_train_8192", 8192, 4096, "bfloat16", "bfloat16", train=True),
        # a decode step's choice among groups under a balancing bias
        _route("route_token_1", 1, 256, 8, "sigmoid", bias=True, groups=8, topk_groups=4),
        # the same for a long prompt
        _route("route_prefill_8192", 8192, 256, 8, "sigmoid", bias=True, groups=8, topk_groups=4),
        # a training step of a softmax router, with the experts' loads and the gradient of the logits
        _route("route_train_4096", 4096, 384, 6, "softmax", load=True, train=True),
        # the router's product of one token, float32 logits of 16-bit rows
        _linear("linear_gate_1", 1, 4096, 384, "bfloat16", out="float32"),
        # a short prompt of an odd length through a biased projection, all of the epilogue
        _linear("linear_ragged_333", 333, 2880, 1440, "float16", bias=True, act="gelu", residual=True),
        # a large prefill batch through one projection of a dense expert: the largest product
        _linear("linear_prefill_8192", 8192, 4096, 8192, "bfloat16", act="silu"),
        # a training step of a biased projection: output, gradients of rows, weights, bias and residual
        _linear("linear_train_4096", 4096, 4096, 2048, "bfloat16", bias=True, act="silu", residual=True, train=True),
        # a prompt through a projection whose weights are kept in 8 bits
        _linear("linear_q8_4096", 4096, 7168, 2048, "e4m3", out="bfloat16"),
    ]


def _norm(name, rows, width, dtype, residual, quant=False, train=False):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual,
            "quant": quant, "train": train}


def _route(name, tokens, experts, top_k, score, dtype="float32", bias=False, groups=1, topk_groups=1, load=False,
           renormalize=True, train=False):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "score": score,
            "dtype": dtype, "bias": bias, "groups": groups, "topk_groups": topk_groups, "load": load,
            "renormalize": renormalize, "train": train}


def _linear(name, rows, in_dims, out_dims, dtype, out="", bias=False, act="", residual=False, train=False):
    return {"name": name, "kind": "linear", "rows": rows, "in_dims": in_dims, "out_dims": out_dims, "dtype": dtype,
            "out": out or dtype, "bias": bias, "act": act, "residual": residual, "train": train}


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["norm", "norm", "route", "route", "linear", "linear", "linear"])
    train = rng.random() < 0.35
    if kind == "norm":
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
        width = rng.choice([2048, 2880, 4096, 7168, 8 * _log(rng, 8, 1024), _log(rng, 16, 8192)])
        quant = not train and rng.random() < 0.4
        residual = rng.choice(["", dtype, dtype, "float32"])
        return _unnamed(_norm("", _log(rng, 1, 8192 if width <= 4096 else 4096), width, dtype, residual, quant, train))
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8, rng.randint(2, 12)])
        experts = groups * rng.randint(2, 384 // groups)
        if groups == 1:
            experts = rng.choice([8, 64, 128, 384, rng.randint(2, 512)])
        topk_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(8, topk_groups * (experts // groups)))
        return _unnamed(_route("", _log(rng, 1, 8192 if experts <= 384 else 4096), experts, top_k,
                               rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]),
                               dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]),
                               bias=rng.random() < 0.5, groups=groups, topk_groups=topk_groups,
                               load=rng.random() < 0.4, renormalize=rng.random() < 0.7, train=train))
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32", "e4m3"])
    in_dims, out_dims = rng.choice([(4096, 2048), (2048, 4096), (4096, 1536), (2880, 1440), (7168, 2048), (4096, 384),
                                    (7168, 256), (8 * rng.randint(8, 512), rng.randint(64, 4096)),
                                    (rng.randint(64, 4096), rng.randint(64, 4096))])
    if dtype == "e4m3":
        in_dims = (in_dims + 15) // 16 * 16
        train = False
    flops = 3e10 if dtype == "float32" else 4e11
    rows = _log(rng, 1, max(1, min(8192, int(flops / (2 * in_dims * out_dims * (3 if train else 1))))))
    out = "" if dtype != "e4m3" else "bfloat16"
    if not train and rng.random() < 0.25:
        out = "float32"
    return _unnamed(_linear("", rows, in_dims, out_dims, dtype, out=out, bias=rng.random() < 0.5,
                            act=rng.choice(["", "", "silu", "gelu", "relu"]), residual=rng.random() < 0.4, train=train))


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

    def normal(self, *shape, dtype=torch.float32, std=1.0, mean=0.0):
        return torch.empty(shape, device=self.dev, dtype=dtype).normal_(mean, std, generator=self.g)


def _e4m3(v, rows):
    """``v`` in 8 bits, and its scales per 128 values of ``rows`` rows."""
    (M, K), Kb, Mb = v.shape, -(-v.shape[1] // _BLOCK), -(-v.shape[0] // rows)
    full = torch.zeros((Mb * rows, Kb * _BLOCK), device=v.device)
    full[:M, :K] = v
    scale = full.view(Mb, rows, Kb, _BLOCK).abs().amax(dim=(1, 3)).clamp(min=1e-4) / 448.0
    q = full.view(Mb, rows, Kb, _BLOCK) / scale[:, None, :, None]
    return q.view(Mb * rows, Kb * _BLOCK)[:M, :K].clamp(-448, 448).to(torch.float8_e4m3fn).contiguous(), scale


def prepare(case, seed):
    g, s = _Inputs(seed), dict(case)
    train = case["train"]
    if case["kind"] == "norm":
        T, n, dtype = case["rows"], case["width"], _DTYPES[case["dtype"]]
        s["x"] = g.normal(T, n, dtype=dtype)
        s["res"] = g.normal(T, n, dtype=_DTYPES[case["residual"]], std=2.0) if case["residual"] else None
        s["w"] = g.normal(n, dtype=dtype, std=0.2, mean=1.0)
        if train:
            s["dy"] = g.normal(T, n, dtype=dtype)
            s["dh"] = None if s["res"] is None else g.normal(T, n, dtype=s["res"].dtype)
        grads = ("x", "res", "w")
    elif case["kind"] == "route":
        T, E = case["tokens"], case["experts"]
        s["z"] = g.normal(T, E, dtype=_DTYPES[case["dtype"]], std=1.5)
        s["b"] = g.normal(E, std=0.05) if case["bias"] else None
        if train:
            s["dw"] = g.normal(T, case["top_k"])
        grads = ("z",)
    else:
        M, K, N = case["rows"], case["in_dims"], case["out_dims"]
        if case["dtype"] == "e4m3":
            s["x"], s["xs"] = _e4m3(g.normal(M, K), 1)
            s["w"], s["ws"] = _e4m3(g.normal(N, K, std=K ** -0.5), _BLOCK)
            dtype = torch.bfloat16
        else:
            dtype = _DTYPES[case["dtype"]]
            s["x"] = g.normal(M, K, dtype=dtype)
            s["w"] = g.normal(N, K, dtype=dtype, std=K ** -0.5)
        od = _DTYPES[case["out"]]
        s["b"] = g.normal(N, dtype=dtype, std=0.5) if case["bias"] else None
        s["res"] = g.normal(M, N, dtype=od) if case["residual"] else None
        if train:
            s["dy"] = g.normal(M, N, dtype=od)
        grads = ("x", "w", "b", "res")
    if train:
        for name in grads:
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# --------------------------------------------------------------------------- one pass


def run(state):
    if own:
        return _OWN[state["kind"]](state)
    with torch.no_grad():
        return _PLAIN[state["kind"]](state)


def _grads(s, outs, douts, names):
    """The gradients of the inputs that there are, by name."""
    names = [n for n in names if s[n] is not None]
    return {"d" + n: g for n, g in zip(names, torch.autograd.grad(outs, [s[n] for n in names], douts))}


def _own_norm(s):
    import keep_amd

    if s["quant"]:
        q = keep_amd.rmsnorm_quant(s["x"], s["w"], _EPS, residual=s["res"], quant_block=_BLOCK)
        return {"q": q[0], "scales": q[1], **({"h": q[2]} if s["res"] is not None else {})}
    y = keep_amd.rmsnorm(s["x"], s["w"], _EPS, residual=s["res"])
    y, h = y if s["res"] is not None else (y, None)
    got = {"y": y} if h is None else {"y": y, "h": h}
    if s["train"]:
        got.update(_grads(s, (y,) if h is None else (y, h), (s["dy"],) if h is None else (s["dy"], s["dh"]),
                          ("x", "res", "w")))
    return got


def _own_route(s):
    import keep_amd

    r = keep_amd.route_experts(s["z"], s["top_k"], bias=s["b"], score_func=s["score"], groups=s["groups"],
                               topk_groups=s["topk_groups"], renormalize=s["renormalize"], count_load=s["load"])
    got = {"idx": r.idx, "weight": r.weight}
    if s["load"]:
        got["load"] = r.load
    if s["train"]:
        got["dz"], = torch.autograd.grad(r.weight, s["z"], s["dw"])
    return got


def _own_linear(s):
    import keep_amd

    more = dict(activation=s["act"] or None, residual=s["res"], out_dtype=_DTYPES[s["out"]])
    if s["dtype"] == "e4m3":
        return {"out": keep_amd.linear_q8(s["x"], s["xs"], s["w"], s["ws"], s["b"], **more)}
    out = keep_amd.linear(s["x"], s["w"], s["b"], **more)
    if not s["train"]:
        return {"out": out}
    return {"out": out, **_grads(s, out, s["dy"], ("x", "w", "b", "res"))}


def _plain_norm(s):
    x, res, w = s["x"].float(), s["res"], s["w"].float()
    h = s["x"] if res is None else (res.float() + x).to(res.dtype)
    hf = h.float()
    r = 1.0 / torch.sqrt((hf * hf).sum(1, keepdim=True) / hf.shape[1] + _EPS)
    y = hf * r * w
    got = {} if res is None else {"h": h}
    if s["quant"]:
        T, n = y.shape
        full = torch.zeros((T, -(-n // _BLOCK) * _BLOCK), device=y.device)
        full[:, :n] = y
        full = full.view(T, -1, _BLOCK)
        scale = full.abs().amax(dim=2).clamp(min=1e-4) / 448.0
        q = (full / scale[:, :, None]).clamp(-448, 448).view(T, -1)[:, :n].to(torch.float8_e4m3fn)
        return {"q": q, "scales": scale, **got}
    got["y"] = y.to(s["x"].dtype)
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dh = r * (g - hf * (r * r * (g * hf).sum(1, keepdim=True) / hf.shape[1]))
        if res is not None:
            dh = dh + s["dh"].float()
            got["dres"] = dh.to(res.dtype)
        got["dx"] = dh.to(s["x"].dtype)
        got["dw"] = (dy * hf * r).sum(0).to(s["w"].dtype)
    return got


def _scores64(z, score):
    if score == "softmax":
        e = torch.exp(z - z.amax(1, keepdim=True))
        return e / e.sum(1, keepdim=True)
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    return torch.sqrt(z.clamp(min=0) + torch.log1p(torch.exp(-z.abs())))


def _take(keys, k):
    """The k largest of each row, in order, the lowest index first among equals."""
    n, at = keys.shape[1], torch.arange(keys.shape[1], device=keys.device)
    keys, got = keys.clone(), []
    for _ in range(k):
        i = torch.where(keys == keys.amax(1, keepdim=True), at, n).amin(1, keepdim=True)
        got.append(i)
        keys.scatter_(1, i, -math.inf)
    return torch.cat(got, 1)


def _plain_route(s):
    """In 64 bits: neighbouring keys of thousands of tokens come closer than 32 bits tell apart."""
    z, k, G = s["z"].double(), s["top_k"], s["groups"]
    T, E = z.shape
    p = _scores64(z, s["score"])
    keys = p if s["b"] is None else p + s["b"].double()
    if s["topk_groups"] < G:
        grouped = keys.view(T, G, E // G)
        top = grouped.amax(2)
        if E // G > 1:
            first = _take(grouped.reshape(T * G, E // G), 1).view(T, G, 1)
            top = top + grouped.scatter(2, first, -math.inf).amax(2)
        kept = torch.zeros((T, G), dtype=torch.bool, device=z.device)
        kept.scatter_(1, _take(top, s["topk_groups"]), True)
        keys = torch.where(kept[:, :, None].expand(T, G, E // G).reshape(T, E), keys, -math.inf)
    idx = _take(keys, k)
    chosen = p.gather(1, idx)
    total = chosen.sum(1, keepdim=True) + 1e-20 if s["renormalize"] else torch.ones((T, 1), device=z.device)
    weight = chosen / total
    got = {"idx": idx.to(torch.int32), "weight": weight.float()}
    if s["load"]:
        got["load"] = torch.zeros(E, dtype=torch.int32, device=z.device).index_add_(
            0, idx.reshape(-1), torch.ones(T * k, dtype=torch.int32, device=z.device))
    if s["train"]:
        g = s["dw"].double()
        if s["renormalize"]:
            g = (g - (g * weight).sum(1, keepdim=True)) / total
        if s["score"] == "softmax":
            dz = -p * (g * chosen).sum(1, keepdim=True)
            dz.scatter_add_(1, idx, g * chosen)
        else:
            zc = z.gather(1, idx)
            slope = chosen * (1 - chosen) if s["score"] == "sigmoid" else 0.5 / (chosen * (1 + torch.exp(-zc)))
            dz = torch.zeros_like(z).scatter_(1, idx, g * slope)
        got["dz"] = dz.to(s["z"].dtype)
    return got


def _scaled(q, scale, rows):
    """8-bit values times their scales, in float32."""
    full = scale.repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(_BLOCK, 1)[:, :q.shape[1]]
    return q.float() * full


def _act(u, act):
    """The activation and its slope."""
    if act == "relu":
        return u.clamp(min=0), (u > 0).to(u.dtype)
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-u))
        return u * p, p * (1 + u * (1 - p))
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(u * math.sqrt(0.5)))
        return u * p, p + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    return u, torch.ones_like(u)


def _plain_linear(s):
    if s["dtype"] == "e4m3":
        x, w = _scaled(s["x"], s["xs"], 1), _scaled(s["w"], s["ws"], _BLOCK)
    else:
        x, w = s["x"].float(), s["w"].float()
    u = torch.mm(x, w.t())
    if s["b"] is not None:
        u = u + s["b"].float()
    v, slope = (u, None) if not s["act"] else _act(u, s["act"])
    if s["res"] is not None:
        v = s["res"].float() + v
    got = {"out": v.to(_DTYPES[s["out"]])}
    if s["train"]:
        du = s["dy"].float() if slope is None else s["dy"].float() * slope
        got["dx"] = torch.mm(du, w).to(s["x"].dtype)
        got["dw"] = torch.mm(du.t(), x).to(s["w"].dtype)
        if s["b"] is not None:
            got["db"] = du.sum(0).to(s["b"].dtype)
        if s["res"] is not None:
            got["dres"] = s["dy"]
    return got


_OWN = {"norm": _own_norm, "route": _own_route, "linear": _own_linear}
_PLAIN = {"norm": _plain_norm, "route": _plain_route, "linear": _plain_linear}


# --------------------------------------------------------------------------- what a pass needs


def _size(dtype):
    return {"float32": 4, "e4m3": 1}.get(dtype, 2)


def work(case):
    if case["kind"] == "norm":
        T, n, size = case["rows"], case["width"], _size(case["dtype"])
        h = _size(case["residual"]) if case["residual"] else 0
        x = T * n * size
        if case["quant"]:
            return {"bytes": x + 2 * T * n * h + n * size + T * n + 4 * T * -(-n // _BLOCK), "flops": 10 * T * n}
        if not case["train"]:
            return {"bytes": 2 * x + 2 * T * n * h + n * size, "flops": 6 * T * n}
        # x, residual, weight, dy and dh in; y, h and the gradients out
        return {"bytes": 4 * x + 4 * T * n * h + 2 * n * size, "flops": 18 * T * n}
    if case["kind"] == "route":
        T, E, k, size = case["tokens"], case["experts"], case["top_k"], _size(case["dtype"])
        moved = T * E * size * (2 if case["train"] else 1) + T * k * (12 if case["train"] else 8)
        return {"bytes": moved + 4 * E * (int(case["bias"]) + int(case["load"])), "flops": (8 + 2 * k) * T * E}
    M, K, N = case["rows"], case["in_dims"], case["out_dims"]
    size, out = _size(case["dtype"]), _size(case["out"])
    x, w, y = M * K * size, N * K * size, M * N * out
    b, res = (N * 2 if case["bias"] else 0), (y if case["residual"] else 0)
    if case["dtype"] == "e4m3":
        scales = 4 * -(-K // _BLOCK) * (M + -(-N // _BLOCK))
        return {"bytes": x + w + y + b + res + scales, "flops": 2 * M * K * N}
    if not case["train"]:
        return {"bytes": x + w + y + b + res, "flops": 2 * M * K * N}
    # x, w, bias, residual and dy in; out, dx, dw and the bias's gradient out
    return {"bytes": 2 * (x + w + y + b) + res, "flops": 6 * M * K * N}


# --------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    return {"norm": _exact_norm, "route": _exact_route, "linear": _exact_linear}[case["kind"]](s)


def _exact_norm(s):
    x, w = s["x"].double(), s["w"].double()
    got = {}
    h = x
    if s["res"] is not None:
        got["h"] = s["res"].double() + x
        h = got["h"].to(s["res"].dtype).double()  # what is normalised is the stream as it is kept
    n = h.shape[1]
    std = torch.sqrt(torch.einsum("ti,ti->t", h, h) / n + _EPS)[:, None]
    unit = h / std
    y = unit * w
    if s["quant"]:
        parts = torch.nn.functional.pad(y.abs(), (0, -n % _BLOCK)).unflatten(1, (-1, _BLOCK))
        scale = parts.max(dim=2).values.clamp(min=1e-4) / 448.0
        got["scales"] = scale
        got["q"] = y / scale.repeat_interleave(_BLOCK, 1)[:, :n]
        return got
    got["y"] = y
    if s["train"]:
        dy = s["dy"].double()
        along = torch.einsum("ti,i,ti->t", dy, w, unit)[:, None] / n
        d = (dy * w - unit * along) / std
        if s["res"] is not None:
            d = d + s["dh"].double()
            got["dres"] = d
        got["dx"] = d
        got["dw"] = torch.einsum("ti,ti->i", dy, unit)
    return got


def _exact_route(s):
    z, k, G = s["z"].double(), s["top_k"], s["groups"]
    T, E = z.shape
    if s["score"] == "softmax":
        p = torch.softmax(z, 1)
    elif s["score"] == "sigmoid":
        p = torch.sigmoid(z)
    else:
        p = torch.logaddexp(z, torch.zeros_like(z)).sqrt()
    keys = p + (s["b"].double() if s["b"] is not None else 0.0)
    order = torch.sort(keys, dim=1, descending=True, stable=True).indices  # the lowest index first among equals
    if s["topk_groups"] < G:
        best = torch.sort(keys.view(T, G, -1), dim=2, descending=True).values[:, :, :2].sum(2)
        rank = torch.argsort(torch.argsort(-best, dim=1, stable=True), dim=1, stable=True)
        out = (rank >= s["topk_groups"]).repeat_interleave(E // G, 1).gather(1, order)
        order = order.gather(1, torch.sort(out.to(torch.int32), dim=1, stable=True).indices)  # chosen groups' first
    idx = order[:, :k]
    zc = z.gather(1, idx)
    top = torch.gather(p, 1, idx)
    weight = top / (top.sum(1, keepdim=True) + 1e-20) if s["renormalize"] else top
    got = {"idx": idx.to(torch.int32), "weight": weight}
    if s["load"]:
        got["load"] = torch.bincount(idx.reshape(-1), minlength=E).to(torch.int32)
    if s["train"]:
        leaf = z.clone().requires_grad_(True)
        with torch.enable_grad():
            if s["score"] == "softmax":
                q = torch.softmax(leaf, 1).gather(1, idx)
            elif s["score"] == "sigmoid":
                q = torch.sigmoid(leaf.gather(1, idx))
            else:
                q = torch.logaddexp(leaf, torch.zeros_like(leaf)).sqrt().gather(1, idx)
            if s["renormalize"]:
                q = q / (q.sum(1, keepdim=True) + 1e-20)
            got["dz"], = torch.autograd.grad(q, leaf, s["dw"].double())
    return got


def _exact_linear(s):
    if s["dtype"] == "e4m3":
        def whole(q, scale, rows):
            q = q.double()
            for i in range(scale.shape[0] if rows > 1 else 0):
                for j in range(scale.shape[1]):
                    q[i * rows:(i + 1) * rows, j * _BLOCK:(j + 1) * _BLOCK] *= scale[i, j].double()
            if rows == 1:
                for j in range(scale.shape[1]):
                    q[:, j * _BLOCK:(j + 1) * _BLOCK] *= scale[:, j:j + 1].double()
            return q
        x, w = whole(s["x"], s["xs"], 1), whole(s["w"], s["ws"], _BLOCK)
    else:
        x, w = s["x"].double(), s["w"].double()
    x.requires_grad_(s["train"])
    w.requires_grad_(s["train"])
    b = None if s["b"] is None else s["b"].double().requires_grad_(s["train"])
    res = None if s["res"] is None else s["res"].double().requires_grad_(s["train"])
    with torch.set_grad_enabled(s["train"]):
        u = x @ w.t()
        if b is not None:
            u = u + b
        f = torch.nn.functional
        v = {"": u, "relu": f.relu(u), "silu": f.silu(u), "gelu": f.gelu(u)}[s["act"]]
        if res is not None:
            v = v + res
    got = {"out": v.detach()}
    if s["train"]:
        leaves = {"dx": x, "dw": w, "db": b, "dres": res}
        leaves = {n: t for n, t in leaves.items() if t is not None}
        got.update(zip(leaves, torch.autograd.grad(v, list(leaves.values()), s["dy"].double())))
    return got
