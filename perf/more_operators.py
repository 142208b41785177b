"""Measured operators: tokens sorted by expert and back, the dense product with its epilogue, and the norms around a block.

A case is one pass through an operator of this framework, of one of seven kinds:

  sort        dispatch.sort_tokens and dispatch.to_experts: the pairs of a router's ids in expert order, their tokens' rows
  back        dispatch.from_experts: the experts' rows weighted and summed per token, onto the shared expert's output
  move        both ways and both gradients, as a tuning step of routed experts has them
  linear      ffn.linear: act(x W^T + bias) + residual
  linear_train   the same with the gradients of x, W, bias (the residual's is the output's own)
  norm        norm.join: the norm after a block, its gate, the scaled residual sum, the norm before the next block
  norm_train  the same with the gradients of the branch, the residual, the gate and both weights

The plain forms compute in fp32 with elementary torch operations; exact() states the definitions in float64. Hidden 4096 with
288 experts, top-8 and intermediate 1024 is one rank's shard of the served layer.
"""
from __future__ import annotations

import importlib
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _framework():
    path = os.path.join(_ROOT, "glm-5.3-flash-dgx-spark-vllm-optimization_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    return importlib.import_module("mi355moe")


def listed():
    return [
        # one user's decode step: eight copies of one token, where the launches count
        {"name": "sort_t1", "kind": "sort", "T": 1, "topk": 8, "n": 288, "total": 288, "H": 4096, "dtype": "bf16"},
        # a long prompt chunk before experts of another kind
        {"name": "sort_t8192", "kind": "sort", "T": 8192, "topk": 8, "n": 288, "total": 288, "H": 4096, "dtype": "bf16"},
        # a ragged batch on an expert-parallel rank that holds a third of the experts, odd row length
        {"name": "back_odd", "kind": "back", "T": 517, "topk": 6, "n": 96, "total": 288, "H": 2051, "shared": True, "dtype": "fp16"},
        # a tuning step of the routed experts: out and back, forward and backward
        {"name": "move_t4096", "kind": "move", "T": 4096, "topk": 8, "n": 288, "total": 288, "H": 4096, "shared": True, "dtype": "bf16"},
        # the shared expert's down projection onto the residual stream, one token
        {"name": "linear_m1", "kind": "linear", "M": 1, "N": 4096, "K": 1024, "bias": False, "act": None, "residual": True, "dtype": "bf16"},
        # a dense layer over a prompt chunk of odd length
        {"name": "linear_m1791", "kind": "linear", "M": 1791, "N": 1024, "K": 4096, "bias": True, "act": "silu", "residual": False,
         "dtype": "fp16"},
        # sizes that are no multiple of anything
        {"name": "linear_odd", "kind": "linear", "M": 333, "N": 2051, "K": 1027, "bias": True, "act": "gelu", "residual": True, "dtype": "bf16"},
        # a tuning step of a dense layer: the largest product
        {"name": "linear_train_m8192", "kind": "linear_train", "M": 8192, "N": 4096, "K": 2048, "bias": True, "act": "gelu_tanh",
         "residual": True, "dtype": "bf16"},
        # between two blocks of one user's decode step
        {"name": "norm_t1", "kind": "norm", "rows": 1, "H": 4096, "gate": "channel", "post": True, "dtype": "bf16", "weights": "bf16"},
        # a ragged batch with one gate value a token, odd row length, fp32 weights
        {"name": "norm_odd", "kind": "norm", "rows": 1237, "H": 4099, "gate": "token", "post": True, "dtype": "fp16", "weights": "fp32"},
        # a long prompt without a gate
        {"name": "norm_t16384", "kind": "norm", "rows": 16384, "H": 4096, "gate": "none", "post": True, "dtype": "bf16", "weights": "bf16"},
        # a tuning step with a gate of a value a channel
        {"name": "norm_train_t8192", "kind": "norm_train", "rows": 8192, "H": 4096, "gate": "channel", "post": True, "dtype": "bf16",
         "weights": "fp32"},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["sort", "back", "move", "linear", "linear", "linear_train", "norm", "norm", "norm_train"])
    if kind in ("sort", "back", "move"):
        total = rng.choice([8, 60, 96, 288, 512])
        n = total if rng.random() < 0.6 else max(1, total // rng.choice([2, 3, 8]))
        c = {"kind": kind, "T": log(1, 4096 if kind == "move" else 8192), "topk": rng.randint(1, 8), "n": n, "total": total,
             "H": log(64, 4096), "dtype": rng.choice(["bf16", "fp16"] if kind == "move" else ["bf16", "bf16", "fp16", "fp32"])}
        if c["dtype"] == "fp32":
            c["T"] = min(c["T"], 4096)
        if kind != "sort":
            c["shared"] = rng.random() < 0.5
        return c
    if kind in ("linear", "linear_train"):
        even = 1 if rng.random() < 0.3 else 8
        K = -(-log(32, 4096 if kind == "linear" else 2048) // even) * even
        N = -(-log(16, 4096) // even) * even
        return {"kind": kind, "M": log(1, 8192), "N": N, "K": K, "bias": rng.random() < 0.6,
                "act": rng.choice([None, "relu", "silu", "gelu", "gelu_tanh"]), "residual": rng.random() < 0.6,
                "dtype": rng.choice(["bf16", "fp16"])}
    H = log(64, 8192)
    if rng.random() < 0.7:
        H = -(-H // 8) * 8
    most = (1 << 26 if kind == "norm" else 1 << 25) // H
    return {"kind": kind, "rows": log(1, min(most, 32768)), "H": H, "gate": rng.choice(["none", "channel", "token", "full"]),
            "post": rng.random() < 0.8, "dtype": rng.choice(["bf16", "fp16"]), "weights": rng.choice(["fp32", "same"])}


# ---------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": dict(case), "fw": _framework() if own else None, "leaves": []}
    train = case["kind"] in ("move", "linear_train", "norm_train")
    if case["kind"] in ("sort", "back", "move"):
        T, k, n, total, H = case["T"], case["topk"], case["n"], case["total"], case["H"]
        # picks without repetition where there are enough experts, some experts taken far more often than others
        score = torch.rand(T, total, generator=g, device="cuda") + 0.3 * torch.rand(total, generator=g, device="cuda")
        s["ids"] = torch.topk(score, min(k, total), dim=1).indices.to(torch.int32)
        s["map"] = None
        if n < total:       # this rank's experts are every (total / n)-th
            m = torch.full((total,), -1, dtype=torch.int64, device="cuda")
            m[torch.arange(n, device="cuda") * (total // n)] = torch.arange(n, device="cuda")
            s["map"] = m
        s["weights"] = torch.softmax(normal(*s["ids"].shape), -1) * 2.5
        s["row"] = _sorted(s["ids"], s["map"], n)[0]
        if own:
            s["plan"] = s["fw"].dispatch.sort_tokens(s["ids"], n, expert_map=s["map"])
        if case["kind"] != "back":
            s["x"] = normal(T, H).to(dt)
        if case["kind"] != "sort":
            s["y"] = normal(s["ids"].numel(), H).to(dt)
            s["shared"] = normal(T, H).to(dt) if case["shared"] else None
        if train:
            s["d_rows"], s["d_out"] = normal(s["ids"].numel(), H).to(dt), normal(T, H).to(dt)
            s["leaves"] = ["x", "y", "weights"]
    elif case["kind"] in ("linear", "linear_train"):
        M, N, K = case["M"], case["N"], case["K"]
        s["x"], s["w"] = normal(M, K).to(dt), (normal(N, K) * (1.5 / math.sqrt(K))).to(dt)
        s["bias"] = (0.5 * normal(N)).to(dt) if case["bias"] else None
        s["residual"] = normal(M, N).to(dt) if case["residual"] else None
        if train:
            s["dy"] = normal(M, N).to(dt)
            s["leaves"] = ["x", "w"] + (["bias"] if case["bias"] else [])
    else:
        R, H = case["rows"], case["H"]
        wt = dt if case["weights"] == "same" else DTYPES[case["weights"]]
        # a block's output and the residual stream it joins, with a few channels far larger than the others
        s["branch"], s["residual"] = normal(R, H), normal(R, H) * 2.0
        s["residual"][:, :: max(1, H // 5)] *= 12.0
        s["branch"], s["residual"] = s["branch"].to(dt), s["residual"].to(dt)
        s["post"] = (1.0 + 0.2 * normal(H)).to(wt) if case["post"] else None
        s["pre"] = (1.0 + 0.2 * normal(H)).to(wt)
        shape = {"none": None, "channel": (H,), "token": (R, 1), "full": (R, H)}[case["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(normal(*shape)).to(dt)
        s["scale"], s["residual_scale"] = 0.5, 1.25
        if train:
            s["ds"], s["dy"] = normal(R, H).to(dt), normal(R, H).to(dt)
            s["leaves"] = [k for k in ("branch", "residual", "post", "gate", "pre") if s[k] is not None]
    if own and train:
        for k in s["leaves"]:
            s[k].requires_grad_()
    return s


def _sorted(ids, expert_map, n):
    """(row [T, topk], pair [P], offsets [n + 1]), int32: the place of every pair in expert order, what is no local expert's
    behind the others and as ~place, and the inverse; where each expert's rows begin."""
    local = ids.reshape(-1).long()
    if expert_map is not None:
        local = expert_map[local]
    local = torch.where((local >= 0) & (local < n), local, n)
    order = torch.argsort(local, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    counts = (local[:, None] == torch.arange(n, device=local.device)).sum(0) if local.numel() * n < 1 << 26 else torch.bincount(local, minlength=n + 1)[:n]
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)])
    row = torch.where(local < n, place, -1 - place)
    pair = torch.where(local[order] < n, order, -1 - order)
    return row.to(torch.int32).reshape(ids.shape), pair.to(torch.int32), offsets.to(torch.int32)


# ---------------------------------------------------------------------------------------------- plain forms


def _act(z, act):
    """(act(z), act'(z))."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0.0), (z > 0).to(z.dtype)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    a = math.sqrt(2.0 / math.pi)
    t = torch.tanh(a * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * a * (1.0 + 3 * 0.044715 * z * z)


def _plain_move(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    k = s["ids"].shape[1]
    if c["kind"] == "back":
        row = s["row"].long()
    else:
        row, pair, offsets = _sorted(s["ids"], s["map"], c["n"])
        token = torch.where(pair >= 0, pair, -1 - pair).long() // k
        rows = (s["x"].float()[token] * (pair >= 0)[:, None]).to(dt)
        if c["kind"] == "sort":
            return {"rows": rows, "row": row, "pair": pair, "offsets": offsets}
        row = row.long()
    here = row >= 0
    at = torch.where(here, row, -1 - row)
    w = torch.where(here, s["weights"], 0.0)
    y = s["y"].float()[at] * here[..., None]
    out = (y * w[..., None]).sum(1)
    if s["shared"] is not None:
        out = out + s["shared"].float()
    if c["kind"] == "back":
        return out.to(dt)
    d_out = s["d_out"].float()
    dx = (s["d_rows"].float()[at] * here[..., None]).sum(1)
    dw = (y * d_out[:, None, :]).sum(-1)
    dy = torch.empty_like(s["y"])
    dy[at.reshape(-1)] = (w[..., None] * d_out[:, None, :]).reshape(-1, c["H"]).to(dt)
    return {"rows": rows, "out": out.to(dt), "dx": dx.to(dt), "dy": dy, "dweights": dw}


def _plain_linear(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.T
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if c["kind"] == "linear":
        return y.to(dt)
    dz = s["dy"].float() * slope
    out = {"y": y.to(dt), "dx": (dz @ w).to(dt), "dw": (dz.T @ x).to(dt)}
    if s["bias"] is not None:
        out["dbias"] = dz.sum(0).to(dt)
    return out


def _rms(v):
    return 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _plain_norm(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    b, res = s["branch"].float(), s["residual"].float()
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    rb = _rms(b) if s["post"] is not None else 1.0
    post = s["post"].float() if s["post"] is not None else 1.0
    pre = s["pre"].float()
    nb = b * rb
    u = nb * post
    t = s["residual_scale"] * res + s["scale"] * gate * u
    rs = _rms(t)
    nt = t * rs
    out = {"s": t.to(dt), "y": (nt * pre).to(dt)}
    if c["kind"] == "norm":
        return out
    dn = s["dy"].float() * pre
    gt = s["ds"].float() + rs * (dn - nt * (nt * dn).mean(-1, keepdim=True))
    out["dresidual"] = (s["residual_scale"] * gt).to(dt)
    out["dpre"] = (s["dy"].float() * nt).sum(0).to(s["pre"].dtype)
    if s["gate"] is not None:
        dg = s["scale"] * gt * u
        out["dgate"] = (dg.sum(0) if c["gate"] == "channel" else dg.sum(-1, keepdim=True) if c["gate"] == "token" else dg).to(dt)
    du = s["scale"] * gate * gt
    if s["post"] is not None:
        out["dpost"] = (du * nb).sum(0).to(s["post"].dtype)
        du = du * post
        du = rb * (du - nb * (nb * du).mean(-1, keepdim=True))
    out["dbranch"] = du.to(dt)
    return out


# ---------------------------------------------------------------------------------------------- the framework's calls


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return _plain_move(s) if kind in ("sort", "back", "move") else _plain_linear(s) if kind in ("linear", "linear_train") else _plain_norm(s)
    fw = s["fw"]
    if kind == "back":
        return fw.dispatch.from_experts(s["y"], s["weights"], s["plan"], shared=s["shared"])
    if kind in ("sort", "move"):
        plan = fw.dispatch.sort_tokens(s["ids"], c["n"], expert_map=s["map"])
        rows = fw.dispatch.to_experts(s["x"], plan)
        if kind == "sort":
            return {"rows": rows, "row": plan.row, "pair": plan.pair, "offsets": plan.offsets}
        out = fw.dispatch.from_experts(s["y"], s["weights"], plan, shared=s["shared"])
        dx, dy, dw = torch.autograd.grad((rows, out), (s["x"], s["y"], s["weights"]), (s["d_rows"], s["d_out"]))
        return {"rows": rows, "out": out, "dx": dx, "dy": dy, "dweights": dw}
    if kind in ("linear", "linear_train"):
        y = fw.ffn.linear(s["x"], s["w"], bias=s["bias"], activation=c["act"], residual=s["residual"])
        if kind == "linear":
            return y
        grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
        return {"y": y, **{"d" + k: v for k, v in zip(s["leaves"], grads)}}
    t, y = fw.norm.join(s["branch"], s["residual"], post=s["post"], gate=s["gate"], pre=s["pre"], eps=EPS, scale=s["scale"],
                        residual_scale=s["residual_scale"])
    if kind == "norm":
        return {"s": t, "y": y}
    grads = dict(zip(s["leaves"], torch.autograd.grad((t, y), [s[k] for k in s["leaves"]], (s["ds"], s["dy"]))))
    out = {"s": t, "y": y, "dresidual": grads["residual"], "dpre": grads["pre"]}
    if s["gate"] is not None:
        out["dgate"] = grads["gate"]
    if s["post"] is not None:
        out["dpost"] = grads["post"]
    out["dbranch"] = grads["branch"]
    return out


# ---------------------------------------------------------------------------------------------- work


def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    kind = case["kind"]
    if kind in ("sort", "back", "move"):
        T, H, k = case["T"], case["H"], min(case["topk"], case["total"])
        P = T * k
        live = P * case["n"] / case["total"]          # the pairs that a local expert takes
        shared = T * H * size if case.get("shared") else 0
        if kind == "sort":
            return {"bytes": 12 * P + T * H * size + P * H * size, "flops": 0}
        if kind == "back":
            return {"bytes": 8 * P + (live + T) * H * size + shared, "flops": 2.0 * live * H}
        return {"bytes": 24 * P + (4 * T + 2 * P + 3 * live) * H * size + shared, "flops": 7.0 * live * H}
    if kind in ("linear", "linear_train"):
        M, N, K = case["M"], case["N"], case["K"]
        b = (M * K + N * K + M * N * (2 if case["residual"] else 1)) * size
        if kind == "linear":
            return {"bytes": b, "flops": 2.0 * M * N * K}
        return {"bytes": b + (M * K + N * K + M * N) * size, "flops": 6.0 * M * N * K}
    R, H = case["rows"], case["H"]
    gate = {"none": 0, "channel": H, "token": R, "full": R * H}[case["gate"]] * size
    b = 4 * R * H * size + 2 * H * 4 + gate
    if kind == "norm":
        return {"bytes": b, "flops": 12.0 * R * H}
    return {"bytes": b + 4 * R * H * size + 2 * H * 4 + gate, "flops": 40.0 * R * H}


# ---------------------------------------------------------------------------------------------- float64


def _exact_move(s):
    c = s["case"]
    T, H, n = c["T"], c["H"], c["n"]
    ids = s["ids"].cpu().numpy()
    k = ids.shape[1]
    where = None if s["map"] is None else s["map"].cpu().numpy()
    # the pairs of expert 0, then those of expert 1, ...: by counting, pair after pair
    local = ids.reshape(-1) if where is None else where[ids.reshape(-1)]
    taken = np.flatnonzero((local >= 0) & (local < n))
    in_order = taken[np.lexsort((taken, local[taken]))]
    P = local.size
    row = np.full(P, -1, dtype=np.int64)
    row[in_order] = np.arange(in_order.size)
    slots = torch.from_numpy(row.reshape(T, k)).cuda()
    tok = torch.from_numpy(in_order // k).cuda()
    live = in_order.size
    rows = torch.zeros(P, H, dtype=torch.float64, device="cuda") if c["kind"] != "back" else None
    if rows is not None:
        rows[:live] = s["x"].detach().double()[tok]
    if c["kind"] == "sort":
        return {"rows": rows, "row": None, "pair": None, "offsets": None}
    w, y = s["weights"].detach().double(), s["y"].detach()
    out = torch.zeros(T, H, dtype=torch.float64, device="cuda") if s["shared"] is None else s["shared"].double()
    dx = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    dw = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    dy = torch.zeros(P, H, dtype=torch.float64, device="cuda") if c["kind"] == "move" else None
    for j in range(k):
        t = torch.nonzero(slots[:, j] >= 0).reshape(-1)
        r = slots[t, j]
        v = y[r].double()
        out[t] += w[t, j, None] * v
        if dy is not None:
            d = s["d_out"][t].double()
            dx[t] += s["d_rows"][r].double()
            dw[t, j] = (v * d).sum(-1)
            dy[r] = w[t, j, None] * d
    return out if dy is None else {"rows": rows, "out": out, "dx": dx, "dy": dy, "dweights": dw}


def _exact_norm(s, leaf):
    gate = leaf["gate"] if s["gate"] is not None else 1.0
    u = leaf["branch"]
    H = u.shape[-1]
    if s["post"] is not None:
        u = u / torch.sqrt(u.square().sum(-1, keepdim=True) / H + EPS) * leaf["post"]
    t = leaf["residual"] * s["residual_scale"] + gate * u * s["scale"]
    return t, t / torch.sqrt(t.square().sum(-1, keepdim=True) / H + EPS) * leaf["pre"]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("sort", "back", "move"):
        return _exact_move(s)
    names = ("x", "w", "bias", "residual") if kind in ("linear", "linear_train") else ("branch", "residual", "post", "gate", "pre")
    leaf = {k: s[k].detach().double() for k in names if s[k] is not None}
    train = kind.endswith("train")
    if train:       # the gradients by the chain rule of torch's own float64 operations
        for k in s["leaves"]:
            leaf[k].requires_grad_()
    if kind in ("linear", "linear_train"):
        z = leaf["x"] @ leaf["w"].t()
        if "bias" in leaf:
            z = z + leaf["bias"]
        f = torch.nn.functional
        y = {None: lambda v: v, "relu": f.relu, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[case["act"]](z)
        if "residual" in leaf:
            y = y + leaf["residual"]
        if not train:
            return y
        grads = torch.autograd.grad(y, [leaf[k] for k in s["leaves"]], s["dy"].double())
        return {"y": y.detach(), **{"d" + k: v for k, v in zip(s["leaves"], grads)}}
    t, y = _exact_norm(s, leaf)
    if not train:
        return {"s": t, "y": y}
    grads = torch.autograd.grad((t, y), [leaf[k] for k in s["leaves"]], (s["ds"].double(), s["dy"].double()))
    return {"s": t.detach(), "y": y.detach(), **{"d" + k: v for k, v in zip(s["leaves"], grads)}}
