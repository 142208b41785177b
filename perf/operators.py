"""Measured operators: microscaled 4-bit experts (MXFP4) and the shared expert's gated feed-forward block.

A case is one call of an operator of this framework, of one of five kinds:

  quant    mxfp4.quant_rows and mxfp4.dequant_rows: rows to e2m1 codes with an e8m0 scale per 32, and back to values
  product  mxfp4.matmul: the product of two MXFP4 matrices, both with their contraction dimension contiguous
  routed   mxfp4.moe_forward_ids: routed SwiGLU experts in MXFP4 from router ids and weights
  gated    ffn.gated: silu(min(g, L)) * clamp(u, -L, L) with [g | u] = x W13^T, the shared expert's block
  train    ffn.gated with its gradients (dx, dW13)

The plain forms compute in fp32 with elementary torch operations; exact() states the definitions in float64. Sizes:
hidden 4096 with 288 experts, top-8 and intermediate 1024 is one rank's shard of the served layer.
"""
from __future__ import annotations

import importlib
import math
import os
import sys

import torch

own = False

LIMIT = 10.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _framework():
    path = os.path.join(_ROOT, "glm-5.3-flash-dgx-spark-vllm-optimization_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    return importlib.import_module("mi355moe")


def listed():
    return [
        # the rows of one decode step before an expert product: the smallest call, where the launch counts
        {"name": "quant_t8", "kind": "quant", "rows": 8, "K": 4096, "dtype": "bf16"},
        # a checkpoint's fp32 rows with an odd row length, converted at load time
        {"name": "quant_odd", "kind": "quant", "rows": 1237, "K": 4099, "dtype": "fp32"},
        # a stacked weight of many experts converted at load time
        {"name": "quant_weights", "kind": "quant", "rows": 32768, "K": 4096, "dtype": "bf16"},
        # one token through a dense projection
        {"name": "product_m1", "kind": "product", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # a ragged batch against a projection whose width is no multiple of a tile, contraction an odd number of blocks
        {"name": "product_m333", "kind": "product", "M": 333, "N": 2050, "K": 2080, "dtype": "fp32"},
        # a long prompt chunk through a dense projection: the largest product
        {"name": "product_m8192", "kind": "product", "M": 8192, "N": 4096, "K": 4096, "dtype": "bf16"},
        # one user's decode step through the routed layer
        {"name": "routed_t1", "kind": "routed", "T": 1, "n": 288, "topk": 8, "K": 4096, "N": 1024, "dtype": "bf16"},
        # 64 streams, one token each: nearly every expert is read for a few rows
        {"name": "routed_t64", "kind": "routed", "T": 64, "n": 288, "topk": 8, "K": 4096, "N": 1024, "dtype": "bf16"},
        # a prompt chunk of odd length
        {"name": "routed_t2047", "kind": "routed", "T": 2047, "n": 288, "topk": 8, "K": 4096, "N": 1024,
         "dtype": "bf16"},
        # the shared expert of one user's decode step
        {"name": "gated_t1", "kind": "gated", "T": 1, "K": 4096, "N": 1024, "dtype": "bf16"},
        # the shared expert over a prompt chunk of odd length
        {"name": "gated_t1791", "kind": "gated", "T": 1791, "K": 4096, "N": 1024, "dtype": "fp16"},
        # a tuning step of a wide shared expert: forward and both gradients, the largest call
        {"name": "train_t8192", "kind": "train", "T": 8192, "K": 4096, "N": 2048, "dtype": "bf16"},
    ]


def draw(rng):
    def log(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(lo, min(hi, step * round(v / step)))

    kind = rng.choice(["quant", "product", "product", "routed", "routed", "gated", "train"])
    if kind == "quant":
        K = log(33, 8192)
        return {"kind": kind, "rows": log(1, (1 << 27) // K), "K": K, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "product":
        N, K = log(24, 4096), log(64, 4096, 32)
        return {"kind": kind, "M": log(1, 8192), "N": N, "K": K, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "routed":
        n = rng.choice([8, 36, 96, 288])
        return {"kind": kind, "T": log(1, 2047), "n": n, "topk": rng.randint(1, 8), "K": log(512, 4096, 32),
                "N": log(128, 1024, 32), "dtype": rng.choice(["bf16", "fp16"])}
    return {"kind": kind, "T": log(1, 8192), "K": log(256, 4096, 8), "N": log(64, 2048, 8),
            "dtype": rng.choice(["bf16", "fp16"])}


# ---------------------------------------------------------------------------------------------- inputs


def _codes(shape, g):
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def _scales(shape, centre, g):
    # a few binades around the centre, as the blocks of a weight or activation matrix have
    return torch.randint(centre - 2, centre + 2, shape, generator=g, device="cuda", dtype=torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    s = {"case": dict(case), "fw": _framework() if own else None}
    if case["kind"] == "quant":
        # rows of different magnitudes with a few outlier columns, as weights and hidden states have
        x = torch.randn(case["rows"], case["K"], generator=g, device="cuda")
        x *= torch.exp(torch.randn(case["rows"], 1, generator=g, device="cuda"))
        x[:, :: max(1, case["K"] // 7)] *= 20.0
        s["x"] = x.to(dt)
    elif case["kind"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"], s["sa"] = _codes((M, K // 2), g), _scales((M, K // 32), 126, g)
        s["w"], s["sw"] = _codes((N, K // 2), g), _scales((N, K // 32), 121, g)
    elif case["kind"] == "routed":
        T, n, k, K, N = case["T"], case["n"], case["topk"], case["K"], case["N"]
        s["x"] = torch.randn(T, K, generator=g, device="cuda").to(dt)
        # scales that bring the gate values to a deviation of 3 to 4, so that some meet the limit
        s["w13"], s["s13"] = _codes((n, 2 * N, K // 2), g), _scales((n, 2 * N, K // 32), 127 - round(math.log2(K) / 2), g)
        s["w2"], s["s2"] = _codes((n, K, N // 2), g), _scales((n, K, N // 32), 122, g)
        score = torch.rand(T, n, generator=g, device="cuda")
        s["ids"] = torch.topk(score, k, dim=1).indices.to(torch.int32)
        s["wts"] = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), -1) * 2.5
        s["plan"] = _plan(s["ids"], n)
        if own:
            s["experts"] = s["fw"].mxfp4.Mxfp4Experts(s["w13"], s["s13"], s["w2"], s["s2"])
    else:
        T, K, N = case["T"], case["K"], case["N"]
        s["x"] = torch.randn(T, K, generator=g, device="cuda").to(dt)
        s["w13"] = (torch.randn(2 * N, K, generator=g, device="cuda") * (3.5 / math.sqrt(K))).to(dt)
        if case["kind"] == "train":
            s["dh"] = torch.randn(T, N, generator=g, device="cuda").to(dt)
            if own:
                s["x"].requires_grad_()
                s["w13"].requires_grad_()
    return s


def _plan(ids, n):
    """The experts that the call reaches, and for each of them the tokens it serves, in rows of one length: (live
    [L], token [L, C], the place of every pair in [L * C])."""
    flat = ids.reshape(-1).long()
    live, which, counts = torch.unique(flat, return_inverse=True, return_counts=True)
    order = torch.argsort(which, stable=True)
    first = torch.cumsum(counts, 0) - counts
    rank = torch.empty_like(flat)
    rank[order] = torch.arange(flat.numel(), device=flat.device) - first[which[order]]
    C = int(counts.max())
    place = which * C + rank
    token = torch.zeros(live.numel() * C, dtype=torch.long, device=flat.device)
    token[place] = torch.arange(flat.numel(), device=flat.device) // ids.shape[1]
    return live, token.reshape(-1, C), place


# ---------------------------------------------------------------------------------------------- plain forms


def _values(codes, scales, K):
    """fp32 values [..., K] of codes [..., ceil(K / 2)] (element 2i in the low four bits) and their block scales."""
    table = torch.tensor(E2M1, dtype=torch.float32, device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :K]
    v = table[c.int()]
    f = torch.where(scales == 255, math.nan, torch.exp2(scales.float() - 127.0))
    return v * f.repeat_interleave(32, -1)[..., :K]


def _rounded(x):
    """fp32 rows as the MXFP4 values nearest to them (ties to even), one power of two per block of 32."""
    rows, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % 32)).reshape(rows, -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1].float() - 3.0).clamp_min(-127.0)
    v = b * torch.exp2(-e)
    a = v.abs()
    q = torch.where(a <= 2.0, torch.round(a * 2.0) / 2.0, torch.where(a <= 4.0, torch.round(a), torch.round(a / 2.0) * 2.0))
    r = torch.sign(v) * q.clamp_max(6.0) * torch.exp2(e)
    return torch.where(torch.isfinite(top), r, math.nan).reshape(rows, -1)[:, :K]


def _act(z):
    g, u = z.chunk(2, -1)
    g, u = g.clamp_max(LIMIT), u.clamp(-LIMIT, LIMIT)
    return g / (1.0 + torch.exp(-g)) * u


def _plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "quant":
        return _rounded(s["x"].float()).to(torch.bfloat16)
    if c["kind"] == "product":
        return (_values(s["a"], s["sa"], c["K"]) @ _values(s["w"], s["sw"], c["K"]).T).to(dt)
    if c["kind"] == "routed":
        live, token, place = s["plan"]
        x = _rounded(s["x"].float())
        h = _act(x[token] @ _values(s["w13"][live], s["s13"][live], c["K"]).transpose(1, 2))
        h = _rounded(h.reshape(-1, c["N"])).reshape(h.shape)
        y = h @ _values(s["w2"][live], s["s2"][live], c["N"]).transpose(1, 2)
        y = y.reshape(-1, c["K"])[place].reshape(c["T"], c["topk"], c["K"])
        return (y * s["wts"][..., None]).sum(1).to(dt)
    x, w = s["x"].float(), s["w13"].float()
    z = x @ w.T
    h = _act(z)
    if c["kind"] == "gated":
        return h.to(dt)
    g, u = z.chunk(2, -1)
    gc, uc, dh = g.clamp_max(LIMIT), u.clamp(-LIMIT, LIMIT), s["dh"].float()
    sg = 1.0 / (1.0 + torch.exp(-gc))
    dg = dh * uc * sg * (1.0 + gc * (1.0 - sg)) * (g <= LIMIT)
    du = dh * gc * sg * (u.abs() <= LIMIT)
    d = torch.cat([dg, du], -1)
    return {"h": h.to(dt), "dx": (d @ w).to(dt), "dw13": (d.T @ x).to(dt)}


# ---------------------------------------------------------------------------------------------- the framework's calls


def run(state):
    if not own:
        return _plain(state)
    s, c = state, state["case"]
    mxfp4, ffn = s["fw"].mxfp4, s["fw"].ffn
    if c["kind"] == "quant":
        q, sc = mxfp4.quant_rows(s["x"])
        return mxfp4.dequant_rows(q, sc, c["K"], out_dtype=torch.bfloat16)
    if c["kind"] == "product":
        return mxfp4.matmul(s["a"], s["sa"], s["w"], s["sw"], out_dtype=DTYPES[c["dtype"]])
    if c["kind"] == "routed":
        return mxfp4.moe_forward_ids(s["experts"], s["x"], s["ids"], s["wts"], limit=LIMIT)
    h = ffn.gated(s["x"], s["w13"], limit=LIMIT)
    if c["kind"] == "gated":
        return h
    dx, dw = torch.autograd.grad(h, (s["x"], s["w13"]), s["dh"])
    return {"h": h, "dx": dx, "dw13": dw}


# ---------------------------------------------------------------------------------------------- work


def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    K = case["K"]
    if case["kind"] == "quant":
        r = case["rows"]
        return {"bytes": r * (K * size + math.ceil(K / 2) + math.ceil(K / 32) + 2 * K), "flops": 0}
    if case["kind"] == "product":
        M, N = case["M"], case["N"]
        return {"bytes": (M + N) * K * 17 / 32 + M * N * size, "flops": 2.0 * M * N * K}
    T, N = case["T"], case["N"]
    if case["kind"] == "routed":
        n, k = case["n"], case["topk"]
        live = n * (1.0 - (1.0 - k / n) ** T)
        return {"bytes": live * 3 * K * N * 17 / 32 + 2 * T * K * size + T * k * 8, "flops": 6.0 * T * k * K * N}
    b = (T * K + 2 * N * K + T * N) * size
    if case["kind"] == "gated":
        return {"bytes": b, "flops": 4.0 * T * K * N}
    return {"bytes": 2 * b, "flops": 12.0 * T * K * N}


# ---------------------------------------------------------------------------------------------- float64


def _unpack64(codes, scales, K):
    even, odd = (codes % 16).long(), torch.div(codes, 16, rounding_mode="floor").long()
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.long, device=codes.device)
    c[..., 0::2], c[..., 1::2] = even, odd
    m, ex = c & 1, (c >> 1) & 3
    mag = torch.where(ex == 0, 0.5 * m.double(), (1.0 + 0.5 * m.double()) * 2.0 ** (ex.double() - 1.0))
    v = torch.where(c >= 8, -mag, mag)[..., :K]
    p = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=codes.device), scales.double() - 127.0)
    block = torch.arange(K, device=codes.device) // 32
    return v * p[..., block]


def _round64(x):
    """float64 rows rounded to MXFP4: the nearest of the eight magnitudes, of two equally near ones the even code."""
    rows, K = x.shape
    out = torch.empty_like(x)
    mags = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)
    mid = (mags[1:] + mags[:-1]) / 2.0
    for k in range(0, K, 2048):
        p = x[:, k:k + 2048]
        w = p.shape[1]
        if w % 32:
            p = torch.cat([p, p.new_zeros(rows, 32 - w % 32)], 1)
        b = p.reshape(rows, -1, 32)
        top = b.abs().max(-1, keepdim=True).values
        # the exponent of the largest value, as the format's fp32 rows have it
        e = torch.floor(torch.log2(top.clamp_min(2.0 ** -149))) - 2.0
        e = torch.where(torch.exp2(e + 3.0) <= top, e + 1.0, torch.where(torch.exp2(e + 2.0) > top, e - 1.0, e))
        s = torch.exp2(e.clamp_min(-127.0))
        a = (b / s).abs()
        below, upto = torch.searchsorted(mid, a.contiguous()), torch.searchsorted(mid, a.contiguous(), right=True)
        code = torch.where(below % 2 == 0, below, upto)
        out[:, k:k + 2048] = (torch.copysign(mags[code], b) * s).reshape(rows, -1)[:, :w]
    return out


def _swiglu64(z, N):
    g = torch.minimum(z[..., :N], z.new_tensor(LIMIT))
    u = torch.maximum(torch.minimum(z[..., N:], z.new_tensor(LIMIT)), z.new_tensor(-LIMIT))
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    s = prepare(case, seed)
    K = case["K"]
    if case["kind"] == "quant":
        return _round64(s["x"].double())
    if case["kind"] == "product":
        return _unpack64(s["a"], s["sa"], K) @ _unpack64(s["w"], s["sw"], K).t().contiguous()
    N = case["N"]
    if case["kind"] == "routed":
        x = _round64(s["x"].double())
        y = torch.zeros(case["T"], K, dtype=torch.float64, device="cuda")
        for e in sorted(set(s["ids"].reshape(-1).tolist())):
            t, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
            h = _swiglu64(x[t] @ _unpack64(s["w13"][e], s["s13"][e], K).t(), N)
            y[t] += (_round64(h) @ _unpack64(s["w2"][e], s["s2"][e], N).t()) * s["wts"][t, slot].double()[:, None]
        return y
    x, w = s["x"].detach().double(), s["w13"].detach().double()
    if case["kind"] == "gated":
        return _swiglu64(x @ w.t(), N)
    # the gradient by the chain rule of torch's own float64 operations
    x.requires_grad_()
    w.requires_grad_()
    h = _swiglu64(x @ w.t(), N)
    dx, dw = torch.autograd.grad(h, (x, w), s["dh"].double())
    return {"h": h, "dx": dx, "dw13": dw}
