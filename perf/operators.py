"""Workloads of the expert-layer operators: root-mean-square norm (with the residual's addition,
8-bit output with row scales, and the gradient) and matrix products grouped by expert (forward,
gradient of the inputs, gradient of the weights).

Every case runs in two forms on the same inputs: `own = False` computes it with elementary torch
operations in 32 bits; `own = True` makes the calls a user makes of bwgemm. `exact` states the
operator in 64 bits. A case is a dict of plain values; `prepare` makes its inputs on the GPU.
"""
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-5
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}

_bw = None


def _bwgemm():
    """The framework's Python face (only where the framework's kernels are asked for)."""
    global _bw
    if _bw is None:
        path = os.path.join(os.getcwd(), "blackwell-tensorcore-kernels_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import bwgemm

        _bw = bwgemm
    return _bw


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoded token: the norm in front of a layer's first FP8 product; latency only
        {"name": "norm_fp8_one_token", "op": "norm", "out": "fp8", "dtype": "bf16", "residual": True,
         "rows": 1, "cols": 8192},
        # a small ragged batch whose row length is no multiple of a 16-byte vector
        {"name": "norm_fp8_odd", "op": "norm", "out": "fp8", "dtype": "f16", "residual": True,
         "rows": 777, "cols": 2049},
        # prefill, or one training step's tokens: bound by memory
        {"name": "norm_fp8_prefill", "op": "norm", "out": "fp8", "dtype": "bf16", "residual": True,
         "rows": 16384, "cols": 8192},
        # norm over each attention head of the queries and keys: many short rows, output in the input's type
        {"name": "norm_heads", "op": "norm", "out": "same", "dtype": "bf16", "residual": False,
         "rows": 131072, "cols": 128},
        # gradient in 32 bits on a small ragged batch (fine-tuning, tests of a training loop)
        {"name": "norm_grad_ragged", "op": "norm_grad", "dtype": "f32", "residual": True, "rows": 1000, "cols": 2050},
        # gradient of a training step's tokens
        {"name": "norm_grad_train", "op": "norm_grad", "dtype": "bf16", "residual": True, "rows": 16384, "cols": 8192},
        # one decoded token sent to 8 of 64 experts: eight products of one row, bound by their weights
        {"name": "experts_fp8_one_token", "op": "experts", "dtype": "fp8", "layout": "nk", "experts": 64, "topk": 8,
         "tokens": 1, "n": 4096, "k": 2048, "skew": 0.5},
        # a decode batch: nearly every expert has a few rows, all weights are read once
        {"name": "experts_fp8_decode", "op": "experts", "dtype": "fp8", "layout": "nk", "experts": 64, "topk": 8,
         "tokens": 128, "n": 4096, "k": 2048, "skew": 1.0},
        # prefill: thousands of rows an expert, bound by the tensor cores
        {"name": "experts_fp8_prefill", "op": "experts", "dtype": "fp8", "layout": "nk", "experts": 16, "topk": 4,
         "tokens": 8192, "n": 8192, "k": 4096, "skew": 0.5},
        # training: gradient of the expert layer's inputs, the same weights read in the other layout
        {"name": "experts_bf16_dgrad", "op": "experts", "dtype": "bf16", "layout": "kn", "experts": 8, "topk": 2,
         "tokens": 16384, "n": 2048, "k": 4096, "skew": 0.5},
        # training: gradient of the expert weights, each expert's rows being the summed dimension
        {"name": "experts_bf16_wgrad", "op": "experts_wgrad", "dtype": "bf16", "experts": 8, "topk": 2,
         "tokens": 16384, "n": 2048, "k": 4096, "skew": 0.5},
        # a short training batch over many small experts: odd row counts, some experts without rows
        {"name": "experts_f16_wgrad_ragged", "op": "experts_wgrad", "dtype": "f16", "experts": 32, "topk": 2,
         "tokens": 250, "n": 520, "k": 1032, "skew": 4.0},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "experts", "experts", "experts", "experts_wgrad"])
    if op in ("norm", "norm_grad"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, min(131072, (1 << 27) // cols))
        c = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "residual": rng.random() < 0.7,
             "rows": rows, "cols": cols}
        if op == "norm":
            c["out"] = rng.choice(["fp8", "fp8", "same"])
        elif c["dtype"] == "f32":
            c["rows"] = max(1, rows // 2)
        return c
    experts = rng.choice([1, 3, 8, 16, 32, 60, 64, 128])
    topk = min(experts, rng.choice([1, 2, 4, 8]))
    wide = experts <= 16
    n = _log(rng, 64, 8192 if wide else 4096) // 8 * 8
    k = _log(rng, 64, 4096) // 16 * 16
    tokens = _log(rng, 1, min(8192 * 4 // topk, int(1.0e12 / (2.0 * topk * n * k)) + 1))
    c = {"op": op, "experts": experts, "topk": topk, "tokens": tokens, "n": n, "k": k,
         "skew": rng.choice([0.0, 0.5, 1.0, 2.0])}
    if op == "experts":
        c["dtype"] = rng.choice(["fp8", "fp8", "bf16", "f16"])
        c["layout"] = "nk" if c["dtype"] == "fp8" else rng.choice(["nk", "kn"])
    else:
        c["dtype"] = rng.choice(["bf16", "f16"])
    return c


def _counts(case):
    """Rows of each expert, most popular first: every token goes to `topk` different experts, whose
    popularity falls as exp(-skew * rank / experts). Depends on the case alone."""
    e, t, k = case["experts"], case["tokens"], case["topk"]
    rs = np.random.RandomState(1000003 * e + 1009 * k + t)
    score = rs.gumbel(size=(t, e)) - case["skew"] * np.arange(e) / e
    chosen = np.argpartition(-score, k - 1, axis=1)[:, :k]
    return np.bincount(chosen.reshape(-1), minlength=e)


# ------------------------------------------------------------------ inputs
def _e4m3(x, scale):
    return (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    dtype = DTYPES[case["dtype"]]
    if case["op"] in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        s = dict(case)
        s["weight"] = (1.0 + normal(cols, std=0.1)).to(dtype)
        if case["op"] == "norm":
            s["x"] = normal(rows, cols).to(dtype)
            s["res"] = normal(rows, cols, std=2.0).to(dtype) if case["residual"] else None
        else:
            s["h"] = normal(rows, cols, std=2.0).to(dtype)  # what the forward pass kept
            s["rstd"] = torch.rsqrt(s["h"].float().square().mean(1) + EPS)
            s["dy"] = normal(rows, cols).to(dtype)
            s["dres"] = normal(rows, cols).to(dtype) if case["residual"] else None
        return s
    counts = _counts(case)[np.random.RandomState(seed % (1 << 32)).permutation(case["experts"])]
    ends = np.cumsum(counts)
    rows, n, k = int(ends[-1]), case["n"], case["k"]
    s = dict(case, rows=rows, most=int(counts.max()), counts=[int(c) for c in counts])
    s["offsets"] = torch.tensor([0] + ends.tolist(), dtype=torch.int32, device="cuda")
    a = normal(rows, k)
    if case["op"] == "experts_wgrad":
        s["x"] = a.to(dtype)
        s["dy"] = normal(rows, n).to(dtype)
        return s
    shape = (case["experts"], n, k) if case["layout"] == "nk" else (case["experts"], k, n)
    std = k ** -0.5
    if case["dtype"] == "fp8":  # one scale a row of activations, one a weight matrix
        s["row_scale"] = a.abs().amax(1) / E4M3_MAX
        s["a"] = _e4m3(a, s["row_scale"][:, None])
        s["b"] = torch.empty(shape, dtype=torch.uint8, device="cuda")
        s["group_scale"] = torch.empty(case["experts"], device="cuda")
        for e in range(case["experts"]):
            w = normal(*shape[1:], std=std)
            s["group_scale"][e] = w.abs().amax() / E4M3_MAX
            s["b"][e] = _e4m3(w, s["group_scale"][e])
    else:
        s["a"] = a.to(dtype)
        s["b"] = torch.empty(shape, dtype=dtype, device="cuda")
        for e in range(case["experts"]):
            s["b"][e] = normal(*shape[1:], std=std)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return {"norm": _norm, "norm_grad": _norm_grad, "experts": _experts, "experts_wgrad": _experts_wgrad}[
        state["op"]](state)


def _norm(s):
    """h = x + residual (kept in the input's type); y = h * rsqrt(mean(h^2) + eps) * weight;
    8-bit output: scale = amax(y) / 448 of each row, q = e4m3(y / scale)."""
    x, res, w = s["x"], s["res"], s["weight"]
    if own:
        bw = _bwgemm()
        if s["out"] == "fp8":
            q, scale, h, rstd = bw.rmsnorm_fp8(x, w, residual=res, eps=EPS)
            out = {"q": q.view(torch.float8_e4m3fn), "row_scale": scale, "rstd": rstd}
        else:
            y, h, rstd = bw.rmsnorm(x, w, residual=res, eps=EPS)
            out = {"y": y, "rstd": rstd}
    else:
        h = x if res is None else (x.float() + res.float()).to(x.dtype)
        hf = h.float()
        rstd = 1.0 / torch.sqrt(hf.square().mean(1) + EPS)
        y = hf * rstd[:, None] * w.float()
        if s["out"] == "fp8":
            scale = y.abs().amax(1) / E4M3_MAX
            q = (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            out = {"q": q, "row_scale": scale, "rstd": rstd}
        else:
            out = {"y": y.to(x.dtype), "rstd": rstd}
    if res is not None:
        out["h"] = h
    return out


def _norm_grad(s):
    """With n = h * rstd: dweight = sum over rows of dy * n;
    dx = rstd * (dy * weight - n * mean(dy * weight * n)) + the gradient that reached h directly."""
    h, w, dy, rstd, dres = s["h"], s["weight"], s["dy"], s["rstd"], s["dres"]
    if own:
        dx, dw = _bwgemm().rmsnorm_backward(dy, h, w, rstd, dresidual=dres)
        return {"dx": dx, "dweight": dw}
    n = h.float() * rstd[:, None]
    dyf = dy.float()
    g = dyf * w.float()
    dx = rstd[:, None] * (g - n * (g * n).mean(1, keepdim=True))
    if dres is not None:
        dx = dx + dres.float()
    return {"dx": dx.to(h.dtype), "dweight": (dyf * n).sum(0)}


def _slots(s):
    """Where each row stands in a batch of experts padded to the longest one: (expert, place)."""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    expert = torch.searchsorted(s["offsets"][1:], row, right=True)
    return expert, (row - s["offsets"][expert]).long()


def _padded(s, rows, slots):
    out = torch.zeros(s["experts"], s["most"], rows.shape[1], device="cuda")
    out[slots] = rows.float()
    return out


def _experts(s):
    """c[row] = a[row] x b[expert of row], times the row's and the expert's scale in 8 bits."""
    a, b = s["a"], s["b"]
    fp8 = s["dtype"] == "fp8"
    if own:
        bw = _bwgemm()
        return {"c": bw.gemm_grouped(a, b, s["offsets"], b_transposed=s["layout"] == "nk",
                                     row_scale=s["row_scale"] if fp8 else None,
                                     group_scale=s["group_scale"] if fp8 else None, out_dtype=bw.OUT_BF16)}
    if fp8:
        a, b = a.view(torch.float8_e4m3fn), b.view(torch.float8_e4m3fn)
    slots = _slots(s)
    b = b.float()
    c = torch.bmm(_padded(s, a, slots), b.transpose(1, 2) if s["layout"] == "nk" else b)[slots]
    if fp8:
        c = c * s["row_scale"][:, None] * s["group_scale"][slots[0]][:, None]
    return {"c": c.to(torch.bfloat16)}


def _experts_wgrad(s):
    """dw[expert] = x[its rows]^T x dy[its rows]: zeros where an expert has no rows."""
    if own:
        bw = _bwgemm()
        return {"dw": bw.gemm_grouped_wgrad(s["x"], s["dy"], s["offsets"], out_dtype=bw.OUT_BF16)}
    slots = _slots(s)
    return {"dw": torch.bmm(_padded(s, s["x"], slots).transpose(1, 2), _padded(s, s["dy"], slots)).to(torch.bfloat16)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        if case["op"] == "norm":
            per = size + (2 * size if case["residual"] else 0) + (1 if case["out"] == "fp8" else size)
            return {"bytes": n * per + cols * size + rows * (8 if case["out"] == "fp8" else 4),
                    "flops": n * (7 if case["out"] == "fp8" else 5)}
        per = 3 * size + (size if case["residual"] else 0)
        return {"bytes": n * per + cols * (size + 4) + rows * 4, "flops": n * 10}
    counts = _counts(case)
    rows, n, k = int(counts.sum()), case["n"], case["k"]
    if case["op"] == "experts_wgrad":
        return {"bytes": rows * (n + k) * size + case["experts"] * n * k * 2, "flops": 2 * rows * n * k}
    scales = (rows + case["experts"]) * 4 if case["dtype"] == "fp8" else 0
    active = int((counts > 0).sum())
    return {"bytes": rows * k * size + active * n * k * size + rows * n * 2 + scales + (case["experts"] + 1) * 4,
            "flops": 2 * rows * n * k}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: t.double()  # noqa: E731
    if case["op"] == "norm":
        x, res, w = s["x"], s["res"], d(s["weight"])
        out = {}
        if res is not None:
            # x + residual of two values of one type is exact in 64 bits; h is held in that type
            x = (d(x) + d(res)).to(x.dtype)
            out["h"] = d(x)
        ms = torch.einsum("rc,rc->r", d(x), d(x)) / case["cols"]
        out["rstd"] = (ms + EPS) ** -0.5
        y = torch.einsum("rc,c,r->rc", d(x), w, out["rstd"])
        if case["out"] == "fp8":
            out["row_scale"] = torch.maximum(y.amax(1), -y.amin(1)) / 448
            out["q"] = y / out["row_scale"].unsqueeze(1)
        else:
            out["y"] = y
        return out
    if case["op"] == "norm_grad":
        h, w, dy, r = d(s["h"]), d(s["weight"]), d(s["dy"]), d(s["rstd"])
        inner = torch.einsum("rc,rc,c->r", dy, h, w)  # <dy * w, h>
        dx = torch.einsum("rc,c,r->rc", dy, w, r) - torch.einsum("rc,r->rc", h, r ** 3 * inner / case["cols"])
        if s["dres"] is not None:
            dx += d(s["dres"])
        return {"dx": dx, "dweight": torch.einsum("rc,rc,r->c", dy, h, r)}
    bounds = np.concatenate([[0], np.cumsum(s["counts"])])
    if case["op"] == "experts_wgrad":
        dw = [d(s["x"][i:j]).T @ d(s["dy"][i:j]) for i, j in zip(bounds, bounds[1:])]
        return {"dw": torch.stack(dw)}
    parts = []
    for e, (i, j) in enumerate(zip(bounds, bounds[1:])):
        a, b = s["a"][i:j], s["b"][e]
        if case["dtype"] == "fp8":
            a = d(a.view(torch.float8_e4m3fn)) * d(s["row_scale"][i:j]).unsqueeze(1)
            b = d(b.view(torch.float8_e4m3fn)) * d(s["group_scale"][e])
        parts.append(d(a) @ (d(b).T if case["layout"] == "nk" else d(b)))
    return {"c": torch.cat(parts)}
