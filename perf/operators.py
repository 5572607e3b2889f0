"""The training-step operators that stand beside orth in a model's update, as cases to measure.

Five operators over two families:

  norm    grad_norm(tensors)                        L2 norm over a list of gradients
  clip    clip_grads(tensors, max_norm, out=...)    the list scaled by min(1, max_norm / (norm + 1e-6)), and the norm
  mm      mm_grouped(x, w, offsets)                 y[t] = w[e(t)] x[t], rows sorted by expert, ragged
  wgrad   mm_grouped_wgrad(dy, x, offsets, ...)     dw[e] = sum over e's rows of dy[t] x[t]^T, in fp32
  step    mm_grouped and its backward by autograd   y, dx and dw of one layer of experts

A case is a dict of plain values.  For the products T is the number of rows, E of experts, N and K the expert matrix
(w is [E, N, K]); `skew` spreads the experts' shares (0: even) and `split` seeds them, so that the row counts belong to
the case and their order among the experts to the seed.
"""
import math
import random

import numpy as np
import torch

own = False   # True: run() makes the framework's calls; False: the plain form

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ----

def listed():
    return [
        # the gradients of one small block, once per step: launch latency
        {"name": "norm_block_fp32", "op": "norm", "kind": "fp32", "count": 14, "rows": 768, "cols": 512, "ragged": False},
        # a large model's gradients in their training type: one pass over 2.3 GB
        {"name": "norm_model_bf16", "op": "norm", "kind": "bf16", "count": 64, "rows": 17408, "cols": 1024,
         "ragged": False},
        # clipping one small block: two dependent passes over little data
        {"name": "clip_block_fp32", "op": "clip", "kind": "fp32", "count": 9, "rows": 768, "cols": 512, "ragged": False},
        # hundreds of gradients of odd sizes and both types: matrices, vectors and scalars
        {"name": "clip_ragged_mixed", "op": "clip", "kind": "mixed", "count": 301, "rows": 1411, "cols": 517,
         "ragged": True},
        # a large model's fp32 gradients, far beyond the caches
        {"name": "clip_model_fp32", "op": "clip", "kind": "fp32", "count": 24, "rows": 17408, "cols": 1024,
         "ragged": False},
        # one decoding step of a few requests: every weight is read once for about one row
        {"name": "mm_token_bf16", "op": "mm", "kind": "bf16", "T": 16, "E": 16, "N": 1024, "K": 2048, "skew": 0.5,
         "split": 1},
        # a short prompt over matrices whose sides are no multiples of anything
        {"name": "mm_odd_bf16", "op": "mm", "kind": "bf16", "T": 1537, "E": 24, "N": 1001, "K": 1111, "skew": 1.0,
         "split": 2},
        # a long prompt or a training batch: bound by the products
        {"name": "mm_batch_bf16", "op": "mm", "kind": "bf16", "T": 16384, "E": 8, "N": 5120, "K": 2048, "skew": 0.3,
         "split": 3},
        # weight gradients at the shapes orth takes, many experts with few rows each: bound by the output
        {"name": "wgrad_tall_bf16", "op": "wgrad", "kind": "bf16", "T": 8191, "E": 32, "N": 768, "K": 512, "skew": 1.0,
         "split": 4},
        # weight gradients of wide experts over a large batch: bound by the products
        {"name": "wgrad_batch_fp16", "op": "wgrad", "kind": "fp16", "T": 32768, "E": 8, "N": 5120, "K": 2048,
         "skew": 0.3, "split": 5},
        # one layer's forward and backward over a small ragged batch, some experts empty
        {"name": "step_ragged_fp16", "op": "step", "kind": "fp16", "T": 4099, "E": 12, "N": 1280, "K": 776, "skew": 2.0,
         "split": 6},
        # one layer's forward and backward in earnest
        {"name": "step_batch_bf16", "op": "step", "kind": "bf16", "T": 16384, "E": 16, "N": 2048, "K": 5120, "skew": 0.5,
         "split": 7},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "clip", "mm", "mm", "wgrad", "step"])
    if op in ("norm", "clip"):
        while True:
            case = {"op": op, "kind": rng.choice(["fp32", "bf16", "mixed"]), "count": _log(rng, 1, 400),
                    "rows": _log(rng, 8, 17408), "cols": _log(rng, 8, 1024), "ragged": rng.random() < 0.5}
            if case["count"] * case["rows"] * case["cols"] <= 24 * 17408 * 1024:
                return case
    while True:
        T, E, N, K = _log(rng, 1, 32768), _log(rng, 1, 128), _log(rng, 64, 6144), _log(rng, 64, 6144)
        if rng.random() < 0.6:   # the usual model widths; the rest stay odd
            N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
        if T * N * K <= 16384 * 2048 * 5120 and E * N * K <= 16 * 2048 * 5120:
            return {"op": op, "kind": rng.choice(["bf16", "fp16"]), "T": T, "E": E, "N": N, "K": K,
                    "skew": rng.choice([0.0, 0.5, 1.0, 2.0]), "split": rng.randrange(1 << 20)}


# ---- inputs ----

def _shapes(case):
    """(rows, cols) of each gradient of a list: equal ones, or for a ragged list odd sizes down to single numbers"""
    if not case["ragged"]:
        return [(case["rows"], case["cols"])] * case["count"]
    rng = random.Random(case["count"] * 7919 + case["rows"])
    shapes = []
    for i in range(case["count"]):
        kind = i % 3
        rows = 1 if kind else max(1, int(case["rows"] * rng.uniform(0.05, 1.0)))
        cols = 1 if kind == 2 and rng.random() < 0.2 else max(1, int(case["cols"] * rng.uniform(0.05, 1.0)))
        shapes.append((rows, cols))
    return shapes


def _types(case):
    if case["kind"] == "mixed":
        return [("bf16", "fp32")[i % 2] for i in range(case["count"])]
    return [case["kind"]] * case["count"]


def _counts(case):
    """rows of each expert, in no order of meaning: a multinomial draw over shares exp(skew * normal)"""
    rng = np.random.default_rng(case["split"])
    share = np.exp(case["skew"] * rng.standard_normal(case["E"]))
    return rng.multinomial(case["T"], share / share.sum())


def _flat(tensors, dtype=None):
    """one zeroed buffer per type of `tensors`, and a view into it for each of them, starting on 64 elements"""
    sizes, at = {}, []
    for t in tensors:
        at.append(sizes.get(t.dtype, 0))
        sizes[t.dtype] = at[-1] + -(-t.numel() // 64) * 64
    flat = {d: torch.zeros(n, dtype=dtype or d, device="cuda") for d, n in sizes.items()}
    return list(flat.values()), [flat[t.dtype][a:a + t.numel()].view(t.shape) for t, a in zip(tensors, at)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("norm", "clip"):
        # layers' gradients differ by orders of magnitude; the clipped ones stay in fp16 and bf16 range
        scales = [10.0 ** random.Random(seed * 31 + i).uniform(-4, 0) for i in range(case["count"])]
        grads = [(torch.randn(r, c, device="cuda", generator=g) * s).to(DTYPES[t])
                 for (r, c), t, s in zip(_shapes(case), _types(case), scales)]
        state = {"op": case["op"], "grads": grads, "max_norm": 1.0}
        if case["op"] == "clip":
            # the clipped gradients go to one flat buffer per type, as an optimizer keeps them
            state["flat"], state["out"] = _flat(grads)
        return state
    dt = DTYPES[case["kind"]]
    T, E, N, K = case["T"], case["E"], case["N"], case["K"]
    counts = np.random.default_rng(seed).permutation(_counts(case))
    state = {"op": case["op"], "offsets": torch.tensor(np.cumsum(counts), dtype=torch.int32, device="cuda"),
             "most": int(counts.max())}
    # unit activations and 1/sqrt(K) weights, as after a norm and at initialisation
    state["x"] = torch.randn(T, K, device="cuda", generator=g).to(dt)
    if case["op"] != "wgrad":
        state["w"] = (torch.randn(E, N, K, device="cuda", generator=g) / math.sqrt(K)).to(dt)
    if case["op"] != "mm":
        state["dy"] = (torch.randn(T, N, device="cuda", generator=g) * 0.1).to(dt)
    if case["op"] == "step":
        state["x"].requires_grad_(True)
        state["w"].requires_grad_(True)
    return state


# ---- one pass ----

def _rows(offsets, T):
    """expert of each row, and the row's place within its expert"""
    t = torch.arange(T, device=offsets.device)
    e = torch.searchsorted(offsets, t.to(offsets.dtype), right=True)
    return e, t - torch.cat([offsets.new_zeros(1), offsets])[e]


def _padded(x, e, p, E, most):
    full = torch.zeros(E, most, x.shape[1], device=x.device)
    full[e, p] = x.float()
    return full


def _plain_products(s):
    x, off = s["x"].detach(), s["offsets"]
    e, p = _rows(off, x.shape[0])
    E, most = off.shape[0], s["most"]
    xp = _padded(x, e, p, E, most)
    if s["op"] == "mm":
        return torch.bmm(xp, s["w"].float().transpose(1, 2))[e, p].to(x.dtype)
    dyp = _padded(s["dy"], e, p, E, most)
    dw = torch.bmm(dyp.transpose(1, 2), xp)
    if s["op"] == "wgrad":
        return dw
    wf = s["w"].detach().float()
    y = torch.bmm(xp, wf.transpose(1, 2))[e, p].to(x.dtype)
    return y, torch.bmm(dyp, wf)[e, p].to(x.dtype), dw.to(x.dtype)


def _plain_lists(s):
    norm = torch.stack([t.float().square().sum(dtype=torch.float64) for t in s["grads"]]).sum().sqrt()
    if s["op"] == "norm":
        return norm.float()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    torch._foreach_copy_(s["out"], [t.float() * coef for t in s["grads"]])
    return s["flat"], norm.float()


def run(state):
    if not own:
        return _plain_lists(state) if state["op"] in ("norm", "clip") else _plain_products(state)
    import spanqr_b200 as spq
    op = state["op"]
    if op == "norm":
        return spq.grad_norm(state["grads"])
    if op == "clip":
        _, norm = spq.clip_grads(state["grads"], state["max_norm"], out=state["out"])
        return state["flat"], norm
    if op == "mm":
        return spq.mm_grouped(state["x"], state["w"], state["offsets"])
    if op == "wgrad":
        return spq.mm_grouped_wgrad(state["dy"], state["x"], state["offsets"], dtype=torch.float32)
    y = spq.mm_grouped(state["x"], state["w"], state["offsets"])
    dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
    return y.detach(), dx, dw


# ---- what a pass cannot do without ----

def work(case):
    if case["op"] in ("norm", "clip"):
        size = {"fp32": 4, "bf16": 2}
        n = sum(r * c for r, c in _shapes(case))
        b = sum(r * c * size[t] for (r, c), t in zip(_shapes(case), _types(case)))
        return {"bytes": b + 4, "flops": 2 * n} if case["op"] == "norm" else {"bytes": 2 * b + 4, "flops": 3 * n}
    T, E, N, K = case["T"], case["E"], case["N"], case["K"]
    used = int((_counts(case) > 0).sum())   # the weights of an expert without rows are not read
    x, y, w = 2 * T * K, 2 * T * N, 2 * used * N * K
    if case["op"] == "mm":
        return {"bytes": x + w + y + 4 * E, "flops": 2 * T * N * K}
    if case["op"] == "wgrad":
        return {"bytes": x + y + 4 * E * N * K + 4 * E, "flops": 2 * T * N * K}
    return {"bytes": 2 * (x + y) + w + 2 * E * N * K + 4 * E, "flops": 6 * T * N * K}


# ---- the definition in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "clip"):
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for t in s["grads"]:
            v = t.double().flatten()
            total += torch.dot(v, v)
        norm = total.sqrt()
        if case["op"] == "norm":
            return norm
        scale = min(1.0, s["max_norm"] / (norm.item() + 1e-6))
        flat, views = _flat(s["grads"], torch.float64)
        for t, v in zip(s["grads"], views):
            v.copy_(t.double() * scale)
        return flat, norm
    x, ends = s["x"].detach(), s["offsets"].tolist()
    T, E, N, K = case["T"], case["E"], case["N"], case["K"]
    y = torch.zeros(T, N, dtype=torch.float64, device="cuda")
    dx = torch.zeros(T, K, dtype=torch.float64, device="cuda")
    dw = torch.zeros(E, N, K, dtype=torch.float64, device="cuda")
    begin = 0
    for e, end in enumerate(ends):
        rows = slice(begin, end)
        begin = end
        xe = x[rows].double()
        if "w" in s:
            we = s["w"][e].detach().double()
            y[rows] = torch.einsum("tk,nk->tn", xe, we)
        if "dy" in s:
            dye = s["dy"][rows].double()
            dw[e] = torch.einsum("tn,tk->nk", dye, xe)
            if "w" in s:
                dx[rows] = torch.einsum("tn,nk->tk", dye, we)
    return {"mm": y, "wgrad": dw, "step": (y, dx, dw)}[case["op"]]
