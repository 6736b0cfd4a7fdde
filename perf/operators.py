"""Workloads of the expert operators (``nerf_amd.expert_ops``: rows grouped by expert, the experts' matrix products and
their gradients) and of the orthogonalised update (``nerf_amd.muon_ops``: Newton-Schulz products, the Muon step).

A workload is a dict of plain values.  ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass through
an operator: in elementary torch operations at 32 bits where ``own`` is false, through the framework's kernels where it is
true.  ``exact`` gives the same outputs from the definition in 64 bits, ``work`` the bytes and operations of a pass.

Definitions.  Row i of a batch belongs to expert index[i]; an index outside [0, E) belongs to no expert.

  plan      counts[e] = |{i : index[i] = e}|, offsets = exclusive sums of counts (E + 1 of them), order = the rows of
            expert 0, 1, ... E - 1, each expert's in ascending order, then the rows of no expert in ascending order.
  linear    y[i] = act(W[index[i]] x[i] + b[index[i]]), 0 for a row of no expert.
  backward  dz[i] = dy[i] (y[i] > 0 if act is relu); dx[i] = W[index[i]]^T dz[i]; dW[e] = sum_{index[i] = e} dz[i] x[i]^T;
            db[e] = sum_{index[i] = e} dz[i].
  schulz    X = G / max(|G|_F, eps); five times X <- a X + (b A + c A^2) X with A = X X^T.
  muon      g = clamp(grad, +-clip); buf <- mu buf + g; O = schulz(g + mu buf);
            p <- (1 - lr wd) p - lr sqrt(max(1, rows / columns)) O.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
MUON = {"lr": 0.02, "momentum": 0.95, "weight_decay": 0.01, "clip_value": 40.0}
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the routing of a training step's few thousand samples over a small set of experts: launch latency
        {"name": "plan_step", "op": "plan", "rows": 2048, "experts": 64, "spread": "router"},
        # a rendered frame's samples over the 16^3 cells of a scene, three quarters of them empty, some samples outside
        {"name": "plan_frame", "op": "plan", "rows": 2000003, "experts": 4096, "spread": "cells"},
        # single tokens of 48 requests through one expert layer: the experts' weights are read once, a row or two each
        {"name": "linear_tokens", "op": "linear", "rows": 48, "experts": 32, "inputs": 1024, "outputs": 2048,
         "dtype": "bf16", "act": "none", "spread": "router"},
        # the first layer of 4096 tiny per-cell networks over a batch of samples: 63 encoding channels -> 32, relu
        {"name": "linear_cells", "op": "linear", "rows": 262147, "experts": 4096, "inputs": 63, "outputs": 32,
         "dtype": "fp32", "act": "relu", "spread": "cells"},
        # a long prompt batch through one expert layer
        {"name": "linear_prompt", "op": "linear", "rows": 32768, "experts": 32, "inputs": 2048, "outputs": 2048,
         "dtype": "bf16", "act": "none", "spread": "router"},
        # the hidden layer of the tiny per-cell networks in a training step
        {"name": "backward_cells", "op": "backward", "rows": 131071, "experts": 4096, "inputs": 32, "outputs": 32,
         "dtype": "fp32", "act": "relu", "spread": "cells"},
        # a few wide experts with the widths of the 8x256 network's skip layer (319 -> 256), fp32
        {"name": "backward_skip", "op": "backward", "rows": 20011, "experts": 8, "inputs": 319, "outputs": 256,
         "dtype": "fp32", "act": "relu", "spread": "router"},
        # a training batch through one expert layer in half precision
        {"name": "backward_batch", "op": "backward", "rows": 16384, "experts": 16, "inputs": 1024, "outputs": 1536,
         "dtype": "fp16", "act": "relu", "spread": "router"},
        # the first-layer gradients of every cell of a 16^3 grid, 32 x 63 each
        {"name": "schulz_cells", "op": "schulz", "batch": 4096, "m": 32, "n": 63, "dtype": "fp32"},
        # wide projections of a larger network
        {"name": "schulz_wide", "op": "schulz", "batch": 2, "m": 1024, "n": 4096, "dtype": "bf16"},
        # the view layers (128 x 283) of the coarse and the fine network: the smallest update
        {"name": "muon_views", "op": "muon", "batch": 2, "m": 128, "n": 283, "dtype": "fp32"},
        # the seven 256 x 256 layers of the coarse and the fine network
        {"name": "muon_hidden", "op": "muon", "batch": 14, "m": 256, "n": 256, "dtype": "fp32"},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["plan", "linear", "linear", "backward", "backward", "schulz", "muon"])
    if op == "plan":
        return {"op": op, "rows": _between(rng, 1, 2000003), "experts": _between(rng, 1, 4096),
                "spread": rng.choice(["router", "cells"])}
    if op in ("linear", "backward"):
        act = rng.choice(["none", "relu"])
        kind = rng.choice(["tokens", "batch", "cells"])
        if kind == "cells":      # thousands of tiny networks
            return {"op": op, "rows": _between(rng, 5000, 262147), "experts": _between(rng, 256, 4096),
                    "inputs": _between(rng, 3, 64), "outputs": _between(rng, 3, 64), "dtype": "fp32", "act": act,
                    "spread": "cells"}
        if kind == "tokens":     # fewer rows than the experts' widths: the weights are what is moved
            return {"op": op, "rows": _between(rng, 1, 256), "experts": _between(rng, 2, 32),
                    "inputs": _between(rng, 64, 1024), "outputs": _between(rng, 64, 2048),
                    "dtype": rng.choice(["fp32", "bf16", "fp16"]), "act": act, "spread": "router"}
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        most = 512 if dtype == "fp32" else 2048
        return {"op": op, "rows": _between(rng, 512, 16384), "experts": _between(rng, 2, 32),
                "inputs": _between(rng, 64, most), "outputs": _between(rng, 64, most), "dtype": dtype, "act": act,
                "spread": "router"}
    if rng.random() < 0.5:       # many small matrices
        m, n, batch = _between(rng, 1, 32), _between(rng, 1, 64), _between(rng, 1, 4096)
    else:                        # a few larger ones
        m, n, batch = _between(rng, 33, 640), _between(rng, 33, 1024), _between(rng, 1, 8)
    if rng.random() < 0.3:
        m, n = n, m
    return {"op": op, "batch": batch, "m": m, "n": n,
            "dtype": "fp32" if op == "muon" else rng.choice(["fp32", "fp32", "bf16", "fp16"])}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _routing(case, g):
    """int32 expert of every row.  "router": uneven popularity; "cells": samples of a scene that fills a quarter of its
    grid, neighbouring rows in the same cell, one in fifty outside the grid."""
    n, experts = case["rows"], case["experts"]
    if case["spread"] == "router":
        popularity = torch.exp(0.7 * torch.randn(experts, device="cuda", generator=g))
        edges = torch.cumsum(popularity / popularity.sum(), 0)
        return torch.searchsorted(edges, torch.rand(n, device="cuda", generator=g)).clamp(max=experts - 1).to(torch.int32)
    used = torch.randperm(experts, device="cuda", generator=g)[: max(1, experts // 4)]
    runs = torch.randint(0, used.numel(), (n // 6 + 1,), device="cuda", generator=g).repeat_interleave(6)[:n]
    index = used[runs]
    outside = torch.rand(n, device="cuda", generator=g) < 0.02
    return torch.where(outside, -1, index).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    dtype = DTYPES[case.get("dtype", "fp32")]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if case["op"] in ("plan", "linear", "backward"):
        state["index"] = index = _routing(case, g)
        kept = index[(index >= 0) & (index < case["experts"])]
        state["longest"] = int(torch.bincount(kept.long(), minlength=1).max()) if kept.numel() else 0
        if case["op"] != "plan":
            n, experts, k, m = case["rows"], case["experts"], case["inputs"], case["outputs"]
            state["x"] = normal(n, k).to(dtype)
            state["weight"] = (normal(experts, m, k) / math.sqrt(k)).to(dtype)
            state["bias"] = (0.1 * normal(experts, m)).to(dtype)
        if case["op"] == "backward":
            state["y"] = torch.relu(normal(n, m)).to(dtype)      # a layer's saved outputs: half of them behind the relu
            state["grad_y"] = (normal(n, m) / math.sqrt(m)).to(dtype)
        return state
    shape = (case["batch"], case["m"], case["n"])
    rank = max(1, min(shape[1:]) // 8)
    # a gradient: a few strong directions over a floor of noise
    grad = 1e-3 * (normal(*shape) + torch.bmm(normal(shape[0], shape[1], rank), normal(shape[0], rank, shape[2])) / math.sqrt(rank))
    if case["op"] == "schulz":
        state["grad"] = grad.to(dtype)
    else:
        state["grad"], state["param"], state["momentum"] = grad, normal(*shape) / math.sqrt(shape[2]), 5e-3 * normal(*shape)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "plan":
        return _plain_plan(state["index"], case["experts"])
    if case["op"] == "linear":
        return _plain_linear(state, case)
    if case["op"] == "backward":
        return _plain_backward(state, case)
    if case["op"] == "schulz":
        return _plain_schulz(state["grad"].float()).to(state["grad"].dtype)
    return _plain_muon(state)


def _own(state, case):
    from nerf_amd import expert_ops, muon_ops
    if case["op"] == "schulz":
        return muon_ops.newton_schulz(state["grad"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    if case["op"] == "muon":
        muon_ops.muon_update(state["param"], state["grad"], state["momentum"], **MUON, nesterov=True, steps=STEPS,
                             coefficients=COEFFICIENTS, eps=EPS)
        return {"param": state["param"], "momentum": state["momentum"]}
    plan = expert_ops.expert_plan(state["index"], case["experts"])
    if case["op"] == "plan":
        return {"counts": plan.counts, "offsets": plan.offsets, "order": plan.order}
    if case["op"] == "linear":
        return expert_ops.expert_linear(state["x"], state["weight"], state["bias"], plan, activation=case["act"])
    y = state["y"] if case["act"] == "relu" else None
    dx, dw, db = expert_ops.expert_linear_backward(state["grad_y"], state["x"], state["weight"], plan, y=y, activation=case["act"])
    return {"x": dx, "weight": dw, "bias": db}


def _plain_plan(index, experts):
    key = torch.where((index >= 0) & (index < experts), index, experts)
    grouped, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(grouped, torch.arange(experts + 1, device=index.device, dtype=key.dtype))
    return {"counts": (offsets[1:] - offsets[:-1]).to(torch.int32), "offsets": offsets.to(torch.int32),
            "order": order.to(torch.int32)}


def _padded(state, case):
    """(rows, there): for each expert, as many places as the longest has rows, the row in each place and whether one is."""
    plan = _plain_plan(state["index"], case["experts"])
    place = torch.arange(max(1, state["longest"]), device=state["index"].device)
    there = place < plan["counts"][:, None]
    at = (plan["offsets"][:-1, None] + place).clamp(max=case["rows"] - 1)
    return plan["order"][at].long(), there


def _unpadded(values, rows, there, n):
    """The places' values back in the order of the rows; places without a row go to an extra row that is cut off."""
    out = torch.zeros((n + 1, values.shape[-1]), dtype=values.dtype, device=values.device)
    out[torch.where(there, rows, n)] = values
    return out[:n]


def _plain_linear(state, case):
    rows, there = _padded(state, case)
    x = state["x"].float()[rows]
    z = torch.bmm(x, state["weight"].float().transpose(1, 2)) + state["bias"].float()[:, None]
    if case["act"] == "relu":
        z = z.clamp(min=0)
    return _unpadded(z, rows, there, case["rows"]).to(state["x"].dtype)


def _plain_backward(state, case):
    rows, there = _padded(state, case)
    dz = state["grad_y"].float()
    if case["act"] == "relu":
        dz = dz * (state["y"] > 0)
    dz = dz[rows] * there[:, :, None]
    dx = _unpadded(torch.bmm(dz, state["weight"].float()), rows, there, case["rows"])
    dw = torch.bmm(dz.transpose(1, 2), state["x"].float()[rows])
    dtype = state["x"].dtype
    return {"x": dx.to(dtype), "weight": dw.to(dtype), "bias": dz.sum(1).to(dtype)}


def _plain_schulz(grad):
    tall = grad.shape[1] > grad.shape[2]
    x = grad.transpose(1, 2).contiguous() if tall else grad
    x = x / torch.sqrt((x.double() * x.double()).sum((1, 2), keepdim=True)).clamp(min=EPS).float()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = torch.bmm(x, x.transpose(1, 2))
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _plain_muon(state):
    param, momentum = state["param"], state["momentum"]
    g = state["grad"].clamp(-MUON["clip_value"], MUON["clip_value"])
    momentum.mul_(MUON["momentum"]).add_(g)
    step = _plain_schulz(g + MUON["momentum"] * momentum)
    rate = MUON["lr"] * math.sqrt(max(1.0, param.shape[1] / param.shape[2]))
    param.mul_(1 - MUON["lr"] * MUON["weight_decay"]).sub_(rate * step)
    return {"param": param, "momentum": momentum}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case.get("dtype", "fp32")]
    if case["op"] == "plan":
        return {"bytes": 8 * case["rows"] + 8 * case["experts"], "flops": 0}
    if case["op"] in ("linear", "backward"):
        n, experts, k, m = case["rows"], case["experts"], case["inputs"], case["outputs"]
        share = 0.25 if case["spread"] == "cells" else 1.0
        reached = min(n, experts * share)                        # experts whose weights have to be read
        rows = n * (0.98 if case["spread"] == "cells" else 1.0)
        if case["op"] == "linear":
            return {"bytes": int(4 * n + size * (n * (k + m) + reached * m * (k + 1))), "flops": int(2 * rows * k * m)}
        saved = n * m if case["act"] == "relu" else 0
        moved = n * (2 * k + m) + saved + reached * m * k + experts * m * (k + 1)
        return {"bytes": int(4 * n + size * moved), "flops": int(4 * rows * k * m)}
    batch, m, n = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    # A and A^2 are symmetric: half of each, then the full product with X
    flops = batch * STEPS * (m * m * n + m * m * m + 2 * m * m * n)
    values = batch * m * n
    return {"bytes": values * (2 * size if case["op"] == "schulz" else 20), "flops": flops}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":     # whole numbers, the same in any precision
        return None
    state = prepare(case, seed)
    if case["op"] in ("schulz", "muon"):
        return _exact_update(case, state)
    index = state["index"].tolist()
    rows_of = {}
    for row, expert in enumerate(index):
        if 0 <= expert < case["experts"]:
            rows_of.setdefault(expert, []).append(row)
    x, w = state["x"], state["weight"]
    if case["op"] == "linear":
        y = torch.zeros(case["rows"], case["outputs"], dtype=torch.float64, device="cuda")
        for e, rows in rows_of.items():
            rows = torch.tensor(rows, device="cuda")
            z = x[rows].double() @ w[e].double().T.contiguous() + state["bias"][e].double()
            y[rows] = z.clamp(min=0) if case["act"] == "relu" else z
        return y
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    db = torch.zeros(state["bias"].shape, dtype=torch.float64, device="cuda")
    for e, rows in rows_of.items():
        rows = torch.tensor(rows, device="cuda")
        dz = state["grad_y"][rows].double()
        if case["act"] == "relu":
            dz = torch.where(state["y"][rows] > 0, dz, 0.0)
        dx[rows] = dz @ w[e].double()
        dw[e] = dz.T.contiguous() @ x[rows].double()
        db[e] = dz.sum(0)
    return {"x": dx, "weight": dw, "bias": db}


def _exact_update(case, state):
    """The iteration acts on the singular values alone: U f(f(...f(s / |s|))) V^T with f(s) = a s + b s^3 + c s^5."""
    source = state["grad"].double().cpu()
    if case["op"] == "muon":
        g = source.clamp(-MUON["clip_value"], MUON["clip_value"])
        momentum = MUON["momentum"] * state["momentum"].double().cpu() + g
        source = g + MUON["momentum"] * momentum
    u, s, vh = torch.linalg.svd(source, full_matrices=False)
    s = s / s.square().sum(1, keepdim=True).sqrt().clamp(min=EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = a * s + b * s ** 3 + c * s ** 5
    step = (u * s[:, None, :]) @ vh
    if case["op"] == "schulz":
        return step.cuda()
    rate = MUON["lr"] * math.sqrt(max(1.0, case["m"] / case["n"]))
    param = (1 - MUON["lr"] * MUON["weight_decay"]) * state["param"].double().cpu() - rate * step
    return {"param": param.cuda(), "momentum": momentum.cuda()}
