"""Routing to experts from logits, and products with 4-bit weights and group scales, as cases to time.

Routing: per row of logits, softmax or sigmoid scores, a bias that takes part in the choice only, experts in groups of which the best are kept,
the top k of what is left and their weights. A NaN or -inf logit, and such a bias, take an expert out of service: it stands behind all others
with weight 0. Without a bias the choice goes by the logits themselves, with one by score + bias in 64 bits; equal choices go to the lower index.

Product: out = x . w^T (+ bias), w = code * scale + bias of its group (32, 64 or 128 elements along a row), codes of 4 bits two a byte, the even
element in the low half; where there are no group biases a code stands for (code - 8) * scale.

Sizes are those of the benchmark's configurations (bench.py) and generic ones inside the operators' documented limits. Logits are N(0, 1.5),
biases N(0, 0.05), weights N(0, 0.02) quantised group by group, activations N(0, 1).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"bf16": 0, "f16": 1, "f32": 2}  # the library's element types; the first two number its metadata types as well
MOST_LOGITS = 16384 * 512
MOST_FLOPS = 2 * 4096 * 8192 * 4096
MOST_WEIGHTS = 201088 * 2880


def _route(rows, experts, top_k, scores, bias=None, groups=1, kept=1, best=1, renormalize=True, scaling=1.0, logits="f32", weights="f16",
           masked=0, pad=0):
    return dict(kind="route", rows=rows, experts=experts, top_k=top_k, scores=scores, bias=bias or "", groups=groups, kept=kept, best=best,
                renormalize=renormalize, scaling=scaling, logits=logits, weights=weights, masked=masked, pad=pad)


def _product(rows, n, k, x="f16", out="f16", meta="bf16", group=64, symmetric=False, bias=False, pad=0):
    return dict(kind="product", rows=rows, n=n, k=k, x=x, out=out, meta=meta, group=group, symmetric=symmetric, bias=bias, pad=pad)


def listed():
    return [
        # the smallest call: one token of the Kimi-Linear shape, whose scores are sigmoids with a balancing bias
        dict(_route(1, 256, 8, "sigmoid", bias="f32", scaling=2.446), name="route_sigmoid_1x256"),
        # 64 sequences, the experts in eight groups of which four are kept
        dict(_route(64, 256, 8, "sigmoid", bias="f32", groups=8, kept=4, best=2, scaling=2.5), name="route_groups_64x256"),
        # the ragged end of a prompt: plain softmax weights, 16-bit logits, six groups by their best expert
        dict(_route(1001, 96, 6, "softmax", groups=6, kept=3, renormalize=False, logits="bf16", masked=5, pad=32), name="route_softmax_1001x96"),
        # a long chunk over many experts, a softmax with a bias
        dict(_route(16384, 512, 10, "softmax", bias="bf16", weights="f32"), name="route_softmax_16384x512"),
        # one token through one projection of a 2,048-wide layer
        dict(_product(1, 2048, 2048), name="product_1x2048x2048"),
        # one token through the output head: the longest read of weights
        dict(_product(1, 201088, 2880, out="f32"), name="product_1x201088x2880"),
        # eight sequences, a token each, a joined projection with a bias
        dict(_product(8, 5120, 2880, meta="f16", bias=True), name="product_8x5120x2880"),
        # the ragged end of a prompt, an odd number of outputs, symmetric weights in small groups
        dict(_product(37, 2049, 2304, x="bf16", out="bf16", group=32, symmetric=True), name="product_37x2049x2304"),
        # 64 sequences, a wide projection
        dict(_product(64, 16384, 2304, group=128), name="product_64x16384x2304"),
        # a short chunk
        dict(_product(300, 4096, 2048, x="bf16", out="bf16"), name="product_300x4096x2048"),
        # the 512-token chunk into a wide projection
        dict(_product(512, 8192, 2048, meta="f16"), name="product_512x8192x2048"),
        # a long chunk: the largest product
        dict(_product(4096, 8192, 4096), name="product_4096x8192x4096"),
    ]


def _log(rng, low, high, step=1):
    return max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + step))) // step * step))


def draw(rng):
    if rng.random() < 0.4:
        groups = rng.choice([1, 1, 2, 4, 8])
        size = max(4, min(_log(rng, 4, 1024), 1024 // groups))
        experts = groups * size
        kept = rng.randint(1, groups)
        return _route(_log(rng, 1, MOST_LOGITS // experts), experts, min(rng.choice([1, 2, 4, 6, 8, 10, 16, 32]), kept * size),
                      rng.choice(["softmax", "sigmoid"]), bias=rng.choice(["", "f32", "bf16", "f16"]), groups=groups, kept=kept,
                      best=rng.choice([1, 2]), renormalize=rng.random() < 0.7, scaling=rng.choice([1.0, 2.5]),
                      logits=rng.choice(["f32", "f32", "bf16", "f16"]), weights=rng.choice(["f16", "f16", "bf16", "f32"]),
                      masked=rng.choice([0, 0, experts // 4]), pad=rng.choice([0, 0, 3]))
    group = rng.choice([32, 64, 64, 128])
    k = _log(rng, group, 8192, group)
    n = _log(rng, 16, min(65536, MOST_WEIGHTS // k))
    return _product(_log(rng, 1, min(8192, MOST_FLOPS // (2 * n * k))), n, k, x=rng.choice(["f16", "f16", "bf16"]),
                    out=rng.choice(["f16", "f16", "bf16", "f32"]), meta=rng.choice(["bf16", "f16"]), group=group,
                    symmetric=rng.random() < 0.3, bias=rng.random() < 0.3, pad=rng.choice([0, 0, 8]))


def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    rows = case["rows"]
    if case["kind"] == "route":
        experts, top_k = case["experts"], case["top_k"]
        moved = rows * (experts * _size(case["logits"]) + top_k * (4 + _size(case["weights"])))
        return dict(bytes=moved + (experts * _size(case["bias"]) if case["bias"] else 0), flops=4 * rows * experts)
    n, k = case["n"], case["k"]
    weights = n * k // 2 + n * (k // case["group"]) * (2 if case["symmetric"] else 4) + (2 * n if case["bias"] else 0)
    return dict(bytes=weights + rows * k * 2 + rows * n * _size(case["out"]), flops=2 * rows * n * k)


# ---------------------------------------------------------------- inputs

def _quantized(n, k, group, meta, symmetric, rng, dev):
    """Codes and group scales (and biases) of N(0, 0.02) rows, some rows at a time."""
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(n, k // group, dtype=DTYPES[meta], device=dev)
    biases = None if symmetric else torch.empty_like(scales)
    for first in range(0, n, 16384):
        rows = slice(first, min(first + 16384, n))
        w = torch.randn(rows.stop - first, k // group, group, generator=rng, device=dev).mul_(0.02)
        if symmetric:
            scales[rows] = (w.abs().amax(-1) / 7.0).to(scales.dtype)
            q = torch.round(w / scales[rows].to(torch.float32)[..., None]) + 8.0
        else:
            low = w.amin(-1)
            scales[rows], biases[rows] = ((w.amax(-1) - low) / 15.0).to(scales.dtype), low.to(scales.dtype)
            q = torch.round((w - biases[rows].to(torch.float32)[..., None]) / scales[rows].to(torch.float32)[..., None])
        q = q.clamp_(0.0, 15.0).to(torch.uint8).reshape(-1, k)
        codes[rows] = q[:, 0::2] | (q[:, 1::2] << 4)
    return codes, scales, biases


def prepare(case, seed):
    dev = torch.device("cuda")
    rng = torch.Generator(device=dev).manual_seed(seed)
    rows = case["rows"]
    st = dict(case=case)
    if case["kind"] == "route":
        experts = case["experts"]
        logits = torch.randn(rows, experts + case["pad"], generator=rng, device=dev).mul_(1.5)
        if case["masked"]:  # experts out of service, the same for every row
            gone = torch.randperm(experts, generator=rng, device=dev)[:case["masked"]]
            logits[:, gone] = -math.inf
        st["logits"] = logits.to(DTYPES[case["logits"]])
        st["bias"] = torch.randn(experts, generator=rng, device=dev).mul_(0.05).to(DTYPES[case["bias"]]) if case["bias"] else None
        if own:
            from shrike_amd import capi
            st["desc"] = capi.RouteDesc(num_experts=experts, top_k=case["top_k"], groups=case["groups"], kept_groups=case["kept"],
                                        group_top=case["best"], renormalize=int(case["renormalize"]), scaling=case["scaling"],
                                        scores=capi.SCORES_SIGMOID if case["scores"] == "sigmoid" else capi.SCORES_SOFTMAX)
        return st
    n, k = case["n"], case["k"]
    st["x"] = torch.randn(rows, k + case["pad"], generator=rng, device=dev).to(DTYPES[case["x"]])
    st["codes"], st["scales"], st["biases"] = _quantized(n, k, case["group"], case["meta"], case["symmetric"], rng, dev)
    st["bias"] = torch.randn(n, generator=rng, device=dev).mul_(0.1).to(DTYPES[case["meta"]]) if case["bias"] else None
    return st


# ---------------------------------------------------------------- one pass

def _run_own(st):
    from shrike_amd import runtime as rt
    case = st["case"]
    rows = case["rows"]
    if case["kind"] == "route":
        top_k = case["top_k"]
        indices = torch.empty(rows, top_k, dtype=torch.int32, device="cuda")
        weights = torch.empty(rows, top_k, dtype=DTYPES[case["weights"]], device="cuda")
        rt.route_rows(st["desc"], st["logits"].data_ptr(), CODES[case["logits"]], st["logits"].stride(0),
                      st["bias"].data_ptr() if case["bias"] else None, CODES[case["bias"] or "f32"], indices.data_ptr(), weights.data_ptr(),
                      CODES[case["weights"]], rows)
        return dict(indices=indices, weights=weights)
    out = torch.empty(rows, case["n"], dtype=DTYPES[case["out"]], device="cuda")
    rt.affine4_product(st["x"].data_ptr(), CODES[case["x"]], st["x"].stride(0), st["codes"].data_ptr(), st["scales"].data_ptr(),
                       None if case["symmetric"] else st["biases"].data_ptr(), CODES[case["meta"]], case["group"],
                       st["bias"].data_ptr() if case["bias"] else None, out.data_ptr(), CODES[case["out"]], case["n"], rows, case["n"], case["k"])
    return out


def _in_service(v):
    """NaN as -inf, +inf as the largest finite value."""
    v = torch.where(torch.isnan(v), -math.inf, v)
    return torch.where(v == math.inf, torch.finfo(torch.float32).max, v)


def _plain_route(st):
    case = st["case"]
    rows, experts, top_k = case["rows"], case["experts"], case["top_k"]
    logits = _in_service(st["logits"][:, :experts].to(torch.float64))
    masked = logits == -math.inf
    if case["scores"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
    else:
        top = logits.amax(-1, keepdim=True)
        e = torch.where(masked, 0.0, torch.exp(logits - torch.where(top == -math.inf, 0.0, top)))
        score = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    if case["bias"]:
        bias = _in_service(st["bias"].to(torch.float64))
        masked = masked | (bias == -math.inf)
        value = score + bias
    else:
        value = score
    choice = torch.where(masked, -math.inf, value if case["bias"] else logits)
    if case["groups"] > 1:
        groups, size = case["groups"], experts // case["groups"]
        if case["best"] == 1:
            best = choice.view(rows, groups, size).amax(-1)
        else:
            v = torch.where(masked, -math.inf, value).view(rows, groups, size).sort(-1, descending=True)[0][..., :2]
            best = torch.where(v[..., 0] == -math.inf, -math.inf, torch.where(v == -math.inf, 0.0, v).sum(-1))
        order = torch.sort(best, dim=-1, descending=True, stable=True)[1][:, :case["kept"]]
        kept = torch.zeros(rows, groups, dtype=torch.bool, device=choice.device)
        kept[torch.arange(rows, device=choice.device)[:, None], order] = True
        kept = kept.repeat_interleave(size, -1)
    else:
        kept = torch.ones_like(masked)
    # three classes behind each other: in service, out of service, not of a kept group
    rank = torch.where(kept, torch.where(masked, 1, 0), 2)
    by_choice = torch.sort(torch.where(masked, 0.0, choice), dim=-1, descending=True, stable=True)[1]
    by_class = torch.sort(rank.gather(-1, by_choice), dim=-1, stable=True)[1]
    indices = by_choice.gather(-1, by_class)[:, :top_k]
    weight = torch.where(masked, 0.0, score).gather(-1, indices)
    if case["renormalize"] and case["scores"] == "softmax":  # = the softmax of the chosen ones: nothing underflows
        chosen = torch.where(masked, -math.inf, logits).gather(-1, indices)
        top = chosen.amax(-1, keepdim=True)
        weight = torch.where(chosen == -math.inf, 0.0, torch.exp(chosen - torch.where(top == -math.inf, 0.0, top)))
    if case["renormalize"]:
        total = weight.sum(-1, keepdim=True)
        weight = torch.where(total > 0.0, weight / total, 0.0)
    return dict(indices=indices.to(torch.int32), weights=(weight * case["scaling"]).to(DTYPES[case["weights"]]))


def _plain_product(st):
    case = st["case"]
    n, k, group = case["n"], case["k"], case["group"]
    x = st["x"][:, :k].to(torch.float32)
    q = torch.stack([st["codes"] & 15, st["codes"] >> 4], -1).view(n, k // group, group).to(torch.float32)
    scale = st["scales"].to(torch.float32)[..., None]
    w = (q - 8.0) * scale if case["symmetric"] else q * scale + st["biases"].to(torch.float32)[..., None]
    y = x @ w.view(n, k).t()
    if case["bias"]:
        y = y + st["bias"].to(torch.float32)
    return y.to(DTYPES[case["out"]])


def run(st):
    if own:
        return _run_own(st)
    return _plain_route(st) if st["case"]["kind"] == "route" else _plain_product(st)


# ---------------------------------------------------------------- the definition, in 64 bits

def _exact_route(case, logits, bias):
    """Rank by rank: the best choice that is left, lowest index first."""
    rows, experts = logits.shape
    dev = logits.device
    finite = torch.nan_to_num(logits, nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf)
    out = finite == -math.inf
    if case["scores"] == "sigmoid":
        score = torch.sigmoid(finite)
    else:
        score = torch.softmax(finite, -1).nan_to_num(0.0)
    by = finite
    value = score
    if bias is not None:
        b = torch.nan_to_num(bias, nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf)
        out = out | (b == -math.inf)
        by = value = score + torch.where(b == -math.inf, 0.0, b)
    left = torch.where(out, -1, 0).expand(rows, experts).clone()  # 0 in service, -1 out of it, -2 not to be taken
    each = torch.arange(rows, device=dev)
    if case["groups"] > 1:
        size = experts // case["groups"]
        marks = torch.full((rows, case["groups"]), -math.inf, dtype=torch.float64, device=dev)
        for g in range(case["groups"]):
            part, gone = slice(g * size, (g + 1) * size), out[:, g * size:(g + 1) * size]
            if case["best"] == 1:
                marks[:, g] = torch.where(gone, -math.inf, by[:, part]).max(-1)[0]
            else:
                v = torch.where(gone, -math.inf, value[:, part])
                first, at = v.max(-1)
                v[each, at] = -math.inf
                second = v.max(-1)[0]
                marks[:, g] = torch.where(first == -math.inf, first, first + torch.where(second == -math.inf, 0.0, second))
        ahead = (marks[:, None, :] > marks[:, :, None]).sum(-1)
        number = torch.arange(case["groups"], device=dev)
        ahead += ((marks[:, None, :] == marks[:, :, None]) & (number[None, None, :] < number[None, :, None])).sum(-1)
        left = torch.where((ahead < case["kept"]).repeat_interleave(size, -1), left, -2)
    indices = torch.empty(rows, case["top_k"], dtype=torch.int64, device=dev)
    for r in range(case["top_k"]):
        best = left.max(-1, keepdim=True)[0]
        v = torch.where(left == best, torch.where(out, 0.0, by), -math.inf)
        hold = (left == best) & (v == v.max(-1, keepdim=True)[0])
        indices[:, r] = torch.where(hold, torch.arange(experts, device=dev), experts).min(-1)[0]
        left[each, indices[:, r]] = -3
    weight = torch.where(out, 0.0, score).gather(-1, indices)
    if case["renormalize"]:
        if case["scores"] == "softmax":
            weight = torch.softmax(torch.where(out, -math.inf, finite).gather(-1, indices), -1).nan_to_num(0.0)
        weight = weight / weight.sum(-1, keepdim=True).clamp(min=5e-324)
    return dict(indices=indices.to(torch.int32), weights=weight * case["scaling"])


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, st["logits"][:, :case["experts"]].double(), st["bias"].double() if case["bias"] else None)
    n, k = case["n"], case["k"]
    x = st["x"][:, :k].double()
    y = torch.empty(case["rows"], n, dtype=torch.float64, device=x.device)
    for first in range(0, n, 32768):
        rows = slice(first, min(first + 32768, n))
        w = torch.empty(rows.stop - first, k, dtype=torch.float64, device=x.device)
        w[:, 0::2], w[:, 1::2] = (st["codes"][rows] % 16).double(), (st["codes"][rows] // 16).double()
        scale = st["scales"][rows].double().repeat_interleave(case["group"], -1)
        w = w * scale + (-8.0 * scale if case["symmetric"] else st["biases"][rows].double().repeat_interleave(case["group"], -1))
        y[:, rows] = torch.matmul(x, w.t())
    return y + st["bias"].double() if case["bias"] else y
