"""Routing from logits in numpy, in 64 bits, rank by rank, and the bound that a kernel's weights are held to."""
from __future__ import annotations

import numpy as np

from shrike_amd import capi
from tests.mx_reference import to_float

BIG = float(np.finfo(np.float32).max)
HALF_STEP = {capi.ELEM_BF16: 2.0 ** -8, capi.ELEM_F16: 2.0 ** -11, capi.ELEM_F32: 2.0 ** -24}  # relative
SMALLEST = {capi.ELEM_BF16: 2.0 ** -134, capi.ELEM_F16: 2.0 ** -25, capi.ELEM_F32: 2.0 ** -150}  # half a subnormal's step


def encode(v, dtype):
    """float64 -> the bits of the nearest fp16, bf16 or fp32 (as the arrays that go to the device)."""
    v = np.asarray(v, np.float64)
    with np.errstate(over="ignore"):
        if dtype == capi.ELEM_F32:
            return v.astype(np.float32)
        if dtype == capi.ELEM_F16:
            return v.astype(np.float16).view(np.uint16)
        u = v.astype(np.float32).view(np.uint32).astype(np.uint64)
    nan = np.isnan(v)
    return np.where(nan, 0x7FC0, (u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)


def decode(bits, dtype):
    return np.asarray(bits).astype(np.float64) if dtype == capi.ELEM_F32 else to_float(bits, dtype)


def desc(experts, top_k, scores=capi.SCORES_SIGMOID, groups=1, kept=1, best=1, renormalize=True, scaling=1.0):
    return capi.RouteDesc(num_experts=experts, top_k=top_k, scores=scores, groups=groups, kept_groups=kept, group_top=best,
                          renormalize=int(renormalize), scaling=scaling)


def _clean(v):
    v = np.where(np.isnan(v), -np.inf, v)
    return np.minimum(v, BIG)


def route(d, logits, bias=None):
    """(indices, weights, relative bound of the weights ahead of their rounding) of float64 rows."""
    rows, experts = logits.shape
    size = experts // d.groups
    indices = np.zeros((rows, d.top_k), np.uint32)
    weights, bound = np.zeros((rows, d.top_k)), np.zeros((rows, d.top_k))
    b = None if bias is None else _clean(np.asarray(bias, np.float64))
    for r in range(rows):
        l = _clean(logits[r])
        out = np.isneginf(l)
        if d.scores == capi.SCORES_SIGMOID:
            with np.errstate(over="ignore"):
                s = 1 / (1 + np.exp(-l))
            far = np.abs(np.where(out, 0, l))
        else:
            top = l.max()
            far = np.where(out, 0, np.minimum(top - l, 800.0)) if top > -np.inf else np.zeros(experts)
            e = np.where(out, 0, np.exp(-far))
            s = e / max(e.sum(), 1e-300)
        by, value = l, s
        if b is not None:
            out = out | np.isneginf(b)
            by = value = s + np.where(np.isneginf(b), 0, b)
        left = np.where(out, 1, 2)  # classes: 2 in service, 1 out of it, 0 not to be taken
        if d.groups > 1:
            marks = []
            for g in range(d.groups):
                at = [e for e in range(g * size, (g + 1) * size) if not out[e]]
                if d.group_top == 1:
                    marks.append(max((by[e] for e in at), default=-np.inf))
                else:
                    two = sorted((value[e] for e in at), reverse=True)[:2]
                    marks.append(sum(two) if two else -np.inf)
            order = sorted(range(d.groups), key=lambda g: (-marks[g], g))
            for g in order[d.kept_groups:]:
                left[g * size:(g + 1) * size] = 0
        order = sorted(range(experts), key=lambda e: (-left[e], 0.0 if out[e] else -by[e], e))[:d.top_k]
        w = np.where(out, 0, s)[order]
        served = ~out[order]
        if d.renormalize:
            if d.scores == capi.SCORES_SOFTMAX and served.any():
                chosen = l[order]
                most = chosen[served].max()
                w = np.where(served, np.exp(np.where(served, np.maximum(chosen - most, -800.0), 0)), 0)
                far_of = np.where(served, np.minimum(most - chosen, 800.0), 0)
            else:
                far_of = far[order]
            total = w.sum()
            w = w / total if total > 0 else np.zeros(d.top_k)
            # the argument's roundings in the sum's terms too, weighted by what they are of it
            spread = (w * far_of).sum()
        else:
            far_of, spread = far[order], (s * far).sum() if d.scores == capi.SCORES_SOFTMAX else 0.0
        indices[r], weights[r] = order, w * d.scaling
        # exp of an argument rounded (three times half a step of it), a few operations, a sum of up to 1,024 terms
        bound[r] = 2.0 ** -19 + (far_of + spread) * 2.0 ** -22
    return indices, weights, bound


def assert_weights(got, want, bound, dtype, what=""):
    g = decode(got, dtype)
    tol = np.abs(want) * (bound + HALF_STEP[dtype] * (1 + bound)) + SMALLEST[dtype] + 2.0 ** -126
    err = np.abs(g - want)
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert np.all(err <= tol), f"{what}: {worst}: {g[worst]} for {want[worst]}, off by {err[worst]:.3e}, {tol[worst]:.3e} allowed"
