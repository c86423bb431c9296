"""shrike_hip_route_rows: what the fast form's words may leave undecided, and the same routes whatever the number of rows."""
import numpy as np
import pytest

from shrike_amd import capi, runtime as rt
from tests import route_reference as ref
from tests.test_route_rows_gpu import F16, F32, SIGMOID, SOFTMAX, call

pytestmark = pytest.mark.gpu

BF16 = capi.ELEM_BF16


def single(v):
    return np.asarray(v, np.float32).astype(np.float64)


def compare(d, logits, bias, rows, what, **how):
    """`rows` rows of these kinds, over and over, against 64 bits; the outputs hold 0xA5 before the call."""
    kinds = len(logits)
    want, weights, bound = ref.route(d, logits, bias)
    order = np.arange(rows) % kinds
    idx, w = call(d, logits[order], bias, weights_type=F32, **how)
    bad = (idx != want[order]).any(1)
    assert not bad.any(), f"{what}, {rows} rows: {bad.sum()} rows, first {np.argmax(bad)}: {idx[np.argmax(bad)]} for {want[order][np.argmax(bad)]}"
    ref.assert_weights(w, weights[order], bound[order], F32, what)
    return idx, w


def near_groups(r, kinds, groups, size, scores, bias, gone):
    """Rows whose third and fourth group in service have sums of their two best that lie 2^-24 ... 2^-17 apart, either way: the fourth's best logit is moved."""
    b = np.zeros(groups * size) if bias is None else bias
    out = []
    for i in range(kinds):
        row = r.normal(0, 1.5, groups * size)
        row[gone * size:(gone + 1) * size] = -np.inf
        row = single(row)

        def sums(l):
            s = 1 / (1 + np.exp(-l)) if scores == SIGMOID else np.exp(l - l.max()) / np.exp(l - l.max()).sum()
            v = np.where(np.isneginf(l), -np.inf, s + b).reshape(groups, size)
            return np.sort(v, 1)[:, -2:].sum(1)

        order = np.argsort(-sums(row))
        third, fourth = order[2], order[3]
        apart = (1 if i % 2 else -1) * 2.0 ** -r.uniform(17, 24)
        at = fourth * size + np.argmax(np.where(np.isneginf(row), -np.inf, row + b * 0)[fourth * size:(fourth + 1) * size])
        low, high = -20.0, 20.0
        for _ in range(60):  # the sums' difference rises with that logit
            row[at] = (low + high) / 2
            s = sums(row)
            low, high = (row[at], high) if s[fourth] - s[third] < apart else (low, row[at])
        out.append(row)
    return single(np.array(out))


@pytest.mark.parametrize("groups,size,top_k", [(8, 32, 8), (8, 32, 24), (16, 32, 8), (8, 20, 6), (6, 16, 8), (12, 8, 20)])
@pytest.mark.parametrize("scores", [SIGMOID, SOFTMAX])
@pytest.mark.parametrize("biased", [False, True])
def test_close_groups_beside_one_out_of_service(gpu, groups, size, top_k, scores, biased):
    """Group 0, and another, with nobody in service, by their logits or by the bias, next to groups whose sums are hardly apart."""
    r = np.random.default_rng(groups * 100 + size)
    experts = groups * size
    for gone in (0, groups - 2):
        bias = single(r.normal(0, 0.05, experts)) if biased else None
        logits = near_groups(r, 128, groups, size, scores, bias, gone)
        d = ref.desc(experts, top_k, scores, groups, 3, 2, scaling=2.5)
        for rows in (1, 128, 9001):
            compare(d, logits, bias, rows, f"group {gone} is gone")
        if biased:  # the same group gone by its bias
            there = logits.copy()
            there[:, gone * size:(gone + 1) * size] = -4.0 if scores == SIGMOID else -np.inf
            by_bias = bias.copy()
            by_bias[gone * size:(gone + 1) * size] = -np.inf
            for rows in (128, 9001):
                compare(d, there, by_bias, rows, f"group {gone} is gone by its bias")
