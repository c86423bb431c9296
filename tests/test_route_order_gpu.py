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


def dominant_rows(experts, lanes):
    """Rows of one expert with nearly all of the softmax and others of 0.97 * 2^-24 of it, where the additions of a sum in order, of a lane's sum in order and
    of a sum in pairs each round them away; the rest is nothing."""
    each, rows = experts // lanes, []
    for small in ([*range(1, each), *(each << j for j in range(10))], [1 << j for j in range(10)], [*range(1, 20)], [*range(1, experts, 37)]):
        row = np.full(experts, -100.0)
        row[0] = 0.0
        row[[e for e in small if e < experts - 1]] = np.log(0.97 * 2.0 ** -24)
        rows.append(row)
    return rows


@pytest.mark.parametrize("experts", [64, 256, 512, 1024])
@pytest.mark.parametrize("groups,best", [(1, 1), (8, 1), (8, 2)])
@pytest.mark.parametrize("renormalize", [False, True])
def test_a_bias_that_cancels_a_dominant_expert(gpu, experts, groups, best, renormalize):
    """What a softmax's sum in fp32 has lost does not move the choices: 64 bits decide between an expert of nearly 1 and a bias of nearly -1, and an expert of
    nothing without a bias."""
    logits = single(np.array(dominant_rows(experts, 64 if experts > 64 else 16) + dominant_rows(experts, 16)))
    d = ref.desc(experts, 1, SOFTMAX, groups, 1, best, renormalize)
    for m in range(-4, 21, 2):
        bias = np.full(experts, -5e-4)
        bias[0], bias[-1] = -1.0 + m * 2.0 ** -24, 0.0
        if best == 2:  # the groups' second experts alike
            bias[1], bias[-2] = -5e-4, -5e-4
        bias = single(bias)
        for rows in (len(logits), 8200):
            compare(d, logits, bias, rows, f"{m} last places")


@pytest.mark.parametrize("experts", [100, 512, 1000, 1024])
@pytest.mark.parametrize("groups,best", [(1, 1), (4, 1), (4, 2)])
def test_one_expert_above_many_equal_ones(gpu, experts, groups, best):
    """One logit above equal ones, each of whose additions rounds the same way, and a bias that lifts one of these to the top one's choice or nearly."""
    r = np.random.default_rng(experts + best)
    d = ref.desc(experts, 1, SOFTMAX, groups, 1, best, False)
    other = experts // max(groups, 2) + 5
    for x in single(r.uniform(4.0, 10.0, 10)):
        row = np.full(experts, -x)
        row[0] = 0.0
        p = np.exp(row) / np.exp(row).sum()
        bias = np.zeros(experts)
        bias[other] = p[0] - p[other]
        bias = single(bias)
        rows = np.tile(row, (48, 1))
        rows[:, other] += np.append(0.0, r.choice([-1.0, 1.0], 47) * 2.0 ** r.uniform(-24, -17, 47)) / p[other]
        for count in (48, 8200):
            compare(d, single(rows), bias, count, f"{x} above the others")


@pytest.mark.parametrize("experts,top_k,groups,kept", [(5, 3, 1, 1), (60, 8, 1, 1), (128, 32, 1, 1), (256, 8, 8, 4), (300, 20, 1, 1), (512, 10, 1, 1), (512, 32, 1, 1), (480, 24, 15, 4),
                                                       (100, 17, 4, 2), (1000, 32, 1, 1)])
@pytest.mark.parametrize("scores", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("biased", [False, True])
def test_a_row_s_routes_are_the_same_bits_in_calls_of_any_size(gpu, experts, top_k, groups, kept, scores, renormalize, biased):
    """The weights in fp32 too, on both sides of where fewer lanes take a row, and of rows that 64 bits decide."""
    r = np.random.default_rng(experts + top_k)
    logits = np.concatenate([r.normal(0, 1.5, (150, experts)), 0.5 + r.integers(-9, 10, (20, experts)) * 2.0 ** -21, r.normal(0, 40, (10, experts))])
    logits[20:30, r.permutation(experts)[:experts // 3]] = -np.inf
    logits[30, 1:], logits[31] = np.nan, -np.inf
    bias = r.normal(0, 0.05, experts) if biased else None
    for logits_type in (F32, F16, BF16):
        for best in (1, 2) if groups > 1 else (1,):
            d = ref.desc(experts, top_k, scores, groups, kept, best, renormalize, 2.5)
            idx, w = call(d, logits, bias, logits_type, weights_type=F32)
            for rows in (1, 8191, 8192, 9001):
                order = (np.arange(rows) * 7 + 3) % len(logits)
                i2, w2 = call(d, logits[order], bias, logits_type, weights_type=F32)
                assert np.array_equal(i2, idx[order])
                bad = (w2.view(np.uint32) != w[order].view(np.uint32)).any(1)
                assert not bad.any(), f"{rows} rows: {bad.sum()} differ, row {order[np.argmax(bad)]}: {w2[np.argmax(bad)]} and {w[order][np.argmax(bad)]}"


@pytest.mark.parametrize("scaling", [3e38, 1e30, 1e10, -1e30, 1e-30, 1e-38])
@pytest.mark.parametrize("rows", [11, 8200])
def test_any_finite_scaling_over_small_sums(gpu, scaling, rows):
    """Chosen sigmoids that sum to 1e-3 ... 1e-29: the scaling over their sum alone may leave fp32, the weights do not."""
    r = np.random.default_rng(11)
    for experts, top_k in ((64, 8), (200, 20)):
        logits = single(r.normal(0, 1, (11, experts)) - np.linspace(5, 68, 11)[:, None])
        d = ref.desc(experts, top_k, SIGMOID, scaling=scaling)
        want, weights, bound = ref.route(d, logits)
        order = np.arange(rows) % 11
        idx, w = call(d, logits[order], weights_type=F32)
        assert np.array_equal(idx, want[order])
        assert np.isfinite(w).all()
        ref.assert_weights(w, weights[order], bound[order], F32, f"{scaling}")


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [7, 8200])
def test_every_nan_is_out_of_service(gpu, kind, rows):
    """Quiet and signalling ones, of either sign, in the logits and in the bias."""
    r = np.random.default_rng(3)
    nans = {F32: (0x7FC00000, 0xFFC00000, 0x7F800001, 0xFF800001, 0x7FFFFFFF), F16: (0x7E00, 0xFE00, 0x7C01, 0xFC01, 0x7FFF), BF16: (0x7FC0, 0xFFC0, 0x7F81, 0xFF81, 0x7FFF)}[kind]
    t = np.uint32 if kind == F32 else np.uint16
    for experts, groups, kept, best in ((64, 1, 1, 1), (256, 8, 4, 2), (256, 8, 4, 1), (1000, 1, 1, 1)):
        for scores, biased in ((SOFTMAX, False), (SIGMOID, True), (SOFTMAX, True)):
            bits = ref.encode(r.normal(0, 1.5, (7, experts)), kind).view(t).copy()
            own = ref.encode(r.normal(0, 0.05, experts), kind).view(t).copy()
            for row in range(7):
                bits[row, r.permutation(experts)[:5 * (row + 1)]] = np.resize(np.array(nans, t), 5 * (row + 1))
            own[r.permutation(experts)[:5]] = np.array(nans, t)
            seen, b = (ref.decode(v.view(np.float32) if kind == F32 else v, kind) for v in (bits, own))
            d = ref.desc(experts, 8, scores, groups, kept, best)
            want, weights, bound = ref.route(d, seen, b if biased else None)
            order = np.arange(rows) % 7
            x, on = rt.dev(np.ascontiguousarray(bits[order])), rt.dev(own)
            idx, w = rt.empty(rows * 32).fill(0xA5), rt.empty(rows * 32).fill(0xA5)
            rt.route_rows(d, x, kind, experts, on if biased else None, kind, idx, w, F32, rows)
            rt.synchronize()
            assert np.array_equal(idx.download(np.uint32, rows * 8).reshape(rows, 8), want[order])
            ref.assert_weights(w.download(np.float32, rows * 8).reshape(rows, 8), weights[order], bound[order], F32)
