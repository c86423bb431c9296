"""shrike_hip_route_rows where choices lie close together: differences around what fp32 and the kernel's words resolve, clusters that are larger than what
is put in order at once, near ties across the end of the route and between groups; in rows of every width, few and many."""
import numpy as np
import pytest

from shrike_amd import capi, runtime as rt
from tests import route_reference as ref
from tests.test_route_rows_gpu import F32, SIGMOID, SOFTMAX, call, check

pytestmark = pytest.mark.gpu

SIZES = [(32, 4), (64, 8), (96, 6), (128, 8), (200, 7), (256, 8), (384, 8), (500, 10), (512, 10), (512, 32), (1024, 32)]


def close_rows(r, experts):
    """Rows with clusters of 2 ... all experts, 2^-12 ... 2^-24 of a unit apart, at several heights."""
    rows = []
    for step in (12, 15, 17, 18, 19, 20, 21, 22, 24):
        for cluster in (2, 5, 20, 40, experts):
            row = r.normal(-1.0, 0.7, experts)
            at = r.permutation(experts)[:min(cluster, experts)]
            row[at] = (1.0 if cluster < 40 else 0.25) + r.integers(-6, 7, len(at)) * 2.0 ** -step
            rows.append(row)
    return np.array(rows, np.float32).astype(np.float64)


@pytest.mark.parametrize("experts,top_k", SIZES)
@pytest.mark.parametrize("scores", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("biased", [False, True])
def test_close_choices(gpu, experts, top_k, scores, biased):
    r = np.random.default_rng(experts * 4 + scores)
    logits = close_rows(r, experts)
    bias = r.integers(-3, 4, experts) * 2.0 ** -20 if biased else None
    for renormalize in (True, False):
        d = ref.desc(experts, top_k, scores, renormalize=renormalize)
        got, bits = check(d, logits, bias, weights_type=F32, what=f"{experts}")
        order = r.permutation(np.arange(9001) % len(logits))  # the same rows among others, where there are many
        i2, b2 = call(d, logits[order], bias, weights_type=F32)
        want = ref.route(d, logits, bias)
        assert np.array_equal(i2, want[0][order]), f"{experts}: {np.argwhere((i2 != want[0][order]).any(1))[:4].ravel()}"
        ref.assert_weights(b2, want[1][order], want[2][order], F32, f"{experts}")


@pytest.mark.parametrize("experts,top_k,groups,kept", [(64, 4, 8, 2), (128, 8, 8, 4), (256, 8, 8, 4), (256, 8, 16, 3), (512, 8, 8, 4), (512, 16, 32, 5), (160, 6, 8, 3)])
@pytest.mark.parametrize("scores", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("best", [1, 2])
def test_close_groups(gpu, experts, top_k, groups, kept, scores, best):
    r = np.random.default_rng(experts + groups)
    logits = close_rows(r, experts)
    size = experts // groups
    near = r.normal(-1.0, 0.5, (24, experts))  # every group's best two are nearly the other groups'
    for i, row in enumerate(near):
        for g in range(groups):
            row[g * size:g * size + 2] = 1.0 + r.integers(-4, 5, 2) * 2.0 ** -(14 + i % 10)
    logits = np.concatenate([logits, near]).astype(np.float32).astype(np.float64)
    for bias in (None, r.integers(-3, 4, experts) * 2.0 ** -20):
        d = ref.desc(experts, top_k, scores, groups, kept, best)
        check(d, logits, bias, weights_type=F32)
        order = r.permutation(np.arange(9001) % len(logits))
        i2, b2 = call(d, logits[order], bias, weights_type=F32)
        want = ref.route(d, logits, bias)
        assert np.array_equal(i2, want[0][order])
        ref.assert_weights(b2, want[1][order], want[2][order], F32)


@pytest.mark.parametrize("experts,top_k", [(64, 8), (128, 32), (256, 8), (512, 10)])
def test_far_and_odd_values_in_many_rows(gpu, experts, top_k):
    """Rows that fp32 words cannot hold, out of service, NaN and infinite, next to ordinary ones in a wave."""
    r = np.random.default_rng(experts)
    logits = r.normal(0, 1.5, (48, experts))
    for i, m in enumerate((-1e30, -3e4, -300.0, -33.0, 33.0, 300.0, 3e4, 1e30)):
        logits[2 * i] += m
    for i, v in enumerate((np.nan, np.inf, -np.inf, np.finfo(np.float32).max, np.finfo(np.float32).min)):
        logits[17 + 2 * i] = v
        logits[27 + 2 * i, r.permutation(experts)[:experts // 2]] = v
    logits[38:44] *= 40
    logits = logits.astype(np.float32).astype(np.float64)
    bias = r.normal(0, 0.05, experts)
    bias[:3] = -np.inf, np.nan, np.inf
    for scores, b in ((SOFTMAX, None), (SIGMOID, None), (SIGMOID, bias.astype(np.float32).astype(np.float64))):
        for renormalize in (True, False):
            d = ref.desc(experts, top_k, scores, renormalize=renormalize)
            want = ref.route(d, logits, b)
            order = r.permutation(np.arange(9001) % len(logits))
            i2, b2 = call(d, logits[order], b, weights_type=F32)
            assert np.array_equal(i2, want[0][order])
            ref.assert_weights(b2, want[1][order], want[2][order], F32)


@pytest.mark.parametrize("rows", [8191, 8192, 8193, 8194, 8195])
@pytest.mark.parametrize("experts,groups,kept", [(64, 1, 1), (512, 1, 1), (256, 8, 4), (320, 1, 1)])
def test_where_one_form_gives_way_to_the_next(gpu, rows, experts, groups, kept):
    r = np.random.default_rng(rows)
    logits = r.normal(0, 1.5, (97, experts)).astype(np.float32).astype(np.float64)
    for kind in (F32, capi.ELEM_F16, capi.ELEM_BF16):
        seen = ref.decode(ref.encode(logits, kind), kind)
        d = ref.desc(experts, 8, SIGMOID, groups, kept, 2, True, 2.5)
        want = ref.route(d, seen)
        order = np.arange(rows) % 97
        i2, b2 = call(d, logits[order], None, logits_type=kind)
        assert np.array_equal(i2, want[0][order])
        ref.assert_weights(b2, want[1][order], want[2][order], capi.ELEM_F16)


@pytest.mark.parametrize("experts,groups,kept,top_k", [(100, 4, 2, 32), (72, 8, 4, 32), (912, 8, 4, 32), (344, 4, 3, 16), (96, 3, 2, 8), (96, 3, 1, 32), (60, 6, 2, 5), (1024, 64, 9, 20),
                                                       (512, 2, 1, 10), (1000, 2, 1, 16), (999, 3, 2, 8), (1023, 33, 5, 32), (992, 62, 7, 16), (77, 7, 3, 8), (650, 26, 4, 8), (30, 15, 4, 6),
                                                       (64, 64, 8, 8), (1024, 2, 1, 32), (510, 17, 3, 9), (144, 9, 2, 8), (128, 2, 1, 8), (20, 5, 2, 3), (3, 3, 2, 2), (48, 16, 3, 9),
                                                       (800, 32, 4, 30)])
def test_groups_of_any_size(gpu, experts, groups, kept, top_k):
    r = np.random.default_rng(experts + groups)
    for scores, best, kind, biased in ((SIGMOID, 2, F32, True), (SOFTMAX, 1, capi.ELEM_BF16, False), (SOFTMAX, 2, capi.ELEM_F16, True), (SIGMOID, 1, F32, False)):
        logits = r.normal(0, 1.5, (53, experts))
        logits[40:, r.permutation(experts)[:experts // 4]] = -np.inf
        logits[45:48, :experts // groups] = np.nan
        logits = ref.decode(ref.encode(logits, kind), kind)
        bias = r.normal(0, 0.05, experts).astype(np.float32).astype(np.float64) if biased else None
        d = ref.desc(experts, top_k, scores, groups, kept, best)
        want = ref.route(d, logits, bias)
        for rows, pad in ((1, 0), (53, 8), (8194, 3)):
            order = np.arange(rows) % 53
            i2, b2 = call(d, logits[order], bias, logits_type=kind, weights_type=F32, pad=pad)
            assert np.array_equal(i2, want[0][order]), f"{rows} rows"
            ref.assert_weights(b2, want[1][order], want[2][order], F32, f"{rows} rows")


@pytest.mark.parametrize("rows", [(1 << 24) - 1, 1 << 24, (1 << 24) + 5, 40_000_000])
def test_more_rows_than_a_launch_takes(gpu, rows):
    r = np.random.default_rng(rows % 1000)
    experts, kinds = 4, 1009
    logits = r.normal(0, 1.5, (kinds, experts))
    bits = ref.encode(logits, capi.ELEM_F16)
    d = ref.desc(experts, 1, SIGMOID, renormalize=False)
    want, weights, bound = ref.route(d, ref.decode(bits, capi.ELEM_F16))
    x = rt.dev(np.tile(bits, (rows // kinds + 1, 1))[:rows])
    idx, w = rt.empty(rows * 4 + 64).fill(0xA5), rt.empty(rows * 4 + 64).fill(0xA5)
    rt.route_rows(d, x, capi.ELEM_F16, experts, None, F32, idx, w, F32, rows)
    rt.synchronize()
    which = np.arange(rows) % kinds
    assert np.array_equal(idx.download(np.uint32, rows), want[which, 0])
    got = w.download(np.float32, rows)
    assert np.array_equal(got, got[:kinds][which])  # (a row's route depends on that row alone)
    ref.assert_weights(got[:kinds, None], weights, bound, F32)
    assert np.all(idx.download(np.uint8, 64, rows * 4) == 0xA5) and np.all(w.download(np.uint8, 64, rows * 4) == 0xA5)
