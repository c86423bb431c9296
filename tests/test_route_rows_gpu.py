"""shrike_hip_route_rows against numpy in 64 bits: indices equal, weights within their rounding."""
import numpy as np
import pytest

from shrike_amd import capi, runtime as rt
from tests import route_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = capi.ELEM_F32, capi.ELEM_F16, capi.ELEM_BF16
SOFTMAX, SIGMOID = capi.SCORES_SOFTMAX, capi.SCORES_SIGMOID


def on_device(a, offset=0):
    """The array on the device, `offset` bytes behind an allocation's start."""
    buf = rt.empty(a.nbytes + offset + 16)
    buf.upload(a.view(np.uint8).reshape(-1), offset)
    return buf


def call(d, logits, bias=None, logits_type=F32, bias_type=F32, weights_type=F16, pad=0, skew=0, stream=None):
    """Runs the call over encoded rows; returns (indices, weight bits). What lies behind the last row has to stay."""
    rows, experts = logits.shape
    host = np.full((rows, experts + pad), np.nan)
    host[:, :experts] = logits
    size = 4 if logits_type == F32 else 2
    x = on_device(ref.encode(host, logits_type), skew * size)
    b = on_device(ref.encode(bias, bias_type), skew * (4 if bias_type == F32 else 2)) if bias is not None else None
    wt = np.float32 if weights_type == F32 else np.uint16
    idx, w = rt.empty((rows + 2) * d.top_k * 4), rt.empty((rows + 2) * d.top_k * 4)
    idx.fill(0xA5), w.fill(0xA5)
    rt.route_rows(d, x.ptr + skew * size, logits_type, experts + pad, b.ptr + skew * (4 if bias_type == F32 else 2) if b else None, bias_type, idx, w,
                  weights_type, rows, stream)
    stream.synchronize() if stream else rt.synchronize()
    n = rows * d.top_k
    assert np.all(idx.download(np.uint8, 8 * d.top_k, 4 * n) == 0xA5)
    assert np.all(w.download(np.uint8, 2 * d.top_k, n * np.dtype(wt).itemsize) == 0xA5)
    return idx.download(np.uint32, n).reshape(rows, d.top_k), w.download(wt, n).reshape(rows, d.top_k)


def check(d, logits, bias=None, logits_type=F32, bias_type=F32, weights_type=F16, what="", **how):
    seen = ref.decode(ref.encode(logits, logits_type), logits_type)
    b = None if bias is None else ref.decode(ref.encode(bias, bias_type), bias_type)
    want, weights, bound = ref.route(d, seen, b)
    got, bits = call(d, logits, bias, logits_type, bias_type, weights_type, **how)
    assert np.array_equal(got, want), f"{what}: row {np.argwhere((got != want).any(1))[0]}: {got[(got != want).any(1)][0]} for {want[(got != want).any(1)][0]}"
    ref.assert_weights(bits, weights, bound, weights_type, what)
    return got, bits


@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 1), (3, 3), (8, 2), (16, 16), (31, 5), (32, 4), (33, 32), (64, 8), (65, 6), (96, 6), (127, 8), (128, 10), (160, 6), (200, 7),
                                           (255, 8), (256, 8), (257, 8), (384, 8), (512, 10), (513, 32), (777, 9), (1000, 16), (1024, 32)])
@pytest.mark.parametrize("scores", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("biased", [False, True])
def test_sizes(gpu, experts, top_k, scores, biased):
    r = np.random.default_rng(experts * 64 + top_k)
    for rows in (1, 5, 131):
        logits = r.normal(0, 1.5, (rows, experts))
        bias = r.normal(0, 0.05, experts) if biased else None
        check(ref.desc(experts, top_k, scores), logits, bias, what=f"{rows} rows")


@pytest.mark.parametrize("groups,size,kept,best", [(8, 32, 4, 2), (8, 32, 3, 1), (4, 16, 1, 2), (2, 2, 1, 2), (2, 1, 1, 1), (2, 1, 1, 2), (64, 16, 7, 2), (64, 1, 32, 1), (64, 1, 32, 2), (6, 16, 3, 1), (6, 27, 2, 2),
                                                   (5, 7, 4, 2), (3, 100, 2, 1), (2, 512, 1, 2), (33, 31, 20, 2), (16, 8, 16, 2), (8, 20, 8, 1), (16, 4, 3, 2), (32, 8, 8, 1), (16, 64, 5, 2)])
@pytest.mark.parametrize("scores", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(gpu, groups, size, kept, best, scores, biased):
    r = np.random.default_rng(groups * 1000 + size)
    experts = groups * size
    for rows in (1, 66):
        logits = r.normal(0, 1.5, (rows, experts))
        bias = r.normal(0, 0.05, experts) if biased else None
        check(ref.desc(experts, min(32, kept * size, 8), scores, groups, kept, best, scaling=2.5), logits, bias, what=f"{rows} rows")


@pytest.mark.parametrize("logits_type", [F32, F16, BF16])
@pytest.mark.parametrize("bias_type", [None, F32, F16, BF16])
@pytest.mark.parametrize("weights_type", [F32, F16, BF16])
def test_types_strides_and_addresses(gpu, logits_type, bias_type, weights_type):
    r = np.random.default_rng(5)
    for experts, groups, kept in ((96, 1, 1), (256, 8, 4), (640, 1, 1)):
        for rows in (3, 90):
            bias = None if bias_type is None else r.normal(0, 0.05, experts)
            for pad, skew in ((0, 0), (1, 1), (4, 0), (13, 3)):
                for renormalize in (True, False):
                    check(ref.desc(experts, 6, SOFTMAX if pad else SIGMOID, groups, kept, 2, renormalize, 1.5), r.normal(0, 1.5, (rows, experts)), bias, logits_type,
                          F32 if bias_type is None else bias_type, weights_type, pad=pad, skew=skew, what=f"{experts} {rows} {pad}")


@pytest.mark.parametrize("scores", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,kept,best", [(1, 1, 1), (8, 3, 1), (8, 3, 2)])
def test_equal_choices_go_to_the_lower_index(gpu, scores, biased, groups, kept, best):
    r = np.random.default_rng(9)
    experts = 128
    logits = r.integers(-2, 3, (70, experts)) * 0.5
    logits[0] = 0.25
    logits[1, :] = np.repeat(r.normal(0, 1, experts // 4), 4)
    logits[2] = -0.0
    logits[2, 5:] = 0.0
    bias = np.tile([0.0, 0.125], experts // 2) if biased else None
    for top_k in (1, 4, 8, 32):
        for kind in (F32, F16, BF16):
            check(ref.desc(experts, top_k, scores, groups, kept, best), logits, bias, kind, what=f"top {top_k}")


@pytest.mark.parametrize("scores", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,kept,best", [(1, 1, 1), (8, 4, 1), (8, 4, 2), (64, 9, 2)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_experts_out_of_service_nan_and_infinities(gpu, scores, biased, groups, kept, best, renormalize):
    r = np.random.default_rng(17)
    experts, rows = 192, 40
    logits = r.normal(0, 1.5, (rows, experts))
    for i, v in enumerate((-np.inf, np.nan, np.finfo(np.float32).min, np.inf)):
        logits[i] = v  # a row of nothing else
        logits[4 + i, r.permutation(experts)[:150]] = v
        logits[8 + i, :180] = v
        logits[12 + i, 1:] = v
        logits[16 + i, r.permutation(experts)[:3]] = v
    logits[20] = np.nan
    logits[20, 77] = -3.0
    logits[21] = -np.inf
    logits[21, 100:103] = (np.nan, np.inf, 2.0)
    bias = None
    if biased:
        bias = r.normal(0, 0.05, experts)
        bias[3], bias[50], bias[51] = -np.inf, np.nan, np.inf
        bias[60:84] = -np.inf
    check(ref.desc(experts, 8, scores, groups, kept, best, renormalize, 2.0), logits, bias, weights_type=F32)
    check(ref.desc(experts, 27, scores, groups, kept if groups < 64 else 20, best, renormalize), logits, bias)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("groups,kept,best", [(1, 1, 1), (4, 2, 2)])
def test_far_logits(gpu, renormalize, groups, kept, best):
    """Scores that fp32 does not hold, and choices that differ by less than it resolves."""
    r = np.random.default_rng(23)
    experts = 64
    logits = np.concatenate([r.normal(0, 1, (8, experts)) + m for m in (-700, -100, -80, -20, 0, 15, 30, 80, 1e30, -1e30)]
                            + [r.normal(0, 200, (16, experts)), 5 + r.normal(0, 1, (8, experts)) * 2.0 ** -18])
    for scores in (SOFTMAX, SIGMOID):
        check(ref.desc(experts, 8, scores, groups, kept, best, renormalize), logits, None, weights_type=F32)
        if scores == SIGMOID:  # (a softmax whose chosen experts underflow in 64 bits has no order but the bias's)
            logits = np.clip(logits, -30, 30)
        check(ref.desc(experts, 8, scores, groups, kept, best, renormalize), logits, r.normal(0, 1, experts) * 2.0 ** -12, weights_type=F32)
        check(ref.desc(experts, 8, scores, groups, kept, best, renormalize), logits, r.normal(0, 1, experts) * 1e6, weights_type=F32)


def test_a_bias_that_moves_every_choice_by_less_than_fp32_resolves(gpu):
    """Choices a few 2^-24 apart, equal but for their bias's last places: 64 bits decide."""
    r = np.random.default_rng(29)
    experts = 256
    logits = np.repeat(r.normal(0, 1, (50, 1)), experts, 1)
    bias = 0.25 + r.permutation(experts) * 2.0 ** -26
    for scores in (SOFTMAX, SIGMOID):
        for groups, kept, best in ((1, 1, 1), (8, 4, 1), (8, 4, 2)):
            check(ref.desc(experts, 8, scores, groups, kept, best), logits, bias, bias_type=F32, weights_type=F32)


def test_many_rows_of_every_width_are_the_rows_alone(gpu):
    """More rows than the launch has places: every row as in a call of its own size."""
    r = np.random.default_rng(31)
    for experts, top_k, groups, kept in ((8, 2, 1, 1), (32, 4, 4, 2), (128, 8, 1, 1), (256, 8, 8, 4), (512, 10, 1, 1)):
        logits = r.normal(0, 1.5, (300, experts))
        bias = r.normal(0, 0.05, experts)
        d = ref.desc(experts, top_k, SIGMOID, groups, kept, 2)
        got, bits = check(d, logits, bias)
        many = 300 * (2_400_000 // 300 // max(1, experts // 8))
        i2, b2 = call(d, np.tile(logits, (many // 300, 1)), bias)
        assert np.array_equal(i2, np.tile(got, (many // 300, 1))) and np.array_equal(b2, np.tile(bits, (many // 300, 1)))
        one_i, one_b = call(d, logits[7:8], bias)
        assert np.array_equal(one_i[0], got[7]) and np.array_equal(one_b[0], bits[7])


def test_rows_past_4_gib_of_logits(gpu):
    r = np.random.default_rng(37)
    experts, rows, stride = 64, 17, 1 << 26
    logits = r.normal(0, 1, (rows, experts)).astype(np.float32)
    x = rt.DeviceBuffer((rows - 1) * stride * 4 + experts * 4)
    for i in range(rows):
        x.upload(logits[i], i * stride * 4)
    idx, w = rt.empty(rows * 32), rt.empty(rows * 32)
    d = ref.desc(experts, 8)
    rt.route_rows(d, x, F32, stride, None, F32, idx, w, F32, rows)
    rt.synchronize()
    want, weights, bound = ref.route(d, logits.astype(np.float64))
    assert np.array_equal(idx.download(np.uint32, rows * 8).reshape(rows, 8), want)
    ref.assert_weights(w.download(np.float32, rows * 8).reshape(rows, 8), weights, bound, F32)


def test_two_streams_and_replays(gpu):
    """Calls at once on two streams, and a captured call replayed over other inputs with eager work between."""
    r = np.random.default_rng(41)
    experts, rows = 256, 700
    d = ref.desc(experts, 8, SIGMOID, 8, 4, 2)
    inputs = [r.normal(0, 1.5, (rows, experts)) for _ in range(4)]
    bias = r.normal(0, 0.05, experts)
    eager = [check(d, v, bias) for v in inputs]
    b = on_device(ref.encode(bias, F32))
    x = [on_device(ref.encode(v, F32)) for v in inputs]
    streams = [rt.Stream(), rt.Stream()]
    outs = [(rt.empty(rows * 32), rt.empty(rows * 16)) for _ in range(4)]
    for i in range(4):
        rt.route_rows(d, x[i], F32, experts, b, F32, *outs[i], F16, rows, streams[i % 2])
    for s in streams:
        s.synchronize()
    for (oi, ow), (gi, gw) in zip(outs, eager):
        assert np.array_equal(oi.download(np.uint32, rows * 8), gi.reshape(-1)) and np.array_equal(ow.download(np.uint16, rows * 8), gw.reshape(-1))
    lib = capi.load()
    s, (oi, ow), fixed = streams[0], outs[0], on_device(ref.encode(inputs[0], F32))
    capi.check(lib.shrike_hip_graph_begin_capture(s.handle), "capture")
    rt.route_rows(d, fixed, F32, experts, b, F32, oi, ow, F16, rows, s)
    graph = lib.shrike_hip_graph_end_capture(s.handle)
    assert graph
    for i in (1, 3, 2, 0, 1):
        fixed.upload(ref.encode(inputs[i], F32).view(np.uint8).reshape(-1))
        call(d, inputs[(i + 1) % 4], bias)
        capi.check(lib.shrike_hip_graph_launch(graph, s.handle), "launch")
        s.synchronize()
        assert np.array_equal(oi.download(np.uint32, rows * 8), eager[i][0].reshape(-1)) and np.array_equal(ow.download(np.uint16, rows * 8), eager[i][1].reshape(-1))
    capi.check(lib.shrike_hip_graph_destroy(graph), "destroy")
