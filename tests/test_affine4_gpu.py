"""shrike_hip_affine4_product against numpy in 64 bits: bit for bit where the sums are exact, within the sums' roundings elsewhere."""
import numpy as np
import pytest

from shrike_amd import capi, runtime as rt
from tests import affine4_reference as ref
from tests.affine4_reference import BF16, F16, F32

pytestmark = pytest.mark.gpu

ROWS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 96, 97, 127, 128, 129, 200, 255, 256, 257, 300, 513]


def exactly(rng, rows, n, k, group=64, x_type=F16, out_type=F16, meta=BF16, symmetric=False, bias=False, **how):
    w = ref.Weights(rng, n, k, group, meta, symmetric, whole=True)
    x = ref.whole_rows(rng, rows, k, x_type)
    b = ref.encode(rng.integers(-9, 10, n) * 0.5, meta) if bias else None
    want = ref.decode(x, x_type) @ w.values.T + (0 if b is None else ref.decode(b, meta))
    ref.assert_exact(ref.run(x, x_type, w, b, out_type, **how), want, out_type, f"{rows} x {n} x {k}, groups of {group}")


def closely(rng, rows, n, k, group=64, x_type=F16, out_type=F16, meta=BF16, symmetric=False, bias=False, **how):
    w = ref.Weights(rng, n, k, group, meta, symmetric)
    x = ref.encode(rng.standard_normal((rows, k)), x_type)
    b = ref.encode(rng.standard_normal(n), meta) if bias else None
    xv = ref.decode(x, x_type)
    want = xv @ w.values.T + (0 if b is None else ref.decode(b, meta))
    bound = ref.bound_of(xv, w) + (0 if b is None else np.abs(ref.decode(b, meta)) * 2.0 ** -23)
    ref.assert_close(ref.run(x, x_type, w, b, out_type, **how), want, bound, out_type, f"{rows} x {n} x {k}, groups of {group}")


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_rows(gpu, rows, x_type):
    r = np.random.default_rng(rows)
    for n, k, group in ((96, 256, 64), (33, 64, 64), (257, 640, 128), (130, 1120, 32), (64, 2048, 64)):
        exactly(r, rows, n, k, group, x_type, F32, symmetric=n == 130)
        closely(r, rows, n, k, group, x_type, F32)


@pytest.mark.parametrize("n", [1, 2, 3, 7, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 191, 255, 256, 257, 384, 511, 513, 1000])
def test_outputs(gpu, n):
    r = np.random.default_rng(n)
    for rows in (1, 3, 16, 40, 70, 150, 300):
        exactly(r, rows, n, 192, 64, F16, F32, bias=True, pad=rows % 3)
        exactly(r, rows, n, 160, 32, BF16, F16, meta=F16, symmetric=True)


@pytest.mark.parametrize("k,group", [(32, 32), (64, 32), (64, 64), (96, 32), (128, 128), (160, 32), (192, 64), (224, 32), (256, 128), (320, 64), (384, 128), (448, 64), (480, 32), (512, 64),
                                     (544, 32), (576, 64), (640, 128), (960, 64), (992, 32), (1024, 128), (1088, 64), (1184, 32), (1408, 128), (2048, 64), (2112, 64), (2304, 32),
                                     (2880, 64), (2944, 128), (4096, 128), (4160, 32), (5760, 64), (8192, 64), (8224, 32)])
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_lengths(gpu, k, group, x_type):
    r = np.random.default_rng(k)
    for rows in (1, 4, 12, 33, 64, 100, 260):
        exactly(r, rows, 70, k, group, x_type, F32, meta=F16 if rows % 2 else BF16, symmetric=rows == 12)
        closely(r, rows, 40, k, group, x_type, F32, meta=BF16 if rows % 2 else F16, symmetric=rows == 33)


@pytest.mark.parametrize("x_type", [F16, BF16])
@pytest.mark.parametrize("meta", [F16, BF16])
@pytest.mark.parametrize("out_type", [F16, BF16, F32])
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_types(gpu, x_type, meta, out_type, symmetric, bias):
    r = np.random.default_rng(3)
    for rows, n, k, group in ((1, 515, 512, 64), (6, 130, 320, 32), (20, 300, 768, 128), (64, 64, 256, 64), (90, 129, 576, 64), (290, 258, 384, 128)):
        for pad, x_pad in ((0, 0), (5, 8), (8, 40)):
            exactly(r, rows, n, k, group, x_type, out_type, meta, symmetric, bias, pad=pad, x_pad=x_pad)
        closely(r, rows, n, k, group, x_type, out_type, meta, symmetric, bias)


@pytest.mark.parametrize("rows", [1, 4, 11, 37, 64, 130, 300])
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_far_values(gpu, rows, x_type):
    """Rows far apart in size, subnormal and largest activations, scales from the type's smallest to where sums still fit."""
    r = np.random.default_rng(rows)
    n, k = 77, 512
    for meta, low in ((F16, -14), (BF16, -60)):
        w = ref.Weights(r, n, k, 64, meta, whole=True)
        spread = 2.0 ** r.integers(low, 1, (n, k // 64))
        w.scale_bits, w.bias_bits = ref.encode(spread, meta), ref.encode(-spread * r.integers(0, 16, (n, k // 64)), meta)
        s, b = (np.repeat(ref.decode(v, meta), 64, 1) for v in (w.scale_bits, w.bias_bits))
        q = np.stack([w.codes & 15, w.codes >> 4], -1).reshape(n, k)
        w.values, w.size = q * s + b, q * s + np.abs(b)
        x = r.standard_normal((rows, k)) * 2.0 ** r.integers(-20 if x_type == F16 else -40, 14, (rows, 1))
        x[0, :] = 65504.0 if x_type == F16 else 3e30
        x[rows // 2, ::2] = 6e-8 if x_type == F16 else 1e-36
        x = ref.encode(x, x_type)
        xv = ref.decode(x, x_type)
        ref.assert_close(ref.run(x, x_type, w, None, F32), xv @ w.values.T, ref.bound_of(xv, w) + 2.0 ** -126, F32, f"{rows} rows")


@pytest.mark.parametrize("rows", [1, 4, 11, 40, 64, 130, 300])
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_nan_and_infinities_stay_in_their_rows_and_outputs(gpu, rows, x_type):
    r = np.random.default_rng(rows)
    n, k = 140, 384
    w = ref.Weights(r, n, k, 64, BF16, whole=True)
    x = ref.whole_rows(r, rows, k, x_type)
    clean = ref.run(x, x_type, w, None, F32)
    bad_row, bad_n = rows // 2, 5
    for v in (np.nan, np.inf, -np.inf):
        y = x.copy()
        y[bad_row, 200] = ref.encode(np.array([v]), x_type)[0]
        got = ref.run(y, x_type, w, None, F32)
        keep = np.arange(rows) != bad_row
        assert np.array_equal(got[keep], clean[keep])
        assert not np.isfinite(got[bad_row]).any()
    for part in ("scale_bits", "bias_bits"):
        w2 = ref.Weights(np.random.default_rng(rows), n, k, 64, BF16, whole=True)
        bits = getattr(w2, part).copy()
        bits[bad_n, 3] = 0x7FC0
        setattr(w2, part, bits)
        got = ref.run(x, x_type, w2, None, F32)
        keep = np.arange(n) != bad_n
        assert np.array_equal(got[:, keep], clean[:, keep])
        assert np.isnan(got[:, bad_n]).all()


@pytest.mark.parametrize("rows", [1, 4, 16, 33, 64, 130, 300])
def test_the_same_bits_again(gpu, rows):
    r = np.random.default_rng(rows)
    w = ref.Weights(r, 300, 1024)
    x = ref.encode(r.standard_normal((rows, 1024)), F16)
    on = w.device()
    first = ref.run(x, F16, w, None, F32, weights=on)
    for _ in range(3):
        assert np.array_equal(ref.run(x, F16, w, None, F32, weights=on), first)


def test_two_streams_and_replays(gpu):
    """Calls at once on two streams, and captured calls replayed over other rows with eager work between."""
    r = np.random.default_rng(7)
    n, k = 500, 768
    w = ref.Weights(r, n, k)
    on = w.device()
    lib = capi.load()
    for rows in (1, 16, 60, 300):
        inputs = [ref.encode(r.standard_normal((rows, k)), F16) for _ in range(3)]
        eager = [ref.run(x, F16, w, weights=on) for x in inputs]
        streams = [rt.Stream(), rt.Stream()]
        x, outs = [rt.dev(v) for v in inputs], [rt.empty(rows * n * 2) for _ in range(3)]
        for i in range(3):
            rt.affine4_product(x[i], F16, k, *on, w.meta, 64, None, outs[i], F16, n, rows, n, k, streams[i % 2])
        for s in streams:
            s.synchronize()
        for o, e in zip(outs, eager):
            assert np.array_equal(o.download(np.uint16, rows * n).reshape(rows, n), e)
        s, fixed, out = streams[0], rt.dev(inputs[0]), outs[0]
        capi.check(lib.shrike_hip_graph_begin_capture(s.handle), "capture")
        rt.affine4_product(fixed, F16, k, *on, w.meta, 64, None, out, F16, n, rows, n, k, s)
        graph = lib.shrike_hip_graph_end_capture(s.handle)
        assert graph
        for i in (1, 2, 0, 1):
            fixed.upload(inputs[i])
            ref.run(inputs[(i + 1) % 3], F16, w, weights=on)
            capi.check(lib.shrike_hip_graph_launch(graph, s.handle), "launch")
            s.synchronize()
            assert np.array_equal(out.download(np.uint16, rows * n).reshape(rows, n), eager[i])
        capi.check(lib.shrike_hip_graph_destroy(graph), "destroy")


@pytest.mark.parametrize("rows", [2, 5, 20, 70, 300])
def test_rows_of_x_and_out_past_4_gib(gpu, rows):
    """Strides that put the later rows past what 32 bits reach, of bytes and of elements."""
    r = np.random.default_rng(rows)
    n, k = 65, 256
    w = ref.Weights(r, n, k, whole=True)
    x = ref.whole_rows(r, rows, k, F16)
    want = ref.encode(ref.decode(x, F16) @ w.values.T, F32)
    stride = ((1 << 33) // 2 // (rows - 1) + 1000) // 8 * 8  # the last row starts 8 GiB in
    far_x = rt.DeviceBuffer(((rows - 1) * stride + k) * 2)
    far_out = rt.DeviceBuffer(((rows - 1) * stride + n) * 4)
    for i in range(rows):
        far_x.upload(x[i], i * stride * 2)
    on = w.device()
    rt.affine4_product(far_x, F16, stride, *on, w.meta, 64, None, far_out, F32, stride, rows, n, k)
    rt.synchronize()
    for i in range(rows):
        assert np.array_equal(far_out.download(np.float32, n, i * stride * 4), want[i]), i


@pytest.mark.parametrize("rows", [1, 8, 40, 64, 130, 300])
def test_weights_past_4_gib(gpu, rows):
    """A head of 4.25 GiB of codes: its first, middle and last outputs."""
    r = np.random.default_rng(rows)
    k, n = 8192, 1114112 + 3
    piece = ref.Weights(r, 512, k, 64, BF16, whole=True)
    codes, scales, biases = rt.DeviceBuffer(n * k // 2), rt.DeviceBuffer(n * k // 32), rt.DeviceBuffer(n * k // 32)
    codes.fill(0x33), scales.fill(0), biases.fill(0)
    places = (0, n // 2 - 100, n - 512)
    for at in places:
        codes.upload(piece.codes, at * k // 2)
        scales.upload(piece.scale_bits, at * k // 32)
        biases.upload(piece.bias_bits, at * k // 32)
    x = ref.whole_rows(r, rows, k, F16)
    out = rt.DeviceBuffer(rows * n * 4)
    dx = rt.dev(x)
    rt.affine4_product(dx, F16, k, codes, scales, biases, BF16, 64, None, out, F32, n, rows, n, k)
    rt.synchronize()
    want = ref.encode(ref.decode(x, F16) @ piece.values.T, F32)
    for i in {0, rows // 2, rows - 1}:
        for at in places:
            assert np.array_equal(out.download(np.float32, 512, (i * n + at) * 4), want[i]), (i, at)
        assert np.all(out.download(np.float32, 1000, (i * n + 4000) * 4) == 0)
