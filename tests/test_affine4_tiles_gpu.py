"""shrike_hip_affine4_product over many rows: every shape of a workgroup (8, 16 or 32 rows with k in parts, tiles of 128 x 128 and of 256 x 256 outputs,
taken as there is work for the device), about where one gives way to the next, with edges, chunks and lengths that do not fill them."""
import numpy as np
import pytest

from shrike_amd import capi, runtime as rt
from tests import affine4_reference as ref
from tests.affine4_reference import BF16, F16, F32
from tests.test_affine4_gpu import closely, exactly

pytestmark = pytest.mark.gpu

# rows and outputs: more than two workgroups a CU of 32 rows x 256 outputs, no more than 256 tiles of 128 x 128; more than 512 of those
MIDDLE = [(65, 25600), (130, 16000), (1700, 1900), (25473, 70)]
LARGE = [(257, 25400), (3600, 3500), (25601, 450), (51100, 129)]


@pytest.mark.parametrize("rows,n", MIDDLE + LARGE)
@pytest.mark.parametrize("k,group", [(32, 32), (64, 64), (128, 128), (288, 32)])
def test_edges(gpu, rows, n, k, group):
    r = np.random.default_rng(rows + k)
    exactly(r, rows, n, k, group, F16 if k % 3 else BF16, F32, meta=F16 if group == 32 else BF16, symmetric=k == 64, bias=k == 128)


@pytest.mark.parametrize("rows,n", [(25473, 70), (1700, 1900), (1800, 7200)])
@pytest.mark.parametrize("k,group", [(64, 32), (96, 32), (128, 64), (160, 32), (192, 64), (256, 32), (320, 64), (384, 128), (448, 64), (480, 32), (512, 128), (544, 32), (576, 64), (640, 128),
                                     (1024, 64), (1056, 32), (1088, 64), (1152, 128), (2304, 64)])
def test_lengths(gpu, rows, n, k, group):
    r = np.random.default_rng(rows + k)
    exactly(r, rows, n, k, group, BF16 if k % 128 else F16, F32, meta=BF16 if k % 64 else F16)


@pytest.mark.parametrize("rows,n", [(300, 500), (1700, 1900), (3600, 3500)])
@pytest.mark.parametrize("x_type", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [False, True])
def test_types(gpu, rows, n, x_type, group, symmetric):
    r = np.random.default_rng(rows + group)
    for out_type, meta, bias, pad, x_pad in ((F16, F16, True, 5, 8), (BF16, BF16, False, 0, 64), (F32, BF16 if symmetric else F16, True, 8, 0)):
        closely(r, rows, n, 640, group, x_type, out_type, meta, symmetric, bias, pad=pad, x_pad=x_pad)


@pytest.mark.parametrize("rows,n", [(8, 4096), (9, 4096), (9, 40000), (16, 8192), (17, 8192), (16, 16384), (17, 16384), (33, 8192), (33, 16384), (64, 16384), (65, 16384), (64, 25600),
                                    (65, 25472), (128, 25600), (129, 25472), (512, 4096), (513, 4096), (512, 4097), (512, 8192), (513, 8192), (2048, 4096), (2048, 4097), (2049, 4096),
                                    (256, 65536), (257, 65536), (4096, 4352), (20000, 32), (20000, 200), (9, 32), (65, 1), (1000, 33), (5000, 40)])
def test_where_one_shape_gives_way_to_the_next(gpu, rows, n):
    r = np.random.default_rng(rows + n)
    for group in (32, 64, 128):
        exactly(r, rows, n, 384, group, F16, F32)


@pytest.mark.parametrize("rows", [1, 2, 20, 64, 70, 300])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_the_longest_rows(gpu, rows, group):
    r = np.random.default_rng(rows)
    exactly(r, rows, 40, 65536, group, F16, F32)
    closely(r, rows, 24, 65536 - 128, group, BF16, F16)


@pytest.mark.parametrize("rows,n", [(600, 5000), (600, 11000), (3700, 3584)])
def test_rows_past_4_gib_in_tiles(gpu, rows, n):
    """Rows of x that a tile reaches by 32 bits from its first, 4 GiB and more behind the first tile's; outputs as far apart."""
    r = np.random.default_rng(rows)
    k = 128
    w = ref.Weights(r, n, k, whole=True)
    x = ref.whole_rows(r, rows, k, F16)
    want = ref.encode(ref.decode(x, F16) @ w.values.T, F32)
    stride = (1 << 33) // 2 // (rows - 1) // 8 * 8 + 1000  # the last row starts 8 GiB in
    assert stride * 512 < 1 << 32
    out_stride = stride + n
    far_x, far_out = rt.DeviceBuffer(((rows - 1) * stride + k) * 2), rt.DeviceBuffer(((rows - 1) * out_stride + n) * 4)
    for i in range(rows):
        far_x.upload(x[i], i * stride * 2)
    rt.affine4_product(far_x, F16, stride, *w.device(), w.meta, 64, None, far_out, F32, out_stride, rows, n, k)
    rt.synchronize()
    for i in range(rows):
        assert np.array_equal(far_out.download(np.float32, n, i * out_stride * 4), want[i]), i


@pytest.mark.parametrize("rows,n", [(3600, 3500), (25473, 70)])
def test_nan_stays_in_its_row_and_output_of_tiles(gpu, rows, n):
    r = np.random.default_rng(5)
    k = 256
    w = ref.Weights(r, n, k, whole=True)
    x = ref.whole_rows(r, rows, k, F16)
    want = ref.decode(x, F16) @ w.values.T
    bad_rows, bad_outputs = [0, 255, 256, 1801, rows - 1], [0, 31, 32, n // 2 + 5, n - 1]
    for i, value in zip(bad_rows, (0x7E00, 0x7C00, 0xFC00, 0x7E00, 0x7C00)):
        x[i, (i * 7) % k] = value
    for i in bad_outputs:
        w.scale_bits[i, i % 4] = 0x7FC0
    got = ref.run(x, F16, w, None, F32)
    assert np.isnan(got[:, bad_outputs]).all() and not np.isfinite(got[bad_rows]).any()
    rest = np.setdiff1d(np.arange(rows), bad_rows)[:, None], np.setdiff1d(np.arange(n), bad_outputs)[None]
    ref.assert_exact(got[rest], want[rest], F32)


@pytest.mark.parametrize("rows", [1, 2, 17, 70, 1700, 3600])
def test_weights_used_by_calls_at_once_and_again(gpu, rows):
    """The same call on two streams at once, over and over: the same bits."""
    r = np.random.default_rng(rows)
    n, k = 3500, 512
    w = ref.Weights(r, n, k)
    x, on = rt.dev(ref.encode(r.standard_normal((rows, k)), F16)), w.device()
    streams, outs = [rt.Stream(), rt.Stream()], [rt.empty(rows * n * 2) for _ in range(2)]
    first = None
    for _ in range(4):
        for s, out in zip(streams, outs):
            out.fill(0xFF)
        rt.synchronize()
        for s, out in zip(streams, outs):
            rt.affine4_product(x, F16, k, *on, w.meta, 64, None, out, F16, n, rows, n, k, s)
        for s, out in zip(streams, outs):
            s.synchronize()
            bits = out.download(np.uint16, rows * n)
            first = bits if first is None else first
            assert np.array_equal(bits, first)


@pytest.mark.parametrize("rows", [8 * 65535 - 1, 8 * 65535, 8 * 65535 + 1, 8 * 65535 + 70, 1 << 20, 1 << 22])
def test_more_rows_than_a_launch_takes(gpu, rows):
    """Whole rows of a few kinds, over and over; every row of the output by its kind."""
    r = np.random.default_rng(rows % 1000)
    n, k, kinds = 24, 64, 61
    w = ref.Weights(r, n, k, whole=True)
    x = ref.whole_rows(r, kinds, k, F16)
    want = ref.encode(ref.decode(x, F16) @ w.values.T, F32)
    which = np.arange(rows) % kinds
    got = ref.run(x[which], F16, w, None, F32)
    assert np.array_equal(got, want[which])


@pytest.mark.parametrize("rows", [1, 3, 20, 70])
@pytest.mark.parametrize("group", [32, 64])
def test_as_many_outputs_as_there_may_be(gpu, rows, group):
    r = np.random.default_rng(rows)
    n, k, piece = 1 << 24, group, 4096
    w = ref.Weights(r, piece, k, group, whole=True)
    x = ref.whole_rows(r, rows, k, F16)
    want = ref.encode(ref.decode(x, F16) @ w.values.T, F32)
    times = n // piece
    codes, scales, biases = (rt.dev(np.tile(v, (times, 1))) for v in (w.codes, w.scale_bits, w.bias_bits))
    out = rt.DeviceBuffer(rows * n * 4)
    dx = rt.dev(x)
    rt.affine4_product(dx, F16, k, codes, scales, biases, w.meta, group, None, out, F32, n, rows, n, k)
    rt.synchronize()
    for i in {0, rows // 2, rows - 1}:
        got = out.download(np.float32, n, i * n * 4).reshape(times, piece)
        assert np.array_equal(got, np.broadcast_to(want[i], got.shape)), i


@pytest.mark.parametrize("rows,n", [(1, 300), (5, 300), (20, 300), (64, 16384), (25473, 70), (3600, 3500)])
@pytest.mark.parametrize("k", [32, 96, 160, 288])
@pytest.mark.parametrize("value", [0x7FC0, 0x7F80])
def test_scales_of_the_next_output_do_not_count(gpu, rows, n, k, value):
    """Rows of an odd number of groups of 32: where the last one ends in the middle of a step, the next output's scales and biases stand behind."""
    r = np.random.default_rng(k)
    w = ref.Weights(r, n, k, 32, whole=True)
    x = ref.whole_rows(r, rows, k, F16)
    want = ref.decode(x, F16) @ w.values.T
    bad = [1, 32, 64, n // 2, n - 1]
    w.scale_bits[bad] = value
    w.bias_bits[bad] = value
    got = ref.run(x, F16, w, None, F32)
    good = np.setdiff1d(np.arange(n), bad)
    ref.assert_exact(np.ascontiguousarray(got[:, good]), want[:, good], F32)


@pytest.mark.parametrize("rows,n", [(1, 301), (4, 301), (20, 301), (64, 16384), (25473, 70), (3600, 3500)])
@pytest.mark.parametrize("k,group", [(96, 32), (320, 64)])
def test_scales_biases_and_outputs_at_addresses_of_their_own_size(gpu, rows, n, k, group):
    r = np.random.default_rng(rows)
    w = ref.Weights(r, n, k, group, F16, whole=True)
    x, own = ref.whole_rows(r, rows, k, F16), ref.encode(r.integers(-9, 10, n) * 0.5, F16)
    want = ref.encode(ref.decode(x, F16) @ w.values.T + ref.decode(own, F16), F16)

    def behind(a, offset):  # the array `offset` bytes behind an allocation's start
        buf = rt.empty(a.nbytes + 64)
        buf.upload(np.ascontiguousarray(a).view(np.uint8).reshape(-1), offset)
        return buf

    dx, codes, scales, biases, bias = rt.dev(x), rt.dev(w.codes), behind(w.scale_bits, 2), behind(w.bias_bits, 6), behind(own, 10)
    out = rt.empty(rows * n * 2 + 64).fill(0xA5)
    rt.affine4_product(dx, F16, k, codes, scales.ptr + 2, biases.ptr + 6, w.meta, group, bias.ptr + 10, out.ptr + 14, F16, n, rows, n, k)
    rt.synchronize()
    assert np.array_equal(out.download(np.uint16, rows * n, 14).reshape(rows, n), want)
    assert np.all(out.download(np.uint8, 14) == 0xA5) and np.all(out.download(np.uint8, 50, rows * n * 2 + 14) == 0xA5)
