"""shrike_hip_affine4_product: the sums of x a group to their last bit, and sums as a whole closer than single bounds hold them."""
import numpy as np
import pytest

from tests import affine4_reference as ref
from tests.affine4_reference import BF16, F16, F32

pytestmark = pytest.mark.gpu

# rows, outputs, k: one row, 8, 16 and 32 rows a workgroup, tiles of 128 x 128 and of 256 x 256
SHAPES = [(1, 300, 640), (5, 300, 640), (20, 70, 640), (64, 16384, 256), (70, 9000, 640), (1700, 1900, 640), (3600, 3500, 640)]


def set_weights(w, codes, scales, biases):
    """Codes [n, k], scales and biases [n, groups] (None: symmetric) in place of what `w` had."""
    w.codes = np.ascontiguousarray((codes[:, 0::2] | codes[:, 1::2] << 4).astype(np.uint8))
    w.scale_bits, w.bias_bits = ref.encode(scales, w.meta), None if biases is None else ref.encode(biases, w.meta)
    s = np.repeat(ref.decode(w.scale_bits, w.meta), w.group, 1)
    w.values = codes * s + (-8.0 * s if biases is None else np.repeat(ref.decode(w.bias_bits, w.meta), w.group, 1))


def long_rows(r, rows, k, x_type, fraction):
    """Values of one sign a row whose sums of 32 and of 64 have up to 24 bits, exactly: large whole ones, and some odd multiples of `fraction`."""
    most = 2048 if x_type == F16 else 256
    x = r.integers(most // 2, most, (rows, k)).astype(np.float64) * (1 if x_type == F16 else 8)
    small = r.random((rows, k)) < 0.1
    x[small] = (2 * r.integers(0, 64, small.sum()) + 1) * fraction
    x *= r.choice([-1.0, 1.0], (rows, 1))
    bits = ref.encode(x, x_type)
    assert np.array_equal(ref.decode(bits, x_type), x)
    return bits


@pytest.mark.parametrize("rows,n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_type", [F16, BF16])
@pytest.mark.parametrize("meta", [F16, BF16])
def test_every_bit_of_a_group_s_sum(gpu, rows, n, k, group, x_type, meta):
    """Outputs that are one group's sum of x, all 24 bits of it, times a power of two: codes of 0, and one bias that is not 0. (The sums of a group of 128 are at
    most 2^18, those of 32 and 64 at most 2^17: multiples of 2^-6 of them fit 24 bits.)"""
    r = np.random.default_rng(rows + group)
    w = ref.Weights(r, n, k, group, meta, whole=True)
    biases = np.zeros((n, k // group))
    biases[np.arange(n), r.integers(0, k // group, n)] = 2.0 ** r.integers(-3, 4, n) * r.choice([-1.0, 1.0], n)
    set_weights(w, np.zeros((n, k), np.uint8), np.ones((n, k // group)), biases)
    x = long_rows(r, rows, k, x_type, 2.0 ** -6)
    want = ref.decode(x, x_type) @ w.values.T
    assert np.array_equal(want.astype(np.float32).astype(np.float64), want)
    ref.assert_exact(ref.run(x, x_type, w, None, F32), want, F32, f"{rows} x {n} x {k}, groups of {group}")


@pytest.mark.parametrize("rows,n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_symmetric_weights_over_sums_of_17_bits(gpu, rows, n, k, group, x_type):
    """One group whose scale is not 0: whole numbers under 2^24 throughout (sums of x * code under 15 * 2^17, of 8 x under 2^20; of a group of 128, values half as large)."""
    r = np.random.default_rng(rows + group)
    w = ref.Weights(r, n, k, group, BF16, symmetric=True, whole=True)
    scales = np.zeros((n, k // group))
    scales[np.arange(n), r.integers(0, k // group, n)] = 2.0 ** r.integers(-3, 4, n)
    set_weights(w, r.integers(0, 16, (n, k)).astype(np.uint8), scales, None)
    most = (2048 if x_type == F16 else 256) // (2 if group == 128 else 1)
    x = ref.encode(r.integers(most // 2, most, (rows, k)).astype(np.float64), x_type)
    ref.assert_exact(ref.run(x, x_type, w, None, F32), ref.decode(x, x_type) @ w.values.T, F32, f"{rows} x {n} x {k}, groups of {group}")


@pytest.mark.parametrize("rows,n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_bit_of_an_fp16_bias(gpu, rows, n, k, group):
    """Biases of 11 bits over sums of up to 13: products of 24."""
    r = np.random.default_rng(rows + group)
    w = ref.Weights(r, n, k, group, F16, whole=True)
    biases = np.zeros((n, k // group))
    biases[np.arange(n), r.integers(0, k // group, n)] = (2 * r.integers(512, 1024, n) + 1) * 2.0 ** -10 * r.choice([-1.0, 1.0], n)
    set_weights(w, np.zeros((n, k), np.uint8), np.ones((n, k // group)), biases)
    x = ref.encode(r.integers(0, 64, (rows, k)).astype(np.float64), F16)
    ref.assert_exact(ref.run(x, F16, w, None, F32), ref.decode(x, F16) @ w.values.T, F32, f"{rows} x {n} x {k}, groups of {group}")


@pytest.mark.parametrize("rows,n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_subnormal_rows_lose_nothing(gpu, rows, n, k, group, x_type):
    """Activations that are subnormal throughout or in part, in whole multiples of the type's smallest (of bf16, with scales that bring the results back)."""
    r = np.random.default_rng(rows + group)
    w = ref.Weights(r, n, k, group, BF16, whole=True)
    step, top = (2.0 ** -24, 1024) if x_type == F16 else (2.0 ** -133, 128)
    codes = np.repeat(r.integers(0, 16, (n, k // 2)), 2, 1).astype(np.uint8)
    scales, biases = np.zeros((n, k // group)), np.zeros((n, k // group))
    at = r.integers(0, k // group, n)
    scales[np.arange(n), at] = 1.0 if x_type == F16 else 2.0 ** 40
    biases[np.arange(n), at] = -scales[np.arange(n), at]
    set_weights(w, codes, scales, biases)
    x = r.integers(-top, top, (rows, k)) * step
    x[1::2] *= np.where(r.random((len(x[1::2]), k)) < 0.5, 2.0, 1.0)  # every second row reaches above the subnormals
    bits = ref.encode(x, x_type)
    ref.assert_exact(ref.run(bits, x_type, w, None, F32), ref.decode(bits, x_type) @ w.values.T, F32, f"{rows} x {n} x {k}, groups of {group}")


@pytest.mark.parametrize("rows,n,k", [(1, 4100, 2880), (5, 900, 2880), (37, 2049, 2304), (64, 16384, 2304), (70, 9000, 640), (1700, 1900, 2880), (3600, 3500, 2880)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_sums_as_a_whole(gpu, rows, n, k, group, x_type):
    """The errors' norm. Their signs are as random as the values', so roundings add up as squares: a group's sum of x * code is at most 16 additions ahead of
    its scaling, and then there are two into the running sum a group (64 of k at most), joined over up to eight parts: each off by half a step, 2^-24, of a
    running sum that is no larger than the products' root of squares, on average. Products that lose some of their 24 bits show as more."""
    if k % group:
        k -= k % group
    r = np.random.default_rng(rows + group)
    w = ref.Weights(r, n, k, group, BF16)
    x = ref.encode(r.standard_normal((rows, k)), x_type)
    xv = ref.decode(x, x_type)
    s = np.repeat(ref.decode(w.scale_bits, BF16), group, 1)
    q = np.stack([w.codes & 15, w.codes >> 4], -1).reshape(n, k)
    squares = (xv ** 2).sum(0) @ ((q * s) ** 2 + np.repeat(ref.decode(w.bias_bits, BF16), group, 1) ** 2).T
    got = ref.decode(ref.run(x, x_type, w, None, F32), F32)
    off = np.sqrt(((got - xv @ w.values.T) ** 2).sum())
    allowed = np.sqrt(squares.sum() * (16 + 2 * (k // min(group, 64)) + 8)) * 2.0 ** -24
    assert off <= allowed, f"off by {off / allowed:.3f} of what is allowed"
