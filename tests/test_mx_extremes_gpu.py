"""NaN, infinities and scales at both ends of their range through every kernel over microscaled blocks: what is not a number stays with the rows and
outputs that it belongs to, and the rest is what it would be without it."""
import numpy as np
import pytest

from shrike_amd import capi
from shrike_amd import synth as S
from tests import mx_reference as R
from tests import test_mx_gpu as base
from tests import test_mx_shapes_gpu as shapes
from tests.test_mx_experts_gpu import Chunk, by_counts

pytestmark = pytest.mark.gpu
F16, BF16 = capi.ELEM_F16, capi.ELEM_BF16
NAN = 255  # a scale byte
PRODUCTS = [(9, 50), (40, 50), (70, 6200), (520, 8200), (1100, 8200)]  # up to 16 rows, up to 64, and tiles of 64, 128 and 256


def same_bits(got, want):
    return (got == want) | ((got & 0x7FFF) + (want & 0x7FFF) == 0)  # (a zero's sign is not the sum's)


# k of 11 and of 37 blocks: scales read byte by byte, and 16 at a time with the last of a row moved up to their places
@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows,n", PRODUCTS)
@pytest.mark.parametrize("k", [352, 1184])
def test_product_keeps_nan_to_its_rows(gpu, x_fmt, rows, n, k):
    rng = np.random.default_rng(rows + n + k)
    x, w = shapes.exact_rows(rng, rows, k, x_fmt), shapes.exact_rows(rng, n, k, R.E2M1)
    want = (R.values(*x, x_fmt) @ R.values(*w, R.E2M1).T).astype(np.float16)
    blocks = k // 32
    bad_rows, bad_columns = {0, rows // 2, rows - 1}, {3, n // 2 + 1, n - 1}
    for i, r in enumerate(sorted(bad_rows)):
        x[1][r, (0, blocks // 2, blocks - 1)[i]] = NAN
    if x_fmt == R.E4M3:  # and a code that is none, the last of its row
        x[0][2, k - 1] = 0xFF
        bad_rows.add(2)
    for i, c in enumerate(sorted(bad_columns)):
        w[1][c, (blocks - 1, 0, blocks // 2)[i]] = NAN
    got = base.run_product(gpu, x, w, x_fmt, None, F16, rows, n, k)
    nan = np.zeros((rows, n), bool)
    nan[sorted(bad_rows)], nan[:, sorted(bad_columns)] = True, True
    assert np.array_equal(np.isnan(got.view(np.float16)), nan)
    assert np.all(same_bits(got, want.view(np.uint16)) | nan)


@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows,n", PRODUCTS)
def test_product_of_scales_that_cancel(gpu, x_fmt, rows, n):
    """Blocks of x up to 2^127 times as large against weights as much smaller, and the other way about: the products are ordinary numbers."""
    k = 608
    rng = np.random.default_rng(rows * n)
    x, w = shapes.exact_rows(rng, rows, k, x_fmt), shapes.exact_rows(rng, n, k, R.E2M1)
    x[1][:], w[1][:] = 127, 127
    want = (R.values(*x, x_fmt) @ R.values(*w, R.E2M1).T).astype(np.float16).view(np.uint16)
    e = rng.integers(-126, 127, k // 32)
    e[[0, -1]], e[[1, -2]] = 127, -127
    x[1][:] += e.astype(np.uint8)
    w[1][:] -= e.astype(np.uint8)
    assert x[1].min() == 0 and x[1].max() == 254 and np.array_equal(x[1][0].astype(int) + w[1][0], np.full(k // 32, 254))
    assert np.all(same_bits(base.run_product(gpu, x, w, x_fmt, None, F16, rows, n, k), want))


@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows,n", PRODUCTS)
def test_product_below_the_normal_range(gpu, x_fmt, rows, n):
    """Outputs of bf16 about 2^-126 and below: the sums keep their subnormal digits, and are rounded once."""
    k = 352
    rng = np.random.default_rng(rows + n)
    for shift in (-124, -130, -138):
        x, w = shapes.exact_rows(rng, rows, k, x_fmt), shapes.exact_rows(rng, n, k, R.E2M1)
        x[1][:] -= np.uint8(-shift // 2)
        w[1][:] -= np.uint8(-shift // 2)
        want = shapes.rounded(R.values(*x, x_fmt) @ R.values(*w, R.E2M1).T, BF16)
        assert np.all(same_bits(base.run_product(gpu, x, w, x_fmt, None, BF16, rows, n, k), want)), shift


@pytest.mark.parametrize("with_delta", [True, False])
def test_norm_of_rows_that_are_not_numbers(gpu, with_delta):
    rows, d = 9, 2880
    rng = np.random.default_rng(4)
    hidden, delta = rng.standard_normal((rows, d)).astype(np.float16), rng.standard_normal((rows, d)).astype(np.float16)
    hidden[1, 2000], hidden[3, 0], hidden[5, d - 1], hidden[7] = np.inf, np.nan, -np.inf, 0.0
    delta[7] = 0.0
    hidden[2, 40], delta[2, 40] = 60000.0, 60000.0  # (their sum is past fp16)
    weight = S.f32_to_bf16_bits(rng.uniform(0.5, 1.5, d).astype(np.float32))
    h, h2, w, dl = gpu.dev(hidden), gpu.dev(hidden), gpu.dev(weight), gpu.dev(delta) if with_delta else None
    want, out, total = gpu.empty(2 * rows * d), gpu.empty(2 * rows * d), gpu.empty(2 * rows * d) if with_delta else None
    codes, scales = gpu.empty(rows * d), gpu.empty(rows * d // 32)
    gpu.residual_add_rmsnorm_bf16w(h2, dl, w, want, d, 1e-6, rows)
    gpu.residual_add_rmsnorm_bf16w_mx8(h, dl, w, total, out, codes, scales, d, 1e-6, rows)
    gpu.synchronize()
    normed = out.download(np.uint16, rows * d)
    assert np.array_equal(normed, want.download(np.uint16, rows * d))
    with np.errstate(invalid="ignore"):
        want_codes, want_scales = R.quantize(R.to_float(normed, F16).reshape(rows, d), R.E4M3)
    assert np.array_equal(scales.download(np.uint8).reshape(rows, -1), want_scales)
    assert np.array_equal(codes.download(np.uint8).reshape(rows, d), want_codes)
    bad = (want_scales == NAN).any(1)
    assert list(np.flatnonzero(bad)) == ([1, 2, 3, 5] if with_delta else [1, 3, 5]) and not want_codes[7].any()


# ---------------------------------------------------------------- the experts

D = 576
# kind, f, experts' rows (a chunk) or tokens of two positions each (single tokens)
KINDS = [("few", 192, 7), ("few", 128, 7), ("few", 320, 6), ("lds", 192, 64), ("thin", 192, (13, 30, 60, 9)), ("runs", 1024, (60, 110, 260, 90))]
EXPERTS = 4


def run(gpu, kind, ex, act, x, tokens, rng):
    """Runs the FFN of that kind. Returns, by pair: token, expert, activations' codes and scales; and a call that holds the outputs, by pair, to
    (values, bounds): of a chunk the pair's row, of single tokens the weighted sum and the residual."""
    if kind in ("thin", "runs"):
        expert = by_counts(rng, tokens)
        chunk = Chunk(gpu, ex, act, x, expert)
        assert chunk.many(len(expert)) == (kind == "runs")
        out, codes, scales = chunk.run(np.arange(len(expert)))

        def check(values, bounds):
            assert np.array_equal(np.isnan(R.to_float(out, F16)), np.isnan(values))
            fine = ~np.isnan(values)
            R.assert_within(out[fine], values[fine], bounds[fine], F16)
        return np.arange(len(expert)), expert, codes, scales, check
    k = 2
    assert ((ex.f + 63) // 64 * tokens * k >= 256) == (kind == "lds") and (D // 16 * tokens <= 256) == (kind == "few")
    expert = rng.integers(0, ex.n, (tokens, k))
    weights = rng.uniform(0.5, 1.0, (tokens, k)).astype(np.float16)
    residual = rng.standard_normal((tokens, D)).astype(np.float16)
    moe = gpu.MoE(D, ex.f, ex.n, k, activation=act, additive_biases=ex.biases)
    y, codes, scales, _ = base.run_decode(gpu, moe, ex, base.make_pool(gpu, ex), expert.astype(np.uint32), x, weights, residual, None, tokens, k)

    def check(values, bounds):
        share = weights.astype(np.float64)[..., None]
        want, bound = residual + (share * values.reshape(tokens, k, D)).sum(1), (share * bounds.reshape(tokens, k, D)).sum(1)
        parts = np.abs(residual) + (share * np.abs(values).reshape(tokens, k, D)).sum(1)
        assert np.array_equal(np.isnan(R.to_float(y, F16)), np.isnan(want))
        fine = ~np.isnan(want)
        # (weighted sums are rounded as often as there are waves with a part of them, 16 at most, and their sum as often again)
        if fine.any():
            R.assert_within(y[fine], want[fine], (bound + 32 * 2.0 ** -24 * parts)[fine], F16)
    return np.repeat(np.arange(tokens), k), expert.reshape(-1), codes, scales, check


def outputs(ex, expert, codes, scales):
    """What the down products of such activations are, with their bounds; NaN where a NaN meets them."""
    values, bounds = np.empty((len(expert), ex.d)), np.empty((len(expert), ex.d))
    with np.errstate(invalid="ignore"):
        for e in set(expert):
            mine = expert == e
            values[mine], bounds[mine] = ex.down(e, (codes[mine], scales[mine]))
    return values, bounds


def assert_blocks(codes, scales, bad, values, bounds):
    """Blocks that are not numbers have a NaN's scale and no codes, and every other has the codes of its values."""
    assert np.array_equal(scales == NAN, bad)
    at = codes.reshape(*bad.shape, 32)
    assert not at[bad].any()
    values, bounds = (v.reshape(*bad.shape, 32)[~bad] for v in (values, bounds))
    R.assert_quantized(at[~bad], scales[~bad][:, None], values, bounds)


@pytest.mark.parametrize("kind,f,tokens", KINDS)
@pytest.mark.parametrize("act", [capi.ACT_GELU_TANH, capi.ACT_SILU, capi.ACT_CLAMPED_SWIGLU])
def test_experts_keep_nan_to_their_rows(gpu, kind, f, tokens, act):
    """A NaN in a gate row, an up row and a down row of three experts, by turns, a fourth without; and in some tokens' rows, as a scale or a code."""
    rng = np.random.default_rng(f + act)
    ex = R.Experts(rng, EXPERTS, D, f, act == capi.ACT_CLAMPED_SWIGLU)
    gate, up, down = [(act + i) % 3 for i in range(3)]
    rows = dict(gate=int(rng.integers(0, f)), up=int(rng.integers(0, f)), down=D - 1)
    for e, name in ((gate, "gate"), (up, "up"), (down, "down")):
        block = int(rng.integers(0, (f if name == "down" else D) // 32))
        scales = ex.parts[e][name][1]
        scales[rows[name], block] = NAN
        ex.blobs[e][getattr(ex.off, name + "_s_off") + rows[name] * scales.shape[1] + block] = NAN
    count = sum(tokens) if isinstance(tokens, tuple) else tokens
    x = R.random_rows(rng, count, D, R.E4M3)
    strange = rng.permutation(count)[:max(2, count // 16)]
    for i, t in enumerate(strange):
        if i % 2:
            x[1][t, int(rng.integers(0, D // 32))] = NAN
        else:
            x[0][t, int(rng.integers(0, D))] = 0x7F
    token, expert, codes, scales, check = run(gpu, kind, ex, act, x, tokens, rng)
    bad = np.zeros(scales.shape, bool)
    bad[np.isin(token, strange)] = True
    bad[expert == gate, rows["gate"] // 32] = True
    bad[expert == up, rows["up"] // 32] = True
    some = np.concatenate([np.flatnonzero(expert == e)[:6] for e in range(EXPERTS)])
    a, da = np.empty((len(some), f)), np.empty((len(some), f))
    with np.errstate(invalid="ignore"):
        for i, p in enumerate(some):
            (a[i],), (da[i],) = ex.act(expert[p], (x[0][token[p]][None], x[1][token[p]][None]), act)
    assert_blocks(codes[some], scales[some], bad[some], a, da)
    assert np.array_equal(scales == NAN, bad) and not codes.reshape(*bad.shape, 32)[bad].any()
    values, bounds = outputs(ex, expert, codes, scales)
    nan = np.repeat(bad.any(1)[:, None], D, axis=1)
    nan[expert == down, D - 1] = True
    assert np.array_equal(np.isnan(values), nan) and not nan.all()
    check(values, bounds)


def glu(g, u, act):
    """The activation in 64 bits, tanh as the logistic function that it is, so that its far ends keep their digits."""
    if act == capi.ACT_CLAMPED_SWIGLU:
        g, u = np.minimum(g, 7.0), np.clip(u, -7.0, 7.0) + 1
        return g / (1 + np.exp(-1.702 * g)) * u
    if act == capi.ACT_SILU:
        return g / (1 + np.exp(-g)) * u
    inner = np.clip(0.7978845608028654 * (g + 0.044715 * g ** 3), -20, 20)
    return g / (1 + np.exp(-2 * inner)) * u


@pytest.mark.parametrize("kind,f,tokens", KINDS)
@pytest.mark.parametrize("act", [capi.ACT_GELU_TANH, capi.ACT_SILU, capi.ACT_CLAMPED_SWIGLU])
def test_experts_whose_activations_leave_fp32(gpu, kind, f, tokens, act):
    """Rows of ones times 2^0, 2^100 or 2^127 at weights of +-1, so that gate and up are +-576, +-576 * 2^100 or infinite, by rows of blocks of which
    gate's are all negative, all positive, all but one negative, or any: an activation that fp32 does not hold makes its block NaN, and no other."""
    rng = np.random.default_rng(f + act + 1)
    ex = R.Experts(rng, EXPERTS, D, f)
    signs = {}
    for e in range(EXPERTS):
        gate = np.full((f // 32, 32), -1.0)
        gate[1::4], gate[2::4, 17] = 1.0, 1.0
        gate[3::4] = rng.choice([-1.0, 1.0], gate[3::4].shape)
        signs[e] = dict(gate=gate.reshape(-1), up=rng.choice([-1.0, 1.0], f))
        for name, n in (("gate", D), ("up", D)):
            codes, scales = ex.parts[e][name]
            codes[:] = np.where(signs[e][name] > 0, 0x22, 0xAA)[:, None]
            scales[:] = 127
            at, s_at = getattr(ex.off, name + "_w_off"), getattr(ex.off, name + "_s_off")
            ex.blobs[e][at:at + codes.size], ex.blobs[e][s_at:s_at + scales.size] = codes.reshape(-1), 127
        scales = ex.parts[e]["down"][1]
        scales[:] = 127 - 24  # (activations of up to 2^18 are many times that in a sum, and the outputs fp16)
        ex.blobs[e][ex.off.down_s_off:ex.off.down_s_off + scales.size] = 127 - 24
    count = sum(tokens) if isinstance(tokens, tuple) else tokens
    power = rng.permutation(np.resize([0, 100, 127], count))
    x = np.full((count, D), 0x38, np.uint8), np.repeat((127 + power)[:, None], D // 32, axis=1).astype(np.uint8)
    token, expert, codes, scales, check = run(gpu, kind, ex, act, x, tokens, rng)
    size = np.where(power == 127, np.inf, D * np.exp2(power.astype(np.float64)))[token][:, None]
    with np.errstate(over="ignore", invalid="ignore"):
        a = glu(np.stack([signs[e]["gate"] for e in expert]) * size, np.stack([signs[e]["up"] for e in expert]) * size, act)
        a = np.where(np.isfinite(a.astype(np.float32)), a, np.nan)
    bad = ~np.isfinite(a).reshape(*scales.shape, 32).all(-1)
    assert bad.any() and not bad.all()
    # (a logistic function of 40 is off by 57.7 * 2^-24 and a few roundings more; one past 2^-126 is nothing in fp32)
    assert_blocks(codes, scales, bad, a, 2.0 ** -16 * np.abs(a) + 2.0 ** -120)
    check(*outputs(ex, expert, codes, scales))
