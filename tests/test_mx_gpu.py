"""The operators over microscaled blocks on the GPU, against tests/mx_reference.py: quantising and back bit for bit, the norm's fp16
rows as the norm's own call gives them and its codes as the quantiser's, products and the experts' FFN within what the matrix
instruction and the roundings can lose."""
import ctypes as C

import numpy as np
import pytest

from shrike_amd import capi
from shrike_amd import synth as S
from tests import mx_reference as R
from tests.test_graph_replay_gpu import capture

pytestmark = pytest.mark.gpu
F16, BF16, F32 = capi.ELEM_F16, capi.ELEM_BF16, capi.ELEM_F32
SIZE = {F16: 2, BF16: 2, F32: 4}


def as_bits(x, dtype):
    """float64 values that the type holds -> its bits."""
    if dtype == F16:
        return x.astype(np.float16).view(np.uint16)
    if dtype == F32:
        return x.astype(np.float32).view(np.uint32)
    return (x.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)


def as_values(bits, dtype):
    if dtype == F32:
        return bits.view(np.float32).astype(np.float64)
    return R.to_float(bits, dtype)


def code_bytes(fmt, d):
    return d if fmt == R.E4M3 else d // 2


def run_quantize(gpu, bits, dtype, stride, fmt, rows, d, ahead=0):
    """bits: [rows, stride] of the source; `ahead`: elements in front of its first."""
    src = gpu.dev(np.concatenate([np.zeros(ahead, bits.dtype), bits.reshape(-1)]))
    n, ns = rows * code_bytes(fmt, d), rows * d // 32
    codes, scales = gpu.empty(n + 64).fill(0xA5), gpu.empty(ns + 64).fill(0xA5)
    gpu.mx_quantize(src.ptr + ahead * bits.itemsize, dtype, stride, fmt, codes, scales, rows, d)
    gpu.synchronize()
    c, s = codes.download(np.uint8), scales.download(np.uint8)
    assert np.all(c[n:] == 0xA5) and np.all(s[ns:ns + 64] == 0xA5), "something behind the last row was written"
    return c[:n].reshape(rows, -1), s[:ns].reshape(rows, -1)


@pytest.mark.parametrize("fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,d,pad,ahead", [(1, 32, 0, 0), (1, 2048, 0, 0), (3, 96, 8, 0), (5, 64, 1, 0), (7, 160, 3, 1), (129, 2880, 40, 8),
                                              (1, 64, 5, 3), (2, 4096, 0, 4), (1000, 32, 0, 0)])
def test_quantize_and_back(gpu, fmt, dtype, rows, d, pad, ahead):
    rng = np.random.default_rng(rows * d + dtype)
    x = rng.standard_normal((rows, d + pad)) * np.exp2(rng.integers(-12, 12, (rows, 1)))
    x[:, ::7] *= np.exp2(rng.integers(-9, 3, x[:, ::7].shape))
    x[rng.random(x.shape) < 0.05] = 0.0
    bits = as_bits(x, dtype)
    x = as_values(bits, dtype)[:, :d]
    codes, scales = run_quantize(gpu, bits, dtype, d + pad, fmt, rows, d, ahead)
    want_codes, want_scales = R.quantize(x, fmt)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)
    # and back, into every type, between filler that stays
    dc, ds = gpu.dev(codes), gpu.dev(scales)
    v = R.values(codes, scales, fmt)
    for out in (F16, BF16, F32):
        stride = d + pad
        to = gpu.empty((ahead + rows * stride) * SIZE[out] + 16).fill(0x5A)
        gpu.mx_dequantize(dc, ds, fmt, to.ptr + ahead * SIZE[out], out, stride, rows, d)
        gpu.synchronize()
        kind = np.uint32 if out == F32 else np.uint16
        got = to.download(kind)[ahead:ahead + rows * stride].reshape(rows, stride)
        assert np.all(got[:, d:] == (0x5A5A5A5A if out == F32 else 0x5A5A))
        if out == F16:
            with np.errstate(over="ignore"):
                want = v.astype(np.float16).view(np.uint16)
        else:
            want = as_bits(v, out)  # bf16 and fp32 hold every value
        assert np.array_equal(got[:, :d], want)


@pytest.mark.parametrize("fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_quantize_any_value(gpu, fmt, dtype):
    """Blocks of zeros of either sign, of the type's smallest and largest values, midpoints between codes, infinities, NaN."""
    rng = np.random.default_rng(5)
    tiny, top = {F16: (2.0 ** -24, 65504.0), BF16: (2.0 ** -133, float(np.float32(3.3895314e38))), F32: (2.0 ** -149, float(np.finfo(np.float32).max))}[dtype]
    grid = R._grid(fmt)
    mid = (grid[1:] + grid[:-1]) / 2
    blocks = [np.zeros(32), np.full(32, -0.0), np.full(32, tiny), np.full(32, -top), np.r_[top, np.full(31, tiny)],
              np.r_[1.0, np.full(31, -2.0 ** -20)], np.r_[np.full(31, tiny), 5 * tiny]]
    for first in range(0, len(mid), 31):  # the format's largest value sets the block's scale
        m = np.resize(mid[first:first + 31], 31)
        blocks += [np.r_[grid[-1], m], np.r_[-grid[-1], -m], np.r_[grid[-1] * 1.1, m]]
    for bad in (np.inf, -np.inf, np.nan):
        for at in (0, 13, 31):
            b = rng.standard_normal(32)
            b[at] = bad
            blocks.append(b)
    with np.errstate(invalid="ignore"):
        bits = as_bits(np.array(blocks), dtype)
    bits = bits.reshape(1, -1)
    x = as_values(bits, dtype)
    codes, scales = run_quantize(gpu, bits, dtype, x.shape[1], fmt, 1, x.shape[1])
    want_codes, want_scales = R.quantize(x, fmt)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)
    assert np.count_nonzero(scales == 255) == 9


@pytest.mark.parametrize("fmt", [R.E4M3, R.E2M1])
def test_dequantize_every_code_at_every_scale(gpu, fmt):
    every = np.arange(256, dtype=np.uint8)
    d = 512 if fmt == R.E2M1 else 256  # a row holds every byte of codes
    codes = np.tile(every, (256, 1))
    scales = np.repeat(every[:, None], d // 32, axis=1)
    dc, ds = gpu.dev(codes), gpu.dev(scales)
    v = R.values(codes, scales, fmt)
    for out in (F32, F16, BF16):
        to = gpu.empty(256 * d * SIZE[out])
        gpu.mx_dequantize(dc, ds, fmt, to, out, d, 256, d)
        gpu.synchronize()
        got = as_values(to.download(np.uint32 if out == F32 else np.uint16).reshape(256, d), out)
        with np.errstate(over="ignore"):
            want = v.astype(np.float32).astype(np.float64)
            if out == F16:
                want = want.astype(np.float16).astype(np.float64)
            if out == BF16:  # to nearest even
                u = want.astype(np.float32).view(np.uint32).astype(np.uint64)
                want = np.where(np.isnan(want), np.nan, ((((u + 0x7FFF + (u >> 16 & 1)) >> 16) << 16).astype(np.uint32)).view(np.float32))
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("rows,d", [(1, 32), (1, 2880), (5, 64), (3, 96), (37, 512), (2, 544), (9, 2048), (4, 4096), (300, 160)])
@pytest.mark.parametrize("with_delta,with_out,in_place", [(True, True, False), (True, False, True), (False, True, False), (False, False, False)])
def test_norm_with_8_bit_rows(gpu, rows, d, with_delta, with_out, in_place):
    rng = np.random.default_rng(rows + d)
    hidden = S.f32_to_f16_bits((3 * rng.standard_normal((rows, d))).astype(np.float32).reshape(-1))
    delta = S.f32_to_f16_bits(rng.standard_normal(rows * d).astype(np.float32))
    weight = S.f32_to_bf16_bits(rng.uniform(0.5, 1.5, d).astype(np.float32))
    h, w = gpu.dev(hidden), gpu.dev(weight)
    dl = gpu.dev(delta) if with_delta else None
    # the call it stands beside
    h2, want_out = gpu.dev(hidden), gpu.empty(2 * rows * d)
    gpu.residual_add_rmsnorm_bf16w(h2, dl, w, want_out, d, 1e-6, rows)
    total = None if not with_delta else h if in_place else gpu.empty(2 * rows * d)
    out = gpu.empty(2 * rows * d) if with_out else None
    codes, scales = gpu.empty(rows * d + 64).fill(0xA5), gpu.empty(rows * d // 32 + 64).fill(0xA5)
    gpu.residual_add_rmsnorm_bf16w_mx8(h, dl, w, total, out, codes, scales, d, 1e-6, rows)
    gpu.synchronize()
    normed = want_out.download(np.uint16, rows * d)
    if with_delta:
        assert np.array_equal(total.download(np.uint16, rows * d), h2.download(np.uint16, rows * d))
    if not in_place:
        assert np.array_equal(h.download(np.uint16, rows * d), hidden)
    if with_out:
        assert np.array_equal(out.download(np.uint16, rows * d), normed)
    want_codes, want_scales = R.quantize(R.to_float(normed, F16).reshape(rows, d), R.E4M3)
    c, s = codes.download(np.uint8), scales.download(np.uint8)
    assert np.array_equal(s[:rows * d // 32].reshape(rows, -1), want_scales)
    assert np.array_equal(c[:rows * d].reshape(rows, d), want_codes)
    assert np.all(c[rows * d:] == 0xA5) and np.all(s[rows * d // 32:rows * d // 32 + 64] == 0xA5)


def run_product(gpu, x, w, x_fmt, bias, dtype, rows, n, k, pad=0, ahead=0, stream=None):
    """Scales and the bias start at odd places on purpose."""
    dx, dw = gpu.dev(x[0]), gpu.dev(w[0])
    sx, sw = gpu.dev(np.r_[np.uint8(255), x[1].reshape(-1)]), gpu.dev(np.r_[np.uint8(255), w[1].reshape(-1)])
    b = gpu.dev(np.r_[np.uint16(0x7FC0), bias]) if bias is not None else None
    stride = n + pad
    out = gpu.empty(2 * (ahead + rows * stride + 32)).fill(0x5A)
    gpu.mx_product(dx, sx.ptr + 1, x_fmt, dw, sw.ptr + 1, b.ptr + 2 if b else None, out.ptr + 2 * ahead, dtype, stride, rows, n, k, stream)
    (stream or gpu).synchronize()
    raw = out.download(np.uint16)
    body = raw[ahead:ahead + rows * stride].reshape(rows, stride)
    assert np.all(raw[:ahead] == 0x5A5A) and np.all(raw[ahead + rows * stride:][:32] == 0x5A5A) and np.all(body[:, n:] == 0x5A5A), "written past the rows"
    return body[:, :n]


@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows,n,k,pad,ahead", [
    (1, 1, 32, 0, 0), (1, 16, 64, 0, 0), (1, 33, 96, 0, 1), (1, 2880, 2880, 0, 0), (2, 31, 128, 3, 0), (7, 64, 160, 0, 0), (15, 100, 256, 4, 0),
    (16, 48, 288, 0, 2), (17, 16, 32, 0, 0), (17, 257, 480, 1, 3), (33, 64, 512, 0, 0), (63, 40, 224, 0, 0), (64, 300, 544, 0, 0), (65, 129, 352, 4, 4),
    (130, 513, 320, 0, 0), (37, 61, 2304, 0, 0), (128, 256, 256, 0, 0), (129, 256, 768, 0, 0), (257, 32, 64, 0, 0), (3, 20, 8192, 0, 0), (20, 20, 8224, 0, 0)])
def test_product(gpu, x_fmt, rows, n, k, pad, ahead):
    rng = np.random.default_rng(rows * 7 + n * 3 + k)
    x, w = R.random_rows(rng, rows, k, x_fmt, 0.7), R.random_rows(rng, n, k, R.E2M1, 0.7)
    dtype = F16 if (rows + n) % 2 else BF16
    bias = (rng.standard_normal(n).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16) if n % 3 else None
    got = run_product(gpu, x, w, x_fmt, bias, dtype, rows, n, k, pad, ahead)
    want, bound = R.product(x, w, x_fmt, max(1, 4_000_000 // (n * k)))
    if bias is not None:
        want = want + R.to_float(bias, BF16)
        bound = bound + 2.0 ** -23 * np.abs(want)
    R.assert_within(got, want, bound, dtype, f"{rows}x{n}x{k}")


@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows", [1, 16, 40, 200])
def test_product_keeps_nan_and_extremes_to_their_rows(gpu, x_fmt, rows):
    n, k = 70, 352
    rng = np.random.default_rng(rows)
    x, w = R.random_rows(rng, rows, k, x_fmt), R.random_rows(rng, n, k, R.E2M1)
    x[1][rows - 1, 3] = 255                       # a NaN block of zeros
    x[0][rows - 1, code_bytes(x_fmt, 96):code_bytes(x_fmt, 128)] = 0
    w[1][n - 1, 10] = 255                         # in the last block of a weight row
    w[1][5, :] = 0                                # 2^-127: all that is left is zeros
    w[1][6, :] = 254                              # 2^127: beyond fp32
    got = R.to_float(run_product(gpu, x, w, x_fmt, None, F16, rows, n, k), F16)
    nan = np.zeros((rows, n), bool)
    nan[rows - 1], nan[:, n - 1] = True, True
    # (row 6: addends of 2^127 and more, of both signs, leave fp32 before they meet: infinite, or an infinity less an infinity)
    others = np.arange(n) != 6
    assert np.array_equal(np.isnan(got[:, others]), nan[:, others]) and not np.any(np.isfinite(got[:, 6]))
    with np.errstate(invalid="ignore"):
        want, bound = R.product(x, w, x_fmt)
    assert np.all(got[:rows - 1, 5] == 0)
    fine = ~nan
    fine[:, 6] = False
    tol = bound[fine] + R.half_step(np.abs(want[fine]) + bound[fine], F16)
    assert np.all(np.abs(got[fine] - want[fine]) <= tol)


def test_product_of_e4m3_nan_codes(gpu):
    rng = np.random.default_rng(3)
    for rows in (2, 40):
        x, w = R.random_rows(rng, rows, 96, R.E4M3), R.random_rows(rng, 20, 96, R.E2M1)
        x[0][1, 95] = 0x7F
        got = R.to_float(run_product(gpu, x, w, R.E4M3, None, F16, rows, 20, 96), F16)
        assert np.array_equal(np.isnan(got).any(1), np.arange(rows) == 1)


def test_product_rows_do_not_depend_on_their_company(gpu):
    """Any row of a chunk alone, up to the chunk's own kernel: same bytes."""
    rng = np.random.default_rng(11)
    x, w = R.random_rows(rng, 150, 480, R.E4M3), R.random_rows(rng, 90, 480, R.E2M1)
    whole = run_product(gpu, x, w, R.E4M3, None, F16, 150, 90, 480)
    part = run_product(gpu, (x[0][70:], x[1][70:]), w, R.E4M3, None, F16, 80, 90, 480)
    assert np.array_equal(whole[70:], part)
    few = run_product(gpu, (x[0][:16], x[1][:16]), w, R.E4M3, None, F16, 16, 90, 480)
    one = run_product(gpu, (x[0][5:6], x[1][5:6]), w, R.E4M3, None, F16, 1, 90, 480)
    assert np.array_equal(few[5:6], one)


# ---------------------------------------------------------------- the experts

def make_pool(gpu, ex, cells=None, chunk_cells=None):
    cells = cells if cells is not None else list(range(ex.n))
    page_rounded = -(-ex.size // capi.POOL_PAGE) * capi.POOL_PAGE
    count = int(max(cells)) + 1
    pool = gpu.ExpertPool(count, ex.size, ex.n, 0 if chunk_cells is None else max(chunk_cells, -(-count // capi.POOL_MAX_CHUNKS)) * page_rounded)
    for e, c in enumerate(cells):
        pool.upload(int(c), ex.blobs[e])
    return pool


DECODE = [  # d, f, experts, top_k, tokens, activation, biases
    (64, 64, 4, 1, 1, capi.ACT_SILU, False), (128, 192, 8, 4, 3, capi.ACT_CLAMPED_SWIGLU, True), (512, 256, 16, 8, 2, capi.ACT_GELU_TANH, False),
    (320, 64, 8, 2, 16, capi.ACT_SILU, True), (64, 704, 5, 3, 2, capi.ACT_CLAMPED_SWIGLU, True), (960, 320, 6, 5, 1, capi.ACT_SILU, False),
    (2880, 128, 4, 4, 1, capi.ACT_CLAMPED_SWIGLU, True), (192, 2304, 3, 2, 1, capi.ACT_GELU_TANH, True)]


def run_decode(gpu, moe, ex, pool, slots, x, weights, residual, hidden, tokens, top_k, stream=None):
    d, f = ex.d, ex.f
    ws = gpu.empty(moe.mx_decode_workspace_bytes(tokens)).fill(0xEE)
    y = gpu.empty(2 * tokens * d + 64).fill(0x5A)
    dh = gpu.dev(hidden) if hidden is not None else None
    keep = [gpu.dev(slots), gpu.dev(x[0]), gpu.dev(x[1]), gpu.dev(weights), gpu.dev(residual) if residual is not None else None]
    moe.encode_mx_decode_ffn(pool, keep[0], ex.off, keep[1], keep[2], keep[3], keep[4], y, dh, ws, top_k, tokens)
    gpu.synchronize()
    raw = y.download(np.uint16)
    assert np.all(raw[tokens * d:] == 0x5A5A)
    acts = ws.download(np.uint8)
    at = -(-tokens * top_k * f // 256) * 256
    return (raw[:tokens * d].reshape(tokens, d), acts[:tokens * top_k * f].reshape(-1, f), acts[at:at + tokens * top_k * f // 32].reshape(-1, f // 32),
            dh.download(np.uint16, tokens * d).reshape(tokens, d) if dh else None)


@pytest.mark.parametrize("d,f,ne,k,tokens,act,biases", DECODE)
def test_decode_ffn(gpu, d, f, ne, k, tokens, act, biases):
    rng = np.random.default_rng(d + f + k)
    ex = R.Experts(rng, ne, d, f, biases)
    cells = list(rng.permutation(ne))
    pool = make_pool(gpu, ex, cells, chunk_cells=2)
    moe = gpu.MoE(d, f, ne, k, activation=act, additive_biases=biases)
    idx = np.array([rng.permutation(ne)[:k] for _ in range(tokens)])
    slots = np.array(cells)[idx].astype(np.uint32)
    if tokens * k > 2:
        slots[0, 0] = capi.SENTINEL
    if tokens > 2:
        slots[1, :] = capi.SENTINEL  # nothing of this token's is there
    x = R.random_rows(rng, tokens, d, R.E4M3)
    weights = rng.uniform(0.05, 1.0, (tokens, k)).astype(np.float16)
    residual = rng.standard_normal((tokens, d)).astype(np.float16) if d != 512 else None
    hidden = rng.standard_normal((tokens, d)).astype(np.float16) if d != 320 else None
    y, codes, scales, h = run_decode(gpu, moe, ex, pool, slots, x, weights, residual, hidden, tokens, k)
    for t in range(tokens):
        want = residual[t].astype(np.float64) if residual is not None else np.zeros(d)
        bound = np.zeros(d)
        parts = np.abs(want)
        for p in range(k):
            row = t * k + p
            if slots[t, p] == capi.SENTINEL:
                assert np.all(codes[row] == 0xEE)  # not computed
                continue
            e = idx[t, p]
            a, da = ex.act(e, (x[0][t:t + 1], x[1][t:t + 1]), act)
            R.assert_quantized(codes[row:row + 1], scales[row:row + 1], a, da, f"activations of token {t}, position {p}")
            o, do = ex.down(e, (codes[row:row + 1], scales[row:row + 1]))
            share = float(weights[t, p])
            want, bound, parts = want + share * o[0], bound + share * do[0], parts + share * np.abs(o[0])
        R.assert_within(y[t], want, bound + 16 * 2.0 ** -24 * parts, F16, f"token {t}")
        if h is not None:
            with np.errstate(over="ignore"):
                assert np.array_equal(h[t], (hidden[t].astype(np.float32) + y[t].view(np.float16).astype(np.float32)).astype(np.float16).view(np.uint16))
        if not np.any(slots[t] != capi.SENTINEL):
            assert np.array_equal(y[t], residual[t].view(np.uint16) if residual is not None else np.zeros(d, np.uint16))
        one = run_decode(gpu, moe, ex, pool, slots[t:t + 1], (x[0][t:t + 1], x[1][t:t + 1]), weights[t:t + 1],
                         residual[t:t + 1] if residual is not None else None, None, 1, k)
        assert np.array_equal(one[0][0], y[t]), "a token of a batch, alone"


GROUPED = [  # d, f, experts, top_k, tokens, activation, biases
    (64, 64, 4, 1, 1, capi.ACT_SILU, False), (128, 192, 8, 4, 37, capi.ACT_CLAMPED_SWIGLU, True), (320, 64, 3, 2, 100, capi.ACT_GELU_TANH, False),
    (192, 320, 2, 1, 300, capi.ACT_SILU, True), (64, 128, 32, 8, 40, capi.ACT_SILU, False), (576, 448, 4, 3, 90, capi.ACT_CLAMPED_SWIGLU, True)]


@pytest.mark.parametrize("d,f,ne,k,tokens,act,biases", GROUPED)
def test_grouped_ffn(gpu, d, f, ne, k, tokens, act, biases):
    rng = np.random.default_rng(d + f + k)
    ex = R.Experts(rng, ne, d, f, biases)
    cells = list(rng.permutation(ne))
    pool = make_pool(gpu, ex, cells, chunk_cells=3)
    absent = ne - 1 if ne > 2 else None
    for e in range(ne):
        if e != absent:
            pool.publish(e, int(cells[e]), capi.RESIDENT)
    moe = gpu.MoE(d, f, ne, k, activation=act, additive_biases=biases)
    pf = gpu.Prefill(moe)
    score = rng.gumbel(size=(tokens, ne)) - 0.8 * np.log1p(np.arange(ne))
    idx = np.argsort(-score, axis=1)[:, :k].astype(np.uint32)
    x = R.random_rows(rng, tokens, d, R.E4M3)
    weights = rng.uniform(0.1, 1, (tokens, k)).astype(np.float16)
    routes = gpu.GroupedRoutesDevice(tokens * k, ne)
    keep = [gpu.dev(idx), gpu.dev(weights), gpu.dev(x[0]), gpu.dev(x[1])]
    pf.group_pairs(keep[0], keep[1], tokens, k, ne, routes, residency=pool.table)
    ws = gpu.empty(pf.mx_ffn_workspace_bytes(routes.max_row_tiles)).fill(0xEE)
    partials = gpu.empty(2 * tokens * k * d + 64).fill(0x5A)
    pf.encode_mx_grouped_expert_gemms(pool, ex.off, routes, keep[2], keep[3], partials, ws, tokens, k)
    gpu.synchronize()
    raw = partials.download(np.uint16)
    assert np.all(raw[tokens * k * d:] == 0x5A5A)
    got = raw[:tokens * k * d].reshape(tokens * k, d)
    table = routes.download()
    rows = routes.max_row_tiles * 64
    acts = ws.download(np.uint8)
    codes, at = acts[:rows * f].reshape(rows, f), -(-rows * f // 256) * 256
    scales = acts[at:at + rows * f // 32].reshape(rows, f // 32)
    seen = np.zeros(tokens * k, bool)
    for number, (cell, start, count, expert) in enumerate(table["row_tiles"]):
        pairs = table["sorted_pairs"][start:start + count]
        out_row = pairs[:, 0] * k + pairs[:, 2]
        seen[out_row] = True
        if expert == absent:
            assert np.all(got[out_row] == 0x5A5A)  # left as they were
            continue
        a, da = ex.act(expert, (x[0][pairs[:, 0]], x[1][pairs[:, 0]]), act)
        here = slice(number * 64, number * 64 + int(count))
        R.assert_quantized(codes[here], scales[here], a, da, f"activations of tile {number}")
        o, do = ex.down(expert, (codes[here], scales[here]))
        R.assert_within(got[out_row], o, do, F16, f"tile {number}")
        assert np.all(codes[number * 64 + int(count):number * 64 + 64] == 0xEE)  # rows behind the tile's
    assert seen.all()
    # a larger bound of tiles, as for several chunks, gives the same bytes
    more = routes.max_row_tiles + 7
    ws2 = gpu.empty(pf.mx_ffn_workspace_bytes(more))
    partials.fill(0x5A)
    pf.encode_mx_grouped_expert_gemms(pool, ex.off, routes, keep[2], keep[3], partials, ws2, tokens, k, max_row_tiles=more)
    gpu.synchronize()
    assert np.array_equal(partials.download(np.uint16), raw)


def test_a_layer_of_them_on_a_stream_and_replayed(gpu):
    """Norm with 8-bit rows, the router over its fp16 rows, the grouping, the experts' FFN, the reduce and the residual add, as a runner
    encodes a chunk; and for its first tokens the decode form over the same rows and cells. On a stream of the caller's, then captured and
    replayed over other inputs with eager work between: every replay gives the eager call's bytes."""
    d, f, ne, k, tokens, few = 256, 192, 16, 4, 75, 3
    rng = np.random.default_rng(77)
    ex = R.Experts(rng, ne, d, f, True)
    cells = [int(c) for c in rng.permutation(ne)]
    pool = make_pool(gpu, ex, cells)
    for e in range(ne):
        pool.publish(e, cells[e], capi.RESIDENT)
    gpu.synchronize()
    moe = gpu.MoE(d, f, ne, k, activation=capi.ACT_CLAMPED_SWIGLU, additive_biases=True)
    stream = gpu.Stream()
    moe.stream = stream
    pf = gpu.Prefill(moe)
    ones = gpu.dev(S.f32_to_bf16_bits(np.ones(max(d, ne), np.float32)))
    zeros = gpu.dev(np.zeros(ne, np.uint16))
    router = gpu.dev((0.2 * rng.standard_normal((ne, d))).astype(np.float16))
    weight = gpu.dev(S.f32_to_bf16_bits(rng.uniform(0.5, 1.5, d).astype(np.float32)))
    hidden, delta = gpu.empty(2 * tokens * d), gpu.empty(2 * tokens * d)
    total, out, codes, scales = gpu.empty(2 * tokens * d), gpu.empty(2 * tokens * d), gpu.empty(tokens * d), gpu.empty(tokens * d // 32)
    idx, w, logits = gpu.empty(4 * tokens * k), gpu.empty(2 * tokens * k), gpu.empty(pf.router_workspace_bytes(tokens, ne, d))
    routes = gpu.GroupedRoutesDevice(tokens * k, ne)
    ws, partials, h2 = gpu.empty(pf.mx_ffn_workspace_bytes(routes.max_row_tiles)), gpu.empty(2 * tokens * k * d), gpu.empty(2 * tokens * d)
    slots, dws, y = gpu.empty(4 * few * k), gpu.empty(moe.mx_decode_workspace_bytes(few)), gpu.empty(2 * few * d)

    def layer():
        gpu.residual_add_rmsnorm_bf16w_mx8(hidden, delta, weight, total, out, codes, scales, d, 1e-6, tokens, stream)
        pf.encode_block(router, None, None, out, ones, ones, zeros, idx, w, logits, tokens, ne, d, k, d)
        pf.group_pairs(idx, w, tokens, k, ne, routes, residency=pool.table)
        pf.encode_mx_grouped_expert_gemms(pool, ex.off, routes, codes, scales, partials, ws, tokens, k)
        pf.encode_reduce_token_major(partials, w, h2, tokens, k, d)
        moe.encode_resolve_batch(idx, pool.table, slots, few * k, ne)
        moe.encode_mx_decode_ffn(pool, slots, ex.off, codes, scales, w, None, y, None, dws, k, few)
        pf.residual_add(total, h2, tokens * d)

    def inputs(seed):
        r = np.random.default_rng(seed)
        hidden.upload(r.standard_normal((tokens, d)).astype(np.float16))
        delta.upload(r.standard_normal((tokens, d)).astype(np.float16))

    def results():
        stream.synchronize()
        return [b.download(t, n) for b, t, n in ((total, np.uint16, tokens * d), (codes, np.uint8, tokens * d), (scales, np.uint8, tokens * d // 32),
                                                 (idx, np.uint32, tokens * k), (partials, np.uint16, tokens * k * d), (h2, np.uint16, tokens * d),
                                                 (y, np.uint16, few * d))]

    inputs(0)
    layer()
    eager = results()
    # the eager layer, against the reference, from the device's own rows and routes
    c, s = eager[1].reshape(tokens, d), eager[2].reshape(tokens, -1)
    want_codes, want_scales = R.quantize(R.to_float(out.download(np.uint16, tokens * d), F16).reshape(tokens, d), R.E4M3)
    assert np.array_equal(c, want_codes) and np.array_equal(s, want_scales)
    route, share = eager[3].reshape(tokens, k), R.to_float(w.download(np.uint16, tokens * k), F16).reshape(tokens, k)
    got = R.to_float(eager[4], F16).reshape(tokens, k, d)
    reduced, one_token = R.to_float(eager[5], F16).reshape(tokens, d), R.to_float(eager[6], F16).reshape(few, d)
    for t in (0, 1, 2, 40, tokens - 1):
        want, bound = np.zeros(d), np.zeros(d)
        for p in range(k):
            e = int(route[t, p])
            a, da = ex.act(e, (c[t:t + 1], s[t:t + 1]), capi.ACT_CLAMPED_SWIGLU)
            # activations within their bound of a border may take either code: an E4M3 step of 2^-3 at most, through the down rows
            q = R.quantize(a, R.E4M3)
            near = np.zeros(f)
            for sign in (-1, 1):
                other = R.quantize(a + sign * da, R.E4M3)
                near = np.maximum(near, np.abs(R.values(*other, R.E4M3) - R.values(*q, R.E4M3))[0])
            o, do = ex.down(e, q)
            do = do[0] + np.abs(R.values(*ex.parts[e]["down"], R.E2M1)) @ near
            tol = do + R.half_step(np.abs(o[0]) + do, F16)
            assert np.all(np.abs(got[t, p] - o[0]) <= tol)
            want, bound = want + share[t, p] * o[0], bound + share[t, p] * (do + R.half_step(np.abs(o[0]) + do, F16))
        tol = bound + R.half_step(np.abs(want) + bound, F16) + 2.0 ** -20 * np.abs(want)
        assert np.all(np.abs(reduced[t] - want) <= tol)
        if t < few:
            assert np.all(np.abs(one_token[t] - want) <= tol)

    graph = capture(gpu, stream, layer)
    other = gpu.empty(1 << 16)
    try:
        for replay in range(4):
            inputs(replay + 1)
            layer()
            eager = results()
            for b in (total, codes, scales, partials, h2, y):
                b.fill(0)
            other.fill(replay)
            gpu.synchronize()
            capi.check(capi.load().shrike_hip_graph_launch(graph, stream.handle), "graph_launch")
            for name, a, b in zip(("total", "codes", "scales", "routes", "partials", "reduced", "y"), eager, results()):
                assert np.array_equal(a, b), f"replay {replay}: {name}"
    finally:
        capi.load().shrike_hip_graph_destroy(graph)
