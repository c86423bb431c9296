"""The operators over microscaled blocks where addresses pass 32 bits, and experts laid out by a caller's own offsets: the far rows, the shifted
parts and the odd addresses give the bytes of a small call over the same numbers."""
import numpy as np
import pytest

from shrike_amd import capi
from shrike_amd import synth as S
from tests import mx_reference as R
from tests import test_mx_gpu as base
from tests.test_mx_experts_gpu import Chunk, by_counts

pytestmark = pytest.mark.gpu
F16 = capi.ELEM_F16


def quantized(gpu, bits, fmt, rows, d):
    return base.run_quantize(gpu, bits.reshape(rows, d), F16, d, fmt, rows, d)


@pytest.mark.parametrize("fmt", [R.E4M3, R.E2M1])
def test_quantize_and_back_past_4_gib(gpu, fmt):
    """fp16 rows of 9.8 GB, codes of 4.9 or 2.5: the first, a middle and the last rows differ from the filler."""
    rows, d, some = 600_000, 8192, 5
    rng = np.random.default_rng(1)
    n = base.code_bytes(fmt, d)
    src, codes, scales = gpu.empty(2 * rows * d).fill(0x3C), gpu.empty(rows * n).fill(0), gpu.empty(rows * d // 32).fill(0)
    marks = {at: S.f32_to_f16_bits(rng.standard_normal(some * d).astype(np.float32)) for at in (0, 300_000, rows - some)}
    for at, bits in marks.items():
        src.upload(bits, 2 * at * d)
    gpu.mx_quantize(src, F16, d, fmt, codes, scales, rows, d)
    gpu.synchronize()
    filler = quantized(gpu, np.full(d, 0x3C3C, np.uint16), fmt, 1, d)
    for at in (7, 524_287, 524_288, rows - some - 1):
        assert np.array_equal(codes.download(np.uint8, n, at * n), filler[0][0]) and np.array_equal(scales.download(np.uint8, d // 32, at * d // 32), filler[1][0])
    values = {}
    for at, bits in marks.items():
        c, s = quantized(gpu, bits, fmt, some, d)
        assert np.array_equal(codes.download(np.uint8, some * n, at * n), c.reshape(-1)), at
        assert np.array_equal(scales.download(np.uint8, some * d // 32, at * d // 32), s.reshape(-1)), at
        values[at] = R.values(c, s, fmt).astype(np.float16).view(np.uint16).reshape(-1)
    src.fill(0)
    gpu.mx_dequantize(codes, scales, fmt, src, F16, d, rows, d)
    gpu.synchronize()
    for at, want in values.items():
        assert np.array_equal(src.download(np.uint16, some * d, 2 * at * d), want), at


def test_rows_further_apart_than_4_gib(gpu):
    d, n, stride = 96, 40, (1 << 32) + 24
    rng = np.random.default_rng(2)
    bits = S.f32_to_f16_bits(rng.standard_normal(2 * d).astype(np.float32)).reshape(2, d)
    far = gpu.empty(2 * (stride + 512)).fill(0x5A)
    for r in range(2):
        far.upload(bits[r], 2 * r * stride)
    codes, scales = gpu.empty(2 * d), gpu.empty(2 * d // 32)
    gpu.mx_quantize(far, F16, stride, R.E4M3, codes, scales, 2, d)
    gpu.synchronize()
    c, s = R.quantize(R.to_float(bits, F16), R.E4M3)
    assert np.array_equal(codes.download(np.uint8, 2 * d).reshape(2, d), c) and np.array_equal(scales.download(np.uint8, 2 * d // 32).reshape(2, -1), s)
    far.fill(0x5A)
    gpu.mx_dequantize(codes, scales, R.E4M3, far, F16, stride, 2, d)
    w = R.random_rows(rng, n, d, R.E2M1)
    dw, ws = gpu.dev(w[0]), gpu.dev(w[1])
    gpu.mx_product(codes, scales, R.E4M3, dw, ws, None, far.ptr + 2 * 256, F16, stride, 2, n, d)
    gpu.synchronize()
    values = R.values(c, s, R.E4M3).astype(np.float16).view(np.uint16)
    want, bound = R.product((c, s), w, R.E4M3)
    for r in range(2):
        row = far.download(np.uint16, 512, 2 * r * stride)
        assert np.array_equal(row[:d], values[r]) and np.all(row[d:256] == 0x5A5A) and np.all(row[256 + n:] == 0x5A5A)
        R.assert_within(row[None, 256:256 + n], want[r:r + 1], bound[r:r + 1], F16)


@pytest.mark.parametrize("with_delta", [True, False])
def test_norm_past_4_gib(gpu, with_delta):
    rows, d, some = 1_200_000, 4096, 4
    rng = np.random.default_rng(3)
    hidden, weight = gpu.empty(2 * rows * d).fill(0x3C), gpu.dev(S.f32_to_bf16_bits(rng.uniform(0.5, 1.5, d).astype(np.float32)))
    delta = gpu.empty(2 * rows * d).fill(0x34) if with_delta else None
    codes, scales = gpu.empty(rows * d).fill(0), gpu.empty(rows * d // 32).fill(0)
    marks = {at: S.f32_to_f16_bits(rng.standard_normal(some * d).astype(np.float32)) for at in (0, 524_286, 1_048_574, rows - some)}
    for at, bits in marks.items():
        hidden.upload(bits, 2 * at * d)
    gpu.residual_add_rmsnorm_bf16w_mx8(hidden, delta, weight, hidden if with_delta else None, None, codes, scales, d, 1e-6, rows)
    gpu.synchronize()
    for at, bits in marks.items():
        h, dl = gpu.dev(bits), gpu.empty(2 * some * d).fill(0x34) if with_delta else None
        out, c, s = gpu.empty(2 * some * d), gpu.empty(some * d), gpu.empty(some * d // 32)
        gpu.residual_add_rmsnorm_bf16w_mx8(h, dl, weight, h if with_delta else None, out, c, s, d, 1e-6, some)
        gpu.synchronize()
        assert np.array_equal(codes.download(np.uint8, some * d, at * d), c.download(np.uint8, some * d)), at
        assert np.array_equal(scales.download(np.uint8, some * d // 32, at * d // 32), s.download(np.uint8, some * d // 32)), at
        assert np.array_equal(hidden.download(np.uint16, some * d, 2 * at * d), h.download(np.uint16, some * d)), at


def test_activations_past_4_gib(gpu):
    """A chunk of 1,050,000 tokens of 61 kinds over two experts: its activations are 4.4 GB, and every row is that of its kind in a small chunk."""
    d, f, ne, tokens, kinds = 64, 4224, 2, 1_050_000, 122
    rng = np.random.default_rng(4)
    ex = R.Experts(rng, ne, d, f, True)
    x = R.random_rows(rng, 61, d, R.E4M3)
    kind = np.arange(kinds)
    small = Chunk(gpu, ex, capi.ACT_SILU, (x[0][kind % 61], x[1][kind % 61]), kind % 2)
    want = small.run(kind)[0]
    of = rng.integers(0, kinds, tokens)
    idx, share, codes, scales = gpu.dev((of % 2).astype(np.uint32)), gpu.dev(np.ones(tokens, np.float16)), gpu.dev(x[0][of % 61]), gpu.dev(x[1][of % 61])
    routes = gpu.GroupedRoutesDevice(tokens, ne)
    ws, out = gpu.empty(small.pf.mx_ffn_workspace_bytes(routes.max_row_tiles)), gpu.empty(2 * tokens * d).fill(0x5A)
    gpu.synchronize()
    small.pf.group_pairs(idx, share, tokens, 1, ne, routes, residency=small.pool.table)
    small.pf.encode_mx_grouped_expert_gemms(small.pool, ex.off, routes, codes, scales, out, ws, tokens, 1)
    gpu.synchronize()
    assert ws.nbytes > 1 << 32 and np.array_equal(out.download(np.uint16, tokens * d).reshape(tokens, d), want[of])


def moved(ex, rng):
    """The same experts with their parts elsewhere in a larger blob: codes at odd multiples of 16, scales at odd addresses, biases at even ones."""
    other = R.Experts.__new__(R.Experts)
    other.__dict__.update(ex.__dict__)
    other.off, at = capi.ExpertOffsets(), 16
    parts = [n + s for n in ("down", "up", "gate") for s in ("_s_off", "_ab_off", "_w_off")]
    sizes = {n + s: size for n, rows, k in (("gate", ex.f, ex.d), ("up", ex.f, ex.d), ("down", ex.d, ex.f))
             for s, size in (("_w_off", rows * k // 2), ("_s_off", rows * k // 32), ("_ab_off", 2 * rows))}
    blobs = [rng.integers(0, 256, ex.size + 4096).astype(np.uint8) for _ in range(ex.n)]
    for part in parts:
        if part.endswith("_ab_off") and not ex.biases:
            continue
        at = at // 32 * 32 + {"_w_off": 48, "_s_off": 33, "_ab_off": 34}[part[part.index("_"):]]
        setattr(other.off, part, at)
        for blob, old in zip(blobs, ex.blobs):
            blob[at:at + sizes[part]] = old[getattr(ex.off, part):getattr(ex.off, part) + sizes[part]]
        at += sizes[part]
    other.blobs, other.size = blobs, ex.size + 4096
    assert at <= other.size
    return other


@pytest.mark.parametrize("biases", [False, True])
@pytest.mark.parametrize("d,f,counts", [(576, 192, (13, 30, 60)), (320, 192, (20, 5, 64)), (576, 1024, (60, 110, 230)), (320, 1024, (256, 64, 80))])
def test_a_chunk_s_experts_laid_out_otherwise(gpu, d, f, counts, biases):
    rng = np.random.default_rng(d + f)
    ex = R.Experts(rng, len(counts), d, f, biases)
    expert = by_counts(rng, counts)
    x = R.random_rows(rng, len(expert), d, R.E4M3)
    every = np.arange(len(expert))
    chunks = [Chunk(gpu, e, capi.ACT_CLAMPED_SWIGLU, x, expert) for e in (ex, moved(ex, rng))]
    assert chunks[0].many(len(every)) == (f == 1024)
    for a, b in zip(*(c.run(every) for c in chunks)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("biases", [False, True])
@pytest.mark.parametrize("d,f,tokens", [(576, 192, 7), (576, 192, 64), (320, 2112, 3)])
def test_single_tokens_experts_laid_out_otherwise(gpu, d, f, tokens, biases):
    rng = np.random.default_rng(d + f + tokens)
    ex, k = R.Experts(rng, 3, d, f, biases), 2
    x = R.random_rows(rng, tokens, d, R.E4M3)
    slots = rng.integers(0, 3, (tokens, k)).astype(np.uint32)
    weights, residual = rng.uniform(0.5, 1, (tokens, k)).astype(np.float16), rng.standard_normal((tokens, d)).astype(np.float16)
    moe = gpu.MoE(d, f, 3, k, activation=capi.ACT_SILU, additive_biases=biases)
    y, codes, scales = [], [], []
    for e in (ex, moved(ex, rng)):
        got = base.run_decode(gpu, moe, e, base.make_pool(gpu, e), slots, x, weights, residual, None, tokens, k)
        y.append(got[0]), codes.append(got[1]), scales.append(got[2])
    for pair in (y, codes, scales):
        assert np.array_equal(*pair)


@pytest.mark.parametrize("f,tokens", [(192, 103), (1024, 400)])
def test_rows_whose_scales_lie_at_odd_addresses(gpu, f, tokens):
    """A chunk's and single tokens' x scales start anywhere."""
    d, ne, few = 576, 3, 5
    rng = np.random.default_rng(f)
    ex = R.Experts(rng, ne, d, f, True)
    x = R.random_rows(rng, tokens, d, R.E4M3)
    chunk = Chunk(gpu, ex, capi.ACT_SILU, x, rng.integers(0, ne, tokens))
    want = chunk.run(np.arange(tokens))[0]
    assert chunk.many(tokens) == (f == 1024)
    routes = gpu.GroupedRoutesDevice(tokens, ne)
    keep = [gpu.dev(chunk.expert), gpu.dev(np.ones(tokens, np.float16)), gpu.dev(x[0])]
    ws, out = gpu.empty(chunk.pf.mx_ffn_workspace_bytes(routes.max_row_tiles)), gpu.empty(2 * tokens * d)
    slots, share, dws, y = gpu.dev(chunk.expert[:few]), gpu.dev(np.ones(few, np.float16)), gpu.empty(chunk.moe.mx_decode_workspace_bytes(few)), gpu.empty(2 * few * d)
    tokens_alone = None
    for ahead in (0, 1, 2, 7, 13):
        scales = gpu.dev(np.r_[np.full(ahead, 255, np.uint8), x[1].reshape(-1)])
        gpu.synchronize()
        chunk.pf.group_pairs(keep[0], keep[1], tokens, 1, ne, routes, residency=chunk.pool.table)
        chunk.pf.encode_mx_grouped_expert_gemms(chunk.pool, ex.off, routes, keep[2], scales.ptr + ahead, out, ws, tokens, 1)
        chunk.moe.encode_mx_decode_ffn(chunk.pool, slots, ex.off, keep[2], scales.ptr + ahead, share, None, y, None, dws, 1, few)
        gpu.synchronize()
        assert np.array_equal(out.download(np.uint16, tokens * d).reshape(tokens, d), want), ahead
        got = y.download(np.uint16, few * d)
        tokens_alone = got if tokens_alone is None else tokens_alone
        assert np.array_equal(got, tokens_alone), ahead
