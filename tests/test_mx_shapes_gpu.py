"""The operators over microscaled blocks where their kernels change over: numbers of rows and workgroups, lengths of k, experts of many
rows, pairs that share a cell, tables that are torn, weights and rows past 4 GiB, calls at once and captured ones. The products here
are of numbers whose sums are exact in fp32, so that an output is the 64-bit sum rounded once, bit for bit."""
import numpy as np
import pytest

from shrike_amd import capi
from tests import mx_reference as R
from tests import test_mx_gpu as base
from tests.test_graph_replay_gpu import capture

pytestmark = pytest.mark.gpu
F16, BF16 = capi.ELEM_F16, capi.ELEM_BF16


def exact_rows(rng, rows, k, fmt):
    """Codes of 0, +-1, +-2 (E4M3) or 0, +-1/2, +-1, +-2 (E2M1) in blocks scaled by 1 or 2: products are multiples of 1/4 up to 16, none less
    than 2^-6 of another, so neither the matrix instruction's groups nor 2^16 of them in fp32 lose a bit."""
    values = np.array([0x00, 0x38, 0x40, 0xB8, 0xC0] if fmt == R.E4M3 else [0, 1, 2, 4, 9, 10, 12], np.uint8)
    codes = values[rng.integers(0, len(values), (rows, k))]
    return R.pack(codes, fmt), rng.integers(127, 129, (rows, k // 32)).astype(np.uint8)


def rounded(v, dtype):
    if dtype == F16:
        return v.astype(np.float16).view(np.uint16)
    u = v.astype(np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def check_exact(gpu, x_fmt, rows, n, k, pad=0, ahead=0, bias=True):
    rng = np.random.default_rng(rows * 7 + n * 3 + k + x_fmt)
    x, w = exact_rows(rng, rows, k, x_fmt), exact_rows(rng, n, k, R.E2M1)
    b = rng.integers(-64, 65, n).astype(np.float32)
    want = R.values(*x, x_fmt) @ R.values(*w, R.E2M1).T
    assert np.array_equal(want, want.astype(np.float32)) and np.abs(want).max() < 65000
    dtype = F16 if (rows + n) % 2 else BF16
    got = base.run_product(gpu, x, w, x_fmt, (b.view(np.uint32) >> 16).astype(np.uint16) if bias else None, dtype, rows, n, k, pad, ahead)
    want = rounded(want + b if bias else want, dtype)
    bad = np.argwhere((got != want) & ~((got & 0x7FFF) + (want & 0x7FFF) == 0))  # (a zero's sign is not the sum's)
    assert len(bad) == 0, f"{len(bad)} outputs differ, the first at {bad[0]}"


# 16, 64 and 65 rows with few outputs: k over the waves; then tiles of 64 x 256, 128 x 256 and 256 x 256 outputs, whole and ragged
@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows,n,k,pad,ahead", [
    (16, 640, 1056, 0, 0), (17, 640, 1056, 0, 0), (64, 641, 96, 0, 1), (65, 700, 2080, 4, 0), (128, 3000, 160, 0, 0), (192, 2000, 224, 1, 0),
    (65, 6200, 160, 0, 0), (70, 6145, 32, 8, 8), (200, 8200, 288, 0, 0), (511, 8191, 96, 1, 3),
    (520, 8200, 160, 0, 0), (900, 8000, 64, 0, 0),
    (1100, 8200, 160, 0, 0), (1281, 7969, 96, 7, 0)])
def test_product_by_rows(gpu, x_fmt, rows, n, k, pad, ahead):
    check_exact(gpu, x_fmt, rows, n, k, pad, ahead)


# every remainder of k: of a step (4 blocks), of the steps whose scales are fetched together (16 blocks, fewer than 16), of a unit
@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows,n", [(9, 50), (70, 6200), (520, 8200), (1100, 8200)])
def test_product_by_k(gpu, x_fmt, rows, n):
    for k in [32 * b for b in (1, 2, 3, 4, 5, 7, 8, 9, 12, 13, 15, 16, 17, 20, 24, 29, 31, 32, 33, 37)]:
        print(f"{rows} x {n} x {k}", flush=True)
        check_exact(gpu, x_fmt, rows, n, k, bias=False)


@pytest.mark.parametrize("x_fmt", [R.E4M3, R.E2M1])
@pytest.mark.parametrize("rows,n,k", [(1, 70, 65536), (16, 33, 65504), (40, 20, 65536), (70, 6200, 4128), (520, 8200, 4192), (1100, 8200, 4224), (100, 8300, 8352)])
def test_product_of_long_rows(gpu, x_fmt, rows, n, k):
    check_exact(gpu, x_fmt, rows, n, k)


def test_a_tile_s_rows_do_not_depend_on_its_height(gpu):
    rng = np.random.default_rng(5)
    x, w = R.random_rows(rng, 1100, 224, R.E4M3), R.random_rows(rng, 8200, 224, R.E2M1)
    whole = base.run_product(gpu, x, w, R.E4M3, None, F16, 1100, 8200, 224)
    for rows in (520, 130):
        assert np.array_equal(base.run_product(gpu, (x[0][-rows:], x[1][-rows:]), w, R.E4M3, None, F16, rows, 8200, 224), whole[-rows:])


@pytest.mark.parametrize("rows", [1, 17, 70])
def test_product_of_weights_past_4_gib(gpu, rows):
    """Weights of 1 but for the last 300 rows', which are of 2: 4.9 GB of codes."""
    n, k, marked = 1_200_000, 8192, 300
    w, ws = gpu.empty(n * k // 2).fill(0x22), gpu.empty(n * k // 32).fill(127)
    w.upload(np.full(marked * k // 2, 0x44, np.uint8), (n - marked) * k // 2)
    x, xs = gpu.empty(rows * k).fill(0x38), gpu.empty(rows * k // 32).fill(127)
    out = gpu.empty(2 * rows * n).fill(0)
    gpu.mx_product(x, xs, R.E4M3, w, ws, None, out, F16, n, rows, n, k)
    gpu.synchronize()
    got = out.download(np.float16).reshape(rows, n)
    assert np.all(got[:, :n - marked] == k) and np.all(got[:, n - marked:] == 2 * k)


def test_product_of_rows_past_4_gib(gpu):
    rows, n, k, marked = 600_000, 16, 8192, 300
    x, xs = gpu.empty(rows * k).fill(0x38), gpu.empty(rows * k // 32).fill(127)
    x.upload(np.full(marked * k, 0x40, np.uint8), (rows - marked) * k)
    w, ws = gpu.empty(n * k // 2).fill(0x22), gpu.empty(n * k // 32).fill(127)
    out = gpu.empty(2 * rows * n).fill(0)
    gpu.mx_product(x, xs, R.E4M3, w, ws, None, out, F16, n, rows, n, k)
    gpu.synchronize()
    got = out.download(np.float16).reshape(rows, n)
    assert np.all(got[:rows - marked] == k) and np.all(got[rows - marked:] == 2 * k)


# experts of so many rows that they are taken in runs of up to 256: one expert, uneven ones, an absent one
@pytest.mark.parametrize("d,f,ne,k,tokens,act,biases", [
    (64, 512, 1, 1, 700, capi.ACT_SILU, True), (128, 1024, 2, 1, 300, capi.ACT_CLAMPED_SWIGLU, True), (192, 2048, 3, 1, 210, capi.ACT_GELU_TANH, False),
    (320, 576, 1, 1, 257, capi.ACT_CLAMPED_SWIGLU, True)])
def test_experts_of_many_rows(gpu, d, f, ne, k, tokens, act, biases):
    assert tokens * k * f >= ne << 17
    base.test_grouped_ffn(gpu, d, f, ne, k, tokens, act, biases)


# and of few, 64 of a tile among them
@pytest.mark.parametrize("d,f,ne,k,tokens,act,biases", [
    (192, 448, 3, 1, 190, capi.ACT_CLAMPED_SWIGLU, True), (1088, 64, 5, 2, 64, capi.ACT_SILU, False), (96 * 4, 832, 2, 2, 33, capi.ACT_GELU_TANH, True),
    (64, 64, 3, 3, 16, capi.ACT_SILU, False)])
def test_experts_of_few_rows(gpu, d, f, ne, k, tokens, act, biases):
    assert tokens * k * f < ne << 17
    base.test_grouped_ffn(gpu, d, f, ne, k, tokens, act, biases)


def grouped_call(gpu, d, f, ne, k, tokens, seed, activation=capi.ACT_SILU, stream=None):
    """Buffers of a call over every expert, present, and the call."""
    rng = np.random.default_rng(seed)
    ex = R.Experts(rng, ne, d, f, True)
    pool = base.make_pool(gpu, ex)
    for e in range(ne):
        pool.publish(e, e, capi.RESIDENT)
    moe = gpu.MoE(d, f, ne, k, activation=activation, additive_biases=True)
    moe.stream = stream
    pf = gpu.Prefill(moe)
    score = rng.gumbel(size=(tokens, ne)) - 0.8 * np.log1p(np.arange(ne))
    idx = gpu.dev(np.argsort(-score, axis=1)[:, :k].astype(np.uint32))
    weights = gpu.dev(rng.uniform(0.1, 1, (tokens, k)).astype(np.float16))
    x = R.random_rows(rng, tokens, d, R.E4M3)
    rows = [gpu.dev(x[0]), gpu.dev(x[1])]
    routes = gpu.GroupedRoutesDevice(tokens * k, ne)
    gpu.synchronize()
    pf.group_pairs(idx, weights, tokens, k, ne, routes, residency=pool.table)
    ws = gpu.empty(pf.mx_ffn_workspace_bytes(routes.max_row_tiles))
    partials = gpu.empty(2 * tokens * k * d).fill(0x5A)
    gpu.synchronize()
    call = lambda: pf.encode_mx_grouped_expert_gemms(pool, ex.off, routes, rows[0], rows[1], partials, ws, tokens, k)  # noqa: E731
    return call, routes, partials, rows, (pool, moe, pf, idx, weights, ws)


@pytest.mark.parametrize("d,f,ne,k,tokens", [(64, 512, 2, 1, 900), (64, 64, 2, 1, 900)])
def test_a_table_with_records_left_out(gpu, d, f, ne, k, tokens):
    """Runs that break off, start late, lie the other way about or are not a run at all: a pair of a record that is there has the whole table's
    row, every other is left as it was."""
    call, routes, partials, _, keep = grouped_call(gpu, d, f, ne, k, tokens, 9)
    call()
    gpu.synchronize()
    whole = partials.download(np.uint16).reshape(tokens * k, d)
    table = routes.download()
    tiles, pairs = table["row_tiles"], table["sorted_pairs"]
    count = len(tiles)
    for there in (list(range(1, count)), [i for i in range(count) if i % 5 != 2], list(range(count))[::-1], list(range(0, count, 2)), [count - 1], [], [3, 4, 5, 6, 7, 0, 1]):
        partials.fill(0x5A)
        raw = np.zeros((routes.max_row_tiles, 4), np.uint32)
        raw[:len(there)] = tiles[there]
        routes.row_tiles.upload(raw.reshape(-1))
        routes.row_tile_count.upload(np.array([len(there)], np.uint32))
        gpu.synchronize()
        call()
        gpu.synchronize()
        want = np.full_like(whole, 0x5A5A)
        for i in there:
            p = pairs[tiles[i][1]:tiles[i][1] + tiles[i][2]]
            want[p[:, 0] * k + p[:, 2]] = whole[p[:, 0] * k + p[:, 2]]
        assert np.array_equal(partials.download(np.uint16).reshape(tokens * k, d), want), there


# one token of a long activation row, the longest rows there are, and of two tokens
@pytest.mark.parametrize("d,f,ne,k,tokens,act,biases", [
    (64, 8192, 3, 2, 1, capi.ACT_SILU, True), (4096, 64, 2, 2, 1, capi.ACT_CLAMPED_SWIGLU, True), (4096, 64, 2, 2, 2, capi.ACT_CLAMPED_SWIGLU, True),
    (192, 4224, 2, 2, 3, capi.ACT_GELU_TANH, False)])
def test_decode_by_workgroups(gpu, d, f, ne, k, tokens, act, biases):
    check_decode(gpu, d, f, ne, k, tokens, act, biases, lambda rng: rng.integers(0, ne, (tokens, k)))


# more than 16 and more than 64 pairs at one cell, the same cell twice in a token, positions that are not there between them
@pytest.mark.parametrize("d,f,ne,k,tokens", [(64, 64, 1, 1, 40), (64, 128, 2, 2, 64), (128, 192, 3, 4, 64), (128, 64, 2, 8, 9)])
def test_decode_of_tokens_that_share_cells(gpu, d, f, ne, k, tokens):
    check_decode(gpu, d, f, ne, k, tokens, capi.ACT_CLAMPED_SWIGLU, True, lambda rng: np.where(rng.random((tokens, k)) < 0.1, -1, rng.integers(0, ne, (tokens, k))))


def check_decode(gpu, d, f, ne, k, tokens, act, biases, choose):
    rng = np.random.default_rng(d + f + k + tokens)
    ex = R.Experts(rng, ne, d, f, biases)
    pool = base.make_pool(gpu, ex)
    moe = gpu.MoE(d, f, max(ne, k), k, activation=act, additive_biases=biases)
    idx = choose(rng)
    slots = np.where(idx < 0, capi.SENTINEL, idx).astype(np.uint32)
    x = R.random_rows(rng, tokens, d, R.E4M3)
    weights = rng.uniform(0.05, 1.0, (tokens, k)).astype(np.float16)
    residual = rng.standard_normal((tokens, d)).astype(np.float16)
    y, codes, scales, _ = base.run_decode(gpu, moe, ex, pool, slots, x, weights, residual, None, tokens, k)
    acts = [ex.act(e, x, act) for e in range(ne)]
    for t in range(tokens):
        want, bound = residual[t].astype(np.float64), np.zeros(d)
        parts = np.abs(want)
        for p in range(k):
            e, row = idx[t, p], t * k + p
            if e < 0:
                assert np.all(codes[row] == 0xEE)
                continue
            R.assert_quantized(codes[row:row + 1], scales[row:row + 1], acts[e][0][t:t + 1], acts[e][1][t:t + 1], f"activations of token {t}, position {p}")
            o, do = ex.down(e, (codes[row:row + 1], scales[row:row + 1]))
            share = float(weights[t, p])
            want, bound, parts = want + share * o[0], bound + share * do[0], parts + share * np.abs(o[0])
        # (a position's weighted sum is rounded as often as there are waves with a part of it, 16 at most, and their sum as often again)
        R.assert_within(y[t], want, bound + 32 * 2.0 ** -24 * parts, F16, f"token {t}")


@pytest.mark.parametrize("d,f,ne,k,tokens", [(64, 512, 1, 1, 600), (128, 192, 4, 2, 100)])
def test_two_chunks_at_once_and_replayed(gpu, d, f, ne, k, tokens):
    """Two captured calls with workspaces of their own, replayed over and over on two streams at the same time, other rows between: every replay
    gives an eager call's bytes."""
    streams = [gpu.Stream(), gpu.Stream()]
    calls = [grouped_call(gpu, d, f, ne, k, tokens, 20 + i, capi.ACT_CLAMPED_SWIGLU, streams[i]) for i in range(2)]
    gpu.synchronize()
    graphs = [capture(gpu, streams[i], calls[i][0]) for i in range(2)]
    try:
        for replay in range(4):
            eager = []
            for call, _, partials, rows, _ in calls:
                x = R.random_rows(np.random.default_rng(100 * replay + len(eager)), tokens, d, R.E4M3)
                rows[0].upload(x[0]), rows[1].upload(x[1])
                gpu.synchronize()
                call()
                for s in streams:
                    s.synchronize()
                eager.append(partials.download(np.uint16))
                partials.fill(0)
            gpu.synchronize()
            for _ in range(3):
                for i in range(2):
                    capi.check(capi.load().shrike_hip_graph_launch(graphs[i], streams[i].handle), "graph_launch")
            for s in streams:
                s.synchronize()
            for i in range(2):
                assert np.array_equal(calls[i][2].download(np.uint16), eager[i]), f"replay {replay}, call {i}"
    finally:
        for g in graphs:
            capi.load().shrike_hip_graph_destroy(g)


def test_products_captured_on_a_stream(gpu):
    """One of each kernel, in one graph, replayed over other rows."""
    rng = np.random.default_rng(31)
    stream = gpu.Stream()
    calls = []
    for x_fmt, rows, n, k in ((R.E4M3, 1, 100, 288), (R.E2M1, 50, 100, 288), (R.E4M3, 70, 6200, 96), (R.E2M1, 520, 8200, 96), (R.E4M3, 1100, 8200, 96)):
        w = exact_rows(rng, n, k, R.E2M1)
        calls.append((x_fmt, rows, n, k, w, gpu.dev(w[0]), gpu.dev(w[1]), gpu.empty(rows * base.code_bytes(x_fmt, k)), gpu.empty(rows * k // 32),
                      gpu.empty(2 * rows * n)))
    gpu.synchronize()

    def body():
        for x_fmt, rows, n, k, _, dw, dws, dx, dxs, out in calls:
            gpu.mx_product(dx, dxs, x_fmt, dw, dws, None, out, F16, n, rows, n, k, stream)
    graph = capture(gpu, stream, body)
    try:
        for replay in range(3):
            want = []
            for x_fmt, rows, n, k, w, _, _, dx, dxs, out in calls:
                x = exact_rows(rng, rows, k, x_fmt)
                dx.upload(x[0]), dxs.upload(x[1])
                out.fill(0x5A)
                want.append((R.values(*x, x_fmt) @ R.values(*w, R.E2M1).T).astype(np.float16))
            gpu.synchronize()
            capi.check(capi.load().shrike_hip_graph_launch(graph, stream.handle), "graph_launch")
            stream.synchronize()
            for c, v in zip(calls, want):
                assert np.array_equal(c[-1].download(np.float16).reshape(v.shape), v), f"replay {replay}: {c[:4]}"
    finally:
        capi.load().shrike_hip_graph_destroy(graph)
