"""Calls of the experts' FFN over microscaled blocks as programs make them at the same time and again: single tokens on two streams, captured and
replayed, and a token that names one expert twice."""
import numpy as np
import pytest

from shrike_amd import capi
from tests import mx_reference as R
from tests import test_mx_gpu as base
from tests.test_graph_replay_gpu import capture

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,f,tokens", [(576, 192, 3), (576, 192, 64), (320, 832, 20)])
def test_single_tokens_on_two_streams_and_replayed(gpu, d, f, tokens):
    """Two captured calls over one pool with workspaces of their own, replayed on two streams at the same time, other rows and routes between: every
    replay gives an eager call's bytes, twice over."""
    rng = np.random.default_rng(d + f + tokens)
    ne, k = 6, 4
    ex = R.Experts(rng, ne, d, f, True)
    pool = base.make_pool(gpu, ex)
    streams, calls = [gpu.Stream(), gpu.Stream()], []
    for s in streams:
        moe = gpu.MoE(d, f, ne, k, activation=capi.ACT_CLAMPED_SWIGLU, additive_biases=True)
        moe.stream = s
        b = dict(moe=moe, slots=gpu.empty(4 * tokens * k), codes=gpu.empty(tokens * d), scales=gpu.empty(tokens * d // 32), w=gpu.empty(2 * tokens * k),
                 residual=gpu.empty(2 * tokens * d), y=gpu.empty(2 * tokens * d), hidden=gpu.empty(2 * tokens * d),
                 ws=gpu.empty(moe.mx_decode_workspace_bytes(tokens)))
        calls.append((b, lambda b=b: b["moe"].encode_mx_decode_ffn(pool, b["slots"], ex.off, b["codes"], b["scales"], b["w"], b["residual"], b["y"], b["hidden"],
                                                                   b["ws"], k, tokens)))

    def load(b, seed):
        r = np.random.default_rng(seed)
        x = R.random_rows(r, tokens, d, R.E4M3)
        b["codes"].upload(x[0]), b["scales"].upload(x[1])
        b["slots"].upload(np.where(r.random((tokens, k)) < 0.1, capi.SENTINEL, r.integers(0, ne, (tokens, k))).astype(np.uint32))
        b["w"].upload(r.uniform(0.1, 1, (tokens, k)).astype(np.float16))
        b["residual"].upload(r.standard_normal((tokens, d)).astype(np.float16))
        b["hidden"].upload(np.zeros((tokens, d), np.float16))
        gpu.synchronize()

    for i, (b, _) in enumerate(calls):
        load(b, i)
    graphs = [capture(gpu, streams[i], calls[i][1]) for i in range(2)]
    try:
        for replay in range(4):
            want = []
            for i, (b, call) in enumerate(calls):
                load(b, 10 * replay + i)
                call()
                streams[i].synchronize()
                want.append(b["y"].download(np.uint16))
                b["y"].fill(0x5A)
                b["hidden"].upload(np.zeros((tokens, d), np.float16))
            gpu.synchronize()
            for _ in range(3):
                for i in range(2):
                    capi.check(capi.load().shrike_hip_graph_launch(graphs[i], streams[i].handle), "graph_launch")
            for i in range(2):
                streams[i].synchronize()
                b = calls[i][0]
                assert np.array_equal(b["y"].download(np.uint16), want[i]), f"replay {replay}, call {i}"
                total = np.zeros(tokens * d, np.float16)  # hidden took y three times
                for _ in range(3):
                    total = (total.astype(np.float32) + want[i][:tokens * d].view(np.float16).astype(np.float32)).astype(np.float16)
                assert np.array_equal(b["hidden"].download(np.float16, tokens * d), total), f"replay {replay}, call {i}: hidden"
    finally:
        for g in graphs:
            capi.load().shrike_hip_graph_destroy(g)


@pytest.mark.parametrize("f,tokens", [(192, 40), (1024, 150)])
def test_a_token_that_names_an_expert_twice(gpu, f, tokens):
    """Each position gets the expert's row, the same bytes in both."""
    d, ne, k = 320, 2, 3
    rng = np.random.default_rng(f)
    ex = R.Experts(rng, ne, d, f)
    pool = base.make_pool(gpu, ex)
    for e in range(ne):
        pool.publish(e, e, capi.RESIDENT)
    moe = gpu.MoE(d, f, 3, k, activation=capi.ACT_SILU)
    pf = gpu.Prefill(moe)
    idx = rng.integers(0, ne, (tokens, k)).astype(np.uint32)
    x = R.random_rows(rng, tokens, d, R.E4M3)
    routes = gpu.GroupedRoutesDevice(tokens * k, 3)
    keep = [gpu.dev(idx), gpu.dev(np.ones((tokens, k), np.float16)), gpu.dev(x[0]), gpu.dev(x[1]), gpu.dev(np.array([2 << 32, 2 << 32 | 1, 0], np.uint64))]
    ws, out = gpu.empty(pf.mx_ffn_workspace_bytes(routes.max_row_tiles)), gpu.empty(2 * tokens * k * d).fill(0x5A)
    gpu.synchronize()
    pf.group_pairs(keep[0], keep[1], tokens, k, 3, routes, residency=keep[4])
    pf.encode_mx_grouped_expert_gemms(pool, ex.off, routes, keep[2], keep[3], out, ws, tokens, k)
    gpu.synchronize()
    got = out.download(np.uint16, tokens * k * d).reshape(tokens, k, d)
    assert (tokens * k * f >= 3 << 17) == (f == 1024)
    rows = {}
    for t in range(tokens):
        for p in range(k):
            assert np.array_equal(got[t, p], rows.setdefault((t, int(idx[t, p])), got[t, p])), (t, p)
    some = rng.permutation(tokens)[:6]
    for e in range(ne):
        a, da = ex.act(e, (x[0][some], x[1][some]), capi.ACT_SILU)
        codes, scales = R.quantize(a, R.E4M3)
        o, do = ex.down(e, (codes, scales))
        near = np.maximum(*(np.abs(R.values(*R.quantize(a + sign * da, R.E4M3), R.E4M3) - R.values(codes, scales, R.E4M3)) for sign in (-1, 1)))
        do = do + near @ np.abs(R.values(*ex.parts[e]["down"], R.E2M1)).T  # (activations so close to a border may take either code)
        for i, t in enumerate(some):
            if (t, e) in rows:
                R.assert_within(rows[t, e][None], o[i:i + 1], do[i:i + 1], capi.ELEM_F16)
