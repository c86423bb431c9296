"""A layer routed from logits, as a host puts it together: norm, the router's 4-bit projection into fp32 logits, the routes, then the routed experts
(grouped for a chunk, resolved cells for single tokens) and a 4-bit projection of their output. Eager, and captured and replayed over other rows."""
import numpy as np
import pytest

from oracle import oracle as O
from shrike_amd import capi, synth as S
from tests import affine4_reference as a4, route_reference as routing
from tests.helpers import Layer, assert_rel_close
from tests.test_decode_gpu import DeviceLayer
from tests.test_prefill_gpu import WorkspaceActs, check_pair_stagewise

pytestmark = pytest.mark.gpu
F32, F16, BF16 = capi.ELEM_F32, capi.ELEM_F16, capi.ELEM_BF16


class Chain:
    """The chain's buffers and calls for up to `t` rows on one stream."""

    def __init__(self, gpu, t, d, f, ne, k, desc, group, head):
        self.gpu, self.t, self.d, self.f, self.ne, self.k, self.desc = gpu, t, d, f, ne, k, desc
        r = np.random.default_rng(d + ne)
        self.L = Layer(0x5EED0061, d, f, ne, k, bits=4)
        self.dl = DeviceLayer(gpu, self.L)
        self.stream = self.dl.moe.stream = gpu.Stream()
        self.router, self.head = a4.Weights(r, ne, d, group), a4.Weights(r, head, d, group, symmetric=True)
        self.router_on, self.head_on = self.router.device(), self.head.device()
        self.bias = routing.encode(r.normal(0, 0.02, ne), F32)
        self.d_bias = gpu.dev(self.bias)
        self.norm_weight = S.f32_to_bf16_bits(r.uniform(0.5, 1.5, d).astype(np.float32))
        self.d_norm = gpu.dev(self.norm_weight)
        self.x, self.normed, self.logits = gpu.empty(t * d * 2), gpu.empty(t * d * 2), gpu.empty(t * ne * 4)
        self.idx, self.w, self.h2, self.out = gpu.empty(t * k * 4), gpu.empty(t * k * 2), gpu.empty(t * d * 2), gpu.empty(t * head * 4)
        self.pf, self.routes = gpu.Prefill(self.dl.moe), gpu.GroupedRoutesDevice(t * k, ne)
        self.partials = gpu.empty(t * k * d * 2)
        self.work = gpu.empty(self.pf.ffn_workspace_bytes(t, self.routes.max_row_tiles))
        self.cells, self.acts = gpu.empty(t * k * 4), gpu.empty(t * k * f * 2)
        self.residual, self.hidden = gpu.dev(np.zeros(t * d, np.uint16)), gpu.empty(t * d * 2)

    def head_of_the_layer(self):
        g, t, d, ne, s = self.gpu, self.t, self.d, self.ne, self.stream
        g.residual_add_rmsnorm_bf16w(self.x, None, self.d_norm, self.normed, d, 1e-6, t, s)
        g.affine4_product(self.normed, F16, d, *self.router_on, BF16, self.router.group, None, self.logits, F32, ne, t, ne, d, s)
        g.route_rows(self.desc, self.logits, F32, ne, self.d_bias, F32, self.idx, self.w, F16, t, s)

    def projection(self):
        n = self.head.n
        self.gpu.affine4_product(self.h2, F16, self.d, *self.head_on, BF16, self.head.group, None, self.out, F32, n, self.t, n, self.d, self.stream)

    def chunk(self):
        self.head_of_the_layer()
        self.pf.group_pairs(self.idx, self.w, self.t, self.k, self.ne, self.routes, residency=self.dl.pool.table)
        self.pf.encode_grouped_expert_gemms(self.dl.pool, self.dl.off, self.routes, self.normed, self.d, self.partials, self.work, self.t, self.k)
        self.pf.encode_reduce_token_major(self.partials, self.w, self.h2, self.t, self.k, self.d)
        self.projection()

    def tokens(self):
        m, dl = self.dl.moe, self.dl
        self.head_of_the_layer()
        m.encode_resolve_batch(self.idx, dl.pool.table, self.cells, self.t * self.k, self.ne)
        m.encode_phase1_batch(dl.pool, self.cells, dl.off, self.normed, self.d, self.acts, self.d, self.f, self.k, self.t)
        m.encode_phase2_batch(dl.pool, self.cells, dl.off, self.acts, self.w, self.residual, self.h2, self.hidden, self.d, self.f, self.k, self.t)
        self.projection()

    def results(self):
        self.stream.synchronize()
        t = self.t
        return dict(normed=self.normed.download(np.uint16, t * self.d).reshape(t, -1), logits=self.logits.download(np.float32, t * self.ne).reshape(t, -1),
                    idx=self.idx.download(np.uint32, t * self.k).reshape(t, -1), w=self.w.download(np.uint16, t * self.k).reshape(t, -1),
                    h2=self.h2.download(np.uint16, t * self.d).reshape(t, -1), out=self.out.download(np.float32, t * self.head.n).reshape(t, -1))

    def check_ends(self, x, got, what):
        """Norm, logits, routes and the last product, each against its reference over the device's own input of it."""
        t, d = self.t, self.d
        for i in range(min(t, 4)):
            row = x[i].copy()
            assert np.array_equal(got["normed"][i], O.residual_add_rmsnorm_bf16w(row, None, self.norm_weight, 1e-6)), f"{what}: norm of row {i}"
        for rows, weights, out, name in ((got["normed"], self.router, got["logits"], "logits"), (got["h2"], self.head, got["out"], "projection")):
            xv = a4.decode(rows, F16)
            a4.assert_close(out, xv @ weights.values.T, a4.bound_of(xv, weights), F32, f"{what}: {name}")
        want, weights, bound = routing.route(self.desc, got["logits"].astype(np.float64), self.bias.astype(np.float64))
        assert np.array_equal(got["idx"], want), f"{what}: routes"
        routing.assert_weights(got["w"], weights, bound, F16, f"{what}: weights")


CASES = [  # rows, d, f, experts, top k, groups, kept, scores, group of the weights, outputs of the projection
    (1, 256, 128, 32, 4, 1, 1, capi.SCORES_SOFTMAX, 64, 33),
    (5, 256, 128, 32, 4, 8, 4, capi.SCORES_SIGMOID, 64, 96),
    (33, 512, 128, 64, 8, 8, 3, capi.SCORES_SIGMOID, 128, 257),
    (130, 256, 128, 48, 4, 1, 1, capi.SCORES_SIGMOID, 32, 300),
]


def make(gpu, rows, d, f, ne, k, groups, kept, scores, group, head):
    return Chain(gpu, rows, d, f, ne, k, routing.desc(ne, k, scores, groups, kept, 2 if groups > 1 else 1, True, 2.5), group, head)


def inputs(c, count):
    return [S.activations_f16(S.SeedTree(0x5EED0062 + i), "x", c.t * c.d).reshape(c.t, c.d) for i in range(count)]


@pytest.mark.parametrize("case", CASES)
def test_a_chunk(gpu, case):
    c = make(gpu, *case)
    x = inputs(c, 1)[0]
    c.x.upload(x.reshape(-1))
    c.chunk()
    got = c.results()
    c.check_ends(x, got, "chunk")
    partials = c.partials.download(np.uint16, c.t * c.k * c.d).reshape(c.t, c.k, c.d)
    acts = WorkspaceActs(c.routes, c.work, c.t, c.d, c.f)
    for tok in sorted({0, c.t // 2, c.t - 1}):
        for rank in range(c.k):
            check_pair_stagewise(c.L, c.L.blobs[int(got["idx"][tok, rank])], got["normed"][tok], acts.row(tok, rank), partials[tok, rank],
                                 f"token {tok} rank {rank}")
    assert np.array_equal(got["h2"].reshape(-1), O.prefill_reduce(partials.reshape(-1), got["w"].reshape(-1), c.t, c.k, c.d))
    # the same rows as single tokens: the decode kernels round once where the chunk's partial rows are rounded first
    c.tokens()
    again = c.results()
    c.check_ends(x, again, "tokens")
    for name in ("normed", "logits", "idx", "w"):
        assert np.array_equal(again[name], got[name]), name
    assert_rel_close(again["h2"].reshape(-1), got["h2"].reshape(-1), "tokens and chunk", tol=2e-3)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("form", ["chunk", "tokens"])
def test_captured_and_replayed(gpu, case, form):
    c = make(gpu, *case)
    lib, rows, eager = capi.load(), inputs(c, 3), []
    for x in rows:
        c.x.upload(x.reshape(-1))
        getattr(c, form)()
        eager.append(c.results())
    capi.check(lib.shrike_hip_graph_begin_capture(c.stream.handle), "capture")
    getattr(c, form)()
    graph = lib.shrike_hip_graph_end_capture(c.stream.handle)
    assert graph
    for i in (1, 0, 2, 0):
        c.x.upload(rows[(i + 1) % 3].reshape(-1))
        getattr(c, form)()  # the program's own work between the replays
        c.stream.synchronize()
        c.x.upload(rows[i].reshape(-1))
        capi.check(lib.shrike_hip_graph_launch(graph, c.stream.handle), "launch")
        got = c.results()
        for name, value in got.items():
            assert np.array_equal(value, eager[i][name]), (i, name)
    capi.check(lib.shrike_hip_graph_destroy(graph), "destroy")
