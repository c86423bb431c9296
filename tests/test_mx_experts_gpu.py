"""The experts' FFN over microscaled blocks in the kernels' long loops: single tokens' gate and up through LDS over several chunks of k, and the tiles
of many rows over rows long enough for 16-byte reads of scales. Against tests/mx_reference.py, and one kernel against another bit for bit."""
import numpy as np
import pytest

from shrike_amd import capi
from tests import mx_reference as R
from tests import test_mx_gpu as base
from tests import test_mx_shapes_gpu as shapes

pytestmark = pytest.mark.gpu
F16 = capi.ELEM_F16


# 256 workgroups and more of gate and up, d of 2 to 12 chunks of 256: whole ones, ends of one block to seven, a last chunk whose second step is empty;
# cells that several pairs share, positions that are not there
@pytest.mark.parametrize("d,f,ne,k,tokens,act,biases", [
    (320, 128, 6, 8, 16, capi.ACT_SILU, True), (512, 192, 5, 8, 16, capi.ACT_CLAMPED_SWIGLU, True), (576, 128, 40, 8, 16, capi.ACT_GELU_TANH, False),
    (768, 64, 9, 8, 32, capi.ACT_SILU, True), (832, 128, 7, 8, 17, capi.ACT_CLAMPED_SWIGLU, False), (1088, 192, 6, 8, 11, capi.ACT_SILU, True),
    (1856, 128, 5, 8, 16, capi.ACT_GELU_TANH, True), (2304, 128, 12, 8, 16, capi.ACT_SILU, False), (2880, 192, 6, 4, 22, capi.ACT_CLAMPED_SWIGLU, True),
    (4032, 64, 4, 4, 64, capi.ACT_SILU, True)])
def test_decode_of_long_rows_through_lds(gpu, d, f, ne, k, tokens, act, biases):
    assert (f + 63) // 64 * tokens * k >= 256 and d > 256
    shapes.check_decode(gpu, d, f, ne, k, tokens, act, biases, lambda rng: np.where(rng.random((tokens, k)) < 0.1, -1, rng.integers(0, ne, (tokens, k))))


class Chunk:
    """A layer's experts, all present, and the grouped FFN over any tokens of rows x = (codes, scales) that go to one expert each."""

    def __init__(self, gpu, ex, act, x, expert):
        self.gpu, self.ex, self.x, self.expert = gpu, ex, x, np.asarray(expert, np.uint32)
        self.pool = base.make_pool(gpu, ex)
        for e in range(ex.n):
            self.pool.publish(e, e, capi.RESIDENT)
        self.moe = gpu.MoE(ex.d, ex.f, ex.n, 1, activation=act, additive_biases=ex.biases)
        self.pf = gpu.Prefill(self.moe)

    def run(self, tokens):
        """(outputs, activations' codes, their scales) of those tokens, in their order."""
        gpu, d, f = self.gpu, self.ex.d, self.ex.f
        n = len(tokens)
        routes = gpu.GroupedRoutesDevice(n, self.ex.n)
        keep = [gpu.dev(self.expert[tokens]), gpu.dev(np.ones(n, np.float16)), gpu.dev(self.x[0][tokens]), gpu.dev(self.x[1][tokens])]
        ws = gpu.empty(self.pf.mx_ffn_workspace_bytes(routes.max_row_tiles)).fill(0xEE)
        out = gpu.empty(2 * n * d).fill(0x5A)
        gpu.synchronize()
        self.pf.group_pairs(keep[0], keep[1], n, 1, self.ex.n, routes, residency=self.pool.table)
        self.pf.encode_mx_grouped_expert_gemms(self.pool, self.ex.off, routes, keep[2], keep[3], out, ws, n, 1)
        gpu.synchronize()
        rows = routes.max_row_tiles * 64
        acts, at = ws.download(np.uint8), -(-rows * f // 256) * 256
        by_row = acts[:rows * f].reshape(rows, f), acts[at:at + rows * f // 32].reshape(rows, f // 32)
        codes, scales = np.empty((n, f), np.uint8), np.empty((n, f // 32), np.uint8)
        table = routes.download()
        for number, (_, start, count, _) in enumerate(table["row_tiles"]):
            token = table["sorted_pairs"][start:start + count, 0]
            codes[token], scales[token] = by_row[0][number * 64:number * 64 + count], by_row[1][number * 64:number * 64 + count]
        return out.download(np.uint16, n * d).reshape(n, d), codes, scales

    def many(self, tokens):
        """Whether that many tokens of a call are taken in runs of up to 256 rows an expert."""
        return tokens * self.ex.f >= self.ex.n << 17


def by_counts(rng, counts):
    """Experts of so many tokens each, in any order."""
    return rng.permutation(np.repeat(np.arange(len(counts)), counts))


# experts of 256, of up to 256, of up to 128 and of up to 64 rows in a run; d of 16 blocks and more, every remainder of the 16 whose scales are read together
@pytest.mark.parametrize("d,f,counts,act,biases", [
    (512, 1024, (300, 100, 37), capi.ACT_SILU, True), (576, 1024, (64, 200, 129), capi.ACT_CLAMPED_SWIGLU, True), (704, 1024, (512, 1, 65), capi.ACT_GELU_TANH, False),
    (960, 1024, (256, 128, 63), capi.ACT_SILU, True), (1024, 1024, (90, 250, 60), capi.ACT_CLAMPED_SWIGLU, False), (1088, 512, (600, 190), capi.ACT_SILU, True),
    (2304, 1088, (150, 80, 140), capi.ACT_SILU, False), (2880, 1024, (255, 66, 64), capi.ACT_CLAMPED_SWIGLU, True)])
def test_experts_of_many_long_rows(gpu, d, f, counts, act, biases):
    rng = np.random.default_rng(d + f + sum(counts))
    ex = R.Experts(rng, len(counts), d, f, biases)
    expert = by_counts(rng, counts)
    x = R.random_rows(rng, len(expert), d, R.E4M3, 0.5)
    chunk = Chunk(gpu, ex, act, x, expert)
    every = np.arange(len(expert))
    assert chunk.many(len(every)) and d >= 512
    out, codes, scales = chunk.run(every)
    # rows of every expert against 64 bits: its first and last, and some between
    for e, count in enumerate(counts):
        mine = np.flatnonzero(expert == e)
        some = mine[sorted({0, count - 1, *rng.integers(0, count, 6)})]
        a, da = ex.act(e, (x[0][some], x[1][some]), act)
        R.assert_quantized(codes[some], scales[some], a, da, f"activations of expert {e}")
        o, do = ex.down(e, (codes[some], scales[some]))
        R.assert_within(out[some], o, do, F16, f"outputs of expert {e}")
    # and every row against calls of fewer tokens, which other kernels take: a pair's row depends on its token and its expert alone
    few = (len(counts) << 17) // f // 2
    for first in range(0, len(every), few):
        part = every[first:first + few]
        assert not chunk.many(len(part))
        for name, whole, alone in zip(("outputs", "activations", "scales"), (out, codes, scales), chunk.run(part)):
            assert np.array_equal(alone, whole[part]), f"{name} of tokens from {first} on"
