"""The microscaled operators without a GPU: what they refuse before anything is launched, the blob's offsets, and the reference that
the GPU tests compare with against known codes."""
import ctypes as C
import errno

import numpy as np
import pytest

from shrike_amd import capi
from tests import mx_reference as R

A = 0x10000  # addresses that are only ever looked at
F16, F32 = capi.ELEM_F16, capi.ELEM_F32
MAXU32 = 0xFFFFFFFF


def refused(rc, word):
    assert rc == errno.EINVAL, rc
    assert word in capi.last_error(), capi.last_error()


QUANTIZE = dict(src=A, dtype=F16, stride=64, fmt=R.E4M3, codes=A, scales=A, rows=2, d=64)


@pytest.mark.parametrize("change,word", [
    (dict(src=None), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(dtype=3), "element type"), (dict(fmt=2), "format"),
    (dict(d=0), "multiple of 32"), (dict(d=48), "multiple of 32"), (dict(stride=63), "stride"), (dict(codes=A + 8), "aligned"), (dict(src=A + 1), "aligned"),
    (dict(src=A + 2, dtype=F32), "aligned"), (dict(rows=1 << 40), "too many"), (dict(rows=1 << 30, stride=1 << 40), "too many"),
    (dict(stride=1 << 41), "too many")])
@pytest.mark.parametrize("back", [False, True])
def test_quantize_refuses(change, word, back):
    a = dict(QUANTIZE, **change)
    lib = capi.load()
    if back:
        refused(lib.shrike_hip_mx_dequantize(None, a["codes"], a["scales"], a["fmt"], a["src"], a["dtype"], a["stride"], a["rows"], a["d"]), word)
    else:
        refused(lib.shrike_hip_mx_quantize(None, a["src"], a["dtype"], a["stride"], a["fmt"], a["codes"], a["scales"], a["rows"], a["d"]), word)


NORM = dict(hidden=A, delta=A, weight=A, total=A, out=A, codes=A, scales=A, d=64, rows=1)


@pytest.mark.parametrize("change,word", [
    (dict(hidden=None), "bound"), (dict(weight=None), "bound"), (dict(codes=None), "bound"), (dict(scales=None), "bound"), (dict(delta=None), "together"),
    (dict(total=None), "together"), (dict(d=0), "multiple"), (dict(d=40), "multiple"), (dict(d=4128), "multiple"), (dict(hidden=A + 2), "aligned"),
    (dict(out=A + 8), "aligned"), (dict(codes=A + 4), "aligned"), (dict(rows=MAXU32), "too many")])
def test_norm_refuses(change, word):
    a = dict(NORM, **change)
    refused(capi.load().shrike_hip_residual_add_rmsnorm_bf16w_mx8(None, a["hidden"], a["delta"], a["weight"], a["total"], a["out"], a["codes"], a["scales"],
                                                                  a["d"], 1e-6, a["rows"]), word)


PRODUCT = dict(x=A, xs=A, fmt=R.E4M3, w=A, ws=A, bias=None, out=A, dtype=F16, stride=16, rows=4, n=16, k=64)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "NULL"), (dict(xs=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"), (dict(out=None), "NULL"), (dict(fmt=2), "format"),
    (dict(dtype=F32), "fp16 or bf16"), (dict(dtype=9), "fp16 or bf16"), (dict(k=0), "k=0"), (dict(k=16), "k=16"), (dict(k=65568), "k=65568"),
    (dict(n=0), "n=0"), (dict(n=(1 << 24) + 1, stride=1 << 25), "not in"), (dict(rows=MAXU32), "too many"), (dict(stride=15), "stride"), (dict(x=A + 8), "aligned"),
    (dict(w=A + 1), "aligned"), (dict(out=A + 1), "aligned"), (dict(bias=A + 1), "aligned")])
def test_product_refuses(change, word):
    a = dict(PRODUCT, **change)
    refused(capi.load().shrike_hip_mx_product(None, a["x"], a["xs"], a["fmt"], a["w"], a["ws"], a["bias"], a["out"], a["dtype"], a["stride"], a["rows"], a["n"],
                                              a["k"]), word)


def test_nothing_to_do_is_no_error():
    lib = capi.load()
    a = QUANTIZE
    assert lib.shrike_hip_mx_quantize(None, a["src"], a["dtype"], a["stride"], a["fmt"], a["codes"], a["scales"], 0, a["d"]) == 0
    assert lib.shrike_hip_mx_dequantize(None, a["codes"], a["scales"], a["fmt"], a["src"], a["dtype"], a["stride"], 0, a["d"]) == 0
    assert lib.shrike_hip_residual_add_rmsnorm_bf16w_mx8(None, A, None, A, None, None, A, A, 64, 1e-6, 0) == 0
    assert lib.shrike_hip_mx_product(None, A, A, 0, A, A, None, A, F16, 16, 0, 16, 64) == 0


class Moe(C.Structure):
    """The head of a handle: what the calls below read of one before they refuse."""
    _fields_ = [("desc", capi.MoEDesc), ("device", C.c_int), ("rest", C.c_void_p * 3)]


def handle(d=128, f=64, biases=0):
    return Moe(capi.MoEDesc(d, f, 8, 4, 4, 0, 0, capi.ACT_SILU, biases, 0, 1.0, 0))


def experts(d=128, f=64, biases=False):
    off = capi.ExpertOffsets()
    size = capi.load().shrike_mx_expert_offsets_make(d, f, int(biases), C.byref(off))
    bases = capi.PoolBases()
    bases.base[0], bases.cells_per_chunk = A, 8
    return off, -(-size // 16) * 16, bases


@pytest.mark.parametrize("change,word", [
    (dict(moe=None), "NULL"), (dict(d=64), "differs"), (dict(f=128), "differs"), (dict(top_k=0), "topK"), (dict(top_k=9), "topK"), (dict(stride=24), "geometry"),
    (dict(cells=0), "geometry"), (dict(base=A + 8), "aligned"), (dict(gate_w_off=8), "multiples of 16"), (dict(up_w_off=1 << 20), "does not fit"),
    (dict(down_s_off=1 << 20), "does not fit"), (dict(x=None), "NULL"), (dict(xs=None), "NULL"), (dict(out=None), "NULL"), (dict(ws=None), "NULL"),
    (dict(x=A + 4), "aligned"), (dict(out=A + 8), "aligned"), (dict(ws=A + 16), "256-byte"), (dict(bytes=100), "needed"), (dict(tokens=MAXU32), "many|needed|GiB"),
    (dict(gate_ab_off=1, biases=1), "even"), (dict(down_ab_off=1 << 20, biases=1), "do not fit")])
@pytest.mark.parametrize("kind", ["grouped", "decode"])
def test_experts_refuse(change, word, kind):
    lib = capi.load()
    biases = change.get("biases", 0)
    moe, (off, stride, bases) = handle(biases=biases), experts(biases=bool(biases))
    for name in ("gate_w_off", "up_w_off", "down_s_off", "gate_ab_off", "down_ab_off"):
        if name in change:
            setattr(off, name, change[name])
    bases.base[0], bases.cells_per_chunk = change.get("base", A), change.get("cells", 8)
    stride = change.get("stride", stride)
    d, f, k, t = change.get("d", 128), change.get("f", 64), change.get("top_k", 4), change.get("tokens", 3)
    h = None if "moe" in change else C.addressof(moe)
    x, xs, out, ws, n = change.get("x", A), change.get("xs", A), change.get("out", A), change.get("ws", A), change.get("bytes", 1 << 20)
    routes = capi.HipGroupedRoutes(A, A, A, A, A)
    if kind == "grouped":
        rc = lib.shrike_hip_mx_grouped_ffn(h, None, C.byref(bases), stride, C.byref(off), C.byref(routes), 8 if t < 99 else 70000, x, xs, out, ws, n, t, d, f, k)
    else:
        rc = lib.shrike_hip_mx_decode_ffn(h, None, C.byref(bases), stride, A, C.byref(off), x, xs, A, None, out, None, ws, n, d, f, k, t)
    assert rc == errno.EINVAL, rc
    assert any(w in capi.last_error() for w in word.split("|")), capi.last_error()


def test_grouped_refuses_routes_that_are_not_bound():
    lib = capi.load()
    moe, (off, stride, bases) = handle(), experts()
    for missing in ("sorted_pairs", "row_tiles", "row_tile_count"):
        routes = capi.HipGroupedRoutes(A, A, A, A, A)
        setattr(routes, missing, None)
        refused(lib.shrike_hip_mx_grouped_ffn(C.addressof(moe), None, C.byref(bases), stride, C.byref(off), C.byref(routes), 8, A, A, A, A, 1 << 20, 3, 128, 64, 4),
                "routes")
    for missing in range(4):
        a = [A] * 4
        a[missing] = None
        refused(lib.shrike_hip_mx_decode_ffn(C.addressof(moe), None, C.byref(bases), stride, a[0], C.byref(off), a[1], A, a[2], None, a[3], None, A, 1 << 20, 128, 64,
                                             4, 3), "NULL")


def test_expert_offsets():
    lib = capi.load()
    off = capi.ExpertOffsets()
    assert lib.shrike_mx_expert_offsets_make(2880, 2880, 1, C.byref(off)) == 3 * 2880 * 2880 * 17 // 32 + 3 * 2880 * 2
    assert (off.gate_w_off, off.gate_s_off, off.up_w_off) == (0, 2880 * 1440, 2880 * 1440 + 2880 * 90)
    assert off.down_ab_off == 3 * 2880 * 2880 * 17 // 32 + 2 * 2880 * 2 and off.gate_b_off == off.up_b_off == off.down_b_off == 0
    assert lib.shrike_mx_expert_offsets_make(2048, 512, 0, C.byref(off)) == 3 * 2048 * 512 * 17 // 32
    for d, f in ((0, 64), (64, 0), (32, 64), (64, 100), (65536, 65536)):
        assert lib.shrike_mx_expert_offsets_make(d, f, 0, C.byref(off)) == 0
    assert lib.shrike_mx_expert_offsets_make(64, 64, 0, None) == 0


def test_the_reference_on_known_codes():
    x = np.zeros((1, 32))
    x[0, :12] = [6, 5, 2.5, 0.25, 0.75, -3.5, 1.75, 0.24, -0.26, 7.9, -0.0, 4.4]
    codes, s = R.quantize(x, R.E2M1)
    assert s[0, 0] == 127
    assert list(R.unpack(codes, R.E2M1)[0, :12]) == [7, 6, 4, 0, 2, 14, 4, 0, 9, 7, 8, 6]
    x[0, :6] = [448, 449, 300, 2.0 ** -9, 2.0 ** -10, 17]
    codes, s = R.quantize(x, R.E4M3)
    assert s[0, 0] == 127 and list(codes[0, :6]) == [0x7E, 0x7E, 0x79, 1, 0, 0x58]
    assert R.quantize(np.full((1, 32), 2.0 ** -140), R.E4M3)[1][0, 0] == 0
    v, sc = R.quantize(np.full((1, 32), np.inf), R.E2M1)
    assert sc[0, 0] == 255 and not v.any() and np.isnan(R.values(v, sc, R.E2M1)).all()
    rng = np.random.default_rng(0)
    x = rng.standard_normal((20, 256))
    for fmt, most in ((R.E4M3, 0.125), (R.E2M1, 0.25)):  # (what saturates: 448 for just under 512, 6 for just under 8)
        codes, s = R.quantize(x, fmt)
        assert np.array_equal(R.quantize(R.values(codes, s, fmt), fmt)[0], codes) or fmt == R.E2M1
        top = np.repeat(np.abs(x.reshape(20, -1, 32)).max(-1), 32, axis=1)
        assert np.all(np.abs(R.values(codes, s, fmt) - x) <= most * top)


@pytest.mark.parametrize("tokens,refusal", [(capi.MX_MAX_DECODE_TOKENS, None), (capi.MX_MAX_DECODE_TOKENS + 1, "many")])
def test_decode_takes_so_many_tokens(tokens, refusal):
    """(As many as it takes are refused for what comes next, the workspace.)"""
    lib = capi.load()
    moe, (off, stride, bases) = handle(), experts()
    refused(lib.shrike_hip_mx_decode_ffn(C.addressof(moe), None, C.byref(bases), stride, A, C.byref(off), A, A, A, None, A, None, A, 0, 128, 64, 4, tokens),
            refusal or "needed")


def test_grouped_refuses_rows_past_4_gib():
    lib = capi.load()
    moe, (off, stride, bases) = handle(), experts()
    routes = capi.HipGroupedRoutes(A, A, A, A, A)
    for rows in (1 << 25, (1 << 32) // 128 - 8):
        refused(lib.shrike_hip_mx_grouped_ffn(C.addressof(moe), None, C.byref(bases), stride, C.byref(off), C.byref(routes), 8, A, A, A, A, 1 << 20, rows, 128, 64, 4),
                "GiB")
