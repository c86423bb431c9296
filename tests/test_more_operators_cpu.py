"""What routing from logits and the 4-bit product refuse, on both sides of each limit. No GPU: an accepted call of no rows launches nothing."""
import ctypes as C
import errno
import math

import numpy as np
import pytest

from shrike_amd import capi
from tests import route_reference as ref

A = 0x10000  # an address that is only ever looked at


def route(d=None, logits=A, logits_type=capi.ELEM_F32, stride=256, bias=A, bias_type=capi.ELEM_F32, idx=A, w=A, weights_type=capi.ELEM_F16, rows=0, **desc):
    if d is None:
        d = ref.desc(**{**dict(experts=256, top_k=8), **desc})
    return capi.load().shrike_hip_route_rows(None, C.byref(d) if d else None, logits, logits_type, stride, bias, bias_type, idx, w, weights_type, rows)


def product(x=A, x_type=capi.ELEM_F16, stride=256, codes=A, scales=A, biases=A, meta=capi.META_BF16, group=64, bias=None, out=A, out_type=capi.ELEM_F16,
            out_stride=100, rows=0, n=100, k=256, w=True):
    p = capi.Projection(codes, scales, biases)
    return capi.load().shrike_hip_affine4_product(None, x, x_type, stride, C.byref(p) if w else None, meta, group, bias, out, out_type, out_stride, rows, n, k)


def refused(rc, word):
    assert rc == errno.EINVAL, rc
    assert word in capi.last_error(), capi.last_error()


@pytest.mark.parametrize("how,word", [
    (dict(logits=None), "NULL"), (dict(idx=None), "NULL"), (dict(w=None), "NULL"), (dict(d=0), "NULL"),
    (dict(logits_type=3), "element type"), (dict(weights_type=7), "element type"), (dict(bias_type=3), "element type"),
    (dict(experts=0, top_k=1), "numExperts"), (dict(experts=1025, stride=2000), "numExperts"),
    (dict(scores=2), "scores"), (dict(groups=0), "groups"), (dict(groups=65, experts=650, stride=700, kept=65), "groups"), (dict(groups=7), "groups"),
    (dict(groups=512, experts=512, stride=512, kept=512), "groups"),
    (dict(groups=8, kept=0), "keptGroups"), (dict(groups=8, kept=9), "keptGroups"), (dict(best=0), "groupTop"), (dict(best=3), "groupTop"),
    (dict(top_k=0), "topK"), (dict(top_k=33), "topK"), (dict(experts=4, top_k=5), "topK"), (dict(experts=64, groups=16, kept=2, top_k=9), "topK"),
    (dict(scaling=math.nan), "scaling"), (dict(scaling=math.inf), "scaling"), (dict(stride=255), "stride"), (dict(stride=(1 << 28) + 1), "stride"),
    (dict(logits=A + 2), "aligned"), (dict(logits=A + 1, logits_type=capi.ELEM_BF16), "aligned"), (dict(idx=A + 2), "aligned"), (dict(w=A + 1), "aligned"),
    (dict(w=A + 2, weights_type=capi.ELEM_F32), "aligned"), (dict(bias=A + 2), "aligned"), (dict(bias=A + 1, bias_type=capi.ELEM_F16), "aligned"),
])
def test_routing_refuses(how, word):
    refused(route(**how), word)
    refused(route(**{**how, "rows": 7}), word)


@pytest.mark.parametrize("how", [
    dict(), dict(experts=1, top_k=1), dict(experts=1024, top_k=32, stride=1024), dict(groups=64, kept=1, top_k=4), dict(experts=64, groups=16, kept=2, top_k=8), dict(best=2),
    dict(groups=64, experts=64, kept=64, best=2), dict(scaling=-1.0), dict(stride=1 << 28), dict(bias=None, bias_type=99), dict(logits=A + 2, logits_type=capi.ELEM_F16),
    dict(logits=A + 4), dict(w=A + 2), dict(bias=A + 2, bias_type=capi.ELEM_BF16),
])
def test_routing_takes_no_rows(how):
    assert route(**how) == 0, capi.last_error()


@pytest.mark.parametrize("how,word", [
    (dict(x=None), "NULL"), (dict(w=False), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(out=None), "NULL"),
    (dict(x_type=capi.ELEM_F32), "rows are"), (dict(meta=2), "metadata"), (dict(out_type=3), "element type"),
    (dict(group=16), "groups of"), (dict(group=0), "groups of"), (dict(group=256), "groups of"), (dict(group=96), "groups of"),
    (dict(k=0), "k="), (dict(k=96), "k="), (dict(k=192, group=128), "k="), (dict(k=48, group=32), "k="), (dict(k=65536 + 64, stride=1 << 20), "k="),
    (dict(n=0), "n="), (dict(n=(1 << 24) + 1, out_stride=1 << 25), "n="), (dict(rows=(1 << 22) + 1), "rows are too many"),
    (dict(stride=248), "stride"), (dict(stride=257), "stride"), (dict(stride=260), "stride"), (dict(stride=(1 << 36) + 8), "stride"),
    (dict(out_stride=99), "stride"), (dict(out_stride=(1 << 36) + 1), "stride"),
    (dict(x=A + 8), "16-byte"), (dict(codes=A + 4), "16-byte"), (dict(scales=A + 1), "aligned"), (dict(biases=A + 1), "aligned"), (dict(bias=A + 1), "aligned"),
    (dict(out=A + 1), "aligned"), (dict(out=A + 2, out_type=capi.ELEM_F32), "aligned"),
])
def test_product_refuses(how, word):
    refused(product(**how), word)
    if "rows" not in how:
        refused(product(**{**how, "rows": 7}), word)


@pytest.mark.parametrize("how", [
    dict(), dict(biases=None), dict(group=32, k=32, stride=32), dict(group=128, k=384, stride=384), dict(k=65536, stride=65536), dict(n=1 << 24, out_stride=1 << 24),
    dict(n=1, out_stride=1), dict(stride=1 << 36), dict(out_stride=1 << 36), dict(scales=A + 2, biases=A + 6, bias=A + 10, out=A + 2), dict(x_type=capi.ELEM_BF16),
    dict(out_type=capi.ELEM_F32, out=A + 4),
])
def test_product_takes_no_rows(how):
    assert product(**how) == 0, capi.last_error()


def test_the_routing_reference_on_rows_worked_by_hand():
    d = ref.desc(6, 2, capi.SCORES_SIGMOID, groups=3, kept=1, best=2, scaling=2.0)
    # choices: groups (0, 1), (2, 3), (4, 5) sum to 1.0, 0.9 + 0.2, 0.5 + 0.5
    idx, w, _ = ref.route(d, np.log(np.array([[1.0, 1.0, 9.0, 0.25, 1.0, 1.0]])))
    assert idx.tolist() == [[2, 3]] and np.allclose(w, [[2 * 0.9 / 1.1, 2 * 0.2 / 1.1]])
    idx, w, _ = ref.route(d, np.log(np.array([[1.0, 1.0, 9.0, 0.25, 1.0, 1.0]])), [0, 0.25, 0, 0, -1, -1])
    assert idx.tolist() == [[1, 0]] and np.allclose(w, [[1.0, 1.0]])
    d = ref.desc(4, 3, capi.SCORES_SOFTMAX, renormalize=False)
    idx, w, _ = ref.route(d, np.array([[np.nan, 0.0, -np.inf, 0.0], [-np.inf] * 4]))
    assert idx.tolist() == [[1, 3, 0], [0, 1, 2]] and np.allclose(w, [[0.5, 0.5, 0.0], [0.0] * 3])
