"""Where the calls' documented limits lie, on both sides of each: what a launch or a 32-bit offset cannot have is refused as an argument, before
anything is launched. No GPU."""
import ctypes as C
import errno

import pytest

from shrike_amd import capi
from tests import test_mx_cpu as base

A = 0x10000  # an address that is only ever looked at


def refused(rc, word):
    assert rc == errno.EINVAL, rc
    assert word in capi.last_error(), capi.last_error()


@pytest.mark.parametrize("rows", [(1 << 32) // 256, 65535 * 1024, 0xFFFFFFFF])
def test_norm_with_8_bit_rows_refuses_more_rows_than_a_launch_has(rows):
    """A workgroup of 256 threads a row: a launch holds fewer than 2^32 threads."""
    refused(capi.load().shrike_hip_residual_add_rmsnorm_bf16w_mx8(None, A, None, A, None, None, A, A, 32, 1e-6, rows), "too many")


@pytest.mark.parametrize("rows", [(1 << 32) // 256, 65535 * 1024, 0xFFFFFFFF])
def test_norm_refuses_more_rows_than_a_launch_has(rows):
    refused(capi.load().shrike_hip_residual_add_rmsnorm_bf16w(None, A, None, A, A, 32, 1e-6, rows), "too many")


@pytest.mark.parametrize("part", ["gate_w_off", "up_w_off", "down_w_off"])
@pytest.mark.parametrize("kind", ["grouped", "decode"])
def test_no_expert_s_codes_lie_in_the_last_line_below_4_gib(part, kind):
    """The loads' offsets from a cell's start are 32 bits, and reach up to a line past a row before they are brought back to its end: past 4 GiB they
    would come back at the cell's start. (What is accepted is refused for what comes next, the workspace.)"""
    lib = capi.load()
    d = f = 64
    codes = d * f // 2
    moe = base.handle(d, f)
    off, _, bases = base.experts(d, f)
    routes = capi.HipGroupedRoutes(A, A, A, A, A)
    last = ((1 << 32) - 1 - 128 - codes) // 16 * 16
    for at, word in ((last, "needed"), (last + 16, "does not fit"), ((1 << 32) - 16 - codes, "does not fit")):
        setattr(off, part, at)
        if kind == "grouped":
            rc = lib.shrike_hip_mx_grouped_ffn(C.addressof(moe), None, C.byref(bases), 1 << 33, C.byref(off), C.byref(routes), 8, A, A, A, A, 0, 3, d, f, 4)
        else:
            rc = lib.shrike_hip_mx_decode_ffn(C.addressof(moe), None, C.byref(bases), 1 << 33, A, C.byref(off), A, A, A, None, A, None, A, 0, d, f, 4, 3)
        refused(rc, word)


@pytest.mark.parametrize("kind", ["grouped", "decode"])
def test_experts_refuse_longer_rows_of_activations_than_a_product_takes(kind):
    """The down product's k is f: 256 rows of it in one tile are reached by 32 bits. (The longest is refused for what comes next, the workspace.)"""
    lib = capi.load()
    d = 64
    routes = capi.HipGroupedRoutes(A, A, A, A, A)
    for f, word in ((capi.MX_MAX_K, "needed"), (capi.MX_MAX_K + 64, "f="), (1 << 25, "f=")):
        moe = base.handle(d, f)
        off, stride, bases = base.experts(d, f)
        if kind == "grouped":
            rc = lib.shrike_hip_mx_grouped_ffn(C.addressof(moe), None, C.byref(bases), stride, C.byref(off), C.byref(routes), 8, A, A, A, A, 0, 3, d, f, 4)
        else:
            rc = lib.shrike_hip_mx_decode_ffn(C.addressof(moe), None, C.byref(bases), stride, A, C.byref(off), A, A, A, None, A, None, A, 0, d, f, 4, 3)
        refused(rc, word)
