"""Where the calls' documented limits lie, on both sides of each: what a launch or a 32-bit offset cannot have is refused as an argument, before
anything is launched. No GPU."""
import errno

import pytest

from shrike_amd import capi

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
