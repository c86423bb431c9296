"""The experts' FFN over microscaled blocks in the kernels' long loops: single tokens' gate and up through LDS over several chunks of k. Against
tests/mx_reference.py."""
import numpy as np
import pytest

from shrike_amd import capi
from tests import test_mx_shapes_gpu as shapes

pytestmark = pytest.mark.gpu


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
