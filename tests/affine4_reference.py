"""Products with 4-bit weights and group scales in numpy, in 64 bits, with the bound that a kernel's result is held to."""
from __future__ import annotations

import numpy as np

from shrike_amd import capi, runtime as rt
from tests.mx_reference import half_step
from tests.route_reference import decode, encode

F32, F16, BF16 = capi.ELEM_F32, capi.ELEM_F16, capi.ELEM_BF16


class Weights:
    """Codes, scales and biases (None: symmetric) of n rows of k; `whole`: powers of two and halves, so that sums are exact."""

    def __init__(self, rng, n, k, group=64, meta=BF16, symmetric=False, whole=False):
        self.n, self.k, self.group, self.meta = n, k, group, meta
        codes = rng.integers(0, 16, (n, k)).astype(np.uint8)
        shape = (n, k // group)
        if whole:
            scales, biases = 2.0 ** rng.integers(-1, 2, shape), rng.integers(-16, 17, shape) * 0.5
        else:
            scales = 0.01 * np.exp(0.5 * rng.standard_normal(shape))
            biases = -7.5 * scales + 0.01 * rng.standard_normal(shape)
        self.scale_bits, self.bias_bits = encode(scales, meta), None if symmetric else encode(biases, meta)
        self.codes = np.ascontiguousarray(codes[:, 0::2] | codes[:, 1::2] << 4)
        s = np.repeat(decode(self.scale_bits, meta), group, 1)
        b = -8.0 * s if symmetric else np.repeat(decode(self.bias_bits, meta), group, 1)
        self.values, self.size = codes * s + b, codes * s + np.abs(b)  # and the sum of the magnitudes that a kernel may add

    def device(self):
        return rt.dev(self.codes), rt.dev(self.scale_bits), None if self.bias_bits is None else rt.dev(self.bias_bits)


def bound_of(x, w):
    """Products are exact in fp32; a group's sum is a chain of up to 64 additions (a group of 128 counts as two), then one or two fused
    steps a group into a running sum, up to 16 such sums joined, the bias vector: each off by 2^-23 of no more than the magnitudes' sum (half a
    step, and as much again should an instruction cut off instead of rounding)."""
    return (np.abs(x) @ w.size.T) * ((64 + 2 * (w.k // min(w.group, 64)) + 17) * 2.0 ** -23)


def run(x_bits, x_type, w, bias_bits=None, out_type=F16, pad=0, x_pad=0, stream=None, weights=None):
    """The call over encoded rows; what lies between and behind the rows has to stay. Returns the output's bits."""
    rows, k = x_bits.shape
    host = np.full((rows, k + x_pad), 0x7E00 if x_type == F16 else 0x7FC0, np.uint16)
    host[:, :k] = x_bits
    codes, scales, biases = weights or w.device()
    t = np.float32 if out_type == F32 else np.uint16
    size = np.dtype(t).itemsize
    stride = w.n + pad
    out = rt.empty((rows + 1) * stride * size + 64)
    out.fill(0xA5)
    dx, db = rt.dev(host), None if bias_bits is None else rt.dev(bias_bits)
    rt.affine4_product(dx, x_type, k + x_pad, codes, scales, biases, w.meta, w.group, db, out, out_type, stride, rows, w.n, k, stream)
    stream.synchronize() if stream else rt.synchronize()
    all_ = out.download(t, (rows + 1) * stride)
    grid = all_.reshape(rows + 1, stride)
    mark = np.frombuffer(b"\xa5" * size, t)[0]
    untouched = grid.copy()
    untouched[:rows, :w.n] = mark
    assert np.all(untouched.view(np.uint8) == 0xA5), "wrote past its outputs"
    return np.ascontiguousarray(grid[:rows, :w.n])


def assert_close(got, want, bound, out_type, what=""):
    g = decode(got, out_type)
    step = np.abs(want) * 2.0 ** -24 + 2.0 ** -149 if out_type == F32 else half_step(np.abs(want) + bound, out_type)
    err, tol = np.abs(g - want), bound + step
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert np.all(err <= tol), f"{what}: {worst}: {g[worst]} for {want[worst]}, off by {err[worst]:.3e}, {tol[worst]:.3e} allowed"


def assert_exact(got, want, out_type, what=""):
    """`want` is what the sums are exactly: the output is it, rounded once."""
    expect = encode(want, out_type)
    bad = np.argwhere(got != expect)
    assert len(bad) == 0, f"{what}: {len(bad)} of {got.size}, first at {bad[0]}: {decode(got, out_type)[tuple(bad[0])]} for {want[tuple(bad[0])]}"


def whole_rows(rng, rows, k, x_type):
    return encode(rng.integers(-2, 3, (rows, k)) * (rng.random((rows, k)) < 0.5), x_type)
