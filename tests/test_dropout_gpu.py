"""GPU: wk_dropout against its definition (oracle/tokens.py) through the C ABI.

Tolerance: which elements stay is exact.  A kept value is f32(x) * f32(1 / (1 - p)) rounded to the type: half a step for
the scale, half a step for the product and, for the 16-bit types, half a step for the result (2^-24 + 2^-24, f16 2^-11 with
2^-25 below its normal range, bf16 2^-8); f64 likewise with 2^-53, and 2^-53 of the oracle's own division."""
import ctypes

import numpy as np
import pytest

from oracle import tokens as ot
from wekua_amd import raw

pytestmark = pytest.mark.gpu

REL = {"f32": 2.0 ** -23, "f64": 2.0 ** -51, "f16": 2.0 ** -11 + 2.0 ** -23, "bf16": 2.0 ** -8 + 2.0 ** -23}


def pack(dtype, x):
    return ot.bf16_bits(x) if dtype == "bf16" else x.astype(raw.real_np_dtype(dtype))


def values(dtype, bits):
    return (ot.bf16_values(bits) if dtype == "bf16" else bits).astype(np.float64)


def close(dtype, got, want):
    err = np.abs(got - want)
    return np.all(err <= REL[dtype] * np.abs(want) * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype == "f16" else 0))


def lay_out(dtype, x, rp, sp, gap):
    """A flat device image of x [depth, rows, cols] with the pitches, `gap` in between."""
    depth, rows, cols = x.shape
    flat = np.full((depth - 1) * sp + (rows - 1) * rp + cols + 5, gap, dtype=raw.real_np_dtype(dtype))
    for d in range(depth):
        for r in range(rows):
            flat[d * sp + r * rp:d * sp + r * rp + cols] = x[d, r]
    return flat


@pytest.mark.parametrize("dtype", ["f32", "f64", "f16", "bf16"])
@pytest.mark.parametrize("shape,pad_x,pad_y,gap", [
    ((1, 1, 1), 0, 0, 0), ((1, 1, 7), 0, 0, 0), ((1, 3, 4), 0, 0, 0), ((1, 5, 13), 0, 0, 0), ((2, 3, 5), 3, 0, 1),
    ((1, 33, 257), 0, 7, 0), ((3, 4, 64), 8, 8, 16), ((1, 9, 1023), 1, 2, 0), ((1, 300, 3), 2, 5, 0),
])
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_against_the_definition(dev, dtype, shape, pad_x, pad_y, gap, p):
    depth, rows, cols = shape
    rng = np.random.RandomState(hash((shape, pad_x)) % 1000)
    x = pack(dtype, rng.randn(*shape) * 3)
    xrp, yrp = cols + pad_x, cols + pad_y
    xsp, ysp = rows * xrp + gap, rows * yrp + gap
    seed, offset = 0xFEDCBA9876543210, (1 << 40) + 7
    poison = pack(dtype, np.full(1, -7.0))[0]
    dx = dev.upload(lay_out(dtype, x, xrp, xsp, poison))
    image = lay_out(dtype, np.full(shape, poison), yrp, ysp, poison)
    dy = dev.upload(image)
    dev.dropout(dtype, shape, dx, xrp, xsp, dy, yrp, ysp, p, seed, offset)
    got = dy.download(image.dtype, image.shape)
    want = ot.dropout(values(dtype, x), p, seed, offset)
    inside = lay_out("i8", np.ones(shape, np.int8), yrp, ysp, 0).astype(bool)
    assert (got[~inside] == poison).all(), "wrote outside the region"
    got = values(dtype, got[inside]).reshape(shape)
    assert np.array_equal(got == 0, want == 0) and close(dtype, got, want)
    if p == 0.0:
        assert np.array_equal(got, values(dtype, x))
    dx.free()
    dy.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_and_the_gradients_mask(dev, dtype):
    """In place gives the same; the gradient passes exactly where the forward pass kept, scaled alike."""
    shape, n = (1, 37, 129), 37 * 129
    rng = np.random.RandomState(3)
    x, g = pack(dtype, rng.rand(n) + 1), pack(dtype, rng.rand(n) + 1)
    bx, by, bg = dev.upload(x), dev.upload(x), dev.upload(g)
    dev.dropout(dtype, shape, bx, 129, n, by, 129, n, 0.25, 5, 9)
    dev.dropout(dtype, shape, bx, 129, n, bx, 129, n, 0.25, 5, 9)
    dev.dropout(dtype, shape, bg, 129, n, bg, 129, n, 0.25, 5, 9)
    y = by.download(x.dtype, (n,))
    assert np.array_equal(y, bx.download(x.dtype, (n,)))
    assert np.array_equal(values(dtype, y) == 0, values(dtype, bg.download(x.dtype, (n,))) == 0)
    for b in (bx, by, bg):
        b.free()


def test_dropped_elements_are_zero_whatever_they_held(dev):
    x = np.full(4096, np.nan, np.float32)
    x[::2] = np.inf
    b = dev.upload(x)
    dev.dropout("f32", (1, 1, 4096), b, 4096, 4096, b, 4096, 4096, 0.5, 1)
    got, keep = b.download(np.float32, (4096,)), ot.dropout_keep(4096, 0.5, 1, 0)
    assert (got[~keep] == 0).all() and not np.isfinite(got[keep]).any()
    dev.dropout("f32", (1, 1, 4096), b, 4096, 4096, b, 4096, 4096, 1.0, 1)
    assert (b.download(np.float32, (4096,)) == 0).all()
    b.free()


def test_count_in_device_memory(dev):
    """offset + *dev_step is one count: the same mask from either, another one for another count; it wraps at 2^64."""
    n = 1000
    one, step = dev.upload(np.ones(n, np.float32)), dev.upload(np.array([2 ** 64 - 3, 4], np.uint64))
    y = dev.malloc(4 * n)

    def mask(offset, at=None):
        dev.dropout("f32", (1, 1, n), one, n, n, y, n, n, 0.5, 11, offset, at)
        return y.download(np.float32, (n,)) != 0
    assert np.array_equal(mask(5), mask(1, step.ptr.value + 8)) and not np.array_equal(mask(5), mask(6))
    assert np.array_equal(mask(8, step), mask(5))
    for b in (one, step, y):
        b.free()


def test_refusals(dev):
    lib, b = dev.lib, dev.malloc(1 << 12)
    p = b.ptr.value

    def call(dtype=8, shape=(1, 2, 4), x=p, xrp=4, xsp=8, y=p, yrp=4, ysp=8, prob=0.1, stream=dev.stream):
        s3 = (ctypes.c_uint64 * 3)(*shape) if shape else None
        return lib.wk_dropout(stream, dtype, s3, x, xrp, xsp, y, yrp, ysp, prob, 1, 0, None)
    assert call() == 0
    for bad in ({"stream": None}, {"shape": None}, {"shape": (0, 2, 4)}, {"shape": (1, 0, 4)}, {"shape": (1, 2, 0)}, {"x": None}, {"y": None},
                {"xrp": 3}, {"yrp": 3}, {"shape": (2, 2, 4), "xsp": 7}, {"prob": -0.1}, {"prob": 1.5}, {"prob": float("nan")},
                {"yrp": 5, "ysp": 10}, {"shape": (2 ** 40, 2 ** 40, 4)}):
        assert call(**bad) == 1, bad
    for dtype in (0, 7, 18, 20, 34, -1):
        assert call(dtype=dtype) == 9, dtype
    dev.sync()
    b.free()


def test_slices_of_one_row(dev):
    """The row pitch of a single row is not walked and may be anything; slices that would lie over each other are refused all the
    same, and so are pitches whose product passes 64 bits."""
    cols = 40
    x = np.arange(1, 3 * cols + 1, dtype=np.float32)
    bx, by = dev.upload(x), dev.upload(np.full(3 * cols, -7, np.float32))
    lib, s3 = dev.lib, ctypes.c_uint64 * 3

    def call(shape, xrp, xsp, yrp, ysp):
        return lib.wk_dropout(dev.stream, 8, s3(*shape), bx.ptr, xrp, xsp, by.ptr, yrp, ysp, 0.25, 6, 0, None)
    for xrp, xsp, yrp, ysp in ((0, cols, 0, cols - 1), (0, cols - 1, 0, cols), (0, 0, cols, cols), (cols, cols, 0, 0), (1, 1, 1, 1)):
        assert call((3, 1, cols), xrp, xsp, yrp, ysp) == 1, (xrp, xsp, yrp, ysp)
    assert call((2, 2, 8), 2 ** 63, 0, 8, 16) == 1 and call((2, 2, 8), 8, 16, 2 ** 63, 0) == 1
    assert (by.download(np.float32, (3 * cols,)) == -7).all()
    want = ot.dropout(x.astype(np.float64), 0.25, 6, 0)
    for pitch in (0, 1, cols, 2 ** 63):
        by.write(np.full(3 * cols, -7, np.float32))
        assert call((3, 1, cols), pitch, cols, pitch, cols) == 0
        got = by.download(np.float32, (3 * cols,)).astype(np.float64)
        assert np.array_equal(got == 0, want == 0) and close("f32", got, want)
    for b in (bx, by):
        b.free()
