"""GPU: wk_f8_quantize and wk_gemm_f8 against their definitions (oracle/tokens.py) through the C ABI.

The quantiser is exact: scales and codes have to be equal.  The product: a block's 128 exact products are summed in f32
(at most 128 roundings of 2^-23, counting a truncating adder), multiplied by a rounded product of two scales (2 * 2^-24) and
added to the running sum (one rounding of 2^-24 per block): (128 + kblocks + 2) * 2^-23 of the sum of magnitudes.  For
16-bit results seven of eight consecutive products may each lose 2^-13 of the largest of them.  Then the bias
(2^-24 of the result and of the sum before it), an activation (slope at most one; tanh and exp within 2^-20), and half a
step of the result's type."""
import ctypes

import numpy as np
import pytest

from oracle import tokens as ot
from wekua_amd import raw

pytestmark = pytest.mark.gpu


def pack(dtype, x):
    return ot.bf16_bits(x) if dtype == "bf16" else x.astype(raw.real_np_dtype(dtype))


def values(dtype, bits):
    return (ot.bf16_values(bits) if dtype == "bf16" else bits).astype(np.float64)


def pitched(a, pitch, gap):
    out = np.full((a.shape[0], pitch), gap, dtype=a.dtype)
    out[:, :a.shape[1]] = a
    return out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 128, 0), (3, 129, 0), (5, 1000, 3), (128, 128, 0), (130, 257, 1), (257, 300, 8), (17, 7, 0)])
def test_quantize(dev, dtype, block_rows, rows, cols, pad):
    rng = np.random.RandomState(rows * 31 + cols)
    x = rng.randn(rows, cols) * np.exp(3 * rng.randn(rows, 1))
    x[rng.rand(rows, cols) < 0.1] = 0
    if rows > 2:
        x[1] = 0                                   # a row of zeros
        x[2] *= 2.0 ** -14                         # small ones
    bits = pack(dtype, np.clip(x, -6e4, 6e4))
    groups, cb = -(-rows // block_rows), -(-cols // 128)
    bx = dev.upload(pitched(bits, cols + pad, pack(dtype, np.full(1, 1e4))[0]))
    bq, bs = dev.upload(np.full((rows, cols + 5), 0xEE, np.uint8)), dev.upload(np.full((groups, cb + 2), -7, np.float32))
    dev.f8_quantize(dtype, rows, cols, bx, cols + pad, block_rows, bq, cols + 5, bs, cb + 2)
    q, s = bq.download(np.uint8, (rows, cols + 5)), bs.download(np.float32, (groups, cb + 2))
    want_q, want_s = ot.f8_quantize(values(dtype, bits), block_rows)
    assert (q[:, cols:] == 0xEE).all() and (s[:, cb:] == -7).all(), "wrote outside the region"
    assert np.array_equal(s[:, :cb], want_s) and np.array_equal(q[:, :cols], want_q)
    for b in (bx, bq, bs):
        b.free()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(dev, block_rows):
    """Infinities, NaN, the type's largest and smallest values, values next to a rounding border."""
    x = np.zeros((128 * 3, 128 * 5), np.float32)
    x[0, :128] = np.linspace(-448, 448, 128)
    x[:1, 128:256] = ((ot.E4M3[:0x7E] + ot.E4M3[1:0x7F]) / 2).astype(np.float32)[-126:].tolist() + [448, 0]
    x[0, 256], x[130, 3], x[131, 140] = np.inf, np.nan, -np.inf
    x[0, 390], x[260, 0], x[260, 130], x[300, 260] = 3.4e38, 1e-38, 1e-45, 448 * 2.0 ** -126
    bx, bq, bs = dev.upload(x), dev.malloc(x.size), dev.malloc(4 * 384 * 5)
    dev.f8_quantize("f32", 384, 640, bx, 640, block_rows, bq, 640, bs, 5)
    want_q, want_s = ot.f8_quantize(x.astype(np.float64), block_rows)
    assert np.array_equal(bs.download(np.float32, want_s.shape), want_s, equal_nan=True)
    assert np.array_equal(bq.download(np.uint8, x.shape), want_q)
    for b in (bx, bq, bs):
        b.free()


def check_gemm(dev, M, N, K, out="f32", bias=False, kind=-1, pads=(0, 0, 0), shift=0, seed=0, codes=None, cut=True):
    rng = np.random.RandomState(seed + M * 7 + N * 3 + K)
    kb = -(-K // 128)
    a = codes(rng, M, K) if codes else ot.e4m3_encode(np.clip(rng.randn(M, K) * 60, -448, 448))
    b = codes(rng, N, K) if codes else ot.e4m3_encode(np.clip(rng.randn(N, K) * 60, -448, 448))
    sa, sb = np.exp(rng.randn(M, kb)).astype(np.float32) / 60, (np.exp(rng.randn(-(-N // 128), kb)) / 60 / np.sqrt(K)).astype(np.float32)
    bi = rng.randn(N).astype(np.float32) if bias else None
    lda, ldb, ldc = K + pads[0], K + pads[1], N + pads[2]
    # everything around the operands is NaN codes and NaN scales: none of it may enter
    fa, fb = (np.concatenate([np.full(shift, 0x7F, np.uint8), pitched(v, ld, 0x7F).reshape(-1)]) for v, ld in ((a, lda), (b, ldb)))
    bufs = [dev.upload(v) for v in (fa, fb, pitched(sa, kb + 1, np.nan), pitched(sb, kb + 3, np.nan))]
    bbias = dev.upload(bi) if bias else None
    poison = pack(out, np.full(1, -7.0))[0]
    bc = dev.upload(np.full((M, ldc), poison))
    dev.gemm_f8(M, N, K, bufs[0].ptr.value + shift, lda, bufs[2], kb + 1, bufs[1].ptr.value + shift, ldb, bufs[3], kb + 3, out, bc, ldc,
                bbias, kind)
    got = bc.download(poison.dtype, (M, ldc))
    assert (got[:, N:] == poison).all(), "wrote outside C"
    got = values(out, got[:, :N])
    want, mag, largest = ot.gemm_f8(a, sa, b, sb, bi, kind, cut)
    tol = (128 + kb + 2) * 2.0 ** -23 * mag + (2.0 ** -23 * (np.abs(want) + mag) if bias else 0)
    tol += 7 * 2.0 ** -13 * largest if out != "f32" else 0
    tol += (2.0 ** -20 if kind >= 0 else 0) + {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[out] * np.abs(want) * 1.01
    tol += 2.0 ** -25 if out == "f16" else 1e-37
    worst = np.max(np.abs(got - want) / tol)
    assert worst <= 1, f"{worst} times the tolerance"
    for b_ in bufs + [bc] + ([bbias] if bias else []):
        b_.free()


@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 16, 128), (16, 1, 127), (2, 3, 129), (7, 130, 300), (16, 128, 256), (17, 129, 511), (33, 257, 1000), (64, 500, 16),
    (100, 100, 100), (128, 128, 128), (129, 127, 384), (256, 256, 512), (300, 200, 2049), (1, 1000, 4096), (5, 2048, 3000), (257, 511, 640)])
def test_gemm_sizes(dev, M, N, K):
    """Rows on 16-byte boundaries behind a gap, and rows that follow each other at whatever K is."""
    check_gemm(dev, M, N, K, pads=(-K % 16, -K % 16 + 16, 3))
    check_gemm(dev, M, N, K, pads=(1 if K % 16 == 0 else 0, 0, 0))


@pytest.mark.parametrize("out", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(65, 70, 1), (100, 100, 100), (65, 300, 129), (129, 127, 384), (257, 511, 640), (300, 200, 2049), (150, 150, 9001), (1000, 140, 255)])
def test_gemm_any_address_16_bit(dev, out, M, N, K):
    """16-bit results of more than 64 rows whose operands' rows begin anywhere: the register-staged tiles with the 8-bit instruction."""
    check_gemm(dev, M, N, K, out, pads=(1 if K % 16 == 0 else 0, 0, 0))
    check_gemm(dev, M, N, K, out, True, 1, pads=(3, 2, 1), shift=7)


@pytest.mark.parametrize("M,N,K,kind", [(2048, 192, 1100, 1), (3600, 3700, 136, -1), (3840, 3584, 640, -1), (3601, 3900, 1280, 0), (700, 2100, 520, -1)])
def test_gemm_large_f16(dev, M, N, K, kind):
    check_gemm(dev, M, N, K, "f16", kind == 0, kind, pads=(-K % 16, -K % 16, 4 if M % 2 else 0), cut=False)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(8, 2048, 4096), (1000, 1300, 2000), (4096, 4096, 4096)])
def test_gemm_same_bits_on_every_run(dev, out, M, N, K):
    """Ten runs one after the other, into buffers that hold something else each time."""
    rng = np.random.RandomState(M)
    kb, ld = -(-K // 128), -(-K // 16) * 16
    a, b = (rng.randint(0, 0x7F, (r, ld)).astype(np.uint8) | (rng.randint(0, 2, (r, ld)) << 7).astype(np.uint8) for r in (M, N))
    bufs = [dev.upload(v) for v in (a, b, np.exp(rng.randn(M, kb)).astype(np.float32), np.exp(rng.randn(-(-N // 128), kb)).astype(np.float32))]
    t = np.uint32 if out == "f32" else np.uint16
    first = None
    for run in range(10):
        bc = dev.upload(np.full((M, N), run, t))
        dev.gemm_f8(M, N, K, bufs[0], ld, bufs[2], kb, bufs[1], ld, bufs[3], kb, out, bc, N)
        got = bc.download(t, (M, N))
        assert first is None or np.array_equal(got, first), run
        first = got
        bc.free()
    for x in bufs:
        x.free()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,kind", [(65, 16, 128, -1), (2048, 192, 1100, 1), (3600, 3700, 136, -1), (3840, 3584, 640, -1), (3601, 3900, 1280, 0), (1, 20000, 512, -1)])
def test_gemm_large(dev, out, M, N, K, kind):
    """Every tile size, whole tiles and ragged ones, one to ten blocks of k with and without a short one behind them, against a
    product in 64 bits; the eight products' largest is bounded by their sum."""
    check_gemm(dev, M, N, K, out, kind == 0, kind, pads=(-K % 16, -K % 16, 4 if M % 2 else 0), cut=False)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 16384, 140), (8, 16421, 256), (17, 16383, 300), (33, 20000, 130), (32, 32768, 64), (64, 33000, 133), (40, 33000, 300), (5, 70001, 129)])
def test_gemm_few_rows_many_columns(dev, out, M, N, K):
    """Both sides of where tiles take over from streaming, and between tiles of 64 and 128 columns."""
    check_gemm(dev, M, N, K, out, True, 1, pads=(-K % 16, -K % 16, 0), cut=False)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bias,kind", [(False, -1), (True, -1), (True, 0), (False, 1)])
@pytest.mark.parametrize("M,N", [(3, 70), (200, 300)])
def test_gemm_epilogue(dev, out, bias, kind, M, N):
    check_gemm(dev, M, N, 272, out, bias, kind, pads=(0, 0, 1))


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [1, 2, 4, 8, 15])
def test_gemm_unaligned_bases_in_tiles(dev, out, shift):
    """More than 64 rows behind a base that is no multiple of 16, rows a multiple of 16 apart and not."""
    check_gemm(dev, 130, 150, 256, out, shift=shift)
    check_gemm(dev, 70, 200, 300, out, shift=shift, pads=(4, 20, 0))


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,pad", [(5, 140, 700, 4), (130, 140, 700, 4), (130, 140, 700, 0), (300, 300, 640, 0)])
def test_gemm_far_scales(dev, out, M, N, K, pad):
    """Scales from 2^-126 to 2^127 whose products f32 holds, large ones against small ones, zero scales, and blocks of zeros under
    products up to 2^127: a zero block adds nothing.  Tolerance as in check_gemm; every product of scales is a power of two here, so exact."""
    rng = np.random.RandomState(M + K)
    kb = -(-K // 128)
    a, b = (ot.e4m3_encode(np.clip(rng.randn(r, K) * 60, -448, 448)) for r in (M, N))
    e = np.array([126, -126, 90, -90, 0, 127])[:kb]                  # of A's scales, block by block; B's the other way
    ea, eb = np.tile(e, (M, 1)), np.tile(-e, (-(-N // 128), 1))
    ea[:, -1], eb[:, -1] = 127, 0                                    # a block of zeros under 2^127
    ea[1::3] -= 2 * (ea[1::3] > -100)                                # rows apart
    sa, sb = (2.0 ** ea).astype(np.float32), (2.0 ** eb).astype(np.float32)
    sa[2, 0] = 0
    a[:, 128 * (kb - 1):] = 0
    a[M - 1, :128] = 0x80                                            # and one of -0 within another row
    lda, ldb = K + pad, K + pad
    bufs = [dev.upload(v) for v in (pitched(a, lda, 0x7F), pitched(b, ldb, 0x7F), sa, sb)]
    bc = dev.malloc(4 * M * N)
    dev.gemm_f8(M, N, K, bufs[0], lda, bufs[2], kb, bufs[1], ldb, bufs[3], kb, out, bc, N)
    got = values(out, bc.download(np.float32 if out == "f32" else np.uint16, (M, N)))
    want, mag, largest = ot.gemm_f8(a, sa, b, sb)
    tol = (128 + kb) * 2.0 ** -23 * mag + (7 * 2.0 ** -13 * largest + 2.0 ** -8 * 1.01 * np.abs(want) if out != "f32" else 2.0 ** -24 * np.abs(want))
    assert (np.abs(got - want) <= tol + 1e-37).all()
    for x in bufs + [bc]:
        x.free()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("M,N,K", [(3, 70, 272), (200, 300, 272), (200, 300, 271), (2048, 520, 128)])
def test_gemm_activation_is_the_element_wise_one(dev, kind, M, N, K):
    """f32 results under an activation are, bit for bit, the plain results that the element-wise activation then runs over: few rows, tiles,
    and operands off 16 bytes; sums from 0 to far where both saturate."""
    rng = np.random.RandomState(M + kind)
    a, b = (ot.e4m3_encode(np.clip(rng.randn(r, K) * 60, -448, 448)) for r in (M, N))
    kb = -(-K // 128)
    sa = (np.exp(3 * rng.randn(M, kb)) / 6000).astype(np.float32)
    bufs = [dev.upload(v) for v in (a, b, sa, np.full((-(-N // 128), kb), 1 / 60, np.float32), rng.randn(N).astype(np.float32))]
    plain, fused = dev.malloc(4 * M * N), dev.malloc(4 * M * N)
    for c, k in ((plain, -1), (fused, kind)):
        dev.gemm_f8(M, N, K, bufs[0], K, bufs[2], kb, bufs[1], K, bufs[3], kb, "f32", c, N, bufs[4], k)
    assert dev.lib.wk_activation(dev.stream, 8, kind, (ctypes.c_uint64 * 3)(1, M, N), plain.ptr, N, M * N) == 0
    assert np.array_equal(fused.download(np.uint32, (M, N)), plain.download(np.uint32, (M, N)))
    for x in bufs + [plain, fused]:
        x.free()


@pytest.mark.parametrize("shift", [1, 4, 8])
def test_gemm_unaligned_bases(dev, shift):
    check_gemm(dev, 40, 150, 256, shift=shift)


@pytest.mark.parametrize("M,N,K", [(4, 64, 300), (130, 140, 300)])
def test_gemm_every_code(dev, M, N, K):
    """All finite codes, denormal ones and both zeros among them."""
    check_gemm(dev, M, N, K, pads=(4, 4, 0), codes=lambda rng, r, k: np.array([c for c in range(256) if c & 0x7F != 0x7F], np.uint8)[rng.randint(0, 254, (r, k))])


def test_gemm_nan_codes_stay_in_their_row_and_column(dev):
    M, N, K = 70, 80, 200
    one = int(ot.e4m3_encode(np.ones(1))[0])
    a, b = np.full((M, 208), one, np.uint8), np.full((N, 208), one, np.uint8)
    a[5, 199], b[77, 0] = 0x7F, 0xFF
    ba, bb = dev.upload(a), dev.upload(b)
    bsa, bsb, bc = dev.upload(np.ones((M, 2), np.float32)), dev.upload(np.ones((1, 2), np.float32)), dev.malloc(4 * M * N)
    dev.gemm_f8(M, N, K, ba, 208, bsa, 2, bb, 208, bsb, 2, "f32", bc, N)
    got = bc.download(np.float32, (M, N))
    hit = np.zeros((M, N), bool)
    hit[5], hit[:, 77] = True, True
    assert np.isnan(got[hit]).all() and (got[~hit] == K).all()
    for x in (ba, bb, bsa, bsb, bc):
        x.free()


def test_gemm_refusals(dev):
    lib, b = dev.lib, dev.malloc(1 << 16)
    p = b.ptr.value
    good = dict(M=8, N=8, K=32, A=p, lda=32, sa=p, sap=1, B=p, ldb=32, sb=p, sbp=1, out=8, C=p + 8192, ldc=8, bias=None, kind=-1)

    def call(stream=dev.stream, **change):
        return lib.wk_gemm_f8(stream, *{**good, **change}.values())
    assert call() == 0
    for bad in ({"M": 0}, {"N": 0}, {"K": 0}, {"A": None}, {"B": None}, {"C": None}, {"sa": None}, {"sb": None}, {"lda": 31}, {"ldb": 31}, {"ldc": 7},
                {"K": 129, "lda": 129, "ldb": 129, "sbp": 2}, {"K": 129, "lda": 129, "ldb": 129, "sap": 2}, {"kind": 2}, {"kind": -2}, {"M": 1 << 31}):
        assert call(**bad) == 1, bad
    assert call(stream=None) == 1
    for out in (9, 4, 34, 20, -1):
        assert call(out=out) == 9
    q = dict(dtype=8, rows=2, cols=8, x=p, pitch=8, block_rows=1, q=p + 8192, q_pitch=8, scales=p + 16384, scale_pitch=1)

    def quant(stream=dev.stream, **change):
        return lib.wk_f8_quantize(stream, *{**q, **change}.values())
    assert quant() == 0
    for bad in ({"rows": 0}, {"cols": 0}, {"x": None}, {"q": None}, {"scales": None}, {"block_rows": 0}, {"block_rows": 64}, {"pitch": 7}, {"q_pitch": 7},
                {"cols": 129, "pitch": 129, "q_pitch": 129}):
        assert quant(**bad) == 1, bad
    assert quant(stream=None) == 1
    for dtype in (9, 0, 34, 20):
        assert quant(dtype=dtype) == 9
    dev.sync()
    b.free()


def test_other_entry_points_refuse_the_new_formats(dev):
    from wekua_amd import _capi
    import ctypes
    lib, b = _capi.load(), dev.malloc(4096)
    s3 = (ctypes.c_uint64 * 3)(1, 4, 4)
    for dt in (32, 33, 34):
        assert lib.wk_gemm(dev.stream, dt, 0, 0, 4, 4, 4, None, b.ptr, 4, b.ptr, 4, None, b.ptr, 4, None, 0) == 9
        assert lib.wk_axpy(dev.stream, dt, s3, b.ptr, 4, 16, b.ptr.value + 2048, 4, 16, None) == 9
        assert lib.wk_fill(dev.stream, dt, b.ptr, s3, 4, 16, b.ptr.value and ctypes.create_string_buffer(16)) == 9
        assert lib.wk_activation(dev.stream, dt, 0, s3, b.ptr, 4, 16) == 9
        assert lib.wk_random_uniform(dev.stream, dt, s3, b.ptr, 4, 16, 1, None, None) == 9
        assert lib.wk_sum_workspace_bytes(dt) >= 0 and lib.wk_gemm_workspace_bytes(dt, 0, 0, 64, 64, 64) == 0
    dev.sync()
    b.free()
