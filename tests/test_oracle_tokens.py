"""CPU: the restatements in oracle/tokens.py against published values, torch's 8-bit type and differences."""
import numpy as np
import pytest

from oracle import tokens as ot


def test_philox_known_answers():
    """The generator's published known answers (Random123 kat_vectors, philox 4x32, 7 and 10 rounds)."""
    ff = [0xFFFFFFFF] * 4
    got = [ot.philox4x32([0, 0, 0, 0], (0, 0), 7)[0], ot.philox4x32([0, 0, 0, 0], (0, 0), 10)[0], ot.philox4x32(ff, ff[:2], 10)[0]]
    want = [[0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48], [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8],
            [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]]
    assert [list(map(int, g)) for g in got] == want


def test_dropout_keeps_about_the_share():
    n = 40000
    for p in (0.1, 0.5, 0.9):
        kept = ot.dropout_keep(n, p, 77, 3).sum()
        assert abs(kept - n * (1 - p)) < 6 * np.sqrt(n * p * (1 - p))
    assert ot.dropout_keep(9, 0.0, 1, 0).all() and not ot.dropout_keep(9, 1.0, 1, 0).any()


def test_e4m3_is_torchs_float8_e4m3fn():
    torch = pytest.importorskip("torch")
    codes = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).float().numpy().astype(np.float64), ot.E4M3, equal_nan=True)
    x = np.concatenate([np.linspace(-448, 448, 20001), np.linspace(-0.05, 0.05, 5001), (ot.E4M3[:0x7E] + ot.E4M3[1:0x7F]) / 2]).astype(np.float32)
    assert np.array_equal(torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), ot.e4m3_encode(x.astype(np.float64)))


def test_bf16_is_torchs():
    torch = pytest.importorskip("torch")
    x = np.random.RandomState(1).randn(5000).astype(np.float32) * 1e3
    assert np.array_equal(torch.from_numpy(x).bfloat16().view(torch.int16).numpy().view(np.uint16), ot.bf16_bits(x))
    assert np.array_equal(ot.bf16_values(ot.bf16_bits(x)), torch.from_numpy(x).bfloat16().float().numpy())


def test_quantize_scale_is_the_least_power_of_two():
    for amax, want in ((448.0, 1.0), (448.001, 2.0), (224.0, 0.5), (1e-30, None), (0.0, 1.0), (2.0 ** -140, 2.0 ** -126)):
        x = np.zeros((1, 5))
        x[0, 3] = -amax
        codes, scales = ot.f8_quantize(x, 1)
        s = float(scales[0, 0])
        assert want is None or s == want
        assert amax <= 448 * s and (s == 2.0 ** -126 or amax == 0 or amax > 224 * s)
        assert abs(ot.E4M3[codes[0, 3]] * s + amax) <= max(amax * 2.0 ** -4, s * 2.0 ** -10)


def test_gradient_against_differences():
    rng = np.random.RandomState(4)
    x, t, w, h = rng.randn(3, 11), np.array([4, -1, 10]), rng.randn(3), rng.randn(3)
    x[1, 2] = -np.inf

    def value(z):
        o = ot.token_logprobs(z, t)
        return (w * o["logprob"] + h * o["entropy"]).sum()
    o = ot.token_logprobs(x, t)
    g = ot.token_logprobs_grad(x, t, o["lse"], o["entropy"], w, h)
    step = 1e-5
    for r in range(3):
        for j in range(11):
            if np.isinf(x[r, j]):
                assert g[r, j] == 0
                continue
            a, b = x.copy(), x.copy()
            a[r, j] += step
            b[r, j] -= step
            assert abs((value(a) - value(b)) / (2 * step) - g[r, j]) < 1e-8


def test_rows_without_a_distribution():
    x = np.array([[-np.inf] * 3, [0, np.nan, 1], [np.inf, 0, 0], [-np.inf, 2, -np.inf]])
    o = ot.token_logprobs(x, np.array([0, 0, 1, 1]), 2)
    assert o["lse"][0] == -np.inf and o["logprob"][0] == -np.inf and o["entropy"][0] == 0 and (o["top_ids"][0] == -1).all()
    assert np.isnan(o["lse"][1:3]).all() and np.isnan(o["top_logprobs"][1:3]).all() and (o["top_ids"][1:3] == -1).all()
    assert o["logprob"][3] == 0 and o["entropy"][3] == 0 and o["top_ids"][3].tolist() == [1, -1]
