"""CPU restatement (numpy, 64 bits) of the operators at the token end of a network: dropout, the 8-bit quantiser and the
block-scaled product, token log probabilities and their gradient.

TEST INFRASTRUCTURE ONLY, like the rest of this package.  The reference has none of these operators: each function
is the definition that include/wekua_hip.h gives, pinned in tests/test_oracle_tokens.py (the generator and
the 8-bit format against published values and torch's type, the gradient against differences).
"""
from __future__ import annotations

import math

import numpy as np

E4M3_MAX = 448.0
BLOCK = 128


# ---- 16-bit types -----------------------------------------------------------------------------------------------------

def bf16_bits(x):
    """float array -> bfloat16 bits (uint16), to nearest, ties to even."""
    u = np.asarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    out = ((u + 0x7FFF + ((u >> np.uint64(16)) & np.uint64(1))) >> np.uint64(16)).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, dtype=np.float32)), np.uint16(0x7FC0), out)


def bf16_values(bits):
    return (np.asarray(bits, dtype=np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


# ---- dropout --------------------------------------------------------------------------------------------------------------

def philox4x32(counter, key, rounds):
    """The four words of Philox4x32 for counters [n, 4] under one key (two words), as the paper writes the round."""
    m0, m1, low = 0xD2511F53, 0xCD9E8D57, 0xFFFFFFFF
    out = []
    for c in np.asarray(counter, dtype=np.uint64).reshape(-1, 4).tolist():
        k = [int(key[0]), int(key[1])]
        for _ in range(rounds):
            a, b = m0 * c[0], m1 * c[2]
            c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        out.append(c)
    return np.array(out, dtype=np.uint64)


def dropout_keep(n, p, seed, count):
    """Which of n elements stay."""
    blocks = (n + 3) // 4
    ctr = [[b & 0xFFFFFFFF, b >> 32, count & 0xFFFFFFFF, count >> 32] for b in range(blocks)]
    words = philox4x32(ctr, (seed & 0xFFFFFFFF, seed >> 32), 7).reshape(-1)[:n]
    return words >= np.uint64(math.floor(p * 2 ** 32))


def dropout(x, p, seed, count):
    """x: float64 values of the logical region."""
    keep = dropout_keep(x.size, p, seed, count).reshape(x.shape)
    with np.errstate(all="ignore"):
        return np.where(keep, x / (1 - p) if p < 1 else 0.0, 0.0)


# ---- 8-bit format ---------------------------------------------------------------------------------------------------------

def e4m3_values():
    """The 256 values: sign, four exponent bits (bias 7), three fraction bits; the code with all of them set is NaN."""
    out = np.empty(256)
    for code in range(256):
        e, f = (code >> 3) & 15, code & 7
        v = math.nan if (code & 0x7F) == 0x7F else f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        out[code] = -v if code & 0x80 else v
    return out


E4M3 = e4m3_values()


def e4m3_encode(x):
    """Nearest code of float64 values within +-448, ties to the even code; NaN to 0x7F."""
    x = np.asarray(x, dtype=np.float64)
    grid = E4M3[:0x7F]                                  # 0 .. 448 ascending
    a = np.abs(x)
    hi = np.clip(np.searchsorted(grid, a, side="left"), 0, 0x7E)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - grid[lo], grid[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = code | np.where(np.signbit(x), 0x80, 0).astype(np.uint8)
    return np.where(np.isnan(x), np.uint8(0x7F), code).astype(np.uint8)


def f8_quantize(x, block_rows):
    """(codes, scales) of float64 values."""
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    codes, scales = np.zeros((rows, cols), np.uint8), np.zeros((rb, cb), np.float32)
    for i in range(rb):
        for j in range(cb):
            at = np.s_[i * block_rows:(i + 1) * block_rows, j * BLOCK:(j + 1) * BLOCK]
            b = x[at]
            amax = np.abs(b).max()
            if not np.isfinite(amax):
                scales[i, j], codes[at] = np.nan, 0x7F
                continue
            e = 0 if amax == 0 else -126
            while amax > E4M3_MAX * 2.0 ** e:
                e += 1
            scales[i, j] = 2.0 ** e
            codes[at] = e4m3_encode(b / 2.0 ** e)
    return codes, scales


def _f8_operand(codes, scales, scale_rows):
    k = codes.shape[1]
    s = np.repeat(np.repeat(scales.astype(np.float64), scale_rows, 0)[:codes.shape[0]], BLOCK, 1)[:, :k]
    return E4M3[codes] * s


def gemm_f8(a, sa, b, sb, bias=None, kind=-1, cut=True):
    """(C, the sum of the products' magnitudes, and that of the largest of each eight consecutive products, or, with
    cut=False, a bound of it that is had faster)."""
    x, w = _f8_operand(a, sa, 1), _f8_operand(b, sb, BLOCK)
    largest = np.zeros((x.shape[0], w.shape[0]))
    for k in range(0, x.shape[1], 8) if cut else ():
        group = np.zeros_like(largest)
        for e in range(k, min(k + 8, x.shape[1])):
            np.maximum(group, np.abs(x[:, e])[:, None] * np.abs(w[:, e]), out=group)
        largest += group
    y = x @ w.T
    if bias is not None:
        y = y + bias.astype(np.float64)
    if kind == 0:
        y = 1 / (1 + np.exp(-y))
    elif kind == 1:
        y = np.tanh(y)
    mag = np.abs(x) @ np.abs(w).T
    return y, mag, largest if cut else mag


# ---- token log probabilities ------------------------------------------------------------------------------------------------

def token_logprobs(x, targets=None, top=0):
    """x: float64 logits [rows, vocab].  A dict with lse, logprob, entropy, top_ids, top_logprobs, and p and d = x - max."""
    rows, vocab = x.shape
    out = {"lse": np.empty(rows), "logprob": np.zeros(rows), "entropy": np.empty(rows), "top_ids": np.full((rows, top), -1, np.int32),
           "top_logprobs": np.full((rows, top), -np.inf)}
    for r in range(rows):
        z = x[r]
        m = z.max()
        t = None if targets is None else int(targets[r])
        if not (m < np.inf):                            # a NaN or +inf
            out["lse"][r] = out["entropy"][r] = np.nan
            out["logprob"][r] = np.nan
            out["top_logprobs"][r] = np.nan
            continue
        if m == -np.inf:
            out["lse"][r], out["entropy"][r] = -np.inf, 0.0
            out["logprob"][r] = 0.0 if t is None or t < 0 else np.nan if t >= vocab else -np.inf
            continue
        d = z - m
        e = np.exp(d)
        s = math.fsum(e)
        out["lse"][r] = m + math.log(s)
        live = e > 0
        out["entropy"][r] = math.log(s) - math.fsum(e[live] * d[live]) / s
        if t is not None and t >= 0:
            out["logprob"][r] = np.nan if t >= vocab else d[t] - math.log(s)
        order = np.argsort(-z, kind="stable")[:top]
        order = order[z[order] > -np.inf]
        out["top_ids"][r, :len(order)] = order
        out["top_logprobs"][r, :len(order)] = d[order] - math.log(s)
    return out


def token_logprobs_grad(x, targets, lse, entropy, w, h):
    """w, h: gradients of the log probabilities and entropies (None: absent); the statistics as they were given."""
    rows, vocab = x.shape
    out = np.zeros((rows, vocab))
    for r in range(rows):
        if lse[r] == -np.inf and (w is None or targets[r] < vocab):
            continue
        with np.errstate(all="ignore"):
            d = x[r] - lse[r]
            p = np.exp(d)
            if w is not None and targets[r] >= 0:
                out[r] -= (w[r] if targets[r] < vocab else np.nan) * p
                if targets[r] < vocab:
                    out[r, targets[r]] += w[r]
            if h is not None:
                out[r] -= h[r] * np.where(p == 0, 0.0, p * (d + entropy[r]))
    return out
