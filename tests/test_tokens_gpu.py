"""GPU: wk_token_logprobs and its gradient against their definitions (oracle/tokens.py) through the C ABI.

Tolerances (u = 2^-24, for f64 logits 2^-53; d = x - max; E1 = sum p|d|, E2 = sum p d^2 of the row, L = vocab / 64 + 64, which
is more than the additions that any element's term goes through).  Everything is computed in f32 (f64):
  d is rounded once; e^d is off by 2 u |d| (its argument: d and the product with log2 e) and 4 u (the instruction)
  S: relative u (2 E1 + 4 + L) =: rs;  ln S: rs + 2 u |ln S|
  logprob: u |d_t| + that + u |result|;  lse: that + u |result|
  U / S: u (2 E2 + 4 E1 + 2 E1 + L E1) + rs E1;  entropy: both, and u |result|
  gradient: p off by u (2 |d| + 6) p with d = x - lse, hence the terms by that times |w| and |h (d + H)|, 4 u of each
  term's size, and half a step of the logits' type
"""
import ctypes

import numpy as np
import pytest

from oracle import tokens as ot
from wekua_amd import raw

pytestmark = pytest.mark.gpu

HALF_STEP = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def pack(dtype, x):
    return ot.bf16_bits(x) if dtype == "bf16" else x.astype(raw.real_np_dtype(dtype))


def values(dtype, bits):
    return (ot.bf16_values(bits) if dtype == "bf16" else bits).astype(np.float64)


def pitched(a, pitch, gap):
    out = np.full((a.shape[0], pitch), gap, dtype=a.dtype)
    out[:, :a.shape[1]] = a
    return out


def same_where_not_finite(got, want):
    bad = ~np.isfinite(want)
    return np.array_equal(got[bad], want[bad], equal_nan=True) and np.isfinite(got[~bad]).all()


def run_forward(dev, dtype, bits, targets, top, pad=0, wide=False, workspace=True, outputs=("logprob", "lse", "entropy"), stream_calls=1):
    rows, vocab = bits.shape
    acc = np.float64 if dtype == "f64" else np.float32
    gap = pack(dtype, np.full(1, np.inf))[0]       # around the rows: would show at once
    bx = dev.upload(pitched(bits, vocab + pad, gap))
    bt = dev.upload(targets.astype(np.int64 if wide else np.int32)) if targets is not None else None
    outs = {n: dev.upload(np.full(rows + 1, -7, acc)) for n in outputs}
    ids, lps = dev.upload(np.full(rows * top + 1, -7, np.int32)), dev.upload(np.full(rows * top + 1, -7, acc))
    n = dev.token_logprobs_workspace_bytes(dtype, rows, vocab, top)
    ws = dev.upload(np.full(n + 64, 0xFF, np.uint8)) if workspace and n else None
    for _ in range(stream_calls):
        dev.token_logprobs(dtype, rows, vocab, bx, vocab + pad, bt, "i64" if wide else "i32", outs.get("logprob"), outs.get("lse"),
                           outs.get("entropy"), top, ids if top else None, lps if top else None, ws, n)
    got = {k: v.download(acc, (rows + 1,)) for k, v in outs.items()}
    gi, gl = ids.download(np.int32, (rows * top + 1,)), lps.download(acc, (rows * top + 1,))
    assert all(v[rows] == -7 for v in got.values()) and gi[-1] == -7 and gl[-1] == -7, "wrote behind the last row"
    if ws is not None:
        assert (ws.download(np.uint8, (n + 64,))[n:] == 0xFF).all(), "wrote behind the workspace"
    got = {k: v[:rows] for k, v in got.items()}
    got["top_ids"], got["top_logprobs"] = gi[:-1].reshape(rows, top), gl[:-1].reshape(rows, top)
    for b in [bx, bt, ws, ids, lps, *outs.values()]:
        if b is not None:
            b.free()
    return got


def check_forward(got, dtype, x, targets, top):
    want = ot.token_logprobs(x, targets, top)
    u = 2.0 ** (-53 if dtype == "f64" else -24)
    rows, vocab = x.shape
    long = vocab / 64 + 64
    assert np.array_equal(got["top_ids"], want["top_ids"])
    for r in range(rows):
        if not np.isfinite(want["lse"][r]):
            for name in ("lse", "logprob", "entropy"):
                if name in got:
                    assert np.array_equal(got[name][r], want[name][r], equal_nan=True), (name, r)
            assert np.array_equal(got["top_logprobs"][r], want["top_logprobs"][r], equal_nan=True)
            continue
        m = x[r].max()
        d = x[r] - m
        p = np.exp(x[r] - want["lse"][r])
        live = p > 0
        e1, e2 = (p[live] * np.abs(d[live])).sum(), (p[live] * d[live] ** 2).sum()
        log_s = want["lse"][r] - m
        rs = u * (2 * e1 + 4 + long)
        tol_log = rs + 2 * u * abs(log_s)
        if "lse" in got:
            assert abs(got["lse"][r] - want["lse"][r]) <= tol_log + 2 * u * abs(want["lse"][r]), ("lse", r)
        if "entropy" in got:
            tol = tol_log + u * (2 * e2 + 6 * e1 + long * e1) + rs * e1 + 2 * u * abs(want["entropy"][r])
            assert abs(got["entropy"][r] - want["entropy"][r]) <= tol, ("entropy", r)
        tops = [(got["top_logprobs"][r, k], want["top_logprobs"][r, k]) for k in range(top)]
        if "logprob" in got:
            tops.append((got["logprob"][r], want["logprob"][r]))
        for g, w in tops:
            if np.isfinite(w):
                assert abs(g - w) <= u * (abs(w) + log_s) + tol_log + 2 * u * abs(w), r
            else:
                assert np.array_equal(g, w, equal_nan=True), r


def logits(rng, rows, vocab, spread=3.0):
    return rng.randn(rows, vocab) * spread


@pytest.mark.parametrize("dtype", ["f32", "f64", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,pad,top", [
    (1, 1, 0, 1), (1, 2, 0, 2), (3, 7, 1, 3), (5, 64, 0, 64), (9, 65, 3, 5), (4, 257, 0, 0), (6, 1000, 8, 20), (2, 1024, 0, 64), (3, 1025, 1, 1),
    (2, 4099, 5, 64), (3, 20011, 0, 5), (1, 70001, 0, 20), (2, 66000, 8, 64), (300, 130, 0, 2), (1, 262144, 0, 7),
])
def test_forward(dev, dtype, rows, vocab, pad, top):
    rng = np.random.RandomState(rows * 7 + vocab)
    bits = pack(dtype, logits(rng, rows, vocab))
    targets = rng.randint(0, vocab, rows)
    targets[0] = vocab - 1
    x = values(dtype, bits)
    first = run_forward(dev, dtype, bits, targets, top, pad, stream_calls=2)
    check_forward(first, dtype, x, targets, top)
    # without a workspace rows are not cut: other sums, the same alternatives
    check_forward(run_forward(dev, dtype, bits, targets, top, pad, wide=True, workspace=False), dtype, x, targets, top)


@pytest.mark.parametrize("dtype", ["f32", "f64", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [3, 130, 1500, 40000])
def test_masks_and_bad_values(dev, dtype, vocab):
    rng = np.random.RandomState(vocab)
    x = logits(rng, 12, vocab)
    low = {"f32": -3.4e38, "f64": -1.7e308, "f16": -65504.0, "bf16": -3.38e38}[dtype]
    x[0] = -np.inf                                    # empty
    x[1, :-1] = -np.inf                               # one left, the last
    x[2, rng.rand(vocab) < 0.9] = -np.inf
    x[2, 0] = 0.5
    x[3, rng.rand(vocab) < 0.9] = low                 # masks of the type's lowest value
    x[3, 0] = 0.5
    x[4] = low                                        # nothing but those
    x[5, vocab // 2] = np.nan
    x[6, vocab - 1] = np.inf
    x[7] = 0.25                                       # all equal: ids by index
    x[8] = np.where(np.arange(vocab) % 2, 1.0, 2.0)   # ties
    x[9] = -np.inf
    x[9, 1] = np.nan
    x[10, :] = 80 + 5 * np.sign(x[10])                # large
    bits = pack(dtype, x)
    targets = np.array([0, vocab - 1, 0, 0, 1, 0, 0, vocab - 1, 1, 0, 2, vocab])
    for top in (0, 3):
        for ws in (True, False):
            check_forward(run_forward(dev, dtype, bits, targets, top, 1, workspace=ws), dtype, values(dtype, bits), targets, top)
    targets[:] = [-1, -100, vocab, 2 ** 31 - 1, -2 ** 31, -1, vocab, -1, 0, 0, 0, 0]
    check_forward(run_forward(dev, dtype, bits, targets, 1), dtype, values(dtype, bits), targets, 1)


def test_ties_across_the_whole_row(dev):
    """Sixty-four alternatives of a row with few distinct values, ascending and descending: always the lowest indexes."""
    vocab = 50000
    x = np.stack([np.arange(vocab) // 1000, -(np.arange(vocab) // 1000), np.arange(vocab) % 7, np.zeros(vocab), np.arange(vocab) / 64]).astype(np.float64)
    for dtype in ("f32", "bf16", "f64"):
        bits = pack(dtype, x)
        for ws in (True, False):
            got = run_forward(dev, dtype, bits, None, 64, outputs=("lse",), workspace=ws)
            assert np.array_equal(got["top_ids"], ot.token_logprobs(values(dtype, bits), None, 64)["top_ids"])


@pytest.mark.parametrize("dtype,rows,vocab,top", [("bf16", 2100, 33001, 5), ("f32", 1050, 33003, 64), ("f32", 600, 60001, 20), ("f64", 40, 430001, 7)])
def test_logits_that_pass_the_cache_by(dev, dtype, rows, vocab, top):
    """More than 128 MB of logits with alternatives, rows whole and cut: thirty rows in turn, of which the copies have the same bits."""
    rng = np.random.RandomState(rows)
    block = pack(dtype, logits(rng, 30, vocab))
    if dtype != "bf16":
        block[3, rng.rand(vocab) < 0.9] = -np.inf
    t = rng.randint(0, vocab, 30)
    bits, targets = np.resize(block, (rows, vocab)), np.resize(t, rows)
    assert bits.nbytes > 128 << 20
    got = run_forward(dev, dtype, bits, targets, top, 1)
    check_forward({n: v[:30] for n, v in got.items()}, dtype, values(dtype, block), t, top)
    for v in got.values():
        assert np.array_equal(v, np.resize(v[:30], v.shape), equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 131072, 20), (3, 20011, 0), (2, 9001, 64)])
def test_a_workspace_that_is_too_small(dev, dtype, rows, vocab, top):
    """Less than the call asks for is as good as none: the same bits, and nothing is written there."""
    rng = np.random.RandomState(rows)
    acc = np.float64 if dtype == "f64" else np.float32
    bits, t = pack(dtype, logits(rng, rows, vocab)), rng.randint(0, vocab, rows).astype(np.int32)
    n = dev.token_logprobs_workspace_bytes(dtype, rows, vocab, top)
    assert n
    bx, bt, ws = dev.upload(bits), dev.upload(t), dev.upload(np.full(n, 0xFF, np.uint8))
    stats, ids, lps = [dev.malloc(rows * acc().itemsize) for _ in range(3)], dev.malloc(4 * rows * top + 4), dev.malloc(8 * rows * top + 8)
    seen = []
    for space, size in ((None, 0), (ws, 0), (ws, 16), (ws, n - 1)):
        dev.token_logprobs(dtype, rows, vocab, bx, vocab, bt, "i32", *stats, top, ids if top else None, lps if top else None, space, size)
        seen.append([b.download(acc, (rows,)) for b in stats] + ([ids.download(np.int32, (rows, top)), lps.download(acc, (rows, top))] if top else []))
    for other in seen[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(seen[0], other))
    assert (ws.download(np.uint8, (n,)) == 0xFF).all()
    got = dict(zip(("logprob", "lse", "entropy"), seen[0][:3]), top_ids=seen[0][3] if top else np.zeros((rows, 0), np.int32),
               top_logprobs=seen[0][4] if top else np.zeros((rows, 0), acc))
    check_forward(got, dtype, values(dtype, bits), t, top)
    for b in (bx, bt, ws, ids, lps, *stats):
        b.free()


@pytest.mark.parametrize("outputs", [("logprob",), ("lse",), ("entropy",), ("logprob", "entropy"), ()])
def test_only_what_is_wanted(dev, outputs):
    rng = np.random.RandomState(8)
    x = logits(rng, 5, 300).astype(np.float32)
    t = rng.randint(0, 300, 5)
    top = 0 if outputs else 4
    check_forward(run_forward(dev, "f32", x, t if "logprob" in outputs else None, top, outputs=outputs), "f32", x.astype(np.float64), t, top)


@pytest.mark.parametrize("dtype", ["f32", "f64", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 2, 0), (5, 63, 1), (4, 257, 0), (7, 1000, 8), (2, 4099, 5), (3, 20011, 0)])
@pytest.mark.parametrize("terms", ["w", "h", "wh"])
def test_gradient(dev, dtype, rows, vocab, pad, terms):
    rng = np.random.RandomState(rows + vocab)
    acc = np.float64 if dtype == "f64" else np.float32
    x = logits(rng, rows, vocab)
    if vocab > 60:
        x[0, rng.rand(vocab) < 0.5] = -np.inf
        x[1, :] = -np.inf                              # empty
    bits = pack(dtype, x)
    xv = values(dtype, bits)
    targets = rng.randint(0, vocab, rows)
    if rows > 2:
        targets[2] = -1
    if rows > 4:
        targets[4] = vocab                             # not a token
    if vocab > 60:
        targets[0] = int(np.argmin(xv[0]))             # a masked one
    o = ot.token_logprobs(xv, targets)
    lse, ent = o["lse"].astype(acc), o["entropy"].astype(acc)
    w = rng.randn(rows).astype(acc) if "w" in terms else None
    h = rng.randn(rows).astype(acc) if "h" in terms else None
    up = {k: dev.upload(v) for k, v in (("lse", lse), ("ent", ent), ("w", w), ("h", h)) if v is not None}
    bt = dev.upload(targets.astype(np.int32))
    poison = pack(dtype, np.full(1, -7.0))[0]
    bx, bg = dev.upload(pitched(bits, vocab + pad, poison)), dev.upload(np.full((rows, vocab + pad + 2), poison))
    args = (bt if w is not None else None, "i32", up["lse"], up["ent"] if h is not None else None, up.get("w"), up.get("h"))
    dev.token_logprobs_grad(dtype, rows, vocab, bx, vocab + pad, *args, bg, vocab + pad + 2)
    got = bg.download(poison.dtype, (rows, vocab + pad + 2))
    assert (got[:, vocab:] == poison).all(), "wrote outside the rows"
    got = values(dtype, got[:, :vocab])
    want = ot.token_logprobs_grad(xv, targets, lse.astype(np.float64), ent.astype(np.float64), w, h)
    u = 2.0 ** (-53 if dtype == "f64" else -24)
    assert same_where_not_finite(got, want)
    with np.errstate(all="ignore"):
        d = xv - lse.astype(np.float64)[:, None]
        p = np.nan_to_num(np.exp(d))                   # a row without a distribution: exactly zeros
        dh = np.where(p > 0, np.abs(d + ent.astype(np.float64)[:, None]), 0)
        terms_size = (np.abs(w)[:, None] if w is not None else 0) * p + (np.abs(h)[:, None] if h is not None else 0) * p * dh
        tol = u * (2 * np.where(p > 0, np.abs(d), 0) + 10) * terms_size + (np.abs(h)[:, None] * p * u * (np.where(p > 0, np.abs(d), 0) + dh) if h is not None else 0)
        tol += (HALF_STEP[dtype] + 2 * u) * np.abs(want) + 2 * u * (np.abs(w)[:, None] if w is not None else 0) * (np.arange(vocab) == targets[:, None])
        tol += {"f16": 2.0 ** -25, "f64": 1e-300}.get(dtype, 1e-37)
    fine = np.isfinite(want)
    assert (np.abs(got - want)[fine] <= tol[fine]).all()
    # in place
    dev.token_logprobs_grad(dtype, rows, vocab, bx, vocab + pad, *args, bx, vocab + pad)
    back = bx.download(poison.dtype, (rows, vocab + pad))
    assert (back[:, vocab:] == poison).all() and np.array_equal(values(dtype, back[:, :vocab]), got, equal_nan=True)
    for b in (bx, bg, bt, *up.values()):
        b.free()


@pytest.mark.parametrize("dtype", ["f32", "f64", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [5, 300, 9001])
def test_gradient_of_empty_rows_and_no_tokens(dev, dtype, vocab):
    """Rows that their mask leaves empty, whose target is a token, none, and not below vocab: zeros, zeros, NaN with a gradient of the
    log probability, and always zeros without one; what forward answers for them beside it."""
    acc = np.float64 if dtype == "f64" else np.float32
    x = np.full((4, vocab), -np.inf)
    targets = np.array([vocab - 1, -1, vocab, 2 ** 31 - 1])
    bits = pack(dtype, x)
    o = run_forward(dev, dtype, bits, targets, 0)
    assert (o["lse"] == -np.inf).all() and (o["entropy"] == 0).all() and np.array_equal(o["logprob"], [-np.inf, 0, np.nan, np.nan], equal_nan=True)
    up = [dev.upload(v) for v in (bits, targets.astype(np.int32), o["lse"], o["entropy"], np.array([np.nan, 3, 0, -1], acc), np.ones(4, acc))]
    bg = dev.malloc(bits.nbytes)
    for w, h in ((up[4], None), (up[4], up[5]), (None, up[5])):
        dev.token_logprobs_grad(dtype, 4, vocab, up[0], vocab, up[1], "i32", up[2], up[3], w, h, bg, vocab)
        got = values(dtype, bg.download(bits.dtype, bits.shape))
        want = ot.token_logprobs_grad(x, targets, o["lse"], o["entropy"], None if w is None else np.array([np.nan, 3, 0, -1]), None if h is None else np.ones(4))
        assert (got[:2] == 0).all() and (np.isnan(got[2:]).all() if w else (got[2:] == 0).all()) and np.array_equal(got, want, equal_nan=True)
    for b in up + [bg]:
        b.free()


def test_gradient_of_the_kernels_own_statistics_against_differences(dev):
    """f64 logits: the gradient from the forward call's lse and entropy against central differences of the forward call."""
    rng = np.random.RandomState(21)
    rows, vocab, step = 4, 37, 1e-6
    x = logits(rng, rows, vocab, 1.5)
    t, w, h = rng.randint(0, vocab, rows), rng.randn(rows), rng.randn(rows)

    def value(z):
        o = run_forward(dev, "f64", z, t, 0)
        return w * o["logprob"] + h * o["entropy"]
    o = run_forward(dev, "f64", x, t, 0)
    up = [dev.upload(v) for v in (x, t.astype(np.int32), o["lse"], o["entropy"], w, h)]
    bg = dev.malloc(8 * rows * vocab)
    dev.token_logprobs_grad("f64", rows, vocab, up[0], vocab, up[1], "i32", up[2], up[3], up[4], up[5], bg, vocab)
    got = bg.download(np.float64, (rows, vocab))
    for j in range(vocab):
        a, b = x.copy(), x.copy()
        a[:, j] += step
        b[:, j] -= step
        # differences: third derivatives (under 10) * step^2, and 2^-53 of the values (under 20) / step
        assert np.abs((value(a) - value(b)) / (2 * step) - got[:, j]).max() < 10 * step ** 2 + 20 * 2.0 ** -52 * 40 / step
    for b in up + [bg]:
        b.free()


def test_refusals(dev):
    lib, b = dev.lib, dev.malloc(1 << 16)
    p = b.ptr.value
    base = dict(dtype=8, rows=2, vocab=8, x=p, pitch=8, t=p + 1024, tt=4, lp=p + 2048, lse=p + 3200, ent=p + 4096, top=2, ids=p + 5120, tl=p + 6144,
                ws=None, n=0)

    def call(stream=dev.stream, **change):
        return lib.wk_token_logprobs(stream, *{**base, **change}.values())
    assert call() == 0 and call(top=0, ids=None, tl=None) == 0 and call(lp=None, t=None) == 0
    for bad in ({"rows": 0}, {"vocab": 0}, {"x": None}, {"pitch": 7}, {"t": None}, {"top": 9}, {"top": 65, "vocab": 100, "pitch": 100}, {"ids": None}, {"tl": None},
                {"lp": None, "lse": None, "ent": None, "top": 0}, {"ws": p + 8}, {"vocab": 1 << 31, "pitch": 1 << 31}):
        assert call(**bad) == 1, bad
    assert call(stream=None) == 1
    for bad in ({"dtype": 4}, {"dtype": 34}, {"dtype": 18}, {"dtype": 20}, {"tt": 5}, {"tt": 8}):
        assert call(**bad) == 9, bad
    g = dict(dtype=8, rows=2, vocab=8, x=p, pitch=8, t=p + 1024, tt=4, lse=p + 2048, ent=p + 3200, w=p + 4096, h=p + 5120, g=p + 6144, gp=8)

    def grad(stream=dev.stream, **change):
        return lib.wk_token_logprobs_grad(stream, *{**g, **change}.values())
    assert grad() == 0 and grad(w=None, t=None) == 0 and grad(h=None, ent=None) == 0
    for bad in ({"rows": 0}, {"vocab": 0}, {"x": None}, {"lse": None}, {"g": None}, {"w": None, "h": None}, {"t": None}, {"ent": None}, {"pitch": 7}, {"gp": 7},
                {"g": p, "gp": 9}):
        assert grad(**bad) == 1, bad
    assert grad(stream=None) == 1
    for bad in ({"dtype": 4}, {"dtype": 33 + 1}, {"tt": 5}):
        assert grad(**bad) == 9, bad
    assert lib.wk_token_logprobs_workspace_bytes(8, 0, 8, 0) == 0 and lib.wk_token_logprobs_workspace_bytes(8, 1, 1 << 17, 65) == 0
    assert lib.wk_token_logprobs_workspace_bytes(4, 1, 1 << 17, 5) == 0 and lib.wk_token_logprobs_workspace_bytes(8, 1, 1 << 17, 5) > 0
    dev.sync()
    b.free()
