"""GPU: the operators at the token end of a network through Tensor, blas, random and nn, alone and as one run: training
(Linear, Dropout, Linear, loss.tokens, backward, an optimiser) and serving (8-bit layer, log probabilities with alternatives).

Tolerances: single operators have theirs in the tests of the C ABI (half a step of the type, and 1e-5 here for f32 statistics of at
most 1000 terms, 1e-12 for f64, both far above vocab * 2^-24 * the few roundings a term goes through); networks in f32 and f64 the
bound of the other network tests, 1e-5 or 1e-12 times sqrt(k) of the largest magnitude.  Differences: central ones of step h in f64
are off by h^2 / 6 of the third derivative and by 2^-53 |loss| / h.
"""
import ctypes

import numpy as np
import pytest

import wekua_amd as wk
from oracle import tokens as ot
from wekua_amd import Context, DeviceType, Pipeline, Tensor, memory, nn
from wekua_amd.raw import real_np_dtype

pytestmark = pytest.mark.gpu

TOL = {"f32": 1e-5, "f64": 1e-12}
STEP = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def env():
    context = Context.initFromDeviceType(DeviceType.all)
    pipeline = Pipeline.init(context.command_queues[0])
    yield context, pipeline
    pipeline.deinit()
    context.deinit()


def pack(dtype, x):
    return ot.bf16_bits(x) if dtype == "bf16" else np.asarray(x).astype(real_np_dtype(dtype))


def values(dtype, bits):
    return (ot.bf16_values(bits) if dtype == "bf16" else bits).astype(np.float64)


def upload(env, dtype, host):
    t = Tensor.alloc(dtype, env[0], env[1], host.shape)
    memory.readFromBuffer(env[1], t, host)
    return t


def download(env, t):
    out = np.empty(t.shape, dtype=real_np_dtype(t.dtype))
    memory.writeToBuffer(env[1], t, out)
    env[1].waitAndCleanup()
    return out


def release(env, *tensors):
    for t in tensors:
        t.release(env[1])


def near(got, want, dtype, k=1):
    assert np.abs(got.astype(np.float64) - want).max() <= TOL[dtype] * np.sqrt(k) * (np.abs(want).max() + 1e-30)


# ---- tensors of the new formats ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "bf16", "f8e4m3"])
@pytest.mark.parametrize("shape", [(1,), (17,), (3, 5), (33, 129), (2, 7, 40)])
def test_storage(env, dtype, shape):
    context, pipeline = env
    rng = np.random.RandomState(len(shape))
    size = real_np_dtype(dtype).itemsize
    host = rng.randint(0, 256, shape + (size,)).astype(np.uint8).view(np.uint8 if size == 1 else np.uint16)[..., 0]
    t = Tensor.alloc(dtype, context, pipeline, shape)
    assert t.shape == shape and t.row_pitch % (16 // size) == 0 and t.size == t.number_of_elements * size
    memory.readFromBuffer(pipeline, t, host.view(real_np_dtype(dtype)))
    other = Tensor.empty(dtype, context, pipeline, shape)
    memory.copy(pipeline, t, other)
    assert np.array_equal(download(env, other).view(host.dtype), host)
    wk.fill.zeroes(pipeline, other)
    assert not download(env, other).view(host.dtype).any()
    if len(shape) > 1:
        turned = Tensor.alloc(dtype, context, pipeline, shape[:-2] + (shape[-1], shape[-2]))
        wk.transpose(pipeline, turned, t, len(shape) - 2, len(shape) - 1)
        assert np.array_equal(download(env, turned).view(host.dtype), host.swapaxes(-1, -2))
        release(env, turned)
    for call in (lambda: wk.fill.one(pipeline, t), lambda: wk.random.uniform(pipeline, t, 1),
                 lambda: wk.blas.axpy(pipeline, t, None, other), lambda: wk.math.dot(pipeline, t, other)):
        with pytest.raises(wk.WekuaError):
            call()
    release(env, t, other)


# ---- the operators alone --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f64", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(5,), (7, 33), (2, 3, 18)])
def test_dropout(env, dtype, shape):
    context, pipeline = env
    n = int(np.prod(shape))
    x = pack(dtype, np.random.RandomState(1).rand(*shape) + 0.5)
    tx, ty, step = upload(env, dtype, x), Tensor.alloc(dtype, context, pipeline, shape), upload(env, "u64", np.array([4], np.uint64))
    wk.random.dropout(pipeline, tx, ty, 0.25, 77, 3, step)
    got, want = values(dtype, download(env, ty)), ot.dropout(values(dtype, x), 0.25, 77, 7)
    assert np.array_equal(got == 0, want == 0) and (np.abs(got - want) <= (STEP[dtype] + 2 * STEP["f64" if dtype == "f64" else "f32"]) * want).all()
    wk.random.dropout(pipeline, tx, tx, 0.25, 77, 7)
    assert np.array_equal(download(env, tx), download(env, ty)) and n
    release(env, tx, ty, step)


def test_dropout_refusals(env):
    context, pipeline = env
    a, b, h = (Tensor.alloc(d, context, pipeline, s) for d, s in (("f32", (3, 4)), ("f32", (4, 3)), ("f16", (3, 4))))
    i, s, c = (Tensor.alloc(d, context, pipeline, (3, 4)) for d in ("i32", "i64", "f8e4m3"))
    for x, y, p, step in ((a, b, .1, None), (a, h, .1, None), (i, i, .1, None), (c, c, .1, None), (a, a, -1, None), (a, a, 2, None), (a, a, .1, s)):
        with pytest.raises(wk.WekuaError):
            wk.random.dropout(pipeline, x, y, p, 1, 0, step)
    release(env, a, b, h, i, s, c)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K,kind", [(1, 5, 9, -1), (19, 130, 300, 1), (200, 260, 520, 0)])
def test_block_scaled_product(env, dtype, M, N, K, kind):
    context, pipeline = env
    rng = np.random.RandomState(M)
    x, w, bias = pack(dtype, rng.randn(M, K)), rng.randn(N, K).astype(np.float32), rng.randn(N).astype(np.float32)
    tx, tw, tb = upload(env, dtype, x), upload(env, "f32", w), upload(env, "f32", bias)
    a, b = wk.blas.BlockScaled.init(context, pipeline, M, K, 1), wk.blas.BlockScaled.init(context, pipeline, N, K, 128)
    a.quantize(pipeline, tx)
    b.quantize(pipeline, tw)
    qa, sa, qb, sb = (download(env, t) for t in (a.codes, a.scales, b.codes, b.scales))
    for got, want in zip((qa, sa, qb, sb), ot.f8_quantize(values(dtype, x), 1) + ot.f8_quantize(w.astype(np.float64), 128)):
        assert np.array_equal(got, want)
    out = "bf16" if dtype == "f32" else "f32"
    c = Tensor.alloc(out, context, pipeline, (M, N))
    for t in (tb, None):
        wk.blas.gemmF8(pipeline, a, b, t, kind, c)
        want, mag, largest = ot.gemm_f8(qa, sa, qb, sb, bias if t is not None else None, kind)
        # f32 results: K roundings of the sums, 8 of the epilogue; others: 7 of each eight products cut at 2^-13 of the largest
        tol = (K + 8) * 2.0 ** -24 * (mag + np.abs(bias)) + 1e-6 * (kind >= 0)
        if out != "f32":
            tol = tol + 7 * 2.0 ** -13 * largest + STEP[out] * np.abs(want)
        assert (np.abs(values(out, download(env, c)) - want) <= tol).all()
    a.deinit(pipeline)
    b.deinit(pipeline)
    release(env, tx, tw, tb, c)


@pytest.mark.parametrize("rows,n,k", [(5, 130, 300), (150, 260, 129)])
def test_product_with_the_weights_turned_around(env, rows, n, k):
    """The gradient of a layer's input: the same codes and scales, transposed, under the quantised gradient of its output."""
    context, pipeline = env
    rng = np.random.RandomState(n)
    w, g = rng.randn(n, k).astype(np.float32), rng.randn(rows, n).astype(np.float32)
    tw, tg, out = upload(env, "f32", w), upload(env, "f32", g), Tensor.alloc("f32", context, pipeline, (rows, k))
    init = wk.blas.BlockScaled.init
    b, turned, a = init(context, pipeline, n, k, 128), init(context, pipeline, k, n, 128), init(context, pipeline, rows, n, 1)
    b.quantize(pipeline, tw)
    a.quantize(pipeline, tg)
    wk.transpose(pipeline, turned.codes, b.codes, 0, 1)
    wk.transpose(pipeline, turned.scales, b.scales, 0, 1)
    wk.blas.gemmF8(pipeline, a, turned, None, -1, out)
    codes, scales = ot.f8_quantize(w.astype(np.float64), 128)
    want, mag, _ = ot.gemm_f8(*ot.f8_quantize(g.astype(np.float64), 1), np.ascontiguousarray(codes.T), np.ascontiguousarray(scales.T))
    assert (np.abs(download(env, out) - want) <= (n + 8) * 2.0 ** -24 * mag).all()
    for m in (a, b, turned):
        m.deinit(pipeline)
    release(env, tw, tg, out)


def test_block_scaled_refusals(env):
    context, pipeline = env
    for rows, cols, block in ((0, 4, 1), (4, 0, 1), (4, 4, 2), (4, 4, 0)):
        with pytest.raises(wk.WekuaError):
            wk.blas.BlockScaled.init(context, pipeline, rows, cols, block)
    a, b, odd = (wk.blas.BlockScaled.init(context, pipeline, r, k, s) for r, k, s in ((3, 64, 1), (5, 64, 128), (5, 65, 128)))
    c, short, i32, f64 = (Tensor.alloc(d, context, pipeline, s) for d, s in
                          (("f32", (3, 5)), ("f32", (3, 4)), ("i32", (3, 5)), ("f64", (5,))))
    for x, y, bias, out in ((b, b, None, c), (a, a, None, c), (a, odd, None, c), (a, b, None, short), (a, b, None, i32), (a, b, f64, c), (a, b, c, c)):
        with pytest.raises(wk.WekuaError):
            wk.blas.gemmF8(pipeline, x, y, bias, -1, out)
    for t in (c, i32, f64):
        with pytest.raises(wk.WekuaError):
            a.quantize(pipeline, t)
    wk.blas.gemmF8(pipeline, a, b, None, -1, c)
    for m in (a, b, odd):
        m.deinit(pipeline)
    release(env, c, short, i32, f64)


@pytest.mark.parametrize("dtype", ["f32", "f64", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top,ids", [(1, 1, 1, "i32"), (3, 1000, 7, "i64"), (40, 77, 0, "i32")])
def test_token_logprobs(env, dtype, rows, vocab, top, ids):
    context, pipeline = env
    rng = np.random.RandomState(rows)
    x = pack(dtype, 2 * rng.randn(rows, vocab))
    t = rng.randint(-1, vocab, rows).astype(real_np_dtype(ids))
    acc = "f64" if dtype == "f64" else "f32"
    tx, tt, grad = upload(env, dtype, x), upload(env, ids, t), Tensor.alloc(dtype, context, pipeline, (rows, vocab))
    w, h = rng.randn(rows).astype(real_np_dtype(acc)), rng.randn(rows).astype(real_np_dtype(acc))
    tw, th = upload(env, acc, w), upload(env, acc, h)
    state = nn.TokenLogProbs.init(dtype, context, pipeline, rows, vocab, top)
    state.forward(pipeline, tx, tt)
    want = ot.token_logprobs(values(dtype, x), t, top)
    for name in ("logprob", "lse", "entropy"):
        assert np.abs(download(env, getattr(state, name)) - want[name]).max() <= TOL[acc] * 10
    if top:
        assert np.array_equal(download(env, state.top_ids).reshape(rows, top), want["top_ids"])
        assert np.abs(download(env, state.top_logprobs).reshape(rows, top) - want["top_logprobs"]).max() <= TOL[acc] * 10
    else:
        assert state.top_ids is None and state.top_logprobs is None
    for gw, gh in ((tw, th), (tw, None), (None, th)):
        state.backward(pipeline, tx, tt, gw, gh, grad)
        want_g = ot.token_logprobs_grad(values(dtype, x), t, want["lse"], want["entropy"], w if gw else None, h if gh else None)
        got = values(dtype, download(env, grad))
        # f16's subnormal values have steps of 2^-24
        assert (np.abs(got - want_g) <= STEP[dtype] * np.abs(want_g) + TOL[acc] * 10 * np.abs(want_g).max() + 2.0 ** -25).all()
    state.forward(pipeline, tx)
    assert np.abs(download(env, state.lse) - want["lse"]).max() <= TOL[acc] * 10
    state.deinit(pipeline)
    release(env, tx, tt, tw, th, grad)


def test_token_logprobs_refusals(env):
    context, pipeline = env
    for dtype, rows, vocab, top in (("f32", 0, 4, 0), ("f32", 4, 0, 0), ("f32", 4, 4, 5), ("f32", 4, 100, 65), ("i32", 4, 4, 0), ("f8e4m3", 4, 4, 0)):
        with pytest.raises(wk.WekuaError):
            nn.TokenLogProbs.init(dtype, context, pipeline, rows, vocab, top)
    state = nn.TokenLogProbs.init("f32", context, pipeline, 3, 10)
    x, wide, half = (Tensor.alloc(d, context, pipeline, s) for d, s in (("f32", (3, 10)), ("f32", (3, 11)), ("bf16", (3, 10))))
    ids, few, u32 = (Tensor.alloc(d, context, pipeline, (s,)) for d, s in (("i32", 3), ("i32", 2), ("u32", 3)))
    w = Tensor.alloc("f64", context, pipeline, (3,))
    for logits, targets in ((wide, ids), (half, ids), (x, few), (x, u32)):
        with pytest.raises(wk.WekuaError):
            state.forward(pipeline, logits, targets)
    state.forward(pipeline, x, ids)
    ok = state.logprob
    for logits, targets, gw, gh, out in ((x, ids, w, None, x), (x, ids, None, None, x), (x, ids, ok, None, half), (x, ids, ok, None, wide),
                                         (x, None, ok, None, x), (x, ids, ids, None, x)):
        with pytest.raises(wk.WekuaError):
            state.backward(pipeline, logits, targets, gw, gh, out)
    state.deinit(pipeline)
    release(env, x, wide, half, ids, few, u32, w)


# ---- layers -----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_dropout_layer(env, dtype):
    context, pipeline = env
    x, g = np.random.RandomState(1).rand(2, 9, 21) + 1
    outer, inner = nn.Sequential.init(dtype), nn.Sequential.init(dtype)
    inner.append(nn.Dropout.init(dtype, context, 21, 0.4, seed=5))
    outer.append(inner)
    cache, other = (nn.Cache.init(context, pipeline, 9, [outer]) for _ in range(2))
    lc, lo = cache.getLayerCache(0), other.getLayerCache(0)
    tx, tg = upload(env, dtype, x), Tensor.alloc(dtype, context, pipeline, (9, 21))
    assert outer.getWeights() == [] and outer.getBias() == [] and outer.getGradients(lc) == []

    def run(c):
        return download(env, outer.forward(pipeline, tx, c))

    def back(c):
        memory.readFromBuffer(pipeline, outer.getSensitivity(c), g)
        outer.backward(pipeline, c, tx, tg)
        return download(env, tg)
    first, second = run(lc), run(lo)       # counts 0 and 1, one on each cache
    near(first, ot.dropout(x, 0.4, 5, 0), dtype)
    near(second, ot.dropout(x, 0.4, 5, 1), dtype)
    near(back(lc), ot.dropout(g, 0.4, 5, 0), dtype)
    near(back(lo), ot.dropout(g, 0.4, 5, 1), dtype)
    outer.setTraining(False)
    assert np.array_equal(run(lc), x.astype(real_np_dtype(dtype))) and np.array_equal(back(lc), g.astype(real_np_dtype(dtype)))
    near(back(lo), ot.dropout(g, 0.4, 5, 1), dtype)     # that pass was in training
    outer.setTraining(True)
    near(run(lc), ot.dropout(x, 0.4, 5, 2), dtype)
    wrong = Tensor.alloc(dtype, context, pipeline, (9, 20))
    with pytest.raises(wk.WekuaError):
        outer.forward(pipeline, wrong, lc)
    for width, p in ((0, .1), (4, -.1), (4, 1.5), (4, float("nan"))):
        with pytest.raises(wk.WekuaError):
            nn.Dropout.init(dtype, context, width, p)
    for c in (cache, other):
        c.deinit(pipeline)
    outer.deinit(pipeline)
    release(env, tx, tg, wrong)


def test_a_refused_pass_leaves_the_dropout_layer_as_it_was(env):
    """Between a forward pass and its backward pass: neither the mask of that pass nor the next pass's count moves."""
    context, pipeline = env
    x, g = np.random.RandomState(8).rand(2, 9, 21).astype(np.float32) + 1
    layer = nn.Sequential.init("f32")
    layer.append(nn.Dropout.init("f32", context, 21, 0.4, seed=5))
    cache = nn.Cache.init(context, pipeline, 9, [layer])
    lc, tx, tg, wrong = cache.getLayerCache(0), upload(env, "f32", x), Tensor.alloc("f32", context, pipeline, (9, 21)), Tensor.alloc("f32", context, pipeline, (9, 20))

    def back(count):
        memory.readFromBuffer(pipeline, layer.getSensitivity(lc), g)
        layer.backward(pipeline, lc, tx, tg)
        near(download(env, tg), ot.dropout(g.astype(np.float64), 0.4, 5, count), "f32")
    near(download(env, layer.forward(pipeline, tx, lc)), ot.dropout(x.astype(np.float64), 0.4, 5, 0), "f32")
    for training in (True, False):
        layer.setTraining(training)
        with pytest.raises(wk.WekuaError):
            layer.forward(pipeline, wrong, lc)
    back(0)
    layer.setTraining(True)
    near(download(env, layer.forward(pipeline, tx, lc)), ot.dropout(x.astype(np.float64), 0.4, 5, 1), "f32")
    back(1)
    cache.deinit(pipeline)
    layer.deinit(pipeline)
    release(env, tx, tg, wrong)


def network(env, dtype, p, sizes=(24, 40, 301)):
    context, pipeline = env
    seq = nn.Sequential.init(dtype)
    seq.append(nn.Linear.init(dtype, context, pipeline, sizes[0], sizes[1], nn.Tanh.init(), seed=3))
    seq.append(nn.Dropout.init(dtype, context, sizes[1], p, seed=9))
    seq.append(nn.Linear.init(dtype, context, pipeline, sizes[1], sizes[2], nn.Identity.init(), seed=4))
    return seq


def oracle_step(x, targets, w, b, p, count):
    """Loss (sum over the rows) and gradients in 64 bits."""
    h = np.tanh(x @ w[0].T + b[0])
    mask = ot.dropout(np.ones_like(h), p, 9, count)
    logits = (h * mask) @ w[1].T + b[1]
    s = ot.token_logprobs(logits, targets)
    g = ot.token_logprobs_grad(logits, targets, s["lse"], s["entropy"], -np.ones(len(x)), None)
    gh = (g @ w[1]) * mask * (1 - h * h)
    return -s["logprob"].sum(), [gh.T @ x, g.T @ (h * mask)], [gh.sum(0), g.sum(0)], logits


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("ids", ["i32", "i64"])
@pytest.mark.parametrize("rows", [1, 37])
def test_training_run(env, dtype, ids, rows):
    """Three steps of the whole network, every gradient against 64 bits, with targets that count nothing, on Adam."""
    context, pipeline = env
    rng = np.random.RandomState(rows)
    x = rng.randn(rows, 24).astype(real_np_dtype(dtype))
    t = rng.randint(0, 301, rows).astype(real_np_dtype(ids))
    t[5::7] = -100
    seq = network(env, dtype, 0.3)
    cache = nn.Cache.init(context, pipeline, rows, [seq])
    lc, opt = cache.getLayerCache(0), nn.optimizers.Adam.init(dtype, 1e-2)
    state = nn.TokenLogProbs.init(dtype, context, pipeline, rows, 301)
    tx, tt, err = upload(env, dtype, x), upload(env, ids, t), np.zeros(1, real_np_dtype(dtype))
    for step in range(3):
        w, b = ([download(env, v).astype(np.float64) for v in vs] for vs in (seq.getWeights(), seq.getBias()))
        loss, gw, gb, logits = oracle_step(x.astype(np.float64), t, w, b, 0.3, step)
        out = seq.forward(pipeline, tx, lc)
        nn.loss.tokens(True, pipeline, out, tt, state, cache, err)
        assert abs(float(err[0]) - loss / rows) <= TOL[dtype] * 10 * max(1, loss / rows)
        near(download(env, out), logits, dtype, 64)
        seq.backward(pipeline, lc, tx)
        for got, want, k in zip(seq.getGradients(lc) + seq.getBiasGradients(lc), gw + gb, (400, 64, 400, 64)):
            near(download(env, got), want, dtype, k)
        opt.step(pipeline, cache)
    state.deinit(pipeline)
    opt.deinit(pipeline)
    cache.deinit(pipeline)
    seq.deinit(pipeline)
    release(env, tx, tt)


def test_gradients_against_differences(env):
    """f64, without dropped elements: the gradient of single weights against central differences of the device's own loss."""
    context, pipeline = env
    rng = np.random.RandomState(2)
    x, t, rows = rng.randn(11, 24), rng.randint(0, 301, 11).astype(np.int32), 11
    seq = network(env, "f64", 0.5)
    seq.setTraining(False)
    cache = nn.Cache.init(context, pipeline, rows, [seq])
    lc, state = cache.getLayerCache(0), nn.TokenLogProbs.init("f64", context, pipeline, rows, 301)
    tx, tt, err = upload(env, "f64", x), upload(env, "i32", t), np.zeros(1)

    def loss(derivative):
        nn.loss.tokens(derivative, pipeline, seq.forward(pipeline, tx, lc), tt, state, cache, err)
        return float(err[0]) * rows
    loss(True)
    seq.backward(pipeline, lc, tx)
    params = seq.getWeights() + seq.getBias()
    grads = [download(env, g) for g in seq.getGradients(lc) + seq.getBiasGradients(lc)]
    for param, grad in zip(params, grads):
        host = download(env, param)
        for at in (np.unravel_index(i, host.shape) for i in rng.randint(0, host.size, 4)):
            h, sides = 1e-5, []
            for sign in (1, -1):
                moved = host.copy()
                moved[at] += sign * h
                memory.readFromBuffer(pipeline, param, moved)
                sides.append(loss(False))
            memory.readFromBuffer(pipeline, param, host)
            # third derivatives of this loss are below 1e3: 1e-10 / 6 * 1e3; 2^-53 * 100 * sqrt(terms) / 1e-5
            assert abs((sides[0] - sides[1]) / (2 * h) - grad[at]) <= 2e-7
    state.deinit(pipeline)
    cache.deinit(pipeline)
    seq.deinit(pipeline)
    release(env, tx, tt)


def test_loss_refusals(env):
    context, pipeline = env
    seq = network(env, "f32", 0.1)
    cache = nn.Cache.init(context, pipeline, 4, [seq])
    good, double, narrow = (nn.TokenLogProbs.init(d, context, pipeline, 4, v) for d, v in (("f32", 301), ("f64", 301), ("f32", 300)))
    out, ids, bad = (Tensor.alloc(d, context, pipeline, s) for d, s in (("f32", (4, 301)), ("i32", (4,)), ("u8", (4,))))
    for o, t, s in ((out, ids, double), (out, ids, narrow), (out, bad, good), (ids, ids, good)):
        with pytest.raises(wk.WekuaError):
            nn.loss.tokens(True, pipeline, o, t, s, cache, None)
    nn.loss.tokens(True, pipeline, out, ids, good, cache, None)
    for s in (good, double, narrow):
        s.deinit(pipeline)
    cache.deinit(pipeline)
    seq.deinit(pipeline)
    release(env, out, ids, bad)


# ---- a run as it would be served ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 70])
def test_serving_run(env, rows):
    """8-bit hidden layer with bias and tanh, 8-bit head, log probabilities with alternatives: each stage against 64 bits on what the
    stage before it gave."""
    context, pipeline = env
    rng = np.random.RandomState(rows)
    k, hidden, vocab, top = 200, 264, 1037, 5
    x, bias = pack("bf16", rng.randn(rows, k)), rng.randn(hidden).astype(np.float32)
    w1, w2 = rng.randn(hidden, k).astype(np.float32) / 14, rng.randn(vocab, hidden).astype(np.float32) / 4
    tx, tb, t1, t2 = upload(env, "bf16", x), upload(env, "f32", bias), upload(env, "f32", w1), upload(env, "f32", w2)
    init = wk.blas.BlockScaled.init
    a1, b1, a2, b2 = (init(context, pipeline, r, c, s) for r, c, s in ((rows, k, 1), (hidden, k, 128), (rows, hidden, 1), (vocab, hidden, 128)))
    h, logits = Tensor.alloc("bf16", context, pipeline, (rows, hidden)), Tensor.alloc("bf16", context, pipeline, (rows, vocab))
    state = nn.TokenLogProbs.init("bf16", context, pipeline, rows, vocab, top)
    b1.quantize(pipeline, t1)
    b2.quantize(pipeline, t2)
    a1.quantize(pipeline, tx)
    wk.blas.gemmF8(pipeline, a1, b1, tb, 1, h)
    a2.quantize(pipeline, h)
    wk.blas.gemmF8(pipeline, a2, b2, None, -1, logits)
    state.forward(pipeline, logits)

    def get(m):
        return download(env, m.codes), download(env, m.scales)

    def product(a, b, bias, kind, got):
        want, mag, largest = ot.gemm_f8(*get(a), *get(b), bias, kind)
        assert (np.abs(got - want) <= 7 * 2.0 ** -13 * largest + 300 * 2.0 ** -24 * (mag + 4) + 2.0 ** -8 * np.abs(want)).all()
    hv, lv = values("bf16", download(env, h)), values("bf16", download(env, logits))
    product(a1, b1, bias, 1, hv)
    codes, scales = ot.f8_quantize(hv, 1)
    assert np.array_equal(get(a2)[0], codes) and np.array_equal(get(a2)[1], scales)
    product(a2, b2, None, -1, lv)
    want = ot.token_logprobs(lv, None, top)
    assert np.array_equal(download(env, state.top_ids).reshape(rows, top), want["top_ids"])
    assert np.abs(download(env, state.top_logprobs).reshape(rows, top) - want["top_logprobs"]).max() <= 1e-4
    assert np.abs(download(env, state.entropy) - want["entropy"]).max() <= 1e-4
    state.deinit(pipeline)
    for m in (a1, b1, a2, b2):
        m.deinit(pipeline)
    release(env, tx, tb, t1, t2, h, logits)


# ---- streams, graphs, long offsets, large sizes (through the C ABI) ---------------------------------------------------------------------

class Step:
    """One training step on raw buffers: dropout counted in device memory, log probabilities of few long rows (which are split),
    their gradient, the gradient's quantised form and two products with it."""
    ROWS, VOCAB, N = 5, 9001, 150

    def __init__(self, dev, seed):
        rng = np.random.RandomState(seed)
        r, v, n = self.ROWS, self.VOCAB, self.N
        self.x = rng.randn(r, v).astype(np.float32)
        self.w = rng.randn(n, v).astype(np.float32)
        self.dev, self.blocks = dev, -(-v // 128)
        self.bufs = {"x": dev.upload(self.x), "t": dev.upload(rng.randint(0, v, r).astype(np.int32)), "minus": dev.upload(-np.ones(r, np.float32)),
                     "step": dev.upload(np.zeros(1, np.uint64)), "wq": dev.malloc(n * v), "ws": dev.malloc(4 * 2 * self.blocks)}
        self.outs = {"y": (np.float32, (r, v)), "lp": (np.float32, (r,)), "lse": (np.float32, (r,)), "ent": (np.float32, (r,)),
                     "ids": (np.int32, (r, 9)), "lps": (np.float32, (r, 9)), "g": (np.float32, (r, v)), "gq": (np.uint8, (r, v)),
                     "gs": (np.float32, (r, self.blocks)), "c": (np.float32, (r, n)), "big": (np.uint16, (n, n))}
        for name, (t, s) in self.outs.items():
            self.bufs[name] = dev.malloc(int(np.prod(s)) * np.dtype(t).itemsize)
        self.wsn = dev.token_logprobs_workspace_bytes("f32", r, v, 9)
        assert self.wsn
        self.bufs["work"] = dev.malloc(self.wsn)
        self.bufs["rq"], self.bufs["rs"] = dev.malloc(n * v), dev.malloc(4 * n * self.blocks)
        tmp = dev.upload(self.w)
        dev.f8_quantize("f32", n, v, tmp, v, 128, self.bufs["wq"], v, self.bufs["ws"], self.blocks)
        dev.f8_quantize("f32", n, v, tmp, v, 1, self.bufs["rq"], v, self.bufs["rs"], self.blocks)
        dev.sync()
        tmp.free()

    def __call__(self, dev=None):
        d, b, r, v, n, k = dev or self.dev, self.bufs, self.ROWS, self.VOCAB, self.N, self.blocks
        d.dropout("f32", (1, r, v), b["x"], v, r * v, b["y"], v, r * v, 0.2, 3, 1, b["step"])
        d.token_logprobs("f32", r, v, b["y"], v, b["t"], "i32", b["lp"], b["lse"], b["ent"], 9, b["ids"], b["lps"], b["work"], self.wsn)
        d.token_logprobs_grad("f32", r, v, b["y"], v, b["t"], "i32", b["lse"], b["ent"], b["minus"], None, b["g"], v)
        d.f8_quantize("f32", r, v, b["g"], v, 1, b["gq"], v, b["gs"], k)
        d.gemm_f8(r, n, v, b["gq"], v, b["gs"], k, b["wq"], v, b["ws"], k, "f32", b["c"], n)
        d.gemm_f8(n, n, v, b["rq"], v, b["rs"], k, b["wq"], v, b["ws"], k, "bf16", b["big"], n)

    def results(self):
        return {name: self.bufs[name].download(t, s) for name, (t, s) in self.outs.items()}

    def clear(self):
        for name, (t, s) in self.outs.items():
            self.bufs[name].write(np.full(s, 77, t))

    def free(self):
        for b in self.bufs.values():
            b.free()


def same(a, b):
    return all(np.array_equal(a[n], b[n], equal_nan=True) for n in a)


def test_products_of_the_run(dev):
    """Both products of the run against 64 bits: what the tests below compare runs with."""
    step = Step(dev, 7)
    step()
    got, k = step.results(), step.blocks
    wq, ws = ot.f8_quantize(step.w.astype(np.float64), 128)
    rq, rs = ot.f8_quantize(step.w.astype(np.float64), 1)
    for name, a, sa, out in (("c", got["gq"], got["gs"], "f32"), ("big", rq, rs, "bf16")):
        want, mag, largest = ot.gemm_f8(a, sa, wq, ws)
        tol = (128 + k + 2) * 2.0 ** -23 * mag + (7 * 2.0 ** -13 * largest + 2.0 ** -8 * 1.01 * np.abs(want) if out != "f32" else 2.0 ** -24 * np.abs(want))
        assert (np.abs(values(out, got[name]) - want) <= tol + 1e-37).all(), name
    step.free()


def test_run_on_two_streams_at_once(dev):
    """Two runs at once, on two streams, give what each gives alone; and so does the same one twice."""
    from wekua_amd import raw
    other = raw.Device(0)
    one, two = Step(dev, 1), Step(other, 2)
    alone = []
    for s in (one, two):
        s()
        alone.append(s.results())
    for s in (one, two):
        s.clear()
    for _ in range(10):
        one()
        two()
    assert same(one.results(), alone[0]) and same(two.results(), alone[1])
    one.free()
    two.free()
    other.close()


def test_captured_run(dev):
    """The run in a graph, replayed with the count moved between the replays, each replay against the same run without a graph."""
    step = Step(dev, 3)
    step()
    dev.sync()
    hip = ctypes.CDLL("libamdhip64.so.7")
    dev.lib.wk_stream_native.restype = ctypes.c_void_p
    stream = ctypes.c_void_p(dev.lib.wk_stream_native(dev.stream))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    try:
        step()
    finally:
        rc = hip.hipStreamEndCapture(stream, ctypes.byref(graph))
    assert rc == 0 and hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    seen = []
    for count in (0, 1, 2, 1):
        step.bufs["step"].write(np.array([count], np.uint64))
        step.clear()
        step()
        want = step.results()
        step.clear()
        assert hip.hipGraphLaunch(run, stream) == 0
        got = step.results()
        assert same(got, want)
        keep = ot.dropout_keep(step.x.size, 0.2, 3, 1 + count).reshape(step.x.shape)
        assert np.array_equal(got["y"] != 0, keep & (step.x != 0))
        seen.append(got["y"])
    assert np.array_equal(seen[1], seen[3]) and not np.array_equal(seen[0], seen[1])
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    step.free()


def test_captured_dropout_layer(env):
    """A network's forward and backward pass in a graph: without a step the replays repeat their masks, with one that is moved by the
    passes in a replay each has new ones, the backward pass the same; the program's own passes between them too."""
    context, pipeline = env
    rng = np.random.RandomState(11)
    x, g = (rng.rand(9, 21) + 1 for _ in range(2))
    layer, inner = nn.Sequential.init("f64"), nn.Sequential.init("f64")
    inner.append(nn.Dropout.init("f64", context, 21, 0.4, seed=5))
    layer.append(inner)
    cache = nn.Cache.init(context, pipeline, 9, [layer])
    lc, tx, tg, step = cache.getLayerCache(0), upload(env, "f64", x), Tensor.alloc("f64", context, pipeline, (9, 21)), upload(env, "u64", np.zeros(1, np.uint64))
    memory.readFromBuffer(pipeline, layer.getSensitivity(lc), g)
    bad = upload(env, "i64", np.zeros(1, np.int64))
    with pytest.raises(wk.WekuaError):
        layer.setStep(bad)
    near(download(env, layer.forward(pipeline, tx, lc)), ot.dropout(x, 0.4, 5, 0), "f64")       # count 0, no step
    layer.setStep(step)
    hip = ctypes.CDLL("libamdhip64.so.7")
    lib = wk._lib()
    lib.wkz_context_stream.restype = ctypes.c_void_p
    dev_lib = wk._capi.load()
    queue = ctypes.c_void_p(lib.wkz_context_stream(context._h, 0))
    dev_lib.wk_stream_native.restype = ctypes.c_void_p
    stream = ctypes.c_void_p(dev_lib.wk_stream_native(queue))
    pipeline.waitAndCleanup()
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    try:
        out = layer.forward(pipeline, tx, lc)                                                     # count 1 + step
        layer.backward(pipeline, lc, tx, tg)
    finally:
        rc = hip.hipStreamEndCapture(stream, ctypes.byref(graph))
    assert rc == 0 and hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    masks = []
    for at in (0, 1, 2, 2):
        memory.readFromBuffer(pipeline, step, np.array([at], np.uint64))
        pipeline.waitAndCleanup()
        wk.fill.zeroes(pipeline, tg)
        assert hip.hipGraphLaunch(run, stream) == 0
        y, dx = download(env, out), download(env, tg)
        near(y, ot.dropout(x, 0.4, 5, 1 + at), "f64")
        near(dx, ot.dropout(g, 0.4, 5, 1 + at), "f64")
        masks.append(y != 0)
    assert np.array_equal(masks[2], masks[3]) and not np.array_equal(masks[0], masks[1]) and not np.array_equal(masks[1], masks[2])
    near(download(env, layer.forward(pipeline, tx, lc)), ot.dropout(x, 0.4, 5, 2 + 2), "f64")   # the host's next count, and the step
    layer.setStep(None)
    layer.backward(pipeline, lc, tx, tg)                                                          # goes by the pass it belongs to
    near(download(env, tg), ot.dropout(g, 0.4, 5, 2 + 2), "f64")
    near(download(env, layer.forward(pipeline, tx, lc)), ot.dropout(x, 0.4, 5, 3), "f64")
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    cache.deinit(pipeline)
    layer.deinit(pipeline)
    release(env, tx, tg, step, bad)


def put(dev, buf, host, pitch):
    """Row by row: `pitch` elements lie between them."""
    host = np.ascontiguousarray(host)
    for r in range(len(host)):
        at = buf.ptr.value + r * pitch * host.itemsize
        assert dev.lib.wk_copy_h2d_rect_async(dev.stream, at, host[r].nbytes, 0, host[r].ctypes.data, host[r].nbytes, 0, host[r].nbytes, 1, 1) == 0
    dev.sync()


def fetch(dev, buf, dtype, shape, pitch):
    out = np.empty(shape, dtype)
    for r in range(shape[0]):
        at = buf.ptr.value + r * pitch * out.itemsize
        assert dev.lib.wk_copy_d2h_rect_async(dev.stream, out[r].ctypes.data, out[r].nbytes, 0, at, out[r].nbytes, 0, out[r].nbytes, 1, 1) == 0
    dev.sync()
    return out


def test_offsets_beyond_32_bits(dev):
    """Rows 2^31 + 8 elements apart (and not a multiple of 8 of them): three of them pass 2^32 elements."""
    rng = np.random.RandomState(4)
    for pitch in (2 ** 31 + 8, 2 ** 31 + 3):
        rows, cols = 4, 700
        room, out = dev.malloc(2 * (3 * pitch + 4096)), dev.malloc(2 * (3 * pitch + 4096))
        x = pack("bf16", rng.randn(rows, cols))
        xv = values("bf16", x)
        put(dev, room, x, pitch)
        dev.dropout("bf16", (1, rows, cols), room, pitch, rows * pitch, out, pitch, rows * pitch, 0.25, 8, 2)
        want = ot.dropout(xv, 0.25, 8, 2)
        got = values("bf16", fetch(dev, out, np.uint16, (rows, cols), pitch))
        assert np.array_equal(got == 0, want == 0) and (np.abs(got - want) <= 2.0 ** -7.9 * np.abs(want)).all()
        t = dev.upload(np.array([3, 699, -1, 0], np.int32))
        lp, lse, ent, w = dev.malloc(16), dev.malloc(16), dev.malloc(16), dev.upload(np.array([1, -2, 3, .5], np.float32))
        dev.token_logprobs("bf16", rows, cols, room, pitch, t, "i32", lp, lse, ent)
        want = ot.token_logprobs(xv, np.array([3, 699, -1, 0]))
        for b, name in ((lp, "logprob"), (lse, "lse"), (ent, "entropy")):
            assert np.abs(b.download(np.float32, (4,)) - want[name]).max() <= 1e-4
        dev.token_logprobs_grad("bf16", rows, cols, room, pitch, t, "i32", lse, ent, w, None, out, pitch)
        want = ot.token_logprobs_grad(xv, np.array([3, 699, -1, 0]), want["lse"], want["entropy"], np.array([1, -2, 3, .5]), None)
        assert np.abs(values("bf16", fetch(dev, out, np.uint16, (rows, cols), pitch)) - want).max() <= 2.0 ** -8 * np.abs(want).max() + 1e-5
        # codes of the rows, 2^31 apart too, and their product with weights 2^26 and more apart
        scales = dev.malloc(4 * 6 * rows)
        dev.f8_quantize("bf16", rows, cols, room, pitch, 1, out, pitch, scales, 6)
        qa, sa = ot.f8_quantize(xv, 1)
        assert np.array_equal(fetch(dev, out, np.uint8, (rows, cols), pitch), qa) and np.array_equal(scales.download(np.float32, (rows, 6)), sa)
        w8, n, far = rng.randn(140, cols), 140, 2 ** 25 + pitch % 8
        qb, sb = ot.f8_quantize(w8, 128)
        put(dev, room, qb, far)
        bs = dev.upload(sb)
        for kind, shape in (("f32", (rows, n)), ("bf16", (rows, n))):
            c = dev.malloc(4 * shape[0] * shape[1])
            dev.gemm_f8(rows, n, cols, out, pitch, scales, 6, room, far, bs, 6, kind, c, n)
            y, mag, largest = ot.gemm_f8(qa, sa, qb, sb)
            got = values(kind, c.download(np.uint16 if kind == "bf16" else np.float32, shape))
            assert (np.abs(got - y) <= 7 * 2.0 ** -13 * largest + 800 * 2.0 ** -24 * mag + 2.0 ** -8 * np.abs(y)).all()
            c.free()
        # the results far apart, and the other operand far apart, of more rows than the kernel for few rows takes
        c = dev.malloc(4 * (2 ** 25 * 140 + 4096))
        dev.gemm_f8(n, rows, cols, room, far, dev_rows := dev.upload(np.repeat(sb, 128, 0)[:n].copy()), 6, out, pitch, sc := dev.upload(sa[:1].copy()), 6,
                    "f32", c, 2 ** 25)
        y, mag, _ = ot.gemm_f8(qb, np.repeat(sb, 128, 0)[:n], qa, sa[:1])
        assert (np.abs(fetch(dev, c, np.float32, (n, rows), 2 ** 25) - y) <= 800 * 2.0 ** -24 * mag).all()
        for b in (room, out, t, lp, lse, ent, w, scales, bs, c, dev_rows, sc):
            b.free()


@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_aligned_rows_far_apart(dev, out):
    """Operands and scales on 16-byte boundaries whose rows lie 2^25 and 2^26 bytes apart, results 2^24 elements: tiles with offsets beyond
    32 bits, ragged on both sides, and a shorter last block."""
    rng = np.random.RandomState(6)
    m, n, k, kb = 140, 150, 400, 4
    lda, ldb, ldc, sap = 2 ** 25, 2 ** 26 + 16, 2 ** 24, 2 ** 22
    a, b = (ot.e4m3_encode(np.clip(rng.randn(r, k) * 60, -448, 448)) for r in (m, n))
    sa, sb = np.exp(rng.randn(m, kb)).astype(np.float32) / 60, np.exp(rng.randn(2, kb)).astype(np.float32) / 60
    size = 4 if out == "f32" else 2
    ba, bb, bsa, bsb, bc = (dev.malloc(v) for v in (m * lda, n * ldb, 4 * m * sap, 4 * 2 * sap, size * m * ldc))
    for buf, host, pitch in ((ba, a, lda), (bb, b, ldb), (bsa, sa, sap), (bsb, sb, sap)):
        put(dev, buf, host, pitch)
    dev.gemm_f8(m, n, k, ba, lda, bsa, sap, bb, ldb, bsb, sap, out, bc, ldc)
    got = values(out, fetch(dev, bc, np.float32 if out == "f32" else np.uint16, (m, n), ldc))
    want, mag, largest = ot.gemm_f8(a, sa, b, sb)
    tol = (128 + kb + 2) * 2.0 ** -23 * mag + (7 * 2.0 ** -13 * largest + 2.0 ** -8 * 1.01 * np.abs(want) if out != "f32" else 2.0 ** -24 * np.abs(want))
    assert (np.abs(got - want) <= tol).all()
    for x in (ba, bb, bsa, bsb, bc):
        x.free()


def test_more_than_the_cache_holds(dev):
    """Sizes beyond which the kernels do not keep their tensors in the last-level cache, looked at in places."""
    rng = np.random.RandomState(5)
    rows, cols = 8200, 8203
    block = pack("bf16", rng.randn(200, cols) + 4)
    x = np.tile(block, (41, 1))
    bx, by = dev.upload(x), dev.malloc(x.nbytes)
    dev.dropout("bf16", (1, rows, cols), bx, cols, x.size, by, cols, x.size, 0.5, 6, 2 ** 40)
    got = by.download(np.uint16, x.shape)
    assert abs((got != 0).mean() - 0.5) <= 6 * 0.5 / np.sqrt(x.size)
    flat, fx = got.reshape(-1), x.reshape(-1)
    for first in (0, 4 * (x.size // 8), x.size // 4 * 4 - 400):
        ctr = [[q & 0xFFFFFFFF, q >> 32, 0, 2 ** 8] for q in range(first // 4, first // 4 + 100)]
        keep = ot.philox4x32(ctr, (6, 0), 7).reshape(-1) >= 2 ** 31
        want = np.where(keep, 2 * values("bf16", fx[first:first + 400]), 0)
        assert np.array_equal(values("bf16", flat[first:first + 400]), want)
    # quantise: rows and weights, 200 rows repeat, so blocks of 128 rows do at 3200
    for block_rows in (1, 128):
        nb, k = -(-rows // block_rows), -(-cols // 128)
        q, s = dev.malloc(rows * cols), dev.malloc(4 * nb * k)
        dev.f8_quantize("bf16", rows, cols, bx, cols, block_rows, q, cols, s, k)
        codes, scales = q.download(np.uint8, (rows, cols)), s.download(np.float32, (nb, k))
        for at in (0, 128 * 13, 8192):
            part = slice(at, min(at + (3 if block_rows == 1 else 128), rows))
            wq, wsc = ot.f8_quantize(values("bf16", x[part]), block_rows)
            assert np.array_equal(codes[part], wq) and np.array_equal(scales[at // block_rows:at // block_rows + len(wsc)], wsc)
        q.free()
        s.free()
    # log probabilities' gradient, logits' own place
    t = np.arange(rows, dtype=np.int32)
    stats = [dev.malloc(4 * rows) for _ in range(3)]
    bt, bw = dev.upload(t), dev.upload(np.full(rows, -1, np.float32))
    dev.token_logprobs("bf16", rows, cols, bx, cols, bt, "i32", *stats)
    dev.token_logprobs_grad("bf16", rows, cols, bx, cols, bt, "i32", stats[1], stats[2], bw, None, bx, cols)
    got = bx.download(np.uint16, x.shape)
    for r in (0, 1, 4100, rows - 1):
        want = ot.token_logprobs(values("bf16", x[r:r + 1]), t[r:r + 1])
        assert abs(stats[0].download(np.float32, (rows,))[r] - want["logprob"][0]) <= 1e-4
        want = ot.token_logprobs_grad(values("bf16", x[r:r + 1]), t[r:r + 1], want["lse"], want["entropy"], np.array([-1.0]), None)
        # 1e-5: d is known to 2^-24 * (|d| < 16) and two more roundings
        assert (np.abs(values("bf16", got[r:r + 1]) - want) <= (2.0 ** -8 + 1e-5) * np.abs(want)).all()
    for b in (bx, by, bt, bw, *stats):
        b.free()


def test_sizes_beyond_one_launch_are_refused(dev):
    """More threads than a launch counts, results in an operand's place: refused on the host."""
    b = dev.malloc(1 << 12)
    p, lib, st = b.ptr.value, dev.lib, dev.stream
    q = p + 2048
    s3 = ctypes.c_uint64 * 3
    for dtype, per in ((8, 4), (9, 4), (32, 8), (33, 8)):
        n = per * 2 ** 32
        assert lib.wk_dropout(st, dtype, s3(1, 1, n), p, n, n, p, n, n, 0.5, 1, 0, None) == 1
        assert lib.wk_dropout(st, dtype, s3(2 ** 16, 2 ** 16, 1), p, 1, 2 ** 16, q, 2, 2 ** 17, 0.5, 1, 0, None) == 1
    for rows, cols in ((2 ** 28, 128), (1, 2 ** 31), (2 ** 31, 1), (2 ** 40 - 1, 2 ** 40 - 1)):
        assert lib.wk_f8_quantize(st, 33, rows, cols, p, cols, 1, q, cols, p + 1024, -(-cols // 128)) == 1
    assert lib.wk_f8_quantize(st, 33, 2 ** 30, 2 ** 29, p, 2 ** 29, 128, q, 2 ** 29, p + 1024, 2 ** 22) == 1
    assert lib.wk_f8_quantize(st, 33, 2, 8, p, 8, 1, p, 8, q, 1) == 1
    assert lib.wk_gemm_f8(st, 1, 2 ** 31 - 1, 16, p, 16, p, 1, q, 16, p, 1, 8, p + 1024, 2 ** 31, None, -1) == 1
    assert lib.wk_gemm_f8(st, 2 ** 30, 2 ** 30, 16, p, 16, p, 1, q, 16, p, 1, 8, p + 1024, 2 ** 31, None, -1) == 1
    for c in (p, q):
        assert lib.wk_gemm_f8(st, 2, 2, 16, p, 16, p + 512, 1, q, 16, p + 512, 1, 8, c, 2, None, -1) == 1
    for rows, vocab in ((2 ** 24, 1025), (2 ** 26, 1024), (2 ** 31, 1), (2, 2 ** 31)):
        assert lib.wk_token_logprobs(st, 8, rows, vocab, p, vocab, None, 4, None, q, None, 0, None, None, None, 0) == 1
    for dtype, rows, vocab in ((8, 2 ** 24, 1), (8, 2 ** 23, 2049), (33, 2 ** 23, 4097), (9, 2 ** 23, 1025)):
        assert lib.wk_token_logprobs_grad(st, dtype, rows, vocab, p, vocab, q, 4, q, None, q, None, p, vocab) == 1
    b.free()
