"""What is measured of the operators at the token end of a network: dropout, the block-scaled 8-bit product
with its quantiser, and the log probabilities of given tokens with their gradient.

`own = False` computes each in its plain form (elementary torch operations in 32 bits, 64 where 32 would lose
what matters, rounded once at the end); `own = True` makes the calls of `wekua_amd.raw.Device` that a program
makes whose tensors live in device memory of its own.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f64": torch.float64}
BLOCK = 128            # elements of k under one scale
E4M3_MAX = 448.0       # largest value of the 8-bit format
WORKSPACE = 32 << 20   # bytes of device memory that the program keeps for calls that want some


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # dropout behind one small layer, where the launch itself counts
        {"name": "dropout-small-f32", "op": "dropout", "rows": 16, "cols": 1024, "pad": 0, "dtype": "f32", "p": 0.1, "back": False},
        # a training step's hidden states, forward and the gradient on its way back, in the type they are kept in
        {"name": "dropout-large-bf16", "op": "dropout", "rows": 8192, "cols": 8192, "pad": 0, "dtype": "bf16", "p": 0.1, "back": True},
        # activations of a decode step of a few sequences, one scale per row and 128 columns
        {"name": "quantize-rows-small", "op": "quantize", "rows": 8, "cols": 8192, "pad": 0, "dtype": "f32", "block_rows": 1},
        # a weight matrix laid out once, one scale per 128 x 128 block
        {"name": "quantize-weights", "op": "quantize", "rows": 8192, "cols": 8192, "pad": 0, "dtype": "f32", "block_rows": 128},
        # a decode step of eight sequences through one matrix: the weights are read once
        {"name": "gemm-f8-decode", "op": "gemm_f8", "m": 8, "n": 8192, "k": 8192, "out": "f32", "bias": True, "act": "none"},
        # ragged in every direction, with the epilogue of a hidden layer and the type this framework's layers have
        {"name": "gemm-f8-ragged", "op": "gemm_f8", "m": 1000, "n": 4095, "k": 4001, "out": "f32", "bias": True, "act": "tanh"},
        # the square product that this repository's benchmark is quoted on
        {"name": "gemm-f8-8192", "op": "gemm_f8", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "bias": False, "act": "none"},
        # one sampled token over a large vocabulary, with the alternatives that a server answers with
        {"name": "logprobs-one-token", "op": "logprobs", "rows": 1, "vocab": 131072, "pad": 0, "dtype": "f32", "top": 20, "masked": 0.0},
        # scoring a text: an odd vocabulary, entropy and five alternatives, some rows under a grammar's mask
        {"name": "logprobs-score-bf16", "op": "logprobs", "rows": 2048, "vocab": 50021, "pad": 11, "dtype": "bf16", "top": 5, "masked": 0.25},
        # a training batch's losses: log probabilities alone
        {"name": "logprobs-train-f32", "op": "logprobs", "rows": 8192, "vocab": 32000, "pad": 0, "dtype": "f32", "top": 0, "masked": 0.0},
        # gradients of the losses and of an entropy bonus, odd sizes
        {"name": "logprobs-grad-f32", "op": "logprobs_grad", "rows": 1000, "vocab": 32003, "pad": 1, "dtype": "f32", "entropy": True, "ignored": 0.2},
        # the largest batch's gradient
        {"name": "logprobs-grad-bf16", "op": "logprobs_grad", "rows": 4096, "vocab": 65536, "pad": 0, "dtype": "bf16", "entropy": False, "ignored": 0.0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("dropout", "quantize", "gemm_f8", "gemm_f8", "logprobs", "logprobs", "logprobs_grad"))
    while True:
        if op == "dropout":
            c = {"op": op, "rows": _log_int(rng, 1, 16384), "cols": _log_int(rng, 1, 16384), "pad": rng.choice((0, 0, 1, 3, 8)),
                 "dtype": rng.choice(("bf16", "f16", "f32", "f64")), "p": rng.choice((0.0, 0.05, 0.1, 0.5, 0.9, 1.0)), "back": rng.random() < 0.5}
            fits = c["rows"] * c["cols"] <= 8192 * 8192 // (2 if c["dtype"] == "f64" else 1)
        elif op == "quantize":
            c = {"op": op, "rows": _log_int(rng, 1, 16384), "cols": _log_int(rng, 1, 16384), "pad": rng.choice((0, 0, 1, 8)),
                 "dtype": rng.choice(("bf16", "f16", "f32")), "block_rows": rng.choice((1, 128))}
            fits = c["rows"] * c["cols"] <= 8192 * 8192
        elif op == "gemm_f8":
            c = {"op": op, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 1, 16384), "k": _log_int(rng, 1, 16384),
                 "out": rng.choice(("f32", "bf16", "f16")), "bias": rng.random() < 0.5, "act": rng.choice(("none", "none", "sigmoid", "tanh"))}
            fits = c["m"] * c["n"] * c["k"] <= 8192 ** 3 // 4
        elif op == "logprobs":
            c = {"op": op, "rows": _log_int(rng, 1, 8192), "vocab": _log_int(rng, 64, 262144), "pad": rng.choice((0, 0, 1, 8)),
                 "dtype": rng.choice(("bf16", "bf16", "f16", "f32", "f32", "f64")), "top": rng.choice((0, 1, 5, 20, 64)),
                 "masked": rng.choice((0.0, 0.0, 0.5))}
            fits = c["rows"] * c["vocab"] <= 1 << 26
        else:
            c = {"op": op, "rows": _log_int(rng, 1, 8192), "vocab": _log_int(rng, 2, 262144), "pad": rng.choice((0, 0, 1, 8)),
                 "dtype": rng.choice(("bf16", "bf16", "f16", "f32", "f32", "f64")), "entropy": rng.random() < 0.5,
                 "ignored": rng.choice((0.0, 0.3))}
            fits = c["rows"] * c["vocab"] <= 1 << 26
        if fits:
            return c


def _size(name):
    return {"f16": 2, "bf16": 2, "f32": 4, "f64": 8}[name]


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def work(c):
    if c["op"] == "dropout":
        n, times = c["rows"] * c["cols"], 2 if c["back"] else 1
        return {"bytes": 2 * n * _size(c["dtype"]) * times, "flops": n * times}
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        scales = (c["rows"] if c["block_rows"] == 1 else _blocks(c["rows"])) * _blocks(c["cols"])
        return {"bytes": n * (_size(c["dtype"]) + 1) + 4 * scales, "flops": 2 * n}
    if c["op"] == "gemm_f8":
        m, n, k = c["m"], c["n"], c["k"]
        scales = (m + _blocks(n)) * _blocks(k) + (n if c["bias"] else 0)
        return {"bytes": (m + n) * k + 4 * scales + m * n * _size(c["out"]), "flops": 2 * m * n * k}
    n, s, a = c["rows"] * c["vocab"], _size(c["dtype"]), 8 if c["dtype"] == "f64" else 4
    if c["op"] == "logprobs":
        return {"bytes": n * s + c["rows"] * (4 + 3 * a + c["top"] * (4 + a)), "flops": 6 * n}
    return {"bytes": 2 * n * s + c["rows"] * (4 + 4 * a), "flops": 5 * n}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _pitched(t, pad):
    """The same values in rows that are `pad` elements further apart."""
    if not pad:
        return t.contiguous()
    wide = torch.zeros((t.shape[0], t.shape[1] + pad), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _empty(rows, cols, pad, dtype):
    return torch.empty((rows, cols + pad), dtype=dtype, device="cuda")[:, :cols]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"case": c, "seed": (seed * 0x9E3779B97F4A7C15 + 1) & (2 ** 64 - 1)}
    if c["op"] == "dropout":
        dt = DTYPES[c["dtype"]]
        s["x"] = _pitched(normal(c["rows"], c["cols"]).to(dt), c["pad"])
        s["y"] = _empty(c["rows"], c["cols"], c["pad"], dt)
        if c["back"]:
            s["dy"] = _pitched(normal(c["rows"], c["cols"]).to(dt), c["pad"])
            s["dx"] = _empty(c["rows"], c["cols"], c["pad"], dt)
        s["offset"] = 3 + seed % 5  # the number of the training step
    elif c["op"] == "quantize":
        # rows and columns of different magnitudes, as activations and weights have them
        x = normal(c["rows"], c["cols"]) * torch.exp(normal(c["rows"], 1)) * torch.exp(normal(1, c["cols"]))
        s["x"] = _pitched(x.clamp_(-3e4, 3e4).to(DTYPES[c["dtype"]]), c["pad"])
        groups = c["rows"] if c["block_rows"] == 1 else _blocks(c["rows"])
        s["q"] = torch.empty((c["rows"], -(-c["cols"] // 16) * 16), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty((groups, _blocks(c["cols"])), dtype=torch.float32, device="cuda")
    elif c["op"] == "gemm_f8":
        m, n, k = c["m"], c["n"], c["k"]
        pitch = -(-k // 16) * 16  # rows start on 16 bytes, as this framework's tensors have them

        def operand(rows):
            q = torch.zeros((rows, pitch), dtype=torch.uint8, device="cuda")
            q[:, :k] = (normal(rows, k) * 100).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
            return q

        s["a"], s["b"] = operand(m), operand(n)
        s["sa"] = torch.exp(normal(m, _blocks(k))) / 100
        s["sb"] = torch.exp(normal(_blocks(n), _blocks(k))) / (100 * math.sqrt(k))
        s["bias"] = normal(n) if c["bias"] else None
        s["out"] = torch.empty((m, n), dtype=DTYPES[c["out"]], device="cuda")
    else:
        rows, vocab, dt = c["rows"], c["vocab"], DTYPES[c["dtype"]]
        acc = torch.float64 if c["dtype"] == "f64" else torch.float32
        x = normal(rows, vocab) * 3
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        likely = torch.rand((rows,), generator=g, device="cuda") < 0.7  # a trained model gives most tokens a high score
        x[torch.arange(rows, device="cuda"), targets.long()] += torch.where(likely, 12.0, 0.0)
        if c["op"] == "logprobs":
            if c["masked"]:  # rows under a mask keep about a third of the vocabulary, and their token
                under = torch.rand((rows, 1), generator=g, device="cuda") < c["masked"]
                out = torch.rand((rows, vocab), generator=g, device="cuda") < 2 / 3
                out[torch.arange(rows, device="cuda"), targets.long()] = False
                x.masked_fill_(under & out, -math.inf)
                if rows > 2:
                    x[1] = -math.inf  # a row that its mask leaves empty
                del out, under
            top = min(c["top"], vocab)
            s["top_ids"] = torch.empty((rows, top), dtype=torch.int32, device="cuda") if top else None
            s["top_logprobs"] = torch.empty((rows, top), dtype=acc, device="cuda") if top else None
            s["top"] = top
            s["workspace"] = torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda")
            for name in ("logprob", "lse", "entropy"):
                s[name] = torch.empty(rows, dtype=acc, device="cuda")
        else:
            if c["ignored"]:
                targets = torch.where(torch.rand((rows,), generator=g, device="cuda") < c["ignored"], -1, targets).to(torch.int32)
            s["logprob_grad"] = (normal(rows) - 1).to(acc) / rows
            s["entropy_grad"] = normal(rows).to(acc) / rows if c["entropy"] else None
            xd = x.to(dt).double()  # what the forward pass kept
            lse = torch.logsumexp(xd, 1)
            s["entropy"] = (lse - (torch.exp(xd - lse[:, None]) * xd).sum(1)).to(acc)
            s["lse"] = lse.to(acc)
            del xd
            s["logits_grad"] = _empty(rows, vocab, c["pad"], dt)
        s["logits"] = _pitched(x.to(dt), c["pad"])
        s["targets"] = targets
    return s


# ---- the framework's calls ----------------------------------------------------------------------------------------------

_dev = None


def _device():
    """The framework's device and stream, opened once as a program does at its start."""
    global _dev
    if _dev is None:
        from wekua_amd import raw
        _dev = raw.Device(0)
    return _dev


def _run_own(s):
    c, dev = s["case"], _device()
    if c["op"] == "dropout":
        shape = (1, c["rows"], c["cols"])
        rp = c["cols"] + c["pad"]
        sp = c["rows"] * rp
        dev.dropout(c["dtype"], shape, s["x"], rp, sp, s["y"], rp, sp, c["p"], s["seed"], s["offset"])
        if not c["back"]:
            return s["y"]
        dev.dropout(c["dtype"], shape, s["dy"], rp, sp, s["dx"], rp, sp, c["p"], s["seed"], s["offset"])
        return s["y"], s["dx"]
    if c["op"] == "quantize":
        dev.f8_quantize(c["dtype"], c["rows"], c["cols"], s["x"], c["cols"] + c["pad"], c["block_rows"], s["q"], s["q"].shape[1],
                        s["scales"], s["scales"].shape[1])
        return s["q"][:, :c["cols"]].view(torch.float8_e4m3fn).float(), s["scales"]
    if c["op"] == "gemm_f8":
        dev.gemm_f8(c["m"], c["n"], c["k"], s["a"], s["a"].shape[1], s["sa"], s["sa"].shape[1], s["b"], s["b"].shape[1], s["sb"],
                    s["sb"].shape[1], c["out"], s["out"], c["n"], s["bias"], {"none": -1, "sigmoid": 0, "tanh": 1}[c["act"]])
        return s["out"]
    rp = c["vocab"] + c["pad"]
    if c["op"] == "logprobs":
        dev.token_logprobs(c["dtype"], c["rows"], c["vocab"], s["logits"], rp, s["targets"], "i32", s["logprob"], s["lse"], s["entropy"],
                           s["top"], s["top_ids"], s["top_logprobs"], s["workspace"], WORKSPACE)
        return s["logprob"], s["lse"], s["entropy"], s["top_ids"], s["top_logprobs"]
    dev.token_logprobs_grad(c["dtype"], c["rows"], c["vocab"], s["logits"], rp, s["targets"], "i32", s["lse"], s["entropy"],
                            s["logprob_grad"], s["entropy_grad"], s["logits_grad"], rp)
    return s["logits_grad"]


# ---- the plain forms ------------------------------------------------------------------------------------------------------

def _mul32(a, b):
    """(high, low) 32-bit words of the product of a constant and 32-bit words held in int64."""
    p = a * b  # wraps past 2^63; the words come out right
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _philox(blocks, seed, offset):
    """Philox4x32 with seven rounds: the four words of counters (block, offset) under key `seed`, one row per block."""
    c = torch.arange(blocks, device="cuda", dtype=torch.int64)
    x0, x1 = c & 0xFFFFFFFF, c >> 32
    x2, x3 = torch.full_like(c, offset & 0xFFFFFFFF), torch.full_like(c, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(7):
        h0, l0 = _mul32(0xD2511F53, x0)
        h1, l1 = _mul32(0xCD9E8D57, x2)
        x0, x1, x2, x3 = h1 ^ x1 ^ k0, l1, h0 ^ x3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack((x0, x1, x2, x3), 1)


def _plain_dropout(s):
    c = s["case"]
    n = c["rows"] * c["cols"]
    words = _philox((n + 3) // 4, s["seed"], s["offset"]).reshape(-1)[:n].reshape(c["rows"], c["cols"])
    keep = words >= int(c["p"] * 2 ** 32)
    wide = torch.float64 if c["dtype"] == "f64" else torch.float32
    scale = torch.tensor(1 / (1 - c["p"]) if c["p"] < 1 else 0.0, dtype=torch.float64).to(wide).item()

    def through(x):
        return torch.where(keep, x.to(wide) * scale, 0.0).to(x.dtype)

    return (through(s["x"]), through(s["dy"])) if c["back"] else through(s["x"])


def _power(e):
    """2^e in 32 bits, by its exponent field (e from -126 on)."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_quantize(s):
    c = s["case"]
    x = s["x"].float()
    rows, cols, br = c["rows"], c["cols"], c["block_rows"]
    rb, cb = -(-rows // br), _blocks(cols)
    padded = torch.zeros((rb * br, cb * BLOCK), device="cuda")
    padded[:rows, :cols] = x
    amax = padded.abs().reshape(rb, br, cb, BLOCK).amax((1, 3))
    f, e = torch.frexp(amax)  # amax = f 2^e, f in [1/2, 1); the format's largest value is 7/8 2^9
    e = torch.clamp(e - 8 - (f <= 0.875).int(), min=-126)
    e = torch.where(amax == 0, 0, e)
    down = _power(-e).repeat_interleave(br, 0).repeat_interleave(BLOCK, 1)
    return (padded * down)[:rows, :cols].to(torch.float8_e4m3fn).float(), _power(e)


def _plain_gemm_f8(s):
    c = s["case"]
    a = s["a"][:, :c["k"]].view(torch.float8_e4m3fn).float() * s["sa"].repeat_interleave(BLOCK, 1)[:, :c["k"]]
    b = s["b"][:, :c["k"]].view(torch.float8_e4m3fn).float() * s["sb"].repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[:c["n"], :c["k"]]
    y = a @ b.t()
    if c["bias"]:
        y = y + s["bias"]
    y = 1 / (1 + torch.exp(-y)) if c["act"] == "sigmoid" else torch.tanh(y) if c["act"] == "tanh" else y
    return y.to(s["out"].dtype)


def _plain_logprobs(s):
    x = s["logits"]
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    z = x.to(acc)
    m = z.amax(1, keepdim=True)
    empty = m == -math.inf
    d = z - torch.where(empty, 0.0, m)
    e = torch.exp(d)
    total = e.sum(1, dtype=torch.float64)  # long sums, of which the small rest counts
    log_total = torch.log(total)
    weighted = torch.where(e > 0, e * d, 0.0).sum(1, dtype=torch.float64)
    empty = empty[:, 0]
    lse = torch.where(empty, -math.inf, m[:, 0].double() + log_total)
    entropy = torch.where(empty, 0.0, log_total - weighted / total)
    t = s["targets"].long()
    score = d.gather(1, t.clamp(min=0)[:, None])[:, 0].double() - log_total
    logprob = torch.where(t < 0, 0.0, torch.where(empty, -math.inf, score)).to(acc)
    lse, entropy = lse.to(acc), entropy.to(acc)
    if not s["top"]:
        return logprob, lse, entropy, None, None
    # the largest scores, equal ones by lowest index: sorted without change of order among equals
    if x.dtype == torch.float64:
        order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :s["top"]]
    else:  # one whole number of both: the score's bits in order above, the index counted down below
        bits = (z + 0.0).view(torch.int32).long()
        key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * 2 ** 31 + (2 ** 31 - 1 - torch.arange(z.shape[1], device="cuda"))
        order = torch.topk(key, s["top"], 1).indices
    score = d.gather(1, order).double() - log_total[:, None]
    gone = z.gather(1, order) == -math.inf
    return logprob, lse, entropy, torch.where(gone, -1, order).to(torch.int32), torch.where(gone, -math.inf, score).to(acc)


def _plain_logprobs_grad(s):
    x = s["logits"]
    acc = s["lse"].dtype
    d = x.to(acc) - s["lse"][:, None]
    p = torch.exp(d)
    t = s["targets"].long()
    w = torch.where(t < 0, 0.0, s["logprob_grad"])
    out = -w[:, None] * p
    out.scatter_add_(1, t.clamp(min=0)[:, None], w[:, None])
    if s["entropy_grad"] is not None:
        out -= s["entropy_grad"][:, None] * torch.where(p > 0, p * (d + s["entropy"][:, None]), 0.0)
    return out.to(x.dtype)


_PLAIN = {"dropout": _plain_dropout, "quantize": _plain_quantize, "gemm_f8": _plain_gemm_f8, "logprobs": _plain_logprobs,
          "logprobs_grad": _plain_logprobs_grad}


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["op"]](s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def _exact_keep(c, s):
    """Which elements stay, from Philox4x32-7 in numpy's unsigned whole numbers."""
    n = c["rows"] * c["cols"]
    u = np.uint64
    ctr = np.zeros((4, (n + 3) // 4), dtype=u)
    ctr[0] = np.arange(ctr.shape[1], dtype=u)
    ctr[2] = u(s["offset"])
    key, low = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32], u(0xFFFFFFFF)
    for r in range(7):
        a, b = u(0xD2511F53) * ctr[0], u(0xCD9E8D57) * ctr[2]
        k = [u((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF), u((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF)]
        ctr = np.stack(((b >> u(32)) ^ ctr[1] ^ k[0], b & low, (a >> u(32)) ^ ctr[3] ^ k[1], a & low))
    return torch.from_numpy((ctr.T.reshape(-1)[:n] >= u(int(c["p"] * 2 ** 32))).reshape(c["rows"], c["cols"])).cuda()


def _exact_e4m3(v):
    """v rounded to the nearest value of the 8-bit format, ties to even: three fraction bits, exponents from -6."""
    _, e = torch.frexp(v)
    step = ((torch.clamp(e.long() - 1, min=-6) - 3 + 1023) << 52).view(torch.float64)
    return torch.round(v / step) * step


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "dropout":
        keep = _exact_keep(c, s)
        got = [torch.where(keep, s[n].double() / (1 - c["p"]) if c["p"] < 1 else 0.0, 0.0) for n in (("x", "dy") if c["back"] else ("x",))]
        return tuple(got) if c["back"] else got[0]
    if c["op"] == "quantize":
        x = torch.nn.functional.pad(s["x"].double(), (0, -c["cols"] % BLOCK, 0, -c["rows"] % c["block_rows"]))
        blocks = x.unflatten(0, (-1, c["block_rows"])).unflatten(2, (-1, BLOCK))
        amax = blocks.abs().amax((1, 3), keepdim=True)
        # the smallest power of two under which the block's largest value fits: counted among all of them
        powers = torch.tensor([2.0 ** e for e in range(-126, 121)], dtype=torch.float64, device="cuda")
        at = torch.searchsorted(powers * E4M3_MAX, amax).clamp(max=len(powers) - 1)
        scale = torch.where(amax > 0, powers[at], 1.0)
        codes = _exact_e4m3(blocks / scale).flatten(2, 3).flatten(0, 1)[:c["rows"], :c["cols"]]
        return codes, scale[:, 0, :, 0]
    if c["op"] == "gemm_f8":
        k = c["k"]
        at = torch.arange(k, device="cuda") // BLOCK
        a = s["a"][:, :k].view(torch.float8_e4m3fn).double() * s["sa"].double()[:, at]
        b = s["b"][:, :k].view(torch.float8_e4m3fn).double() * s["sb"].double()[torch.arange(c["n"], device="cuda") // BLOCK][:, at]
        y = torch.matmul(a, b.t()) + (s["bias"].double() if c["bias"] else 0.0)
        return torch.sigmoid(y) if c["act"] == "sigmoid" else torch.tanh(y) if c["act"] == "tanh" else y
    z = s["logits"].double()
    lp = torch.log_softmax(z, 1)
    t = s["targets"].long()
    if c["op"] == "logprobs":
        empty = torch.isinf(z).all(1)
        pick = lp[torch.arange(len(t), device="cuda"), t.clamp(min=0)]
        logprob = torch.where(t < 0, 0.0, torch.where(empty, -math.inf, pick))
        entropy = torch.where(empty, 0.0, -torch.nan_to_num(torch.exp(lp) * lp, nan=0.0).sum(1))
        best = torch.sort(lp, dim=1, descending=True, stable=True).values[:, :s["top"]] if s["top"] else None
        if best is not None:
            best = torch.where(empty[:, None], -math.inf, best)
        return logprob, torch.logsumexp(z, 1), entropy, None, best
    # the given statistics are inputs: the gradient is the formula's at them
    lp = z - s["lse"].double()[:, None]
    p = torch.exp(lp)
    hot = torch.zeros_like(p)
    hot[torch.arange(len(t), device="cuda"), t.clamp(min=0)] = (t >= 0).double()
    out = torch.where(t >= 0, s["logprob_grad"].double(), 0.0)[:, None] * (hot - p)
    if c["entropy"]:
        out = out - s["entropy_grad"].double()[:, None] * p * (lp + s["entropy"].double()[:, None])
    return out
