"""Three operators of a training step, as cases with sizes, in plain torch and as calls of this framework.

* ``linear``    a linear layer in 8-bit floating point: activations and gradients are quantised with one power-of-two scale for
                each 1 x 128 piece, weights with one for each 128 x 128 block; product, input gradient and weight gradient.
* ``forward``   the forward pass of such a layer alone, as in an evaluation pass.
* ``quantize``  the quantisation alone, along the rows and along the columns of an activation.
* ``ortho``     orthogonalising a batch of matrices by Newton-Schulz products.
* ``muon``      the optimizer step built on it: momentum, orthogonalised update, decay, fp32 master and bf16 weight.
* ``embedding`` lookup with a scale, and the gradient added to the table's rows by sorted tokens.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 128
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
MOMENTUM, DECAY, LR = 0.95, 0.01, 2e-4      # the last two: what TrainConfig has
#: (bits of the mantissa, smallest exponent, exponent e of the largest value 0.875 * 2^e, torch type)
FORMATS = {"e4m3": (3, -6, 9, torch.float8_e4m3fn), "e5m2": (2, -14, 16, torch.float8_e5m2)}


def _linear(name, tokens, n_in, n_out, grad="e4m3"):
    return {"name": name, "kind": "linear", "tokens": tokens, "n_in": n_in, "n_out": n_out, "grad": grad}


def _embedding(name, tokens, hidden, vocab, start, scale, skew, padded):
    return {"name": name, "kind": "embedding", "tokens": tokens, "hidden": hidden, "vocab": vocab, "start": start, "scale": scale,
            "skew": skew, "padded": padded}


def listed():
    return [
        # gate and up projection of the configured 8B model over one nanobatch of 2 x 4096 tokens
        _linear("linear_8b_fc1", 8192, 4096, 28672),
        # the same layer of the 1.7B model over a ragged batch, gradients in the format with the wider range
        _linear("linear_ragged", 3799, 2048, 12288, "e5m2"),
        # a short ragged batch through a small layer: launches decide
        _linear("linear_small", 328, 1032, 776),
        # evaluation of a few tokens: the weight is what has to be read
        {"name": "forward_few", "kind": "forward", "tokens": 17, "n_in": 4096, "n_out": 6144},
        # activations behind the 8B model's SwiGLU, along the rows for the product and along the columns for the weight gradient
        {"name": "quantize_acts", "kind": "quantize", "rows": 8192, "cols": 14336},
        # gate and up projection of the smoke model: launches decide
        {"name": "ortho_smoke", "kind": "ortho", "batch": 1, "rows": 2048, "cols": 512},
        # matrices of sizes that fit no tile
        {"name": "ortho_ragged", "kind": "ortho", "batch": 3, "rows": 333, "cols": 1000},
        # optimizer step of the 8B model's QKV projection (more rows than columns) and of its down projection (fewer)
        {"name": "muon_8b_qkv", "kind": "muon", "rows": 6144, "cols": 4096},
        {"name": "muon_8b_fc2", "kind": "muon", "rows": 4096, "cols": 14336},
        # the smoke model's table under uniform tokens
        _embedding("embedding_smoke", 512, 512, 2048, 0, 1.0, 1, 0.0),
        # the 8B model's table, 2 x 4096 tokens whose frequencies fall off as those of a text
        _embedding("embedding_8b", 8192, 4096, 128256, 0, 64.0, 4, 0.0),
        # third of eight shards of the 1.7B model's table, a batch of 8 x 4096 of which a third is padding
        _embedding("embedding_shard", 32768, 2048, 18992, 37984, 1.0, 2, 0.33),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "forward", "quantize", "ortho", "muon", "embedding", "embedding"))
    if kind in ("linear", "forward"):
        # feature counts are multiples of 8: rows of bf16 operands start on 16 bytes
        while True:
            c = {"kind": kind, "tokens": _log_int(rng, 1, 9000), "n_in": 8 * _log_int(rng, 8, 1792),
                 "n_out": 8 * _log_int(rng, 8, 3584)}
            if kind == "linear":
                c["grad"] = rng.choice(("e4m3", "e4m3", "e5m2"))
            if c["tokens"] * c["n_in"] * c["n_out"] <= 8192 * 4096 * 28672:
                return c
    if kind == "quantize":
        while True:
            c = {"kind": kind, "rows": _log_int(rng, 1, 20000), "cols": 8 * _log_int(rng, 1, 2048)}
            if c["rows"] * c["cols"] <= 8192 * 14336:
                return c
    if kind in ("ortho", "muon"):
        while True:
            c = {"kind": kind, "rows": _log_int(rng, 16, 14336), "cols": _log_int(rng, 16, 14336)}
            if kind == "ortho":
                c["batch"] = rng.choice((1, 1, 2, 5))
            a, b = min(c["rows"], c["cols"]), max(c["rows"], c["cols"])
            if c.get("batch", 1) * a * a * (2 * b + a) <= 4096 * 4096 * (2 * 14336 + 4096):
                return c
    shards = rng.choice((1, 1, 4, 8))
    vocab = _log_int(rng, 500, 150000) // shards + 1
    return {"kind": "embedding", "tokens": _log_int(rng, 1, 33000), "hidden": 8 * _log_int(rng, 8, 512), "vocab": vocab,
            "start": vocab * rng.randint(0, shards - 1), "scale": rng.choice((1.0, 64.0, 45.254833995939045)),
            "skew": rng.choice((1, 2, 4)), "padded": rng.choice((0.0, 0.0, 0.3, 0.9))}


# ----------------------------------------------------------------------------- states
def prepare(case, seed):
    torch.cuda.set_device(DEVICE)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=gen)

    def outliers(*shape, std):       # a few features are far larger than the others, as in trained models
        t = randn(*shape, std=std)
        hot = torch.rand(shape[-1], device=DEVICE, generator=gen) < 0.01
        return t.mul_(torch.where(hot, 30.0, 1.0).to(t.dtype))

    kind = case["kind"]
    if kind in ("linear", "forward"):
        t, i, o = case["tokens"], case["n_in"], case["n_out"]
        s = {"x": outliers(t, i, std=1.0), "w": randn(o, i, std=0.02)}
        if kind == "linear":
            s |= {"dy": outliers(t, o, std=1e-4), "main_grad": randn(o, i, std=1e-3, dtype=torch.float32)}
    elif kind == "quantize":
        s = {"x": outliers(case["rows"], case["cols"], std=1.0)}
    elif kind == "ortho":
        s = {"x": randn(case["batch"], case["rows"], case["cols"], std=1e-3, dtype=torch.float32)}
    elif kind == "muon":
        shape = (case["rows"], case["cols"])
        s = {"g": randn(*shape, std=1e-3, dtype=torch.float32), "m": randn(*shape, std=3e-3, dtype=torch.float32),
             "master": randn(*shape, std=0.02, dtype=torch.float32)}
        s["p"] = s["master"].to(torch.bfloat16)
    else:
        t, h, v, start = case["tokens"], case["hidden"], case["vocab"], case["start"]
        total = max(v, start + v, 4 * start)        # tokens of other shards are in the batch too
        u = torch.rand(t, device=DEVICE, generator=gen, dtype=torch.float64)
        tok = ((u ** case["skew"]) * total).long().clamp_(max=total - 1)
        tok = tok[torch.randperm(t, device=DEVICE, generator=gen)]
        if case["padded"]:
            tok[int(t * (1 - case["padded"])):] = start + v // 2
        s = {"tokens": tok, "weight": randn(v, h, std=0.02), "dout": randn(t, h, std=1e-3),
             "grad": randn(v, h, std=1e-4, dtype=torch.float32)}
    return s | {"case": dict(case)}


# ----------------------------------------------------------------------------- plain forms
def _scale_bytes(exponent):
    """``[rows, pieces]`` exponents + 127 as they are laid out for the product: four pieces of 128 rows are 512 bytes, row ``r``
    of them at ``(r % 32) * 16 + (r // 32) * 4``; what lies past the edge is 0."""
    r, p = exponent.shape
    rt, pt = -(-r // 128), -(-p // 4)
    e = torch.zeros(rt * 128, pt * 4, dtype=torch.uint8, device=exponent.device)
    e[:r, :p] = (exponent + 127).to(torch.uint8)
    return e.view(rt, 4, 32, pt, 4).permute(0, 3, 2, 1, 4).contiguous()


def _power(e):
    """2 to whole exponents, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64).float()


def _quantize(x, fmt, square=False):
    """Rows of ``x`` in 8 bits: values, exponents of the scales of 128 columns (and 128 rows, if ``square``), what they stand for."""
    _, _, top, dtype = FORMATS[fmt]
    r, c = x.shape
    pad = torch.zeros(-(-r // 128) * 128 if square else r, -(-c // 128) * 128, device=x.device)
    pad[:r, :c] = x.float()
    blocks = pad.view(-1, 128 if square else 1, pad.shape[1] // 128, 128)
    amax = blocks.abs().amax(dim=(1, 3))
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - top + (m > 0.875), -127).clamp(min=-127)
    if square:
        e = e.repeat_interleave(128, 0)[:r]
    pad = pad[:r].view(r, -1, 128)
    q = (pad * _power(-e)[:, :, None]).to(dtype)
    back = (q.float() * _power(e)[:, :, None]).view(r, -1)[:, :c]
    return q.view(r, -1)[:, :c].contiguous(), _scale_bytes(e), back


def _newton_schulz(x):
    a, b, c = COEFFICIENTS
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    for _ in range(STEPS):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def _muon_scale(case):
    return 0.2 * math.sqrt(max(case["rows"], case["cols"]))


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _run_own(state, case, kind)
    if kind in ("linear", "forward"):
        x, w = state["x"], state["w"]
        _, _, xr = _quantize(x, "e4m3")
        _, _, wr = _quantize(w, "e4m3", square=True)
        y = (xr @ wr.t()).to(x.dtype)
        if kind == "forward":
            return {"y": y}
        dy, fmt = state["dy"], case["grad"]
        _, _, dr = _quantize(dy, fmt)
        dx = (dr @ wr).to(dy.dtype)
        del dr
        _, _, dc = _quantize(dy.t(), fmt)
        _, _, xc = _quantize(x.t(), "e4m3")
        state["main_grad"].addmm_(dc, xc.t())
        return {"y": y, "dx": dx, "dw": state["main_grad"]}
    if kind == "quantize":
        q, s, _ = _quantize(state["x"], "e4m3")
        qc, sc, _ = _quantize(state["x"].t(), "e4m3")
        return {"rows": q, "row_scales": s, "cols": qc, "col_scales": sc}
    if kind == "ortho":
        return {"o": _newton_schulz(state["x"]).to(torch.bfloat16)}
    if kind == "muon":
        m, master = state["m"], state["master"]
        m.mul_(MOMENTUM).add_(state["g"])
        o = _newton_schulz(state["g"] + MOMENTUM * m).to(torch.bfloat16)       # the update, as the operator above returns it
        master.mul_(1 - LR * DECAY).sub_(o, alpha=LR * _muon_scale(case))
        state["p"].copy_(master)
        return {"o": o, "m": m, "master": master, "p": state["p"]}
    idx = state["tokens"] - case["start"]
    here = (idx >= 0) & (idx < case["vocab"])
    idx = torch.where(here, idx, 0)
    out = state["weight"][idx].float() * case["scale"] * here[:, None]
    state["grad"].index_add_(0, idx, state["dout"].float() * case["scale"] * here[:, None])
    return {"out": out.to(torch.bfloat16), "grad": state["grad"]}


def _run_own(state, case, kind):
    from kareus_b200 import kernels as K
    if kind in ("linear", "forward"):
        x, w = state["x"], state["w"]
        if kind == "forward":
            xr, _ = K.fp8_quantize(x)
            wr, _ = K.fp8_quantize(w, square=True)
            return {"y": K.fp8_gemm(xr, wr)}
        xr, xc = K.fp8_quantize(x, cols=True)
        wr, wc = K.fp8_quantize(w, cols=True, square=True)
        y = K.fp8_gemm(xr, wr)
        dr, dc = K.fp8_quantize(state["dy"], cols=True, fmt=case["grad"])
        dx = K.fp8_gemm(dr, wc)
        dw = K.fp8_gemm(dc, xc, accumulate=state["main_grad"])
        return {"y": y, "dx": dx, "dw": dw}
    if kind == "quantize":
        r, c = K.fp8_quantize(state["x"], cols=True)
        return {"rows": r.data, "row_scales": r.scales, "cols": c.data, "col_scales": c.scales}
    if kind == "ortho":
        return {"o": K.orthogonalize(state["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}
    if kind == "muon":
        o = K.muon_step(state["p"], state["g"], state["m"], state["master"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY,
                        scale=_muon_scale(case), nesterov=True, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        return {"o": o, "m": state["m"], "master": state["master"], "p": state["p"]}
    out = K.embedding_fwd(state["tokens"], state["weight"], case["start"], scale=case["scale"])
    K.embedding_bwd(state["dout"], state["tokens"], state["grad"], case["start"], scale=case["scale"], order="sorted")
    return {"out": out, "grad": state["grad"]}


# ----------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind in ("linear", "forward"):
        t, i, o = case["tokens"], case["n_in"], case["n_out"]
        if kind == "forward":
            return {"bytes": 2.0 * (t * i + o * i + t * o), "flops": 2.0 * t * i * o}
        # x, w and dy read, y and dx written in 16 bits; the fp32 gradient read and written
        return {"bytes": 2.0 * (2 * t * i + 2 * t * o + o * i) + 8.0 * o * i, "flops": 6.0 * t * i * o}
    if kind == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": 4.0 * n + n / 64.0, "flops": 4.0 * n}
    if kind in ("ortho", "muon"):
        a, b = sorted((case["rows"], case["cols"]))
        n = case.get("batch", 1)
        # X Xt and its square are symmetric: half of their products
        flops = n * STEPS * (a * a * b + a ** 3 + 2.0 * a * a * b)
        # ortho: fp32 in, bf16 out; muon: gradient read, momentum and master read and written, update and weight written
        return {"bytes": (6.0 if kind == "ortho" else 24.0) * n * a * b, "flops": flops}
    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    rows = min(t, v)
    # looked-up rows read and written in 16 bits, the gradient read in 16 bits, its rows' sums read and written in 32
    return {"bytes": 2.0 * rows * h + 4.0 * t * h + 8.0 * rows * h + 16.0 * t, "flops": 2.0 * t * h}


# ----------------------------------------------------------------------------- 64 bits
def _exact_quantize(x, fmt, square=False):
    """(values in 8 bits, exponents, what they stand for), all in 64 bits, from the definition: the smallest power of two under
    which the piece fits the format, and the nearest value of the format, ties to the even one."""
    mantissa, low, top, _ = FORMATS[fmt]
    x = x.double()
    r, c = x.shape
    largest = 0.875 * 2.0 ** top
    limits = torch.tensor([largest * 2.0 ** k for k in range(-127, 125)], dtype=torch.float64, device=x.device)
    powers = torch.tensor([2.0 ** k for k in range(-160, 161)], dtype=torch.float64, device=x.device)
    exps = torch.empty(r, -(-c // 128), dtype=torch.int64, device=x.device)
    scale = torch.empty(r, c, dtype=torch.float64, device=x.device)
    for p in range(exps.shape[1]):
        piece = x[:, p * 128:(p + 1) * 128].abs().amax(dim=1)
        if square:
            piece = torch.cat([b.amax().expand(b.numel()) for b in piece.split(128)])
        exps[:, p] = torch.bucketize(piece, limits) - 127
        scale[:, p * 128:(p + 1) * 128] = powers[exps[:, p] + 160][:, None]
    v = x / scale
    at = torch.bucketize(v.abs().clamp(min=2.0 ** low), powers, right=True) - 1 - 160       # 2^at <= |v| < 2^(at + 1)
    step = powers[at - mantissa + 160]
    del at
    q = torch.round(v / step) * step
    return q, exps, q * scale


def _exact_ns(x):
    x = x.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            g = x @ x.transpose(-1, -2)
            gx = g @ x
            x = a * x + b * gx + c * (g @ gx)
        else:
            g = x.transpose(-1, -2) @ x
            xg = x @ g
            x = a * x + b * xg + c * (xg @ g)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("linear", "forward"):
        xr = _exact_quantize(s["x"], "e4m3")[2]
        wr = _exact_quantize(s["w"], "e4m3", square=True)[2]
        y = xr @ wr.t()
        if kind == "forward":
            return {"y": y}
        del xr
        dx = _exact_quantize(s["dy"], case["grad"])[2] @ wr
        del wr
        xc = _exact_quantize(s["x"].t(), "e4m3")[2]
        dw = s["main_grad"].double() + _exact_quantize(s["dy"].t(), case["grad"])[2] @ xc.t()
        return {"y": y, "dx": dx, "dw": dw}
    if kind == "quantize":
        return {"rows": _exact_quantize(s["x"], "e4m3")[0], "row_scales": None,
                "cols": _exact_quantize(s["x"].t(), "e4m3")[0], "col_scales": None}
    if kind == "ortho":
        return {"o": _exact_ns(s["x"])}
    if kind == "muon":
        g = s["g"].double()
        m = MOMENTUM * s["m"].double() + g
        o = _exact_ns(g + MOMENTUM * m)
        master = s["master"].double() * (1 - LR * DECAY) - LR * _muon_scale(case) * o
        return {"o": o, "m": m, "master": master, "p": master}
    idx = s["tokens"] - case["start"]
    keep = torch.nonzero((idx >= 0) & (idx < case["vocab"])).flatten()
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=idx.device)
    out[keep] = s["weight"].double()[idx[keep]] * case["scale"]
    grad = s["grad"].double()
    grad.index_put_((idx[keep],), s["dout"].double()[keep] * case["scale"], accumulate=True)
    return {"out": out, "grad": grad}
