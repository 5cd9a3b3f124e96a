"""Operators of language models served in 8 bits: hidden states to codes, linear
layers on codes, logits to tokens.

  linear   rows brought to 8-bit codes with a scale each, with what stands in front
           of a layer (nothing, an RMS norm, a swish gate), and the layer's product
  product  a layer's product alone, of codes that are there already
  sample   a token for each row of logits: temperature, top-k, top-p, min-p

Codes of activations have a scale for each row (token), codes of weights one for
each column (channel).  Rows of logits have their own settings, and a number in
[0, 1) each that their token follows from.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6
_held = {}


# ---- cases -------------------------------------------------------------------
def _linear(front, dtype, m, k, n, out, bias=False):
    return {"kind": "linear", "front": front, "dtype": dtype, "m": m, "k": k, "n": n, "out": out, "bias": bias, "along_k": True}


def _product(m, k, n, out, bias=False, along_k=True):
    return {"kind": "product", "m": m, "k": k, "n": n, "out": out, "bias": bias, "along_k": along_k}


def _sample(dtype, rows, words, spread, pad=0):
    return {"kind": "sample", "dtype": dtype, "rows": rows, "words": words, "spread": spread, "pad": pad}


def listed():
    return [dict(c, name=name) for name, c in (
        # one chat, one token: norm and the product of queries, keys and values; one call's latency
        ("linear_f16_token", _linear("rms", "f16", 1, 2048, 2560, "f16")),
        # a step of decoding for a batch of chats: norm and the way up
        ("linear_bf16_step", _linear("rms", "bf16", 48, 4096, 12288, "bf16")),
        # the gate and the way down of a batch of prompts
        ("linear_bf16_gate", _linear("gate", "bf16", 4000, 12288, 4096, "bf16")),
        # odd sizes, rows in f32, with a bias
        ("linear_f32_odd", _linear("none", "f32", 333, 1001, 777, "bf16", bias=True)),
        # logits of a few chats over a large vocabulary
        ("product_f32_head", _product(5, 4096, 131072, "f32")),
        # weights that lie along the channels, ragged sizes, a bias
        ("product_f16_ragged", _product(777, 1008, 1400, "f16", bias=True, along_k=False)),
        # a prompt
        ("product_bf16_prompt", _product(4096, 4096, 8192, "bf16")),
        # what a server gathers of prompts in a step
        ("product_bf16_prompts", _product(16384, 4096, 12288, "bf16", bias=True)),
        # one chat's next token
        ("sample_f32_one", _sample("f32", 1, 65536, 3.0)),
        # a few chats over an odd vocabulary in rows with some room behind
        ("sample_f16_odd", _sample("f16", 7, 100003, 2.0, pad=29)),
        # a step of decoding
        ("sample_bf16_step", _sample("bf16", 48, 131072, 3.0)),
        # many answers to the same question, drawn widely
        ("sample_f32_many", _sample("f32", 256, 131072, 1.2)),
    )]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over its logarithm: most are a multiple of 64 or 16 as layers have them, others any."""
    n = _log(rng, lo, hi)
    step = rng.choice([64, 64, 16, 1])
    return max(step, n // step * step)


def draw(rng):
    """One of the three kinds over its whole range, cut to what the listed ones cost."""
    kind = rng.choice(["linear", "linear", "product", "product", "sample", "sample"])
    if kind == "sample":
        c = _sample(rng.choice(["f32", "f32", "bf16", "f16"]), _log(rng, 1, 256), _log(rng, 500, 200000),
                    round(rng.uniform(0.8, 4.0), 2), rng.choice([0, 0, rng.randint(1, 64)]))
        while c["rows"] * c["words"] > 256 * 131072:
            c["rows"] = (c["rows"] + 1) // 2
        return c
    m, k, n = _log(rng, 1, 16384), _size(rng, 64, 16384), _size(rng, 64, 32768)
    if kind == "linear":
        front = rng.choice(["none", "rms", "rms", "gate"])
        c = _linear(front, rng.choice(["bf16", "bf16", "f16", "f32"]), m, k, n, rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.3)
    else:
        c = _product(m, k, n, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.3, rng.random() < 0.75)
    while 2 * c["m"] * c["k"] * c["n"] > 1.6e12:
        c["m"] = (c["m"] + 1) // 2
    return c


# ---- inputs ------------------------------------------------------------------
def _normal(gen, shape, dtype=torch.float32, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _uniform(gen, n):
    return torch.rand([n], generator=gen, device="cuda", dtype=torch.float32)


def _codes(gen, rows, k):
    """Codes as rows of about normal values have them: the largest of a row at 127."""
    return _normal(gen, [rows, k], std=32.0).round_().clamp_(-127, 127).to(torch.int8)


def _pick(gen, n, values, dtype):
    at = torch.randint(0, len(values), [n], generator=gen, device="cuda")
    return torch.tensor(values, device="cuda", dtype=dtype)[at]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "sample":
        b, v = c["rows"], c["words"]
        whole = _normal(gen, [b, v + c["pad"]], std=c["spread"])
        # a few words that fit
        at = torch.randint(0, v, [b, 24], generator=gen, device="cuda")
        whole.scatter_add_(1, at, _uniform(gen, b * 24).view(b, 24).mul_(4.0 * c["spread"]))
        s["logits"] = whole.to(_DT[c["dtype"]])[:, :v]
        s["uniform"] = _uniform(gen, b)
        s["temperature"] = _pick(gen, b, [0.0, 0.6, 0.8, 1.0, 1.0, 1.3], torch.float32)
        s["top_k"] = _pick(gen, b, [0, 0, 1, 40, 200, v // 3], torch.int32)
        s["top_p"] = _pick(gen, b, [1.0, 0.95, 0.9, 0.8, 0.5], torch.float32)
        s["min_p"] = _pick(gen, b, [0.0, 0.0, 0.02, 0.1], torch.float32)
        s["token"] = torch.empty([b], device="cuda", dtype=torch.int32)
        s["probability"] = torch.empty([b], device="cuda", dtype=torch.float32)
        return s
    m, k, n = c["m"], c["k"], c["n"]
    if c["kind"] == "linear":
        dt = _DT[c["dtype"]]
        if c["front"] == "gate":  # what one product of both gives
            s["x"], s["up"] = _normal(gen, [m, 2 * k], dt).split(k, 1)
        else:
            s["x"] = _normal(gen, [m, k], dt)
        if c["front"] == "rms":
            s["weight"] = _normal(gen, [k], std=0.1).add_(1.0).to(dt)
        s["a"] = torch.empty([m, k], device="cuda", dtype=torch.int8)
        s["a_scale"] = torch.empty([m], device="cuda", dtype=torch.float32)
    else:
        s["a"] = _codes(gen, m, k)
        s["a_scale"] = _uniform(gen, m).mul_(0.01).add_(0.02)
    s["b"] = _codes(gen, n, k).T if c["along_k"] else _codes(gen, k, n)
    s["b_scale"] = _uniform(gen, n).mul_(0.2).add_(0.9).mul_(0.03 / math.sqrt(k))
    if c["bias"]:
        s["bias"] = _normal(gen, [n], _DT[c["out"]], 0.2)
    s["out"] = torch.empty([m, n], device="cuda", dtype=_DT[c["out"]])
    return s


# ---- the framework's calls ---------------------------------------------------
def _plan(s):
    """Descriptors, workspace and the pointers: what a program makes once for buffers that it keeps."""
    from fusilli_amd import capi
    c = s["case"]
    if not _held:
        _held["stream"] = torch.cuda.Stream()
        _held["ctx"] = capi.Context(torch.cuda.current_device(), _held["stream"].cuda_stream)
    _held["stream"].wait_stream(torch.cuda.current_stream())
    ctx = _held["ctx"]
    types = {torch.bfloat16: capi.BFLOAT16, torch.float16: capi.HALF, torch.float32: capi.FLOAT, torch.int8: capi.INT8}
    desc = {n: capi.TensorDesc.make(t.shape, t.stride(), types[t.dtype]) for n, t in s.items()
            if isinstance(t, torch.Tensor) and t.dtype in types}
    p = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    if c["kind"] == "sample":
        d = capi.SampleDesc()
        d.logits = desc["logits"]
        d.has_temperature = d.has_top_k = d.has_top_p = d.has_min_p = 1
        s["room"] = room = torch.empty(max(ctx.sample_workspace(d), 1), device="cuda", dtype=torch.uint8)
        ws = room.data_ptr()

        def call():
            ctx.sample(d, p["logits"], p["uniform"], p["token"], temperature=p["temperature"], top_k=p["top_k"],
                       top_p=p["top_p"], min_p=p["min_p"], probability=p["probability"], workspace=ws)
        s["plan"] = call
        return call
    d = capi.MatmulQuantizedDesc()
    d.a, d.b, d.c, d.out = desc["a"], desc["b"], desc["out"], desc["out"]
    d.out_dtype = types[s["out"].dtype]
    d.a_scale_stride = d.b_scale_stride = 1
    if "bias" in s:
        d.has_bias, d.bias_dtype, d.bias_stride = 1, types[s["bias"].dtype], 1

    def multiply():
        ctx.matmul_quantized(d, p["a"], p["b"], p["a_scale"], p["b_scale"], p["out"], bias=p.get("bias"))
    call = multiply
    if c["kind"] == "linear":
        f = capi.QuantizeRowsDesc()
        f.x, f.q, f.scale_stride = desc["x"], desc["a"], 1
        f.front = capi.QUANTIZE_FRONT[{"none": "NONE", "rms": "RMSNORM", "gate": "SWISH_GATE"}[c["front"]]]
        if "up" in s:
            f.up = desc["up"]
        if "weight" in s:
            f.has_weight, f.weight_dtype, f.weight_stride, f.epsilon = 1, types[s["weight"].dtype], 1, _EPS

        def call():
            ctx.quantize_rows(f, p["x"], p["a"], p["a_scale"], up=p.get("up"), weight=p.get("weight"))
            multiply()
    s["plan"] = call
    return call


# ---- the plain forms ---------------------------------------------------------
def _plain_quantize(s):
    y = s["x"].float()
    if "weight" in s:
        y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + _EPS) * s["weight"].float()
    elif "up" in s:
        y = y / (1.0 + torch.exp(-y)) * s["up"].float()
    most = y.abs().amax(1, keepdim=True)
    by = torch.where(most > 0, 127.0 / most, torch.zeros_like(most))
    s["a"].copy_((y * by).round_())
    s["a_scale"].copy_((most / 127.0)[:, 0])


def _plain_product(s):
    y = s["a"].float() @ s["b"].float()
    y.mul_(s["a_scale"][:, None]).mul_(s["b_scale"])
    if "bias" in s:
        y.add_(s["bias"].float())
    s["out"].copy_(y)


def _plain_sample(s):
    l = s["logits"].float()
    v = l.shape[1]
    l, order = torch.sort(l, dim=1, descending=True, stable=True)
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])[:, None].double()
    l = l.double()
    w = ((l - l[:, :1]) / t).exp_()
    run = w.cumsum(1)
    place = torch.arange(v, device="cuda")
    # the first k, of them the shortest prefix with a share p, of that what reaches min_p of the largest
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > v), v, s["top_k"]).long()[:, None]
    share = s["top_p"].double()[:, None] * run.gather(1, k - 1)
    p = torch.where(s["top_p"][:, None] < 1, (run < share).sum(1, keepdim=True) + 1, v)
    m = (w >= s["min_p"].double()[:, None]).sum(1, keepdim=True)
    kept = torch.minimum(torch.minimum(k, p), m).clamp_(1, v)
    kept = torch.where(greedy[:, None], torch.ones_like(kept), kept)
    total = run.gather(1, kept - 1)
    at = ((run <= s["uniform"].double()[:, None] * total) & (place < kept)).sum(1, keepdim=True)
    at = torch.minimum(at, kept - 1)
    s["token"].copy_(order.gather(1, at)[:, 0])
    s["probability"].copy_((w.gather(1, at) / total)[:, 0])


def _outputs(s):
    if "token" in s:
        return {"token": s["token"], "probability": s["probability"]}
    return {"out": s["out"], "a_scale": s["a_scale"]} if s["case"]["kind"] == "linear" else s["out"]


def run(state):
    s = state
    if own:
        (s.get("plan") or _plan(s))()
        return _outputs(s)
    if s["case"]["kind"] == "sample":
        _plain_sample(s)
        return _outputs(s)
    if s["case"]["kind"] == "linear":
        _plain_quantize(s)
    _plain_product(s)
    return _outputs(s)


# ---- what a pass cannot do without -------------------------------------------
def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (c["words"] * size[c["dtype"]] + 28), "flops": 0}
    m, k, n = c["m"], c["k"], c["n"]
    b = k * n + m * n * size[c["out"]] + 4 * (m + n) + (n * size[c["out"]] if c["bias"] else 0)
    if c["kind"] == "product":
        b += m * k
    else:  # (codes between the two are a pass's own business)
        b += (2 if c["front"] == "gate" else 1) * m * k * size[c["dtype"]] + (k * size[c["dtype"]] if c["front"] == "rms" else 0)
    return {"bytes": b, "flops": 2 * m * k * n}


# ---- the definition in 64 bits -----------------------------------------------
def _exact_row(logits, u, t, k, p, least):
    """(place of the token among the ordered, its probability) of one row on the host."""
    import numpy as np
    l = logits[np.lexsort((np.arange(logits.size), -logits))]
    if t <= 0:
        return 1.0
    w = np.exp((l - l[0]) / t)
    n = k if 0 < k < w.size else w.size
    if p < 1:
        n = min(n, int(np.searchsorted(np.cumsum(w[:n]), p * w[:n].sum(), side="left")) + 1)
    n = max(1, min(n, int((w >= least).sum())))
    at = min(int(np.searchsorted(np.cumsum(w[:n]), u * w[:n].sum(), side="right")), n - 1)
    return float(w[at] / w[:n].sum())


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "sample":
        rows = s["logits"].double().cpu().numpy()
        each = zip(rows, *(s[x].double().tolist() for x in ("uniform", "temperature", "top_k", "top_p", "min_p")))
        chances = [_exact_row(row, u, t, int(k), p, least) for row, u, t, k, p, least in each]
        return {"token": None, "probability": torch.tensor(chances, dtype=torch.float64)}
    a, scale = s["a"].double(), s["a_scale"].double()
    if c["kind"] == "linear":
        y = s["x"].double()
        if c["front"] == "rms":
            y = y / (y.pow(2).sum(1, keepdim=True) / c["k"] + _EPS).sqrt() * s["weight"].double()
        if c["front"] == "gate":
            y = y * torch.sigmoid(y) * s["up"].double()
        scale = y.abs().max(1).values / 127
        a = (y / scale.clamp(min=1e-300)[:, None]).round()
    out = torch.empty([c["m"], c["n"]], device="cuda", dtype=torch.float64)
    b = s["b"].double() * s["b_scale"].double()
    for i in range(0, c["m"], 4096):
        out[i:i + 4096] = scale[i:i + 4096, None] * a[i:i + 4096] @ b
    if c["bias"]:
        out += s["bias"].double()
    return {"out": out, "a_scale": scale} if c["kind"] == "linear" else out
