"""Serving operators of language models: prompts of different lengths in one
batch, and a key / value cache in pages that single tokens attend over.

  packed  attention over packed prompts, causal or not, grouped heads
  append  positions rotated into queries and keys, keys and values put into
          their pages, in 16 bits or in 4 with a scale and a low value per group
  read    a cache's rows brought back to packed rows (a cached prefix in front
          of a prompt's next chunk, a sequence that moves)
  paged   attention of each sequence's newest tokens over its pages

Sequences share three small tensors: `offsets` (B + 1; where each sequence's
rows start), `lengths` (B; keys in the cache, this call's tokens among them) and
`pages` (B x most pages).  Row i of a sequence's n rows has the place
length - n + i in the cache.
"""
import itertools
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}
_held = {}


# ---- cases -------------------------------------------------------------------
def _heads(dtype, hq, hkv, d):
    return {"dtype": dtype, "hq": hq, "hkv": hkv, "d": d}


def _packed(heads, seqs, longest, mix, causal=True, fused=False):
    return {"kind": "packed", **heads, "seqs": seqs, "longest": longest, "mix": mix, "causal": causal,
            "fused": fused}


def _append(heads, seqs, longest, mix, past, page, group=0, rotary=0, interleaved=False):
    return {"kind": "append", **heads, "seqs": seqs, "longest": longest, "mix": mix, "past": past,
            "page": page, "group": group, "rotary": rotary or heads["d"], "interleaved": interleaved}


def _read(heads, seqs, longest, mix, page, group=0):
    return {"kind": "read", **heads, "seqs": seqs, "longest": longest, "mix": mix, "page": page,
            "group": group}


def _paged(heads, seqs, longest, mix, new, page, group=0):
    return {"kind": "paged", **heads, "seqs": seqs, "longest": longest, "mix": mix, "new": new,
            "page": page, "group": group}


def listed():
    small, wide = _heads("f16", 16, 4, 64), _heads("bf16", 32, 8, 128)
    return [dict(c, name=name) for name, c in (
        # a few short questions at once: one call's latency
        ("packed_f16_short", _packed(small, 5, 100, 1)),
        # what a server gathers in a step: chats of very different lengths
        ("packed_bf16_ragged", _packed(wide, 24, 2048, 2, fused=True)),
        # documents
        ("packed_bf16_long", _packed(wide, 2, 8192, 3, fused=True)),
        # texts to be embedded, every token sees every other
        ("packed_f16_both_ways", _packed(_heads("f16", 12, 12, 64), 32, 512, 4, causal=False)),
        # one token each of some sequences goes into a 16-bit cache
        ("append_f16_tokens", _append(small, 7, 1, 5, 300, 16, rotary=32, interleaved=True)),
        # whole prompts go in: queries and keys rotated on the way
        ("append_bf16_prompts", _append(wide, 24, 2048, 6, 0, 64)),
        # the same into 4 bits, and what the cache then holds
        ("append_bf16_int4_prompts", _append(wide, 24, 2048, 7, 0, 64, group=64)),
        # a short prefix out of a 16-bit cache
        ("read_f16_prefix", _read(small, 3, 200, 8, 16)),
        # long prefixes out of 4 bits
        ("read_bf16_int4_prefixes", _read(wide, 8, 8192, 9, 64, group=64)),
        # one chat, one token
        ("paged_f16_single", _paged(small, 1, 333, 10, 1, 16)),
        # a full step of decoding over 16-bit pages
        ("paged_bf16_decode", _paged(wide, 32, 8192, 11, 1, 16)),
        # more and longer chats in 4 bits, some tokens drafted ahead
        ("paged_bf16_int4_draft", _paged(wide, 64, 16384, 12, 3, 64, group=64)),
    )]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_heads(rng):
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    return _heads(rng.choice(["bf16", "bf16", "f16"]), hkv * rng.choice([1, 2, 3, 4, 4, 7, 8]), hkv,
                  rng.choice([64, 128, 128]))


def _draw_group(rng, d):
    return rng.choice([0, 0, 32, 64, d])


def _draw_any(rng):
    kind, h, mix = rng.choice(["packed", "packed", "append", "read", "paged", "paged"]), _draw_heads(rng), rng.randrange(1 << 30)
    seqs, longest, page = _log(rng, 1, 64), _log(rng, 1, 8192), rng.choice([16, 16, 32, 64, 128])
    if kind == "packed":
        return _packed(h, seqs, longest, mix, rng.random() < 0.8, rng.random() < 0.5)
    if kind == "append":
        rotary = rng.choice([h["d"], h["d"], h["d"] // 2, 48])
        return _append(h, seqs, rng.choice([1, _log(rng, 1, 2048)]), mix, rng.choice([0, _log(rng, 1, 4096)]), page,
                       _draw_group(rng, h["d"]), rotary, rng.random() < 0.3)
    if kind == "read":
        return _read(h, seqs, longest, mix, page, _draw_group(rng, h["d"]))
    return _paged(h, seqs, _log(rng, 1, 16384), mix, rng.choice([1, 1, 1, 2, 4, rng.randint(1, 8)]), page,
                  _draw_group(rng, h["d"]))


def draw(rng):
    """One of the four kinds; sequences and lengths over their whole range, cut to what the listed ones cost (and
    scores of equally long prompts to what a plain form of them holds)."""
    c = _draw_any(rng)
    room = {"packed": 3.5e9, "append": 1.5e6 * 32, "read": 64e3 * 8, "paged": 1e6 * 8}[c["kind"]]
    while True:
        w, many = work(c), c["seqs"] * c["longest"]
        size = {"packed": many * c["longest"] * c["hq"], "append": many * c["hq"], "read": many * c["hkv"],
                "paged": many * c["hkv"]}[c["kind"]]
        if w["flops"] <= 5.5e11 and w["bytes"] <= 5e8 and size <= room:
            return c
        c["seqs"], c["longest"] = ((c["seqs"] + 1) // 2, c["longest"]) if c["seqs"] > 1 else (1, c["longest"] * 3 // 4)


def _lens(c):
    """Rows of each sequence: the longest, and others spread over their logarithm down to a sixteenth of it."""
    rng, top = random.Random(c["mix"]), c["longest"]
    lens = [top] + [_log(rng, max(1, top / 16), top) for _ in range(c["seqs"] - 1)]
    rng.shuffle(lens)
    return lens


def _rows_and_keys(c):
    """Per sequence: rows of this call, and keys that it has with them."""
    lens = _lens(c)
    if c["kind"] == "paged":
        return [min(c["new"], n) for n in lens], lens
    if c["kind"] == "append" and c["past"]:
        rng = random.Random(c["mix"] + 1)
        return lens, [n + _log(rng, max(1, c["past"] / 16), c["past"]) for n in lens]
    return lens, lens


# ---- inputs ------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(_DT[dtype])


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lens):
    return list(itertools.accumulate(lens, initial=0))


def _rotation(places, rotary):
    """Row p: the cosines of p's angles, then their sines."""
    step = 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = torch.arange(places, device="cuda", dtype=torch.float64)[:, None] * step
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    hq, hkv, d, dt = c["hq"], c["hkv"], c["d"], c["dtype"]
    rows, keys = _rows_and_keys(c)
    t = sum(rows)
    s = {"case": c, "offsets": _int32(_starts(rows)), "most": max(rows)}
    if c["kind"] == "packed" and c["fused"]:  # what one product of all three gives
        whole = _normal(gen, [t, (hq + 2 * hkv) * d], dt)
        cut = (0, hq * d, (hq + hkv) * d, (hq + 2 * hkv) * d)
        s["q"], s["k"], s["v"] = (whole[:, a:b].unflatten(1, (-1, d)) for a, b in zip(cut, cut[1:]))
    elif c["kind"] in ("packed", "append"):
        s["q"] = _normal(gen, [t, hq, d], dt)
        s["k"], s["v"] = (_normal(gen, [t, hkv, d], dt) for _ in range(2))
    elif c["kind"] == "paged":
        s["q"] = _normal(gen, [t, hq, d], dt)
    if c["kind"] in ("packed", "paged"):
        s["o"] = torch.empty([t, hq, d], device="cuda", dtype=_DT[dt])
    else:
        s["k_out"] = torch.empty([t, hkv, d], device="cuda", dtype=_DT[dt])
    if c["kind"] == "append":
        s["q_out"] = torch.empty([t, hq, d], device="cuda", dtype=_DT[dt])
        s["rotation"] = _rotation(max(keys), c["rotary"])
    if c["kind"] == "read" or (c["kind"] == "append" and c["group"]):
        s["k_read"], s["v_read"] = (torch.empty([t, hkv, d], device="cuda", dtype=_DT[dt]) for _ in range(2))
    if c["kind"] != "packed":
        # every sequence's pages lie anywhere in a pool with room for some more
        page = c["page"]
        need = [-(-n // page) for n in keys]
        pool = sum(need) + 8
        order = torch.randperm(pool, generator=gen, device="cuda").tolist()
        most = max(need)
        at = _starts(need)
        s["pages"] = _int32([order[a:a + n] + [0] * (most - n) for a, n in zip(at, need)])
        s["lengths"] = _int32(keys)
        for x in "kv":
            if not c["group"]:
                s[x + "_cache"] = _normal(gen, [pool, hkv, page, d], dt)
                continue
            n = d // c["group"]
            s[x + "_cache"] = torch.randint(0, 256, [pool, hkv, page, d // 2], generator=gen, device="cuda", dtype=torch.uint8)
            # what groups of normal values have: about four deviations, from two below the mean
            scale = torch.rand([pool, hkv, page, n], generator=gen, device="cuda").mul_(0.1).add_(0.25)
            low = torch.rand([pool, hkv, page, n], generator=gen, device="cuda").mul_(-0.8).sub_(1.8)
            s[x + "_params"] = torch.stack([scale, low], -1).flatten(3).half()
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
    types = {torch.bfloat16: capi.BFLOAT16, torch.float16: capi.HALF, torch.float32: capi.FLOAT, torch.uint8: capi.UINT8}
    desc = {n: capi.TensorDesc.make(t.shape, t.stride(), types[t.dtype]) for n, t in s.items()
            if isinstance(t, torch.Tensor) and t.dtype in types}
    p = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    ctx = _held["ctx"]
    if c["kind"] != "packed":
        cache, at = capi.CacheDesc(), capi.CachePointers()
        for x in ("k", "v"):
            setattr(cache, x, desc[x + "_cache"])
            setattr(at, x, p[x + "_cache"])
            if c["group"]:
                setattr(cache, x + "_params", desc[x + "_params"])
                setattr(at, x + "_params", p[x + "_params"])
        cache.batch, cache.pages_per_sequence = s["pages"].shape
        cache.page_stride = s["pages"].stride(0)
        at.pages, at.lengths = p["pages"], p["lengths"]
    if c["kind"] == "packed":
        d = capi.SdpaPackedDesc()
        d.q, d.k, d.v, d.o = (desc[n] for n in "qkvo")
        d.batch, d.is_causal = c["seqs"], int(c["causal"])
        s["room"] = room = torch.empty(max(ctx.sdpa_packed_workspace(d), 1), device="cuda", dtype=torch.uint8)
        ws = room.data_ptr()

        def call():
            ctx.sdpa_packed_fwd(d, p["q"], p["k"], p["v"], p["offsets"], p["o"], workspace=ws)
    elif c["kind"] == "paged":
        d = capi.SdpaPagedDesc()
        d.q, d.o, d.cache, d.is_causal = desc["q"], desc["o"], cache, 1
        s["room"] = room = torch.empty(max(ctx.sdpa_paged_workspace(d), 1), device="cuda", dtype=torch.uint8)
        ws = room.data_ptr()

        def call():
            ctx.sdpa_paged_fwd(d, at, p["q"], p["offsets"], p["o"], workspace=ws)
    elif c["kind"] == "read":
        d = capi.CacheReadDesc()
        d.cache, d.k, d.v = cache, desc["k_read"], desc["v_read"]

        def call():
            ctx.cache_read(d, at, p["offsets"], p["k_read"], p["v_read"])
    else:
        d = capi.CacheAppendDesc()
        d.cache, d.interleaved = cache, int(c["interleaved"])
        d.q, d.k, d.v, d.rotation, d.q_out, d.k_out = (desc[n] for n in ("q", "k", "v", "rotation", "q_out", "k_out"))
        back = capi.CacheReadDesc()
        if c["group"]:
            back.cache, back.k, back.v = cache, desc["k_read"], desc["v_read"]

        def call():
            ctx.cache_append(d, at, p["k"], p["v"], p["offsets"], q=p["q"], rotation=p["rotation"],
                             q_out=p["q_out"], k_out=p["k_out"])
            if c["group"]:
                ctx.cache_read(back, at, p["offsets"], p["k_read"], p["v_read"])
    s["plan"] = call
    return call


# ---- the plain forms ---------------------------------------------------------
def _places(s):
    """Per packed row: its sequence and its place among that sequence's keys."""
    t = (s.get("q") if "q" in s else s["k_out"]).shape[0]
    row = torch.arange(t, device="cuda")
    at = s["offsets"].long()
    seq = torch.bucketize(row, at[1:], right=True)
    n = at[1:] - at[:-1]
    keys = s["lengths"].long() if "lengths" in s else n
    return seq, row - at[seq], keys[seq] - n[seq] + row - at[seq]


def _padded(x, seq, i, seqs, most):
    """Packed rows [T, H, D] as [seqs, H, most, D] in f32, zeros behind each sequence."""
    out = torch.zeros([seqs, most, *x.shape[1:]], device="cuda", dtype=torch.float32)
    out[seq, i] = x.float()
    return out.transpose(1, 2)


def _values(codes, params):
    """What 4-bit codes and their groups' (scale, low) pairs stand for, in f32."""
    pair = params.float().unflatten(-1, (-1, 2))
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (pair.shape[-2], -1))
    return (code * pair[..., :1] + pair[..., 1:]).flatten(-2)


def _attend(s, q, k, v, seq, i, place, keys, causal):
    """softmax(q k^T / sqrt(d)) v of padded [seqs, hq, rows, d] against [seqs, hkv, most keys, d]."""
    c = s["case"]
    b, h, r, d = q.shape
    q = q.reshape(b, c["hkv"], -1, d)  # heads that share keys side by side
    x = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(b, h, r, -1)
    key = torch.arange(x.shape[-1], device="cuda")
    top = torch.zeros([b, r], device="cuda", dtype=torch.long)
    top[seq, i] = place if causal else keys[seq] - 1
    x.masked_fill_((key > top[:, :, None])[:, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    y = torch.matmul(x.view(b, c["hkv"], -1, x.shape[-1]), v).view(b, h, r, d).div_(x.sum(-1, keepdim=True))
    return s["o"].copy_(y.transpose(1, 2)[seq, i])


def _plain_packed(s):
    c = s["case"]
    seq, i, place = _places(s)
    q, k, v = (_padded(s[x], seq, i, c["seqs"], s["most"]) for x in "qkv")
    return _attend(s, q, k, v, seq, i, place, (s["offsets"][1:] - s["offsets"][:-1]).long(), c["causal"])


def _plain_paged(s):
    c = s["case"]
    seq, i, place = _places(s)
    pages = s["pages"].long()
    k, v = ((_values(s[x + "_cache"][pages], s[x + "_params"][pages]) if c["group"] else s[x + "_cache"][pages].float())
            .transpose(1, 2).flatten(2, 3) for x in "kv")
    return _attend(s, _padded(s["q"], seq, i, c["seqs"], s["most"]), k, v, seq, i, place, s["lengths"].long(), True)


def _rotated(x, table, place, interleaved):
    """The first dims of x [T, H, D] turned by their place's angles, in f32, rounded once."""
    half = table.shape[1] // 2
    cos, sin = table[place][:, None].split(half, -1)
    y = x.float()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    return y.to(x.dtype)


def _codes(x, group):
    """4-bit codes of 16-bit x [T, H, D] and the (scale, low) pairs of its groups."""
    y = x.float().unflatten(-1, (-1, group))
    low = y.amin(-1, keepdim=True).half()
    wide = (y.amax(-1, keepdim=True) - low.float()).clamp_(min=0)
    scale = (wide / torch.full_like(wide, 15.0)).half()
    by = torch.where(scale > 0, torch.ones_like(wide) / scale.float(), torch.zeros_like(wide))
    code = ((y - low.float()) * by).round_().clamp_(0, 15).to(torch.uint8).flatten(-2)
    return code[..., ::2] | code[..., 1::2] << 4, torch.stack([scale, low], -1).flatten(2)


def _plain_append(s):
    c = s["case"]
    seq, _, place = _places(s)
    s["q_out"].copy_(_rotated(s["q"], s["rotation"], place, c["interleaved"]))
    s["k_out"].copy_(_rotated(s["k"], s["rotation"], place, c["interleaved"]))
    page, at = s["pages"][seq, place // c["page"]].long(), place % c["page"]
    if not c["group"]:
        s["k_cache"][page, :, at] = s["k_out"]
        s["v_cache"][page, :, at] = s["v"]
        return
    s["k_cache"][page, :, at], s["k_params"][page, :, at] = _codes(s["k_out"], c["group"])
    s["v_cache"][page, :, at], s["v_params"][page, :, at] = _codes(s["v"], c["group"])


def _plain_read(s):
    c = s["case"]
    seq, _, place = _places(s)
    page, at = s["pages"][seq, place // c["page"]].long(), place % c["page"]
    k, v = ((_values(s[x + "_cache"][page, :, at], s[x + "_params"][page, :, at]) if c["group"] else s[x + "_cache"][page, :, at])
            for x in "kv")
    s["k_read"].copy_(k)
    s["v_read"].copy_(v)


def _outputs(s):
    if "o" in s:
        return s["o"]
    names = ("q_out", "k_out", "k_read", "v_read") if "k_read" in s else ("q_out", "k_out", "k_cache", "v_cache")
    if s["case"]["kind"] == "read":
        names = ("k_read", "v_read")
    return {n: s[n] for n in names}


def run(state):
    s = state
    if own:
        (s.get("plan") or _plan(s))()
        return _outputs(s)
    kind = s["case"]["kind"]
    if kind == "packed":
        _plain_packed(s)
    elif kind == "paged":
        _plain_paged(s)
    else:
        if kind == "append":
            _plain_append(s)
        if "k_read" in s:
            _plain_read(s)
    return _outputs(s)


# ---- what a pass cannot do without -------------------------------------------
def work(case):
    c = case
    rows, keys = _rows_and_keys(c)
    t, hq, hkv, d = sum(rows), c["hq"], c["hkv"], c["d"]
    small = 4 * (2 * c["seqs"] + 1)
    if c["kind"] == "packed":
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in rows)
        return {"bytes": 2 * t * d * 2 * (hq + hkv) + small, "flops": 4 * pairs * hq * d}
    row = hkv * (d // 2 + 4 * d // c["group"] if c["group"] else 2 * d)  # of K or V in the cache
    table = small + sum(4 * -(-n // c["page"]) for n in keys)
    if c["kind"] == "paged":
        pairs = sum(r * n - r * (r - 1) // 2 for r, n in zip(rows, keys))
        return {"bytes": 2 * row * sum(keys) + 4 * t * hq * d + table, "flops": 4 * pairs * hq * d}
    if c["kind"] == "read":
        return {"bytes": 2 * t * (row + 2 * hkv * d) + table, "flops": 0}
    # q, k, v and the angles in; q, k and the cache's rows out, with 4 bits what they stand for too
    more = 4 * hkv * d if c["group"] else 0
    return {"bytes": t * (4 * hq * d + 6 * hkv * d + 4 * c["rotary"] + 2 * row + more) + table,
            "flops": 3 * t * (hq + hkv) * c["rotary"]}


# ---- the definition in 64 bits -----------------------------------------------
def _exact_rows(x, group, params, page, at):
    """Cache rows at (page, at) as [rows, heads, d] in f64."""
    x = x[page, :, at]
    if not group:
        return x.double()
    pair = params[page, :, at].double()
    full = torch.empty([*x.shape[:2], 2 * x.shape[2]], device="cuda", dtype=torch.float64)
    full[:, :, 0::2], full[:, :, 1::2] = x.remainder(16).double(), x.div(16, rounding_mode="floor").double()
    scale, low = (pair[:, :, j::2].repeat_interleave(group, 2) for j in (0, 1))
    return full * scale + low


def _exact_softmax(q, k, v, first, causal):
    """Rows q [n, hq, d], the first of them at place `first`, over k and v [m, hkv, d], all in f64."""
    n, hq, d = q.shape
    m, hkv, _ = k.shape
    out = torch.empty_like(q)
    for h in range(hq):
        kk, vv = k[:, h * hkv // hq], v[:, h * hkv // hq]
        for a in range(0, n, 4096):
            x = q[a:a + 4096, h] @ kk.T / math.sqrt(d)
            if causal:
                place = torch.arange(first + a, first + a + x.shape[0], device="cuda")
                x = x.masked_fill(torch.arange(m, device="cuda")[None] > place[:, None], -math.inf)
            w = torch.softmax(x, 1)
            out[a:a + 4096, h] = w @ vv
    return out


def _exact_turn(x, table, place, interleaved):
    z = x.double()
    r = table.shape[1]
    pair = z[..., :r].unflatten(-1, (-1, 2)) if interleaved else torch.stack(z[..., :r].chunk(2, -1), -1)
    turn = torch.complex(*table.double()[place].chunk(2, -1))[:, None]
    pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    z[..., :r] = pair.flatten(-2) if interleaved else torch.cat(pair.unbind(-1), -1)
    return z


def _exact_held(x, group):
    """What a group's 4-bit codes of x [T, H, D] stand for."""
    y = x.double().unflatten(-1, (-1, group))
    low = y.min(-1, keepdim=True).values.half().double()
    scale = ((y.max(-1, keepdim=True).values - low).clamp(min=0) / 15).half().double()
    code = torch.where(scale > 0, (y - low) / scale, 0).round().clamp(0, 15)
    return (low + scale * code).flatten(-2)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    rows, keys = _rows_and_keys(c)
    if c["kind"] in ("packed", "paged") and 8 * c["d"] * c["hq"] * sum(r * n for r, n in zip(rows, keys)) > 1e14:
        return None
    start, outs, k_at, v_at, q_at = _starts(rows), [], [], [], []
    k_cache, v_cache = ((s[x + "_cache"].double() if c["kind"] == "append" and not c["group"] else None) for x in "kv")
    for b, (n, m) in enumerate(zip(rows, keys)):
        here = slice(start[b], start[b] + n)
        if c["kind"] == "packed":
            outs.append(_exact_softmax(*(s[x][here].double() for x in "qkv"), 0, c["causal"]))
            continue
        place = torch.arange(0 if c["kind"] == "paged" else m - n, m, device="cuda")
        page, at = s["pages"][b].long()[place // c["page"]], place % c["page"]
        if c["kind"] != "append":
            k, v = (_exact_rows(s[x + "_cache"], c["group"], s.get(x + "_params"), page, at) for x in "kv")
            if c["kind"] == "paged":
                outs.append(_exact_softmax(s["q"][here].double(), k, v, m - n, True))
            k_at.append(k)
            v_at.append(v)
            continue
        q_at.append(_exact_turn(s["q"][here], s["rotation"], place, c["interleaved"]))
        k = _exact_turn(s["k"][here], s["rotation"], place, c["interleaved"])
        outs.append(k)
        if c["group"]:
            k_at.append(_exact_held(k.to(s["k"].dtype), c["group"]))
            v_at.append(_exact_held(s["v"][here], c["group"]))
        else:
            k_cache[page, :, at] = k
            v_cache[page, :, at] = s["v"][here].double()
    if c["kind"] in ("packed", "paged"):
        return torch.cat(outs)
    if c["kind"] == "read":
        return {"k_read": torch.cat(k_at), "v_read": torch.cat(v_at)}
    out = {"q_out": torch.cat(q_at), "k_out": torch.cat(outs)}
    if c["group"]:
        return {**out, "k_read": torch.cat(k_at), "v_read": torch.cat(v_at)}
    return {**out, "k_cache": k_cache, "v_cache": v_cache}
