"""
The operators of a decoding step on one MI355X, as cases with sizes: what `bergen_amd`'s entry points compute, in their plain form
(elementary torch operations) and through those entry points (`own`).

  rotary    RMS norm of query and key heads + rotary positions                      bergen_amd.qk_norm_rotary
  cache     a chunk written into a paged key-value cache, the context read back     bergen_amd.kv_cache_write, kv_cache_read
  paged     attention of one new token per sequence over that cache                 bergen_amd.paged_attention
  logprobs  log probabilities of given tokens, entropy, top alternatives            bergen_amd.token_logprobs
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "int8": 1, "e4m3": 1}


# ---- cases ------------------------------------------------------------------------------------------------------------------

def _rotary(name, tokens, hq, hk, dim, rotary, dtype, far=32768, norm=True, interleaved=False):
    return {"name": name, "op": "rotary", "tokens": tokens, "hq": hq, "hk": hk, "dim": dim, "rotary": rotary, "dtype": dtype, "far": far,
            "norm": norm, "interleaved": interleaved}


def _cache(name, write, read, heads, dim, page, dtype, cache):
    return {"name": name, "op": "cache", "write": write, "read": read, "heads": heads, "dim": dim, "page": page, "dtype": dtype, "cache": cache}


def _paged(name, batch, short, long, hq, hk, dim, page, dtype, cache, softcap=0.0, window=0, alibi=False):
    return {"name": name, "op": "paged", "batch": batch, "short": short, "long": long, "hq": hq, "hk": hk, "dim": dim, "page": page,
            "dtype": dtype, "cache": cache, "softcap": softcap, "window": window, "alibi": alibi}


def _logprobs(name, rows, vocab, given, top, dtype, banned=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "given": given, "top": top, "dtype": dtype, "banned": banned}


def listed():
    return [
        # one layer of one decoding step of 16 sequences: latency
        _rotary("rotary step", 16, 32, 8, 128, 128, "bf16"),
        # the prompts of a batch of questions with their passages, one layer
        _rotary("rotary prompt", 16384, 32, 8, 128, 128, "bf16"),
        # heads of 64 as this repository's encoders have them, half of each rotated in neighbouring pairs, no norm, an odd count of rows
        _rotary("rotary halves fp32", 4111, 12, 12, 64, 32, "fp32", far=1000000, norm=False, interleaved=True),
        # 8 new tokens of one sequence into an 8-bit cache, and its short context back: latency
        _cache("cache step", 8, 300, 8, 128, 16, "bf16", "int8"),
        # a chunk of a long prompt into an e4m3 cache, and the whole context back for the chunk's attention
        _cache("cache chunk", 8192, 65536, 8, 128, 64, "bf16", "e4m3"),
        # one question, a short context: latency
        _paged("paged one", 1, 700, 700, 32, 8, 128, 16, "bf16", "bf16"),
        # questions with the passages that retrieval found for them, lengths as ragged as those
        _paged("paged batch", 64, 90, 8191, 32, 8, 128, 16, "bf16", "bf16"),
        # few sequences with very long contexts, an e4m3 cache
        _paged("paged long", 3, 100001, 131072, 32, 8, 128, 64, "bf16", "e4m3"),
        # every head its own keys (12 x 64 as BERT-base), an int8 cache, capped scores, a distance bias, a window
        _paged("paged capped", 37, 1, 6000, 12, 12, 64, 32, "fp16", "int8", softcap=30.0, window=4096, alibi=True),
        # yes / no of one prompt over BERT's vocabulary, in fp32: latency
        _logprobs("logprobs yes no", 1, 30522, 2, 5, "fp32"),
        # the next tokens of a batch over a large vocabulary with its padding banned
        _logprobs("logprobs step", 61, 120064, 1, 20, "bf16", banned=256),
        # every token of a batch of answers: their likelihood under the model
        _logprobs("logprobs answers", 4096, 128000, 1, 8, "bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm, odd ones among them."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "cache", "paged", "paged", "logprobs"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        group = rng.choice([1, 2, 4, 8])
        hk = rng.choice([1, 2, 4, 8, 12])
        hq = min(64, hk * group) // hk * hk
        tokens = max(1, min(_spread(rng, 1, 16384), 16384 * 40 * 128 // ((hq + hk) * dim * 2)))
        c = _rotary("", tokens, hq, hk, dim, rng.choice([dim, dim // 2]), rng.choice(["bf16", "fp16", "fp32"]), _spread(rng, 512, 1000000),
                    rng.random() < 0.7, rng.random() < 0.3)
    elif op == "cache":
        heads, dim = rng.choice([1, 2, 4, 8, 12]), rng.choice([64, 96, 128, 256])
        read = max(2, min(_spread(rng, 16, 65536), 60000 * 8 * 128 // (heads * dim * 2)))
        c = _cache("", min(read, _spread(rng, 1, 8192)), read, heads, dim, rng.choice([8, 16, 32, 64, 128]), rng.choice(["bf16", "fp16", "fp32"]),
                   rng.choice(["int8", "e4m3", "e4m3", "int8", "bf16", "fp16"]))
    elif op == "paged":
        dtype = rng.choice(["bf16", "fp16"])
        dim, hk = rng.choice([64, 96, 128, 256]), rng.choice([1, 2, 4, 8, 12])
        hq = hk * rng.choice([1, 2, 4, 5, 8, 16])
        long = _spread(rng, 1, 131072)
        batch = max(1, min(_spread(rng, 1, 256), 260000 * 8 * 128 // (long * hk * dim)))
        if batch * long * max(hk * dim, hq * 32) > 260000 * 8 * 128:
            long = max(1, 260000 * 8 * 128 // (batch * max(hk * dim, hq * 32)))
        c = _paged("", batch, _spread(rng, 1, long), long, hq, hk, dim, rng.choice([8, 16, 32, 64, 128]), dtype,
                   rng.choice([dtype, dtype, "int8", "e4m3"]), rng.choice([0.0, 0.0, 30.0, 50.0]), rng.choice([0, 0, _spread(rng, 64, 4096)]),
                   rng.random() < 0.25)
    else:
        vocab = _spread(rng, 1000, 262144)
        rows = max(1, min(_spread(rng, 1, 4096), 4096 * 64000 // vocab))
        c = _logprobs("", rows, vocab, rng.choice([1, 1, 2, 5]), rng.choice([0, 1, 5, 8, 20, 50]), rng.choice(["bf16", "fp16", "fp32"]),
                      rng.choice([0, 0, vocab // 100]))
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _heads(g, tokens, heads, dim, dtype):
    """Vectors of heads as projections give them: some channels an order larger than the others, each token with its own size."""
    x = _normal(g, tokens, heads, dim)
    x *= torch.exp(0.7 * _normal(g, 1, heads, dim)) * torch.exp(0.3 * _normal(g, tokens, 1, 1))
    return x.to(dtype)


def _lengths(case):
    """The sequences' lengths: the case's own, evenly from its shortest to its longest."""
    b, lo, hi = case["batch"], case["short"], case["long"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _stored(g, shape, cache):
    """A cache's content, and the scale of each vector where it holds 8 bits."""
    if cache in ("fp16", "bf16"):
        return _normal(g, *shape, dtype=DTYPES[cache]), None
    x = _normal(g, *shape, dtype=torch.float16)
    if cache == "int8":
        codes = x.mul_(40).clamp_(-127, 127).round_().to(torch.int8)
        return codes, torch.rand(shape[:-1], generator=g, device="cuda") * 0.02 + 0.015
    codes = x.mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return codes, torch.exp2(torch.randint(-8, -5, shape[:-1], generator=g, device="cuda").float())


def prepare(case, seed):
    g = _gen(seed)
    c, op = dict(case), case["op"]
    if op == "rotary":
        dtype = DTYPES[c["dtype"]]
        qkv = _heads(g, c["tokens"], c["hq"] + 2 * c["hk"], c["dim"], dtype)  # as one projection writes them, side by side
        s = {"q": qkv[:, : c["hq"]], "k": qkv[:, c["hq"]: c["hq"] + c["hk"]],
             "positions": torch.randint(0, c["far"], (c["tokens"],), generator=g, device="cuda"),
             "inv_freq": 10000.0 ** (-torch.arange(0, c["rotary"], 2, device="cuda", dtype=torch.float64) / c["rotary"])}
        s["qw"] = (1 + 0.2 * _normal(g, c["dim"])).to(dtype) if c["norm"] else None
        s["kw"] = (1 + 0.2 * _normal(g, c["dim"])).to(dtype) if c["norm"] else None
    elif op == "cache":
        page = c["page"]
        pages = -(-c["read"] // page) + 3
        shape = (pages, c["heads"], page, c["dim"])
        s = {}
        s["kc"], s["ks"] = _stored(g, shape, c["cache"])
        s["vc"], s["vs"] = _stored(g, shape, c["cache"])
        s["k"] = _heads(g, c["write"], c["heads"], c["dim"], DTYPES[c["dtype"]])
        s["v"] = _normal(g, c["write"], c["heads"], c["dim"]).to(DTYPES[c["dtype"]])
        order = torch.randperm(pages, generator=g, device="cuda")[: -(-c["read"] // page)]  # the sequence's pages
        slots = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[: c["read"]].contiguous()
        s["read"] = slots
        s["slots"] = slots[c["read"] - c["write"]:].contiguous()
    elif op == "paged":
        page, b = c["page"], c["batch"]
        lengths = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")[torch.randperm(b, generator=g, device="cuda")].contiguous()
        wide = -(-c["long"] // page)
        need = sum(-(-n // page) for n in _lengths(c))
        shape = (need + 1, c["hk"], page, c["dim"])
        s = {"lengths": lengths}
        s["kc"], s["ks"] = _stored(g, shape, c["cache"])
        s["vc"], s["vs"] = _stored(g, shape, c["cache"])
        own_pages = (lengths.long() + page - 1) // page
        at = torch.arange(wide, device="cuda")
        first = own_pages.cumsum(0) - own_pages
        used = at < own_pages[:, None]
        s["table"] = torch.where(used, torch.randperm(need + 1, generator=g, device="cuda")[(first[:, None] + at).clamp_(max=need)], 0).int()
        s["q"] = 2 * _normal(g, b, c["hq"], c["dim"]).to(DTYPES[c["dtype"]])
        s["slopes"] = torch.exp2(-8.0 * (torch.arange(c["hq"], device="cuda") + 1) / c["hq"]).float() if c["alibi"] else None
    else:
        x = _normal(g, c["rows"], c["vocab"], dtype=DTYPES[c["dtype"]]).mul_(2.5)
        at = torch.randint(0, c["vocab"] - c["banned"], (c["rows"], 3), generator=g, device="cuda")
        x.scatter_add_(1, at, (9 + 4 * _normal(g, c["rows"], 3)).to(x.dtype))  # the few tokens that carry most of the mass
        if c["banned"]:
            x[:, c["vocab"] - c["banned"]:] = -math.inf
        some = torch.randint(0, c["vocab"] - c["banned"], (c["rows"], c["given"]), generator=g, device="cuda")
        s = {"logits": x, "targets": torch.cat([at[:, :1], some[:, 1:]], 1).contiguous()}
    s["case"] = c
    return s


# ---- the operators' plain forms ---------------------------------------------------------------------------------------------

def _turned(y, cos, sin, rotary, interleaved):
    r, rest = y[..., :rotary], y[..., rotary:]
    if interleaved:
        u, v = r[..., 0::2], r[..., 1::2]
        return torch.cat([torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2), rest], -1)
    u, v = r[..., : rotary // 2], r[..., rotary // 2:]
    return torch.cat([u * cos - v * sin, v * cos + u * sin, rest], -1)


def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def one(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        return _turned(y, cos, sin, c["rotary"], c["interleaved"]).to(x.dtype)

    return {"q": one(s["q"], s["qw"]), "k": one(s["k"], s["kw"])}


def _plain_codes(x, cache):
    """x as the cache holds it: codes and the scale of each vector."""
    if cache in ("fp16", "bf16"):
        return x.to(DTYPES[cache]), None
    most = x.float().abs().amax(-1)
    if cache == "int8":
        scale = (most.double() / 127).float().clamp(min=2.0 ** -126)
        return (x.double() / scale.double()[..., None]).round().to(torch.int8), scale
    part, power = torch.frexp(most)
    scale = torch.exp2((power - 9 + (part > 0.875).int()).clamp(min=-126).float())
    return (x.float() / scale[..., None]).to(torch.float8_e4m3fn), scale


def _plain_cache(s):
    c = s["case"]
    page, offset = s["slots"] // c["page"], s["slots"] % c["page"]
    rpage, roffset = s["read"] // c["page"], s["read"] % c["page"]

    def one(x, codes, scales):
        new, scale = _plain_codes(x, c["cache"])
        bits = codes.view(torch.int8) if scale is not None else codes
        bits[page, :, offset] = new.view(bits.dtype)
        back = codes.view(bits.dtype)[rpage, :, roffset].view(codes.dtype).float()
        if scale is not None:
            scales[page, :, offset] = scale
            back = back * scales[rpage, :, roffset][..., None]
        return back.to(x.dtype)

    return {"k": one(s["k"], s["kc"], s["ks"]), "v": one(s["v"], s["vc"], s["vs"])}


def _gathered(codes, scales, table):
    """The sequences' vectors, [batch, heads, width, dim] in 32 bits."""
    b, w = table.shape
    _, h, page, d = codes.shape
    x = codes.view(torch.int8)[table.long()].view(codes.dtype) if scales is not None else codes[table.long()]
    x = x.transpose(1, 2).reshape(b, h, w * page, d).float()
    if scales is not None:
        x *= scales[table.long()].transpose(1, 2).reshape(b, h, w * page, 1)
    return x


def _plain_paged(s):
    c, n = s["case"], s["lengths"].long()[:, None, None, None]
    q = s["q"].float().reshape(c["batch"], c["hk"], c["hq"] // c["hk"], c["dim"])
    k = _gathered(s["kc"], s["ks"], s["table"])
    x = torch.matmul(q, k.transpose(2, 3)) * c["dim"] ** -0.5
    del k
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    t = torch.arange(x.shape[-1], device="cuda")
    if c["alibi"]:
        x = x - s["slopes"].reshape(c["hk"], -1, 1) * (n - 1 - t)
    gone = (t >= n) | (t < n - c["window"]) if c["window"] else t >= n
    x = x.masked_fill(gone, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.masked_fill(m == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    v = _gathered(s["vc"], s["vs"], s["table"])
    out = torch.matmul(p, v) / total.masked_fill(total == 0, 1)
    lse = (m + torch.log(total))[..., 0]
    return {"out": out.reshape(s["q"].shape).to(s["q"].dtype), "lse": lse.reshape(c["batch"], c["hq"])}


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    weighted = ((x - m).masked_fill(e == 0, 0) * e).sum(-1, keepdim=True)
    r = {"logprobs": x.gather(1, s["targets"]) - lse, "entropy": (torch.log(total) - weighted / total)[:, 0]}
    del e
    if c["top"]:
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + (c["vocab"] - 1 - torch.arange(c["vocab"], device="cuda"))
        r["top_ids"] = order.topk(c["top"], -1).indices
        r["top_logprobs"] = x.gather(1, r["top_ids"]) - lse
    return r


def _own(s):
    import bergen_amd
    c = s["case"]
    if c["op"] == "rotary":
        q, k = bergen_amd.qk_norm_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6,
                                         interleaved=c["interleaved"])
        return {"q": q, "k": k}
    if c["op"] == "cache":
        bergen_amd.kv_cache_write(s["k"], s["v"], s["slots"], s["kc"], s["vc"], k_scale=s["ks"], v_scale=s["vs"])
        k, v = bergen_amd.kv_cache_read(s["read"], s["kc"], s["vc"], k_scale=s["ks"], v_scale=s["vs"], dtype=s["k"].dtype)
        return {"k": k, "v": v}
    if c["op"] == "paged":
        out, lse = bergen_amd.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lengths"], k_scale=s["ks"], v_scale=s["vs"],
                                              softcap=c["softcap"], window=c["window"], alibi_slopes=s["slopes"], return_lse=True)
        return {"out": out, "lse": lse}
    r = bergen_amd.token_logprobs(s["logits"], s["targets"], top=c["top"])
    d = {"logprobs": r.logprobs, "entropy": r.entropy}
    if c["top"]:
        d["top_ids"], d["top_logprobs"] = r.top_ids, r.top_logprobs
    return d


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "cache": _plain_cache, "paged": _plain_paged, "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "rotary":
        heads = c["tokens"] * (c["hq"] + c["hk"])
        return {"bytes": 2 * heads * c["dim"] * BYTES[c["dtype"]] + 8 * c["tokens"], "flops": heads * (3 * c["rotary"] + (4 * c["dim"] if c["norm"] else 0))}
    if c["op"] == "cache":
        outside, inside = c["dim"] * BYTES[c["dtype"]], c["dim"] * BYTES[c["cache"]] + (4 if BYTES[c["cache"]] == 1 else 0)
        rows = c["write"] + c["read"]
        return {"bytes": 2 * rows * c["heads"] * (outside + inside) + 8 * rows, "flops": 4 * rows * c["heads"] * c["dim"]}
    if c["op"] == "paged":
        seen = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
        vector = c["dim"] * BYTES[c["cache"]] + (4 if BYTES[c["cache"]] == 1 else 0)
        rows = c["batch"] * c["hq"]
        return {"bytes": 2 * seen * c["hk"] * vector + 2 * rows * c["dim"] * BYTES[c["dtype"]] + 4 * rows + 4 * seen // c["page"],
                "flops": 4 * seen * c["hq"] * c["dim"]}
    cells = c["rows"] * c["vocab"]
    return {"bytes": cells * BYTES[c["dtype"]] + c["rows"] * (12 * c["given"] + 4 + 12 * c["top"]), "flops": 5 * cells}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------------

def _exact_rotary(s):
    c = s["case"]
    half = c["rotary"] // 2
    first = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else half)
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double().outer(s["inv_freq"]))
    r = {}
    for name, w in (("q", s["qw"]), ("k", s["kw"])):
        y = s[name].double().clone()
        if w is not None:
            y /= torch.sqrt((y * y).sum(-1, keepdim=True) / c["dim"] + 1e-6)
            y *= w.double()
        pairs = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z[:, None]
        y[..., first], y[..., second] = pairs.real, pairs.imag
        r[name] = y
    return r


def _exact_codes(x, cache):
    """What a cache of 8 bits gives back for vectors x, in 64 bits."""
    x = x.double()
    most = x.abs().max(-1, keepdim=True).values
    if cache == "int8":
        scale = torch.clamp((most / 127).float(), min=2.0 ** -126).double()
        return torch.round(x / scale) * scale
    scale = torch.ones_like(most)
    for power in range(-126, 121):  # the least power of two that lets the largest value be held
        scale = torch.where(most > 448 * 2.0 ** (power - 1), torch.full_like(most, 2.0 ** power), scale) if power > -126 else torch.full_like(most, 2.0 ** power)
    y = x / scale
    grid = torch.exp2(torch.clamp(torch.frexp(y).exponent.double() - 1, min=-6) - 3)  # the spacing of 4-bit significands there
    return torch.round(y / grid) * grid * scale


def _exact_cache(s):
    c = s["case"]
    r = {}
    for name in ("k", "v"):
        codes, scales = s[name + "c"], s[name + "s"]
        flat = codes.float().double().transpose(1, 2).reshape(-1, c["heads"], c["dim"])
        if scales is not None:
            flat = flat * scales.double().transpose(1, 2).reshape(-1, c["heads"], 1)
            flat[s["slots"]] = _exact_codes(s[name], c["cache"])
        else:
            flat[s["slots"]] = s[name].to(DTYPES[c["cache"]]).double()
        r[name] = flat[s["read"]]
    return r


def _exact_paged(s):
    c = s["case"]
    group = c["hq"] // c["hk"]
    outs, sums = [], []
    for b, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - c["window"]) if c["window"] else 0
        pages = s["table"][b, : -(-n // c["page"])].long()
        kv = []
        for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
            x = codes.view(torch.int8)[pages].view(codes.dtype) if scales is not None else codes[pages]
            x = x.float().double()
            if scales is not None:
                x = x * scales[pages].double()[..., None]
            kv.append(x.permute(1, 0, 2, 3).reshape(c["hk"], -1, c["dim"])[:, lo:n])
        q = s["q"][b].double().reshape(c["hk"], group, c["dim"])
        x = torch.stack([q[h] @ kv[0][h].t().contiguous() for h in range(c["hk"])]).reshape(c["hq"], -1) / math.sqrt(c["dim"])
        if c["softcap"]:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        if c["alibi"]:
            x = x - s["slopes"].double()[:, None] * torch.arange(n - 1 - lo, -1, -1, device="cuda")
        if n == 0:
            outs.append(torch.zeros(c["hq"], c["dim"], dtype=torch.float64, device="cuda"))
            sums.append(torch.full((c["hq"],), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        lse = torch.logsumexp(x, -1)
        p = torch.exp(x - lse[:, None]).reshape(c["hk"], group, -1)
        outs.append(torch.cat([p[h] @ kv[1][h] for h in range(c["hk"])]))
        sums.append(lse)
    return {"out": torch.stack(outs), "lse": torch.stack(sums)}


def _exact_logprobs(s):
    c = s["case"]
    parts = {"logprobs": [], "entropy": [], "top_ids": [], "top_logprobs": []}
    step = max(1, 50_000_000 // c["vocab"])
    for at in range(0, c["rows"], step):
        lp = torch.log_softmax(s["logits"][at: at + step].double(), -1)
        parts["logprobs"].append(torch.gather(lp, 1, s["targets"][at: at + step]))
        parts["entropy"].append(torch.special.entr(torch.exp(lp)).sum(-1))
        if c["top"]:
            ids = torch.sort(s["logits"][at: at + step], dim=-1, descending=True, stable=True).indices[:, : c["top"]]
            parts["top_ids"].append(ids)
            parts["top_logprobs"].append(torch.gather(lp, 1, ids))
    return {name: torch.cat(v) for name, v in parts.items() if v}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "cache": _exact_cache, "paged": _exact_paged, "logprobs": _exact_logprobs}[case["op"]](s)
