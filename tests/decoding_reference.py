"""Plain implementations, in 64 bits, of the decoding operators (bergen_amd/decoding.py), with bounds on how far a kernel that
computes in 32 bits and rounds once may be from them.  Used by the tests only."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative to the value
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}               # half a step among fp16's subnormals


def assert_within(got, want, bound, what):
    """|got - want| <= bound elementwise (want in 64 bits); infinities and NaN in the same places."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities differ"
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, (f"{what}: {int((over > 0).sum())} of {over.numel()} values are off, by up to {float(over.max()):.3g} "
                                                        f"over a bound of {float(bound[fine][over.argmax()]):.3g}")


def rotary(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False):
    """-> (value, bound).  In 32 bits: the sum of D squares is off by at most (D / lanes + 6 + 1) roundings, half of that reaches the
    reciprocal root; the root, the quotient, two products and the pair's two products and sum add 8 more; the fraction of a turn (at most
    1/2) is rounded to 2^-24 of itself, which is at most pi 2^-24 of an angle; cos and sin are good to 4 x 2^-24.  32 x 2^-24 of |u| + |v| covers them
    for D <= 256 (16 elements a lane).  The angle itself, a, is a product in 64 bits here (off by 2^-53 a) and, in the kernel, that product times 1 / (2 pi)
    (two roundings and the constant's own 2^-54: 2.5 x 2^-53 a): 4 x 2^-53 a of |u| + |v| more, which counts from positions of 1e8 on."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
    half = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    out, size = y.clone(), 32 * 2.0 ** -24 * y.abs()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    u, v = y[..., a], y[..., b]
    out[..., a], out[..., b] = u * c - v * s, v * c + u * s
    both = (u.abs() + v.abs()) * (32 * 2.0 ** -24 + 4 * 2.0 ** -53 * angle.abs()[:, None])
    size[..., a], size[..., b] = both, both
    return out, HALF[x.dtype] * out.abs() + TINY[x.dtype] + size


def quantise(x, dtype):
    """Vectors x [..., dim] as a cache holds them -> (codes' values in 64 bits, scales or None)."""
    if dtype not in (torch.int8, torch.float8_e4m3fn):
        return x.to(dtype).double(), None
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], torch.zeros_like(x), x)
    amax = x.abs().amax(-1)
    if dtype == torch.int8:
        scale = (amax / 127).float().clamp(min=2.0 ** -126)
        codes = torch.round(x / scale.double()[..., None])  # (to even; the quotient of such numbers is no nearer a border than 64 bits tell)
    else:
        e = torch.full_like(amax, -126)
        for p in range(-126, 121):
            e = torch.where(amax > 448 * 2.0 ** p, torch.full_like(e, p + 1), e)
        scale = torch.exp2(e).float()
        y = x / scale.double()[..., None]
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -40))), min=-6) - 3)
        codes = torch.round(y / step) * step
    return codes, torch.where(bad, torch.full_like(scale, math.nan), scale)


def gather(codes, scales, table, n, page):
    """The n tokens of one sequence: [heads, n, dim] in 64 bits, and which of them are there."""
    pages = codes.shape[0]
    t = torch.arange(n)
    entry = table[t // page].long()
    there = (entry >= 0) & (entry < pages)
    entry = entry.clamp(0, max(0, pages - 1))
    bits = codes.view(torch.int8)[entry, :, t % page].view(codes.dtype) if codes.element_size() == 1 else codes[entry, :, t % page]
    x = bits.float().double()
    if scales is not None:
        x = x * scales.double()[entry, :, t % page][..., None]
    return x.transpose(0, 1), there


def attention(q, k_cache, v_cache, table, lengths, scale=None, k_scale=None, v_scale=None, softcap=0.0, window=0, slopes=None):
    """-> (out, bound, lse, bound).  A score: D exact products summed in 32 bits, at most (D + 8) 2^-24 of the sum of their magnitudes, and a few
    roundings of the score itself (8 x 2^-24 of it, of the cap and of the distance bias); e^d of that bounds a weight's relative error, twice that the
    quotient's.  The sums over the tokens: a lane adds at most len / 32 + 40 terms.  Weights held as two bf16 numbers keep 2^-17."""
    q, k_cache, v_cache, table = q.cpu(), k_cache.cpu(), v_cache.cpu(), table.cpu()
    k_scale, v_scale, slopes = (None if x is None else x.cpu() for x in (k_scale, v_scale, slopes))
    batch, hq, dim = q.shape
    hk, page = k_cache.shape[1], k_cache.shape[2]
    group = hq // hk
    scale = dim ** -0.5 if scale is None else scale
    out, obound = torch.zeros(batch, hq, dim, dtype=torch.float64), torch.zeros(batch, hq, dim, dtype=torch.float64)
    lse, lbound = torch.full((batch, hq), -math.inf, dtype=torch.float64), torch.zeros(batch, hq, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        n = max(0, min(n, table.shape[1] * page))
        lo = max(0, n - window) if window else 0
        if n == 0:
            continue
        k, there = gather(k_cache, k_scale, table[b], n, page)
        v, _ = gather(v_cache, v_scale, table[b], n, page)
        keep = there & (torch.arange(n) >= lo)
        if not keep.any():
            continue
        k, v = k[:, keep].repeat_interleave(group, 0), v[:, keep].repeat_interleave(group, 0)
        x = q[b].double()
        s = (x[:, None] * k).sum(-1) * scale
        err = (dim + 8) * 2.0 ** -24 * abs(scale) * (x[:, None] * k).abs().sum(-1) + 8 * 2.0 ** -24 * s.abs()
        if softcap:
            s = softcap * torch.tanh(s / softcap)
            err = err + 8 * 2.0 ** -24 * softcap
        if slopes is not None:
            far = (n - 1 - torch.arange(n)[keep]).double() * slopes.double()[:, None]
            s = s - far
            err = err + 8 * 2.0 ** -24 * far.abs()
        total = torch.logsumexp(s, -1)
        p = torch.exp(s - total[:, None])
        err = err + 4 * 2.0 ** -24 * ((s - s.amax(-1, keepdim=True)).abs() * (p > 1e-30))
        d = (p * err).sum(-1) + 2.0 ** -24 * (8 + total.abs())  # of the sum of weights, and of lse
        adds = (n / 32 + 40) * 2.0 ** -24
        lse[b], lbound[b] = total, d + adds
        out[b] = (p[..., None] * v).sum(1)
        size = (p[..., None] * v.abs()).sum(1)
        obound[b] = HALF[q.dtype] * out[b].abs() + TINY[q.dtype] + (2 * (p[..., None] * err[..., None] * v.abs()).sum(1)
                                                                  + size * (d[:, None] + 2 * adds + 2.0 ** -17)) * 1.01
    return out, obound, lse, lbound


def logprobs(logits, targets, top):
    """-> dict of (value, bound); ids without a bound.  In 32 bits: an exponent (x - m) log2(e) is off by 2^-23 of itself, e^ of it by that times
    |x - m|, which with e^-|x - m| averages below the entropy's terms; a lane adds at most vocab / 256 + 80 terms."""
    x = logits.cpu().double()
    t = targets.cpu().reshape(x.shape[0], -1)
    vocab = x.shape[1]
    bad = torch.isnan(x).any(-1) | (x == math.inf).any(-1)
    none = (x == -math.inf).all(-1) & ~bad
    m = torch.where(bad | none, torch.zeros(()).double(), x.amax(-1))
    z = torch.where((bad | none)[:, None], torch.zeros(()).double(), x - m[:, None])
    lse = torch.logsumexp(z, -1)
    p = torch.exp(z - lse[:, None])
    mean = (p * torch.where(p > 0, -z, torch.zeros(()).double())).sum(-1)  # of |x - m|
    entropy = torch.special.entr(p).sum(-1)
    d = 2.0 ** -23 * (mean + 4) + (vocab / 256 + 80) * 2.0 ** -24         # of the sum, relative
    given = z.gather(1, t.clamp(0, vocab - 1)) - lse[:, None]
    gbound = (d + 2.0 ** -23 * lse.abs())[:, None] + 2.0 ** -23 * given.abs()
    given = torch.where(none[:, None], torch.full_like(given, -math.inf), given)
    given = torch.where((t >= vocab) | ((t >= 0) & bad[:, None]), torch.full_like(given, math.nan), given)
    given = torch.where(t < 0, torch.zeros_like(given), given)
    gbound = torch.where(torch.isfinite(gbound), gbound, torch.zeros_like(gbound))
    second = (p * torch.where(p > 0, z * z, torch.zeros(()).double())).sum(-1)
    ebound = d * (2 + entropy + mean) + 2.0 ** -23 * (second + mean + entropy + 1)
    entropy = torch.where(bad, torch.full_like(entropy, math.nan), torch.where(none, torch.zeros_like(entropy), entropy))
    order = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    r = {"logprobs": (given.reshape(targets.shape), gbound.reshape(targets.shape)), "entropy": (entropy, ebound)}
    if top:
        nan_last = torch.sort(torch.isnan(x).int(), dim=-1, stable=True).indices  # NaN behind -inf
        by_value = torch.sort(order.gather(1, nan_last), dim=-1, descending=True, stable=True).indices
        ids = nan_last.gather(1, by_value)[:, :top]
        lp = z.gather(1, ids) - lse[:, None]
        lp = torch.where(none[:, None], torch.full_like(lp, -math.inf), lp)
        lp = torch.where(bad[:, None], torch.full_like(lp, math.nan), lp)
        b = (d + 2.0 ** -23 * lse.abs())[:, None] + 2.0 ** -23 * torch.where(torch.isfinite(lp), lp.abs(), torch.zeros_like(lp))
        r["top_ids"], r["top_logprobs"] = ids, (lp, b)
    return r
