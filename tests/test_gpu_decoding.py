"""GPU: the decoding operators (bergen_amd/decoding.py) against plain implementations in 64 bits (tests/decoding_reference.py, which
derives the bounds), at the sizes, strides, masks and values where they can go wrong, and a whole decoding step of them."""
import math

import pytest
import torch

import bergen_amd
import decoding_reference as ref

pytestmark = pytest.mark.gpu

BF, HF, F32, I8, E4 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
CACHES = [BF, HF, I8, E4]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ---- rotary ----------------------------------------------------------------------------------------------------------------

def check_rotary(q, k, positions, inv_freq, qw=None, kw=None, interleaved=False, inplace=False, eps=1e-6):
    wants = [ref.rotary(x.clone(), positions, inv_freq, w, eps, interleaved) for x, w in ((q, qw), (k, kw))]
    got = bergen_amd.qk_norm_rotary(q, k, positions, inv_freq, q_weight=qw, k_weight=kw, eps=eps, interleaved=interleaved, inplace=inplace)
    if inplace:
        assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k.data_ptr()
    for name, x, (want, bound) in zip("qk", got, wants):
        ref.assert_within(x, want, bound, name)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, nq, nk, dim, rot", [
    (1, 1, 1, 16, 16), (1, 32, 8, 128, 128), (7, 4, 4, 64, 32), (33, 12, 12, 64, 64), (5, 5, 1, 80, 80), (9, 3, 1, 96, 48), (130, 2, 1, 256, 256),
    (3, 64, 8, 128, 64), (300, 1, 1, 16, 16), (4, 3, 2, 100, 100), (4, 2, 2, 7, 4), (5, 3, 1, 1, 0), (6, 2, 1, 250, 30), (2, 40, 1, 128, 0), (11, 2, 2, 72, 24)])
def test_rotary(dtype, interleaved, tokens, nq, nk, dim, rot):
    g = gen(tokens * dim + nq)
    q, k = randn(g, tokens, nq, dim, dtype=dtype), 3 * randn(g, tokens, nk, dim, dtype=dtype)
    pos = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    f = bergen_amd.rotary_frequencies(rot)
    w = [1 + 0.3 * randn(g, dim) for _ in range(2)]
    check_rotary(q, k, pos, f, w[0].to(dtype), w[1].to(dtype), interleaved)
    check_rotary(q, k, pos.int(), f, None, w[1], interleaved)
    check_rotary(q, k, pos, f, None, None, interleaved, inplace=True)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_strides(dtype):
    """Slices of one projection, rows that start off a 16-byte border, heads-first storage, in place inside a larger matrix."""
    g = gen(3)
    f, pos, w = bergen_amd.rotary_frequencies(64), torch.arange(9, device="cuda"), 1 + 0.1 * randn(g, 64, dtype=dtype)
    qkv = randn(g, 9, 10, 64, dtype=dtype)
    rest = qkv[:, 8:].clone()
    check_rotary(qkv[:, :6], qkv[:, 6:8], pos, f, w, w)
    before = qkv._version
    check_rotary(qkv[:, :6], qkv[:, 6:8], pos, f, w, w, inplace=True)
    assert qkv._version > before                                # autograd is told
    assert torch.equal(qkv[:, 8:], rest)
    odd = randn(g, 9 * 10 * 65 + 1, dtype=dtype)[1:].view(9, 10, 65)
    check_rotary(odd[:, :6, :64], odd[:, 6:8, 1:], pos, f, w, w)
    check_rotary(odd[:, :6, :64], odd[:, 6:8, 1:], pos, f, w, w, True, inplace=True)
    first = randn(g, 10, 9, 64, dtype=dtype).transpose(0, 1)
    check_rotary(first[:, :6], first[:, 6:], pos, f, w, None)
    shared = randn(g, 1, 10, 64, dtype=dtype).expand(9, 10, 64)  # (read, not written)
    check_rotary(shared[:, :6], shared[:, 6:], pos, f, w, w)


@pytest.mark.parametrize("dtype, dim", [(BF, 64), (BF, 50), (F32, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_place_between_heads(dtype, dim, interleaved):
    """[tokens, heads, 3, dim]: each head's query, key and value side by side.  The values, and what a call on copies gives, stay as they are."""
    g = gen(12)
    f, pos, w = bergen_amd.rotary_frequencies(dim), torch.arange(9, device="cuda"), 1 + 0.1 * randn(g, dim, dtype=dtype)
    x = randn(g, 9, 6, 3, dim, dtype=dtype)
    want = bergen_amd.qk_norm_rotary(x[:, :, 0].contiguous(), x[:, :, 1].contiguous(), pos, f, w, w, interleaved=interleaved)
    values = x[:, :, 2].clone()
    check_rotary(x[:, :, 0], x[:, :, 1], pos, f, w, w, interleaved, inplace=True)
    for i in (0, 1):
        assert torch.equal(x[:, :, i], want[i])
    assert torch.equal(x[:, :, 2], values)


def test_rotary_far_positions_and_values():
    g = gen(4)
    f = bergen_amd.rotary_frequencies(128, theta=500000.0, scale=0.25)
    pos = torch.tensor([0, 1, 131071, 1 << 20, (1 << 31) - 1, (1 << 40) + 3, -7, -(1 << 33)], device="cuda")
    q, k = randn(g, 8, 4, 128), randn(g, 8, 2, 128)
    check_rotary(q, k, pos, f)
    check_rotary(q, k, pos, f, interleaved=True)
    w = torch.ones(128, device="cuda")
    check_rotary(q * 1e-12, k * 0, pos, f, w, w)            # eps decides; a vector of zeros stays zero
    check_rotary(q * 1e15, k * 1e-30, pos, f, w, w, eps=0.0 + 1e-30)
    bad = q.clone()
    bad[2, 1, 5], bad[3, 0, 7] = math.nan, math.inf
    out, _ = bergen_amd.qk_norm_rotary(bad, k, pos, f, w, w)
    good = torch.ones(8, 4, dtype=torch.bool)
    good[2, 1] = good[3, 0] = False
    want, _ = bergen_amd.qk_norm_rotary(q, k, pos, f, w, w)
    assert torch.equal(out.cpu()[good], want.cpu()[good])     # a bad vector spoils none of its neighbours
    assert torch.isnan(out[2, 1]).all()


@pytest.mark.parametrize("dim, interleaved", [(128, False), (128, True), (100, False), (30, True)])
def test_rotary_sines(dim, interleaved):
    """Pairs (1, 0) come out as the cosine and sine themselves, with no rounding but their own: half a step of fp32, the angle's three roundings in 64 bits (the
    test's own product is one more) and the series' 2^-36."""
    pos = torch.cat([torch.arange(2000), torch.tensor([131071, 1 << 20, (1 << 31) - 1])]).cuda()
    f = torch.cat([bergen_amd.rotary_frequencies(dim)[: dim // 2 - 5], torch.tensor([math.pi / 4, math.pi / 2, math.pi, -math.pi / 2, -0.1], device="cuda").double()])
    a, b = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
    q = torch.zeros(len(pos), 1, dim, device="cuda")
    q[..., a] = 1
    out, _ = bergen_amd.qk_norm_rotary(q, q, pos, f, interleaved=interleaved)
    angle = pos.cpu().double()[:, None] * f.cpu()
    for got, want in ((out[:, 0, a], angle.cos()), (out[:, 0, b], angle.sin())):
        ref.assert_within(got, want, 2.0 ** -24 * want.abs() + 4 * 2.0 ** -53 * angle.abs() + 2.0 ** -36, "sine")


def test_rotary_of_nothing():
    q, k = torch.zeros(0, 4, 64, dtype=BF, device="cuda"), torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    a, b = bergen_amd.qk_norm_rotary(q, k, torch.zeros(0, dtype=torch.int64, device="cuda"), bergen_amd.rotary_frequencies(64))
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)


# ---- cache -----------------------------------------------------------------------------------------------------------------

def read_bound(values, dtype):
    return (ref.HALF[dtype] + 2.0 ** -24) * values.abs() + ref.TINY[dtype]  # the product in 32 bits, then the type


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("tokens, heads, dim, page", [(1, 1, 16, 8), (37, 3, 64, 16), (130, 8, 128, 64), (9, 2, 80, 8), (20, 1, 256, 1024), (11, 3, 100, 32),
                                                      (7, 2, 1, 8), (5, 4, 250, 16)])
def test_cache(cache, dtype, tokens, heads, dim, page):
    g = gen(tokens + dim)
    pages = -(-tokens // page) + 2
    c = bergen_amd.kv_cache(pages, heads, page, dim, cache)
    for t in (c.k_cache, c.v_cache):
        t.view(torch.int8 if t.element_size() == 1 else torch.int16).fill_(7)
    if c.k_scale is not None:
        c.k_scale.fill_(3), c.v_scale.fill_(3)
    before = [t.clone() for t in c if t is not None]
    k, v = 10 * randn(g, tokens, heads, dim, dtype=dtype), (randn(g, tokens, heads, dim) * torch.exp(4 * randn(g, tokens, heads, 1))).to(dtype)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].contiguous()
    slots[tokens // 2] = -1
    bergen_amd.kv_cache_write(k, v, slots, *c)
    back = bergen_amd.kv_cache_read(slots, *c, dtype=F32)
    kept = slots.cpu() >= 0
    for x, got, codes, scale in ((k, back[0], c.k_cache, c.k_scale), (v, back[1], c.v_cache, c.v_scale)):
        want, s = ref.quantise(x.cpu(), cache)
        p, o = slots.cpu()[kept] // page, slots.cpu()[kept] % page
        stored = codes.cpu().float().double()[p, :, o] if cache != E4 else codes.cpu().view(I8)[p, :, o].view(E4).float().double()
        assert torch.equal(stored, want[kept]), "codes"           # whole numbers and whole roundings: no tolerance
        if s is not None:
            assert torch.equal(torch.nan_to_num(scale.cpu()[p, :, o], 7.0), torch.nan_to_num(s[kept], 7.0)), "scales"  # (NaN: fp16's infinities)
            want = want * s.double()[..., None]
        ref.assert_within(got.cpu()[kept], want[kept], read_bound(want[kept], F32), "read")
        assert not got.cpu()[~kept].any()
        low = bergen_amd.kv_cache_read(slots, *c, dtype=dtype)[0 if codes is c.k_cache else 1]
        ref.assert_within(low.cpu()[kept], want[kept], read_bound(want[kept], dtype), "read, its own type")
    # what no slot names is as it was
    touched = torch.zeros(pages, page, dtype=torch.bool)
    touched.view(-1)[slots.cpu()[kept]] = True
    for now, was in zip([t for t in c if t is not None], before):
        a, b = (x.view(torch.int8).cpu() if x.element_size() == 1 else x.cpu() for x in (now, was))
        assert torch.equal(a.transpose(1, 2)[~touched], b.transpose(1, 2)[~touched])


@pytest.mark.parametrize("cache", [BF, E4])
def test_a_write_is_told_to_autograd(cache):
    """A backward pass that needs what the cache held before a write is refused, as after torch's own writes in place."""
    c = bergen_amd.kv_cache(2, 1, 8, 16, cache)
    held = c.v_scale if cache is E4 else c.v_cache
    w = torch.ones_like(held, requires_grad=True)
    y = (w * held).sum()
    with torch.no_grad():
        bergen_amd.kv_cache_write(torch.ones(1, 1, 16, device="cuda"), torch.ones(1, 1, 16, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), *c)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("dim", [64, 50])
@pytest.mark.parametrize("cache", [I8, E4])
def test_quantising_borders(cache, dim):
    """Vectors whose quotients fall on and next to the borders between codes; zeros, the smallest and largest numbers, infinities and NaN."""
    rows = []
    for amax in (127.0, 127.0 * 3, 1.0, 448.0, 449.0, 1e-3, 3e38, 2e-38, 1e-44, 0.0):
        x = torch.linspace(-1, 1, dim, dtype=torch.float64) * amax
        x[0] = amax
        rows.append(x.float())
        half = ((torch.arange(dim) % 126) + 0.5) * (amax / 127)          # ties of int8, as near as fp32 gives them
        half[0] = amax
        rows += [half.float(), torch.nextafter(half.float(), torch.zeros(dim)).clamp(max=amax), half.float() * -1]
        tie = torch.tensor([17.0, 19, 21, 1.0625, 1.1875, 2 ** -10, 3 * 2 ** -10, 2 ** -9])  # ties of e4m3's grid, at its largest scale and below
        rows.append(torch.cat([torch.tensor([448.0]), tie.repeat(dim)[: dim - 1]]) * (2.0 ** -7 if amax == 1.0 else 1.0))
    x = torch.stack(rows)[:, None].cuda()
    bad = x[:3].clone()
    bad[0, 0, 3], bad[1, 0, 4], bad[2, 0, 5] = math.nan, math.inf, -math.inf
    x = torch.cat([x, bad])
    c = bergen_amd.kv_cache(16, 1, 8, dim, cache)
    slots = torch.arange(x.shape[0], device="cuda")
    bergen_amd.kv_cache_write(x, x, slots, *c)
    codes, scale = ref.quantise(x.cpu(), cache)
    n = x.shape[0]
    stored = c.k_cache.cpu().float().reshape(-1, 1, dim)[:n].double()
    assert torch.equal(stored, codes) and torch.equal(c.v_cache.cpu().float().reshape(-1, 1, dim)[:n].double(), codes)
    assert torch.equal(torch.nan_to_num(c.k_scale.cpu().reshape(-1, 1)[:n], 5.0), torch.nan_to_num(scale, 5.0))
    back = bergen_amd.kv_cache_read(slots, *c, dtype=F32)[0].cpu()
    assert torch.isnan(back[-3:]).all() and torch.isfinite(back[:-3]).all()


def test_cache_slots_outside():
    c = bergen_amd.kv_cache(2, 2, 8, 32, I8)
    k = randn(gen(1), 5, 2, 32)
    slots = torch.tensor([-1, 16, 3, 1 << 40, -(1 << 50)], device="cuda")
    bergen_amd.kv_cache_write(k, k, slots, *c)
    assert int((c.k_scale != 0).sum()) == 2 and (c.k_scale[0, :, 3] != 0).all()
    a, b = bergen_amd.kv_cache_read(slots, *c, dtype=HF)
    assert not a[[0, 1, 3, 4]].any() and not b[[0, 1, 3, 4]].any() and a[2].any()
    bergen_amd.kv_cache_write(k[:0], k[:0], slots[:0], *c)
    assert bergen_amd.kv_cache_read(slots[:0], *c)[0].shape == (0, 2, 32)


@pytest.mark.parametrize("cache", [BF, I8])
def test_an_empty_cache(cache):
    """No pages: every slot and every table entry is outside it.  Sizes are still checked."""
    c = bergen_amd.kv_cache(0, 2, 16, 64, cache)
    k, slots = torch.ones(3, 2, 64, dtype=BF, device="cuda"), torch.tensor([0, -1, 5], device="cuda")
    bergen_amd.kv_cache_write(k, k, slots, *c)
    for x in bergen_amd.kv_cache_read(slots, *c):
        assert x.shape == (3, 2, 64) and not x.any()
    q, n = torch.ones(2, 4, 64, dtype=BF, device="cuda"), torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    out, lse = bergen_amd.paged_attention(q, c.k_cache, c.v_cache, torch.zeros(2, 300, dtype=torch.int32, device="cuda"), n, k_scale=c.k_scale,
                                          v_scale=c.v_scale, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    c = bergen_amd.kv_cache(0, 2, 12, 64, cache)
    for call in (lambda: bergen_amd.kv_cache_write(k, k, slots, *c), lambda: bergen_amd.kv_cache_read(slots, *c)):
        with pytest.raises(RuntimeError, match="page_size 12"):
            call()


def test_cache_strides():
    g = gen(2)
    qkv = randn(g, 6, 7, 48, dtype=BF)
    odd = randn(g, 6, 3, 49, dtype=BF)
    for k, v in ((qkv[:, 3:5], qkv[:, 5:]), (odd[:, :2, 1:], odd[:, 1:, :48])):
        for cache in (BF, I8):
            c = bergen_amd.kv_cache(1, 2, 8, 48, cache)
            d = bergen_amd.kv_cache(1, 2, 8, 48, cache)
            slots = torch.arange(6, device="cuda")
            bergen_amd.kv_cache_write(k, v, slots, *c)
            bergen_amd.kv_cache_write(k.contiguous(), v.contiguous(), slots, *d)
            for a, b in zip(c, d):
                assert a is None or torch.equal(a, b)


# ---- attention -------------------------------------------------------------------------------------------------------------

def made_cache(g, pages, heads, page, dim, cache, spoil=True):
    """A cache full of numbers; spoil: garbage that only tokens behind a sequence's end may hold (set by the caller)."""
    c = bergen_amd.kv_cache(pages, heads, page, dim, cache)
    rows = pages * page
    k, v = randn(g, rows, heads, dim), randn(g, rows, heads, dim) * torch.exp(randn(g, rows, heads, 1))
    bergen_amd.kv_cache_write(k, v, torch.arange(rows, device="cuda"), *c)
    return c


def table_for(g, lengths, page, pages, extra=1):
    wide = max([-(-n // page) for n in lengths] + [0]) + extra
    order, at = torch.randperm(pages, generator=g, device="cuda").int(), 0
    t = torch.full((len(lengths), wide), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths):
        need = -(-n // page)
        t[b, :need] = order[at: at + need]
        at += need
    return t


def spoil_tails(c, table, lengths, page):
    """NaN behind the end of each sequence's last page, in codes (16 bits) or scales (8 bits)."""
    for b, n in enumerate(lengths):
        if n % page:
            last = int(table[b, n // page])
            for codes, scale in ((c.k_cache, c.k_scale), (c.v_cache, c.v_scale)):
                if scale is not None:
                    scale[last, :, n % page:] = math.nan
                else:
                    codes[last, :, n % page:] = math.nan


def check_attention(q, c, table, lengths, window=0, softcap=0.0, slopes=None, scale=None):
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = bergen_amd.paged_attention(q, c.k_cache, c.v_cache, table, n, scale=scale, k_scale=c.k_scale, v_scale=c.v_scale, softcap=softcap,
                                          window=window, alibi_slopes=slopes, return_lse=True)
    want, bound, wlse, lbound = ref.attention(q, c.k_cache, c.v_cache, table, n, scale, c.k_scale, c.v_scale, softcap, window, slopes)
    ref.assert_within(lse, wlse, lbound, "lse")
    ref.assert_within(out, want, bound, "out")
    return out, lse


LENGTHS = [0, 1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 127, 128, 129, 200, 300]


@pytest.mark.parametrize("cache", ["own", I8, E4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq, hk, dim, page", [(1, 1, 16, 8), (8, 2, 64, 16), (32, 8, 128, 16), (12, 12, 64, 32), (6, 2, 80, 8), (5, 1, 96, 64),
                                               (16, 1, 256, 16), (20, 1, 128, 128), (33, 1, 48, 16), (4, 2, 240, 1024), (7, 7, 112, 8)])
def test_attention(cache, dtype, hq, hk, dim, page):
    g = gen(hq * dim + page)
    pages = sum(-(-n // page) for n in LENGTHS) + 3
    c = made_cache(g, pages, hk, page, dim, dtype if cache == "own" else cache)
    table = table_for(g, LENGTHS, page, pages)
    spoil_tails(c, table, LENGTHS, page)
    q = 2 * randn(g, len(LENGTHS), hq, dim, dtype=dtype)
    check_attention(q, c, table, LENGTHS)
    slopes = torch.exp2(-8 * torch.rand(hq, generator=g, device="cuda"))
    check_attention(q, c, table, LENGTHS, window=33, softcap=20.0, slopes=slopes, scale=0.3)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 5000])
@pytest.mark.parametrize("cache", [BF, I8])
def test_attention_windows(window, cache):
    g = gen(window)
    lengths = [1, 31, 32, 33, 64, 65, 1000, 2049]
    pages = sum(-(-n // 16) for n in lengths)
    c = made_cache(g, pages, 2, 16, 64, cache)
    check_attention(randn(g, 8, 4, 64, dtype=BF), c, table_for(g, lengths, 16, pages, 0), lengths, window=window)


@pytest.mark.parametrize("cache", [HF, I8, E4])
def test_attention_of_long_sequences(cache):
    """More than one split, ragged: the longest fills all of them, the shortest one."""
    g = gen(9)
    lengths = [20011, 1, 0, 4097, 511, 512, 513, 19999]
    pages = sum(-(-n // 32) for n in lengths) + 1
    c = made_cache(g, pages, 2, 32, 128, cache)
    table = table_for(g, lengths, 32, pages)
    spoil_tails(c, table, lengths, 32)
    q = 3 * randn(g, 8, 10, 128, dtype=HF)
    check_attention(q, c, table, lengths)
    check_attention(q, c, table, lengths, window=6000, softcap=30.0)
    one = check_attention(q[3:4], c, table[3:4], lengths[3:4])
    assert torch.equal(one[0], check_attention(q[3:4], c, table[3:4], lengths[3:4])[0])  # the same call, the same bits


@pytest.mark.parametrize("softcap", [127.0, 129.0, 1e4, 1e7, 1e30])
@pytest.mark.parametrize("cache, dim", [(BF, 64), (I8, 128), (E4, 256)])
def test_attention_with_a_high_cap(cache, dim, softcap):
    """A cap far above the scores leaves them as they are, to their own roundings: tanh adds less than 14 x 2^-24 of a score, and the plain bound holds
    dim + 16 of those.  Below 128 the cap's own 8 x 2^-24 is allowed for."""
    g = gen(int(softcap % 1000) + dim)
    lengths = [1, 40, 333]
    c = made_cache(g, 40, 2, 16, dim, cache)
    table = table_for(g, lengths, 16, 40)
    q, n = 6 * randn(g, 3, 4, dim, dtype=BF), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got, lse = bergen_amd.paged_attention(q, c.k_cache, c.v_cache, table, n, k_scale=c.k_scale, v_scale=c.v_scale, softcap=softcap, return_lse=True)
    want, cap_bound, wlse, cap_lbound = ref.attention(q, c.k_cache, c.v_cache, table, n, None, c.k_scale, c.v_scale, softcap)
    _, bound, _, lbound = ref.attention(q, c.k_cache, c.v_cache, table, n, None, c.k_scale, c.v_scale)
    ref.assert_within(lse, wlse, cap_lbound if softcap < 128 else 2 * lbound, "lse")
    ref.assert_within(got, want, cap_bound if softcap < 128 else 2 * bound, "out")


@pytest.mark.parametrize("cache", [BF, I8, E4])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_attention_where_the_distance_decides(dim, cache):
    """Keys of zeros: the weights are the slopes' alone, another one in each of 20 heads of a group (16 and 4 of them in a workgroup)."""
    g = gen(dim)
    lengths = [1, 33, 200, 1500]
    pages = sum(-(-n // 16) for n in lengths)
    c = made_cache(g, pages, 2, 16, dim, cache)
    c.k_cache.view(torch.int8 if cache != BF else torch.int16).zero_()
    slopes = torch.exp2(-12 * torch.rand(40, generator=g, device="cuda"))
    check_attention(randn(g, 4, 40, dim, dtype=BF), c, table_for(g, lengths, 16, pages, 0), lengths, slopes=slopes)


def test_attention_of_queries_off_a_border():
    """Dense queries that start 2 bytes behind a 16-byte border, and slices of rows of odd length, give what aligned ones do."""
    g = gen(14)
    c, n = made_cache(g, 12, 2, 16, 64, BF), torch.tensor([20, 60], dtype=torch.int32, device="cuda")
    table = table_for(g, [20, 60], 16, 12, 0)
    q = randn(g, 2, 4, 64, dtype=BF)
    want = bergen_amd.paged_attention(q, c.k_cache, c.v_cache, table, n)
    off = torch.empty(513, dtype=BF, device="cuda")[1:].view(2, 4, 64).copy_(q)
    odd = torch.empty(2, 4, 65, dtype=BF, device="cuda")[..., 1:].copy_(q)
    assert off.is_contiguous() and off.data_ptr() % 16 == 2
    for x in (off, odd):
        assert torch.equal(bergen_amd.paged_attention(x, c.k_cache, c.v_cache, table, n), want)


@pytest.mark.parametrize("cache", [BF, I8])
def test_attention_without_some_pages(cache):
    """Table entries outside the cache: their tokens are left out; where all are, zeros and -inf.  Lengths outside the table's width."""
    g = gen(5)
    c = made_cache(g, 12, 2, 8, 64, cache)
    table = torch.tensor([[0, -1, 2, 99, 4], [-1, -1, -1, -1, -1], [12, 1 << 30, -5, 3, 5], [6, 7, 8, 9, 10], [11, 1, 0, 2, 3]], dtype=torch.int32, device="cuda")
    q = randn(g, 5, 8, 64, dtype=BF)
    out, lse = check_attention(q, c, table, [40, 40, 37, 1000000, -3])
    assert not out[1].any() and (lse[1] == -math.inf).all() and not out[4].any()
    out, lse = check_attention(q, c, table, [16, 5, 20, 40, 0], window=3)  # a window that ends in a missing page
    assert (lse[0] == -math.inf).all() and not out[0].any()


def test_attention_values():
    """Keys that leave one token all the weight, equal scores, infinite and NaN entries of tokens that count and of tokens that do not."""
    g = gen(6)
    for cache in (BF, HF):
        c = bergen_amd.kv_cache(8, 1, 16, 64, cache)
        c.k_cache.zero_(), c.v_cache.copy_(randn(g, 8, 1, 16, 64))
        q = torch.ones(1, 2, 64, dtype=cache, device="cuda")
        table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
        check_attention(q, c, table, [100])                        # all scores equal
        c.k_cache[3, 0, 5] = 30.0                                  # one far above: e^-1920 underflows
        check_attention(q, c, table, [100], scale=1.0)
        c.k_cache[3, 0, 5] = 0
        c.v_cache[6, 0, 4:] = math.inf                             # token 100 and later do not count
        c.k_cache[6, 0, 4:] = math.nan
        c.v_cache[7] = math.nan
        check_attention(q, c, table, [100])
        c.v_cache[2, 0, 1, 7] = math.inf                           # token 33, dim 7
        out, lse = check_attention(q, c, table, [100])
        assert torch.isinf(out[0, :, 7]).all() and torch.isfinite(lse).all()
        out, lse = check_attention(q, c, table, [100], window=60)   # ... outside the window
        assert torch.isfinite(out).all()
        c.k_cache[2, 0, 1] = math.nan
        out, _ = check_attention(q, c, table, [100], window=60)
        out = bergen_amd.paged_attention(q, c.k_cache, c.v_cache, table, torch.tensor([100], dtype=torch.int32, device="cuda"))
        assert torch.isnan(out).all()


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1.0, 1e4, 1e30])
def test_attention_scales_of_values(size):
    """8-bit values of very different sizes next to each other, bf16 queries far outside fp16's range."""
    g = gen(7)
    for cache in (I8, E4):
        c = bergen_amd.kv_cache(10, 2, 32, 64, cache)
        rows = 320
        k = randn(g, rows, 2, 64)
        v = randn(g, rows, 2, 64) * torch.exp(6 * randn(g, rows, 2, 1)) * size
        bergen_amd.kv_cache_write(k, v, torch.arange(rows, device="cuda"), *c)
        table = torch.randperm(10, generator=g, device="cuda").int()[None]
        q = (randn(g, 1, 8, 64) * 1e8).to(BF)
        q[0, 0], q[0, 1] = 0, 1e-20
        check_attention(q, c, table, [311], scale=1e-9)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cache", [I8, E4])
@pytest.mark.parametrize("far", [1e6, 1e12, 1e25, 1e-25])
def test_attention_of_large_values_without_weight(cache, dim, far):
    """8-bit values that are far larger than those that count (or far smaller) and weigh next to nothing: the distance bias leaves e^-100 and less of
    the tokens before the last 100, and in the last sequence a score of its own decides."""
    g = gen(dim)
    lengths = [400, 130, 1500, 300]
    pages = sum(-(-n // 16) for n in lengths)
    c = bergen_amd.kv_cache(pages, 2, 16, dim, cache)
    rows = pages * 16
    table = table_for(g, lengths, 16, pages, 0)
    k, v = torch.zeros(rows, 2, dim, device="cuda"), randn(g, rows, 2, dim)
    for b, n in enumerate(lengths):
        t = torch.arange(n, device="cuda")
        slot = table[b].long()[t // 16] * 16 + t % 16
        v[slot[: max(0, n - 110)]] *= far
        if b == 3:
            k[slot[7]], v[slot[7]] = 300.0, 1.0
    bergen_amd.kv_cache_write(k, v, torch.arange(rows, device="cuda"), *c)
    q = torch.ones(4, 8, dim, dtype=BF, device="cuda")
    check_attention(q, c, table, lengths, slopes=torch.linspace(1.0, 1.5, 8, device="cuda"))


@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("cache", [I8, E4])
@pytest.mark.parametrize("large", [2.0 ** 20, 2.0 ** 26, 2.0 ** 40])
def test_attention_of_queries_with_a_large_element(cache, dim, large):
    """bf16 queries whose largest element meets zeros in the keys: the scores are the small elements' alone."""
    g = gen(dim)
    lengths = [1, 40, 333]
    c = bergen_amd.kv_cache(40, 2, 16, dim, cache)
    k = randn(g, 640, 2, dim)
    k[:, :, 5] = 0
    bergen_amd.kv_cache_write(k, randn(g, 640, 2, dim), torch.arange(640, device="cuda"), *c)
    q = 3 * randn(g, 3, 4, dim, dtype=BF)
    q[:, :3, 5] = torch.tensor([large, -large, large / 8], device="cuda").to(BF)  # (the fourth head has none)
    check_attention(q, c, table_for(g, lengths, 16, 40), lengths)
    bad = q.clone()
    bad[1, 0, 7], bad[2, 1, 9] = math.inf, math.nan                               # infinite and NaN elements stay with their head
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    table = table_for(gen(1), lengths, 16, 40)
    want, got = (bergen_amd.paged_attention(x, c.k_cache, c.v_cache, table, n, k_scale=c.k_scale, v_scale=c.v_scale) for x in (q, bad))
    assert torch.isnan(got[1, 0]).all() and torch.isnan(got[2, 1]).all()
    keep = torch.ones(3, 4, dtype=torch.bool)
    keep[1, 0] = keep[2, 1] = False
    assert torch.equal(got.cpu()[keep], want.cpu()[keep])


def test_attention_far_into_a_cache():
    """Offsets past 2^31 bytes: 8-bit pages at the end of a cache of 2.5 GB each for keys and values."""
    g = gen(8)
    pages, heads, page, dim = 9600, 8, 256, 128
    kc, vc = (torch.zeros(pages, heads, page, dim, dtype=I8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, heads, page, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 31
    c = bergen_amd.KVCache(kc, vc, ks, vs)
    slots = torch.cat([torch.arange(9598 * page, 9598 * page + 200), torch.arange(9000 * page, 9001 * page)]).cuda()
    k, v = randn(g, 456, heads, dim), randn(g, 456, heads, dim)
    bergen_amd.kv_cache_write(k, v, slots, *c)
    a, b = bergen_amd.kv_cache_read(slots, *c, dtype=F32)
    codes, s = ref.quantise(k.cpu(), I8)
    want = codes * s.double()[..., None]
    ref.assert_within(a, want, read_bound(want, F32), "read")
    assert int((ks != 0).sum()) == 456 * heads
    table = torch.tensor([[9000, 9598]], dtype=torch.int32, device="cuda")
    q = randn(g, 1, 16, dim, dtype=BF)
    near = bergen_amd.KVCache(kc[[9000, 9598]], vc[[9000, 9598]], ks[[9000, 9598]], vs[[9000, 9598]])
    got = bergen_amd.paged_attention(q, kc, vc, table, torch.tensor([456], dtype=torch.int32, device="cuda"), k_scale=ks, v_scale=vs)
    want, _ = check_attention(q, near, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), [456])
    assert torch.equal(got, want)


@pytest.mark.parametrize("cache", [BF, E4])
def test_attention_with_a_wide_table(cache):
    """A table far wider than most sequences need, and more splits wanted than there are: a long sequence takes longer ones."""
    g = gen(12)
    lengths = [33000] + [60] * 63 + [0, 16385]
    pages = sum(-(-n // 8) for n in lengths)
    c = made_cache(g, pages, 24, 8, 16, cache)
    table = table_for(g, lengths, 8, pages, extra=12000)
    check_attention(randn(g, len(lengths), 24, 16, dtype=BF), c, table, lengths)


def test_attention_strides():
    g = gen(10)
    c = made_cache(g, 6, 2, 16, 64, BF)
    wide = torch.arange(12, dtype=torch.int32, device="cuda").reshape(2, 6)
    table = (wide % 6)[:, :3]
    qkv = randn(g, 2, 9, 64, dtype=BF)
    a, _ = check_attention(qkv[:, :8], c, table, [40, 48])
    assert torch.equal(a, check_attention(qkv[:, :8].contiguous(), c, table.contiguous(), [40, 48])[0])
    odd = randn(g, 2, 8, 67, dtype=BF)[..., 3:]
    check_attention(odd, c, table, [40, 48])
    check_attention(qkv[:0, :8], c, table[:0], [])
    check_attention(qkv[:, :8], c, table[:, :0], [4, 5])  # a table of no pages: nothing there


# ---- log probabilities -----------------------------------------------------------------------------------------------------

def check_logprobs(x, t, top):
    got, want = bergen_amd.token_logprobs(x, t, top=top), ref.logprobs(x, t, top)
    ref.assert_within(got.logprobs, *want["logprobs"], "logprobs")
    ref.assert_within(got.entropy, *want["entropy"], "entropy")
    assert got.top_ids.shape == (x.shape[0], top)
    if top:
        assert torch.equal(got.top_ids.cpu(), want["top_ids"]), "ids"
        ref.assert_within(got.top_logprobs, *want["top_logprobs"], "top_logprobs")
    return got


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (2, 7), (5, 63), (4, 64), (3, 65), (2, 511), (2, 513), (3, 2049), (1, 30522), (7, 8193), (2, 50257),
                                         (1300, 300), (1, 262143)])
def test_logprobs(dtype, rows, vocab):
    g = gen(rows + vocab)
    x = (2 * randn(g, rows, vocab)).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    for top in (0, 1, 5, 20, 64):
        if top <= vocab:
            check_logprobs(x, t, top)
    more = torch.randint(-1, vocab + 1, (rows, 3), generator=g, device="cuda")
    check_logprobs(x, more, min(4, vocab))
    check_logprobs(x, t[:, None][:, :0].contiguous(), min(2, vocab))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_logprobs_rows_and_ties(dtype):
    """Equal logits, rising and falling rows, one certain token, large offsets, banned tokens, rows of nothing, NaN and infinities."""
    n = 9001
    ramp = torch.linspace(-30, 30, n)
    rows = [torch.zeros(n), ramp, -ramp, torch.full((n,), -math.inf), torch.full((n,), 3.0), torch.round(ramp), -torch.round(ramp).abs()]
    one = torch.full((n,), -40.0)
    one[4321] = 0
    banned = ramp.clone()
    banned[::2] = -math.inf
    single = torch.full((n,), -math.inf)
    single[77] = 5.0
    offset = ramp / 10 + 1000
    nan, inf, both = ramp.clone(), ramp.clone(), ramp.clone()
    nan[5000], inf[123], both[1], both[2] = math.nan, math.inf, math.nan, math.inf
    few = torch.full((n,), math.nan)
    few[[10, 8000]] = torch.tensor([1.0, 2.0])
    signs = torch.zeros(n)
    signs[::3] = -0.0                                          # -0 and 0 are equal logits
    rows.append(signs)
    x = torch.stack(rows + [one, banned, single, offset, nan, inf, both, few]).to(dtype).cuda()
    t = torch.tensor([0, 8999, 77, 4321, 10], device="cuda").expand(x.shape[0], 5).contiguous()
    for top in (1, 3, 50, 64):
        check_logprobs(x, t, top)
    r = bergen_amd.token_logprobs(x, t, top=3)
    assert r.top_ids[0].tolist() == [0, 1, 2] and r.entropy[3] == 0 and (r.logprobs[3] == -math.inf).all()
    assert abs(float(r.entropy[0]) - math.log(n)) < 1e-5 and torch.isnan(r.logprobs[12]).all()


@pytest.mark.parametrize("dtype, bits, signalling", [(BF, torch.int16, 0x7f81), (F32, torch.int32, 0x7f800001), (HF, torch.int16, 0x7c01)])
def test_logprobs_next_to_a_signalling_nan(dtype, bits, signalling):
    """It spoils its row's probabilities, as any NaN does, and hides no alternative: the largest logit beside it, in each place of a 16-byte vector."""
    g = gen(8)
    x, t = randn(g, 300, 50000, dtype=dtype), torch.zeros(300, dtype=torch.int64, device="cuda")
    rows, at = torch.arange(16, device="cuda"), 40000 + torch.arange(16, device="cuda")
    x[rows, at] = 50.0
    x.view(bits)[rows, at ^ 1] = signalling
    r = bergen_amd.token_logprobs(x, t, top=4)
    assert torch.equal(r.top_ids[:16, 0], at)
    assert torch.isnan(r.logprobs[:16]).all() and torch.isnan(r.top_logprobs[:16]).all() and torch.isfinite(r.logprobs[16:]).all()
    whole = x.float().nan_to_num(nan=-math.inf)  # (every alternative of these rows is a number)
    assert torch.equal(r.top_ids, torch.sort(whole, dim=-1, descending=True, stable=True).indices[:, :4])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_logprobs_of_a_types_limits(dtype):
    """The type's lowest value as a mask, in a whole row too (which is then uniform), its largest, its smallest, and a row of NaN alone."""
    low, high, n = torch.finfo(dtype).min, torch.finfo(dtype).max, 5000
    g = torch.Generator().manual_seed(3)
    some = torch.randn(n, generator=g)
    masked, above = some.clone(), some.clone()
    masked[::3], above[4000] = low, high
    late = torch.full((n,), low)
    late[4999] = -5.0
    rows = [torch.full((n,), low), masked, above, late, torch.full((n,), high), torch.full((n,), torch.finfo(dtype).tiny), torch.full((n,), math.nan)]
    x = torch.stack(rows).to(dtype).cuda()
    t = torch.tensor([0, 4000, 4999], device="cuda").expand(len(rows), 3).contiguous()
    for top in (0, 5):
        r = check_logprobs(x, t, top)
    for i in (0, 4, 5):
        assert abs(float(r.entropy[i]) - math.log(n)) < 1e-5 and torch.allclose(r.logprobs[i], torch.full((3,), -math.log(n), device="cuda"), atol=1e-5)
    assert torch.isnan(r.logprobs[6]).all() and r.top_ids[6].tolist() == [0, 1, 2, 3, 4]
    parts = torch.full((1, 70000), low, device="cuda", dtype=dtype)       # several parts of a row
    parts[0, 69000] = low / 2
    check_logprobs(parts, torch.tensor([69000], device="cuda"), 3)


def masked_rows(dtype, mask, n):
    """Rows of n logits beside, below or above the finite value `mask`: it alone, two allowed tokens in many places, one maximum, steps of one unit up and down."""
    base = torch.tensor(mask, dtype=dtype).double()
    unit = 2.0 ** (math.floor(math.log2(abs(float(base)))) - {F32: 23, BF: 7}[dtype])
    rows = [torch.full((n,), float(base), dtype=torch.float64)]
    for yes, no in ((3, 4), (n // 2, n - 3), (n - 1, 70), (0, n // 3)):
        x = torch.full((n,), float(base), dtype=torch.float64)
        x[yes], x[no] = 1.5, 0.25
        rows.append(x)
    one = torch.full((n,), -math.inf, dtype=torch.float64)
    one[n // 2 + 5] = base
    steps = torch.arange(n, dtype=torch.float64) % 97
    up = base + unit * torch.div(torch.arange(n), n // 60, rounding_mode="floor")  # a new maximum in every part of the row
    rows += [one, base + unit * steps, base - unit * steps, up, up.flip(0), torch.where(steps == 5, -base, base)]
    return torch.stack(rows).to(dtype).cuda()


@pytest.mark.parametrize("mask", [-1e4, -1e5, -1048573.0, -1.0486e6, -1e7, -1e9, -1e10, -1e11, -1e12, -1e20, -1e30])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_of_finite_masks(dtype, mask):
    """Every magnitude of the maximum, on both sides of zero, in a row of several parts and in rows that one workgroup walks in several steps."""
    for sign in (1, -1):
        x = masked_rows(dtype, sign * mask, 20011)
        t = torch.tensor([3, 10005, 20010, 0, 777], device="cuda").expand(x.shape[0], 5).contiguous()
        for top in (0, 5):
            r = check_logprobs(x, t, top)
            assert torch.isfinite(r.entropy).all()
        many = bergen_amd.token_logprobs(x.repeat(100, 1), t.repeat(100, 1), top=5)     # 1100 rows: each in one part
        want = ref.logprobs(x, t, 5)
        for i in (0, 1, 99):
            part = slice(i * len(x), (i + 1) * len(x))
            ref.assert_within(many.logprobs[part], *want["logprobs"], "logprobs")
            ref.assert_within(many.entropy[part], *want["entropy"], "entropy")
            ref.assert_within(many.top_logprobs[part], *want["top_logprobs"], "top_logprobs")
            assert torch.equal(many.top_ids[part].cpu(), want["top_ids"])
    parts = torch.full((1, 70000), mask, device="cuda", dtype=dtype)                    # several parts, allowed tokens in the last one only
    parts[0, 69990], parts[0, 69999] = 2.0, 1.0
    check_logprobs(parts, torch.tensor([[69990, 69999]], device="cuda"), 3)


def test_entropy_of_a_nearly_certain_row():
    """p = 1 - 1e-9: the entropy is kept, not rounded to 0."""
    x = torch.full((2, 1000), -math.inf, device="cuda")
    x[:, 500], x[0, 3], x[1, 900] = 10.0, 10.0 - 20.7, 10.0 - 80.0
    r = check_logprobs(x, torch.tensor([500, 500], device="cuda"), 2)
    for i, d in ((0, 20.7), (1, 80.0)):
        d = 10.0 - float(x[i, 3 if i == 0 else 900])
        p = math.exp(-d) / (1 + math.exp(-d))
        want = p * (d + math.log1p(math.exp(-d))) + (1 - p) * math.log1p(math.exp(-d))
        assert abs(float(r.entropy[i]) - want) < 1e-5 * want


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_strides(dtype):
    """Rows off a 16-byte border (every offset), rows of a wider matrix whose other columns must not be seen."""
    g = gen(1)
    for cut in range(9):
        wide = randn(g, 5, 2100, dtype=dtype)
        wide[:, :cut], wide[:, cut + 1500:] = math.inf, math.nan
        check_logprobs(wide[:, cut: cut + 1500], torch.arange(5, device="cuda"), 10)
    check_logprobs(randn(g, 1, 700, dtype=dtype).expand(3, 700), torch.arange(3, device="cuda"), 3)
    assert bergen_amd.token_logprobs(wide[:0, :99], torch.zeros(0, dtype=torch.int64, device="cuda"), top=4).top_ids.shape == (0, 4)


# ---- refusals that need a device, streams, graphs --------------------------------------------------------------------------

def test_refusals_on_the_device():
    q = torch.zeros(2, 4, 64, dtype=BF, device="cuda")
    f = bergen_amd.rotary_frequencies(64)
    with pytest.raises(ValueError, match="positions is on cpu"):
        bergen_amd.qk_norm_rotary(q, q, torch.zeros(2, dtype=torch.int64), f)
    with pytest.raises(ValueError, match="no backward pass"):
        bergen_amd.qk_norm_rotary(q.clone().requires_grad_(), q, torch.zeros(2, dtype=torch.int64, device="cuda"), f)
    with torch.no_grad():
        bergen_amd.qk_norm_rotary(q.clone().requires_grad_(), q, torch.zeros(2, dtype=torch.int64, device="cuda"), f)
    with pytest.raises(RuntimeError, match="at most 64"):
        bergen_amd.token_logprobs(torch.zeros(1, 100, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), top=65)
    with pytest.raises(ValueError, match="top 11"):
        bergen_amd.token_logprobs(torch.zeros(1, 10, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), top=11)
    c = bergen_amd.kv_cache(2, 1, 16, 72, BF)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        bergen_amd.paged_attention(torch.zeros(1, 1, 72, dtype=BF, device="cuda"), c.k_cache, c.v_cache, torch.zeros(1, 2, dtype=torch.int32, device="cuda"),
                                   torch.ones(1, dtype=torch.int32, device="cuda"))


class Step:
    """One decoding step of a small decoder: 2 layers, a paged cache, the answer's first token's log probabilities."""

    def __init__(self, cache, batch=5, seed=0, hq=8, hk=2, dim=64, page=16, vocab=5003):
        g = gen(seed)
        self.hq, self.hk, self.dim, self.page, self.batch, self.vocab = hq, hk, dim, page, batch, vocab
        d = self.width = hq * dim
        self.layers = []
        self.pages = 20 * batch + 1
        for _ in range(2):
            c = made_cache(g, self.pages, hk, page, dim, cache)
            self.layers.append((randn(g, (hq + 2 * hk) * dim, d, dtype=BF) * d ** -0.5, randn(g, d, d, dtype=BF) * d ** -0.5,
                                1 + 0.2 * randn(g, dim, dtype=BF), 1 + 0.2 * randn(g, dim, dtype=BF), c))
        self.head = randn(g, vocab, d, dtype=BF) * d ** -0.5 * 3
        self.x = randn(g, batch, d, dtype=BF)
        self.table = torch.randperm(self.pages, generator=g, device="cuda")[: 20 * batch].reshape(batch, 20).int()
        self.lengths = torch.randint(1, 20 * page - 8, (batch,), generator=g, device="cuda").int()
        self.targets = torch.randint(0, vocab, (batch, 2), generator=g, device="cuda")
        self.f = bergen_amd.rotary_frequencies(dim)

    def slots(self):
        at = (self.lengths - 1).long()
        return (self.table.gather(1, (at // self.page)[:, None])[:, 0].long() * self.page + at % self.page).contiguous()

    def run(self):
        x, slots, pos = self.x, self.slots(), (self.lengths - 1).contiguous()
        for wqkv, wo, qw, kw, c in self.layers:
            qkv = (x @ wqkv.t()).view(self.batch, -1, self.dim)
            q, k = bergen_amd.qk_norm_rotary(qkv[:, : self.hq], qkv[:, self.hq: self.hq + self.hk], pos, self.f, qw, kw)
            bergen_amd.kv_cache_write(k, qkv[:, self.hq + self.hk:], slots, *c)
            o = bergen_amd.paged_attention(q, c.k_cache, c.v_cache, self.table, self.lengths, k_scale=c.k_scale, v_scale=c.v_scale)
            x = x + o.view(self.batch, -1) @ wo.t()
        return bergen_amd.token_logprobs(x @ self.head.t(), self.targets, top=5)

    def plain(self):
        """The same in 64 bits, with the roundings of what is kept in memory (activations, cache) where the step has them."""
        x, slots = self.x.double().cpu(), self.slots().cpu()
        for wqkv, wo, qw, kw, c in self.layers:
            r = lambda z: z.to(BF).double()  # noqa: E731
            qkv = r(x @ wqkv.double().cpu().t()).view(self.batch, -1, self.dim)
            q, k = qkv[:, : self.hq], qkv[:, self.hq: self.hq + self.hk]
            pos, f = (self.lengths - 1).cpu(), self.f.cpu()
            q = ref.rotary(q.to(BF), pos, f, qw.cpu())[0].to(BF)
            k = ref.rotary(k.to(BF), pos, f, kw.cpu())[0].to(BF)
            store = [z.cpu().clone() if z is not None else None for z in c]
            for new, i in ((k, 0), (qkv[:, self.hq + self.hk:].to(BF), 1)):
                codes, scale = ref.quantise(new, store[i].dtype)
                p, o = slots // self.page, slots % self.page
                if scale is not None:
                    store[i].view(I8)[p, :, o] = codes.float().to(store[i].dtype).view(I8)
                    store[2 + i][p, :, o] = scale
                else:
                    store[i][p, :, o] = codes.to(store[i].dtype)
            out = ref.attention(q, store[0], store[1], self.table, self.lengths.cpu(), None, store[2], store[3])[0]
            x = r(x + r(r(out).reshape(self.batch, -1) @ wo.double().cpu().t()))
        return ref.logprobs((x @ self.head.double().cpu().t()).to(BF), self.targets, 5)


@pytest.mark.parametrize("cache", [BF, I8, E4])
def test_a_decoding_step(cache):
    """All operators as a decoder runs them, against the same step in 64 bits.  Between the two lie only roundings that fall on another side of
    a border (bf16 activations of 2^-8 relative, a code): logits of size ~3 then differ by a few bf16 steps, 0.1 at most."""
    s = Step(cache)
    want, got = s.plain(), s.run()
    assert float((got.logprobs.cpu().double() - want["logprobs"][0]).abs().max()) < 0.1
    assert float((got.entropy.cpu().double() - want["entropy"][0]).abs().max()) < 0.1
    assert (got.top_ids[:, 0].cpu() == want["top_ids"][:, 0]).float().mean() >= 0.6


@pytest.mark.parametrize("cache", [BF, I8])
def test_a_captured_step_replays(cache):
    """Two steps captured into graphs (their workspaces are their own), replayed in turn with new inputs and eager work between: bit for bit the eager results."""
    steps = [Step(cache, seed=1), Step(cache, seed=2, batch=3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in steps:
            s.run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    for turn in range(4):
        for s in steps:
            s.x.copy_(randn(gen(100 + turn), s.batch, s.width, dtype=BF))
            s.lengths.copy_(torch.randint(1, 300, (s.batch,), generator=gen(turn), device="cuda").int())
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        captured = [[t.clone() for t in o] for o in outs]
        torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        for s, c in zip(steps, captured):
            for a, b in zip(s.run(), c):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls on two streams at once, on data of their own: each has its own workspace."""
    g = gen(11)
    lengths = [5000, 4000]
    sets = []
    for _ in range(2):
        pages = sum(-(-n // 16) for n in lengths)
        c = made_cache(g, pages, 2, 16, 64, BF)
        sets.append((randn(g, 2, 8, 64, dtype=BF), c, table_for(g, lengths, 16, pages, 0), randn(g, 2, 60000)))
    n, t = torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor([5, 9], device="cuda")

    def run(q, c, table, x):
        return [bergen_amd.paged_attention(q, c.k_cache, c.v_cache, table, n), *bergen_amd.token_logprobs(x, t, top=9)]
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
