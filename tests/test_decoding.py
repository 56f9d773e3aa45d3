"""CPU: the decoding operators' checks of arguments (bergen_amd/decoding.py and the C entry points), which come before anything
touches a device, and the reference's own formulas against torch's."""
import ctypes
import math

import pytest
import torch

import bergen_amd
import decoding_reference as ref
from bergen_amd import _lib

P = ctypes.c_void_p(4096)  # an address that no refused call reads


def _refused(match, fn, *a, **k):
    with pytest.raises(ValueError, match=match):
        fn(*a, **k)


def _rotary_args(t=3, hq=4, hk=2, d=64, r=64, dtype=torch.bfloat16):
    return dict(q=torch.zeros(t, hq, d, dtype=dtype), k=torch.zeros(t, hk, d, dtype=dtype), positions=torch.zeros(t, dtype=torch.int64),
                inv_freq=torch.zeros(r // 2, dtype=torch.float64))


_QKV = torch.zeros(3, 8, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("change, match", [
    (dict(q=torch.zeros(3, 4, dtype=torch.bfloat16)), r"q must be \[tokens, heads, dim\]"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float64)), "float16, bfloat16 or float32"),
    (dict(k=torch.zeros(3, 2, 32, dtype=torch.bfloat16)), "k must be"),
    (dict(k=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), "k must be"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float16)), "k must be"),
    (dict(positions=torch.zeros(3)), "positions"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), "positions"),
    (dict(inv_freq=torch.zeros(32)), "inv_freq must be float64"),
    (dict(inv_freq=torch.zeros(33, dtype=torch.float64)), "rotary_dim at most 64"),
    (dict(q_weight=torch.zeros(32, dtype=torch.bfloat16)), "q_weight"),
    (dict(q_weight=torch.zeros(64, dtype=torch.float16)), "q_weight"),
    (dict(q_weight=torch.zeros(64), k_weight=torch.zeros(64, dtype=torch.bfloat16)), "one type"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)[..., ::2]), "dense"),
    (dict(q=torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, 4, 64), inplace=True), "overlaps itself"),
    (dict(q=_QKV[:, :4], k=_QKV[:, 3:5], inplace=True), "q and k overlap"),
    (dict(q=_QKV[:, :4], k=_QKV[:, :4], inplace=True), "q and k overlap"),
    (dict(q=_QKV[:1, :4], k=_QKV[:1, 3:], positions=torch.zeros(1, dtype=torch.int64), inplace=True), "q and k overlap"),
    (dict(q=_QKV[:, :4], k=_QKV[:, 4:6], inplace=True), "must be on the GPU"),
    (dict(q=_QKV[:1, :4], k=_QKV[:1, 4:], positions=torch.zeros(1, dtype=torch.int64), inplace=True), "must be on the GPU"),
    (dict(q=_QKV[:, :4].clone(), k=_QKV[:, :4], inplace=True), "must be on the GPU"),
    (dict(), "must be on the GPU"),
])
def test_rotary_refusals(change, match):
    _refused(match, bergen_amd.qk_norm_rotary, **{**_rotary_args(), **change})


def _views(*made):
    buf = torch.zeros(4000, dtype=torch.bfloat16)
    return [buf.as_strided(size, stride, 1000 + at) for size, stride, at in made]


@pytest.mark.parametrize("q, k", [
    (((5, 4, 16), (192, 48, 1), 0), ((5, 4, 16), (192, 48, 1), 16)),       # [tokens, heads, 3, dim]: queries and keys of each head side by side
    (((5, 4, 16), (192, 48, 1), 16), ((5, 4, 16), (192, 48, 1), 0)),
    (((5, 4, 16), (192, 48, 1), 0), ((5, 1, 16), (192, 48, 1), 32)),       # one key head between the queries' heads
    (((5, 4, 16), (192, 48, 1), 0), ((5, 2, 16), (192, 96, 1), 64)),       # every other head
    (((1, 4, 16), (7, 48, 1), 0), ((1, 4, 16), (9, 48, 1), 16)),
    (((4, 5, 16), (16, 128, 1), 0), ((4, 5, 16), (16, 128, 1), 64)),       # heads first
    (((3, 2, 8), (21, 10, 1), 0), ((3, 2, 2), (21, 10, 1), 8)),            # the last head ends in the next row's gap
    (((2, 3, 1), (5, 2, 1), 0), ((2, 2, 1), (5, 2, 1), 1)),
])
def test_what_lies_between_may_be_written_in_place(q, k):
    from bergen_amd import decoding
    q, k = _views(q, k)
    for t in (q, k):
        decoding._distinct("q", t)
    decoding._apart(q, k)
    decoding._apart(k, q)


def test_overlaps_are_found():
    """All small lattices around each other: refused exactly where they share an element."""
    import itertools
    import random
    from bergen_amd import decoding
    rng, shared, apart = random.Random(0), 0, 0
    for _ in range(4000):
        d, h, t = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 4])
        by_head = d * rng.choice([1, 1, 2, 3]) + rng.choice([0, 0, 1])
        strides = (rng.choice([by_head * h, by_head * h + 1, 2 * by_head * h]), by_head, 1) if rng.random() < 0.8 else (d, d * t * rng.choice([1, 2]), 1)
        other = strides if rng.random() < 0.7 else (strides[0], strides[1] * 2, 1)
        q, k = _views(((t, h, d), strides, 0), ((t, rng.choice([1, h]), d), other, rng.randint(-30, 30)))
        at = [{v.storage_offset() + sum(i * s for i, s in zip(x, v.stride())) for x in itertools.product(*map(range, v.shape))} for v in (q, k)]
        if any(len(a) < v.numel() for a, v in zip(at, (q, k))):
            continue
        if at[0] & at[1]:
            shared += 1
            _refused("q and k overlap", decoding._apart, q, k)
        else:
            apart += 1
            decoding._apart(q, k)
    assert shared > 1000 and apart > 1000


def _cache_args(dtype=torch.int8, pages=2, heads=3, page=16, dim=32):
    c = bergen_amd.kv_cache(pages, heads, page, dim, dtype, device="cpu")
    return dict(k_cache=c.k_cache, v_cache=c.v_cache, k_scale=c.k_scale, v_scale=c.v_scale)


def test_cache_refusals():
    k = torch.zeros(5, 3, 32)
    slots = torch.zeros(5, dtype=torch.int64)
    base = dict(k=k, v=k, slots=slots, **_cache_args())
    for change, match in [(dict(k=torch.zeros(5, 2, 32)), "k has shape"), (dict(v=torch.zeros(4, 3, 32)), "v must have"),
                          (dict(v=k.half()), "v must have"), (dict(slots=slots.int()), "slots"), (dict(slots=slots[:4]), "slots"),
                          (dict(k_scale=None), "needs k_scale"), (dict(v_scale=torch.zeros(2, 3, 16).double()), "needs v_scale"),
                          (dict(v_cache=torch.zeros(2, 3, 16, 32)), "v_cache must have"),
                          (dict(k_cache=torch.zeros(2, 3, 16, 32), v_cache=torch.zeros(2, 3, 16, 32)), "k_cache must be"),
                          (dict(k_cache=base["k_cache"].transpose(0, 1), v_cache=base["v_cache"].transpose(0, 1)), "contiguous"),
                          (dict(), "must be on the GPU")]:
        _refused(match, bergen_amd.kv_cache_write, **{**base, **change})
    same = _cache_args()
    _refused("the same memory", bergen_amd.kv_cache_write, k, k, slots, **dict(same, v_cache=same["k_cache"]))
    half = dict(_cache_args(torch.float16), k_scale=torch.zeros(2, 3, 16))
    _refused("has no scales", bergen_amd.kv_cache_read, slots, **half)
    _refused("dtype must be", bergen_amd.kv_cache_read, slots, **_cache_args(), dtype=torch.int8)
    _refused("must be on the GPU", bergen_amd.kv_cache_read, slots, **_cache_args())
    _refused("a cache holds", bergen_amd.kv_cache, 1, 1, 16, 32, torch.float32, device="cpu")


def test_cache_memory_that_is_shared():
    """Keys and values are written at once: caches, scales, or codes and scales that meet anywhere are refused; those that lie side by side are not."""
    k, slots = torch.zeros(5, 3, 32), torch.zeros(5, dtype=torch.int64)
    a = _cache_args()
    both = torch.zeros(3, 3, 16, 32, dtype=torch.int8)
    scales = torch.zeros(3, 3, 16)
    raw = torch.zeros(4 * 3072, dtype=torch.int8)
    for change, match in [(dict(v_scale=a["k_scale"]), "k_scale and v_scale are the same memory"), (dict(k_cache=both[:2], v_cache=both[1:]), "share some"),
                          (dict(k_cache=both[1:], v_cache=both[:2]), "share some"), (dict(k_scale=scales[:2], v_scale=scales[1:]), "share some"),
                          (dict(k_cache=raw[:3072].view(2, 3, 16, 32), k_scale=raw[3008:3392].view(torch.float32).view(2, 3, 16)), "codes and its scales"),
                          (dict(v_cache=raw[3072:6144].view(2, 3, 16, 32), k_scale=raw[2816:3200].view(torch.float32).view(2, 3, 16)), "codes and its scales"),
                          (dict(k_cache=raw[:3072].view(2, 3, 16, 32), v_cache=raw[3072:6144].view(2, 3, 16, 32), k_scale=raw[6144:6528].view(torch.float32).view(2, 3, 16),
                                v_scale=raw[6528:6912].view(torch.float32).view(2, 3, 16)), "must be on the GPU")]:
        _refused(match, bergen_amd.kv_cache_write, k, k, slots, **{**a, **change})
    half = torch.zeros(3, 3, 16, 32, dtype=torch.float16)
    _refused("share some", bergen_amd.kv_cache_write, k, k, slots, half[:2], half[1:])
    two = torch.zeros(4, 3, 16, 32, dtype=torch.float16)
    _refused("must be on the GPU", bergen_amd.kv_cache_write, k, k, slots, two[:2], two[2:])


def test_attention_refusals():
    base = dict(q=torch.zeros(2, 6, 32, dtype=torch.bfloat16), block_table=torch.zeros(2, 4, dtype=torch.int32),
                lengths=torch.zeros(2, dtype=torch.int32), **_cache_args())
    for change, match in [(dict(q=torch.zeros(2, 6, 32)), "q must be float16 or bfloat16"), (dict(q=torch.zeros(2, 6, 48, dtype=torch.bfloat16)), "q has shape"),
                          (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), "block_table"), (dict(block_table=torch.zeros(2, 4).long()), "block_table"),
                          (dict(lengths=torch.zeros(2)), "lengths"), (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
                          (dict(window=-1), "window"), (dict(window=1 << 32), "window"), (dict(alibi_slopes=torch.zeros(3)), "alibi_slopes"), (_cache_args(torch.float16), "the cache must be"),
                          (dict(), "must be on the GPU")]:
        _refused(match, bergen_amd.paged_attention, **{**base, **change})


def test_logprobs_refusals():
    x, t = torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64)
    for a, match in [((x.double(), t), "logits must be"), ((x[0], t), "logits must be"), ((x[:, :0], t), "not empty"), ((x.t(), t), "dense"),
                     ((x, t.int()), "targets"), ((x, t[:1]), "targets"), ((x, t, 10), "top 10 of 9"),
                     ((x, t, -1), "top -1"), ((x, t, 1 << 32), "top"), ((x, t), "must be on the GPU")]:
        _refused(match, bergen_amd.token_logprobs, *a)


def test_refused_by_the_c_entry_points():
    """Sizes, types, null buffers and short workspaces are refused before any device is looked for, each with its message."""
    lib, E, U = _lib.lib(), _lib.BH_EINVAL, _lib.BH_EUNSUPPORTED
    H, B, F, I8, E4 = _lib.BH_F16, _lib.BH_BF16, _lib.BH_F32, _lib.BH_I8, _lib.BH_E4M3

    def rotary(dtype=B, tokens=2, nq=2, nk=1, dim=64, rot=64, pos=P, inv=P, qw=None, wt=B, eps=1e-6, q=P):
        return lib.bh_op_qk_norm_rotary(q, 128, 64, P, 128, 64, P, 64, 64, P, 64, 64, dtype, tokens, nq, nk, dim, rot, pos, 1, inv, qw, None, wt, eps, 0, None)

    for code, k in [(E, dict(dtype=I8)), (E, dict(dtype=9)), (E, dict(qw=P, wt=H)), (E, dict(tokens=-1)), (E, dict(nq=0)), (E, dict(eps=-1.0)),
                    (E, dict(eps=math.nan)), (U, dict(dim=257)), (U, dict(dim=0)), (E, dict(rot=66)), (E, dict(rot=63)), (E, dict(rot=-2)),
                    (U, dict(tokens=1 << 31)), (U, dict(tokens=1 << 30)), (U, dict(tokens=1 << 24, dim=63, rot=62)), (E, dict(q=None)), (E, dict(pos=None)), (E, dict(inv=None))]:
        assert rotary(**k) == code, k
        assert lib.bh_last_error(), k
    assert rotary(tokens=0) == _lib.BH_OK

    def write(dtype=B, cache=I8, tokens=2, heads=2, dim=64, pages=4, page=16, k=P, slots=P, scale=P, fn=lib.bh_op_kv_write):
        return fn(k, 128, 64, P, 128, 64, dtype, slots, tokens, heads, dim, P, P, scale, scale, cache, pages, page, None)

    for fn in (lib.bh_op_kv_write, lib.bh_op_kv_read):
        for code, k in [(E, dict(dtype=I8)), (E, dict(cache=F)), (E, dict(cache=7)), (E, dict(tokens=-1)), (E, dict(heads=0)), (E, dict(pages=0)),
                        (U, dict(dim=257)), (U, dict(page=4)), (U, dict(page=24)), (U, dict(page=2048)), (E, dict(k=None)), (E, dict(slots=None)),
                        (E, dict(scale=None)), (U, dict(tokens=1 << 40)), (U, dict(tokens=1 << 30)), (U, dict(tokens=1 << 28, dim=63))]:
            assert write(fn=fn, **k) == code, k
        assert write(fn=fn, tokens=0) == _lib.BH_OK

    def attend(dtype=B, cache=B, batch=2, hq=8, hk=2, dim=64, page=16, width=4, q=P, kc=P, scale=None, s=0.125, cap=0.0, window=0, ws=P, n=1 << 40, pages=9,
               q_seq=512):
        return lib.bh_op_paged_attention(q, q_seq, 64, dtype, kc, P, scale, scale, cache, pages, page, P, width, width, P, batch, hq, hk, dim, s, cap,
                                         window, None, P, None, ws, n, None)

    for code, k in [(E, dict(dtype=F)), (E, dict(cache=H)), (E, dict(cache=F)), (E, dict(batch=-1)), (E, dict(hq=7)), (E, dict(hk=0)), (U, dict(dim=72)),
                    (U, dict(dim=272)), (U, dict(page=4)), (U, dict(page=48)), (E, dict(width=-1)), (U, dict(batch=65536)), (U, dict(width=1 << 30)),
                    (E, dict(s=math.nan)), (E, dict(cap=-1.0)), (E, dict(cap=math.inf)), (E, dict(cap=math.nan)), (E, dict(window=-1)), (E, dict(q=None)),
                    (E, dict(kc=None)), (E, dict(cache=E4)), (E, dict(pages=-1)), (U, dict(cache=I8, scale=ctypes.c_void_p(4100))), (U, dict(q=ctypes.c_void_p(4098))), (U, dict(q_seq=511)),
                    (E, dict(width=4096, n=1024)), (E, dict(width=4096, ws=None)), (E, dict(width=4096, ws=ctypes.c_void_p(4104)))]:
        assert attend(**k) == code, k
        assert lib.bh_last_error(), k
    assert attend(batch=0) == _lib.BH_OK
    size = lib.bh_op_paged_attention_workspace
    assert size(2, 8, 2, 64, 16, 4096, 0) > 0 and size(0, 8, 2, 64, 16, 4096, 0) == 0
    assert size(2, 7, 2, 64, 16, 4, 0) == E and size(2, 8, 2, 60, 16, 4, 0) == U and size(2, 8, 2, 64, 16, 4, -1) == E

    def logp(dtype=F, rows=2, vocab=100, given=1, top=5, x=P, t=P, ids=P, ws=P, n=1 << 40, stride=100):
        return lib.bh_op_token_logprobs(x, stride, dtype, rows, vocab, t, given, top, P, P, P, ids, ws, n, None)

    for code, k in [(E, dict(dtype=I8)), (E, dict(rows=-1)), (E, dict(vocab=0)), (E, dict(top=101)), (E, dict(top=-1)), (U, dict(top=65)), (E, dict(given=-1)),
                    (E, dict(stride=99)), (E, dict(x=None)), (E, dict(t=None)), (E, dict(ids=None)), (U, dict(vocab=(1 << 30) + 1, stride=1 << 31)),
                    (U, dict(rows=(1 << 24) + 1)), (E, dict(x=ctypes.c_void_p(4098))), (E, dict(vocab=100000, stride=100000, n=8)),
                    (E, dict(vocab=100000, stride=100000, ws=None)), (U, dict(rows=1 << 24))]:
        assert logp(**k) == code, k
    assert logp(rows=0) == _lib.BH_OK
    assert lib.bh_op_token_logprobs_workspace(1, 100000, F, 5) > 0 and lib.bh_op_token_logprobs_workspace(100000, 1000, F, 5) == 0
    assert lib.bh_op_token_logprobs_workspace(1, 100, F, 101) == E


def test_registers_as_the_makefile_builds():
    """The decoding operators' kernels with their own flags: nothing in scratch, and 8-bit attention of heads up to 128 in 3 waves a SIMD (of 64: 4)."""
    import os
    import re
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bergen_amd", "csrc")
    jobs = []
    for src in ("decode_ops", "paged_attention", "token_logprobs"):
        line = [w for w in subprocess.run(["make", "-n", "-W", f"{src}.hip", f"../lib/obj/{src}.o"], cwd=csrc, capture_output=True, text=True, check=True).stdout.splitlines()
                if f"-c {src}.hip" in w][0].split()
        assert "-packed-fp32-ops" in line
        jobs.append(subprocess.Popen(line[: line.index("-o")] + ["-o", os.devnull, "-Rpass-analysis=kernel-resource-usage"], cwd=csrc, stderr=subprocess.PIPE, text=True))
    seen = 0
    for job in jobs:
        text = job.communicate()[1]
        assert job.returncode == 0, text[-2000:]
        for block in text.split("Function Name: ")[1:]:
            name = block.split()[0]
            value = {k.strip(): int(v) for k, v in re.findall(r"remark:\s+([A-Za-z ]+?)(?: \[[^\]]*\])?: (\d+)", block)}
            seen += 1
            assert value["ScratchSize"] == 0 and value["VGPRs Spill"] == 0, (name, value)
            form = re.search(r"bh_paged_attention_kernelIDF16.Li([34])ELi(64|128)E", name)
            if form:
                assert value["Occupancy"] >= {"64": 4, "128": 3}[form.group(2)], (name, value)
    assert seen > 60


def test_older_entry_points_still_refuse_the_new_types():
    lib = _lib.lib()
    h = ctypes.c_void_p()
    for t in (_lib.BH_BF16, _lib.BH_I8, _lib.BH_E4M3):
        assert lib.bh_index_create(ctypes.byref(h), 10, 64, t, 0) in (_lib.BH_EINVAL, _lib.BH_EUNSUPPORTED)


def test_a_gradient_is_refused_while_it_is_recorded():
    from bergen_amd import decoding
    leaf = torch.zeros(2, requires_grad=True)
    with pytest.raises(ValueError, match="k requires a gradient"):
        decoding._one_device("q k", torch.zeros(2), leaf)
    with torch.no_grad(), pytest.raises(ValueError, match="must be on the GPU"):
        decoding._one_device("q k", torch.zeros(2), leaf)


def test_a_tangent_is_refused():
    """Forward-mode differentiation: requires_grad is False, and the tangent would be lost; under no_grad() it lives on, in inference mode it does not."""
    import torch.autograd.forward_ad as fwd
    a = _rotary_args()
    x, t = torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64)
    with fwd.dual_level():
        for name in ("q", "k"):
            dual = {**a, name: fwd.make_dual(a[name], torch.ones_like(a[name]))}
            assert not dual[name].requires_grad
            for inplace in (False, True):
                _refused(f"{name} carries a tangent", bergen_amd.qk_norm_rotary, **dual, inplace=inplace)
            with torch.no_grad():
                _refused(f"{name} carries a tangent", bergen_amd.qk_norm_rotary, **dual)
            with torch.inference_mode():
                _refused("must be on the GPU", bergen_amd.qk_norm_rotary, **dual)
        w = fwd.make_dual(torch.ones(64), torch.ones(64))
        _refused("k_weight carries a tangent", bergen_amd.qk_norm_rotary, **a, k_weight=w)
        _refused("logits carries a tangent", bergen_amd.token_logprobs, fwd.make_dual(x, x), t)
        c = _cache_args()
        k, slots = torch.zeros(5, 3, 32), torch.zeros(5, dtype=torch.int64)
        _refused("v carries a tangent", bergen_amd.kv_cache_write, k, fwd.make_dual(k.clone(), k), slots, **c)
        _refused("v_scale carries a tangent", bergen_amd.kv_cache_read, slots, **{**c, "v_scale": fwd.make_dual(c["v_scale"], c["v_scale"].clone())})
        _refused("must be on the GPU", bergen_amd.token_logprobs, x, t)


@pytest.mark.filterwarnings("ignore")
def test_a_trace_is_refused():
    a, c = _rotary_args(), _cache_args()
    k, slots = torch.zeros(5, 3, 32), torch.zeros(5, dtype=torch.int64)
    q, table, n = torch.zeros(2, 6, 32, dtype=torch.bfloat16), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    calls = [(lambda x: bergen_amd.qk_norm_rotary(**{**a, "q": x}), a["q"]), (lambda x: bergen_amd.token_logprobs(x, slots[:2]).logprobs, torch.zeros(2, 9)),
             (lambda x: bergen_amd.kv_cache_write(x, k, slots, **c), k), (lambda x: bergen_amd.kv_cache_read(x, **c), slots),
             (lambda x: bergen_amd.paged_attention(x, c["k_cache"], c["v_cache"], table, n, k_scale=c["k_scale"], v_scale=c["v_scale"]), q)]
    for call, x in calls:
        _refused("cannot be traced", torch.jit.trace, call, x)
        _refused("must be on the GPU", call, x)


def test_rotary_frequencies():
    f = bergen_amd.rotary_frequencies(8, 100.0, 0.5, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, 0.5 * torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert bergen_amd.rotary_frequencies(0, device="cpu").numel() == 0
    _refused("even", bergen_amd.rotary_frequencies, 7, device="cpu")


def test_the_reference_against_torch():
    """The 64-bit formulas agree with torch's own functions where torch has one."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 301, generator=g)
    r = ref.logprobs(x, torch.arange(5), 7)
    lp = torch.log_softmax(x.double(), -1)
    assert torch.allclose(r["logprobs"][0], lp[torch.arange(5), torch.arange(5)], atol=1e-12)
    assert torch.allclose(r["entropy"][0], torch.distributions.Categorical(logits=x.double()).entropy(), atol=1e-12)
    assert torch.equal(r["top_ids"], x.topk(7).indices)
    y = torch.randn(1000, generator=g) * 200
    codes, scale = ref.quantise(y[None], torch.float8_e4m3fn)
    assert torch.equal(codes[0], (y / scale).to(torch.float8_e4m3fn).double()) and 224 < float(y.abs().max() / scale) <= 448
    codes, scale = ref.quantise(y[None], torch.int8)
    assert float(codes.abs().max()) == 127
    c = bergen_amd.kv_cache(3, 2, 8, 16, torch.float16, device="cpu")
    c.k_cache.normal_(generator=g), c.v_cache.normal_(generator=g)
    q = torch.randn(1, 4, 16, generator=g).half()
    out, _, lse, _ = ref.attention(q, c.k_cache, c.v_cache, torch.tensor([[2, 0]], dtype=torch.int32), torch.tensor([13]))
    k, v = (torch.cat([z[2], z[0]], 1)[:, :13].double().repeat_interleave(2, 0) for z in (c.k_cache, c.v_cache))
    want = torch.nn.functional.scaled_dot_product_attention(q[0].double()[:, None], k, v)[:, 0]
    assert torch.allclose(out[0], want, atol=1e-12)
