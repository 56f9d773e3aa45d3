"""
Operators of a decoding step on hand-written HIP kernels: what a decoder that answers from the retrieved passages, or scores them by
the log probability of a token, runs next to its matrix products (the reference reaches such models through
AutoModelForCausalLM, models/generators/llm.py).

  rotary_frequencies   the rotary positions' inverse frequencies, in 64 bits (made once)
  qk_norm_rotary       RMS norm of each query / key head and rotary positions, in one pass
  kv_cache             an empty paged key-value cache: fp16, bf16, int8 or e4m3
  kv_cache_write       keys and values into their slots, quantised on the way
  kv_cache_read        slots back as vectors
  paged_attention      attention of one new token per sequence over that cache
  token_logprobs       log probabilities of given tokens, entropy, likeliest alternatives

They take device tensors, ENQUEUE on the current stream of the tensors' device and return (the other entry points of this package wait); they can
be captured into a graph, but not traced (torch.jit.trace).  They run inference only: a tensor that requires a gradient is refused while gradients are recorded,
and one that carries a tangent (forward-mode differentiation).
"""
import collections

import torch
from torch.autograd import forward_ad

from . import _lib

_FLOATS = {torch.float16: _lib.BH_F16, torch.bfloat16: _lib.BH_BF16, torch.float32: _lib.BH_F32}
_CACHES = {torch.float16: _lib.BH_F16, torch.bfloat16: _lib.BH_BF16, torch.int8: _lib.BH_I8, torch.float8_e4m3fn: _lib.BH_E4M3}
_SCALED = (torch.int8, torch.float8_e4m3fn)

TokenLogprobs = collections.namedtuple("TokenLogprobs", "logprobs entropy top_logprobs top_ids")

_ready = set()

# the current stream's handle: current_stream() builds an object around it, which takes longer than the launch it is wanted for
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
# (likewise: the index without the question whether CUDA is initialised, which a tensor on the GPU has answered)
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_tracing = torch._C._get_tracing_state


def _fail(message):
    raise ValueError(message)


def _one_device(names, *tensors):
    """Every tensor (None: not given) on one GPU, and none that waits for a gradient or carries a tangent; -> that GPU's index.  names: theirs, for a refusal."""
    index = tensors[0].get_device()
    grad = torch.is_grad_enabled()
    if _tracing() is not None:
        _fail("torch.jit.trace would record the outputs' memory and none of the work: these operators cannot be traced")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():  # (inside forward_ad.dual_level(); under no_grad() too)
        for name, t in zip(names.split(), tensors):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _fail(f"{name} carries a tangent and there is no derivative here")
    for t in tensors:
        if t is not None and (t.get_device() != index or (grad and t.requires_grad)):
            for name, t in zip(names.split(), tensors):
                if t is not None and t.get_device() != index:
                    _fail(f"{name} is on {t.device}, expected {tensors[0].device}")
                if t is not None and grad and t.requires_grad:
                    _fail(f"{name} requires a gradient and there is no backward pass here: call under torch.no_grad()")
    if index < 0:
        _fail(f"tensors must be on the GPU, got them on {tensors[0].device}")
    if index not in _ready:
        with torch.cuda.device(index):
            _lib.init(index)  # once per device: is it a gfx950 part
        _ready.add(index)
    return index


def _call(index, fn, *args):
    """fn(*args, stream) with GPU `index` as the current device, on its current stream."""
    if _current() == index:
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc:
        _lib.check(rc)


def _empty_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(name, t):
    """[tokens, heads, dim] with the last dimension dense -> its sizes, the strides of the first two, its address."""
    if t.dim() != 3:
        _fail(f"{name} must be [tokens, heads, dim], got {tuple(t.shape)}")
    if t.dtype not in _FLOATS:
        _fail(f"{name} must be float16, bfloat16 or float32, got {t.dtype}")
    tokens, heads, dim = t.shape
    by_token, by_head, dense = t.stride()
    if dense != 1 and dim > 1:
        _fail(f"{name}'s last dimension must be dense")
    return tokens, heads, dim, by_token, by_head, t.data_ptr()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _distinct(name, t):
    """An output whose elements share no memory (an expanded view would)."""
    room = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda p: p[1]):
        if size > 1:
            if not (stride >= room):
                _fail(f"{name} overlaps itself (shape {tuple(t.shape)}, strides {t.stride()}): it cannot be written")
            room += stride * (size - 1)


def _meet(at, a, b):
    """Whether two lattices share an element: a and b, [(size, stride)] with the longest stride first, none overlapping itself, b's first element `at`
    elements behind a's.  The rows of one that reach the other are looked at in turn, those of both by their difference where they are equally far apart."""
    if not a and not b:
        return at == 0
    (n, step_a), (m, step_b) = (a or [(1, 0)])[0], (b or [(1, 0)])[0]
    step = max(step_a, step_b)
    rest_a, rest_b = a[1:] if step_a == step else a, b[1:] if step_b == step else b
    reach_a, reach_b = (sum((size - 1) * by for size, by in x) for x in (rest_a, rest_b))
    first, last = 1 - n if step_a == step else 0, m - 1 if step_b == step else 0  # b's row less a's
    near = range(max(first, -((at + reach_b) // step)), min(last, (reach_a - at) // step) + 1)
    return len(near) > 1000 or any(_meet(at + j * step, rest_a, rest_b) for j in near)


def _apart(q, k):
    """q's and k's memory does not meet: separate ranges, separate columns of rows that are equally far apart, or heads between each other's."""
    if 0 in q.shape or 0 in k.shape:
        return
    ends = [sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1 for t in (q, k)]
    at, off = divmod(k.data_ptr() - q.data_ptr(), q.element_size())
    if at >= ends[0] or -at >= ends[1] + (off > 0):
        return
    row = q.stride(0)
    if q.shape[0] > 1 and k.stride(0) == row and not off:
        cols = [e - (t.shape[0] - 1) * row for e, t in zip(ends, (q, k))]
        if at % row >= cols[0] and at % row + cols[1] <= row:
            return
    dims = [sorted(((n, st) for n, st in zip(t.shape, t.stride()) if n > 1), key=lambda p: -p[1]) for t in (q, k)]
    if off or _meet(at, *dims):
        _fail("q and k overlap: they cannot be written in place")


def rotary_frequencies(rotary_dim, theta=10000.0, scale=1.0, device="cuda"):
    """inv_freq[j] = scale * theta^(-2 j / rotary_dim), j < rotary_dim / 2, float64: what `qk_norm_rotary` turns a pair by, per position."""
    if not (rotary_dim >= 0 and rotary_dim % 2 == 0):
        _fail(f"rotary_dim must be even, got {rotary_dim}")
    j = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    return float(scale) * float(theta) ** (-j / max(1, rotary_dim))


def _weight(name, w, dim, dtype):
    if w.dim() != 1 or w.shape[0] != dim or not (w.dtype == dtype or w.dtype == torch.float32) or not w.is_contiguous():
        _fail(f"{name} must be contiguous [{dim}], {dtype} or float32")
    return w.dtype


def qk_norm_rotary(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, inplace=False):
    """RMS norm of each head of q [tokens, n_q, dim] and k [tokens, n_k, dim], then rotary positions, in one pass -> (q, k).

    positions [tokens] int32 / int64; inv_freq [rotary_dim / 2] float64 (`rotary_frequencies`): the pair (j, j + rotary_dim / 2) — or (2 j, 2 j + 1)
    with interleaved — is turned by positions * inv_freq[j]; elements behind rotary_dim stay.  q_weight, k_weight [dim], of q's type
    or float32; None: that side is not normalised.  q and k are float16, bfloat16 or float32, any strides with a dense last
    dimension (slices of one projection).  inplace: into q and k themselves.
    """
    tokens, nq, dim, q0, q1, qp = _rows("q", q)
    tokens_k, nk, dim_k, k0, k1, kp = _rows("k", k)
    dtype = q.dtype
    if k.dtype != dtype or tokens_k != tokens or dim_k != dim:
        _fail(f"k must be [{tokens}, heads, {dim}] {dtype}, got {tuple(k.shape)} {k.dtype}")
    wide = positions.dtype == torch.int64
    if not (wide or positions.dtype == torch.int32) or positions.dim() != 1 or positions.shape[0] != tokens:
        _fail(f"positions must be int32 or int64 [{tokens}]")
    rotary = 2 * inv_freq.numel()
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or rotary > dim:
        _fail(f"inv_freq must be float64 [rotary_dim / 2], rotary_dim at most {dim}")
    if not (positions.is_contiguous() and inv_freq.is_contiguous()):
        _fail("positions and inv_freq must be contiguous")
    wtype = _weight("q_weight", q_weight, dim, dtype) if q_weight is not None else None
    if k_weight is not None:
        was, wtype = wtype, _weight("k_weight", k_weight, dim, dtype)
        if was not in (None, wtype):
            _fail("q_weight and k_weight must have one type")
    if inplace:
        _distinct("q", q)
        _distinct("k", k)
        _apart(q, k)
    device = _one_device("q k positions inv_freq q_weight k_weight", q, k, positions, inv_freq, q_weight, k_weight)
    if inplace:
        qo, ko, qo0, qo1, ko0, ko1 = q, k, q0, q1, k0, k1
    else:
        qo, ko, qo0, qo1, ko0, ko1 = _empty_like(q), _empty_like(k), nq * dim, dim, nk * dim, dim
    _call(device, _lib.lib().bh_op_qk_norm_rotary, qp, q0, q1, qo.data_ptr(), qo0, qo1, kp, k0, k1, ko.data_ptr(), ko0, ko1, _FLOATS[dtype], tokens,
          nq, nk, dim, rotary, positions.data_ptr(), wide, inv_freq.data_ptr(), _ptr(q_weight), _ptr(k_weight), _FLOATS[wtype or dtype],
          float(eps), bool(interleaved))
    if inplace:
        torch.autograd.graph.increment_version((q, k))
    return qo, ko


KVCache = collections.namedtuple("KVCache", "k_cache v_cache k_scale v_scale")


def kv_cache(pages, heads, page_size, dim, dtype=torch.bfloat16, device="cuda"):
    """An empty paged cache -> KVCache(k_cache, v_cache [pages, heads, page_size, dim], k_scale, v_scale [pages, heads, page_size] or None).

    The operators take page sizes that are a power of two, 8 .. 1024, and dim up to 256 (`paged_attention`: multiples of 16).
    """
    if not (dtype in _CACHES):
        _fail(f"a cache holds float16, bfloat16, int8 or float8_e4m3fn, got {dtype}")
    shape = (pages, heads, page_size, dim)
    made = [torch.zeros(shape, dtype=torch.int8 if dtype in _SCALED else dtype, device=device).view(dtype) for _ in range(2)]
    scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) if dtype in _SCALED else None for _ in range(2)]
    return KVCache(*made, *scales)


def _cache_tensors(k_cache, v_cache, k_scale, v_scale):
    """-> the cache's sizes and whether it is scaled."""
    kind, shape = k_cache.dtype, k_cache.shape
    if k_cache.dim() != 4 or kind not in _CACHES:
        _fail(f"k_cache must be [pages, heads, page_size, dim], float16, bfloat16, int8 or float8_e4m3fn; got {tuple(shape)} {kind}")
    if v_cache.shape != shape or v_cache.dtype != kind:
        _fail("v_cache must have k_cache's shape and type")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        _fail("k_cache and v_cache must be contiguous")
    scaled = kind in _SCALED
    if scaled:
        scales = shape[:3]
        for s in (k_scale, v_scale):
            if s is None or s.shape != scales or s.dtype != torch.float32 or not s.is_contiguous():
                _fail(f"an 8-bit cache needs {'k_scale' if s is k_scale else 'v_scale'}: contiguous float32 {tuple(scales)}")
    elif k_scale is not None or v_scale is not None:
        _fail(f"a cache of {kind} has no scales")
    return shape, scaled


def kv_cache_write(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    """Rows k, v [tokens, heads, dim] (float16, bfloat16 or float32) into their slots (int64 [tokens]; page * page_size + offset) of the cache.

    A slot outside the cache, -1 for padding, is skipped; the slots of one call must differ, and k and v must not be vectors of the cache that it
    writes.  8-bit caches: int8 with scale = amax / 127 and the
    exact quotient rounded to nearest even; float8_e4m3fn with the least power of two that keeps amax within 448.  A vector that holds an
    infinity or a NaN reads back as NaN.
    """
    (pages, heads, page, dim), scaled = _cache_tensors(k_cache, v_cache, k_scale, v_scale)
    tokens, heads_k, dim_k, k0, k1, kp = _rows("k", k)
    *same, v0, v1, vp = _rows("v", v)
    if heads_k != heads or dim_k != dim:
        _fail(f"k has shape {tuple(k.shape)}, the cache {heads} heads of {dim}")
    if same != [tokens, heads, dim] or v.dtype != k.dtype:
        _fail("v must have k's shape and type")
    if slots.dtype != torch.int64 or slots.dim() != 1 or slots.shape[0] != tokens or not slots.is_contiguous():
        _fail(f"slots must be contiguous int64 [{tokens}]")
    kc, vc = k_cache.data_ptr(), v_cache.data_ptr()
    vectors = pages * heads * page
    size = vectors * dim * (1 if scaled else 2)
    if kc < vc + size and vc < kc + size:
        _fail("k_cache and v_cache are the same memory, or share some")
    ks = vs = None
    if scaled:
        ks, vs, size_s = k_scale.data_ptr(), v_scale.data_ptr(), 4 * vectors
        if ks < vs + size_s and vs < ks + size_s:
            _fail("k_scale and v_scale are the same memory, or share some")
        if kc - size_s < ks < kc + size or kc - size_s < vs < kc + size or vc - size_s < ks < vc + size or vc - size_s < vs < vc + size:
            _fail("the cache's codes and its scales share memory")
    device = _one_device("k v slots k_cache v_cache k_scale v_scale", k, v, slots, k_cache, v_cache, k_scale, v_scale)
    if not pages:
        pages, tokens = 1, 0  # every slot is outside it: the sizes are checked, nothing is written
    _call(device, _lib.lib().bh_op_kv_write, kp, k0, k1, vp, v0, v1, _FLOATS[k.dtype], slots.data_ptr(), tokens, heads, dim, kc, vc, ks, vs,
          _CACHES[k_cache.dtype], pages, page)
    torch.autograd.graph.increment_version((k_cache, v_cache, k_scale, v_scale) if scaled else (k_cache, v_cache))


def kv_cache_read(slots, k_cache, v_cache, k_scale=None, v_scale=None, dtype=torch.bfloat16):
    """The slots' keys and values (int64 [tokens]) as `dtype` -> (k, v) [tokens, heads, dim]; zeros for a slot outside the cache."""
    (pages, heads, page, dim), _ = _cache_tensors(k_cache, v_cache, k_scale, v_scale)
    if dtype not in _FLOATS:
        _fail(f"dtype must be float16, bfloat16 or float32, got {dtype}")
    if slots.dim() != 1 or slots.dtype != torch.int64 or not slots.is_contiguous():
        _fail("slots must be contiguous int64 [tokens]")
    device = _one_device("slots k_cache v_cache k_scale v_scale", slots, k_cache, v_cache, k_scale, v_scale)
    tokens = slots.shape[0]
    k = slots.new_empty((tokens, heads, dim), dtype=dtype)
    v = torch.empty_like(k)
    if not pages:
        pages, tokens = 1, 0
        k.zero_(), v.zero_()
    _call(device, _lib.lib().bh_op_kv_read, k.data_ptr(), heads * dim, dim, v.data_ptr(), heads * dim, dim, _FLOATS[dtype], slots.data_ptr(), tokens,
          heads, dim, k_cache.data_ptr(), v_cache.data_ptr(), _ptr(k_scale), _ptr(v_scale), _CACHES[k_cache.dtype], pages, page)
    return k, v


def paged_attention(q, k_cache, v_cache, block_table, lengths, scale=None, k_scale=None, v_scale=None, softcap=0.0, window=0,
                    alibi_slopes=None, return_lse=False):
    """Attention of one new token per sequence over a paged cache: q [batch, n_q, dim] -> out, or (out, lse) with return_lse.

    q is float16 or bfloat16, dim a multiple of 16 up to 256; the cache (`kv_cache`) q's type, int8 or float8_e4m3fn with its scales;
    n_q a multiple of the cache's heads.  lengths [batch] int32: tokens of each sequence in the cache, its newest among them;
    block_table [batch, width] int32: their pages in order.  A length is taken as 0 .. width * page_size, and the tokens of an entry
    outside the cache's pages are left out.  scale: 1 / sqrt(dim) unless given.  softcap c > 0: scores c tanh(s / c).  alibi_slopes [n_q]
    float32: minus slope times the distance.  window w > 0: the last w tokens only.  lse [batch, n_q] float32: log of the sum of e^score.
    A sequence with nothing left gives zeros and -inf.  Scores, their sums and the outputs' are in 32 bits; weights are kept to 2^-17 of themselves (bf16 cache) or 2^-22 (fp16,
    8-bit), where weights below 2^-39 of a head's largest are left out.
    """
    (pages, heads, page, dim), scaled = _cache_tensors(k_cache, v_cache, k_scale, v_scale)
    batch, nq, dim_q, q0, q1, qp = _rows("q", q)
    dtype = q.dtype
    if dim_q != dim:
        _fail(f"q has shape {tuple(q.shape)}, the cache heads of {dim}")
    if dtype == torch.float32:
        _fail(f"q must be float16 or bfloat16, got {dtype}")
    if not scaled and k_cache.dtype != dtype:
        _fail(f"the cache must be {dtype}, int8 or float8_e4m3fn, got {k_cache.dtype}")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != batch:
        _fail(f"block_table must be int32 [{batch}, width]")
    width, (t0, dense) = block_table.shape[1], block_table.stride()
    if dense != 1 and width > 1:
        _fail("block_table's rows must be dense")
    if not pages:
        width = 0  # no entry names a page of it
    if lengths.dtype != torch.int32 or lengths.dim() != 1 or lengths.shape[0] != batch or not lengths.is_contiguous():
        _fail(f"lengths must be contiguous int32 [{batch}]")
    if alibi_slopes is not None and (alibi_slopes.dim() != 1 or alibi_slopes.shape[0] != nq or alibi_slopes.dtype != torch.float32
                                     or not alibi_slopes.is_contiguous()):
        _fail(f"alibi_slopes must be contiguous float32 [{nq}]")
    if not 0 <= window < 1 << 31:
        _fail(f"window must be 0 or a count of tokens, got {window}")
    device = _one_device("q k_cache v_cache block_table lengths k_scale v_scale alibi_slopes", q, k_cache, v_cache, block_table, lengths, k_scale,
                         v_scale, alibi_slopes)
    if qp % 16 or q0 % 8 or q1 % 8:
        q = q.clone(memory_format=torch.contiguous_format)  # (contiguous() would hand back a dense one that starts off a border)
        q0, q1, qp = nq * dim, dim, q.data_ptr()
    lib = _lib.lib()
    need = lib.bh_op_paged_attention_workspace(batch, nq, heads, dim, page, width, int(window))
    if need < 0:
        _lib.check(need)
    out = _empty_like(q)
    lse = q.new_empty((batch, nq), dtype=torch.float32) if return_lse else None
    # (made anew for each call: two calls at once, or two captured graphs, must not share one)
    work = lengths.new_empty(need, dtype=torch.uint8) if need else None
    _call(device, lib.bh_op_paged_attention, qp, q0, q1, _FLOATS[dtype], k_cache.data_ptr(), v_cache.data_ptr(), _ptr(k_scale), _ptr(v_scale),
          _CACHES[k_cache.dtype], pages, page, block_table.data_ptr(), t0, width, lengths.data_ptr(), batch, nq, heads, dim,
          float(dim ** -0.5 if scale is None else scale), float(softcap), int(window), _ptr(alibi_slopes), out.data_ptr(), _ptr(lse), _ptr(work), need)
    return (out, lse) if return_lse else out


def token_logprobs(logits, targets, top=0):
    """Log probabilities of given tokens, entropy and the `top` likeliest tokens of each row, in one pass over logits [rows, vocab].

    logits: float16, bfloat16 or float32 with dense rows; targets: int64 [rows] or [rows, given].  -> TokenLogprobs(logprobs float32 of targets'
    shape, entropy float32 [rows] in nats, top_logprobs float32 and top_ids int64 [rows, top] in the order logit descending, id ascending).
    A negative target's log probability is 0 (padding), one beyond the vocabulary NaN.  -inf logits carry no probability; a row of nothing
    else has log probabilities -inf and entropy 0; a row with a NaN or +inf has NaN.  top is at most 64.
    """
    if logits.dim() != 2 or logits.dtype not in _FLOATS:
        _fail(f"logits must be [rows, vocab], float16, bfloat16 or float32; got {tuple(logits.shape)} {logits.dtype}")
    (rows, vocab), (by_row, dense) = logits.shape, logits.stride()
    if vocab < 1 or (dense != 1 and vocab > 1):
        _fail("logits' rows must be dense and not empty")
    given = targets.dim()
    if targets.dtype != torch.int64 or not 1 <= given <= 2 or targets.shape[0] != rows or not targets.is_contiguous():
        _fail(f"targets must be contiguous int64 [{rows}] or [{rows}, given]")
    given = 1 if given == 1 else targets.shape[1]
    if not 0 <= top <= vocab:
        _fail(f"top {top} of {vocab} tokens")
    device = _one_device("logits targets", logits, targets)
    if rows > 1 and by_row < vocab:
        logits, by_row = logits.contiguous(), vocab
    lib, code, top = _lib.lib(), _FLOATS[logits.dtype], int(top)
    need = lib.bh_op_token_logprobs_workspace(rows, vocab, code, top)
    if need < 0:
        _lib.check(need)
    logprobs = logits.new_empty(targets.shape, dtype=torch.float32)
    entropy = logits.new_empty((rows,), dtype=torch.float32)
    top_logprobs = logits.new_empty((rows, top), dtype=torch.float32)
    top_ids = targets.new_empty((rows, top))
    work = targets.new_empty(need, dtype=torch.uint8) if need else None
    _call(device, lib.bh_op_token_logprobs, logits.data_ptr(), by_row, code, rows, vocab, targets.data_ptr(), given, top, logprobs.data_ptr(),
          entropy.data_ptr(), top_logprobs.data_ptr(), top_ids.data_ptr(), _ptr(work), need)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)
