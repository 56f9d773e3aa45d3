// token_logprobs.hip — log probabilities of given tokens, entropy and the likeliest alternatives of each row of logits, in one pass.
//
//   lse = m + log sum_i e^(x_i - m),   logprob = x_target - lse,   H = log sum_i e^(x_i - m) - (sum_i (x_i - m) e^(x_i - m)) / (sum_i e^(x_i - m))
//
// A wave keeps ONE running maximum m for its 64 lanes (it changes a handful of times over a row; a maximum per lane would change in
// some lane at nearly every step) and per lane the sums of e^(x - m) and (x - m) e^(x - m) in fp32.  The sum leaves out the
// maximum's own 1: log1p of the rest keeps the entropy of a row that is nearly certain.
// Top alternatives: the wave's 64 best (value, index) keys live sorted across its lanes; a block of 8 elements per lane is looked at
// only if its maximum beats the k-th key, what does goes into a buffer in LDS, and 64 of those are sorted in at a time.
// -inf (banned tokens) carries no probability; a row of nothing else has log probabilities -inf and entropy 0.  A row that holds a
// NaN or +inf has NaN log probabilities and entropy; its alternatives are ordered with NaN below -inf.  Ties go to the lower index.
// Bound: HBM (every logit is read once); ~9 vector instructions per logit.
#include "bh_decode.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int MAX_TOP = 64, WAVES = 4, THREADS = 64 * WAVES;

struct LogprobArgs {
    const void* x;
    long long stride;           // of a row, in elements
    const long long* targets;   // [rows][given]
    float *logprobs, *entropy, *top_logprobs;
    long long* top_ids;
    float* part_stats;          // [rows][parts][4]
    u64* part_keys;             // [rows][parts][top]
    int rows, vocab, given, top, parts;
    int per_part;               // 16-byte vectors of a part
};

// The distribution seen so far: 1 + rest is the sum of 2^(x2 - m2) over it, x2 = x log2(e), and first the sum of (x2 - m2) 2^(x2 - m2).
struct Seen {
    float m, rest, first;
    bool bad;  // a NaN was among it
};

__device__ __forceinline__ Seen joined(const Seen& a, const Seen& b) {
    const bool swap = b.m > a.m;
    const Seen hi = swap ? b : a, lo = swap ? a : b;
    Seen r = hi;
    r.bad = a.bad || b.bad;
    if (lo.m == -INFINITY) return r;  // nothing in it
    const float by = (lo.m - hi.m) * LOG2E, f = __builtin_amdgcn_exp2f(by), n = 1.0f + lo.rest;
    r.rest = hi.rest + f * n;
    if (f > 0.f) r.first = hi.first + f * (lo.first + by * n);
    return r;
}

// Order of the alternatives: the key of value x at index i; NaN is below -inf.  0 is no key at all.
__device__ __forceinline__ u64 key_of(float x, int i) {
    return ((u64)(x == x ? bh_ordf(x) : BH_ORD_NEG_INF - 1) << 32) | (u64)(~(unsigned)i);
}

template <typename E>
struct Vec {
    static constexpr int N = 16 / sizeof(E);
};

// The elements of 16-byte vector v of a row whose first element sits `off` elements behind a 16-byte border; what lies outside the
// row comes as -inf and has no index in [0, vocab).
template <typename E>
__device__ __forceinline__ void load_vector(const E* row, int off, int vocab, long long v, float (&x)[Vec<E>::N]) {
    constexpr int N = Vec<E>::N;
    const long long e0 = v * N - off;
    if (e0 >= 0 && e0 + N <= vocab) {
        typedef E vec __attribute__((ext_vector_type(N)));
        const vec w = *reinterpret_cast<const vec*>(row + e0);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = (float)w[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = e0 + e >= 0 && e0 + e < vocab ? (float)row[e0 + e] : -INFINITY;
    }
}

// What the waves of a workgroup found, joined by its first wave and written down: as the row's result, or as one part of it.
struct Shared {
    float stats[WAVES][4];
    u64 keys[WAVES][64];
};

__device__ __forceinline__ void finish(const LogprobArgs& a, int row, int part, int parts, Shared& sh, int lane, int wave, const Seen& mine, u64 key) {
    if (lane == 0) {
        sh.stats[wave][0] = mine.m;
        sh.stats[wave][1] = mine.rest;
        sh.stats[wave][2] = mine.first;
        sh.stats[wave][3] = mine.bad ? 1.f : 0.f;
    }
    if (a.top) sh.keys[wave][lane] = key;
    __syncthreads();
    if (wave) return;
    Seen s = mine;
    for (int w = 1; w < WAVES; ++w) s = joined(s, Seen{sh.stats[w][0], sh.stats[w][1], sh.stats[w][2], sh.stats[w][3] != 0.f});
    if (a.top) {
        u64 acc[1] = {key};
        for (int w = 1; w < WAVES; ++w) {
            const u64 b[1] = {sh.keys[w][lane]};
            bh_wave_merge_top<1>(acc, b, lane);
        }
        key = acc[0];
    }
    if (parts > 1) {
        const long long at = (long long)row * parts + part;
        if (lane == 0) *reinterpret_cast<floatx4*>(a.part_stats + 4 * at) = floatx4{s.m, s.rest, s.first, s.bad ? 1.f : 0.f};
        if (lane < a.top) a.part_keys[at * a.top + lane] = key;
        return;
    }
    const float log_sum = log1pf(s.rest);
    const bool bad = s.bad || s.m == INFINITY, none = s.m == -INFINITY;
    const float gone = bad ? __uint_as_float(0x7fc00000u) : -INFINITY;  // of every token of a bad or an empty row
    if (lane == 0) a.entropy[row] = bad ? gone : none ? 0.f : log_sum - LN2 * s.first / (1.0f + s.rest);
    if (lane < a.top) {
        const unsigned o = (unsigned)(key >> 32);
        const float x = bh_unordf(o);
        a.top_ids[(long long)row * a.top + lane] = (long long)bh_key_row(key);
        a.top_logprobs[(long long)row * a.top + lane] = bad || none ? gone : (x - s.m) - log_sum;
    }
}

// log probabilities of the row's given tokens; every lane of the wave that finish() leaves has the result's parts again from LDS
template <typename E>
__device__ __forceinline__ void given_tokens(const LogprobArgs& a, int row, const Seen& s, int lane) {
    const E* x = static_cast<const E*>(a.x) + row * a.stride;
    const float log_sum = log1pf(s.rest);
    const bool bad = s.bad || s.m == INFINITY, none = s.m == -INFINITY;
    for (int g = lane; g < a.given; g += 64) {
        const long long t = a.targets[(long long)row * a.given + g];
        float r = 0.f;  // a negative target names no token
        if (t >= a.vocab || (t >= 0 && bad))
            r = __uint_as_float(0x7fc00000u);
        else if (t >= 0)
            r = none ? -INFINITY : ((float)x[t] - s.m) - log_sum;
        a.logprobs[(long long)row * a.given + g] = r;
    }
}

__device__ __forceinline__ float wave_max(float v) {
    for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

template <typename E, bool TOP>
__global__ void __launch_bounds__(THREADS) bh_token_logprobs_kernel(LogprobArgs a) {
    constexpr int N = Vec<E>::N, U = 4, HOLD = 64 + 64 * N;  // a buffer takes one block on top of what does not fill a list yet
    __shared__ Shared sh;
    __shared__ u64 buffer[TOP ? WAVES : 1][TOP ? HOLD : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const E* x = static_cast<const E*>(a.x) + row * a.stride;
    const int off = (int)(((uintptr_t)x & 15) / sizeof(E));
    const long long vectors = ((long long)a.vocab + off + N - 1) / N;
    const long long v0 = (long long)part * a.per_part;
    const long long v1 = v0 + a.per_part < vectors ? v0 + a.per_part : vectors;

    Seen s{-INFINITY, 0.f, 0.f, false};  // m, bad: the wave's; rest, first: the lane's
    float m2 = 0.f;                      // m log2(e), rounded (0 while there is nothing but -inf): what the exponents are taken from, and
    float off2 = 0.f;                    // what the rounding left of it: 2^off2 is the maximum's own weight, put right at the end
    u64 best = 0, bar = 0;               // the lane's key of the wave's list; the k-th key: what is not above it cannot be among the k
    float bar_x = __uint_as_float(0x7fc00000u);  // its value; a NaN lets every block through
    int held = 0;
    bool first_block = true;

    auto flush = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes of the wave wrote what this one reads
        for (int at = 0; at < held; at += 64) {
            u64 b[1] = {at + lane < held ? buffer[TOP ? wave : 0][at + lane] : 0}, acc[1] = {best};
            bh_wave_sort_desc<1>(b, lane);
            bh_wave_merge_top<1>(acc, b, lane);
            best = acc[0];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        held = 0;
        const u64 kth = bh_shfl64(best, a.top - 1);
        if (kth > bar) bar = kth;
        if (bar) bar_x = bh_unordf((unsigned)(bar >> 32));
    };

    for (long long base = v0; base < v1; base += U * THREADS) {
        float xs[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = base + u * THREADS + threadIdx.x;
            if (v < v1)
                load_vector(x, off, a.vocab, v, xs[u]);
            else
#pragma unroll
                for (int e = 0; e < N; ++e) xs[u][e] = -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float most = xs[u][0];
            bool nan = most != most;
#pragma unroll
            for (int e = 1; e < N; ++e) {
                most = fmaxf(most, xs[u][e]);
                nan |= xs[u][e] != xs[u][e];
            }
            const bool look = nan || !(most <= (TOP ? bar_x : s.m));
            bool skip = false;  // the lane whose element became the maximum leaves its 1 out
            if (__any(look)) {
                if (__any(nan)) s.bad = true;
                const float top_x = wave_max(most);
                if (top_x > s.m) {
                    if (s.m > -INFINITY && top_x < INFINITY) {
                        const float by = m2 - __fmul_rn(top_x, LOG2E), f = __builtin_amdgcn_exp2f(by);
                        if (lane == 0) {  // the old maximum is one of many now
                            const float own = __builtin_amdgcn_exp2f(off2);
                            s.rest += own;
                            s.first = fmaf(off2, own, s.first);
                        }
                        s.first = f > 0.f ? f * (s.first + by * s.rest) : 0.f;
                        s.rest *= f;
                    }
                    s.m = top_x;
                    m2 = __fmul_rn(top_x, LOG2E);
                    off2 = top_x < INFINITY ? fmaf(top_x, LOG2E, -m2) : 0.f;
                    skip = lane == __ffsll((unsigned long long)__ballot(most == top_x)) - 1;
                }
                if (TOP) {
                    const long long i0 = (base + u * THREADS + threadIdx.x) * N - off;
                    const bool inside = base + u * THREADS + threadIdx.x < v1;
                    if (first_block) {
                        // a first bar: the k-th of the lanes' best elements (k of the block are at least as good)
                        u64 k[1] = {0};
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (inside && i0 + e >= 0 && i0 + e < a.vocab) {
                                const u64 ke = key_of(xs[u][e], (int)(i0 + e));
                                k[0] = k[0] > ke ? k[0] : ke;
                            }
                        bh_wave_sort_desc<1>(k, lane);
                        const u64 kth = bh_shfl64(k[0], a.top - 1);
                        if (kth) {
                            bar = kth - 1;
                            bar_x = bh_unordf((unsigned)(bar >> 32));
                        }
                        first_block = false;
                    }
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const u64 k = inside && i0 + e >= 0 && i0 + e < a.vocab ? key_of(xs[u][e], (int)(i0 + e)) : 0;
                        const unsigned long long who = __ballot(k > bar);
                        if (k > bar) buffer[wave][held + __popcll(who & ((1ull << lane) - 1))] = k;
                        held += __popcll(who);
                    }
                    if (held >= 64) flush();
                }
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float t = fmaxf(fmaf(xs[u][e], LOG2E, -m2), -1000.0f);  // (-inf: 2^-1000 is 0, and so is its product)
                float p = __builtin_amdgcn_exp2f(t);
                if (skip && xs[u][e] == s.m) {
                    p = 0.f;
                    skip = false;
                }
                s.rest += p;
                s.first = fmaf(t, p, s.first);
            }
        }
    }
    if (TOP) flush();
    s.rest = bh_group_sum(s.rest, 64);
    s.first = bh_group_sum(s.first, 64);
    s.first = __builtin_amdgcn_exp2f(-off2) * (s.first - off2 * s.rest);  // from m2 to m itself
    s.rest *= __builtin_amdgcn_exp2f(-off2);
    finish(a, row, part, a.parts, sh, lane, wave, s, best);
    if (wave || a.parts > 1) return;
    Seen all = s;
    for (int w = 1; w < WAVES; ++w) all = joined(all, Seen{sh.stats[w][0], sh.stats[w][1], sh.stats[w][2], sh.stats[w][3] != 0.f});
    given_tokens<E>(a, row, all, lane);
}

// Joins the parts of a row: one workgroup a row, wave w the parts w, w + 4, ...
template <typename E>
__global__ void __launch_bounds__(THREADS) bh_token_logprobs_join_kernel(LogprobArgs a) {
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x;
    Seen s{-INFINITY, 0.f, 0.f, false};
    u64 acc[1] = {0};
    for (int p = wave; p < a.parts; p += WAVES) {
        const long long at = (long long)row * a.parts + p;
        const floatx4 f = *reinterpret_cast<const floatx4*>(a.part_stats + 4 * at);
        s = joined(s, Seen{f[0], f[1], f[2], f[3] != 0.f});
        if (a.top) {
            const u64 b[1] = {lane < a.top ? a.part_keys[at * a.top + lane] : 0};
            bh_wave_merge_top<1>(acc, b, lane);
        }
    }
    finish(a, row, 0, 1, sh, lane, wave, s, acc[0]);
    if (wave) return;
    Seen all = s;
    for (int w = 1; w < WAVES; ++w) all = joined(all, Seen{sh.stats[w][0], sh.stats[w][1], sh.stats[w][2], sh.stats[w][3] != 0.f});
    given_tokens<E>(a, row, all, lane);
}

// How a row is cut: enough workgroups for the chip (4 on each of 256 CUs) where there are few rows, parts of at least 4 vectors a
// thread, whole steps of a workgroup.
void cut(int64_t rows, int64_t vocab, int32_t dtype, int* parts, int* per_part) {
    const int64_t n = 16 / (int64_t)bh_dtype_size(dtype);
    const int64_t vectors = (vocab + n - 1) / n + 1;  // (+ 1: a row that starts behind a 16-byte border)
    const int64_t step = 4 * THREADS, steps = (vectors + step - 1) / step;
    int64_t want = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    if (want > steps) want = steps;
    const int64_t per = (steps + want - 1) / want;
    *per_part = (int)(per * step);
    *parts = (int)((steps + per - 1) / per);
}

template <typename E>
void launch(const LogprobArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((long long)a.rows * a.parts));
    if (a.top)
        hipLaunchKernelGGL((bh_token_logprobs_kernel<E, true>), grid, dim3(THREADS), 0, st, a);
    else
        hipLaunchKernelGGL((bh_token_logprobs_kernel<E, false>), grid, dim3(THREADS), 0, st, a);
    if (a.parts > 1) hipLaunchKernelGGL((bh_token_logprobs_join_kernel<E>), dim3((unsigned)a.rows), dim3(THREADS), 0, st, a);
}

int check_sizes(int64_t rows, int64_t vocab, int32_t dtype, int32_t top) {
    if (!bh_is_float(dtype)) return bh_fail(BH_EINVAL, "bad dtype %d (fp16, bf16 or fp32)", dtype);
    if (rows < 0 || vocab < 1) return bh_fail(BH_EINVAL, "bad sizes");
    if (top < 0 || top > vocab) return bh_fail(BH_EINVAL, "top %d of %lld tokens", top, (long long)vocab);
    if (top > MAX_TOP) return bh_fail(BH_EUNSUPPORTED, "top %d (at most %d)", top, MAX_TOP);
    if (vocab > (1 << 30) || rows > (1 << 24)) return bh_fail(BH_EUNSUPPORTED, "more than 2^24 rows or 2^30 tokens");
    return BH_OK;
}

}  // namespace

extern "C" {

int64_t bh_op_token_logprobs_workspace(int64_t n_rows, int64_t vocab, int32_t dtype, int32_t top) {
    const int rc = check_sizes(n_rows, vocab, dtype, top);
    if (rc) return rc;
    if (n_rows == 0) return 0;
    int parts, per;
    cut(n_rows, vocab, dtype, &parts, &per);
    return parts > 1 ? n_rows * parts * (16 + 8 * (int64_t)top) : 0;
}

int bh_op_token_logprobs(const void* logits, int64_t row_stride, int32_t dtype, int64_t n_rows, int64_t vocab, const int64_t* targets,
                         int32_t n_given, int32_t top, float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids,
                         void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_sizes(n_rows, vocab, dtype, top);
    if (rc) return rc;
    if (n_given < 0) return bh_fail(BH_EINVAL, "bad sizes");
    if (n_rows > 1 && row_stride < vocab) return bh_fail(BH_EINVAL, "rows overlap (stride %lld, %lld tokens)", (long long)row_stride, (long long)vocab);
    if (n_rows == 0) return BH_OK;
    if (!logits || !entropy || (n_given && (!targets || !logprobs)) || (top && (!top_logprobs || !top_ids)))
        return bh_fail(BH_EINVAL, "null buffer");
    if ((uintptr_t)logits % bh_dtype_size(dtype)) return bh_fail(BH_EINVAL, "logits are not aligned to their type");
    LogprobArgs a{};
    cut(n_rows, vocab, dtype, &a.parts, &a.per_part);
    const int64_t need = a.parts > 1 ? n_rows * a.parts * (16 + 8 * (int64_t)top) : 0;
    if (need && (!workspace || workspace_bytes < need || !bh_aligned16(workspace)))
        return bh_fail(BH_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed: %lld given", (long long)need, (long long)workspace_bytes);
    if (n_rows * a.parts > 0x7fffffffll) return bh_fail(BH_EUNSUPPORTED, "too many rows");
    a.x = logits;
    a.stride = row_stride;
    a.targets = reinterpret_cast<const long long*>(targets);
    a.logprobs = logprobs, a.entropy = entropy, a.top_logprobs = top_logprobs;
    a.top_ids = reinterpret_cast<long long*>(top_ids);
    a.part_stats = static_cast<float*>(workspace);
    a.part_keys = reinterpret_cast<u64*>(static_cast<char*>(workspace) + 16 * n_rows * a.parts);
    a.rows = (int)n_rows, a.vocab = (int)vocab, a.given = n_given, a.top = top;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == BH_F16)
        launch<_Float16>(a, st);
    else if (dtype == BH_BF16)
        launch<__bf16>(a, st);
    else
        launch<float>(a, st);
    BH_HIP_TRY(hipGetLastError());
    return BH_OK;
}

}  // extern "C"
