// token_logprobs.hip — log probabilities of given tokens, entropy and the likeliest alternatives of each row of logits, in one pass.
//
//   lse = m + log sum_i e^(x_i - m),   logprob = x_target - lse,   H = log sum_i e^(x_i - m) - (sum_i (x_i - m) e^(x_i - m)) / (sum_i e^(x_i - m))
//
// A wave keeps ONE running maximum m for its 64 lanes (it changes a handful of times over a row; a maximum per lane would change in
// some lane at nearly every step) and per lane the sums of e^(x - m) and (x - m) e^(x - m) in fp32.  The sum leaves out the
// maximum's own 1: log1p of the rest keeps the entropy of a row that is nearly certain.
// Top alternatives: the wave's 64 best (value, index) keys live sorted across its lanes; elements are looked at only where the step's
// maximum beats the k-th key, and each that does takes its place at once, so that the bar is never stale (about k ln(n / 2048) of a wave's n).
// -inf (banned tokens) carries no probability; a row of nothing else has log probabilities -inf and entropy 0.  A row that holds a
// NaN or +inf has NaN log probabilities and entropy; its alternatives are ordered with NaN below -inf.  Ties go to the lower index.
// Bound: HBM and the vector units alike: a logit takes 9.2 of their issue slots (its exponential 4), which is as long as 2 bytes take from HBM.
// Measured, 4096 rows of 128000 in bf16: 164 us = 6.4 TB/s without alternatives, 201 us with 8, 247 with 20 (the candidates' instructions; about
// 30 of each wave's 32000 for 8; in the first 10 ms of a load, while the card's clock settles, up to 290 with 8).  61 rows of 120064, 20 alternatives: 16 + 8 us
// (the first step's candidates go in one by one, in an order that the join makes anew), 8 + 4 without; one row of 30522 in fp32, 5: 7 + 5 us (latency).
#include "bh_decode.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
// Beyond this magnitude of the running maximum m the exponents are taken from m itself.  Below it m log2(e) < 2^20.53, so that what its rounding leaves is at
// most 2^-4 (2^off2 of 0.957 .. 1.045); it grows with m, and from about 3e9 on 2^off2 is infinity or zero.
constexpr float FAR = 0x1p20f;
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

// Order of the alternatives: the key of value x at index i; NaN is below -inf, and -0 is 0.  0 is no key at all.
__device__ __forceinline__ u64 key_of(float x, int i) {
    return ((u64)(x == x ? bh_ordf(x + 0.0f) : BH_ORD_NEG_INF - 1) << 32) | (u64)(~(unsigned)i);
}

template <typename E>
struct Vec {
    static constexpr int N = 16 / sizeof(E);
    typedef E type __attribute__((ext_vector_type(N)));
};

// The 16-byte vector v of a row whose first element sits `off` elements behind a 16-byte border; what lies outside the row, or behind
// the part's last vector, comes as -inf.
template <typename E>
__device__ __forceinline__ typename Vec<E>::type load_vector(const E* row, int off, int vocab, long long v, long long v1) {
    typedef typename Vec<E>::type vec;
    constexpr int N = Vec<E>::N;
    const long long e0 = v * N - off;
    vec w;
    if (v < v1 && e0 >= 0 && e0 + N <= vocab) {
        w = __builtin_nontemporal_load(reinterpret_cast<const vec*>(row + e0));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = v < v1 && e0 + e >= 0 && e0 + e < vocab ? row[e0 + e] : (E)-INFINITY;
    }
    return w;
}

// What a workgroup joins: the distributions its waves (or a row's parts) saw and, in `sorted` lists of `top` keys, their best.
template <int KEYS>
struct Shared {
    alignas(16) float stats[WAVES][4];
    u64 bar, low;
    int count;
    u64 keys[KEYS];
};

// The best `top` of n_lists sorted lists, out(rank, key) for each, by the whole workgroup: what reaches a bar that `top` keys reach is
// collected and ranked by counting.  Two bars do: the best of the lists' last keys (`top` keys of that list), which is the higher one for few lists, and
// the least of their r-th, r = top / n_lists rounded up (r keys of each), for many.  Ranks that have no key: out(rank, 0).
template <int KEYS, typename Get, typename Out>
__device__ __forceinline__ void join_lists(Shared<KEYS>& sh, int n_lists, int top, Get get, Out out) {
    const int tid = threadIdx.x;
    if (tid == 0) sh.bar = 0, sh.low = ~0ull, sh.count = 0;
    __syncthreads();
    const int r = (top + n_lists - 1) / n_lists;
    for (int l = tid; l < n_lists; l += THREADS) {
        atomicMax(&sh.bar, get(l, top - 1));
        atomicMin(&sh.low, get(l, r - 1));
    }
    __syncthreads();
    const u64 bar = sh.bar > sh.low ? sh.bar : sh.low;
    for (int i = tid; i < n_lists * top; i += THREADS) {
        const int l = i / top;
        const u64 k = get(l, i - l * top);
        if (k && k >= bar) sh.keys[atomicAdd(&sh.count, 1)] = k;
    }
    __syncthreads();
    const int n = sh.count;
    for (int i = tid; i < n; i += THREADS) {
        const u64 k = sh.keys[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += sh.keys[j] > k ? 1 : 0;
        if (rank < top) out(rank, k);
    }
    for (int i = n + tid; i < top; i += THREADS) out(i, 0);
}

// A row's results, by the whole workgroup: `lists` sorted lists of keys, and what was seen in sh.stats.
template <typename E, int KEYS, typename Get>
__device__ __forceinline__ void finish(const LogprobArgs& a, int row, Shared<KEYS>& sh, int lists, Get get) {
    Seen s{-INFINITY, 0.f, 0.f, false};
    for (int w = 0; w < WAVES; ++w) s = joined(s, Seen{sh.stats[w][0], sh.stats[w][1], sh.stats[w][2], sh.stats[w][3] != 0.f});
    const float log_sum = log1pf(s.rest);
    const bool bad = s.bad || s.m == INFINITY, none = s.m == -INFINITY;
    const float gone = bad ? __uint_as_float(0x7fc00000u) : -INFINITY;  // of every token of a bad or an empty row
    if (threadIdx.x == 0) a.entropy[row] = bad ? gone : none ? 0.f : log_sum - LN2 * s.first / (1.0f + s.rest);
    const E* x = static_cast<const E*>(a.x) + row * a.stride;
    for (int g = threadIdx.x; g < a.given; g += THREADS) {
        const long long t = a.targets[(long long)row * a.given + g];
        float r = 0.f;  // a negative target names no token
        if (t >= a.vocab || (t >= 0 && bad))
            r = __uint_as_float(0x7fc00000u);
        else if (t >= 0)
            r = none ? -INFINITY : ((float)x[t] - s.m) - log_sum;
        a.logprobs[(long long)row * a.given + g] = r;
    }
    if (a.top)
        join_lists(sh, lists, a.top, get, [&](int rank, u64 key) {
            a.top_ids[(long long)row * a.top + rank] = (long long)bh_key_row(key);
            a.top_logprobs[(long long)row * a.top + rank] = bad || none ? gone : (bh_key_score(key) - s.m) - log_sum;
        });
}

__device__ __forceinline__ float wave_max(float v) {
    for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

// the largest of three, NaN left out; as the one instruction (fmaxf first makes every operand that came from memory a quiet NaN if it is one)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// the value of the lane before (lane 0: nothing that is used)
__device__ __forceinline__ u64 lane_before(u64 v) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)v, 0x138 /* wave_shr:1 */, 0xf, 0xf, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), 0x138, 0xf, 0xf, false);
    return ((u64)hi << 32) | lo;
}

// A number that at least k of the wave's lanes reach with theirs, the largest with 16 leading bits only: found bit by bit by
// counting (a full sort of the lanes takes four times as long, and a bar that is a little low lets one or two elements more through).
__device__ __forceinline__ unsigned reached_by(unsigned v, int k) {
    unsigned t = 0;
    for (int bit = 31; bit >= 16; --bit) {
        const unsigned c = t | (1u << bit);
        if (__popcll(__ballot(v >= c)) >= k) t = c;
    }
    return t;
}

template <typename E, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) bh_token_logprobs_kernel(LogprobArgs a) {
    constexpr int MANY = 8, N = Vec<E>::N, U = 4;  // elements of a vector, vectors of a lane's step
    typedef float Step __attribute__((ext_vector_type(U * N)));
    // the mode register's IEEE bit off: with it a maximum of a number and a signalling NaN is NaN, and the number would be lost to the alternatives
    __builtin_amdgcn_s_setreg(1 /* MODE */ | 9 << 6 /* bit 9 */ | 0 << 11 /* one bit */, 0);
    __shared__ Shared<TOP ? WAVES * 64 : 1> sh;
    __shared__ u64 lists[TOP ? WAVES * 64 : 1];  // the waves' own
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const E* x = static_cast<const E*>(a.x) + row * a.stride;
    const int off = (int)(((uintptr_t)x & 15) / sizeof(E));
    const long long vectors = ((long long)a.vocab + off + N - 1) / N;
    const long long v0 = (long long)part * a.per_part;
    const long long v1 = v0 + a.per_part < vectors ? v0 + a.per_part : vectors;

    Seen s{-INFINITY, 0.f, 0.f, false};  // m: the wave's; rest, first: the lane's
    float m2 = 0.f;                      // m log2(e), rounded (0 while there is nothing but -inf): what the exponents are taken from, and
    float off2 = 0.f;                    // what the rounding left of it: 2^off2 is the maximum's own weight, put right at the end
    bool huge = false;                   // m is beyond FAR (masked tokens of -1e10, the type's lowest value): exponents from m itself, m2 and off2 are 0
    u64 best = 0, bar = 0;               // the lane's key of the wave's list; the k-th key: what is not above it cannot be among the k
    float bar_x = __uint_as_float(0x7fc00000u);  // its value; a NaN lets everything through

    // the indices of this part's elements; what lies outside (a row's ends, vectors that were not loaded) has none of them
    const int i_first = v0 * N - off > 0 ? (int)(v0 * N - off) : 0;
    const unsigned i_count = (unsigned)((v1 * N - off < a.vocab ? (int)(v1 * N - off) : a.vocab) - i_first);
    // The elements of a step take their places in the list: those in its places `places` (bit b = u N + e: the lanes' elements e of their vectors
    // u, index i0 + u THREADS N + e) that beat the bar.  Few places, as in all steps but the first: one after the other, the registers chosen
    // by a scalar.  Many: one element of each lane at a time, read again, sorted and merged.  (Neither is there once for each of the 32 places: as it
    // was, most of 37 us for 61 rows went into fetching instructions.  Which elements beat the bar is kept in scalars: as bits of
    // each lane it took 24 vector instructions for a vector, not 8, and these are what the kernel is bound by.)
    auto take = [&](const Step& xs, unsigned places, int i0) {
        auto new_bar = [&]() {
            const int k = a.top - 1;
            const unsigned high = __builtin_amdgcn_readlane((int)(best >> 32), k);
            const u64 kth = ((u64)high << 32) | (unsigned)__builtin_amdgcn_readlane((int)best, k);
            if (kth > bar) bar = kth, bar_x = bh_unordf(high);
        };
        auto insert = [&](u64 key, unsigned long long who) {  // the keys of the lanes `who`, as long as they beat the bar
            while (who) {
                const int l = __ffsll(who) - 1;
                const u64 k = ((u64)(unsigned)__builtin_amdgcn_readlane((int)(key >> 32), l) << 32) | (unsigned)__builtin_amdgcn_readlane((int)key, l);
                const int at = __popcll(__ballot(best > k));
                const u64 before = lane_before(best);
                best = lane < at ? best : lane == at ? k : before;
                new_bar();
                who &= who - 1;
                who &= __ballot(key > bar);
            }
        };
        if (__popc(places) > MANY) {
            unsigned look = 0;
            for (; places; places &= places - 1) {
                const int b = __ffs((int)places) - 1;
                look |= !(xs[b] <= bar_x) ? 1u << b : 0;
            }
            for (; __any(look != 0); look &= look - 1) {
                const int b = __ffs((int)look) - 1, i = i0 + (b / N) * THREADS * N + b % N;
                u64 key[1] = {0}, acc[1] = {best};
                if (look != 0 && (unsigned)(i - i_first) < i_count) key[0] = key_of((float)x[i], i);
                const unsigned long long who = __ballot(key[0] > bar);
                if (__popcll(who) > 12) {
                    bh_wave_sort_desc<1>(key, lane);
                    bh_wave_merge_top<1>(acc, key, lane);
                    best = acc[0];
                    new_bar();
                } else {
                    insert(key[0], who);
                }
            }
            return;
        }
        for (; places; places &= places - 1) {
            const int b = __ffs((int)places) - 1, i = i0 + (b / N) * THREADS * N + b % N;
            const u64 key = (unsigned)(i - i_first) < i_count ? key_of(xs[b], i) : 0;
            insert(key, __ballot(key > bar));
        }
    };

    typename Vec<E>::type w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = load_vector(x, off, a.vocab, v0 + u * THREADS + threadIdx.x, v1);
    for (long long base = v0; base < v1; base += U * THREADS) {
        Step xs;
        float most[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int e = 0; e < N; ++e) xs[u * N + e] = (float)w[u][e];
            most[u] = N == 8 ? max3(max3(xs[u * N + 0], xs[u * N + 1], xs[u * N + 2]), max3(xs[u * N + 3], xs[u * N + 4], xs[u * N + 5]), max3(xs[u * N + 6], xs[u * N + 6], xs[u * N + N - 1]))
                             : max3(xs[u * N + 0], xs[u * N + 1], max3(xs[u * N + 2], xs[u * N + 2], xs[u * N + 3]));
        }
        if (base + U * THREADS < v1) {  // the next step's loads run beside this one's arithmetic
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = load_vector(x, off, a.vocab, base + (U + u) * THREADS + threadIdx.x, v1);
        }
        const float step_most = max3(most[0], most[1], max3(most[2], most[2], most[3]));
        if (TOP && __any(!(step_most <= bar_x))) {
            if (base == v0) {
                // a first bar, just below what k of the lanes' largest reach (k elements of the step are at least as good)
                const unsigned o = step_most == step_most ? bh_ordf(step_most + 0.0f) : 0;
                const unsigned kth = reached_by(o, a.top);
                if (kth > BH_ORD_NEG_INF) {
                    bar = ((u64)kth << 32) - 1;
                    bar_x = bh_unordf(kth - (kth == 0x80000000u ? 2 : 1));  // (one below 0 is -0, which is not less)
                }
            }
            unsigned places = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (__any(!(most[u] <= bar_x))) {  // (what was seen before this step has lower indices: equal values stay out)
#pragma unroll
                    for (int e = 0; e < N; ++e) places |= __any(!(xs[u * N + e] <= bar_x)) ? 1u << (u * N + e) : 0;
                }
            take(xs, places, (int)((base + threadIdx.x) * N - off));
        }
        if (__any(step_most > s.m)) {  // a new maximum: a few times in a row
            const float top_x = wave_max(step_most);
            const bool far = fabsf(top_x) > FAR;
            float top2 = far ? 0.f : top_x * LOG2E;
            asm("" : "+v"(top2));  // the ROUNDED product in every use: fused into the difference below it moved the sums by up to 2^off2 (5e-3 at 1e5)
            const float top_off = far ? 0.f : fmaf(top_x, LOG2E, -top2);
            if (s.m > -INFINITY && top_x < INFINITY) {
                // from the old base to the new one; each is its maximum's exponent less its off2
                const float by = huge || far ? (s.m - top_x) * LOG2E + (top_off - off2) : m2 - top2, f = __builtin_amdgcn_exp2f(by);
                if (lane == 0) {  // the old maximum is one of many now
                    const float own = __builtin_amdgcn_exp2f(off2);
                    s.rest += own;
                    s.first = fmaf(off2, own, s.first);
                }
                s.first = f > 0.f ? f * (s.first + by * s.rest) : 0.f;
                s.rest *= f;
            }
            s.m = top_x;
            huge = far;
            m2 = top2;
            off2 = top_off;
            // its own 1 is left out: one element that equals it, of one lane
            bool mine = lane == __ffsll((unsigned long long)__ballot(step_most == top_x)) - 1;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (mine && xs[u * N + e] == top_x) {
                        xs[u * N + e] = -INFINITY;
                        mine = false;
                    }
            if (top_x == INFINITY) s.rest = __uint_as_float(0x7fc00000u);
        }
        if (__any(huge)) {
#pragma unroll
            for (int b = 0; b < U * N; ++b) xs[b] -= s.m;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float t = fmaf(xs[u * N + e], LOG2E, -m2), p = __builtin_amdgcn_exp2f(t);
                s.rest += p;                              // (a NaN stays in it)
                s.first = fmaf(fmaxf(t, -1000.0f), p, s.first);  // (-inf: p is 0, and so is its product with -1000)
            }
    }
    s.rest = bh_group_sum(s.rest, 64);
    s.first = bh_group_sum(s.first, 64);
    s.bad = s.rest != s.rest;
    s.first = __builtin_amdgcn_exp2f(-off2) * (s.first - off2 * s.rest);  // from m2 to m itself
    s.rest *= __builtin_amdgcn_exp2f(-off2);
    if (lane == 0) *reinterpret_cast<floatx4*>(sh.stats[wave]) = floatx4{s.m, s.rest, s.first, s.bad ? 1.f : 0.f};
    if (TOP) lists[wave * 64 + lane] = best;
    __syncthreads();
    const auto get = [&](int l, int i) { return lists[TOP ? l * 64 + i : 0]; };
    if (a.parts == 1) {
        finish<E>(a, row, sh, WAVES, get);
        return;
    }
    const long long at = (long long)row * a.parts + part;
    if (threadIdx.x == 0) {
        Seen all = s;
        for (int w = 1; w < WAVES; ++w) all = joined(all, Seen{sh.stats[w][0], sh.stats[w][1], sh.stats[w][2], sh.stats[w][3] != 0.f});
        *reinterpret_cast<floatx4*>(a.part_stats + 4 * at) = floatx4{all.m, all.rest, all.first, all.bad ? 1.f : 0.f};
    }
    if (TOP) join_lists(sh, WAVES, a.top, get, [&](int rank, u64 key) { a.part_keys[at * a.top + rank] = key; });
}

constexpr int JOIN_KEYS = 2048;  // parts times top: 16 KiB of LDS

// Joins the parts of a row: one workgroup a row, wave w the distributions of its quarter of them.
template <typename E>
__global__ void __launch_bounds__(THREADS) bh_token_logprobs_join_kernel(LogprobArgs a) {
    __shared__ Shared<JOIN_KEYS> sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x;
    Seen s{-INFINITY, 0.f, 0.f, false};
    for (int p = threadIdx.x; p < a.parts; p += THREADS) {
        const floatx4 f = *reinterpret_cast<const floatx4*>(a.part_stats + 4 * ((long long)row * a.parts + p));
        s = joined(s, Seen{f[0], f[1], f[2], f[3] != 0.f});
    }
    for (int d = 1; d < 64; d <<= 1)
        s = joined(s, Seen{__shfl_xor(s.m, d), __shfl_xor(s.rest, d), __shfl_xor(s.first, d), (bool)__shfl_xor((int)s.bad, d)});
    if (lane == 0) *reinterpret_cast<floatx4*>(sh.stats[wave]) = floatx4{s.m, s.rest, s.first, s.bad ? 1.f : 0.f};
    __syncthreads();
    const u64* keys = a.part_keys + (long long)row * a.parts * a.top;
    finish<E>(a, row, sh, a.parts, [&](int l, int i) { return keys[l * a.top + i]; });
}

// How a row is cut: enough workgroups for the chip (4 on each of 256 CUs) where there are few rows, parts of at least 4 vectors a
// thread, whole steps of a workgroup.
void cut(int64_t rows, int64_t vocab, int32_t dtype, int32_t top, int* parts, int* per_part) {
    const int64_t n = 16 / (int64_t)bh_dtype_size(dtype);
    const int64_t vectors = (vocab + n - 1) / n + 1;  // (+ 1: a row that starts behind a 16-byte border)
    const int64_t step = 4 * THREADS, steps = (vectors + step - 1) / step;
    int64_t want = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    if (want > steps) want = steps;
    if (top > 0 && want > JOIN_KEYS / top) want = JOIN_KEYS / top;
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
    cut(n_rows, vocab, dtype, top, &parts, &per);
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
    cut(n_rows, vocab, dtype, top, &a.parts, &a.per_part);
    const int64_t need = a.parts > 1 ? n_rows * a.parts * (16 + 8 * (int64_t)top) : 0;
    if (need && (!workspace || workspace_bytes < need || !bh_aligned16(workspace)))
        return bh_fail(BH_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed: %lld given", (long long)need, (long long)workspace_bytes);
    if (n_rows * a.parts >= 1 << 24) return bh_fail(BH_EUNSUPPORTED, "too many rows");
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
