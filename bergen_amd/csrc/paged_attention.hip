// paged_attention.hip — attention of one new token per sequence over a paged key-value cache, split over the cache's length.
//
//   s_t = scale q . k_t;  capped: s = c tanh(s / c);  distance bias: s -= slope (len - 1 - t);  t in [max(0, len - window), len)
//   out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),   lse = m + log sum_t e^(s_t - m)       (nothing left: out 0, lse -inf)
//
// Bound: HBM, by the cache's bytes — each key and value is read once for the whole group of query heads that shares it.  A query
// head alone makes 1 flop per byte, a group of 8 makes 8; on the vector units 8 would already take all their cycles, so both products run
// on the matrix cores, 16 heads wide whether there are 16 or 1 (the matrix pipe is busy 5 % of the time for 4 heads a group in bf16).
// Measured: 64 sequences of 90..8191 tokens, 8 key heads of 128, bf16: 186 us = 5.8 TB/s (the loads alone take as long); 3 of 100001..131072 tokens, e4m3:
// 126 us = 5.8 TB/s on some cards, 145 on others; 37 of 1..6000, window 4096, 12 heads of 64 without groups, int8: 43 us = 3.7 TB/s (the loads alone 31 us: the
// vector instructions of a tile are the same for 1 head as for 16).  64 of 90..4095, 8 key heads of 256: 253 us in bf16, 139 in e4m3 (4.3 and 4.0 TB/s, one
// wave a SIMD: registers); of 96: 92 and 47.
//
// A wave takes 32 tokens of one key head at a time and needs no LDS for them:
//   S^T = K Q^T     two tiles of 16 tokens.  Row i of tile u is token 8 (i / 4) + 4 u + i % 4, so that lane (g, n) — g = lane / 16,
//                   n = lane % 16 — ends up with the scores of the 8 CONSECUTIVE tokens 8 g .. 8 g + 7 of head n;
//   O^T += V^T P^T  wants in lane (g, n) the weights of 8 tokens of head n: those 8, as they are.  Its V^T operand, lane (g, i),
//                   wants the same 8 tokens of one dim; the lane loads D / 16 consecutive dims of each of them (a group's 16 lanes: a
//                   whole row) and turns its own little block round with byte permutes.
// Keys: lane (g, i) loads 16 bytes of its row, groups side by side.  8-bit codes become numbers of the queries' type, and values fp16, exactly, between
// load and MFMA; the keys' scale multiplies the score, the values' scale the weight.
// Weights reach the MFMA as a sum of two numbers of its type (hi + lo): bf16 alone would keep 2^-8 of a weight, as much as the output's own rounding;
// two keep 2^-17 (a third, the whole weight, costs 1 % of the time).  fp16 weights (8-bit caches: their products with the values' scales) are held times 2^14 so
// that small ones do not become subnormal: two keep 2^-22 of them, and leave out 2^-39 of the sequence's largest.
//
// Pages are 8..1024 tokens (a power of two): 8 consecutive tokens share one.  A table entry outside [0, pages) names a page that is
// not there: its tokens are left out.  What lies behind a sequence's end is neither counted nor multiplied (its values
// are replaced by zeros: 0 x NaN is NaN).
#include <type_traits>

#include "bh_decode.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int WAVES = 4, TILE = 32;  // waves of a workgroup, which take its tiles by turns; tokens of a tile

struct PagedArgs {
    const void* q;
    long long q_seq, q_head;  // strides in elements
    void* out;                // [batch][hq][dim]
    float* lse;               // [batch][hq] or null
    const void *k, *v;
    const float *k_scale, *v_scale, *slopes;
    const int* table;
    long long table_stride;
    const int* lengths;
    float* part_stats;  // [batch][hq][splits][2]: m log2(e), sum
    float* part_out;    // [batch][hq][splits][dim], not yet divided
    int batch, hq, hk, group, blocks, dim, n_pages, page_log2, table_width;
    int splits, per_split;  // of a sequence at most; tokens of one, for the longest that the table allows
    int work;               // batch times key heads (times blocks of 16 query heads), at most 256
    int window;
    float scale, softcap;
};

template <typename E>
struct Mma;
template <>
struct Mma<_Float16> {
    typedef half8 frag;
    static __device__ __forceinline__ floatx4 mul(frag a, frag b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<__bf16> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ floatx4 mul(frag a, frag b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// A load of what is not read again: the lines need not stay (bf16 cache of 1.08 GB, 64 sequences: 186 us, 201 us with plain loads).
// Not for 8-bit keys wider than 64 bytes, whose lines two instructions share: those were fetched twice (0.73 GB: 148 and 145 us).
template <typename T>
__device__ __forceinline__ T streamed(const unsigned char* p) {
    typedef unsigned words __attribute__((ext_vector_type(sizeof(T) / 4)));
    return __builtin_bit_cast(T, __builtin_nontemporal_load(reinterpret_cast<const words*>(p)));
}

// A sequence's tokens that count, [start, len), and its splits: `per` tokens each from `first` on, the tile that start lies in.
struct Range {
    int start, len, first, per, live;
};
__device__ __forceinline__ Range range_of(const PagedArgs& a, int seq) {
    Range r;
    const long long most = (long long)a.table_width << a.page_log2;
    r.len = a.lengths[seq];
    r.len = r.len < 0 ? 0 : r.len > most ? (int)most : r.len;
    r.start = a.window > 0 && r.len > a.window ? r.len - a.window : 0;
    r.first = r.start & ~(TILE - 1);
    // as many tokens as a sequence of its own length would get (a wide table says little of what is in use); longer ones where the splits run out
    constexpr int STEP = WAVES * TILE;
    const int tokens = r.len - r.first, share = (tokens + a.splits - 1) / a.splits;
    const long long even = (long long)tokens * a.work / 256;
    r.per = even < a.per_split ? (int)even : a.per_split;
    r.per = ((r.per > share ? r.per : share) + STEP - 1) / STEP * STEP;
    r.per = r.per < STEP ? STEP : r.per;
    r.live = (tokens + r.per - 1) / r.per;
    return r;
}

__device__ __forceinline__ float over_groups_max(float v) {  // over the 4 lanes with the same lane % 16
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// the power of two at or above v >= 0, 2^126 at most
__device__ __forceinline__ float power_above(float v) {
    const unsigned b = __float_as_uint(v);
    return b > 0x7e800000u ? 0x1p126f : __uint_as_float((b + 0x7fffffu) & 0x7f800000u);
}
// 2^n / p, p a power of two between 2^(n - 126) and 2^126
__device__ __forceinline__ float over_power(int n, float p) { return __uint_as_float(((unsigned)(254 + n) << 23) - __float_as_uint(p)); }

// two codes of a word, the lower two or (which = 1) the upper two, as two fp16
template <int CACHE>
__device__ __forceinline__ unsigned two_f16(unsigned word, int which) {
    if (CACHE == BH_I8) {
        // 1024 + (code + 128) as fp16 is the byte 0x64 over the code with its top bit flipped; minus 1152 is exact
        const unsigned u = word ^ 0x80808080u;
        const unsigned w = __builtin_amdgcn_perm(0x64646464u, u, which ? 0x04030402u : 0x04010400u);
        half2v h = __builtin_bit_cast(half2v, w);
        h -= (half2v){(_Float16)1152.f, (_Float16)1152.f};
        return __builtin_bit_cast(unsigned, h);
    }
    return which ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, true))
                 : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, false));
}

// the same as two of the queries' type: codes have at most 8 significant bits, which bf16 keeps as well
template <typename E, int CACHE>
__device__ __forceinline__ unsigned two_keys(unsigned word, int which) {
    if constexpr (std::is_same<E, _Float16>::value) return two_f16<CACHE>(word, which);
    if constexpr (CACHE == BH_E4M3)
        return which ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.0f, true))
                     : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.0f, false));
    // a code as fp32 ends in 16 zero bits: its upper half is the bf16
    const float lo = (float)(int)__builtin_amdgcn_sbfe((int)word, which ? 16 : 0, 8), hi = (float)(int)__builtin_amdgcn_sbfe((int)word, which ? 24 : 8, 8);
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// E: the queries' type; CACHE: BH_F16 / BH_BF16 (E's own), BH_I8, BH_E4M3; DP: head dim, rounded up to 64, 128 or 256 (EXACT: is it).
// ONE_PAGE: pages of 32 tokens and more, so that a tile lies in one.
template <typename E, int CACHE, int DP, bool EXACT, bool ONE_PAGE>
__global__ void __launch_bounds__(64 * WAVES, DP == 256 ? 1 : DP == 64 ? 4 : EXACT || CACHE == BH_I8 || CACHE == BH_E4M3 ? 3 : 2) bh_paged_attention_kernel(PagedArgs a) {
    constexpr bool SCALED = CACHE == BH_I8 || CACHE == BH_E4M3;
    typedef typename std::conditional<SCALED, _Float16, E>::type M;  // the type of the weights' and values' MFMAs; the scores' is E
    typedef typename Mma<M>::frag frag;
    typedef typename Mma<E>::frag key_frag;
    constexpr int ES = SCALED ? 1 : 2;            // bytes of a cached element
    constexpr int KS = DP / 32;                   // steps of S^T
    constexpr int KL = KS * 8 * ES / 16;          // 16-byte loads of a key row per lane
    constexpr int NJ = DP / 16;                   // dims of a value row per lane = tiles of O^T
    constexpr int VW = NJ * ES / 4;               // their words
    constexpr bool F16 = std::is_same<M, _Float16>::value;
    constexpr float HOLD = F16 ? 14.f : 0.f;      // weights are held times 2^HOLD
    constexpr float LEAST = 0x1p-112f;            // least unit of the values' scales times weights: 2^HOLD over it is finite, and a scale of 2^-126 keeps all its bits

    __shared__ key_frag sh_q[KS][64];  // registers are short; each wave writes the same and reads what it wrote
    __shared__ float sh_stats[WAVES][2][16];
    __shared__ float sh_out[WAVES][16][DP + 4];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    // (splits slowest: workgroups go to the XCDs in turn, and with the splits side by side the XCDs that get every sequence's
    // first ones would have far more to do than those that get the last ones, which most sequences do not have)
    const int split = blockIdx.z, seq = blockIdx.y;
    const int hk = blockIdx.x / a.blocks, block = blockIdx.x - hk * a.blocks;
    const int hq0 = hk * a.group + 16 * block;                       // the first of this workgroup's query heads
    const int heads = a.group - 16 * block < 16 ? a.group - 16 * block : 16;

    const Range range = range_of(a, seq);
    const int len = range.len, start = range.start, live_splits = range.live;
    if (split >= live_splits && split > 0) return;
    const int lo = range.first + split * range.per;
    const int hi = lo + range.per < len ? lo + range.per : len;

    // ---- the queries, operand B of S^T: lane (g, n) holds head n, dims as its key chunks
    const bool head_live = n < heads;
    const E* qp = static_cast<const E*>(a.q) + seq * a.q_seq + (long long)(hq0 + (head_live ? n : 0)) * a.q_head;
    float unit = a.scale * LOG2E;  // of a score, in powers of two
    {
        float top = 0.f;
        key_frag qs[KS];
        (void)qs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = SCALED ? 16 * ((s >> 1) * 4 + g) + 8 * (s & 1) : 8 * (4 * s + g);
            typedef E vec __attribute__((ext_vector_type(8)));
            vec x = {};
            if (head_live && d < a.dim) x = *reinterpret_cast<const vec*>(qp + d);
            if constexpr (std::is_same<E, M>::value) {
                sh_q[s][lane] = x;
            } else {
                qs[s] = x;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf((float)x[e]));
            }
        }
        if constexpr (!std::is_same<E, M>::value) {
            // bf16 queries against 8-bit keys: times the power of two that brings the head's largest to 2^7..2^8, exact but below 2^-133 of it.  The
            // codes are as large as the scales make them, and the sum of products with them must not leave fp32's range.  (As fp16, like the weights,
            // the elements of a head whose largest is 2^24 times theirs and more would lose bits)
            top = over_groups_max(top);
            int e = (int)(__float_as_uint(top) >> 23) - 127;
            e = e > 126 ? 126 : e < -112 ? -112 : e;
            const float up = ldexpf(1.f, 7 - e);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                key_frag f;
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = (E)((float)qs[s][i] * up);
                sh_q[s][lane] = f;
            }
            unit *= ldexpf(1.f, e - 7);
        }
    }
    const float slope = a.slopes && head_live ? a.slopes[hq0 + n] * LOG2E : 0.f;
    if (DP > 64) {
        if (g == 0) sh_stats[wave][0][n] = slope;  // (kept there until the wave's own m comes; heads of 64 keep it in a register)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the other lanes of the wave read it: not before the store
    }
    const float cap = a.softcap * LOG2E, cap_unit = a.softcap > 0.f ? 2.f / a.softcap : 0.f;

    float m, total;  // of head n: the same m in its 4 lanes; each lane's own sum, times 2^HOLD (scaled: as it is)
    // scaled: a power of two for head n that o and the held products (weight times value's scale) count in: no product is above it when it is held,
    // and their largest not far below it, however the scales compare (counting in the scales alone gave 0 beside values of 1e12 that weigh e^-100;
    // this costs a steep distance bias 1.2 us of 42, heads of 256 2 %).  slack: what the weights have lost since it was set
    float unit_v, slack;
    floatx4 o[NJ];

    const int* table = a.table + seq * a.table_stride;
    const int in_page = (1 << a.page_log2) - 1, last = a.table_width - 1;
    const int row = EXACT ? DP * ES : a.dim * ES;  // bytes
    // what a lane loads of a row: key bytes at 16 (4 s + g), value bytes at NJ ES n; behind the row's end (dim < DP) its first bytes instead
    int key_at[KL];
#pragma unroll
    for (int s = 0; s < KL; ++s) key_at[s] = EXACT || 16 * (4 * s + g) < row ? 16 * (4 * s + g) : 0;
    const int value_at = EXACT || NJ * n < a.dim ? NJ * ES * n : 0;
    const unsigned char* kc = static_cast<const unsigned char*>(a.k);
    const unsigned char* vc = static_cast<const unsigned char*>(a.v);

    // The page of the lane's 8 tokens (8 g..) of a tile (behind the table's end its last).  Where a tile has one page it is the
    // same for the whole wave and comes as a scalar, on a counter of its own
    auto page_of = [&](int t0) {
        const int t = t0 + (ONE_PAGE ? 0 : 8 * g);
        const int at = t >> a.page_log2;
        return table[at < last ? at : last];
    };
    auto there_at = [&](int page) { return (unsigned)page < (unsigned)a.n_pages; };
    // the vector of token t, a multiple of 8, in the cache; of token 0 of page 0 where there is no such page
    auto vector_at = [&](int t, int page) {
        const bool there = there_at(page);
        return (((long long)((there ? page : 0) * (long long)a.hk + hk)) << a.page_log2) + (there ? t & in_page : 0);
    };
    uint4 kr[2][KL];
    unsigned vreg[8][VW];
    float ks[8], vs[8];
    const int key_row = 8 * (n >> 2) + (n & 3);
    auto load_keys = [&](int t0, int page) {
        auto from = [&](const unsigned char* p, int off) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int s = 0; s < KL; ++s) {
                    const unsigned char* q = p + (off + 4 * u * row + key_at[s]);
                    kr[u][s] = KL > 1 && SCALED ? *reinterpret_cast<const uint4*>(q) : streamed<uint4>(q);
                }
        };
        if constexpr (ONE_PAGE) {
            const long long at = vector_at(t0, page);
            from(kc + at * row, key_row * row);
            if constexpr (SCALED) bh_load8(a.k_scale + at + 8 * g, ks);
        } else {
            const int key_page = __shfl(page, 16 * (n >> 2));  // of the lanes whose own tokens these are
            from(kc + vector_at(t0 + 8 * (n >> 2), key_page) * row, (n & 3) * row);
            if constexpr (SCALED) bh_load8(a.k_scale + vector_at(t0 + 8 * g, page), ks);
        }
    };
    auto load_values = [&](int t0, int page) {
        auto from = [&](const unsigned char* p, int off) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const unsigned char* q = p + (off + r * row);
                if constexpr (VW == 1) {
                    vreg[r][0] = streamed<unsigned>(q);
                } else if constexpr (VW == 2) {
                    const uint2 x = streamed<uint2>(q);
                    vreg[r][0] = x.x, vreg[r][1] = x.y;
                } else {
#pragma unroll
                    for (int w = 0; w < VW; w += 4) {
                        const uint4 x = streamed<uint4>(q + 4 * w);
                        vreg[r][w] = x.x, vreg[r][w + 1] = x.y, vreg[r][w + 2] = x.z, vreg[r][w + 3] = x.w;
                    }
                }
            }
        };
        if constexpr (ONE_PAGE) {
            const long long at = vector_at(t0, page);
            from(vc + at * row, 8 * g * row + value_at);
            if constexpr (SCALED) bh_load8(a.v_scale + at + 8 * g, vs);
        } else {
            const long long at = vector_at(t0 + 8 * g, page);
            from(vc + at * row, value_at);
            if constexpr (SCALED) bh_load8(a.v_scale + at, vs);
        }
    };

    // lo can be zero or below: an infinite value, times it, spoils what hi made of it.  Where a sum came out as NaN, the walk is taken once
    // more with hi alone, for those sums only
    bool both = true;
    for (;; both = false) {
        m = -INFINITY, total = 0.f, unit_v = LEAST, slack = 1.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j] = floatx4{0.f, 0.f, 0.f, 0.f};
        int t0 = lo + wave * TILE;
        int next_page = 0;
        bool there = false;
        if (t0 < hi) {
            const int page = page_of(t0);
            next_page = page_of(t0 + WAVES * TILE);
            there = there_at(page);
            load_keys(t0, page);
            load_values(t0, page);
        }
        // A tile's keys are asked for as soon as the tile before has used its own, its values likewise: no registers but one tile's.  Its
        // pages are asked for a tile earlier, before those loads: loads come back in order, and a page asked for behind a tile's values
        // would make the next tile's keys wait for them
        while (t0 < hi) {
            const int next = t0 + WAVES * TILE;
            int after_page = 0;
            const bool whole = t0 >= start && t0 + TILE <= hi && __all(there);

            // ---- S^T
            if (!EXACT) {
#pragma unroll
                for (int s = 0; s < KL; ++s)
                    if (16 * (4 * s + g) >= row) kr[0][s] = kr[1][s] = uint4{0, 0, 0, 0};
            }
            int q_lane = lane;
            // (or the loads move out of the loop, into the registers that they are to spare; heads of 64 have those)
            if constexpr (DP > 64) asm volatile("" : "+v"(q_lane));
            floatx4 st[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    key_frag kf;
                    if constexpr (SCALED) {
                        const uint4 c = kr[u][s >> 1];
                        const unsigned w0 = s & 1 ? c.z : c.x, w1 = s & 1 ? c.w : c.y;
                        const uint4 f = {two_keys<E, CACHE>(w0, 0), two_keys<E, CACHE>(w0, 1), two_keys<E, CACHE>(w1, 0), two_keys<E, CACHE>(w1, 1)};
                        kf = __builtin_bit_cast(key_frag, f);
                    } else {
                        kf = __builtin_bit_cast(key_frag, kr[u][s]);
                    }
                    st[u] = Mma<E>::mul(kf, sh_q[s][q_lane], st[u]);
                }
            float x[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = st[r >> 2][r & 3] * (SCALED ? ks[r] * unit : unit);
            if (next < hi) {
                after_page = page_of(next + WAVES * TILE);
                load_keys(next, next_page);
            }

            // ---- softmax: the lane's 8 tokens of head n
            auto capped = [&](float x) {
                const float e2 = __builtin_amdgcn_exp2f(fminf(x * cap_unit, 64.f));  // e^(2 s / c)
                return x == x ? cap * (e2 - 1.f) * __builtin_amdgcn_rcpf(e2 + 1.f) : x;
            };
            if (a.softcap > 128.f) {
                // e2 - 1 keeps 2^-23 of 1, which times a large cap is more than a score may be off by: below c / 4 tanh's series, whose first
                // term left out is 9e-9 of the score.  (Being there it costs low caps 2 us of 44, in a loop of its own as well; both forms with a
                // choice for each score cost 5)
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float z = x[r] * cap_unit * (0.5f * LN2), z2 = z * z;
                    const float series = x[r] + x[r] * (z2 * (-1.f / 3 + z2 * (2.f / 15 + z2 * (-17.f / 315 + z2 * (62.f / 2835)))));
                    x[r] = fabsf(z) < 0.25f ? series : capped(x[r]);
                }
            } else if (a.softcap > 0.f) {
#pragma unroll
                for (int r = 0; r < 8; ++r) x[r] = capped(x[r]);
            }
            if (a.slopes) {
                const float by = DP > 64 ? sh_stats[wave][0][n] : slope;
#pragma unroll
                for (int r = 0; r < 8; ++r) x[r] -= by * (float)(len - 1 - t0 - 8 * g - r);
            }
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int t = t0 + 8 * g + r;
                    const bool counts = there && t < hi && t >= start;
                    if (!counts) {
                        x[r] = -INFINITY;
                        if (SCALED) vs[r] = 0.f;
#pragma unroll
                        for (int w = 0; w < VW; ++w) vreg[r][w] = 0;
                    }
                }
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            if (__any(top > m)) {  // (a few times at the start of a walk, then hardly ever)
                const float now = fmaxf(m, over_groups_max(top));
                const float fade = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - now);
                m = now;
                total *= fade;
                float by = fade;
                if constexpr (SCALED) {
                    slack *= fade;
                    if (__any(slack < 0x1p-12f)) {  // (a large scale whose weight is gone must not hide the ones to come; until then they are held times 2^2 and keep 2^-27)
                        const float to = fmaxf(LEAST, power_above(unit_v * slack));
                        by = unit_v * fade * over_power(0, to);  // at most 2^12: o is in 32 bits
                        unit_v = to, slack = 1.f;
                    }
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j) o[j] *= by;
            }
            const float base = m == -INFINITY ? 0.f : SCALED ? m : m - HOLD;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                x[r] = __builtin_amdgcn_exp2f(x[r] - base);
                total += x[r];
                if constexpr (SCALED) x[r] *= vs[r];
            }
            // (the sum now, not when there is time for it: the weights would wait beside the products, and 8-bit heads of 80, 96 and 112 have no registers
            // for both in 3 waves a SIMD: 64 sequences of 4000 tokens, 8 key heads of 96, e4m3: 73 us, 85 in 2 waves.  Heads of 64 lose 5 of 45 us by it)
            if constexpr (SCALED && DP == 128 && !EXACT) asm volatile("" : "+v"(total));
            float per = 1.f;
            if constexpr (SCALED) {
                float big = fabsf(x[0]);
#pragma unroll
                for (int r = 1; r < 8; ++r) big = fmaxf(big, fabsf(x[r]));
                if (__any(big > unit_v)) {
                    const float to = fmaxf(unit_v, power_above(over_groups_max(big))), shrink = unit_v * over_power(0, to);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) o[j] *= shrink;
                    slack = to > unit_v ? 1.f : slack;
                    unit_v = to;
                }
                per = over_power(14, unit_v);
            }
            frag hi_p, lo_p;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float p = SCALED ? x[r] * per : x[r];
                // one value for both: left alone, the compiler rounds the product above to fp16 once in a fused instruction for hi and once
                // by way of fp32 for what hi is subtracted from, and where those fall on different sides lo belongs to another hi
                asm("" : "+v"(p));
                hi_p[r] = (M)p;
                lo_p[r] = (M)(p - (float)hi_p[r]);
            }
            if (!both) {
#pragma unroll
                for (int r = 0; r < 8; ++r) lo_p[r] = (M)0.f;
            }

            // ---- O^T
            if constexpr (SCALED) {
#pragma unroll
                for (int w = 0; w < VW; ++w) {  // 4 dims of 8 tokens
                    unsigned f[4][4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {  // tokens 2 h, 2 h + 1
                        const unsigned e01 = __builtin_amdgcn_perm(vreg[2 * h + 1][w], vreg[2 * h][w], 0x05010400u);
                        const unsigned e23 = __builtin_amdgcn_perm(vreg[2 * h + 1][w], vreg[2 * h][w], 0x07030602u);
                        f[0][h] = two_f16<CACHE>(e01, 0);
                        f[1][h] = two_f16<CACHE>(e01, 1);
                        f[2][h] = two_f16<CACHE>(e23, 0);
                        f[3][h] = two_f16<CACHE>(e23, 1);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const frag vf = __builtin_bit_cast(frag, (uint4{f[e][0], f[e][1], f[e][2], f[e][3]}));
                        o[4 * w + e] = Mma<M>::mul(vf, hi_p, o[4 * w + e]);
                        o[4 * w + e] = Mma<M>::mul(vf, lo_p, o[4 * w + e]);
                    }
                }
            } else {
#pragma unroll
                for (int w = 0; w < VW; ++w) {  // 2 dims of 8 tokens
                    uint4 f0, f1;
                    f0.x = __builtin_amdgcn_perm(vreg[1][w], vreg[0][w], 0x05040100u), f1.x = __builtin_amdgcn_perm(vreg[1][w], vreg[0][w], 0x07060302u);
                    f0.y = __builtin_amdgcn_perm(vreg[3][w], vreg[2][w], 0x05040100u), f1.y = __builtin_amdgcn_perm(vreg[3][w], vreg[2][w], 0x07060302u);
                    f0.z = __builtin_amdgcn_perm(vreg[5][w], vreg[4][w], 0x05040100u), f1.z = __builtin_amdgcn_perm(vreg[5][w], vreg[4][w], 0x07060302u);
                    f0.w = __builtin_amdgcn_perm(vreg[7][w], vreg[6][w], 0x05040100u), f1.w = __builtin_amdgcn_perm(vreg[7][w], vreg[6][w], 0x07060302u);
                    const frag v0 = __builtin_bit_cast(frag, f0), v1 = __builtin_bit_cast(frag, f1);
                    o[2 * w] = Mma<M>::mul(v0, hi_p, o[2 * w]);
                    o[2 * w + 1] = Mma<M>::mul(v1, hi_p, o[2 * w + 1]);
                    if (both) {
                        o[2 * w] = Mma<M>::mul(v0, lo_p, o[2 * w]);
                        o[2 * w + 1] = Mma<M>::mul(v1, lo_p, o[2 * w + 1]);
                    }
                }
            }
            if (next < hi) load_values(next, next_page);
            t0 = next, there = there_at(next_page), next_page = after_page;
        }
        if (SCALED || !both) break;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) odd |= o[j][r] != o[j][r] && (EXACT || NJ * (4 * g + r) + j < a.dim);
        if (!__any(odd)) break;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sh_out[wave][n][NJ * (4 * g + r) + j] = o[j][r];
    }
    total *= F16 && !SCALED ? 0x1p-14f : 1.f;

    // ---- the workgroup's waves joined
    total = over_groups_sum(total);
    if (g == 0) {
        sh_stats[wave][0][n] = m;
        sh_stats[wave][1][n] = total;
    }
    __syncthreads();
    float all = sh_stats[0][0][n];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) all = fmaxf(all, sh_stats[w][0][n]);
    const float base = all == -INFINITY ? 0.f : all;
    const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - base - HOLD) * (SCALED ? unit_v : 1.f);
    // lane (g, n), tile j, element r: head n, dim NJ (4 g + r) + j
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float& to = sh_out[wave][n][NJ * (4 * g + r) + j];
            const float x = !SCALED && !both && to == to ? to : o[j][r];
            to = m == -INFINITY ? 0.f : x * mine;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * a.dim; i += 64 * WAVES) {
        const int h = i / a.dim, d = i - h * a.dim;
        float top = sh_stats[0][0][h], sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = fmaxf(top, sh_stats[w][0][h]);
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            sum += sh_stats[w][1][h] * __builtin_amdgcn_exp2f(sh_stats[w][0][h] - from);
            x += sh_out[w][h][d];
        }
        const long long at = (long long)seq * a.hq + hq0 + h;
        if (live_splits > 1) {
            a.part_out[(at * a.splits + split) * a.dim + d] = x;
            if (d == 0) {
                a.part_stats[2 * (at * a.splits + split)] = top;
                a.part_stats[2 * (at * a.splits + split) + 1] = sum;
            }
        } else {
            static_cast<E*>(a.out)[at * a.dim + d] = (E)(sum > 0.f || sum != sum ? x / sum : 0.f);
            if (d == 0 && a.lse) a.lse[at] = sum > 0.f || sum != sum ? LN2 * (top + __builtin_amdgcn_logf(sum)) : -INFINITY;
        }
    }
}

// Joins the splits of one query head: a workgroup a head.  The splits' weights go to LDS; then 4 dims a thread, the splits by turns (8 of them
// at a time for a head of 128), 4 loads in flight.
template <typename E>
__global__ void __launch_bounds__(256) bh_paged_attention_join_kernel(PagedArgs a) {
    extern __shared__ __attribute__((aligned(16))) float weight[];  // [splits]
    __shared__ float sh[4];
    __shared__ floatx4 sh_out[256];
    const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
    const int live = range_of(a, seq).live;
    if (live <= 1) return;  // written by its only workgroup
    const long long at = (long long)seq * a.hq + head;
    const float* stats = a.part_stats + 2 * at * a.splits;
    float top = -INFINITY;
    for (int s = tid; s < live; s += 256) top = fmaxf(top, stats[2 * s]);
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    if ((tid & 63) == 0) sh[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
    const float from = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int s = tid; s < live; s += 256) {
        const float w = __builtin_amdgcn_exp2f(stats[2 * s] - from);
        weight[s] = w;
        sum += stats[2 * s + 1] * w;
    }
    sum = bh_group_sum(sum, 64);
    __syncthreads();
    if ((tid & 63) == 0) sh[tid >> 6] = sum;
    __syncthreads();
    sum = sh[0] + sh[1] + sh[2] + sh[3];
    const int quads = a.dim >> 2, wide = 1 << (32 - __clz(quads - 1));  // threads of one split: a power of two, 4..64
    const int d = tid & (wide - 1), turns = 256 / wide;
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
    if (d < quads) {
        const floatx4* part = reinterpret_cast<const floatx4*>(a.part_out + at * a.splits * a.dim) + d;
#pragma unroll 4
        for (int s = tid / wide; s < live; s += turns) x += part[(long long)s * quads] * weight[s];
    }
    sh_out[tid] = x;
    __syncthreads();
    if (tid < a.dim) {
        float y = 0.f;
        for (int i = 0; i < turns; ++i) y += sh_out[(tid >> 2) + i * wide][tid & 3];
        static_cast<E*>(a.out)[at * a.dim + tid] = (E)(sum > 0.f || sum != sum ? y / sum : 0.f);
        if (tid == 0 && a.lse) a.lse[at] = sum > 0.f || sum != sum ? LN2 * (top + __builtin_amdgcn_logf(sum)) : -INFINITY;
    }
}

// How the cache's length is split, by the longest length that the table allows (the lengths themselves are on the device); range_of does the same
// again for each sequence's own.  A CU takes about 30 GB/s whatever runs on it (700 tokens of one key head in one workgroup of 4
// waves or of 8: 12 us), so few sequences are spread over all 256 of them, down to 128 tokens a workgroup (one tile a wave: 6.7 us); beyond
// that fewer, longer splits cost less (64 sequences, up to 8191 tokens: 194 / 187 / 192 us in splits of 512 / 1024 / 2048; a window of
// 4096 on 444 heads: 41 / 43 / 53).  The join is a second launch of 3.7 us and more: none up to 768 tokens (8 heads, 700 tokens: 12.0 against 6.6 + 3.7
// and a launch), nor up to 2048 where the sequences alone fill the chip (32 sequences, up to 2000 tokens: 43.4 against 45.4 + 4.6).  At most
// 16384 workgroups, or 16 splits, however wide the table (65 thousand that find nothing to do take 20 us, and each split its workspace): a sequence
// that is longer than that many splits takes longer ones.
void split_length(int64_t batch, int64_t blocks, int64_t longest, int32_t window, int* splits, int* per_split) {
    if (window > 0 && window + TILE < longest) longest = window + TILE;  // (a window's start is rounded down to a tile)
    const int64_t work = batch * blocks, step = WAVES * TILE;
    int64_t per = (longest * work / 256 + step - 1) / step * step;
    per = per < step ? step : per > 1024 ? 1024 : per;
    if (longest <= 768 || (longest <= 2048 && work >= 256)) per = (longest + step - 1) / step * step;
    *per_split = (int)(per < step ? step : per);
    int64_t n = (longest + *per_split - 1) / *per_split, most = work > 1024 ? 16 : work < 4 ? 4096 : 16384 / work;
    *splits = (int)(n < 1 ? 1 : n < most ? n : most);
}

template <typename E, int CACHE, int DP, bool EXACT>
void launch_split(const PagedArgs& a, hipStream_t st) {
    const dim3 grid(a.hk * a.blocks, a.batch, a.splits), block(64 * WAVES);
    if (a.page_log2 >= 5)
        hipLaunchKernelGGL((bh_paged_attention_kernel<E, CACHE, DP, EXACT, true>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((bh_paged_attention_kernel<E, CACHE, DP, EXACT, false>), grid, block, 0, st, a);
}

template <typename E, int CACHE>
void launch_dim(const PagedArgs& a, hipStream_t st) {
    if (a.dim == 64)
        launch_split<E, CACHE, 64, true>(a, st);
    else if (a.dim == 128)
        launch_split<E, CACHE, 128, true>(a, st);
    else if (a.dim < 128)
        launch_split<E, CACHE, 128, false>(a, st);
    else
        launch_split<E, CACHE, 256, false>(a, st);
    if (a.splits > 1) hipLaunchKernelGGL((bh_paged_attention_join_kernel<E>), dim3(a.hq, a.batch), dim3(256), a.splits * sizeof(float), st, a);
}

int check_sizes(int32_t batch, int32_t hq, int32_t hk, int32_t dim, int32_t page_size, int32_t width) {
    if (batch < 0 || hq <= 0 || hk <= 0 || width < 0) return bh_fail(BH_EINVAL, "bad sizes");
    if (hq % hk) return bh_fail(BH_EINVAL, "%d query heads on %d key heads", hq, hk);
    if (dim < 16 || dim > 256 || dim % 16) return bh_fail(BH_EUNSUPPORTED, "head_dim %d (a multiple of 16, 16..256)", dim);
    if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1)))
        return bh_fail(BH_EUNSUPPORTED, "page_size %d (a power of two, 8..1024)", page_size);
    if (batch > 65535 || hq > 65535 || (long long)width * page_size > (1 << 30))
        return bh_fail(BH_EUNSUPPORTED, "more than 65535 sequences or heads, or 2^30 tokens of a sequence");
    return BH_OK;
}

}  // namespace

extern "C" {

int64_t bh_op_paged_attention_workspace(int32_t batch, int32_t n_q_heads, int32_t n_k_heads, int32_t head_dim, int32_t page_size,
                                        int32_t table_width, int32_t window) {
    const int rc = check_sizes(batch, n_q_heads, n_k_heads, head_dim, page_size, table_width);
    if (rc) return rc;
    if (window < 0) return bh_fail(BH_EINVAL, "bad window");
    if (batch == 0) return 0;
    int splits, per;
    split_length(batch, (int64_t)n_k_heads * ((n_q_heads / n_k_heads + 15) / 16), (int64_t)table_width * page_size, window, &splits, &per);
    return splits > 1 ? (int64_t)batch * n_q_heads * splits * (2 + (int64_t)head_dim) * 4 : 0;
}

int bh_op_paged_attention(const void* q, int64_t q_seq, int64_t q_head, int32_t dtype, const void* k_cache, const void* v_cache,
                          const float* k_scale, const float* v_scale, int32_t cache_dtype, int64_t n_pages, int32_t page_size,
                          const int32_t* table, int64_t table_stride, int32_t table_width, const int32_t* lengths, int32_t batch,
                          int32_t n_q_heads, int32_t n_k_heads, int32_t head_dim, float scale, float softcap, int32_t window,
                          const float* slopes, void* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_sizes(batch, n_q_heads, n_k_heads, head_dim, page_size, table_width);
    if (rc) return rc;
    if (dtype != BH_F16 && dtype != BH_BF16) return bh_fail(BH_EINVAL, "bad dtype %d (fp16 or bf16)", dtype);
    const bool scaled = cache_dtype == BH_I8 || cache_dtype == BH_E4M3;
    if (!scaled && cache_dtype != dtype) return bh_fail(BH_EINVAL, "bad cache dtype %d (the queries' own %d, int8 or e4m3)", cache_dtype, dtype);
    if (!(scale == scale) || !(softcap >= 0.f) || softcap == __builtin_inff() || window < 0)
        return bh_fail(BH_EINVAL, "bad scale, softcap or window");
    if (n_pages < 0 || n_pages > 0x7fffffff) return bh_fail(BH_EINVAL, "bad sizes");
    if (batch == 0) return BH_OK;
    if (!q || !lengths || !out || (table_width && (!table || !k_cache || !v_cache))) return bh_fail(BH_EINVAL, "null buffer");
    if (scaled && table_width && (!k_scale || !v_scale)) return bh_fail(BH_EINVAL, "an 8-bit cache needs the scales of keys and values");
    if (!bh_aligned16(k_scale) || !bh_aligned16(v_scale)) return bh_fail(BH_EUNSUPPORTED, "scales must be 16-byte aligned");
    if (!bh_aligned16(q) || !bh_aligned16(k_cache) || !bh_aligned16(v_cache) || (q_seq | q_head) % 8)
        return bh_fail(BH_EUNSUPPORTED, "queries and cache must be 16-byte aligned");
    PagedArgs a{};
    a.group = n_q_heads / n_k_heads;
    a.blocks = (a.group + 15) / 16;
    split_length(batch, (int64_t)n_k_heads * a.blocks, (int64_t)table_width * page_size, window, &a.splits, &a.per_split);
    const int64_t parts = a.splits > 1 ? (int64_t)batch * n_q_heads * a.splits : 0, need = parts * (2 + (int64_t)head_dim) * 4;
    if (need && (!workspace || workspace_bytes < need || !bh_aligned16(workspace)))
        return bh_fail(BH_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed: %lld given", (long long)need, (long long)workspace_bytes);
    a.q = q, a.q_seq = q_seq, a.q_head = q_head, a.out = out, a.lse = lse;
    a.k = k_cache, a.v = v_cache, a.k_scale = k_scale, a.v_scale = v_scale, a.slopes = slopes;
    a.table = table, a.table_stride = table_stride, a.lengths = lengths;
    a.part_out = static_cast<float*>(workspace);
    a.part_stats = a.part_out + parts * head_dim;
    a.work = (int64_t)batch * n_k_heads * a.blocks < 256 ? batch * n_k_heads * a.blocks : 256;
    a.batch = batch, a.hq = n_q_heads, a.hk = n_k_heads, a.dim = head_dim, a.n_pages = (int)n_pages;
    a.page_log2 = bh_ceil_log2(page_size), a.table_width = n_pages ? table_width : 0;
    a.window = window, a.scale = scale, a.softcap = softcap;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == BH_F16) {
        if (cache_dtype == BH_F16)
            launch_dim<_Float16, BH_F16>(a, st);
        else if (cache_dtype == BH_I8)
            launch_dim<_Float16, BH_I8>(a, st);
        else
            launch_dim<_Float16, BH_E4M3>(a, st);
    } else {
        if (cache_dtype == BH_BF16)
            launch_dim<__bf16, BH_BF16>(a, st);
        else if (cache_dtype == BH_I8)
            launch_dim<__bf16, BH_I8>(a, st);
        else
            launch_dim<__bf16, BH_E4M3>(a, st);
    }
    BH_HIP_TRY(hipGetLastError());
    return BH_OK;
}

}  // extern "C"
