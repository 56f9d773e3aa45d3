// decode_ops.hip — the memory-bound operators of a decoding step: RMS norm of query / key heads with rotary positions in the same
// pass, and the paged key-value cache's write and read, plain or in 8 bits with a scale per token and head.
//
// All three move vectors of one (token, head): D elements, D <= 256.  The wide kernels give a lane two 16-byte pieces of a vector
// and a vector 1..32 lanes, a power of two, so that sums and maxima over it are 0..5 exchanges between neighbouring lanes and nothing
// passes through LDS; they need whole pieces and 16-byte rows.  Everything else (odd D, unaligned views) runs on the narrow
// kernels: one wave per vector, one element per lane and step.
// Bound: HBM (each element is read once and written once).  Measured: norm + rotary of 16384 tokens of 32 + 8 heads of 128, bf16: 68 us = 4.9 TB/s (a copy: 4.9);
// 8192 such tokens in fp32, pairs side by side: 65 us = 5.1 TB/s; 65536 tokens of 8 heads of 128 read from an e4m3 cache of 64-token pages as bf16: 70 us = 5.8
// TB/s; 8192 written: 17 us = 3.0 TB/s, most of it waiting (a group of lanes moves one vector and ends).  Rows that the narrow kernels take, 4096 tokens of
// 32 + 8 heads of 100 in bf16: 50 us where a copy takes 13.
#include "bh_decode.h"

namespace {

constexpr int MAX_D = 256;

// ---- norm + rotary ---------------------------------------------------------------------------------------------------------

struct RotaryArgs {
    const void *q, *k;
    void *q_out, *k_out;
    long long q_tok, q_head, qo_tok, qo_head, k_tok, k_head, ko_tok, ko_head;  // strides in elements
    const void *qw, *kw;
    const void* pos;
    const double* inv_freq;
    long long n_tokens;
    int nq, nk, dim, rot, tb;  // tb: tokens of a workgroup
    int lanes_log2;            // lanes of a vector (wide kernel)
    float eps;
    bool pos64, w32, interleaved;
};

// cos and sin of pos * f, f in radians per position.  The angle is formed, reduced to a fraction of a turn and to |x| <= pi / 4 in 64 bits, and so are
// the two Taylor series (the terms left out are below 2^-37 there): the results are the nearest fp32 numbers but for ties that close.  (A fraction
// narrowed to fp32 before its sine moves the angle by up to 2^-23.4, which doubled the outputs that round the other way than the exact ones in bf16.)
__device__ __forceinline__ void angle_of(double pos, double f, float& c, float& s) {
    double t = pos * f * 0.15915494309189533577;  // 1 / (2 pi)
    t -= rint(t);
    const double quarters = rint(4.0 * t), x = (t - 0.25 * quarters) * 6.283185307179586477, z = x * x;
    const double sn = x + x * z * (-1.0 / 6 + z * (1.0 / 120 + z * (-1.0 / 5040 + z * (1.0 / 362880 + z * (-1.0 / 39916800)))));
    const double cs = 1.0 + z * (-0.5 + z * (1.0 / 24 + z * (-1.0 / 720 + z * (1.0 / 40320 + z * (-1.0 / 3628800 + z * (1.0 / 479001600))))));
    const float a = (float)cs, b = (float)sn;
    const bool odd = fabs(quarters) == 1.0;                           // (a NaN: no quarter at all, and both series are NaN)
    const bool half = fabs(quarters) == 2.0, third = quarters < 0.0;  // -1 quarter: three of them
    const float u = odd ? b : a, v = odd ? a : b;
    c = half || (odd && !third) ? -u : u;
    s = half || (odd && third) ? -v : v;
}

__device__ __forceinline__ double position(const RotaryArgs& a, long long t) {
    return a.pos64 ? (double)static_cast<const long long*>(a.pos)[t] : (double)static_cast<const int*>(a.pos)[t];
}

// C elements of E at p (of 16 bytes, or 8 where the other side is fp32) as fp32, and back, rounded once.
template <typename E, int C>
__device__ __forceinline__ void load16(const E* p, float (&x)[C]) {
    typedef E vec __attribute__((ext_vector_type(C)));
    const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int e = 0; e < C; ++e) x[e] = (float)v[e];
}
template <typename E, int C>
__device__ __forceinline__ void store16(E* p, const float (&x)[C]) {
    typedef E vec __attribute__((ext_vector_type(C)));
    vec v;
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = (E)x[e];
    *reinterpret_cast<vec*>(p) = v;
}
template <typename E, int C>
__device__ __forceinline__ void weights(const RotaryArgs& a, const void* w, int d, float (&x)[C]) {
    if (a.w32) {
#pragma unroll
        for (int e = 0; e < C; e += 4) load16<float, 4>(static_cast<const float*>(w) + d + e, reinterpret_cast<float(&)[4]>(x[e]));
    } else {
        load16<E, C>(static_cast<const E*>(w) + d, x);
    }
}

// A workgroup takes `tb` tokens with all their heads: the sines of a token are computed once, into LDS, and shared by its heads
// (64 for a head of 128; per head they would cost 40 times as much as the norm).  A lane holds two pieces of 16 bytes (C elements) of a vector, at
// C i of either half: of the rotated part's halves, so that a pair stays in one lane, of the rest's behind them, or, with pairs
// side by side, of the vector's.  Neighbouring lanes load neighbouring pieces.
template <typename E>
__global__ void __launch_bounds__(256) bh_qk_norm_rotary_kernel(RotaryArgs a) {
    constexpr int C = 16 / sizeof(E);
    extern __shared__ __attribute__((aligned(16))) float trig[];  // [tb][2][rot / 2]
    const int half = a.rot >> 1;
    const long long t0 = (long long)blockIdx.x * a.tb;
    const int nt = a.n_tokens - t0 < a.tb ? (int)(a.n_tokens - t0) : a.tb;
    for (int i = threadIdx.x; i < nt * half; i += 256) {
        const int t = i / half, j = i - t * half;
        float c, s;
        angle_of(position(a, t0 + t), a.inv_freq[j], c, s);
        trig[t * a.rot + j] = c;
        trig[t * a.rot + half + j] = s;
    }
    __syncthreads();
    const int heads = a.nq + a.nk, lanes = 1 << a.lanes_log2;
    const int i = threadIdx.x & (lanes - 1), in_first = half / C;  // lanes of the rotated part, where its halves are paired
    const bool live = 2 * C * i < a.dim;
    int d0, d1;
    if (a.interleaved)
        d0 = C * i, d1 = a.dim / 2 + C * i;
    else if (i < in_first)
        d0 = C * i, d1 = half + C * i;
    else
        d0 = a.rot + C * (i - in_first), d1 = a.rot + (a.dim - a.rot) / 2 + C * (i - in_first);
    for (int v = threadIdx.x >> a.lanes_log2; v < nt * heads; v += 256 >> a.lanes_log2) {
        const int t = v / heads, h = v - t * heads;
        const bool is_q = h < a.nq;
        const E* src = is_q ? static_cast<const E*>(a.q) + (t0 + t) * a.q_tok + h * a.q_head
                            : static_cast<const E*>(a.k) + (t0 + t) * a.k_tok + (h - a.nq) * a.k_head;
        E* dst = is_q ? static_cast<E*>(a.q_out) + (t0 + t) * a.qo_tok + h * a.qo_head
                      : static_cast<E*>(a.k_out) + (t0 + t) * a.ko_tok + (h - a.nq) * a.ko_head;
        const void* w = is_q ? a.qw : a.kw;
        float x[C] = {}, y[C] = {};
        if (live) {
            load16<E, C>(src + d0, x);
            load16<E, C>(src + d1, y);
        }
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < C; ++e) ss += x[e] * x[e] + y[e] * y[e];
            const float r = 1.0f / sqrtf(bh_group_sum(ss, lanes) / (float)a.dim + a.eps);
            if (live) {
                float wx[C], wy[C];
                weights<E, C>(a, w, d0, wx);
                weights<E, C>(a, w, d1, wy);
#pragma unroll
                for (int e = 0; e < C; ++e) {
                    x[e] *= r * wx[e];
                    y[e] *= r * wy[e];
                }
            }
        }
        if (!live) continue;
        const float *cos_t = &trig[t * a.rot], *sin_t = cos_t + half;
        if (a.interleaved) {
            auto turn = [&](float(&z)[C], int d) {
                if (d >= a.rot) return;
#pragma unroll
                for (int e = 0; e < C / 2; ++e) {
                    const float c = cos_t[d / 2 + e], s = sin_t[d / 2 + e], u = z[2 * e], p = z[2 * e + 1];
                    z[2 * e] = u * c - p * s;
                    z[2 * e + 1] = p * c + u * s;
                }
            };
            turn(x, d0);
            turn(y, d1);
        } else if (i < in_first) {
#pragma unroll
            for (int e = 0; e < C; ++e) {
                const float c = cos_t[d0 + e], s = sin_t[d0 + e], u = x[e], p = y[e];
                x[e] = u * c - p * s;
                y[e] = p * c + u * s;
            }
        }
        store16<E, C>(dst + d0, x);
        store16<E, C>(dst + d1, y);
    }
}

// Any D <= 256 and any strides: a workgroup takes one token, a wave one head at a time, lane l the elements l, l + 64, ...  A
// vector's elements and their partners are all read before any of it is written (the norm's sum waits for them), so it also runs in place.
template <typename E>
__global__ void __launch_bounds__(256) bh_qk_norm_rotary_any_kernel(RotaryArgs a) {
    extern __shared__ __attribute__((aligned(16))) float trig[];  // [2][rot / 2]
    __shared__ float vec[4][MAX_D];
    const int half = a.rot >> 1, lane = threadIdx.x & 63;
    const long long t = blockIdx.x;
    for (int j = threadIdx.x; j < half; j += 256) {
        float c, s;
        angle_of(position(a, t), a.inv_freq[j], c, s);
        trig[j] = c;
        trig[half + j] = s;
    }
    __syncthreads();
    for (int h = threadIdx.x >> 6; h < a.nq + a.nk; h += 4) {
        const bool is_q = h < a.nq;
        const E* src = is_q ? static_cast<const E*>(a.q) + t * a.q_tok + h * a.q_head
                            : static_cast<const E*>(a.k) + t * a.k_tok + (h - a.nq) * a.k_head;
        E* dst = is_q ? static_cast<E*>(a.q_out) + t * a.qo_tok + h * a.qo_head
                      : static_cast<E*>(a.k_out) + t * a.ko_tok + (h - a.nq) * a.ko_head;
        const void* w = is_q ? a.qw : a.kw;
        float x[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int d = lane + 64 * n;
            x[n] = d < a.dim ? (float)src[d] : 0.f;
        }
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int n = 0; n < 4; ++n) ss += x[n] * x[n];
            const float r = 1.0f / sqrtf(bh_group_sum(ss, 64) / (float)a.dim + a.eps);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int d = lane + 64 * n;
                if (d < a.dim) x[n] *= r * (a.w32 ? static_cast<const float*>(w)[d] : (float)static_cast<const E*>(w)[d]);
            }
        }
        // the partner of element d sits in another lane and step: by way of LDS, the wave's own (16 exchanges between lanes took a
        // third longer)
        float o[4];
        float* mine = vec[threadIdx.x >> 6];
#pragma unroll
        for (int n = 0; n < 4; ++n)
            if (lane + 64 * n < a.dim) mine[lane + 64 * n] = x[n];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int d = lane + 64 * n;
            o[n] = x[n];
            if (d >= a.rot) continue;
            const int j = a.interleaved ? d >> 1 : (d < half ? d : d - half);
            const int p = a.interleaved ? d ^ 1 : (d < half ? d + half : d - half);
            const bool first = a.interleaved ? !(d & 1) : d < half;
            const float other = mine[p];
            o[n] = first ? x[n] * trig[j] - other * trig[half + j] : x[n] * trig[j] + other * trig[half + j];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int d = lane + 64 * n;
            if (d < a.dim) dst[d] = (E)o[n];
        }
    }
}

// ---- key-value cache -------------------------------------------------------------------------------------------------------

struct CacheArgs {
    const void* src[2];        // write: keys, values
    void* dst[2];              // read: keys, values
    long long tok[2], head[2];  // their strides in elements
    void* codes[2];            // [pages][heads][page][dim]
    float* scale[2];           // [pages][heads][page], 8-bit caches
    const long long* slots;
    long long n_tokens, n_slots;
    int heads, dim, page_log2, lanes_log2;
};

// Where head h's vector of a slot starts in the cache, in vectors.
__device__ __forceinline__ long long vector_of(const CacheArgs& a, long long slot, int h) {
    const long long page = slot >> a.page_log2, offset = slot & ((1ll << a.page_log2) - 1);
    return (((page * a.heads + h) << a.page_log2) + offset);
}

// How a cache type holds a vector whose largest magnitude has the bits `most` (as of a non-negative fp32; beyond infinity's: a NaN).
// CODE 0 / 1: fp16 / bf16.  BH_I8: scale = amax / 127, at least the smallest normal number, so that the products with its reciprocal
// stay finite.  BH_E4M3: the least power of two with amax <= 448 * scale: scaling by it is exact, the code is one rounding.
// A vector that holds an infinity or a NaN gets the scale NaN and reads back as NaN, whole.
template <int CACHE>
__device__ __forceinline__ float scale_of(unsigned most) {
    if (most >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    const float amax = __uint_as_float(most);
    if (CACHE == BH_I8) return fmaxf(amax / 127.0f, 0x1p-126f);
    // amax = f * 2^e, 1 <= f < 2; 448 = 1.75 * 2^8.  A subnormal amax has e < -126 and takes the smallest scale as well
    const int e = (int)(most >> 23) - 127 - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
    return ldexpf(1.0f, e < -126 ? -126 : e);
}

// x / s to the nearest whole number, ties to even, of the exact quotient: the product with the rounded reciprocal is off by less
// than one, and x - n s is exact in one fma (both are multiples of 2^-25 s, and at most s), so its comparison with s / 2 decides.
__device__ __forceinline__ int int8_code(float x, float s, float inv) {
    float n = rintf(x * inv);
    const float r = 2.0f * fmaf(-n, s, x), m = fabsf(r);
    if (m > s || (m == s && ((int)n & 1))) n += r > 0.f ? 1.0f : -1.0f;
    return (int)n;
}

__device__ __forceinline__ unsigned pack4_int8(const float* x, float s, float inv) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (unsigned)(int8_code(x[i], s, inv) & 0xff) << (8 * i);
    return w;
}
__device__ __forceinline__ unsigned pack4_e4m3(const float* x, float inv) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, w, true);
}

__device__ __forceinline__ void unpack4_int8(unsigned w, float s, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)((int)(w << (24 - 8 * i)) >> 24) * s;
}
__device__ __forceinline__ void unpack4_e4m3(unsigned w, float s, float* x) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * s;
    x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * s;
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * s;
    x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * s;
}

template <int CACHE>
struct cache_elem {
    typedef unsigned char type;
};
template <>
struct cache_elem<BH_F16> {
    typedef _Float16 type;
};
template <>
struct cache_elem<BH_BF16> {
    typedef __bf16 type;
};

// C codes of a piece, in C / 4 words.
template <int CACHE, int C>
__device__ __forceinline__ void store_codes(unsigned char* p, const float (&x)[C], float s, float inv, bool good) {
    typedef unsigned words __attribute__((ext_vector_type(C / 4)));
    words w;
#pragma unroll
    for (int i = 0; i < C / 4; ++i) {
        unsigned c;
        if constexpr (CACHE == BH_I8)
            c = pack4_int8(x + 4 * i, s, inv);
        else
            c = pack4_e4m3(x + 4 * i, inv);
        w[i] = good ? c : 0;
    }
    *reinterpret_cast<words*>(p) = w;
}

// grid.y: 0 keys, 1 values.  A lane has a piece of 16 bytes of the row (C elements) at C i of either half of the vector: neighbouring lanes
// read and write next to each other on both sides (with one piece of 32 or 64 bytes a lane fp32 rows came at 3.8 TB/s).
template <typename E, int CACHE>
__global__ void __launch_bounds__(256) bh_kv_write_kernel(CacheArgs a) {
    typedef typename cache_elem<CACHE>::type T;
    constexpr int C = 16 / sizeof(E);
    const int kv = blockIdx.y, lanes = 1 << a.lanes_log2, i = threadIdx.x & (lanes - 1);
    const long long v = ((long long)blockIdx.x * 256 + threadIdx.x) >> a.lanes_log2;
    if (v >= a.n_tokens * a.heads) return;  // whole groups
    const long long t = v / a.heads;
    const int h = (int)(v - t * a.heads);
    const long long slot = a.slots[t];
    if (slot < 0 || slot >= a.n_slots) return;
    const int d0 = C * i, d1 = a.dim / 2 + C * i;
    const E* src = static_cast<const E*>(a.src[kv]) + t * a.tok[kv] + h * a.head[kv];
    const long long at = vector_of(a, slot, h);
    T* dst = static_cast<T*>(a.codes[kv]) + at * a.dim;
    const bool live = 2 * C * i < a.dim;
    float x[C] = {}, y[C] = {};
    if (live) {
        load16<E, C>(src + d0, x);
        load16<E, C>(src + d1, y);
    }
    if constexpr (CACHE == BH_F16 || CACHE == BH_BF16) {
        if (live) {
            store16<T, C>(dst + d0, x);
            store16<T, C>(dst + d1, y);
        }
    } else {
        unsigned most = 0;
#pragma unroll
        for (int e = 0; e < C; ++e) {
            const unsigned p = __float_as_uint(x[e]) & 0x7fffffffu, q = __float_as_uint(y[e]) & 0x7fffffffu;
            most = most > p ? most : p;
            most = most > q ? most : q;
        }
        const float s = scale_of<CACHE>(bh_group_umax(most, lanes));
        if (i == 0) a.scale[kv][at] = s;
        if (!live) return;
        const float inv = 1.0f / s;
        store_codes<CACHE, C>(dst + d0, x, s, inv, s == s);
        store_codes<CACHE, C>(dst + d1, y, s, inv, s == s);
    }
}

template <typename E, int CACHE>
__global__ void __launch_bounds__(256) bh_kv_write_any_kernel(CacheArgs a) {
    typedef typename cache_elem<CACHE>::type C;
    const int kv = blockIdx.y, lane = threadIdx.x & 63;
    const long long v = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (v >= a.n_tokens * a.heads) return;
    const long long t = v / a.heads;
    const int h = (int)(v - t * a.heads);
    const long long slot = a.slots[t];
    if (slot < 0 || slot >= a.n_slots) return;
    const E* src = static_cast<const E*>(a.src[kv]) + t * a.tok[kv] + h * a.head[kv];
    const long long at = vector_of(a, slot, h);
    C* dst = static_cast<C*>(a.codes[kv]) + at * a.dim;
    float x[4];
    unsigned most = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int d = lane + 64 * n;
        x[n] = d < a.dim ? (float)src[d] : 0.f;
        const unsigned p = __float_as_uint(x[n]) & 0x7fffffffu;
        most = most > p ? most : p;
    }
    float s = 1.f, inv = 1.f;
    bool good = true;
    if constexpr (CACHE == BH_I8 || CACHE == BH_E4M3) {
        s = scale_of<CACHE>(bh_group_umax(most, 64));
        if (lane == 0) a.scale[kv][at] = s;
        good = s == s;
        inv = 1.0f / s;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int d = lane + 64 * n;
        if (d >= a.dim) continue;
        if constexpr (CACHE == BH_I8)
            dst[d] = good ? (unsigned char)(int8_code(x[n], s, inv) & 0xff) : 0;
        else if constexpr (CACHE == BH_E4M3)
            dst[d] = good ? (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(x[n] * inv, 0.f, 0, false) & 0xff) : 0;
        else
            dst[d] = (C)x[n];
    }
}

template <int CACHE, int C>
__device__ __forceinline__ void load_codes(const unsigned char* p, float s, float (&x)[C]) {
    typedef unsigned words __attribute__((ext_vector_type(C / 4)));
    const words w = *reinterpret_cast<const words*>(p);
#pragma unroll
    for (int i = 0; i < C / 4; ++i) {
        if constexpr (CACHE == BH_I8)
            unpack4_int8(w[i], s, x + 4 * i);
        else
            unpack4_e4m3(w[i], s, x + 4 * i);
    }
}

template <typename E, int CACHE>
__global__ void __launch_bounds__(256) bh_kv_read_kernel(CacheArgs a) {
    typedef typename cache_elem<CACHE>::type T;
    constexpr int C = 16 / sizeof(E);
    const int kv = blockIdx.y, lanes = 1 << a.lanes_log2, i = threadIdx.x & (lanes - 1);
    const long long v = ((long long)blockIdx.x * 256 + threadIdx.x) >> a.lanes_log2;
    if (v >= a.n_tokens * a.heads || 2 * C * i >= a.dim) return;
    const long long t = v / a.heads;
    const int h = (int)(v - t * a.heads);
    const long long slot = a.slots[t];
    const int d0 = C * i, d1 = a.dim / 2 + C * i;
    E* dst = static_cast<E*>(a.dst[kv]) + t * a.tok[kv] + h * a.head[kv];
    float x[C] = {}, y[C] = {};
    if (slot >= 0 && slot < a.n_slots) {
        const long long at = vector_of(a, slot, h);
        const T* src = static_cast<const T*>(a.codes[kv]) + at * a.dim;
        if constexpr (CACHE == BH_F16 || CACHE == BH_BF16) {
            load16<T, C>(src + d0, x);
            load16<T, C>(src + d1, y);
        } else {
            const float s = a.scale[kv][at];
            load_codes<CACHE, C>(src + d0, s, x);
            load_codes<CACHE, C>(src + d1, s, y);
        }
    }
    store16<E, C>(dst + d0, x);
    store16<E, C>(dst + d1, y);
}

template <typename E, int CACHE>
__global__ void __launch_bounds__(256) bh_kv_read_any_kernel(CacheArgs a) {
    typedef typename cache_elem<CACHE>::type C;
    const int kv = blockIdx.y, lane = threadIdx.x & 63;
    const long long v = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (v >= a.n_tokens * a.heads) return;
    const long long t = v / a.heads;
    const int h = (int)(v - t * a.heads);
    const long long slot = a.slots[t];
    const bool there = slot >= 0 && slot < a.n_slots;
    E* dst = static_cast<E*>(a.dst[kv]) + t * a.tok[kv] + h * a.head[kv];
    const long long at = there ? vector_of(a, slot, h) : 0;
    const C* src = static_cast<const C*>(a.codes[kv]) + at * a.dim;
    float s = 1.f;
    if constexpr (CACHE == BH_I8 || CACHE == BH_E4M3) s = there ? a.scale[kv][at] : 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int d = lane + 64 * n;
        if (d >= a.dim) continue;
        float x = 0.f;
        if (there) {
            if constexpr (CACHE == BH_I8)
                x = (float)(signed char)src[d] * s;
            else if constexpr (CACHE == BH_E4M3)
                x = __builtin_amdgcn_cvt_f32_fp8((int)src[d], 0) * s;
            else
                x = (float)src[d];
        }
        dst[d] = (E)x;
    }
}

template <typename E, int CACHE>
void launch_cache(const CacheArgs& a, bool write, bool wide, hipStream_t st) {
    const long long vectors = a.n_tokens * a.heads;
    const dim3 grid((unsigned)(wide ? ((vectors << a.lanes_log2) + 255) / 256 : (vectors + 3) / 4), 2);
    if (write && wide)
        hipLaunchKernelGGL((bh_kv_write_kernel<E, CACHE>), grid, dim3(256), 0, st, a);
    else if (write)
        hipLaunchKernelGGL((bh_kv_write_any_kernel<E, CACHE>), grid, dim3(256), 0, st, a);
    else if (wide)
        hipLaunchKernelGGL((bh_kv_read_kernel<E, CACHE>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((bh_kv_read_any_kernel<E, CACHE>), grid, dim3(256), 0, st, a);
}

template <typename E>
void launch_cache_of(int cache, const CacheArgs& a, bool write, bool wide, hipStream_t st) {
    switch (cache) {
        case BH_F16: return launch_cache<E, BH_F16>(a, write, wide, st);
        case BH_BF16: return launch_cache<E, BH_BF16>(a, write, wide, st);
        case BH_I8: return launch_cache<E, BH_I8>(a, write, wide, st);
        default: return launch_cache<E, BH_E4M3>(a, write, wide, st);
    }
}

// Arguments that the cache's write and read share.
int cache_call(bool write, const void* const (&x)[2], const long long (&tok)[2], const long long (&head)[2], int32_t dtype,
               const int64_t* slots, int64_t n_tokens, int32_t n_heads, int32_t head_dim, void* const (&codes)[2], float* const (&scale)[2],
               int32_t cache_dtype, int64_t n_pages, int32_t page_size, hipStream_t st) {
    if (!bh_is_float(dtype)) return bh_fail(BH_EINVAL, "bad dtype %d (fp16, bf16 or fp32)", dtype);
    if (cache_dtype == BH_F32 || !bh_dtype_size(cache_dtype)) return bh_fail(BH_EINVAL, "bad cache dtype %d (fp16, bf16, int8 or e4m3)", cache_dtype);
    const bool scaled = bh_dtype_size(cache_dtype) == 1;
    if (n_tokens < 0 || n_heads <= 0 || n_pages <= 0) return bh_fail(BH_EINVAL, "bad sizes");
    if (head_dim < 1 || head_dim > MAX_D) return bh_fail(BH_EUNSUPPORTED, "head_dim %d (1..%d)", head_dim, MAX_D);
    if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1)))
        return bh_fail(BH_EUNSUPPORTED, "page_size %d (a power of two, 8..1024)", page_size);
    if (n_tokens == 0) return BH_OK;
    if (!x[0] || !x[1] || !slots || !codes[0] || !codes[1]) return bh_fail(BH_EINVAL, "null buffer");
    if (scaled && (!scale[0] || !scale[1])) return bh_fail(BH_EINVAL, "an 8-bit cache needs the scales of keys and values");
    CacheArgs a{};
    const long long per16 = 16 / (long long)bh_dtype_size(dtype);
    bool wide = head_dim % (2 * per16) == 0;
    for (int kv = 0; kv < 2; ++kv) {
        a.src[kv] = x[kv];
        a.dst[kv] = const_cast<void*>(x[kv]);
        a.tok[kv] = tok[kv];
        a.head[kv] = head[kv];
        a.codes[kv] = codes[kv];
        a.scale[kv] = scaled ? scale[kv] : nullptr;
        wide = wide && bh_aligned16(x[kv]) && bh_aligned16(codes[kv]) && tok[kv] % per16 == 0 && head[kv] % per16 == 0;
    }
    a.slots = reinterpret_cast<const long long*>(slots);
    a.n_tokens = n_tokens;
    a.n_slots = (long long)n_pages * page_size;
    a.heads = n_heads;
    a.dim = head_dim;
    a.page_log2 = bh_ceil_log2(page_size);
    a.lanes_log2 = wide ? bh_ceil_log2((int)(head_dim / (2 * per16))) : 0;
    // (2^24 workgroups of 256 threads are as many as a grid's first dimension can have)
    if (n_tokens > (1ll << 40) / n_heads || ((n_tokens * n_heads) << (wide ? a.lanes_log2 : 6)) >> 32)
        return bh_fail(BH_EUNSUPPORTED, "too many head vectors in one call");
    if (dtype == BH_F16)
        launch_cache_of<_Float16>(cache_dtype, a, write, wide, st);
    else if (dtype == BH_BF16)
        launch_cache_of<__bf16>(cache_dtype, a, write, wide, st);
    else
        launch_cache_of<float>(cache_dtype, a, write, wide, st);
    BH_HIP_TRY(hipGetLastError());
    return BH_OK;
}

template <typename E>
void launch_rotary(const RotaryArgs& a, bool wide, hipStream_t st) {
    const size_t lds = (size_t)(wide ? a.tb : 1) * a.rot * sizeof(float);
    if (wide)
        hipLaunchKernelGGL((bh_qk_norm_rotary_kernel<E>), dim3((unsigned)((a.n_tokens + a.tb - 1) / a.tb)), dim3(256), lds, st, a);
    else
        hipLaunchKernelGGL((bh_qk_norm_rotary_any_kernel<E>), dim3((unsigned)a.n_tokens), dim3(256), lds, st, a);
}

}  // namespace

extern "C" {

int bh_op_qk_norm_rotary(const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok, int64_t qo_head, const void* k,
                         int64_t k_tok, int64_t k_head, void* k_out, int64_t ko_tok, int64_t ko_head, int32_t dtype, int64_t n_tokens,
                         int32_t n_q_heads, int32_t n_k_heads, int32_t head_dim, int32_t rotary_dim, const void* positions,
                         int32_t positions_i64, const double* inv_freq, const void* q_weight, const void* k_weight, int32_t weight_dtype,
                         float eps, int32_t interleaved, void* stream) {
    if (!bh_is_float(dtype)) return bh_fail(BH_EINVAL, "bad dtype %d (fp16, bf16 or fp32)", dtype);
    if ((q_weight || k_weight) && weight_dtype != dtype && weight_dtype != BH_F32)
        return bh_fail(BH_EINVAL, "bad weight dtype %d (the heads' own or fp32)", weight_dtype);
    if (n_tokens < 0 || n_q_heads <= 0 || n_k_heads <= 0 || !(eps >= 0.f)) return bh_fail(BH_EINVAL, "bad sizes or eps");
    if (head_dim < 1 || head_dim > MAX_D) return bh_fail(BH_EUNSUPPORTED, "head_dim %d (1..%d)", head_dim, MAX_D);
    if (rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1))
        return bh_fail(BH_EINVAL, "rotary_dim %d (even, 0..head_dim %d)", rotary_dim, head_dim);
    if (n_tokens > 0x7fffffffll || n_q_heads > 65535 || n_k_heads > 65535) return bh_fail(BH_EUNSUPPORTED, "too many tokens or heads");
    if (n_tokens == 0) return BH_OK;
    if (!q || !q_out || !k || !k_out || (rotary_dim && (!positions || !inv_freq))) return bh_fail(BH_EINVAL, "null buffer");
    const long long per16 = 16 / (long long)bh_dtype_size(dtype);
    const bool wide = head_dim % (2 * per16) == 0 && rotary_dim % (2 * per16) == 0 && bh_aligned16(q) && bh_aligned16(k) && bh_aligned16(q_out) &&
                      bh_aligned16(k_out) && bh_aligned16(q_weight) && bh_aligned16(k_weight) &&
                      (q_tok | q_head | qo_tok | qo_head | k_tok | k_head | ko_tok | ko_head) % per16 == 0;
    RotaryArgs a{};
    a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
    a.q_tok = q_tok, a.q_head = q_head, a.qo_tok = qo_tok, a.qo_head = qo_head;
    a.k_tok = k_tok, a.k_head = k_head, a.ko_tok = ko_tok, a.ko_head = ko_head;
    a.qw = q_weight, a.kw = k_weight;
    a.pos = positions, a.pos64 = positions_i64 != 0, a.inv_freq = inv_freq;
    a.n_tokens = n_tokens, a.nq = n_q_heads, a.nk = n_k_heads, a.dim = head_dim, a.rot = rotary_dim;
    a.w32 = weight_dtype == BH_F32, a.interleaved = interleaved != 0, a.eps = eps;
    a.lanes_log2 = wide ? bh_ceil_log2((int)(head_dim / (2 * per16))) : 0;
    // tokens of a workgroup: enough for two steps of its 256 threads where a token has few heads; the sines stay within 16 KiB of LDS
    const int lanes = (n_q_heads + n_k_heads) << a.lanes_log2;
    a.tb = lanes >= 512 ? 1 : 512 / lanes;
    if (n_tokens / (wide ? a.tb : 1) >= (1 << 24) - 1) return bh_fail(BH_EUNSUPPORTED, "too many tokens in one call");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == BH_F16)
        launch_rotary<_Float16>(a, wide, st);
    else if (dtype == BH_BF16)
        launch_rotary<__bf16>(a, wide, st);
    else
        launch_rotary<float>(a, wide, st);
    BH_HIP_TRY(hipGetLastError());
    return BH_OK;
}

int bh_op_kv_write(const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok, int64_t v_head, int32_t dtype,
                   const int64_t* slots, int64_t n_tokens, int32_t n_heads, int32_t head_dim, void* k_cache, void* v_cache, float* k_scale,
                   float* v_scale, int32_t cache_dtype, int64_t n_pages, int32_t page_size, void* stream) {
    return cache_call(true, {k, v}, {k_tok, v_tok}, {k_head, v_head}, dtype, slots, n_tokens, n_heads, head_dim, {k_cache, v_cache},
                      {k_scale, v_scale}, cache_dtype, n_pages, page_size, static_cast<hipStream_t>(stream));
}

int bh_op_kv_read(void* k, int64_t k_tok, int64_t k_head, void* v, int64_t v_tok, int64_t v_head, int32_t dtype, const int64_t* slots,
                  int64_t n_tokens, int32_t n_heads, int32_t head_dim, const void* k_cache, const void* v_cache, const float* k_scale,
                  const float* v_scale, int32_t cache_dtype, int64_t n_pages, int32_t page_size, void* stream) {
    return cache_call(false, {k, v}, {k_tok, v_tok}, {k_head, v_head}, dtype, slots, n_tokens, n_heads, head_dim,
                      {const_cast<void*>(k_cache), const_cast<void*>(v_cache)}, {const_cast<float*>(k_scale), const_cast<float*>(v_scale)},
                      cache_dtype, n_pages, page_size, static_cast<hipStream_t>(stream));
}

}  // extern "C"
