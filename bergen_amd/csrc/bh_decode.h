// bh_decode.h — what the operators of a decoding step share (decode_ops.hip, paged_attention.hip, token_logprobs.hip): element
// types, group reductions.
#pragma once
#include "bh_device.h"
#include "bh_host.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

inline size_t bh_dtype_size(int32_t dtype) {
    return dtype == BH_F32 ? 4 : dtype == BH_F16 || dtype == BH_BF16 ? 2 : dtype == BH_I8 || dtype == BH_E4M3 ? 1 : 0;
}
inline bool bh_is_float(int32_t dtype) { return dtype == BH_F16 || dtype == BH_BF16 || dtype == BH_F32; }

inline bool bh_aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 8 consecutive numbers at p (16-byte aligned).
__device__ __forceinline__ void bh_load8(const float* p, float (&x)[8]) {
    const floatx4 a = *reinterpret_cast<const floatx4*>(p), b = *reinterpret_cast<const floatx4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
    }
}

// Reductions over aligned groups of `size` lanes (a power of two).
__device__ __forceinline__ float bh_group_sum(float v, int size) {
    for (int m = 1; m < size; m <<= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ unsigned bh_group_umax(unsigned v, int size) {
    for (int m = 1; m < size; m <<= 1) {
        const unsigned o = __shfl_xor(v, m);
        v = v > o ? v : o;
    }
    return v;
}

// Smallest power of two >= n, as its exponent (n >= 1).
inline int bh_ceil_log2(int n) {
    int s = 0;
    while ((1 << s) < n) ++s;
    return s;
}
