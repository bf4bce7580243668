// The 8-bit decode cache: e4m3 codes in a ring with one fp32 power-of-two scale
// per (block of slots, head); shared by the write / read kernels (kv8.hip) and
// the decode attention over it (attn_decode_kv8.hip).
//
// Ring of S_ring = n_meta + ctx slots per (b, h): metadata position -n_meta + s
// in slot s < n_meta, the token at position p >= 0 in slot n_meta + p % ctx. A
// row whose newest position is `last` holds S = n_meta + min(last + 1, ctx)
// rows (none if that is <= 0: the row is not in use).
#pragma once
#include "common.h"

constexpr int KV8_MAX_HS = 128;

// rows in the window whose newest position is `last`
__host__ __device__ __forceinline__ int kv8_window(int64_t last, int n_meta, int ctx) {
    const int64_t n = last + 1 < ctx ? last + 1 : ctx;
    return n + n_meta > 0 ? (int)(n + n_meta) : 0;
}
// a % n for a >= 0: by a 32-bit division wherever that does (the 64-bit one is a
// long scalar sequence at the head of every workgroup)
__host__ __device__ __forceinline__ int kv8_mod(int64_t a, int n) {
    return a >> 32 ? (int)(a % n) : (int)((uint32_t)a % (uint32_t)n);
}
// ring offset of the window's first token (0 until the ring wraps)
__host__ __device__ __forceinline__ int kv8_first(int64_t last, int ctx) {
    return last + 1 > ctx ? kv8_mod(last + 1, ctx) : 0;
}
__host__ __device__ __forceinline__ bool kv8_block_ok(int64_t block) {
    return block == 16 || block == 32 || block == 64 || block == 128;
}

// four e4m3 codes -> fp32 (exact)
__device__ __forceinline__ f32x4 kv8_dec4(uint32_t c) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    return (f32x4){a[0], a[1], b[0], b[1]};
}
// four fp32 in [-448, 448] (or NaN) -> e4m3, nearest even
__device__ __forceinline__ uint32_t kv8_enc4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// exponent e >= -126 of the smallest power of two 2^e with amax <= 448 * 2^e
// (amax finite, >= 0): 448 = 1.75 * 2^8
__device__ __forceinline__ int kv8_scale_exp(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
    return e < -126 ? -126 : e;  // also for a zero or subnormal amax
}
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
