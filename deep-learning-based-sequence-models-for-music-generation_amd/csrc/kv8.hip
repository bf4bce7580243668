// Writing the 8-bit decode cache and reading it back (kv8.h; the keys and
// values that models/transformer/model_transformer.py:54-82 recomputes for the
// whole window per generated token, scripts/generate.py:26-31).
//
// Write. T new rows at positions p0 .. p0+T-1 of a row of the batch. A block of
// slots is touched when one of its slots takes a new row; its contents after
// the write are C(r) = x(r) for new rows and code(r) * scale for the rows that
// stay, its scale is the smallest power of two 2^e (e >= -126) with
// |C| <= 448 * 2^e over its finite contents, and code(r) = e4m3(C(r) / 2^e):
// a function of the block's contents alone, so the order of writes does not
// matter and a scale falls again once a large row has been overwritten. A power
// of two costs no accuracy against amax / 448 (e4m3 keeps 3 bits of mantissa
// down to 2^-6 of the scale, 16 octaves below its largest value) and makes the
// re-coding of the rows that stay exact, except where a code falls below 2^-6
// of the new scale: each element is rounded once, not once per step.
// One workgroup per (touched block, K | V, head, row of the batch), the block's
// contents in registers between the maximum and the store, 8 values per lane
// and chunk.
//
// Read. Elementwise: 8 codes per lane, in window order (oldest first).
#include "kv8.h"

namespace {

constexpr int NT = 256;

struct WriteArgs {
    const void* src[2];
    uint8_t* code[2];
    float* scale[2];
    int64_t sb, st;  // strides of src (elements): row of the batch, token; heads are hs apart
    const int64_t* pos;
    int64_t pos_stride, T;
    int H, hs, S_ring, n_meta, block, nblk, nb, all, vec;
};

__device__ __forceinline__ void load8(float* v, const bf16* p, int vec) {
    if (vec) {
        const bf16x8 x = *(const bf16x8*)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)p[e];
    }
}
__device__ __forceinline__ void load8(float* v, const float* p, int vec) {
    if (vec) {
        const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p[e];
    }
}

// +-448 for what lies outside (infinities too); NaN stays
__device__ __forceinline__ float sat(float x) { return x > 448.f ? 448.f : (x < -448.f ? -448.f : x); }

template <typename T, int NC>
__global__ __launch_bounds__(NT) void kv8_write_kernel(WriteArgs a) {
    __shared__ float red[NT / 64];
    const int tid = threadIdx.x;
    int id = blockIdx.x;
    const int i = id % a.nb;
    id /= a.nb;
    const int kv = id & 1;
    id >>= 1;
    const int h = id % a.H;
    const int64_t b = id / a.H;
    const int ctx = a.S_ring - a.n_meta;
    const int64_t p0 = a.pos[b * a.pos_stride], last = p0 + a.T - 1;
    if (p0 < -a.n_meta) return;  // the row is not in use (uniform)
    // the i-th touched block: from the first new row's slot, round the ring
    int blk = i;
    if (!a.all) {
        const int s = p0 < 0 ? (int)p0 + a.n_meta : a.n_meta + kv8_mod(p0, ctx);
        blk = s / a.block + i;
        if (blk >= a.nblk) blk += a.n_meta / a.block - a.nblk;
    }
    const int s0 = blk * a.block, cpr = a.hs >> 3, rows = min(a.block, a.S_ring - s0), n = rows * cpr;
    const int lm = last >= 0 ? kv8_mod(last, ctx) : 0;
    uint8_t* code = a.code[kv] + ((b * a.H + h) * a.S_ring + s0) * a.hs;
    float* scale = a.scale[kv] + (b * a.H + h) * a.nblk + blk;
    const T* src = (const T*)a.src[kv] + b * a.sb + (int64_t)h * a.hs;
    const float s_old = *scale;

    float v[NC][8];
    int kind[NC];  // 0: no row there, 1: stays, 2: new
    float m = 0.f;
    bool any = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int q = c * NT + tid;
        kind[c] = 0;
        if (q < n) {
            const int r = q / cpr, s = s0 + r;
            int64_t t;  // index of the new token in this slot (negative: an older one)
            bool there;
            if (s < a.n_meta) {
                t = (int64_t)(s - a.n_meta) - p0;
                there = s - a.n_meta <= last;
            } else {
                int d = lm - (s - a.n_meta);  // how far behind `last` the slot's position is
                d += d < 0 ? ctx : 0;
                t = a.T - 1 - d;
                there = d <= last;
            }
            kind[c] = !there ? 0 : (t >= 0 ? 2 : 1);
            if (kind[c] == 2) {
                load8(v[c], src + t * a.st + (q - r * cpr) * 8, a.vec);
            } else if (kind[c] == 1) {
                const uint2 w = *(const uint2*)(code + q * 8);
                const f32x4 lo = kv8_dec4(w.x), hi = kv8_dec4(w.y);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[c][e] = lo[e] * s_old, v[c][4 + e] = hi[e] * s_old;
            }
            any |= kind[c] == 2;
            if (kind[c]) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = fabsf(v[c][e]);
                    m = x <= 3.402823466e38f ? fmaxf(m, x) : m;  // infinities saturate, NaN stays NaN
                }
            }
        }
    }
    m = wave_max(m);
    if ((tid & 63) == 0) red[tid >> 6] = m;
    if (!__syncthreads_or(any)) return;  // no new row in this block (uniform)
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const int e = kv8_scale_exp(m);
    const float s_new = kv8_pow2(e), inv = kv8_pow2(-e);
    if (tid == 0) *scale = s_new;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (kind[c] == 2 || (kind[c] == 1 && s_new != s_old)) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = sat(v[c][k] * inv);
            *(uint2*)(code + (c * NT + tid) * 8) =
                make_uint2(kv8_enc4(y[0], y[1], y[2], y[3]), kv8_enc4(y[4], y[5], y[6], y[7]));
        }
    }
}

struct ReadArgs {
    const uint8_t* code[2];
    const float* scale[2];
    void* out[2];
    const int64_t* pos;
    int64_t pos_stride, total;  // 8-value chunks of one output
    int H, hs, S_ring, n_meta, block, nblk, first, n;
};

__device__ __forceinline__ void put8(bf16* p, f32x4 a, f32x4 b) {
    *(bf16x8*)p = (bf16x8){(bf16)a[0], (bf16)a[1], (bf16)a[2], (bf16)a[3], (bf16)b[0], (bf16)b[1], (bf16)b[2], (bf16)b[3]};
}
__device__ __forceinline__ void put8(float* p, f32x4 a, f32x4 b) {
    *(f32x4*)p = a;
    *(f32x4*)(p + 4) = b;
}

// grid: (chunks of one (b, h)'s rows, K | V x head, row of the batch)
template <typename T>
__global__ __launch_bounds__(NT) void kv8_read_kernel(ReadArgs a) {
    const int h = blockIdx.y >> 1, kv = blockIdx.y & 1;
    const int64_t b = blockIdx.z;
    const int cpr = a.hs >> 3, ctx = a.S_ring - a.n_meta;
    const int64_t q = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (q >= (int64_t)a.n * cpr) return;
    const int r = (int)(q / cpr), c = (int)(q - (int64_t)r * cpr) * 8, w = a.first + r;
    const int64_t last = a.pos[b * a.pos_stride];
    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    if (w < kv8_window(last, a.n_meta, ctx)) {
        int s = w;
        if (w >= a.n_meta) {
            s += kv8_first(last, ctx);
            s -= s >= a.S_ring ? ctx : 0;
        }
        const int64_t bh = b * a.H + h;
        const uint2 x = *(const uint2*)(a.code[kv] + (bh * a.S_ring + s) * a.hs + c);
        const float f = a.scale[kv][bh * a.nblk + s / a.block];
        lo = kv8_dec4(x.x) * f;
        hi = kv8_dec4(x.y) * f;
    }
    put8((T*)a.out[kv] + ((b * a.H + h) * a.n + r) * a.hs + c, lo, hi);
}

int check_cache(const char* fn, const void* kc, const float* ks, const void* vc, const float* vs, int64_t B, int64_t H,
                int64_t hs, int64_t S_ring, int64_t n_meta, int64_t block, const int64_t* pos, int64_t pos_stride) {
    MSQ_CHECK_ARG(kc && ks && vc && vs && pos, "%s: null pointer", fn);
    MSQ_CHECK_ARG(hs > 0 && hs <= KV8_MAX_HS && hs % 8 == 0, "%s: head size %lld (8 | hs <= %d)", fn, (long long)hs,
                  KV8_MAX_HS);
    MSQ_CHECK_ARG(B > 0 && B <= 65535 && H > 0 && H <= 32767 && n_meta >= 0 && S_ring > n_meta && S_ring <= (1 << 30),
                  "%s: bad sizes (B %lld, H %lld, ring %lld, metadata %lld)", fn, (long long)B, (long long)H,
                  (long long)S_ring, (long long)n_meta);
    MSQ_CHECK_ARG(kv8_block_ok(block), "%s: block %lld (16, 32, 64 or 128 slots)", fn, (long long)block);
    MSQ_CHECK_ARG(pos_stride == 0 || pos_stride == 1, "%s: pos_stride %lld (0 or 1)", fn, (long long)pos_stride);
    MSQ_CHECK_ARG((((uintptr_t)kc | (uintptr_t)vc) & 7) == 0, "%s: the cache is not 8-byte aligned", fn);
    return MSQ_OK;
}

template <typename T>
void launch_write(const WriteArgs& a, unsigned grid, int nc, hipStream_t s) {
    if (nc <= 1) hipLaunchKernelGGL((kv8_write_kernel<T, 1>), dim3(grid), dim3(NT), 0, s, a);
    else if (nc <= 2) hipLaunchKernelGGL((kv8_write_kernel<T, 2>), dim3(grid), dim3(NT), 0, s, a);
    else if (nc <= 4) hipLaunchKernelGGL((kv8_write_kernel<T, 4>), dim3(grid), dim3(NT), 0, s, a);
    else hipLaunchKernelGGL((kv8_write_kernel<T, 8>), dim3(grid), dim3(NT), 0, s, a);
}

}  // namespace

extern "C" int64_t msq_kv8_blocks(int64_t S_ring, int64_t block) {
    return kv8_block_ok(block) && S_ring > 0 ? (S_ring + block - 1) / block : -1;
}

extern "C" int msq_kv8_write(int dtype, void* kc, float* ks, void* vc, float* vs, const void* k, const void* v,
                             int64_t ld_b, int64_t ld_t, int64_t B, int64_t T, int64_t H, int64_t hs, int64_t S_ring,
                             int64_t n_meta, int64_t block, const int64_t* pos, int64_t pos_stride, void* stream) {
    const int rc = check_cache("msq_kv8_write", kc, ks, vc, vs, B, H, hs, S_ring, n_meta, block, pos, pos_stride);
    if (rc) return rc;
    MSQ_CHECK_ARG(k && v, "msq_kv8_write: null pointer");
    MSQ_CHECK_ARG(dtype == MSQ_BF16 || dtype == MSQ_F32, "msq_kv8_write: dtype %d", dtype);
    MSQ_CHECK_ARG(T > 0 && T <= (1 << 30), "msq_kv8_write: %lld new rows", (long long)T);
    MSQ_CHECK_ARG(ld_b >= 0 && ld_t >= 0, "msq_kv8_write: negative strides");
    WriteArgs a;
    a.src[0] = k; a.src[1] = v;
    a.code[0] = (uint8_t*)kc; a.code[1] = (uint8_t*)vc;
    a.scale[0] = ks; a.scale[1] = vs;
    a.sb = ld_b; a.st = ld_t;
    a.pos = pos; a.pos_stride = pos_stride;
    a.T = T;
    a.H = (int)H; a.hs = (int)hs; a.S_ring = (int)S_ring; a.n_meta = (int)n_meta; a.block = (int)block;
    a.nblk = (int)msq_kv8_blocks(S_ring, block);
    // T consecutive slots, split at most once by the ring's end, touch at most
    // T / block + 4 blocks; where that could reach round the ring (T >= ctx always
    // does) every block of it is visited, once
    const int64_t nb = T == 1 ? 1 : T / block + 4;
    a.all = nb >= a.nblk - n_meta / block;
    a.nb = a.all ? a.nblk : (int)nb;
    a.vec = ((ld_b | ld_t) & 7) == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    const int64_t grid = (int64_t)a.nb * 2 * H * B;
    MSQ_CHECK_ARG(grid < (1ll << 31), "msq_kv8_write: %lld workgroups", (long long)grid);
    const int nc = (int)((block * (hs / 8) + NT - 1) / NT);
    if (dtype == MSQ_BF16) launch_write<bf16>(a, (unsigned)grid, nc, (hipStream_t)stream);
    else launch_write<float>(a, (unsigned)grid, nc, (hipStream_t)stream);
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}

extern "C" int msq_kv8_read(int dtype, void* k, void* v, const void* kc, const float* ks, const void* vc,
                            const float* vs, int64_t B, int64_t H, int64_t hs, int64_t S_ring, int64_t n_meta,
                            int64_t block, const int64_t* pos, int64_t pos_stride, int64_t first, int64_t rows,
                            void* stream) {
    const int rc = check_cache("msq_kv8_read", kc, ks, vc, vs, B, H, hs, S_ring, n_meta, block, pos, pos_stride);
    if (rc) return rc;
    MSQ_CHECK_ARG(k && v, "msq_kv8_read: null pointer");
    MSQ_CHECK_ARG(dtype == MSQ_BF16 || dtype == MSQ_F32, "msq_kv8_read: dtype %d", dtype);
    MSQ_CHECK_ARG(first >= 0 && rows > 0 && first + rows <= S_ring, "msq_kv8_read: rows %lld .. %lld of a ring of %lld",
                  (long long)first, (long long)(first + rows), (long long)S_ring);
    MSQ_CHECK_ARG((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "msq_kv8_read: the outputs are not 16-byte aligned");
    ReadArgs a;
    a.code[0] = (const uint8_t*)kc; a.code[1] = (const uint8_t*)vc;
    a.scale[0] = ks; a.scale[1] = vs;
    a.out[0] = k; a.out[1] = v;
    a.pos = pos; a.pos_stride = pos_stride;
    a.H = (int)H; a.hs = (int)hs; a.S_ring = (int)S_ring; a.n_meta = (int)n_meta; a.block = (int)block;
    a.nblk = (int)msq_kv8_blocks(S_ring, block);
    a.first = (int)first; a.n = (int)rows;
    a.total = rows * (hs / 8);
    const dim3 grid((unsigned)((a.total + NT - 1) / NT), (unsigned)(2 * H), (unsigned)B);
    if (dtype == MSQ_BF16) hipLaunchKernelGGL(kv8_read_kernel<bf16>, grid, dim3(NT), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(kv8_read_kernel<float>, grid, dim3(NT), 0, (hipStream_t)stream, a);
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}
