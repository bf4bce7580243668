// Writing the 8-bit decode cache and reading it back (kv8.h; the keys and
// values that models/transformer/model_transformer.py:54-82 recomputes for the
// whole window per generated token, scripts/generate.py:26-31).
//
// Write. T new rows at positions p0 .. p0+T-1 of a row of the batch. A block of
// slots is touched when one of its slots takes a new row; its contents after
// the write are C(r) = x(r) for new rows and code(r) * scale for the rows that
// stay, its scale is the smallest power of two 2^e (e >= -126) with
// |C| <= 448 * 2^e over its finite contents, and code(r) = e4m3(C(r) / 2^e). The
// scale is a function of C alone and falls again once a large row has been
// overwritten. A power of two costs no accuracy against amax / 448 (e4m3 keeps 3
// bits of mantissa down to 2^-6 of the scale, 15 octaves below its largest value)
// and makes the re-coding of the rows that stay exact, except where a code falls
// below 2^-6 of the new scale and is rounded again, to a multiple of 2^-9 of it;
// what that takes does not come back when the scale falls. Only a scale above
// all those the block had before can do it, and each is at least twice the last:
// an element is off by at most 2^-4 |x| + 2^-9 of the largest scale since.
// One workgroup per (touched block, K | V, head, row of the batch), the block's
// contents in registers between the maximum and the store, 8 values per lane
// and chunk.
//
// Read. Elementwise: 8 (fp32: 4) codes per lane and pass, in window order (oldest first).
// Both are bound by their bytes; what is read or written once goes past the caches
// (a prompt of 32 x 2054 rows x 8 heads of 128: 82 us without, 71 us with that).
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

// 8 consecutive values as loaded: 16 bytes of bf16, 32 of fp32
template <typename T> struct Raw8 {
    static constexpr int W = sizeof(T) / 2;
    u32x4 w[W];
    __device__ __forceinline__ void load(const T* p, int vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = __builtin_nontemporal_load((const u32x4*)p + i);
        } else {
            union { u32x4 u[W]; T t[8]; } r;
#pragma unroll
            for (int e = 0; e < 8; ++e) r.t[e] = p[e];
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = r.u[i];
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (W == 2) return __uint_as_float(w[e >> 2][e & 3]);
        return __uint_as_float(e & 1 ? w[0][e >> 1] & 0xffff0000u : w[0][e >> 1] << 16);
    }
};
__device__ __forceinline__ float code8(uint2 w, int e) { return kv8_dec4(e & 4 ? w.y : w.x)[e & 3]; }
// NaN does not count, infinities only with finite = false
__device__ __forceinline__ float abs_max(float m, float x, bool finite) {
    x = fabsf(x);
    return finite && !(x <= 3.402823466e38f) ? m : fmaxf(m, x);
}

// +-top for what lies outside (infinities too); NaN stays
__device__ __forceinline__ float sat(float x, float top) { return x > top ? top : (x < -top ? -top : x); }

template <typename T, int NC>
__global__ __launch_bounds__(NT) void kv8_write_kernel(WriteArgs a) {
    __shared__ float red[NT / 64];
    const int tid = threadIdx.x;
    int id = blockIdx.x;
    const int h = id % a.H;  // the heads of a token lie side by side
    id /= a.H;
    const int kv = id & 1;
    id >>= 1;
    const int i = id % a.nb;
    const int64_t b = id / a.nb;
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
    const int s0 = blk * a.block, cpr = a.hs >> 3, rpp = NT / cpr, rows = min(a.block, a.S_ring - s0);
    const int row = tid / cpr, col = (tid - row * cpr) * 8;  // of each pass over rpp rows
    const int lm = last >= 0 ? kv8_mod(last, ctx) : 0;
    uint8_t* code = a.code[kv] + ((b * a.H + h) * a.S_ring + s0) * a.hs + col;
    float* scale = a.scale[kv] + (b * a.H + h) * a.nblk + blk;
    const T* src = (const T*)a.src[kv] + b * a.sb + (int64_t)h * a.hs + col;
    const float s_old = *scale;

    Raw8<T> v[NC];   // new rows
    uint2 old[NC];   // rows that stay
    int kind[NC];    // 0: no row there, 1: stays, 2: new
    bool any = false, stay = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int r = c * rpp + row, s = s0 + r;
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
        kind[c] = row >= rpp || r >= rows || !there ? 0 : (t >= 0 ? 2 : 1);
        any |= kind[c] == 2;
        stay |= kind[c] == 1;
        if (kind[c] == 2) v[c].load(src + t * a.st, a.vec);
    }
    stay = __any(stay);  // (uniform over the wave)
    if (stay) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (kind[c] == 1) old[c] = *(const uint2*)(code + (c * rpp + row) * a.hs);
    }
    auto block_max = [&](bool finite) {
        float m = 0.f;
        if (stay) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (kind[c] == 1)
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = abs_max(m, code8(old[c], e) * s_old, finite);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (kind[c] == 2)
#pragma unroll
                for (int e = 0; e < 8; ++e) m = abs_max(m, v[c].get(e), finite);
        m = wave_max(m);
        if ((tid & 63) == 0) red[tid >> 6] = m;
        any = __syncthreads_or(any);
        return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    };
    float m = block_max(false);
    if (!any) return;  // no new row in this block (uniform)
    const bool wild = m == INFINITY;  // (uniform) else no value lies outside +-448 of the scale
    if (wild) {
        __syncthreads();
        m = block_max(true);
    }
    const int e = kv8_scale_exp(m);
    const float s_new = kv8_pow2(e), inv = kv8_pow2(-e);
    // at the largest scale the code 256 stands for 2^128, which would come back as an infinity: 240 is
    // no further than 2^-4 from any finite value there
    const float top = e == 120 ? 240.f : 448.f;
    const bool clip = wild || e == 120;  // (uniform)
    if (tid == 0) *scale = s_new;
    const bool recode = s_new != s_old;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (kind[c] == 2 || (stay && kind[c] == 1 && recode)) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = kind[c] == 2 ? v[c].get(k) * inv : code8(old[c], k) * s_old * inv;
            if (clip)
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = sat(y[k], top);
            const uint64_t lo = kv8_enc4(y[0], y[1], y[2], y[3]), hi = kv8_enc4(y[4], y[5], y[6], y[7]);
            __builtin_nontemporal_store(lo | hi << 32, (uint64_t*)(code + (c * rpp + row) * a.hs));
        }
    }
}

struct ReadArgs {
    const uint8_t* code[2];
    const float* scale[2];
    void* out[2];
    const int64_t* pos;
    int64_t pos_stride;
    int H, hs, S_ring, n_meta, block_log2, nblk, first, n;
};
constexpr int READ_PASSES = 2;  // rows of a workgroup, in units of those that its lanes take at once
                                // (a window of 32 x 2054 rows x 8 heads of 128: 77, 64, 68 us for 1, 2, 4)

// 16 bytes of values per lane and store, so that a wave's store covers whole lines
template <typename T> struct Out;
template <> struct Out<bf16> {
    static constexpr int N = 8;
    typedef uint64_t code;
    static __device__ __forceinline__ void put(bf16* p, code x, float f) {
        const f32x4 a = kv8_dec4((uint32_t)x) * f, b = kv8_dec4((uint32_t)(x >> 32)) * f;
        union { bf16x8 v; u32x4 u; } r;
        r.v = (bf16x8){(bf16)a[0], (bf16)a[1], (bf16)a[2], (bf16)a[3], (bf16)b[0], (bf16)b[1], (bf16)b[2], (bf16)b[3]};
        __builtin_nontemporal_store(r.u, (u32x4*)p);
    }
};
template <> struct Out<float> {
    static constexpr int N = 4;
    typedef uint32_t code;
    static __device__ __forceinline__ void put(float* p, code x, float f) {
        __builtin_nontemporal_store(kv8_dec4(x) * f, (f32x4*)p);
    }
};

// grid: (groups of rows, K | V x head, row of the batch)
template <typename T>
__global__ __launch_bounds__(NT) void kv8_read_kernel(ReadArgs a) {
    typedef typename Out<T>::code code_t;
    const int h = blockIdx.y >> 1, kv = blockIdx.y & 1;
    const int64_t b = blockIdx.z, bh = b * a.H + h;
    const int cpr = a.hs / Out<T>::N, ctx = a.S_ring - a.n_meta, rpp = NT / cpr;  // lanes of a row, rows per pass
    const int row = threadIdx.x / cpr, c = (threadIdx.x - row * cpr) * Out<T>::N;
    if (row >= rpp) return;
    const int64_t last = a.pos[b * a.pos_stride];
    const int S = kv8_window(last, a.n_meta, ctx), shift = kv8_first(last, ctx);
    const uint8_t* code = a.code[kv] + bh * a.S_ring * a.hs + c;
    const float* scale = a.scale[kv] + bh * a.nblk;
    T* out = (T*)a.out[kv] + bh * a.n * a.hs + c;
    code_t x[READ_PASSES];
    float f[READ_PASSES];
#pragma unroll
    for (int p = 0; p < READ_PASSES; ++p) {
        const int64_t r = (int64_t)blockIdx.x * (READ_PASSES * rpp) + p * rpp + row;
        x[p] = 0;
        f[p] = 0.f;
        if (r < a.n && a.first + r < S) {
            int s = a.first + (int)r;
            if (s >= a.n_meta) {
                s += shift;
                s -= s >= a.S_ring ? ctx : 0;
            }
            x[p] = __builtin_nontemporal_load((const code_t*)(code + (int64_t)s * a.hs));
            f[p] = scale[s >> a.block_log2];
        }
    }
#pragma unroll
    for (int p = 0; p < READ_PASSES; ++p) {
        const int64_t r = (int64_t)blockIdx.x * (READ_PASSES * rpp) + p * rpp + row;
        if (r < a.n) Out<T>::put(out + r * a.hs, x[p], f[p]);
    }
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
    MSQ_CHECK_ARG(grid * NT < (1ll << 32), "msq_kv8_write: %lld workgroups (%d rows of the batch x %d heads x %d blocks), "
                  "a launch takes under %lld", (long long)grid, (int)B, (int)H, a.nb, (1ll << 32) / NT);
    const int rpp = NT / (int)(hs / 8), nc = ((int)block + rpp - 1) / rpp;  // <= 8
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
    a.H = (int)H; a.hs = (int)hs; a.S_ring = (int)S_ring; a.n_meta = (int)n_meta;
    a.block_log2 = __builtin_ctz((unsigned)block);
    a.nblk = (int)msq_kv8_blocks(S_ring, block);
    a.first = (int)first; a.n = (int)rows;
    const int64_t group = READ_PASSES * (NT / (hs / (dtype == MSQ_BF16 ? Out<bf16>::N : Out<float>::N)));
    MSQ_CHECK_ARG((rows + group - 1) / group * NT < (1ll << 32), "msq_kv8_read: %lld rows, a launch takes under %lld",
                  (long long)rows, (1ll << 32) / NT * group);
    const dim3 grid((unsigned)((rows + group - 1) / group), (unsigned)(2 * H), (unsigned)B);
    if (dtype == MSQ_BF16) hipLaunchKernelGGL(kv8_read_kernel<bf16>, grid, dim3(NT), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(kv8_read_kernel<float>, grid, dim3(NT), 0, (hipStream_t)stream, a);
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}
