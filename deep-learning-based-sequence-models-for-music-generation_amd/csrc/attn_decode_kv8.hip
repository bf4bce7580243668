// Decode step of the relative-position attention (HeadRelPos,
// model_transformer.py:54-82, the LAST row of a window) over the 8-bit cache
// (kv8.h): for each (b, h)
//   out = softmax_j((q . k_j + q . R[w(j)]) * scale) . v_j,  k_j = code * scale
// over the S keys of the row's window, w(j) = the key's position in it (slot j
// itself until the ring wraps). Rows whose window is empty get zeros.
//
// Split over the keys: one workgroup per (chunk of slots, h, b); a key is
// spread over a 16-lane group, 8 values per lane, and every group keeps its own
// running maximum and sum (one pass, no exchange inside the loop); the groups
// and waves are joined at the end, the chunks by a second kernel.
#include "kv8.h"

namespace {

constexpr int NT = 256, HS = KV8_MAX_HS, GROUPS = 16, UN = 4, STEP = GROUPS * UN;

typedef float f32x8 __attribute__((ext_vector_type(8)));

struct Args {
    const void* q;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const void* R;
    void* out;
    float *po, *pml;
    const int64_t* pos;
    int64_t pos_stride, ldq, ldo, S_max;
    int H, hs, S_ring, n_meta, block, nblk, chunk, nsplit;
    float scale;
};

__device__ __forceinline__ f32x8 ld8(const bf16* p) {
    const bf16x8 x = *(const bf16x8*)p;
    return (f32x8){(float)x[0], (float)x[1], (float)x[2], (float)x[3], (float)x[4], (float)x[5], (float)x[6], (float)x[7]};
}
__device__ __forceinline__ f32x8 ld8(const float* p) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
    return (f32x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ f32x8 ld8(const uint8_t* p) {
    const uint2 x = *(const uint2*)p;
    const f32x4 a = kv8_dec4(x.x), b = kv8_dec4(x.y);
    return (f32x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// 2^(x - m) with an empty maximum read as 0 (x is then -inf too)
__device__ __forceinline__ float pexp(float x, float m) {
    return __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.f : m));
}

template <typename T>
__global__ __launch_bounds__(NT) void decode_kv8_kernel(Args a) {
    __shared__ float part[4][HS];
    __shared__ float wm[4], wl[4];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int l16 = lane & 15, grp = w * 4 + (lane >> 4);
    const int c = blockIdx.x, h = blockIdx.y, hs = a.hs, ctx = a.S_ring - a.n_meta;
    const int64_t b = blockIdx.z, bh = b * a.H + h;
    const int64_t last = a.pos[b * a.pos_stride];
    const int S = kv8_window(last, a.n_meta, ctx), first = kv8_first(last, ctx), s0 = c * a.chunk;
    if (s0 >= S && a.nsplit > 1) return;  // chunk past the window (uniform)
    const int d0 = 8 * l16;
    const bool dok = d0 < hs;
    const uint8_t* kc = a.kc + bh * a.S_ring * hs + d0;
    const uint8_t* vc = a.vc + bh * a.S_ring * hs + d0;
    const float *ks = a.ks + bh * a.nblk, *vs = a.vs + bh * a.nblk;
    const T* R = (const T*)a.R + (int64_t)h * a.S_max * hs + d0;
    f32x8 q = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (dok) q = ld8((const T*)a.q + b * a.ldq + (int64_t)h * hs + d0);
    const float sc = a.scale * 1.44269504088896340736f;  // scores in base 2

    float m = -INFINITY, l = 0.f, o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
    const int s1 = min(S, s0 + a.chunk);
    for (int t = s0; t < s1; t += STEP) {
        float x[UN];
        f32x8 v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int s = min(t + u * GROUPS + grp, s1 - 1);  // rows past the chunk: masked below
            int j = s;
            if (s >= a.n_meta) {
                j -= first;
                j += j < a.n_meta ? ctx : 0;
            }
            float acc = 0.f, rel = 0.f;
            v[u] = q;
            if (dok) {
                const f32x8 k = ld8(kc + (int64_t)s * hs), r = ld8(R + (int64_t)j * hs);
                v[u] = ld8(vc + (int64_t)s * hs);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc = fmaf(k[e], q[e], acc), rel = fmaf(r[e], q[e], rel);
            }
            acc = fmaf(acc, ks[s / a.block], rel);
#pragma unroll
            for (int k = 8; k > 0; k >>= 1) acc += __shfl_xor(acc, k, 64);
            x[u] = t + u * GROUPS + grp < s1 ? acc * sc : -INFINITY;
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < UN; ++u) mn = fmaxf(mn, x[u]);
        const float f = pexp(m, mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= f;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const float p = pexp(x[u], m);
            const int s = min(t + u * GROUPS + grp, s1 - 1);
            l += p;
            const float pv = p * vs[s / a.block];
            if (t + u * GROUPS + grp < s1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = fmaf(pv, v[u][e], o[e]);
            }
        }
    }
    // the 4 key groups of the wave
    float M = fmaxf(m, __shfl_xor(m, 16, 64));
    M = fmaxf(M, __shfl_xor(M, 32, 64));
    const float f = pexp(m, M);
    l *= f;
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        o[e] *= f;
        o[e] += __shfl_xor(o[e], 16, 64);
        o[e] += __shfl_xor(o[e], 32, 64);
    }
    if (lane < 16 && dok) {
#pragma unroll
        for (int e = 0; e < 8; ++e) part[w][d0 + e] = o[e];
    }
    if (lane == 0) wm[w] = M, wl[w] = l;
    __syncthreads();
    M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    float acc = 0.f, L = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float g = pexp(wm[i], M);
        L = fmaf(g, wl[i], L);
        if (tid < hs) acc = fmaf(g, part[i][tid], acc);
    }
    if (a.nsplit == 1) {
        if (tid < hs) ((T*)a.out)[b * a.ldo + (int64_t)h * hs + tid] = (T)(S > 0 ? acc / L : 0.f);
        return;
    }
    const int64_t pi = bh * a.nsplit + c;
    if (tid < hs) a.po[pi * hs + tid] = acc;
    if (tid == 0) a.pml[2 * pi] = M, a.pml[2 * pi + 1] = L;
}

// out[b, h] = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c over the chunks of the window
template <typename T>
__global__ __launch_bounds__(HS) void decode_kv8_join_kernel(Args a) {
    const int tid = threadIdx.x, h = blockIdx.x, hs = a.hs;
    const int64_t b = blockIdx.y, base = (b * a.H + h) * a.nsplit;
    const int S = kv8_window(a.pos[b * a.pos_stride], a.n_meta, a.S_ring - a.n_meta);
    const int nc = (S + a.chunk - 1) / a.chunk;
    float M = -INFINITY;
    for (int c = 0; c < nc; ++c) M = fmaxf(M, a.pml[2 * (base + c)]);
    float L = 0.f, acc = 0.f;
    for (int c = 0; c < nc; ++c) {
        const float f = pexp(a.pml[2 * (base + c)], M);
        L = fmaf(f, a.pml[2 * (base + c) + 1], L);
        if (tid < hs) acc = fmaf(f, a.po[(base + c) * hs + tid], acc);
    }
    if (tid < hs) ((T*)a.out)[b * a.ldo + (int64_t)h * hs + tid] = (T)(S > 0 ? acc / L : 0.f);
}

// slots per workgroup: enough workgroups for the 256 CUs, whole steps of the loop
int chunk_of(int64_t B, int64_t H, int64_t S_ring) {
    const int64_t want = (S_ring * B * H + 2047) / 2048;
    const int64_t c = (want + STEP - 1) / STEP * STEP;
    return (int)std::min<int64_t>(c, (S_ring + STEP - 1) / STEP * STEP);
}
int64_t splits(int64_t B, int64_t H, int64_t S_ring) {
    const int c = chunk_of(B, H, S_ring);
    return (S_ring + c - 1) / c;
}

}  // namespace

extern "C" size_t msq_relattn_decode_kv8_workspace(int64_t B, int64_t H, int64_t hs, int64_t S_ring) {
    if (B <= 0 || H <= 0 || hs <= 0 || S_ring <= 0) return 0;
    const int64_t n = splits(B, H, S_ring);
    return n > 1 ? (size_t)(B * H * n * (hs + 2)) * sizeof(float) : 0;
}

extern "C" int msq_relattn_decode_kv8(int dtype, void* out, int64_t ldo, const void* q, int64_t ldq, const void* kc,
                                      const float* ks, const void* vc, const float* vs, const void* R, int64_t S_max,
                                      int64_t B, int64_t H, int64_t hs, int64_t S_ring, int64_t n_meta, int64_t block,
                                      const int64_t* pos, int64_t pos_stride, float scale, void* ws, size_t ws_bytes,
                                      void* stream) {
    const char* fn = "msq_relattn_decode_kv8";
    MSQ_CHECK_ARG(out && q && kc && ks && vc && vs && R && pos, "%s: null pointer", fn);
    MSQ_CHECK_ARG(dtype == MSQ_BF16 || dtype == MSQ_F32, "%s: dtype %d", fn, dtype);
    MSQ_CHECK_ARG(hs > 0 && hs <= HS && hs % 8 == 0, "%s: head size %lld (8 | hs <= %d)", fn, (long long)hs, HS);
    MSQ_CHECK_ARG(B > 0 && B <= 65535 && H > 0 && H <= 32767 && n_meta >= 0 && S_ring > n_meta && S_ring <= (1 << 30),
                  "%s: bad sizes (B %lld, H %lld, ring %lld, metadata %lld)", fn, (long long)B, (long long)H,
                  (long long)S_ring, (long long)n_meta);
    MSQ_CHECK_ARG(S_max >= S_ring, "%s: %lld relative rows for a ring of %lld", fn, (long long)S_max, (long long)S_ring);
    MSQ_CHECK_ARG(kv8_block_ok(block), "%s: block %lld (16, 32, 64 or 128 slots)", fn, (long long)block);
    MSQ_CHECK_ARG(pos_stride == 0 || pos_stride == 1, "%s: pos_stride %lld (0 or 1)", fn, (long long)pos_stride);
    MSQ_CHECK_ARG(ldq >= H * hs && ldo >= H * hs && ldq % 8 == 0, "%s: bad leading dims", fn);
    MSQ_CHECK_ARG((((uintptr_t)q | (uintptr_t)R) & 15) == 0 && (((uintptr_t)kc | (uintptr_t)vc) & 7) == 0,
                  "%s: q and R have to be 16-byte, the cache 8-byte aligned", fn);
    const size_t need = msq_relattn_decode_kv8_workspace(B, H, hs, S_ring);
    MSQ_CHECK_ARG(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0),
                  "%s: workspace of %zu bytes (16-B aligned) needed, %zu given", fn, need, ws_bytes);
    Args a;
    a.q = q; a.kc = (const uint8_t*)kc; a.vc = (const uint8_t*)vc; a.ks = ks; a.vs = vs; a.R = R; a.out = out;
    a.pos = pos; a.pos_stride = pos_stride; a.ldq = ldq; a.ldo = ldo; a.S_max = S_max;
    a.H = (int)H; a.hs = (int)hs; a.S_ring = (int)S_ring; a.n_meta = (int)n_meta; a.block = (int)block;
    a.nblk = (int)((S_ring + block - 1) / block);
    a.chunk = chunk_of(B, H, S_ring);
    a.nsplit = (int)splits(B, H, S_ring);
    a.po = (float*)ws;
    a.pml = (float*)ws + B * H * a.nsplit * hs;
    a.scale = scale;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)a.nsplit, (unsigned)H, (unsigned)B), jgrid((unsigned)H, (unsigned)B);
    if (dtype == MSQ_BF16) {
        hipLaunchKernelGGL(decode_kv8_kernel<bf16>, grid, dim3(NT), 0, s, a);
        if (a.nsplit > 1) hipLaunchKernelGGL(decode_kv8_join_kernel<bf16>, jgrid, dim3(HS), 0, s, a);
    } else {
        hipLaunchKernelGGL(decode_kv8_kernel<float>, grid, dim3(NT), 0, s, a);
        if (a.nsplit > 1) hipLaunchKernelGGL(decode_kv8_join_kernel<float>, jgrid, dim3(HS), 0, s, a);
    }
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}
