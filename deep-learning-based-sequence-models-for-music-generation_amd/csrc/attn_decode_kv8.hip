// Decode step of the relative-position attention (HeadRelPos,
// model_transformer.py:54-82, the LAST row of a window) over the 8-bit cache
// (kv8.h): for each (b, h)
//   out = softmax_j((q . k_j + q . R[w(j)]) * scale) . v_j,  k_j = code * scale
// over the S keys of the row's window, w(j) = the key's position in it (slot j
// itself until the ring wraps). Rows whose window is empty get zeros.
//
// Bound by the cache's bytes (2 hs per key and (b, h)); R comes from L2.
// Split over the keys (flash decoding): one workgroup of 4 waves per (chunk of
// slots, h, b). A key is spread over LPK lanes, VPL values each (16-byte loads of
// 16 codes where the head size allows it), so a wave's load covers 64 / LPK
// consecutive slots; every such key group keeps its own running maximum, sum and
// output (one pass, no exchange inside the loop but the LPK-lane sum of a
// score). Groups and waves are joined at the end, the chunks of a row by a second
// kernel.
#include "kv8.h"

namespace {

constexpr int HS = KV8_MAX_HS;
constexpr float LOG2E = 1.44269504088896340736f;

struct Args {
    const void* q;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const void* R;
    void* out;
    float *po, *pml;
    const int64_t* pos;
    int64_t pos_stride, ldq, ldo, S_max;
    int B, H, hs, S_ring, n_meta, block_log2, nblk, chunk, nsplit, waves, remap;
    float scale;
};

// 2^(x - m) with an empty maximum read as 0 (x is then -inf too)
__device__ __forceinline__ float pexp(float x, float m) {
    return __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.f : m));
}

// N values of a row as the lane holds them
template <typename T, int N> struct Row;
template <int N> struct Row<bf16, N> {
    u32x4 v[N / 8];
    __device__ __forceinline__ void load(const bf16* p) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) v[i] = ((const u32x4*)p)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) v[i] = (u32x4){0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ bf16x2 pair(int i) const {
        const uint32_t x = v[i >> 2][i & 3];  // a value: __builtin_bit_cast of a vector's element reads element 0
        return __builtin_bit_cast(bf16x2, x);
    }
    __device__ __forceinline__ float dot(const Row& o) const {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) a = __builtin_amdgcn_fdot2_f32_bf16(pair(i), o.pair(i), a, false);
        return a;
    }
};
template <int N> struct Row<float, N> {
    f32x4 v[N / 4];
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) v[i] = ((const f32x4*)p)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) v[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ float dot(const Row& o) const {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) a = fmaf(v[i >> 2][i & 3], o.v[i >> 2][i & 3], a);
        return a;
    }
};
template <int N> struct Codes {
    uint32_t v[N / 4];
    // read once: not to push the rows of R out of the L2
    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (N == 16) {
            const u32x4 x = __builtin_nontemporal_load((const u32x4*)p);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = x[i];
        } else {
            const uint64_t x = __builtin_nontemporal_load((const uint64_t*)p);
            v[0] = (uint32_t)x, v[1] = (uint32_t)(x >> 32);
        }
    }
    // e4m3 is exact in bf16: two products per instruction
    __device__ __forceinline__ float dot(const Row<bf16, N>& q) const {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            a = __builtin_amdgcn_fdot2_f32_bf16(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, false),
                                                q.pair(2 * i), a, false);
            a = __builtin_amdgcn_fdot2_f32_bf16(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, true),
                                                q.pair(2 * i + 1), a, false);
        }
        return a;
    }
    __device__ __forceinline__ float dot(const Row<float, N>& q) const {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const f32x4 c = kv8_dec4(v[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) a = fmaf(c[e], q.v[i][e], a);
        }
        return a;
    }
    __device__ __forceinline__ void add_to(float* o, float p) const {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const f32x4 c = kv8_dec4(v[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * i + e] = fmaf(p, c[e], o[4 * i + e]);
        }
    }
};

template <typename T, int VPL, int LPK, int NW>
__global__ __launch_bounds__(64 * NW) void decode_kv8_kernel(Args a) {
    constexpr int GW = 64 / LPK;                       // keys per load of a wave
    constexpr int UN = VPL * sizeof(T) > 32 ? 2 : 4;   // loads of a wave in flight: 64 registers
    constexpr int STEP = NW * GW * UN;
    __shared__ float part[NW][HS];
    __shared__ float wm[NW], wl[NW];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, grp = lane / LPK;
    // workgroups go round the 8 XCDs: the chunks and rows of a head, which read the
    // same rows of R, on one XCD (remap 2: 8 | H), else those of a (h, chunk) pair
    // (remap 1); the rows of the batch side by side
    int h, c;
    int64_t b;
    if (a.remap) {
        const int x = blockIdx.x & 7, i = blockIdx.x >> 3, k = i / a.B;
        b = i - k * a.B;
        if (a.remap == 2) {
            h = k / a.nsplit;
            c = k - h * a.nsplit;
            h = h * 8 + x;
        } else {
            const int pair = k * 8 + x;
            if (pair >= a.H * a.nsplit) return;
            h = pair / a.nsplit;
            c = pair - h * a.nsplit;
        }
    } else {
        const int pair = blockIdx.x / a.B;
        b = blockIdx.x - pair * a.B;
        h = pair / a.nsplit;
        c = pair - h * a.nsplit;
    }
    const int hs = a.hs, ctx = a.S_ring - a.n_meta;
    const int64_t bh = b * a.H + h, last = a.pos[b * a.pos_stride];
    const int S = kv8_window(last, a.n_meta, ctx), first = kv8_first(last, ctx), s0 = c * a.chunk;
    const int n = min(S - s0, a.chunk);  // keys of this chunk
    if (n <= 0 && a.nsplit > 1) return;  // no key in this chunk (uniform)
    const int d0 = VPL * (lane % LPK);
    const bool dok = d0 < hs;
    const uint8_t* kc = a.kc + (bh * a.S_ring + s0) * hs + d0;
    const uint8_t* vc = a.vc + (bh * a.S_ring + s0) * hs + d0;
    const float *ks = a.ks + bh * a.nblk, *vs = a.vs + bh * a.nblk;
    const T* R = (const T*)a.R + (int64_t)h * a.S_max * hs + d0;
    Row<T, VPL> q;
    q.zero();
    if (dok) q.load((const T*)a.q + b * a.ldq + (int64_t)h * hs + d0);
    const float sc = a.scale * LOG2E;  // scores in base 2

    float m = -INFINITY, l = 0.f, o[VPL];
#pragma unroll
    for (int e = 0; e < VPL; ++e) o[e] = 0.f;
    for (int t = w * GW * UN; t < n; t += STEP) {
        Codes<VPL> k[UN], v[UN];
        Row<T, VPL> r[UN];
        float fk[UN], fv[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int s = min(t + u * GW + grp, n - 1);  // rows past the chunk: masked below
            int j = s0 + s;
            fk[u] = ks[j >> a.block_log2];
            fv[u] = vs[j >> a.block_log2];
            if (j >= a.n_meta) {
                j -= first;
                j += j < a.n_meta ? ctx : 0;
            }
            if (dok) {
                k[u].load(kc + (uint32_t)(s * hs));
                r[u].load(R + (int64_t)j * hs);
                v[u].load(vc + (uint32_t)(s * hs));
            }
        }
        float x[UN], mn = m;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            x[u] = dok ? fmaf(k[u].dot(q), fk[u], r[u].dot(q)) : 0.f;
#pragma unroll
            for (int i = LPK / 2; i > 0; i >>= 1) x[u] += __shfl_xor(x[u], i, 64);
            x[u] = t + u * GW + grp < n ? x[u] * sc : -INFINITY;
            mn = fmaxf(mn, x[u]);
        }
        if (__any(mn > m)) {  // else the factor is 1
            const float f = pexp(m, mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int e = 0; e < VPL; ++e) o[e] *= f;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const float p = pexp(x[u], m);
            l += p;
            if (dok && t + u * GW + grp < n) v[u].add_to(o, p * fv[u]);
        }
    }
    // the key groups of the wave
    float M = m;
#pragma unroll
    for (int i = LPK; i < 64; i <<= 1) M = fmaxf(M, __shfl_xor(M, i, 64));
    const float f = pexp(m, M);
    l *= f;
#pragma unroll
    for (int e = 0; e < VPL; ++e) o[e] *= f;
#pragma unroll
    for (int i = LPK; i < 64; i <<= 1) {
        l += __shfl_xor(l, i, 64);
#pragma unroll
        for (int e = 0; e < VPL; ++e) o[e] += __shfl_xor(o[e], i, 64);
    }
    if (lane < LPK && dok) {
#pragma unroll
        for (int e = 0; e < VPL; ++e) part[w][d0 + e] = o[e];
    }
    if (lane == 0) wm[w] = M, wl[w] = l;
    __syncthreads();
    M = wm[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) M = fmaxf(M, wm[i]);
    float acc = 0.f, L = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
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

// out[b, h] = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c over the chunks that hold keys,
// HS chunks at a time. (Joined instead by the workgroup that is done last: with the
// parts written past the L2 the same time, with fences around them four to ten times
// the whole kernel's.)
template <typename T>
__global__ __launch_bounds__(HS) void decode_kv8_join_kernel(Args a) {
    __shared__ float f[HS], l[HS];
    const int tid = threadIdx.x, hs = a.hs;
    const int64_t b = blockIdx.y, bh = b * a.H + blockIdx.x, base = bh * a.nsplit;
    const f32x2* ml = (const f32x2*)a.pml + base;
    const float* po = a.po + base * hs + tid;
    const int S = kv8_window(a.pos[b * a.pos_stride], a.n_meta, a.S_ring - a.n_meta);
    const int nc = (S + a.chunk - 1) / a.chunk;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int c0 = 0; c0 < nc; c0 += HS) {
        const int n = min(HS, nc - c0);
        f32x2 x = {-INFINITY, 0.f};
        if (tid < n) x = ml[c0 + tid];
        f[tid] = x[0];
        __syncthreads();
        float Mn = M;
        for (int i = 0; i < n; ++i) Mn = fmaxf(Mn, f[i]);
        __syncthreads();
        f[tid] = pexp(x[0], Mn);
        l[tid] = x[1];
        __syncthreads();
        const float r = pexp(M, Mn);
        M = Mn;
        acc *= r;
        L *= r;
        for (int i = 0; i < n; i += 4) {
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = tid < hs && i + k < n ? po[(int64_t)(c0 + i + k) * hs] : 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) acc = fmaf(f[i + k], o[k], acc), L = fmaf(f[i + k], l[i + k], L);
        }
        __syncthreads();
    }
    if (tid < hs) ((T*)a.out)[b * a.ldo + (int64_t)blockIdx.x * hs + tid] = (T)(nc > 0 ? acc / L : 0.f);
}

struct Plan {
    int64_t chunk, nsplit;
    int waves;
};
// How a row's ring is cut. A workgroup streams at its CU's share of the memory's
// rate (some 19 KB/us of 4.8 TB/s), so a cut into n chunks takes ceil(B H n /
// 256) / n times a whole row, and a join of some 4 us more: the n that fill one
// to four rounds of the 256 CUs are weighed. 64 rows x 8 heads x 2054 keys of 128
// run uncut in 52 us (in 4 chunks 55, in 8 57); 8 rows in 4 chunks 15 us (uncut
// 25); 4 rows x 16 heads x 16385 keys of 64 in 4 chunks 35 us (uncut 89). Rows at
// positions of their own are cut into 10 workgroups a CU, for the long ones not to
// be left over (24 rows x 16 heads of up to 16385 keys: 119 us; uncut 178). Eight
// waves a workgroup where each has a pass or more over the loop, else four.
Plan plan_of(int64_t B, int64_t H, int64_t hs, int64_t S_ring, bool ragged) {
    // no chunk under 32 KB, what four waves have in flight at once
    const int64_t U = B * H, most = std::max<int64_t>(1, S_ring * hs * 2 / 32768);
    const double row = (double)S_ring * hs * 2 / 19e3;
    int64_t best = 1;
    double cost = row * ((U + 255) / 256);
    for (int k = 1; k <= 4; ++k) {
        const int64_t n = std::min(most, 256 * k / U);
        if (n <= best) continue;
        const double c = row * ((U * n + 255) / 256) / n + 4.0;
        if (c < cost) cost = c, best = n;
    }
    if (ragged) best = std::max(best, std::min(most, (2560 + U - 1) / U));
    Plan p;
    p.chunk = ((S_ring + best - 1) / best + 31) / 32 * 32;
    p.nsplit = (S_ring + p.chunk - 1) / p.chunk;
    const int64_t unit = hs > 64 ? 32 : hs > 32 ? 64 : hs > 16 ? 128 : 256;  // keys of a wave in flight
    p.waves = p.chunk >= 12 * unit && !ragged ? 8 : 4;
    return p;
}

template <typename T, int VPL, int LPK>
void launch_one(const Args& a, unsigned grid, hipStream_t s) {
    if (a.waves == 8) hipLaunchKernelGGL((decode_kv8_kernel<T, VPL, LPK, 8>), dim3(grid), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((decode_kv8_kernel<T, VPL, LPK, 4>), dim3(grid), dim3(256), 0, s, a);
}
template <typename T>
void launch(const Args& a, unsigned grid, hipStream_t s) {
    // 16 codes per lane where the rows are 16-byte aligned
    if (a.hs % 16 == 0 && (((uintptr_t)a.kc | (uintptr_t)a.vc) & 15) == 0) {
        if (a.hs <= 16) launch_one<T, 16, 1>(a, grid, s);
        else if (a.hs <= 32) launch_one<T, 16, 2>(a, grid, s);
        else if (a.hs <= 64) launch_one<T, 16, 4>(a, grid, s);
        else launch_one<T, 16, 8>(a, grid, s);
    } else {
        if (a.hs <= 8) launch_one<T, 8, 1>(a, grid, s);
        else if (a.hs <= 16) launch_one<T, 8, 2>(a, grid, s);
        else if (a.hs <= 32) launch_one<T, 8, 4>(a, grid, s);
        else if (a.hs <= 64) launch_one<T, 8, 8>(a, grid, s);
        else launch_one<T, 8, 16>(a, grid, s);
    }
    if (a.nsplit > 1)
        hipLaunchKernelGGL(decode_kv8_join_kernel<T>, dim3((unsigned)a.H, (unsigned)a.B), dim3(HS), 0, s, a);
}

}  // namespace

extern "C" size_t msq_relattn_decode_kv8_workspace(int64_t B, int64_t H, int64_t hs, int64_t S_ring) {
    if (B <= 0 || H <= 0 || hs <= 0 || S_ring <= 0) return 0;
    const int64_t n = plan_of(B, H, hs, S_ring, true).nsplit;  // no fewer than with one position for all
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
    a.B = (int)B; a.H = (int)H; a.hs = (int)hs; a.S_ring = (int)S_ring; a.n_meta = (int)n_meta;
    a.block_log2 = __builtin_ctz((unsigned)block);
    a.nblk = (int)((S_ring + block - 1) / block);
    const Plan p = plan_of(B, H, hs, S_ring, pos_stride != 0);
    a.chunk = (int)p.chunk;
    a.nsplit = (int)p.nsplit;
    a.waves = p.waves;
    MSQ_CHECK_ARG((int64_t)a.chunk * hs < (1ll << 31), "%s: a ring of %lld for %lld x %lld heads", fn, (long long)S_ring,
                  (long long)B, (long long)H);  // 32-bit offsets inside a chunk
    a.po = (float*)ws;
    a.pml = (float*)ws + B * H * a.nsplit * hs;
    a.scale = scale;
    const int64_t pairs = H * a.nsplit;
    a.remap = H % 8 == 0 ? 2 : pairs >= 32;  // fewer would leave XCDs without work
    const int64_t grid = (a.remap ? (pairs + 7) / 8 * 8 : pairs) * B;
    MSQ_CHECK_ARG(grid * 64 * a.waves < (1ll << 32), "%s: %lld workgroups (%lld rows x %lld heads x %d chunks), a launch "
                  "takes under %lld", fn, (long long)grid, (long long)B, (long long)H, a.nsplit, (1ll << 26) / a.waves);
    if (dtype == MSQ_BF16) launch<bf16>(a, (unsigned)grid, (hipStream_t)stream);
    else launch<float>(a, (unsigned)grid, (hipStream_t)stream);
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}
