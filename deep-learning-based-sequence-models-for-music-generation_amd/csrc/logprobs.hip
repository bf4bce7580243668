// Log probabilities of given tokens, entropy and the top alternatives of rows of
// logits, and their gradient (what torch.nn.CrossEntropyLoss, train_parallel.py:
// 156,179, and torch.topk, scripts/generate.py:66-74, compute in part):
//   lp_i = x_i - M - log s,   s = sum e^(x_i - M),  M = max x
//   H    = -sum p_i lp_i = log s - t / s,   t = sum (x_i - M) e^(x_i - M)
//   dx_i = sum_k g_k ([i = id_k] - p_i) + g_y ([i = y] - p_i) - g_H p_i (lp_i + H)
// A row without a finite logit (all -inf) has no distribution: lp = -inf,
// H = 0, gradient 0. NaN or +inf in a row makes its lp, H and gradient NaN.
// Tokens outside [0, V) (padding) get lp = 0 and no gradient from g_y. The top
// alternatives are ordered by value, equal ones by index; NaN counts as largest.
//
// One workgroup per row. A row whose address is not 16-byte aligned is read as
// the aligned 16-byte vectors that cover it, the ones at its ends by element.
#include "common.h"

namespace {

constexpr int MAXTOP = 32, CAP = 512;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };

struct FwdArgs {
    const void* x;
    int64_t ld, V;
    const int64_t* tok;
    float *lp, *ent, *stats, *top_lp;
    int64_t* top_id;
    int top;
};

template <typename T>
__device__ __forceinline__ float elem(u32x4 v, int e);
template <>
__device__ __forceinline__ float elem<float>(u32x4 v, int e) { return __uint_as_float(v[e]); }
template <>
__device__ __forceinline__ float elem<bf16>(u32x4 v, int e) {
    return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
}

// the row as aligned vectors: vector j holds elements j * N - off .. + N - 1
template <typename T>
struct Row {
    const T* x;
    int64_t V;
    int off;
    __device__ __forceinline__ Row(const void* base, int64_t row, int64_t ld, int64_t V_)
        : x((const T*)base + row * ld), V(V_), off((int)(((uintptr_t)x & 15) / sizeof(T))) {}
    __device__ __forceinline__ int64_t vecs() const { return (V + off + Vec<T>::N - 1) / Vec<T>::N; }
    // elements outside the row read as -inf
    __device__ __forceinline__ u32x4 load(int64_t j) const {
        const int64_t i0 = j * Vec<T>::N - off;
        if (i0 >= 0 && i0 + Vec<T>::N <= V) return *(const u32x4*)(x + i0);
        union { u32x4 v; T t[Vec<T>::N]; } r;
#pragma unroll
        for (int e = 0; e < Vec<T>::N; ++e) r.t[e] = i0 + e >= 0 && i0 + e < V ? x[i0 + e] : (T)-INFINITY;
        return r.v;
    }
};

// order of the values as unsigned integers, -0 = +0, NaN largest (above +inf,
// 0xff800000, and below the bound ~0 that no key of an element reaches)
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xff800001u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)ordered(x) << 32 | (0xffffffffu - i); }

template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) s += red[i];
    return s;
}
template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) s = fmaxf(s, red[i]);
    return s;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void token_logprobs_kernel(FwdArgs a) {
    __shared__ float red[NT / 64];
    __shared__ uint64_t kred[NT / 64];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Row<T> R(a.x, row, a.ld, a.V);
    const int64_t nv = R.vecs();
    float m = -INFINITY;
    for (int64_t j = tid; j < nv; j += NT) {
        const u32x4 v = R.load(j);
#pragma unroll
        for (int e = 0; e < Vec<T>::N; ++e) m = fmaxf(m, elem<T>(v, e));
    }
    const float M = block_max<NT>(m, red), Mf = M == -INFINITY ? 0.f : M;
    float s = 0.f, t = 0.f;
    for (int64_t j = tid; j < nv; j += NT) {
        const u32x4 v = R.load(j);
#pragma unroll
        for (int e = 0; e < Vec<T>::N; ++e) {
            const float d = elem<T>(v, e) - Mf, p = __builtin_amdgcn_exp2f(d * LOG2E);
            s += p;
            t = fmaf(fmaxf(d, -1e30f), p, t);  // d = -inf: p = 0
        }
    }
    s = block_sum<NT>(s, red);
    t = block_sum<NT>(t, red);
    const float ls = M == -INFINITY ? s : logf(s);  // no finite logit: 0, or NaN if one is
    if (tid == 0) {
        const int64_t y = a.tok[row];
        a.lp[row] = y >= 0 && y < a.V ? (M == -INFINITY && s == 0.f ? -INFINITY : ((float)R.x[y] - M) - ls) : 0.f;
        a.ent[row] = M == -INFINITY && s == 0.f ? 0.f : ls - t / s;
        if (a.stats) a.stats[2 * row] = M, a.stats[2 * row + 1] = ls;
    }
    uint64_t prev = ~0ull;
    for (int k = 0; k < a.top; ++k) {  // the largest key below the one before
        uint64_t best = 0;
        for (int64_t j = tid; j < nv; j += NT) {
            const u32x4 v = R.load(j);
#pragma unroll
            for (int e = 0; e < Vec<T>::N; ++e) {
                const int64_t i = j * Vec<T>::N - R.off + e;
                const uint64_t key = key_of(elem<T>(v, e), (uint32_t)i);
                if (i >= 0 && i < a.V && key < prev && key > best) best = key;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, o, 64);
            best = other > best ? other : best;
        }
        __syncthreads();
        if ((tid & 63) == 0) kred[tid >> 6] = best;
        __syncthreads();
        best = kred[0];
#pragma unroll
        for (int i = 1; i < NT / 64; ++i) best = kred[i] > best ? kred[i] : best;
        prev = best;
        if (tid == 0) {
            const uint32_t i = 0xffffffffu - (uint32_t)best;
            a.top_id[row * a.top + k] = i;
            a.top_lp[row * a.top + k] = M == -INFINITY && s == 0.f ? -INFINITY : ((float)R.x[i] - M) - ls;
        }
    }
}

struct BwdArgs {
    const void* x;
    void* dx;
    int64_t ld, ldd, V;
    const int64_t *tok, *top_id;
    const float *g_lp, *g_ent, *g_top, *stats, *ent;
    int top;
};

template <typename T, int NT>
__global__ __launch_bounds__(NT) void token_logprobs_bwd_kernel(BwdArgs a) {
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Row<T> R(a.x, row, a.ld, a.V);
    T* dx = (T*)a.dx + row * a.ldd;
    const float M = a.stats[2 * row], ls = a.stats[2 * row + 1];
    const int64_t y = a.tok[row];
    const float gy = a.g_lp && y >= 0 && y < a.V ? a.g_lp[row] : 0.f, gh = a.g_ent ? a.g_ent[row] : 0.f;
    float c = gy;
    if (a.g_top)
        for (int k = 0; k < a.top; ++k) c += a.g_top[row * a.top + k];
    c = -c - gh * a.ent[row];
    const bool empty = M == -INFINITY && ls == 0.f;
    for (int64_t i = tid; i < a.V; i += NT) {
        const float lp = ((float)R.x[i] - M) - ls, p = __builtin_amdgcn_exp2f(lp * LOG2E);
        float d = p * fmaf(-gh, fmaxf(lp, -1e30f), c);
        if (i == y) d += gy;
        if (a.g_top)
            for (int k = 0; k < a.top; ++k) d += a.top_id[row * a.top + k] == i ? a.g_top[row * a.top + k] : 0.f;
        dx[i] = (T)(empty ? 0.f : d);
    }
}

}  // namespace

extern "C" int msq_token_logprobs(float* logprob, float* entropy, float* stats, int64_t* top_ids, float* top_logprobs,
                                  const void* logits, int dtype, int64_t ld, const int64_t* tokens, int64_t rows,
                                  int64_t V, int64_t top, void* stream) {
    const char* fn = "msq_token_logprobs";
    MSQ_CHECK_ARG(logprob && entropy && logits && tokens, "%s: null pointer", fn);
    MSQ_CHECK_ARG(dtype == MSQ_BF16 || dtype == MSQ_F32, "%s: dtype %d", fn, dtype);
    MSQ_CHECK_ARG(rows > 0 && rows < (1ll << 31) && V > 0 && V < (1ll << 31) && ld >= 0,
                  "%s: bad sizes (%lld rows of %lld, stride %lld)", fn, (long long)rows, (long long)V, (long long)ld);
    MSQ_CHECK_ARG(top >= 0 && top <= MAXTOP && top <= V, "%s: %lld alternatives of %lld (at most %d)", fn,
                  (long long)top, (long long)V, MAXTOP);
    MSQ_CHECK_ARG(top == 0 || (top_ids && top_logprobs), "%s: null pointer", fn);
    const FwdArgs a{logits, ld, V, tokens, logprob, entropy, stats, top_logprobs, top_ids, (int)top};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MSQ_BF16) hipLaunchKernelGGL((token_logprobs_kernel<bf16, 256>), dim3((unsigned)rows), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((token_logprobs_kernel<float, 256>), dim3((unsigned)rows), dim3(256), 0, s, a);
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}

extern "C" int msq_token_logprobs_bwd(void* dlogits, int64_t ldd, const float* g_logprob, const float* g_entropy,
                                      const float* g_top, const float* stats, const float* entropy,
                                      const int64_t* top_ids, int64_t top, const void* logits, int dtype, int64_t ld,
                                      const int64_t* tokens, int64_t rows, int64_t V, void* stream) {
    const char* fn = "msq_token_logprobs_bwd";
    MSQ_CHECK_ARG(dlogits && stats && entropy && logits && tokens, "%s: null pointer", fn);
    MSQ_CHECK_ARG(dtype == MSQ_BF16 || dtype == MSQ_F32, "%s: dtype %d", fn, dtype);
    MSQ_CHECK_ARG(rows > 0 && rows < (1ll << 31) && V > 0 && V < (1ll << 31) && ld >= 0 && ldd >= V,
                  "%s: bad sizes (%lld rows of %lld, strides %lld, %lld)", fn, (long long)rows, (long long)V,
                  (long long)ld, (long long)ldd);
    MSQ_CHECK_ARG(top >= 0 && top <= MAXTOP, "%s: %lld alternatives (at most %d)", fn, (long long)top, MAXTOP);
    MSQ_CHECK_ARG(!g_top || (top_ids && top > 0), "%s: the alternatives' gradient needs their ids", fn);
    const BwdArgs a{logits, dlogits, ld, ldd, V, tokens, top_ids, g_logprob, g_entropy, g_top, stats, entropy, (int)top};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MSQ_BF16)
        hipLaunchKernelGGL((token_logprobs_bwd_kernel<bf16, 256>), dim3((unsigned)rows), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((token_logprobs_bwd_kernel<float, 256>), dim3((unsigned)rows), dim3(256), 0, s, a);
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}
