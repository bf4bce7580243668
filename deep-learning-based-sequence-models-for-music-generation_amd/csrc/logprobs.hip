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
// One workgroup per row. Forward: bound by the row's bytes, and close behind by
// the VALU (some 12 operations an element at 13 that fit under 6 TB/s of bf16, the
// exponential alone 4): the row is read once, into registers (up to 9 vectors of
// 16 bytes a lane), the maximum taken first so that no running sum is rescaled.
// Longer rows are streamed with a running maximum (and read a second time for
// the top alternatives). A row whose address is not 16-byte aligned is read as the
// aligned 16-byte vectors that cover it, the ones at its ends by element.
//
// Top k without sorting: of the maxima of 64 sets of lanes the k-th largest is a
// bound that at least k elements reach and hardly more do (k (1 + k / 128) or so
// for values in no order). It is found by bisection over the upper 16 bits of the
// values' order, with a ballot a bit. The vectors that hold such elements are
// listed in LDS, the elements ranked by (value, index). A row of many equal
// values, or whose values above a large tie lie in fewer than k sets of lanes, may
// list more than fit; it is then searched k times (top_slow: 4096 bf16 rows of 17914
// with 127 events above 0 elsewhere, 32 alternatives: 1.08 ms; 39 us for values in
// no order, and 55 in fp32, where the 127 lie in 32 vectors).
#include "common.h"

namespace {

constexpr int MAXTOP = 32, VCAP = 128, CAP = 256;  // a row of under 32 vectors fits whole
constexpr float LOG2E = 1.44269504088896340736f;

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };

struct FwdArgs {
    const void* x;
    int64_t ld, V;
    const int64_t* tok;
    float *lp, *ent, *stats, *top_lp;
    int64_t* top_id;
    int64_t rows;
    int top;
};

// A row of one wave needs no barrier: LDS operations of a wave are in order. Such
// rows go four to a workgroup.
template <int NT>
__device__ __forceinline__ void row_sync() {
    if constexpr (NT > 64) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}
constexpr int rows_per_block(int NT) { return NT == 64 ? 4 : 1; }

template <typename T>
__device__ __forceinline__ float elem(u32x4 v, int e);
template <>
__device__ __forceinline__ float elem<float>(u32x4 v, int e) { return __uint_as_float(v[e]); }
template <>
__device__ __forceinline__ float elem<bf16>(u32x4 v, int e) {
    return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
}
template <typename T>
__device__ __forceinline__ float vec_max(u32x4 v) {
    float m = elem<T>(v, 0);
#pragma unroll
    for (int e = 1; e < Vec<T>::N; ++e) m = fmaxf(m, elem<T>(v, e));
    return m;
}

// the row as aligned vectors: vector j holds elements j * N - off .. + N - 1
template <typename T>
struct Row {
    static constexpr int N = Vec<T>::N;
    const T* x;
    int64_t V;
    int off;
    __device__ __forceinline__ Row(const void* base, int64_t row, int64_t ld, int64_t V_)
        : x((const T*)base + row * ld), V(V_), off((int)(((uintptr_t)x & 15) / sizeof(T))) {}
    __device__ __forceinline__ int64_t vecs() const { return (V + off + N - 1) / N; }
    __device__ __forceinline__ int64_t at(int64_t j) const { return j * N - off; }
    __device__ __forceinline__ bool whole(int64_t j) const { return at(j) >= 0 && at(j) + N <= V; }
    // elements outside the row read as -inf; KEEP: the row is read again soon
    template <bool KEEP = true>
    __device__ __forceinline__ u32x4 inner(int64_t j) const {  // of a whole vector
        const T* p = x + at(j);
        return KEEP ? *(const u32x4*)p : __builtin_nontemporal_load((const u32x4*)p);
    }
    __device__ __forceinline__ u32x4 edge(int64_t j) const {
        const int64_t i0 = at(j);
        union { u32x4 v; T t[N]; } r;
#pragma unroll
        for (int e = 0; e < N; ++e) r.t[e] = i0 + e >= 0 && i0 + e < V ? x[i0 + e] : (T)-INFINITY;
        return r.v;
    }
    static __device__ __forceinline__ u32x4 none() {
        union { u32x4 v; T t[N]; } r;
#pragma unroll
        for (int e = 0; e < N; ++e) r.t[e] = (T)-INFINITY;
        return r.v;
    }
    __device__ __forceinline__ u32x4 load(int64_t j) const { return whole(j) ? inner(j) : edge(j); }
};

// order of the values as unsigned integers, -0 = +0, NaN largest (above +inf,
// 0xff800000, and below the bound ~0 that no key of an element reaches)
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xff800001u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)ordered(x) << 32 | (0xffffffffu - i); }
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

// a value that at least k of the wave's 64 values g reach and no more than about k do
__device__ __forceinline__ float kth_bound(float g, int k) {
    const uint32_t o = ordered(g);
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t c = t | 1u << bit;
        if (__popcll(__ballot(o >= c)) >= k) t = c;  // (uniform)
    }
    // the value of that order; -inf where fewer than k sets hold a finite one
    return t <= ordered(-INFINITY) ? -INFINITY : __uint_as_float(t & 0x80000000u ? t ^ 0x80000000u : ~t);
}

// running sums of a row against the maximum m: s = sum e^(x - m), t = sum (x - m) e^(x - m)
struct Sums {
    float s = 0.f, t = 0.f;
    template <typename T>
    __device__ __forceinline__ void add(u32x4 v, float m) {
#pragma unroll
        for (int e = 0; e < Vec<T>::N; ++e) {
            const float d = elem<T>(v, e) - m, p = __builtin_amdgcn_exp2f(d * LOG2E);
            s += p;
            t = fmaf(fmaxf(d, -1e30f), p, t);  // d = -inf: p = 0
        }
    }
    // to the maximum m + d, d >= 0 (or m = -inf: the sums are 0, or NaN)
    __device__ __forceinline__ void rescale(float d) {
        const float f = __builtin_amdgcn_exp2f(-d * LOG2E);
        t = f * fmaf(-fminf(d, 1e30f), s, t);
        s *= f;
    }
};
__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

// The largest elements by repeated search (many equal values, or NaN)
template <typename T, int NT>
__device__ void top_slow(const Row<T>& R, int top, uint64_t* kred, uint64_t* out) {
    const int tid = threadIdx.x % NT;
    const int64_t nv = R.vecs();
    uint64_t prev = ~0ull;
    for (int k = 0; k < top; ++k) {  // the largest key below the one before
        uint64_t best = 0;
        for (int64_t j = tid; j < nv; j += NT) {
            const u32x4 v = R.load(j);
#pragma unroll
            for (int e = 0; e < Vec<T>::N; ++e) {
                const int64_t i = R.at(j) + e;
                const uint64_t key = key_of(elem<T>(v, e), (uint32_t)i);
                if (i >= 0 && i < R.V && key < prev && key > best) best = key;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, o, 64);
            best = other > best ? other : best;
        }
        row_sync<NT>();
        if ((tid & 63) == 0) kred[tid >> 6] = best;
        row_sync<NT>();
        best = kred[0];
#pragma unroll
        for (int i = 1; i < NT / 64; ++i) best = kred[i] > best ? kred[i] : best;
        prev = best;  // top <= V: there is one
        if (tid == 0) out[k] = best;
    }
    row_sync<NT>();
}

// NV > 0: the row in registers, NV vectors a lane; NV = 0: streamed. KEEP: a
// backward pass will read the rows again (4096 fp32 rows, both passes: 152 us, 173
// with loads past the caches; alone they cost 4096 bf16 rows 34 us, and 31 past)
template <typename T, int NT, int NV, bool KEEP>
__global__ __launch_bounds__(NT * rows_per_block(NT), NT == 1024 ? 8 : 6) void token_logprobs_kernel(FwdArgs a) {
    constexpr int W = NT / 64, N = Vec<T>::N, NR = NV ? NV : 1, UN = 4, RB = rows_per_block(NT);
    __shared__ float lmax_[RB][NT], rs_[RB][W], rt_[RB][W];
    __shared__ u32x4 vecs_[RB][VCAP];
    __shared__ uint32_t vec_at_[RB][VCAP];
    __shared__ uint64_t list_[RB][CAP], best_[RB][MAXTOP];
    __shared__ int count_[RB][2];
    const int tid = threadIdx.x % NT, lane = tid & 63, w = tid >> 6, sub = threadIdx.x / NT;
    const int64_t row = (int64_t)blockIdx.x * RB + sub;
    if (RB > 1 && row >= a.rows) return;
    float *lmax = lmax_[sub], *rs = rs_[sub], *rt = rt_[sub];
    int* count = count_[sub];
    const Row<T> R(a.x, row, a.ld, a.V);
    const int64_t nv = R.vecs();
    int64_t y = 0;
    float xy = 0.f;
    if (tid == 0) {
        count[0] = count[1] = 0;
        y = a.tok[row];
        if (y >= 0 && y < a.V) xy = (float)R.x[y];
    }
    // whether this wave's i-th vectors hold any of the row (uniform; the count is made
    // opaque between the passes, or the compiler copies what follows for each of its values)
    int left = __builtin_amdgcn_readfirstlane((int)min(nv, (int64_t)1 << 30) - w * 64);
    auto live = [&](int i) { return i * NT < left; };
    u32x4 v[NR];
    float vm[NR], m = -INFINITY;
    Sums sum;
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) v[i] = R.whole(i * NT + tid) ? R.template inner<KEEP>(i * NT + tid) : R.none();
        // the row's first and last vector, where they are not whole
        const int je = (int)nv - 1;
        if (tid == 0 && !R.whole(0)) v[0] = R.edge(0);
        if (je > 0 && tid == je % NT && !R.whole(je)) {
            const u32x4 u = R.edge(je);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i == je / NT) v[i] = u;
        }
        asm volatile("" : "+s"(left));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            vm[i] = -INFINITY;
            if (live(i)) vm[i] = vec_max<T>(v[i]);
            m = fmaxf(m, vm[i]);
        }
    } else {
        for (int64_t j = tid; j < nv; j += UN * NT) {
            u32x4 u[UN];
            float mn = m;
#pragma unroll
            for (int i = 0; i < UN; ++i) u[i] = R.load(j + i * NT);
#pragma unroll
            for (int i = 0; i < UN; ++i) mn = fmaxf(mn, vec_max<T>(u[i]));
            const float mf = finite_or_0(mn);
            sum.rescale(m == -INFINITY ? 0.f : mn - m);
            m = mn;
#pragma unroll
            for (int i = 0; i < UN; ++i) sum.template add<T>(u[i], mf);
        }
    }
    float g = m;
    if constexpr (W > 1) {
        lmax[tid] = m;
        row_sync<NT>();
        g = lmax[lane];
#pragma unroll
        for (int i = 1; i < W; ++i) g = fmaxf(g, lmax[i * 64 + lane]);
    }
    // every wave: from the maxima of 64 sets of lanes the row's maximum and the bound for the top k
    const float tau = a.top ? kth_bound(g, a.top) : 0.f;
    g = wave_max(g);
    const float M = g, Mf = finite_or_0(M);
    auto push = [&](u32x4 u, int64_t j) {
        const int at = atomicAdd(&count[0], 1);
        if (at < VCAP) vecs_[sub][at] = u, vec_at_[sub][at] = (uint32_t)j;
    };
    if constexpr (NV > 0) {
        asm volatile("" : "+s"(left));
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) sum.template add<T>(v[i], Mf);
        asm volatile("" : "+s"(left));
        if (a.top)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (live(i) && vm[i] >= tau) push(v[i], i * NT + tid);
    } else {
        sum.rescale(m == -INFINITY ? 0.f : M - m);
        if (a.top && m >= tau)
            for (int64_t j = tid; j < nv; j += NT) {
                const u32x4 u = R.load(j);
                if (vec_max<T>(u) >= tau) push(u, j);
            }
    }
    float s = wave_sum(sum.s), t = wave_sum(sum.t);
    if constexpr (W > 1) {
        if (lane == 0) rs[w] = s, rt[w] = t;
        row_sync<NT>();
        s = rs[0], t = rt[0];
#pragma unroll
        for (int i = 1; i < W; ++i) s += rs[i], t += rt[i];
    }
    const bool empty = M == -INFINITY && s == 0.f;   // no distribution
    const float ls = M == -INFINITY ? s : logf(s);   // no finite logit: 0, or NaN if one is
    if (tid == 0) {
        a.lp[row] = y >= 0 && y < a.V ? (empty ? -INFINITY : (xy - M) - ls) : 0.f;
        a.ent[row] = empty ? 0.f : ls - t / s;
        if (a.stats) a.stats[2 * row] = M, a.stats[2 * row + 1] = ls;
    }
    if (!a.top) return;
    if constexpr (W == 1) row_sync<NT>();
    uint64_t* list = list_[sub];
    auto put = [&](int k, uint64_t key) {
        const uint32_t i = key_index(key);
        a.top_id[row * a.top + k] = i;
        a.top_lp[row * a.top + k] = empty ? -INFINITY : ((float)R.x[i] - M) - ls;
    };
    // the listed vectors' elements that reach the bound
    const int nvec = min(count[0], VCAP + 1);
    if (nvec <= VCAP) {
        for (int c = tid; c < nvec * N; c += NT) {
            const float f = elem<T>(vecs_[sub][c / N], c % N);
            const int64_t i = R.at(vec_at_[sub][c / N]) + c % N;
            if (f >= tau && i >= 0 && i < a.V) {
                const int at = atomicAdd(&count[1], 1);
                if (at < CAP) list[at] = key_of(f, (uint32_t)i);
            }
        }
    }
    row_sync<NT>();
    const int n = count[1];
    if (nvec > VCAP || n > CAP || s != s) {  // (uniform) too many for the lists, or NaN, which no bound reaches
        top_slow<T, NT>(R, a.top, list, best_[sub]);
        if (tid < a.top) put(tid, best_[sub][tid]);
        return;
    }
    for (int c = tid; c < n; c += NT) {
        const uint64_t key = list[c];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += list[i] > key;
        if (rank < a.top) put(rank, key);
    }
}

struct BwdArgs {
    const void* x;
    void* dx;
    int64_t ld, ldd, V;
    const int64_t *tok, *top_id;
    const float *g_lp, *g_ent, *g_top, *stats, *ent;
    int64_t rows;
    int top;
};

template <typename T>
__device__ __forceinline__ u32x4 pack(const float* d);
template <>
__device__ __forceinline__ u32x4 pack<float>(const float* d) {
    return (u32x4){__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3])};
}
template <>
__device__ __forceinline__ u32x4 pack<bf16>(const float* d) {
    union { bf16x8 b; u32x4 u; } r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.b[e] = (bf16)d[e];
    return r.u;
}

// Streamed: read and written once, bound by that. Rows are taken last first, so
// that what the forward pass read last is found in the memory-side cache, and the
// gradient is stored past the caches, so that it stays there (4096 x 17914 fp32,
// both passes: 184 us; last row first 183; stores past the caches 160; both 152).
// The given token's and the alternatives' elements are written again at the end,
// with their own terms.
template <typename T, int NT>
__global__ __launch_bounds__(NT * rows_per_block(NT)) void token_logprobs_bwd_kernel(BwdArgs a) {
    constexpr int N = Vec<T>::N, UN = 2, RB = rows_per_block(NT);
    const int tid = threadIdx.x % NT, w0 = tid & ~63;
    const int64_t row = a.rows - 1 - ((int64_t)blockIdx.x * RB + threadIdx.x / NT);
    if (RB > 1 && row < 0) return;
    const Row<T> R(a.x, row, a.ld, a.V);
    T* dx = (T*)a.dx + row * a.ldd;
    const bool same = (((uintptr_t)dx ^ (uintptr_t)R.x) & 15) == 0;  // both rows' vectors coincide
    const float M = a.stats[2 * row], ls = a.stats[2 * row + 1], ls2 = ls * LOG2E;
    const int64_t y = a.tok[row], nv = R.vecs();
    const float gy = a.g_lp && y >= 0 && y < a.V ? a.g_lp[row] : 0.f, gh = a.g_ent ? a.g_ent[row] : 0.f;
    float c = gy;
    if (a.g_top)
        for (int k = 0; k < a.top; ++k) c += a.g_top[row * a.top + k];
    const bool empty = M == -INFINITY && ls == 0.f;
    // -p sum g - g_H p (lp + H). No product exceeds the result's size (a loss scale may
    // bring gradients near the largest number), and lp of a masked element, whose p is 0,
    // is kept finite: p is 0 from lp = -104 on, H is at most log V
    const float lsh = ls - a.ent[row];
    auto smooth = [&](float x) {
        const float d = x - M, p = __builtin_amdgcn_exp2f(fmaf(d, LOG2E, -ls2));
        return empty ? 0.f : -fmaf(p, c, gh * p * fmaxf(d - lsh, -256.f));
    };
    for (int64_t j1 = 0; j1 < nv; j1 += UN * NT) {
        const int64_t j0 = j1 + tid;
        u32x4 v[UN];
        auto live = [&](int u) { return j1 + u * NT + w0 < nv; };  // (uniform over the wave)
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (live(u)) v[u] = R.load(j0 + u * NT);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (!live(u)) break;
            float d[N];
#pragma unroll
            for (int e = 0; e < N; ++e) d[e] = smooth(elem<T>(v[u], e));
            const int64_t i0 = R.at(j0 + u * NT);
            if (same && i0 >= 0 && i0 + N <= a.V) {
                __builtin_nontemporal_store(pack<T>(d), (u32x4*)(dx + i0));
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (i0 + e >= 0 && i0 + e < a.V) dx[i0 + e] = (T)d[e];
            }
        }
    }
    // the rest overwrites elements that other lanes have written: their stores first
    if constexpr (NT > 64) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"), __builtin_amdgcn_wave_barrier();
    const int picks = 1 + (a.g_top ? a.top : 0);
    if (tid < picks) {
        const int64_t i = tid == 0 ? y : a.top_id[row * a.top + tid - 1];
        if (i >= 0 && i < a.V && !empty) {
            float d = smooth((float)R.x[i]) + (i == y ? gy : 0.f);  // every pick of one element gives the same
            for (int k = 0; k < picks - 1; ++k) d += a.top_id[row * a.top + k] == i ? a.g_top[row * a.top + k] : 0.f;
            dx[i] = (T)d;
        }
    }
}

// A launch takes fewer than 2^32 lanes; a row up to 1024 of them. More rows go in several.
constexpr int64_t LAUNCH_ROWS = (1ll << 22) - 1;
template <typename T>
T* shift(T* p, int64_t n) { return p ? p + n : p; }

// the variant goes by the rows of the whole call
template <typename T, bool KEEP>
void launch_fwd(const FwdArgs& all, int64_t r0, int64_t n, hipStream_t s) {
    const int64_t rows = all.rows;
    FwdArgs a = all;
    a.x = (const T*)a.x + r0 * a.ld;
    a.tok += r0, a.lp += r0, a.ent += r0, a.stats = shift(a.stats, 2 * r0);
    a.top_id = shift(a.top_id, r0 * a.top), a.top_lp = shift(a.top_lp, r0 * a.top);
    a.rows = n;
    const int64_t vecs = (a.V + 2 * (Vec<T>::N - 1)) / Vec<T>::N;  // whatever the row's alignment
#define FWD(NT, NV)                                                                                      \
    do {                                                                                                 \
        if (vecs <= NT * NV) {                                                                           \
            constexpr int RB = rows_per_block(NT);                                                       \
            const dim3 g((unsigned)((n + RB - 1) / RB));                                                 \
            hipLaunchKernelGGL((token_logprobs_kernel<T, NT, NV, KEEP>), g, dim3(NT * RB), 0, s, a);     \
            return;                                                                                      \
        }                                                                                                \
    } while (0)
    // many rows: as few lanes a row as hold it, for many rows a CU (4096 bf16 rows of 17914 with 5 alternatives:
    // 31 us, 57 with 1024 lanes; 65536 of 568: 32, 85 with 256); few: as many lanes as help
    FWD(64, 1);
    if (rows >= 1024) {
        FWD(64, 3);
        FWD(64, 9);
        FWD(256, 9);
        FWD(512, 9);
    } else {
        FWD(256, 1);
    }
    FWD(1024, 1);
    FWD(1024, 2);
    FWD(1024, 9);
#undef FWD
    hipLaunchKernelGGL((token_logprobs_kernel<T, 1024, 0, KEEP>), dim3((unsigned)n), dim3(1024), 0, s, a);
}
template <typename T>
void launch_bwd(const BwdArgs& all, int64_t r0, int64_t n, hipStream_t s) {
    const int64_t rows = all.rows, vecs = all.V / Vec<T>::N;
    BwdArgs a = all;
    a.x = (const T*)a.x + r0 * a.ld, a.dx = (T*)a.dx + r0 * a.ldd;
    a.tok += r0, a.stats += 2 * r0, a.ent += r0;
    a.g_lp = shift(a.g_lp, r0), a.g_ent = shift(a.g_ent, r0);
    a.g_top = shift(a.g_top, r0 * a.top), a.top_id = shift(a.top_id, r0 * a.top);
    a.rows = n;
    const dim3 g((unsigned)n);
    // long rows by 1024 lanes (rows of 17914 fp32, both passes: 4096 in 146 us, 16384 in 578; by 256 lanes 154 and
    // 618), others by 256 (65536 rows of 17914 bf16: 1251 us, 1284 by 1024): even near 2500 vectors
    if (vecs <= 256)
        hipLaunchKernelGGL((token_logprobs_bwd_kernel<T, 64>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, s, a);
    else if (rows >= 1024 && vecs <= 2560) hipLaunchKernelGGL((token_logprobs_bwd_kernel<T, 256>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((token_logprobs_bwd_kernel<T, 1024>), g, dim3(1024), 0, s, a);
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
    const FwdArgs a{logits, ld, V, tokens, logprob, entropy, stats, top_logprobs, top_ids, rows, (int)top};
    hipStream_t s = (hipStream_t)stream;
    for (int64_t r = 0; r < rows; r += LAUNCH_ROWS) {
        const int64_t n = std::min(LAUNCH_ROWS, rows - r);
        if (dtype == MSQ_BF16) stats ? launch_fwd<bf16, true>(a, r, n, s) : launch_fwd<bf16, false>(a, r, n, s);
        else stats ? launch_fwd<float, true>(a, r, n, s) : launch_fwd<float, false>(a, r, n, s);
    }
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
    const BwdArgs a{logits, dlogits, ld, ldd, V, tokens, top_ids, g_logprob, g_entropy, g_top, stats, entropy, rows, (int)top};
    for (int64_t r = (rows - 1) / LAUNCH_ROWS * LAUNCH_ROWS; r >= 0; r -= LAUNCH_ROWS) {  // last rows first
        const int64_t n = std::min(LAUNCH_ROWS, rows - r);
        if (dtype == MSQ_BF16) launch_bwd<bf16>(a, r, n, (hipStream_t)stream);
        else launch_bwd<float>(a, r, n, (hipStream_t)stream);
    }
    MSQ_LAUNCH_CHECK();
    return MSQ_OK;
}
