// Log probabilities of given tokens with entropy, rank and top alternatives from logits rows, and their gradient
// (sm_100a).  No counterpart in the reference, whose call sites stop at the token.
//
// With z = x / T and c = log2(e) / T, everything is kept in base 2 around a reference R = fl(m c) of the running
// maximum m: y_i = fma(x_i, c, -R) (one rounding of the exact x_i c - R, and R drops out of every difference, so R
// need not be exact), S = sum 2^y, U = sum 2^y y.  Then logprob = (y_t - log2 S) ln 2 and the entropy
// H = (log2 S - U / S) ln 2: U <= 0 but for R's rounding (at most 2^-5 of S), so that nothing cancels.  S and U are fp32
// per thread (a few hundred terms each) and merged pairwise; a merge of two references shifts y by R_a - R_b.
// Beyond |R| = 2^20 (finite masks, logits by the million, small temperatures) y = (x - m) c instead (lp_far).  A masked (-inf) element adds nothing; a row with nothing left has logprob -inf, entropy 0
// and gradient 0; NaN or +inf anywhere makes the row NaN, as a softmax gives it.
//
// Forward, one pass over the row by bulk copies into a ring of shared-memory chunks (a thread's registers do not bound
// the bytes in flight), 128 or 256 threads per row where rows are many, else 512 and a cluster of CTAs per row while rows
// are few; many short rows without alternatives take a warp each, from registers.  Two elements share one packed fp32 operation, and a bf16 pair one maximum and one comparison: about 6
// instructions an element, so that bf16 rows stay bound by HBM.  The rank counts the elements before the token in (value
// descending, id ascending) order: an element before the token counts when x >= x_t, i.e. x > pred(x_t), one after it
// when x > x_t, so a vector needs one threshold.  Top alternatives: the
// top-th largest of the warps' largest thread maxima bounds the CTA's top-th value from below (each is a distinct
// element), and what reaches the bound is listed, element by element of the threads whose maximum does, and ordered by
// rank counting.  Where the CTA's part of the row fits the ring this happens once, from shared memory, after the last
// chunk.  Longer parts list on the way, with a bound from the first chunk that is taken again after 4, 16, .. chunks, so
// that about 3 `top` elements are listed while what was read grows fourfold.  Where too few threads hold anything (short
// or masked rows) every finite element is listed and the first masked ids fill what is missing.  A list that overflows is
// made again in a second pass (L2) from a last bound, and where ties overflow that too, by an exact radix select.
//
// Backward, elementwise: dx = (g_lp ([i = t] - p) - g_H p (log p + H)) / T with p = 2^(y - log2 S) recomputed from
// the saved reference: one read and one write of the row.
#include <cooperative_groups.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "../../include/b2s_sampler.h"
#include "b2s_device.cuh"
#include "b2s_logprobs.cuh"

namespace cg = cooperative_groups;

namespace b2s {

int cuda_fail(cudaError_t e);

cudaError_t device_sms(int* sms) {
    static std::atomic<int> cached[64];  // 0: not asked yet; a device's count never changes, so racing writers agree
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64 && cached[dev].load(std::memory_order_relaxed) > 0) {
        *sms = cached[dev].load(std::memory_order_relaxed);
        return cudaSuccess;
    }
    e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess && dev >= 0 && dev < 64) cached[dev].store(*sms, std::memory_order_relaxed);
    return e;
}

static std::atomic<long long> g_wait_limit{GM_WAIT};
long long wait_limit() { return g_wait_limit.load(std::memory_order_relaxed); }

namespace {

constexpr int LP_CAP = 512;      // candidate list entries per CTA
constexpr int LP_GATHER = 64;    // thread maxima gathered per CTA, at most
constexpr int LP_MAX_TOP = 32;
constexpr int LP_KEPT = 128;     // words of the histogram's room
constexpr int LP_U = 4;          // vectors per thread and chunk

// The largest float below x (x not NaN); NaN for -inf, whose "x > pred" must hold for every element.
__device__ __forceinline__ float pred_float(float x) {
    if (x == f_ninf()) return __int_as_float(0x7fffffff);
    if (x == 0.0f) return __int_as_float((int)0x80000001u);
    const int b = __float_as_int(x);
    return __int_as_float(x > 0.0f ? b - 1 : b + 1);
}

template <typename E>
struct LpElem;
template <>
struct LpElem<float> {
    static constexpr int EPV = 4;
    typedef float Thr;
    static __device__ __forceinline__ Thr threshold(float xt) { return xt; }
    static __device__ __forceinline__ Thr threshold_before(float xt) { return pred_float(xt); }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
    static __device__ __forceinline__ float batch_max(const uint4 (&q)[LP_U]) {
        float m = __uint_as_float(q[0].x);
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            m = fmax_nan(m, fmax_nan(__uint_as_float(q[u].x), __uint_as_float(q[u].y)));
            m = fmax_nan(m, fmax_nan(__uint_as_float(q[u].z), __uint_as_float(q[u].w)));
        }
        return m;
    }
    static __device__ __forceinline__ float vec_max(uint4 q) {
        return fmax_nan(fmax_nan(__uint_as_float(q.x), __uint_as_float(q.y)), fmax_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
    // elements above the threshold, or NaN
    static __device__ __forceinline__ int count_above(uint4 q, Thr t) {
        return !(__uint_as_float(q.x) <= t) + !(__uint_as_float(q.y) <= t) + !(__uint_as_float(q.z) <= t) +
               !(__uint_as_float(q.w) <= t);
    }
    static __device__ __forceinline__ float ld(const void* p, int64_t i) { return __ldg(static_cast<const float*>(p) + i); }
    static __device__ __forceinline__ float ld_shared(const uint4* p, int j) { return reinterpret_cast<const float*>(p)[j]; }
    static __device__ __forceinline__ void unpack(uint4 q, float (&x)[4]) {
        x[0] = __uint_as_float(q.x); x[1] = __uint_as_float(q.y); x[2] = __uint_as_float(q.z); x[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    static __device__ __forceinline__ void st(void* p, int64_t i, float v) { static_cast<float*>(p)[i] = v; }
};
template <>
struct LpElem<__nv_bfloat16> {
    static constexpr int EPV = 8;
    typedef __nv_bfloat162 Thr;
    static __device__ __forceinline__ __nv_bfloat162 as2(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
    static __device__ __forceinline__ Thr both(uint32_t bits) { return as2(bits | bits << 16); }
    static __device__ __forceinline__ Thr threshold(float xt) { return both(__float_as_uint(xt) >> 16); }
    // the largest bf16 below xt; NaN for -inf
    static __device__ __forceinline__ Thr threshold_before(float xt) {
        const uint32_t b = __float_as_uint(xt) >> 16;
        if (xt == f_ninf()) return both(0x7fffu);
        if (xt == 0.0f) return both(0x8001u);
        return both(xt > 0.0f ? b - 1u : b + 1u);
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
    static __device__ __forceinline__ float batch_max(const uint4 (&q)[LP_U]) {
        __nv_bfloat162 m = as2(q[0].x);
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            m = __hmax2_nan(m, __hmax2_nan(as2(q[u].x), as2(q[u].y)));
            m = __hmax2_nan(m, __hmax2_nan(as2(q[u].z), as2(q[u].w)));
        }
        return fmax_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ float vec_max(uint4 q) {
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(as2(q.x), as2(q.y)), __hmax2_nan(as2(q.z), as2(q.w)));
        return fmax_nan(__low2float(m), __high2float(m));
    }
    // elements above the threshold, or NaN: a true comparison is a 0xffff half, whose low byte is -1
    static __device__ __forceinline__ int count_above(uint4 q, Thr t) {
        int n = __dp4a((int)__hgtu2_mask(as2(q.x), t), 0x00010001, 0);
        n = __dp4a((int)__hgtu2_mask(as2(q.y), t), 0x00010001, n);
        n = __dp4a((int)__hgtu2_mask(as2(q.z), t), 0x00010001, n);
        n = __dp4a((int)__hgtu2_mask(as2(q.w), t), 0x00010001, n);
        return -n;
    }
    static __device__ __forceinline__ float ld(const void* p, int64_t i) {
        return bf16_bits_to_f(__ldg(static_cast<const unsigned short*>(p) + i));
    }
    static __device__ __forceinline__ float ld_shared(const uint4* p, int j) {
        return bf16_bits_to_f(reinterpret_cast<const unsigned short*>(p)[j]);
    }
    static __device__ __forceinline__ void unpack(uint4 q, float (&x)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    }
    // one rounding to bf16, the element type of the logits whose gradient this is
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void st(void* p, int64_t i, float v) {
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    }
};

// order key of a value: NaN above every number, the zeros equal
__device__ __forceinline__ uint32_t rank_key(float x) { return x != x ? 0xffffffffu : okey(x); }
// (value descending, id ascending) as one word: the larger word comes first
__device__ __forceinline__ unsigned long long rank_word(float x, int id) {
    return ((unsigned long long)rank_key(x) << 32) | (0xffffffffu - (uint32_t)id);
}
__device__ __forceinline__ int word_id(unsigned long long w) { return (int)(0xffffffffu - (uint32_t)w); }

struct LpLists {
    alignas(16) uint32_t gather[LP_GATHER];
    uint32_t bound;  // the last bound, 0: none
    int n_list;
    int ties[16];
    alignas(16) uint32_t hist[256];
    uint32_t ctl[2];
    unsigned long long list[LP_CAP];
    unsigned long long top[LP_MAX_TOP];      // this CTA's best, in order (0: none)
    unsigned long long all[8 * LP_MAX_TOP];  // the cluster's, in its first CTA
};
struct LpNoLists {};
template <int NTH, bool TOP>
struct LpShared : std::conditional_t<TOP, LpLists, LpNoLists> {
    static constexpr int WARPS = NTH / 32;
    uint64_t full[6], empty[6];
    float wmax[WARPS];
    float wS[WARPS], wU[WARPS];
    int wcount[WARPS];
    int failed;
    int loaded;  // chunks asked for, by thread 0
    LpState total[8];  // the cluster's states and counts, in its first CTA
    int total_count[8];
};

struct LpArgs {
    const void* logits;
    int64_t stride;
    int V, per, top, stages;
    float c;
    long long wait;  // clocks a wait takes at most; 0: nothing is loaded and the rows count as given up
    const int64_t* tokens;
    float *logprob, *entropy;
    int64_t *rank, *top_ids;
    float* top_logprobs;
    float4* stats;
    uint32_t* status;
};

// A thread's running statistics: two lanes of S and U that packed operations add to.
struct LpThread {
    float m;
    float2 S, U;
};
__device__ __forceinline__ void lp_thread_rescale(LpThread& s, float m, float c) {
    if (s.m != f_ninf()) {
        const float d = lp_shift(s.m, m, c), f = ex2(d);
        s.U = make_float2(f * __fmaf_rn(d, s.S.x, s.U.x), f * __fmaf_rn(d, s.S.y, s.U.y));
        s.S = make_float2(f * s.S.x, f * s.S.y);
    }
    s.m = m;
}
// One value, by the thread's first lane, whatever the reference.
__device__ __forceinline__ void lp_thread_add(LpThread& s, float x, float c) {
    const float m = fmax_nan(s.m, x);
    if (!(fabsf(m) <= 3.402823466e38f)) {
        s.m = m;
        return;
    }
    if (m > s.m) lp_thread_rescale(s, m, c);
    const float y = lp_y(x, s.m, c), e = ex2(y);
    s.S.x += e;
    s.U.x = __fmaf_rn(e, y, s.U.x);
}
// LP_U vectors whose maximum is bm: the maximum moved, then packed sums.
template <typename E>
__device__ __forceinline__ void lp_thread_batch(LpThread& s, const uint4 (&q)[LP_U], float bm, float c) {
    if (!(bm <= s.m)) {  // larger, or NaN
        const float m = fmax_nan(s.m, bm);
        if (fabsf(m) <= 3.402823466e38f) lp_thread_rescale(s, m, c);
        else s.m = m;
    }
    if (!(fabsf(s.m) <= 3.402823466e38f)) return;  // NaN or +inf (the row's outcome), or nothing but -inf so far
    const float R = __fmul_rn(s.m, c);
    if (!lp_far(R)) {
        const float2 c2 = make_float2(c, c), r2 = make_float2(-R, -R);
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            float x[LpElem<E>::EPV];
            LpElem<E>::unpack(q[u], x);
#pragma unroll
            for (int j = 0; j < LpElem<E>::EPV; j += 2) {
                float2 y = __ffma2_rn(make_float2(x[j], x[j + 1]), c2, r2);
                y = make_float2(fmaxf(y.x, -200.0f), fmaxf(y.y, -200.0f));  // a masked element: 0 * -200
                const float2 e = make_float2(ex2(y.x), ex2(y.y));
                s.S = __fadd2_rn(s.S, e);
                s.U = __ffma2_rn(e, y, s.U);
            }
        }
    } else {  // a reference far from zero: (x - m) c
        const float2 c2 = make_float2(c, c), m2 = make_float2(-s.m, -s.m);
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            float x[LpElem<E>::EPV];
            LpElem<E>::unpack(q[u], x);
#pragma unroll
            for (int j = 0; j < LpElem<E>::EPV; j += 2) {
                float2 y = __fmul2_rn(__fadd2_rn(make_float2(x[j], x[j + 1]), m2), c2);
                y = make_float2(fmaxf(y.x, -200.0f), fmaxf(y.y, -200.0f));
                const float2 e = make_float2(ex2(y.x), ex2(y.y));
                s.S = __fadd2_rn(s.S, e);
                s.U = __ffma2_rn(e, y, s.U);
            }
        }
    }
}

// The top `need` words of elements [0, n) of this CTA's part of the row (element i has id lo + i), exactly, whatever
// the ties: the need-th largest value by radix select, then everything above it and the first ties in id order.
// Every thread calls it; sh.list holds min(need, n) words afterwards.
template <typename E, int NTH>
__device__ __noinline__ void exact_top(LpLists& sh, const void* rowp, int lo, int n, int need) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    need = min(need, n);
    auto key = [&](int i) { return rank_key(LpElem<E>::ld(rowp, lo + i)); };
    __syncthreads();
    const uint32_t kth = block_kth_largest<NTH>(n, need, key, sh.hist, sh.ctl);
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NTH) {
        const float x = LpElem<E>::ld(rowp, lo + i);
        if (rank_key(x) > kth) sh.list[atomicAdd(&sh.n_list, 1)] = rank_word(x, lo + i);  // fewer than need <= LP_CAP
    }
    __syncthreads();
    int have = sh.n_list;
    for (int b = 0; b < n && have < need; b += NTH) {
        const int i = b + tid;
        const float x = i < n ? LpElem<E>::ld(rowp, lo + i) : 0.0f;
        const bool tie = i < n && rank_key(x) == kth;
        const uint32_t who = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) sh.ties[warp] = __popc(who);
        __syncthreads();
        int at = have, total = 0;
#pragma unroll
        for (int w = 0; w < NTH / 32; ++w) {
            at += w < warp ? sh.ties[w] : 0;
            total += sh.ties[w];
        }
        at += __popc(who & ((1u << lane) - 1u));
        if (tie && at < need) sh.list[at] = rank_word(x, lo + i);
        have += total;
        __syncthreads();
    }
    if (tid == 0) sh.n_list = need;
    __syncthreads();
}

// How many of the n words of `list` come before the i-th (i < n), by 8 lanes a word; the warp calls it converged.
__device__ __forceinline__ int rank_of(const unsigned long long* list, int n, int i) {
    const unsigned long long w = i < n ? list[i] : 0ull;
    int r = 0;
#pragma unroll 2
    for (int j = threadIdx.x & 7; j < n; j += 8) r += list[j] > w;
    r += __shfl_xor_sync(0xffffffffu, r, 1);
    r += __shfl_xor_sync(0xffffffffu, r, 2);
    return r + __shfl_xor_sync(0xffffffffu, r, 4);
}
// Orders n words (distinct) of `list` into out[0 .. top): out[k] the k-th largest, 0 where there are fewer.
template <int NTH>
__device__ __forceinline__ void order_words(const unsigned long long* list, int n, unsigned long long* out, int top) {
    for (int k = threadIdx.x; k < top; k += NTH)
        if (k >= n) out[k] = 0ull;
    for (int b = 0; b < n; b += NTH / 8) {
        const int i = b + (int)(threadIdx.x >> 3), r = rank_of(list, n, i);
        if ((threadIdx.x & 7) == 0 && i < n && r < top) out[r] = list[i];
    }
}

// Whether a value reaches the bound (as a value: NaN does).
__device__ __forceinline__ bool reaches(float x, float bound) { return !(x < bound); }
__device__ __forceinline__ float bound_value(uint32_t bound) {
    return bound == 0xffffffffu || bound > 0xff800000u ? __int_as_float(0x7f800000) : okey_to_f(bound);  // NaN only: +inf
}

// The bound (see above) from this thread's maximum so far: an order key that at least `top` elements reach, or, where
// there are fewer maxima than that, the one above -inf's.  Every thread calls it.  A gathered word is a key without its
// last 6 bits and the complement of its place, so that words differ; the bound they give is lower by less than 64 keys.
// The first `warps` warps hold something.
template <int NTH>
__device__ __noinline__ float top_bound(LpLists& sh, int top, int warps, float tmax) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // enough rounds for `top` maxima and a few to spare
    const int rounds = min(LP_GATHER / warps, (top + warps - 1) / warps + 2), gathered = rounds * warps;
    uint32_t k = tmax == f_ninf() ? 0u : rank_key(tmax);
#pragma unroll 1
    for (int g = 0; g < (warp < warps ? rounds : 0); ++g) {
        const uint32_t mx = __reduce_max_sync(0xffffffffu, k);
        const int at = warp * rounds + g;
        if (lane == 0) sh.gather[at] = (mx & ~63u) | (63u - (uint32_t)at);
        const uint32_t who = __ballot_sync(0xffffffffu, k == mx);
        if (lane == __ffs(who) - 1) k = 0u;
    }
    if (tid >= gathered && tid < LP_GATHER) sh.gather[tid] = 63u - (uint32_t)tid;
    __syncthreads();
    if (tid < LP_GATHER) {
        const uint32_t mine = sh.gather[tid];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < LP_GATHER; j += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(&sh.gather[j]);
            r += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
        }
        if (r == top - 1) sh.bound = mine & ~63u;
    }
    __syncthreads();
    return bound_value(sh.bound ? sh.bound : rank_key(f_ninf()) + 1u);
}

// Appends the lanes' elements that reach the bound, one shared atomic for all of them; the warp calls it converged.
__device__ __forceinline__ void offer(LpLists& sh, float bound, bool there, float x, int id) {
    const int lane = threadIdx.x & 31;
    const bool pass = there && reaches(x, bound);
    const uint32_t who = __ballot_sync(0xffffffffu, pass);
    if (who == 0u) return;
    int at = 0;
    if (lane == 0) at = atomicAdd(&sh.n_list, __popc(who));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
    if (pass && at < LP_CAP) sh.list[at] = rank_word(x, id);
}
template <typename E>
__device__ __noinline__ void offer_vec(LpLists& sh, float bound, bool there, uint4 q, int id) {
    if (!__any_sync(0xffffffffu, there && reaches(LpElem<E>::vec_max(q), bound))) return;
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {  // a word at a time, the next one moved to the front
        if (LpElem<E>::EPV == 4) {
            offer(sh, bound, there, __uint_as_float(q.x), id + j);
        } else {
            offer(sh, bound, there, __uint_as_float(q.x << 16), id + 2 * j);
            offer(sh, bound, there, __uint_as_float(q.x & 0xffff0000u), id + 2 * j + 1);
        }
        q.x = q.y;
        q.y = q.z;
        q.z = q.w;
    }
}

// The `top` best words of this CTA's part into sh.top, from the list (n_list entries offered).
template <typename E, int NTH>
__device__ __forceinline__ void finish_top(LpLists& sh, int top, int warps, float tmax, const unsigned char* rowp, int lo,
                                           int n, int nh, int nv, const uint4* vp) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __syncthreads();
    if (sh.n_list > LP_CAP) {  // again, with the bound that all maxima give
        const float bound = top_bound<NTH>(sh, top, warps, tmax);
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
#pragma unroll 1
        for (int b = warp * 32; b < nv; b += NTH) {
            if (*reinterpret_cast<volatile int*>(&sh.n_list) > LP_CAP) break;
            const int v = b + lane;
            offer_vec<E>(sh, bound, v < nv, v < nv ? ldg_stream(vp + v) : LpElem<E>::nothing(), lo + nh + v * LpElem<E>::EPV);
        }
        if (warp == 0) {  // the ragged ends: fewer than 16 elements
            const int tail = n - nh - nv * LpElem<E>::EPV;
            const int i = lane < 16 ? (lane < nh ? lane : n) : (lane - 16 < tail ? n - tail + lane - 16 : n);
            offer(sh, bound, i < n, i < n ? LpElem<E>::ld(rowp, lo + i) : 0.0f, lo + i);
        }
        __syncthreads();
        if (sh.n_list > LP_CAP) exact_top<E, NTH>(sh, rowp, lo, n, top);
    } else if (sh.n_list < top && warp == 0) {
        // every finite element is listed; the masked ones follow in id order
        int have = sh.n_list;
        __syncwarp();
        const int need = min(top, n);
        for (int b = 0; b < n && have < need; b += 32) {
            const bool tie = b + lane < n && LpElem<E>::ld(rowp, lo + b + lane) == f_ninf();
            const uint32_t who = __ballot_sync(0xffffffffu, tie);
            const int at = have + __popc(who & ((1u << lane) - 1u));
            if (tie && at < need) sh.list[at] = rank_word(f_ninf(), lo + b + lane);
            have = min(need, have + __popc(who));
        }
        if (lane == 0) sh.n_list = have;
    }
    __syncthreads();
    const unsigned long long* list = sh.list;
    int listed = sh.n_list;
    if (listed > 2 * top + 64) {  // listed on the way, with lower bounds: what the last one leaves, where that is less
        const float bound = top_bound<NTH>(sh, top, warps, tmax);
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
        unsigned long long* kept = reinterpret_cast<unsigned long long*>(sh.hist);  // the radix select is done with it
        const unsigned long long least = (unsigned long long)rank_key(bound) << 32;
        for (int b = 0; b < listed; b += NTH) {
            const unsigned long long w = b + tid < listed ? sh.list[b + tid] : 0ull;
            if (w >= least) {
                const int at = atomicAdd(&sh.n_list, 1);
                if (at < LP_KEPT) kept[at] = w;
            }
        }
        __syncthreads();
        if (sh.n_list <= LP_KEPT) {
            list = kept;
            listed = sh.n_list;
        }
    }
    order_words<NTH>(list, listed, sh.top, top);
}

template <typename E, int NTH, bool TOP>
__global__ void __launch_bounds__(NTH, 1024 / NTH) token_logprobs_kernel(const LpArgs a) {
    constexpr int EPV = LpElem<E>::EPV, ES = 16 / EPV, WARPS = NTH / 32;
    constexpr int VPC = LP_U * NTH;  // vectors per chunk
    __shared__ LpShared<NTH, TOP> sh;
    extern __shared__ __align__(128) unsigned char ring[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
    const int r = (int)(blockIdx.x / C);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned char* rowp = static_cast<const unsigned char*>(a.logits) + (int64_t)r * a.stride * ES;
    const int lo = min(a.V, crank * a.per), hi = min(a.V, lo + a.per), n = hi - lo;

    // the 16-byte interior [v0, v0 + nv vectors) of the part, a ragged head and tail
    const uintptr_t A = reinterpret_cast<uintptr_t>(rowp) + (uintptr_t)lo * ES;
    const int nh = min(n, (int)(((16 - (A & 15)) & 15) / ES));
    const int nv = (n - nh) / EPV;
    const int i0 = lo + nh;             // id of the interior's first element
    const int nt = n - nh - nv * EPV;   // tail elements
    const uint4* vp = reinterpret_cast<const uint4*>(rowp + (int64_t)i0 * ES);
    const int chunks = (nv + VPC - 1) / VPC;
    auto load_chunk = [&](int k) {  // by one thread
        const int s = k % a.stages, cnt = min(VPC, nv - k * VPC);
        mbar_arrive_expect_tx(&sh.full[s], (uint32_t)cnt * 16u);
        bulk_g2s(ring + (size_t)s * VPC * 16, vp + (int64_t)k * VPC, (uint32_t)cnt * 16u, &sh.full[s]);
        sh.loaded = k + 1;
    };
    if (C > 1) cluster_arrive_relaxed();  // waited for before the first store to another CTA
    if (tid == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], WARPS);
        }
        fence_mbar_init();
        sh.failed = a.wait <= 0;
        sh.loaded = 0;
        if constexpr (TOP) sh.n_list = sh.bound = 0;
    }
    pdl_wait_then_release();
    bool bad = a.wait <= 0;  // a wait gave up: nothing more is read, the barriers are still met
    if (tid == 0 && !bad)
        for (int k = 0; k < min(chunks, a.stages); ++k) load_chunk(k);
    const int64_t tok = a.tokens ? a.tokens[r] : -1;
    const bool has_tok = tok >= 0 && tok < a.V;
    const int t = has_tok ? (int)tok : -1;
    const float xt = has_tok ? LpElem<E>::ld(rowp, t) : 0.0f;
    const typename LpElem<E>::Thr thr_after = LpElem<E>::threshold(xt), thr_before = LpElem<E>::threshold_before(xt);
    const int tv = t >= i0 ? min(nv, (t - i0) / EPV) : 0;  // vectors below it lie before the token

    LpThread s;
    s.m = f_ninf();
    s.S = s.U = make_float2(0.0f, 0.0f);
    int cnt = 0;
    auto one = [&](float x, int id) {
        lp_thread_add(s, x, a.c);
        cnt += id != t && (x > xt || x != x || (id < t && x == xt));
    };
    if (tid < nh) one(LpElem<E>::ld(rowp, lo + tid), lo + tid);
    if (tid >= 32 && tid < 32 + nt) one(LpElem<E>::ld(rowp, hi - nt + tid - 32), hi - nt + tid - 32);
    __syncthreads();  // the mbarriers are there

    int slot = 0;
    uint32_t ph = 0;
    float bound = 0.0f;
    const int warps = min(WARPS, (max(nv, 64) + 31) / 32);  // warps that hold something (the ragged ends: two)
    for (int k = 0; k < chunks; ++k) {
        // refill the chunk before this one: its readers have had a whole chunk's time
        if (tid == 0 && k > 0 && k - 1 + a.stages < chunks && !bad) {
            const int ps = (k - 1) % a.stages;
            if (gm_wait<false>(&sh.empty[ps], (uint32_t)((k - 1) / a.stages) & 1u, a.wait)) load_chunk(k - 1 + a.stages);
            else sh.failed = 1;
        }
        if (!bad && !gm_wait<false>(&sh.full[slot], ph, a.wait)) {
            sh.failed = 1;
            bad = true;
        }
        const uint4* buf = reinterpret_cast<const uint4*>(ring + (size_t)slot * VPC * 16);
        const int left = bad ? 0 : nv - k * VPC;  // vectors of this chunk
        float bm;
        {
            uint4 q[LP_U];
            if (left >= VPC) {
#pragma unroll
                for (int u = 0; u < LP_U; ++u) q[u] = buf[tid + u * NTH];
            } else {
#pragma unroll
                for (int u = 0; u < LP_U; ++u) q[u] = tid + u * NTH < left ? buf[tid + u * NTH] : LpElem<E>::nothing();
            }
            bm = LpElem<E>::batch_max(q);
            lp_thread_batch<E>(s, q, bm, a.c);
            // the vector that holds the token counts as behind it here
            const int before = tv - k * VPC;  // vectors of this chunk before it
            if (before <= 0 || before >= VPC) {
                const typename LpElem<E>::Thr thr = before <= 0 ? thr_after : thr_before;
#pragma unroll
                for (int u = 0; u < LP_U; ++u) cnt += LpElem<E>::count_above(q[u], thr);
            } else {
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
                    cnt += LpElem<E>::count_above(q[u], tid + u * NTH < before ? thr_before : thr_after);
            }
        }
        if constexpr (TOP) {
            if (chunks > a.stages) {
                if (k == 0 || k == 3 || (k & 15) == 15) bound = top_bound<NTH>(sh, a.top, warps, s.m);
                // the shares that reach it, an element per lane
                for (uint32_t hits = __ballot_sync(0xffffffffu, reaches(bm, bound)); hits; hits &= hits - 1) {
                    const int v = (tid & ~31) + __ffs(hits) - 1 + lane / EPV * NTH;
                    const bool there = lane < LP_U * EPV && v < left;
                    const float x = there ? LpElem<E>::ld_shared(buf + v, lane % EPV) : 0.0f;
                    offer(sh, bound, there, x, i0 + (k * VPC + v) * EPV + lane % EPV);
                }
            }
        }
        if (chunks > a.stages) {
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&sh.empty[slot])) : "memory");
        }
        if (++slot == a.stages) {
            slot = 0;
            ph ^= 1;
        }
    }
    // the elements of the token's own vector before it that tie with it
    if (tid == 0 && t >= i0 && t < i0 + nv * EPV)
        for (int i = i0 + tv * EPV; i < t; ++i) cnt += LpElem<E>::ld(rowp, i) == xt;
    // a NaN token compares false with everything, so every element was counted: the ones before it are the NaN ones with
    // a smaller id
    if (has_tok && xt != xt) {
        cnt = 0;
        for (int i = lo + tid; i < min(hi, t); i += NTH) {
            const float x = LpElem<E>::ld(rowp, i);
            cnt += x != x;
        }
    }
    const float tmax = s.m;  // this thread's maximum (NaN if it saw one)
    if constexpr (TOP) {
        if (chunks <= a.stages) {  // the whole part lies in shared memory
            bound = top_bound<NTH>(sh, a.top, warps, tmax);
            const uint4* buf = reinterpret_cast<const uint4*>(ring);
            for (uint32_t hits = __ballot_sync(0xffffffffu, reaches(tmax, bound)); hits; hits &= hits - 1) {
                // a vector of the thread's share per lane (at most 24), then the elements of those that reach it
                const int v = (tid & ~31) + __ffs(hits) - 1 + lane * NTH;
                const bool there = v < nv && !bad;
                for (uint32_t vecs = __ballot_sync(0xffffffffu, there && reaches(LpElem<E>::vec_max(buf[there ? v : 0]), bound));
                     vecs; vecs &= vecs - 1) {
                    const int w = (tid & ~31) + __ffs(hits) - 1 + (__ffs(vecs) - 1) * NTH, j = lane & (EPV - 1);
                    offer(sh, bound, lane < EPV, LpElem<E>::ld_shared(buf + w, j), i0 + w * EPV + j);
                }
            }
        }
        if (warp < 2) {  // the ragged ends
            const bool head = tid < nh, tail = tid >= 32 && tid < 32 + nt;
            const int id = head ? lo + tid : hi - nt + tid - 32;
            offer(sh, bound, head || tail, head || tail ? LpElem<E>::ld(rowp, id) : 0.0f, id);
        }
    }
    // the CTA's maximum (NaN wins), then sums relative to it
    float m = s.m;
    {
        const uint32_t key = __reduce_max_sync(0xffffffffu, rank_key(m));
        m = key == 0xffffffffu ? __int_as_float(0x7fffffff) : okey_to_f(key);
    }
    if (lane == 0) sh.wmax[warp] = m;
    __syncthreads();
    m = sh.wmax[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m = fmax_nan(m, sh.wmax[w]);
    if (sh.failed) m = __int_as_float(0x7fffffff);
    float S = 0.0f, U = 0.0f;
    if (fabsf(m) <= 3.402823466e38f && s.m != f_ninf()) {
        lp_thread_rescale(s, m, a.c);
        S = s.S.x + s.S.y;
        U = s.U.x + s.U.y;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        S += __shfl_xor_sync(0xffffffffu, S, o);
        U += __shfl_xor_sync(0xffffffffu, U, o);
    }
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) {
        sh.wS[warp] = S;
        sh.wU[warp] = U;
        sh.wcount[warp] = cnt;
    }
    if constexpr (TOP) finish_top<E, NTH>(sh, a.top, warps, tmax, rowp, lo, n, nh, nv, vp);
    __syncthreads();
    LpState w;
    w.m = m;
    w.S = w.U = 0.0f;
    int c2 = 0;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
        w.S += sh.wS[k];
        w.U += sh.wU[k];
        c2 += sh.wcount[k];
    }
    if (sh.failed) c2 = -1;
    if (C > 1) {  // every CTA hands its state, count and best words to the first one
        __syncwarp();
        cluster_wait();
        LpShared<NTH, TOP>* first = cluster.map_shared_rank(&sh, 0);
        if (tid == 0) {
            first->total[crank] = w;
            first->total_count[crank] = c2;
        }
        if constexpr (TOP)
            if (tid < a.top) first->all[crank * a.top + tid] = sh.top[tid];
        __syncwarp();
        cluster_arrive_release();
        cluster_wait();
        if (crank == 0) {  // every warp for itself: the maximum, then one rescaling and a sum over the parts
            LpState o;
            o.m = f_ninf();
            o.S = o.U = 0.0f;
            c2 = 0;
            if (lane < C) {
                o = sh.total[lane];
                c2 = sh.total_count[lane];
            }
            const uint32_t key = __reduce_max_sync(0xffffffffu, rank_key(o.m));
            w.m = key == 0xffffffffu ? __int_as_float(0x7fffffff) : okey_to_f(key);
            if (fabsf(w.m) <= 3.402823466e38f && o.m != f_ninf()) lp_rescale(o, w.m, a.c);
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                o.S += __shfl_xor_sync(0xffffffffu, o.S, d);
                o.U += __shfl_xor_sync(0xffffffffu, o.U, d);
            }
            w.S = o.S;
            w.U = o.U;
            c2 = __any_sync(0xffffffffu, c2 < 0) ? -1 : __reduce_add_sync(0xffffffffu, c2);
        }
    }
    if (crank == 0) {
        const LpFinal f = lp_final(w, a.c);
        if (tid == 0) {
            if (a.logprob) a.logprob[r] = has_tok ? lp_value(xt, f, a.c) : 0.0f;
            if (a.entropy) a.entropy[r] = f.entropy;
            if (a.rank) a.rank[r] = has_tok ? (int64_t)c2 : -1;
            if (a.stats) a.stats[r] = make_float4(f.m, f.R, f.log2S, f.entropy);
            if (a.status && tok >= a.V) atomicOr(a.status, B2S_STATUS_TOKEN_RANGE);
        }
        if constexpr (TOP) {
            // the cluster's lists (C x top words, each in order) into one; no alternatives where a wait gave up
            const int n_all = c2 < 0 ? 0 : C * a.top;
            if (c2 < 0 && tid < a.top) {
                a.top_ids[(int64_t)r * a.top + tid] = -1;
                a.top_logprobs[(int64_t)r * a.top + tid] = __int_as_float(0x7fffffff);
            }
            const unsigned long long* src = C > 1 ? sh.all : sh.top;
            for (int b = 0; b < n_all; b += NTH / 8) {
                const int i = b + (tid >> 3), rk = C > 1 ? rank_of(src, n_all, i) : i;
                const unsigned long long w64 = i < n_all ? src[i] : 0ull;
                if ((tid & 7) == 0 && w64 != 0ull && rk < a.top) {
                    const uint32_t key = (uint32_t)(w64 >> 32);
                    const float x = key == 0xffffffffu ? __int_as_float(0x7fffffff) : okey_to_f(key);
                    a.top_ids[(int64_t)r * a.top + rk] = word_id(w64);
                    a.top_logprobs[(int64_t)r * a.top + rk] = lp_value(x, f, a.c);
                }
            }
        }
    }
    if (sh.failed && tid == 0) {  // copies still in flight write this CTA's shared memory: wait for them
        if (a.status) atomicOr(a.status, B2S_STATUS_WAIT_TIMEOUT);
        for (int k = max(0, sh.loaded - a.stages); k < sh.loaded; ++k)
            gm_wait<false>(&sh.full[k % a.stages], (uint32_t)(k / a.stages) & 1u);
    }
}

// A warp per row, for many short rows without alternatives: no shared memory and no barriers, the next vectors in flight in
// registers while the current ones are added.  Bound by instruction issue on bf16 rows (120000 of 1000: issue active 77 %,
// IPC 3.1, ALU 61 %, DRAM 33 %; 30000 of 6562: IPC 3.0, DRAM 53 %), by HBM on the longest fp32 ones
// (microseconds, a CTA of 128 threads per row / this kernel: 30000 rows of 1000 bf16 89.5 / 21.2, 8192 of 6562 bf16 40.3 /
// 24.8, 4000 of 15000 fp32 46.9 / 40.4, 5.9 TB/s).  A lane adds up to a 64th of a row into each of its sums.
constexpr int LPW_NT = 256;
template <typename E>
__global__ void __launch_bounds__(LPW_NT, 4) token_logprobs_warp_kernel(const LpArgs a, int rows) {
    constexpr int EPV = LpElem<E>::EPV, ES = 16 / EPV;
    pdl_wait_then_release();
    const int r = (int)blockIdx.x * (LPW_NT / 32) + (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= rows) return;
    const unsigned char* rowp = static_cast<const unsigned char*>(a.logits) + (int64_t)r * a.stride * ES;
    const int n = a.V, nh = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(rowp) & 15)) & 15) / ES));
    const int nv = (n - nh) / EPV, nt = n - nh - nv * EPV;
    const uint4* vp = reinterpret_cast<const uint4*>(rowp + (int64_t)nh * ES);
    uint4 q[LP_U];
    auto load = [&](int v0) {
#pragma unroll
        for (int u = 0; u < LP_U; ++u) q[u] = v0 + 32 * u + lane < nv ? ldg_stream(vp + v0 + 32 * u + lane) : LpElem<E>::nothing();
    };
    load(0);
    const int64_t tok = a.tokens ? a.tokens[r] : -1;
    const bool has_tok = tok >= 0 && tok < a.V;
    const int t = has_tok ? (int)tok : -1;
    const float xt = has_tok ? LpElem<E>::ld(rowp, t) : 0.0f;
    const typename LpElem<E>::Thr thr_after = LpElem<E>::threshold(xt), thr_before = LpElem<E>::threshold_before(xt);
    const int tv = t >= nh ? min(nv, (t - nh) / EPV) : 0;  // vectors below it lie before the token
    LpThread s;
    s.m = f_ninf();
    s.S = s.U = make_float2(0.0f, 0.0f);
    int cnt = 0;
    const int end = lane < nh ? lane : (lane >= 16 && lane < 16 + nt ? n - nt + lane - 16 : -1);  // the ragged ends
    if (end >= 0) {
        const float x = LpElem<E>::ld(rowp, end);
        lp_thread_add(s, x, a.c);
        cnt += end != t && (x > xt || x != x || (end < t && x == xt));
    }
    for (int v0 = 0; v0 < nv; v0 += 32 * LP_U) {
        uint4 now[LP_U];
#pragma unroll
        for (int u = 0; u < LP_U; ++u) now[u] = q[u];
        load(v0 + 32 * LP_U);
        lp_thread_batch<E>(s, now, LpElem<E>::batch_max(now), a.c);
#pragma unroll
        for (int u = 0; u < LP_U; ++u)  // the vector that holds the token counts as behind it here
            cnt += LpElem<E>::count_above(now[u], v0 + 32 * u + lane < tv ? thr_before : thr_after);
    }
    // the elements of the token's own vector before it that tie with it
    const int i = nh + tv * EPV + lane;
    if (t >= nh && t < nh + nv * EPV && i < t) cnt += LpElem<E>::ld(rowp, i) == xt;
    if (has_tok && xt != xt) {  // a NaN token: the NaN elements before it
        cnt = 0;
        for (int j = lane; j < t; j += 32) {
            const float x = LpElem<E>::ld(rowp, j);
            cnt += x != x;
        }
    }
    const uint32_t key = __reduce_max_sync(0xffffffffu, rank_key(s.m));
    LpState w;
    w.m = key == 0xffffffffu ? __int_as_float(0x7fffffff) : okey_to_f(key);
    w.S = w.U = 0.0f;
    if (fabsf(w.m) <= 3.402823466e38f && s.m != f_ninf()) {
        lp_thread_rescale(s, w.m, a.c);
        w.S = s.S.x + s.S.y;
        w.U = s.U.x + s.U.y;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        w.S += __shfl_xor_sync(0xffffffffu, w.S, o);
        w.U += __shfl_xor_sync(0xffffffffu, w.U, o);
    }
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    const LpFinal f = lp_final(w, a.c);
    if (lane == 0) {
        if (a.logprob) a.logprob[r] = has_tok ? lp_value(xt, f, a.c) : 0.0f;
        if (a.entropy) a.entropy[r] = f.entropy;
        if (a.rank) a.rank[r] = has_tok ? (int64_t)cnt : -1;
        if (a.stats) a.stats[r] = make_float4(f.m, f.R, f.log2S, f.entropy);
        if (a.status && tok >= a.V) atomicOr(a.status, B2S_STATUS_TOKEN_RANGE);
    }
}

// dx for one chunk of a row per G threads: a CTA (bound by HBM: 2048 x 151936 bf16 188 us, the copy's rate), or, for many
// short rows, a whole row per warp.
constexpr int LPG_NT = 256;
constexpr int LPG_U = 8;  // vectors in flight per thread
template <typename E, int G>
__global__ void __launch_bounds__(LPG_NT) token_logprobs_grad_kernel(const void* logits, int64_t stride, int rows, int V,
                                                                     int chunk_vecs, int chunks, const int64_t* tokens,
                                                                     float c, float inv_t, const float4* stats,
                                                                     const float* g_lp, const float* g_h, void* out,
                                                                     int64_t ostride) {
    constexpr int EPV = LpElem<E>::EPV;
    constexpr int ES = 16 / EPV;
    pdl_wait_then_release();
    int r = (int)(blockIdx.x / chunks), ch = (int)(blockIdx.x % chunks), tid = threadIdx.x;
    if constexpr (G == 32) {  // a row per warp, in one chunk
        r = (int)blockIdx.x * (LPG_NT / 32) + (int)(threadIdx.x >> 5), ch = 0, tid = threadIdx.x & 31;
        if (r >= rows) return;
    }
    const unsigned char* rowp = static_cast<const unsigned char*>(logits) + (int64_t)r * stride * ES;
    unsigned char* outp = static_cast<unsigned char*>(out) + (int64_t)r * ostride * ES;
    const float4 st = stats[r];
    const int64_t tok = tokens ? tokens[r] : -1;
    const LpGrad g(st, tok >= 0 && tok < V ? (int)tok : -1, g_lp ? g_lp[r] : 0.0f, g_h ? g_h[r] : 0.0f, inv_t);
    // vectors of the output row; the input is read as vectors where it has the same alignment
    const int nh = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(outp) & 15)) & 15) / ES));
    const int nv = (V - nh) / EPV;
    const bool same = ((reinterpret_cast<uintptr_t>(rowp) - reinterpret_cast<uintptr_t>(outp)) & 15) == 0;
    if (ch == 0) {
        if (tid < nh) LpElem<E>::st(outp, tid, g.at(LpElem<E>::ld(rowp, tid), tid, c));
        const int i = nh + nv * EPV + tid;
        if (i < V) LpElem<E>::st(outp, i, g.at(LpElem<E>::ld(rowp, i), i, c));
    }
    const int v1 = min(nv, (ch + 1) * chunk_vecs), tv = g.t >= nh ? (g.t - nh) / EPV : -1;
    const uint4* vp = reinterpret_cast<const uint4*>(rowp + (int64_t)nh * ES);
    for (int v0 = ch * chunk_vecs + tid; v0 < v1; v0 += LPG_U * G) {
        uint4 q[LPG_U];
#pragma unroll
        for (int u = 0; u < LPG_U; ++u) {
            const int v = v0 + u * G;
            if (v < v1) {
                if (same) {
                    q[u] = ldg_stream(vp + v);
                } else {
                    float x[EPV];
#pragma unroll
                    for (int j = 0; j < EPV; ++j) x[j] = LpElem<E>::ld(rowp, nh + v * EPV + j);
                    q[u] = LpElem<E>::pack(x);  // the values themselves: nothing is rounded
                }
            }
        }
#pragma unroll
        for (int u = 0; u < LPG_U; ++u) {
            const int v = v0 + u * G;
            if (v < v1) {
                float x[EPV];
                LpElem<E>::unpack(q[u], x);
#pragma unroll
                for (int j = 0; j < EPV; ++j) x[j] = g.rest(x[j], c);
                if (v == tv) {
#pragma unroll
                    for (int j = 0; j < EPV; ++j) x[j] += nh + v * EPV + j == g.t ? g.bump : 0.0f;
                }
                __stcs(reinterpret_cast<uint4*>(outp + (int64_t)nh * ES) + v, LpElem<E>::pack(x));
            }
        }
    }
}

template <typename K, typename... Args>
cudaError_t launch(K kernel, int64_t blocks, int threads, uint32_t smem, int cluster, void* stream, Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The forward kernel on `rows` rows, C CTAs of NTH threads each.  A ring of three chunks keeps the copies going (96 KB of
// 512 threads, 48 of 256, 24 of 128: all 1024 threads that the registers allow fit an SM); with alternatives the whole
// part where it fits those, 48 KB of 128 threads (four CTAs an SM), or 192 of 512 where an SM has one CTA anyway.
template <typename E, int NTH, bool TOP>
cudaError_t launch_rows(LpArgs a, int rows, int C, int es, int sms, void* stream) {
    constexpr uint32_t CHUNK = LP_U * NTH * 16;
    a.per = ((a.V + C - 1) / C + 15) / 16 * 16;
    const int chunks = (int)(((int64_t)a.per * es + CHUNK - 1) / CHUNK);
    a.stages = chunks < 3 ? (chunks < 1 ? 1 : chunks) : 3;
    if (TOP && chunks <= (NTH == 128 || (int64_t)rows * C <= sms ? 6 : 3)) a.stages = chunks < 1 ? 1 : chunks;
    const auto kernel = token_logprobs_kernel<E, NTH, TOP>;
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(6 * CHUNK));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    return launch(kernel, (int64_t)rows * C, NTH, a.stages * CHUNK, C, stream, a);
}

}  // namespace
}  // namespace b2s

extern "C" {

int b2s_wait_limit(int64_t clocks, int64_t* previous) {
    using namespace b2s;
    const long long before =
        clocks < 0 ? wait_limit() : g_wait_limit.exchange(clocks < GM_WAIT ? clocks : GM_WAIT, std::memory_order_relaxed);
    if (previous) *previous = before;
    return B2S_OK;
}

int b2s_token_logprobs(const void* logits, int32_t logits_dtype, int32_t rows, int32_t vocab, int64_t row_stride,
                       const int64_t* tokens, float temperature, int32_t top, float* logprob, float* entropy,
                       int64_t* rank, int64_t* top_ids, float* top_logprobs, float* stats, uint32_t* status,
                       void* stream) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || top < 0 || row_stride < vocab) return B2S_ERR_INVALID;
    if (logits_dtype != B2S_DTYPE_F32 && logits_dtype != B2S_DTYPE_BF16) return B2S_ERR_INVALID;
    if (!lp_temperature_ok(temperature)) return B2S_ERR_INVALID;
    if (top > vocab) return B2S_ERR_INVALID;
    if (top > LP_MAX_TOP || vocab > LP_MAX_SIZE || rows > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
    if (rows == 0) return B2S_OK;
    if (!logits || (top && (!top_ids || !top_logprobs)) || (stats && (reinterpret_cast<uintptr_t>(stats) & 15)))
        return B2S_ERR_INVALID;
    const int es = logits_dtype == B2S_DTYPE_BF16 ? 2 : 4;
    if ((reinterpret_cast<uintptr_t>(logits) & (es - 1)) != 0) return B2S_ERR_INVALID;
    int sms = 0;
    const cudaError_t de = device_sms(&sms);
    if (de != cudaSuccess) return cuda_fail(de);
    LpArgs a;
    a.logits = logits;
    a.stride = row_stride;
    a.V = vocab;
    a.top = top;
    a.c = lp_scale(temperature);
    a.wait = wait_limit();
    a.tokens = tokens;
    a.logprob = logprob;
    a.entropy = entropy;
    a.rank = rank;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.stats = reinterpret_cast<float4*>(stats);
    a.status = status;
    const bool bf = logits_dtype == B2S_DTYPE_BF16;
    const int64_t row_bytes = (int64_t)vocab * es;
    cudaError_t e;
    // Many rows: a CTA each, of 128 threads up to 64 KB (1065 rows of 31 KB: 512 threads 13.3 us, 128 11.9) and of 256 beyond
    // (2048 rows of 297 KB: 512 threads 142 us, 128 132, 256 129).  With alternatives 256 from 24 KB on, which leaves an SM
    // its 1024 threads beside whole rows in shared memory.  Few rows: clusters of 512 threads.
    //
    // Without alternatives a warp per row once that fills the SMs' warps, or where a row is a few vectors per lane (a CTA / a
    // warp: 300 rows of 700 bf16 3.4 / 2.9 us, 300 of 6562 4.4 / 6.5, 1200 of 6562 8.7 / 9.1, 2000 of 18664 20.5 / 20.3,
    // 2000 of 30000 32.3 / 30.1, 4000 of 64000 107.4 / 106.6).
    if (!top && ((rows >= 2 * sms && row_bytes <= 4 * 1024) || (rows >= 12 * sms && row_bytes <= 64 * 1024))) {
        const int64_t blocks = ((int64_t)rows + LPW_NT / 32 - 1) / (LPW_NT / 32);
        e = bf ? launch(token_logprobs_warp_kernel<__nv_bfloat16>, blocks, LPW_NT, 0u, 0, stream, a, (int)rows)
               : launch(token_logprobs_warp_kernel<float>, blocks, LPW_NT, 0u, 0, stream, a, (int)rows);
    } else if (rows >= 2 * sms && row_bytes <= (top ? 24 : 64) * 1024) {
        e = top ? (bf ? launch_rows<__nv_bfloat16, 128, true>(a, rows, 1, es, sms, stream)
                      : launch_rows<float, 128, true>(a, rows, 1, es, sms, stream))
                : (bf ? launch_rows<__nv_bfloat16, 128, false>(a, rows, 1, es, sms, stream)
                      : launch_rows<float, 128, false>(a, rows, 1, es, sms, stream));
    } else if (rows >= 2 * sms) {
        e = top ? (bf ? launch_rows<__nv_bfloat16, 256, true>(a, rows, 1, es, sms, stream)
                      : launch_rows<float, 256, true>(a, rows, 1, es, sms, stream))
                : (bf ? launch_rows<__nv_bfloat16, 256, false>(a, rows, 1, es, sms, stream)
                      : launch_rows<float, 256, false>(a, rows, 1, es, sms, stream));
    } else {
        int C = 1;
        while (C < 8 && (int64_t)rows * C * 2 <= 2 * sms && row_bytes / (C * 2) >= 16 * 1024) C <<= 1;
        e = top ? (bf ? launch_rows<__nv_bfloat16, 512, true>(a, rows, C, es, sms, stream)
                      : launch_rows<float, 512, true>(a, rows, C, es, sms, stream))
                : (bf ? launch_rows<__nv_bfloat16, 512, false>(a, rows, C, es, sms, stream)
                      : launch_rows<float, 512, false>(a, rows, C, es, sms, stream));
    }
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

int b2s_token_logprobs_grad(const void* logits, int32_t logits_dtype, int32_t rows, int32_t vocab, int64_t row_stride,
                            const int64_t* tokens, float temperature, const float* stats, const float* grad_logprob,
                            const float* grad_entropy, void* grad_logits, int64_t grad_row_stride, void* stream) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || row_stride < vocab || grad_row_stride < vocab) return B2S_ERR_INVALID;
    if (logits_dtype != B2S_DTYPE_F32 && logits_dtype != B2S_DTYPE_BF16) return B2S_ERR_INVALID;
    if (!lp_temperature_ok(temperature)) return B2S_ERR_INVALID;
    if (vocab > LP_MAX_SIZE || rows > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
    if (rows == 0) return B2S_OK;
    const int es = logits_dtype == B2S_DTYPE_BF16 ? 2 : 4;
    if (!logits || !stats || !grad_logits || (reinterpret_cast<uintptr_t>(stats) & 15) ||
        (reinterpret_cast<uintptr_t>(logits) & (es - 1)) || (reinterpret_cast<uintptr_t>(grad_logits) & (es - 1)))
        return B2S_ERR_INVALID;
    const int epv = 16 / es;
    int sms = 0;
    const cudaError_t de = device_sms(&sms);
    if (de != cudaSuccess) return cuda_fail(de);
    const int64_t row_bytes = (int64_t)vocab * es;
    // A CTA / a warp per row (us): 300 x 2040 bf16 3.6 / 3.9, 600 x 2040 4.3 / 4.0, 2000 x 4000 10.7 / 10.2, 2000 x 6562 13.0 /
    // 15.3, 4000 x 6562 25.6 / 24.9, 8192 x 8000 53.1 / 49.8, 30000 x 1000 80.7 / 28.4, 8192 x 6562 fp32 65.2 / 72.7.
    const bool warp = row_bytes <= 8 * 1024 ? rows >= 4 * sms : row_bytes <= 16 * 1024 && rows >= 24 * sms;
    const int chunk_vecs = warp ? vocab / epv + 1 : LPG_NT * LPG_U;
    const int64_t chunks = warp ? 1 : ((int64_t)vocab / epv + chunk_vecs - 1) / chunk_vecs;
    const int64_t nch = chunks < 1 ? 1 : chunks;
    if (nch * rows > INT32_MAX) return B2S_ERR_UNSUPPORTED;
    const float c = lp_scale(temperature), inv = (float)(1.0 / (double)temperature);
    const float4* st = reinterpret_cast<const float4*>(stats);
    const int64_t per = warp ? LPG_NT / 32 : 1, blocks = (nch * rows + per - 1) / per;
    auto go = [&](auto kernel) {
        return launch(kernel, blocks, LPG_NT, 0u, 0, stream, logits, row_stride, (int)rows, (int)vocab, chunk_vecs, (int)nch,
                      tokens, c, inv, st, grad_logprob, grad_entropy, grad_logits, grad_row_stride);
    };
    cudaError_t e;
    if (logits_dtype == B2S_DTYPE_BF16)
        e = warp ? go(token_logprobs_grad_kernel<__nv_bfloat16, 32>) : go(token_logprobs_grad_kernel<__nv_bfloat16, LPG_NT>);
    else
        e = warp ? go(token_logprobs_grad_kernel<float, 32>) : go(token_logprobs_grad_kernel<float, LPG_NT>);
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

}  // extern "C"
