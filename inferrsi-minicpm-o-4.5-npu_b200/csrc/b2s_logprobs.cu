// Log probabilities of given tokens with entropy, rank and top alternatives from logits rows, and their gradient
// (sm_100a).  No counterpart in the reference, whose call sites stop at the token.
//
// With z = x / T and c = log2(e) / T, everything is kept in base 2 around a reference R = fl(m c) of the running
// maximum m: y_i = fma(x_i, c, -R) (one rounding of the exact x_i c - R, and R drops out of every difference, so R
// need not be exact), S = sum 2^y, U = sum 2^y y.  Then logprob = (y_t - log2 S) ln 2 and the entropy
// H = (log2 S - U / S) ln 2: U <= 0, so H is a sum of two non-negative terms and nothing cancels.  S and U are fp32
// per thread (a few hundred terms each) and merged pairwise; a merge of two references shifts y by R_a - R_b.
// Rows whose reference overflows (|m| c beyond fp32: a mask of the type's lowest value throughout) use
// y = (x - m) c instead.  A masked (-inf) element adds nothing; a row with nothing left has logprob -inf, entropy 0
// and gradient 0; NaN or +inf anywhere makes the row NaN, as a softmax gives it.
//
// Forward, one pass over the row: a cluster of CTAs per row (several while rows are few), each thread streaming
// 16-byte vectors.  The rank counts the elements before the token in (value descending, id ascending) order:
// an element before the token counts when x >= x_t, i.e. x > pred(x_t), one after it when x > x_t, so a vector needs
// one threshold.  Top alternatives: pass 1 leaves each thread's maximum; the top-th largest of the warps' largest
// maxima bounds the CTA's top-th value from below; only the shares of threads that reach it are read again (from L2),
// their elements above the bound listed and ordered by rank counting.  Lists that overflow (more ties than the list
// holds) take an exact radix select over the CTA's part of the row.
//
// Backward, elementwise: dx = (g_lp ([i = t] - p) - g_H p (log p + H)) / T with p = 2^(y - log2 S) recomputed from
// the saved reference: one read and one write of the row.
#include <cooperative_groups.h>
#include <string.h>

#include "../../include/b2s_sampler.h"
#include "b2s_device.cuh"
#include "b2s_logprobs.cuh"

namespace cg = cooperative_groups;

namespace b2s {

int cuda_fail(cudaError_t e);

cudaError_t device_sms(int* sms) {
    static int cached[64] = {};  // 0: not asked yet; a device's count never changes, so racing writers agree
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64 && cached[dev] > 0) {
        *sms = cached[dev];
        return cudaSuccess;
    }
    e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess && dev >= 0 && dev < 64) cached[dev] = *sms;
    return e;
}

namespace {

constexpr int LP_CAP = 512;      // candidate list entries per CTA
constexpr int LP_GATHER = 4;     // thread maxima gathered per warp (16 warps x 4 = 64 >= the largest top)
constexpr int LP_MAX_TOP = 32;
constexpr int LP_U = 4;          // vectors per thread and batch

template <typename E>
struct LpElem;
template <>
struct LpElem<float> {
    static constexpr int EPV = 4;
    static __device__ __forceinline__ float ld(const void* p, int64_t i) { return __ldg(static_cast<const float*>(p) + i); }
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
    static __device__ __forceinline__ float ld(const void* p, int64_t i) {
        return bf16_bits_to_f(__ldg(static_cast<const unsigned short*>(p) + i));
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

// The largest float below x (x not NaN); NaN for -inf, whose "x > pred" must hold for every element.
__device__ __forceinline__ float pred_float(float x) {
    if (x == f_ninf()) return __int_as_float(0x7fffffff);
    if (x == 0.0f) return __int_as_float((int)0x80000001u);
    const int b = __float_as_int(x);
    return __int_as_float(x > 0.0f ? b - 1 : b + 1);
}

struct LpShared {
    LpState warp[NWARP];
    int count[NWARP];
    int has_nan[NWARP];
    uint32_t gather[NWARP * LP_GATHER];
    int n_list;
    int red[NWARP + 1];
    uint32_t hist[256];
    uint32_t ctl[2];
    unsigned long long list[LP_CAP];
    unsigned long long top[LP_MAX_TOP];  // this CTA's best, in order (0: none)
    LpState total;                       // this CTA's state and count, read by the cluster's first CTA
    int total_count;
};

struct LpArgs {
    const void* logits;
    int64_t stride;
    int V, per, top;
    float c;
    const int64_t* tokens;
    float *logprob, *entropy;
    int64_t *rank, *top_ids;
    float* top_logprobs;
    float4* stats;
    uint32_t* status;
};

// The top `need` words of elements [0, n) of this CTA's part of the row (element i has id lo + i), exactly, whatever
// the ties: the need-th largest value by radix select, then everything above it and the first ties in id order.
// Every thread calls it; sh.list holds min(need, n) words afterwards.
template <typename E>
__device__ __noinline__ void exact_top(LpShared& sh, const void* rowp, int lo, int n, int need) {
    const int tid = threadIdx.x;
    need = min(need, n);
    auto key = [&](int i) { return rank_key(LpElem<E>::ld(rowp, lo + i)); };
    __syncthreads();
    const uint32_t kth = block_kth_largest(n, need, key, sh.hist, sh.ctl);
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
        const float x = LpElem<E>::ld(rowp, lo + i);
        if (rank_key(x) > kth) sh.list[atomicAdd(&sh.n_list, 1)] = rank_word(x, lo + i);  // fewer than need <= LP_CAP
    }
    __syncthreads();
    int have = sh.n_list;
    for (int b = 0; b < n && have < need; b += NT) {
        const int i = b + tid;
        const float x = i < n ? LpElem<E>::ld(rowp, lo + i) : 0.0f;
        const int tie = i < n && rank_key(x) == kth;
        int total;
        const int before = block_excl_scan_i(tie, sh.red, &total);
        if (tie && have + before < need) sh.list[have + before] = rank_word(x, lo + i);
        have += total;
        __syncthreads();
    }
    if (tid == 0) sh.n_list = need;
    __syncthreads();
}

// Orders n words (distinct) of `list` into out[0 .. top): out[k] the k-th largest, 0 where there are fewer.
__device__ __forceinline__ void order_words(const unsigned long long* list, int n, unsigned long long* out, int top) {
    for (int k = threadIdx.x; k < top; k += NT)
        if (k >= n) out[k] = 0ull;
    for (int i = threadIdx.x; i < n; i += NT) {
        const unsigned long long w = list[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += list[j] > w;
        if (r < top) out[r] = w;
    }
}

template <typename E, bool TOP>
__global__ void __launch_bounds__(NT, 2) token_logprobs_kernel(const LpArgs a) {
    constexpr int EPV = LpElem<E>::EPV;
    constexpr int ES = 16 / EPV;
    __shared__ LpShared sh;
    pdl_wait_then_release();
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
    const int r = (int)(blockIdx.x / C);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned char* rowp = static_cast<const unsigned char*>(a.logits) + (int64_t)r * a.stride * ES;
    const int lo = min(a.V, crank * a.per), hi = min(a.V, lo + a.per), n = hi - lo;

    const int64_t tok = a.tokens ? a.tokens[r] : -1;
    const bool has_tok = tok >= 0 && tok < a.V;
    const int t = has_tok ? (int)tok : -1;
    const float xt = has_tok ? LpElem<E>::ld(rowp, t) : 0.0f;
    const float thr_after = xt, thr_before = pred_float(xt);

    // the 16-byte interior [v0, v0 + nv vectors) of the part, a ragged head and tail
    const uintptr_t A = reinterpret_cast<uintptr_t>(rowp) + (uintptr_t)lo * ES;
    int nh = (int)(((16 - (A & 15)) & 15) / ES);
    nh = min(nh, n);
    const int nv = (n - nh) / EPV;
    const int i0 = lo + nh;             // id of the interior's first element
    const int nt = n - nh - nv * EPV;   // tail elements
    const uint4* vp = reinterpret_cast<const uint4*>(rowp + (int64_t)i0 * ES);

    LpState s;
    s.m = f_ninf();
    s.S = 0.0f;
    s.U = 0.0f;
    int cnt = 0;
    auto one = [&](float x, int id) {
        lp_add(s, x, a.c);
        cnt += !(x <= (id < t ? thr_before : thr_after)) && id != t;
    };
    if (tid < nh) one(LpElem<E>::ld(rowp, lo + tid), lo + tid);
    if (tid >= 32 && tid < 32 + nt) one(LpElem<E>::ld(rowp, hi - nt + tid - 32), hi - nt + tid - 32);

    for (int b = tid; b < nv; b += LP_U * NT) {
        uint4 q[LP_U];
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
            if (b + u * NT < nv) q[u] = ldg_stream(vp + b + u * NT);
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            const int v = b + u * NT;
            if (v < nv) {
                float x[EPV];
                LpElem<E>::unpack(q[u], x);
                lp_add_many<EPV>(s, x, a.c);
                const int id = i0 + v * EPV;
                if (t < id || t >= id + EPV) {
                    const float thr = id < t ? thr_before : thr_after;
#pragma unroll
                    for (int j = 0; j < EPV; ++j) cnt += !(x[j] <= thr);
                } else {
#pragma unroll
                    for (int j = 0; j < EPV; ++j) cnt += !(x[j] <= (id + j < t ? thr_before : thr_after)) && id + j != t;
                }
            }
        }
    }
    // a NaN token: NaN compares false with everything, so every element was counted; the elements before it are the
    // NaN ones with a smaller id
    if (has_tok && xt != xt) {
        cnt = 0;
        for (int i = lo + tid; i < min(hi, t); i += NT) {
            const float x = LpElem<E>::ld(rowp, i);
            cnt += x != x;
        }
    }

    const float tmax = s.m;  // this thread's maximum (NaN if it saw one)
    if (TOP) {
        // the warp's LP_GATHER largest thread maxima (0: no such thread)
        uint32_t k = tmax == f_ninf() ? 0u : rank_key(tmax);
#pragma unroll
        for (int g = 0; g < LP_GATHER; ++g) {
            const uint32_t mx = __reduce_max_sync(0xffffffffu, k);
            if (lane == 0) sh.gather[warp * LP_GATHER + g] = mx;
            const uint32_t who = __ballot_sync(0xffffffffu, k == mx);
            if (lane == __ffs(who) - 1) k = 0u;
        }
        if (tid == 0) sh.n_list = 0;
    }
    // merge the warp's, then the CTA's states and counts
    lp_warp_merge(s, a.c);
    cnt = warp_sum_i(cnt);
    if (lane == 0) {
        sh.warp[warp] = s;
        sh.count[warp] = cnt;
    }
    __syncthreads();
    if (warp == 0) {
        LpState w;
        w.m = f_ninf();
        w.S = w.U = 0.0f;
        int c2 = 0;
        if (lane < NWARP) {
            w = sh.warp[lane];
            c2 = sh.count[lane];
        }
        lp_warp_merge(w, a.c);
        c2 = warp_sum_i(c2);
        if (lane == 0) {
            sh.total = w;
            sh.total_count = c2;
        }
    }
    if (TOP) {
        // tau: the top-th largest gathered maximum, each a distinct element, so at least `top` elements reach it
        const uint32_t g0 = sh.gather[lane], g1 = sh.gather[32 + lane];
        int r0 = 0, r1 = 0;
#pragma unroll 8
        for (int j = 0; j < NWARP * LP_GATHER; ++j) {
            const uint32_t o = sh.gather[j];
            r0 += o > g0 || (o == g0 && j < lane);
            r1 += o > g1 || (o == g1 && j < 32 + lane);
        }
        const uint32_t tau = __reduce_max_sync(0xffffffffu, r0 == a.top - 1 ? g0 : r1 == a.top - 1 ? g1 : 0u);
        // pass 2: the shares whose maximum reaches tau, one warp per share
        uint32_t hits = __ballot_sync(0xffffffffu, (tmax == f_ninf() ? 0u : rank_key(tmax)) >= tau);
        auto offer = [&](float x, int id) {
            if (rank_key(x) >= tau) {
                const int p = atomicAdd(&sh.n_list, 1);
                if (p < LP_CAP) sh.list[p] = rank_word(x, id);
            }
        };
        while (hits) {
            if (*reinterpret_cast<volatile int*>(&sh.n_list) > LP_CAP) break;  // the exact path will take it
            const int h = (warp << 5) + __ffs(hits) - 1;
            hits &= hits - 1;
            for (int v = h + lane * NT; v < nv; v += 32 * NT) {
                float x[EPV];
                LpElem<E>::unpack(ldg_stream(vp + v), x);
#pragma unroll
                for (int j = 0; j < EPV; ++j) offer(x[j], i0 + v * EPV + j);
            }
            if (lane == 0 && h < nh) offer(LpElem<E>::ld(rowp, lo + h), lo + h);
            if (lane == 0 && h >= 32 && h < 32 + nt) offer(LpElem<E>::ld(rowp, hi - nt + h - 32), hi - nt + h - 32);
        }
        __syncthreads();
        if (sh.n_list > LP_CAP) exact_top<E>(sh, rowp, lo, n, a.top);
        order_words(sh.list, sh.n_list, sh.top, a.top);
    }
    if (C > 1) cluster.sync();
    else __syncthreads();

    if (crank == 0) {
        LpState w = sh.total;
        int c2 = sh.total_count;
        for (int k = 1; k < C; ++k) {
            const LpShared* o = cluster.map_shared_rank(&sh, k);
            w = lp_merge(w, o->total, a.c);
            c2 += o->total_count;
        }
        const LpFinal f = lp_final(w, a.c);
        if (tid == 0) {
            float lp = 0.0f;
            if (has_tok) lp = lp_value(xt, f, a.c);
            if (a.logprob) a.logprob[r] = lp;
            if (a.entropy) a.entropy[r] = f.entropy;
            if (a.rank) a.rank[r] = has_tok ? (int64_t)c2 : -1;
            if (a.stats) a.stats[r] = make_float4(f.m, f.R, f.log2S, f.entropy);
            if (a.status && tok >= a.V) atomicOr(a.status, B2S_STATUS_TOKEN_RANGE);
        }
        if (TOP) {
            // the cluster's lists (C x top words, each in order) into one
            int n_all = 0;
            if (C > 1) {
                __syncthreads();
                for (int i = tid; i < C * a.top; i += NT) {
                    const LpShared* o = cluster.map_shared_rank(&sh, i / a.top);
                    sh.list[i] = o->top[i % a.top];
                }
                n_all = C * a.top;
                __syncthreads();
            }
            const unsigned long long* src = C > 1 ? sh.list : sh.top;
            if (C == 1) n_all = a.top;
            for (int i = tid; i < n_all; i += NT) {
                const unsigned long long w64 = src[i];
                int rk = i;
                if (C > 1) {
                    rk = 0;
                    for (int j = 0; j < n_all; ++j) rk += src[j] > w64;
                }
                if (w64 != 0ull && rk < a.top) {
                    const int id = word_id(w64);
                    a.top_ids[(int64_t)r * a.top + rk] = id;
                    a.top_logprobs[(int64_t)r * a.top + rk] = lp_value(LpElem<E>::ld(rowp, id), f, a.c);
                }
            }
        }
    }
    if (C > 1) cluster.sync();  // the first CTA has read the others' shared memory
}

// dx for one chunk of a row per CTA.
constexpr int LPG_NT = 256;
template <typename E>
__global__ void __launch_bounds__(LPG_NT) token_logprobs_grad_kernel(const void* logits, int64_t stride, int V,
                                                                     int chunk_vecs, int chunks, const int64_t* tokens,
                                                                     float c, float inv_t, const float4* stats,
                                                                     const float* g_lp, const float* g_h, void* out,
                                                                     int64_t ostride) {
    constexpr int EPV = LpElem<E>::EPV;
    constexpr int ES = 16 / EPV;
    pdl_wait_then_release();
    const int r = (int)(blockIdx.x / chunks), ch = (int)(blockIdx.x % chunks);
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
        if ((int)threadIdx.x < nh) LpElem<E>::st(outp, threadIdx.x, g.at(LpElem<E>::ld(rowp, threadIdx.x), threadIdx.x, c));
        const int i = nh + nv * EPV + (int)threadIdx.x;
        if (i < V) LpElem<E>::st(outp, i, g.at(LpElem<E>::ld(rowp, i), i, c));
    }
    const int v1 = min(nv, (ch + 1) * chunk_vecs);
    for (int v = ch * chunk_vecs + (int)threadIdx.x; v < v1; v += LPG_NT) {
        const int id = nh + v * EPV;
        float x[EPV];
        if (same) {
            LpElem<E>::unpack(ldg_stream(reinterpret_cast<const uint4*>(rowp + (int64_t)id * ES)), x);
        } else {
#pragma unroll
            for (int j = 0; j < EPV; ++j) x[j] = LpElem<E>::ld(rowp, id + j);
        }
#pragma unroll
        for (int j = 0; j < EPV; ++j) x[j] = g.at(x[j], id + j, c);
        *reinterpret_cast<uint4*>(outp + (int64_t)id * ES) = LpElem<E>::pack(x);
    }
}

template <typename K, typename... Args>
cudaError_t launch(K kernel, int64_t blocks, int threads, int cluster, void* stream, Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
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

}  // namespace
}  // namespace b2s

extern "C" {

int b2s_token_logprobs(const void* logits, int32_t logits_dtype, int32_t rows, int32_t vocab, int64_t row_stride,
                       const int64_t* tokens, float temperature, int32_t top, float* logprob, float* entropy,
                       int64_t* rank, int64_t* top_ids, float* top_logprobs, float* stats, uint32_t* status,
                       void* stream) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || top < 0 || row_stride < vocab) return B2S_ERR_INVALID;
    if (logits_dtype != B2S_DTYPE_F32 && logits_dtype != B2S_DTYPE_BF16) return B2S_ERR_INVALID;
    if (!lp_temperature_ok(temperature)) return B2S_ERR_INVALID;
    if (top > vocab) return B2S_ERR_INVALID;
    if (top > LP_MAX_TOP) return B2S_ERR_UNSUPPORTED;
    if (rows == 0) return B2S_OK;
    if (!logits || (top && (!top_ids || !top_logprobs)) || (stats && (reinterpret_cast<uintptr_t>(stats) & 15)))
        return B2S_ERR_INVALID;
    const int es = logits_dtype == B2S_DTYPE_BF16 ? 2 : 4;
    if ((reinterpret_cast<uintptr_t>(logits) & (es - 1)) != 0) return B2S_ERR_INVALID;
    int sms = 0;
    const cudaError_t de = device_sms(&sms);
    if (de != cudaSuccess) return cuda_fail(de);
    int C = 1;
    while (C < 8 && (int64_t)rows * C * 2 <= 2 * sms && (int64_t)vocab * es / (C * 2) >= 16 * 1024) C <<= 1;
    const int per = ((vocab + C - 1) / C + 15) / 16 * 16;
    LpArgs a;
    a.logits = logits;
    a.stride = row_stride;
    a.V = vocab;
    a.per = per;
    a.top = top;
    a.c = lp_scale(temperature);
    a.tokens = tokens;
    a.logprob = logprob;
    a.entropy = entropy;
    a.rank = rank;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.stats = reinterpret_cast<float4*>(stats);
    a.status = status;
    const bool bf = logits_dtype == B2S_DTYPE_BF16;
    const cudaError_t e =
        top ? (bf ? launch(token_logprobs_kernel<__nv_bfloat16, true>, (int64_t)rows * C, NT, C, stream, a)
                  : launch(token_logprobs_kernel<float, true>, (int64_t)rows * C, NT, C, stream, a))
            : (bf ? launch(token_logprobs_kernel<__nv_bfloat16, false>, (int64_t)rows * C, NT, C, stream, a)
                  : launch(token_logprobs_kernel<float, false>, (int64_t)rows * C, NT, C, stream, a));
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

int b2s_token_logprobs_grad(const void* logits, int32_t logits_dtype, int32_t rows, int32_t vocab, int64_t row_stride,
                            const int64_t* tokens, float temperature, const float* stats, const float* grad_logprob,
                            const float* grad_entropy, void* grad_logits, int64_t grad_row_stride, void* stream) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || row_stride < vocab || grad_row_stride < vocab) return B2S_ERR_INVALID;
    if (logits_dtype != B2S_DTYPE_F32 && logits_dtype != B2S_DTYPE_BF16) return B2S_ERR_INVALID;
    if (!lp_temperature_ok(temperature)) return B2S_ERR_INVALID;
    if (rows == 0) return B2S_OK;
    const int es = logits_dtype == B2S_DTYPE_BF16 ? 2 : 4;
    if (!logits || !stats || !grad_logits || (reinterpret_cast<uintptr_t>(stats) & 15) ||
        (reinterpret_cast<uintptr_t>(logits) & (es - 1)) || (reinterpret_cast<uintptr_t>(grad_logits) & (es - 1)))
        return B2S_ERR_INVALID;
    const int epv = 16 / es;
    const int chunk_vecs = LPG_NT * 8;
    const int64_t chunks = ((int64_t)vocab / epv + chunk_vecs - 1) / chunk_vecs;
    const int64_t nch = chunks < 1 ? 1 : chunks;
    if (nch * rows > INT32_MAX) return B2S_ERR_UNSUPPORTED;
    const float c = lp_scale(temperature), inv = (float)(1.0 / (double)temperature);
    const float4* st = reinterpret_cast<const float4*>(stats);
    const cudaError_t e =
        logits_dtype == B2S_DTYPE_BF16
            ? launch(token_logprobs_grad_kernel<__nv_bfloat16>, nch * rows, LPG_NT, 0, stream, logits, row_stride,
                     (int)vocab, chunk_vecs, (int)nch, tokens, c, inv, st, grad_logprob, grad_entropy, grad_logits,
                     grad_row_stride)
            : launch(token_logprobs_grad_kernel<float>, nch * rows, LPG_NT, 0, stream, logits, row_stride, (int)vocab,
                     chunk_vecs, (int)nch, tokens, c, inv, st, grad_logprob, grad_entropy, grad_logits, grad_row_stride);
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

}  // extern "C"
