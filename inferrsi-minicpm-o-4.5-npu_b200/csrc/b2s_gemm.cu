// The product kernel and what is built on it: the head's log probabilities (logits never written), their gradient,
// the projection with bias, activation and residual in its epilogue, and its gradient.  No counterpart in the
// reference, whose call sites use F.linear.
#include <string.h>

#include <mutex>

#include "b2s_gemm.cuh"

namespace b2s {

int cuda_fail(cudaError_t e);
int tensor_map_2d(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int64_t outer_stride, int box_inner,
                  int box_outer);

namespace {

__device__ __forceinline__ void tile_of(const GemmArgs& a, int64_t t, int* mt, int* nt) {
    const int64_t per = (int64_t)GM_GROUP * a.tiles_n;
    const int g = (int)(t / per), in = (int)(t % per);
    const int gm = min(GM_GROUP, a.tiles_m - g * GM_GROUP);
    *mt = g * GM_GROUP + in % gm;
    *nt = in / gm;
}

// The epilogue of one thread's row of a tile: columns [n0, n0 + TN) from tensor memory at `tm`.
template <int TN, int EPI>
__device__ __forceinline__ void epilogue_row(const GemmArgs& a, uint32_t tm, int row, int n0, int nt) {
    const bool live = row < a.M;
    if constexpr (EPI == EPI_LINEAR || EPI == EPI_STORE) {
        unsigned char* out = static_cast<unsigned char*>(a.out) + (int64_t)row * a.out_stride * 2;
#pragma unroll 1
        for (int q = 0; q < TN / 32; ++q) {
            float v[32];
            tmem_ld32(tm + 32u * q, v);
            const int n = n0 + 32 * q;
            if (live && n < a.N) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int ng = n + 8 * g;
                    if (ng < a.N) {
                        float* w = v + 8 * g;
                        if constexpr (EPI == EPI_LINEAR) {
                            if (a.bias) {
                                float b[8];
                                load8(a.bias, ng, a.N, true, b);
#pragma unroll
                                for (int j = 0; j < 8; ++j) w[j] += b[j];
                            }
                            // the saved pre-activation is bf16, like the tensors around it: the slope taken from it
                            // is off by half a bf16 step of z times the activation's curvature, less than dz's own
                            // rounding to the tensor cores' bf16
                            if (a.preact)
                                store8(static_cast<unsigned char*>(a.preact) + (int64_t)row * a.pre_stride * 2, ng, a.N,
                                       true, w);
                            if (a.act != ACT_NONE) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) w[j] = act_apply(w[j], a.act);
                            }
                            if (a.residual) {
                                float r[8];
                                load8(static_cast<const unsigned char*>(a.residual) + (int64_t)row * a.res_stride * 2,
                                      ng, a.N, a.res_vec, r);
#pragma unroll
                                for (int j = 0; j < 8; ++j) w[j] += r[j];
                            }
                        }
                        store8(out, ng, a.N, a.out_vec, w);
                    }
                }
            }
        }
    } else if constexpr (EPI == EPI_LSE) {
        const int64_t tok = live ? a.tokens[row] : -1;
        LpState s;
        s.m = f_ninf();
        s.S = s.U = 0.0f;
#pragma unroll 1
        for (int q = 0; q < TN / 32; ++q) {
            float v[32];
            tmem_ld32(tm + 32u * q, v);
            const int n = n0 + 32 * q;
            if (n < a.N) {
                if (tok >= n && tok < min(n + 32, a.N)) {
                    float tv = v[0];
#pragma unroll
                    for (int j = 1; j < 32; ++j) tv = tok == n + j ? v[j] : tv;
                    a.token_value[row] = tv;
                }
                if (n + 32 > a.N) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = n + j < a.N ? v[j] : f_ninf();
                }
                lp_add_many<32>(s, v, a.c);
            }
        }
        if (live) a.part[(int64_t)row * a.tiles_n + nt] = make_float4(s.m, s.S, s.U, 0.0f);
    } else {
        const int64_t tok = live ? a.tokens[row] : -1;
        const float4 st = live ? a.stats[row] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const LpGrad g(st, tok >= 0 && tok < a.N ? (int)tok : -1, live && a.g_lp ? a.g_lp[row] : 0.0f,
                       live && a.g_h ? a.g_h[row] : 0.0f, a.inv_t);
        unsigned char* out = static_cast<unsigned char*>(a.out) + (int64_t)row * a.out_stride * 2;
#pragma unroll 1
        for (int q = 0; q < TN / 32; ++q) {
            float v[32];
            tmem_ld32(tm + 32u * q, v);
            const int n = n0 + 32 * q;
            if (live && n < a.N) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = g.at(v[j], n + j, a.c);
                // dz is rounded to bf16 once: it is the tensor cores' operand in both gradient products
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + 8 * j < a.N) store8(out, n + 8 * j, a.N, a.out_vec, v + 8 * j);
            }
        }
    }
}

template <int TN, bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(GM_THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                const __grid_constant__ GemmArgs a) {
    constexpr int ST = gm_stages(TN);
    constexpr uint32_t STAGE = gm_stage_bytes(TN);
    constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)AMN << 15) | ((uint32_t)BMN << 16) |
                               ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(GM_M >> 4) << 24);
    extern __shared__ __align__(128) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base_u = smem_u32(smem_raw);
    unsigned char* sm = smem_raw + (((base_u + 1023u) & ~1023u) - base_u);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + ST * STAGE);
    uint64_t* empty = full + ST;
    uint64_t* tfull = empty + ST;   // [2] an accumulator is complete
    uint64_t* tempty = tfull + 2;   // [2] an accumulator has been read
    uint64_t* drain = tempty + 2;   // every MMA issued has completed (only after a failure)
    uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tslot + 1);
    volatile int* issued = fail + 1;    // stage loads issued
    volatile int* consumed = fail + 2;  // stage loads seen to land

    if (tid == 0) {
        prefetch_tensormap(&amap);
        prefetch_tensormap(&bmap);
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&tfull[s], 1);
            mbar_init(&tempty[s], 128);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
        *fail = 0;
        *issued = 0;
        *consumed = 0;
    }
    if (warp == 5) tmem_alloc(tslot, 2 * TN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    pdl_wait_then_release();

    const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
    if (warp == 4) {
        if (lane == 0) {  // loads
            int it = 0;
            bool ok = true;
            for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                int mt, nt;
                tile_of(a, t, &mt, &nt);
                for (int kb = 0; kb < a.nkb; ++kb, ++it) {
                    const int s = it % ST;
                    if (it >= ST && !mbar_wait_bounded(&empty[s], (uint32_t)(it / ST - 1) & 1u, HEAD_WAIT_NS)) {
                        *fail = 1;
                        ok = false;
                        break;
                    }
                    if (*fail) {
                        ok = false;
                        break;
                    }
                    unsigned char* sa = sm + s * STAGE;
                    unsigned char* sb = sa + GM_A_BYTES;
                    mbar_arrive_expect_tx(&full[s], STAGE);  // parts outside the tensors are filled with zeros
                    if constexpr (AMN) {
#pragma unroll
                        for (int j = 0; j < GM_M / 64; ++j)
                            tma_load_2d(sa + 8192 * j, &amap, mt * GM_M + 64 * j, kb * GM_KB, &full[s]);
                    } else {
                        tma_load_2d(sa, &amap, kb * GM_KB, mt * GM_M, &full[s]);
                    }
                    if constexpr (BMN) {
#pragma unroll
                        for (int j = 0; j < TN / 64; ++j)
                            tma_load_2d(sb + 8192 * j, &bmap, nt * TN + 64 * j, kb * GM_KB, &full[s]);
                    } else {
                        tma_load_2d(sb, &bmap, kb * GM_KB, nt * TN, &full[s]);
                    }
                }
            }
            *issued = it;
        }
    } else if (warp == 5) {
        if (lane == 0) {  // MMAs
            int it = 0, i = 0;
            bool ok = true;
            for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++i) {
                const int acc = i & 1;
                if (i >= 2 && !mbar_wait_bounded(&tempty[acc], (uint32_t)(i / 2 - 1) & 1u, HEAD_WAIT_NS)) {
                    *fail = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(acc * TN);
                for (int kb = 0; kb < a.nkb; ++kb) {
                    const int s = it % ST;
                    if (*fail || !mbar_wait_bounded(&full[s], (uint32_t)(it / ST) & 1u, HEAD_WAIT_NS)) {
                        *fail = 1;
                        ok = false;
                        break;
                    }
                    ++it;
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(sm + s * STAGE), b0 = a0 + GM_A_BYTES;
#pragma unroll
                    for (int k = 0; k < GM_KB / 16; ++k)
                        umma_bf16(d, AMN ? umma_desc_mn128(a0 + 2048u * k) : umma_desc_sw128(a0 + 32u * k),
                                  BMN ? umma_desc_mn128(b0 + 2048u * k) : umma_desc_sw128(b0 + 32u * k), IDESC,
                                  (kb | k) != 0 ? 1u : 0u);
                    umma_commit(&empty[s]);
                }
                if (ok) umma_commit(&tfull[acc]);
            }
            *consumed = it;
            if (*fail) {
                umma_commit(drain);
                mbar_wait_bounded(drain, 0u, HEAD_WAIT_NS);
            }
        }
    } else {
        int i = 0;
        for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
            int mt, nt;
            tile_of(a, t, &mt, &nt);
            const int acc = i & 1;
            const bool ok = mbar_wait_bounded(&tfull[acc], (uint32_t)(i / 2) & 1u, HEAD_WAIT_NS);
            if (!__all_sync(0xffffffffu, ok) || *fail) {
                *fail = 1;
                break;
            }
            tc_fence_after();
            epilogue_row<TN, EPI>(a, tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)(acc * TN),
                                  mt * GM_M + warp * 32 + lane, nt * TN, nt);
            tc_fence_before();
            mbar_arrive(&tempty[acc]);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*fail && tid == 0) {
        if (a.status) atomicOr(a.status, B2S_STATUS_WAIT_TIMEOUT);
        // loads issued but not seen landing still write this CTA's shared memory
        for (int it = *consumed; it < *issued; ++it)
            mbar_wait_bounded(&full[it % ST], (uint32_t)(it / ST) & 1u, HEAD_WAIT_NS);
    }
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * TN);
    }
}

template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, uint32_t smem, void* stream, A... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// An operand of a product: rows of `k` elements `stride` apart (k contiguous), or, transposed, k rows of `m` elements.
struct Operand {
    const void* base;
    int64_t stride;
};

template <int TN, bool AMN, bool BMN, int EPI>
int gemm_tn(const Operand& A, const Operand& B, int64_t K, GemmArgs a, void* stream) {
    CUtensorMap amap, bmap;
    int rc = AMN ? tensor_map_2d(&amap, A.base, a.M, K, A.stride, 64, GM_KB)
                 : tensor_map_2d(&amap, A.base, K, a.M, A.stride, GM_KB, GM_M);
    if (rc == B2S_OK)
        rc = BMN ? tensor_map_2d(&bmap, B.base, a.N, K, B.stride, 64, GM_KB)
                 : tensor_map_2d(&bmap, B.base, K, a.N, B.stride, GM_KB, TN);
    if (rc != B2S_OK) return rc;
    a.tiles_m = (a.M + GM_M - 1) / GM_M;
    a.tiles_n = (a.N + TN - 1) / TN;
    a.nkb = (int)((K + GM_KB - 1) / GM_KB);
    int sms = 0;
    cudaError_t e = device_sms(&sms);
    if (e != cudaSuccess) return cuda_fail(e);
    const auto kernel = gemm_kernel<TN, AMN, BMN, EPI>;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gm_smem(TN));
    if (e != cudaSuccess) return cuda_fail(e);
    const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
    e = launch_pdl(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), GM_THREADS, gm_smem(TN), stream, amap, bmap, a);
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

int tile_cols(int M, int N) {
    int sms = 0;
    if (device_sms(&sms) != cudaSuccess) sms = 148;
    const int64_t mt = (M + GM_M - 1) / GM_M;
    for (int tn = 256; tn > 64; tn >>= 1)
        if (mt * ((N + tn - 1) / tn) >= sms) return tn;
    return 64;
}

template <bool AMN, bool BMN, int EPI>
int gemm(const Operand& A, const Operand& B, int64_t K, const GemmArgs& a, void* stream) {
    switch (tile_cols(a.M, a.N)) {
        case 256: return gemm_tn<256, AMN, BMN, EPI>(A, B, K, a, stream);
        case 128: return gemm_tn<128, AMN, BMN, EPI>(A, B, K, a, stream);
        default: return gemm_tn<64, AMN, BMN, EPI>(A, B, K, a, stream);
    }
}

// ------------------------------------------------------------------ the head's log probabilities

constexpr int LM_NT = 128;
// One CTA per row: the column tiles' states into the row's outputs.
__global__ void __launch_bounds__(LM_NT) lmhead_merge_kernel(const float4* part, int tiles, const float* token_value,
                                                             const int64_t* tokens, int V, float c, float* logprob,
                                                             float* entropy, float4* stats, uint32_t* status) {
    pdl_wait_then_release();
    __shared__ LpState sw[LM_NT / 32];
    const int r = blockIdx.x, tid = threadIdx.x;
    LpState s;
    s.m = f_ninf();
    s.S = s.U = 0.0f;
    for (int i = tid; i < tiles; i += LM_NT) {
        const float4 p = part[(int64_t)r * tiles + i];
        LpState o;
        o.m = p.x;
        o.S = p.y;
        o.U = p.z;
        s = lp_merge(s, o, c);
    }
    lp_warp_merge(s, c);
    if ((tid & 31) == 0) sw[tid >> 5] = s;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < LM_NT / 32; ++w) s = lp_merge(s, sw[w], c);
        const LpFinal f = lp_final(s, c);
        const int64_t tok = tokens[r];
        const bool has = tok >= 0 && tok < V;
        if (logprob) logprob[r] = has ? lp_value(token_value[r], f, c) : 0.0f;
        if (entropy) entropy[r] = f.entropy;
        if (stats) stats[r] = make_float4(f.m, f.R, f.log2S, f.entropy);
        if (status && tok >= V) atomicOr(status, B2S_STATUS_TOKEN_RANGE);
    }
}

// ------------------------------------------------------------------ the projection's elementwise gradient

// dz = dy act'(z) (bf16, rows dz_stride apart) and the sums of its columns over this CTA's rows: 32 groups of 8
// columns x 8 rows in turn per CTA; the sums (fp32, of the unrounded dz) go to part[blockIdx.y][n], or, with one
// part, straight to the bias gradient.
constexpr int DZ_NT = 256;
__global__ void __launch_bounds__(DZ_NT) linear_dz_kernel(const void* dy, int64_t dy_stride, int dy_vec, const void* z,
                                                          int64_t z_stride, int act, int rows, int N, int rows_per,
                                                          void* dz, int64_t dz_stride, float* part, void* db) {
    pdl_wait_then_release();
    __shared__ float red[8][32][9];
    const int cg = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int n = (blockIdx.x * 32 + cg) * 8;
    const int r0 = blockIdx.y * rows_per, r1 = min(rows, r0 + rows_per);
    float sum[8] = {};
    if (n < N) {
        for (int r = r0 + rl; r < r1; r += 8) {
            float g[8];
            load8(static_cast<const unsigned char*>(dy) + (int64_t)r * dy_stride * 2, n, N, dy_vec, g);
            if (act != ACT_NONE) {
                float x[8];
                load8(static_cast<const unsigned char*>(z) + (int64_t)r * z_stride * 2, n, N, true, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] *= act_slope(x[j], act);
            }
            if (dz) store8(static_cast<unsigned char*>(dz) + (int64_t)r * dz_stride * 2, n, N, true, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += g[j];
        }
    }
    if (!part && !db) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[rl][cg][j] = sum[j];
    __syncthreads();
    const int i = threadIdx.x, c = i >> 3, j = i & 7;  // one column per thread
    float s = red[0][c][j];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][c][j];
    const int col = blockIdx.x * 256 + i;
    if (col < N) {
        if (part) part[(int64_t)blockIdx.y * N + col] = s;
        else static_cast<__nv_bfloat16*>(db)[col] = __float2bfloat16_rn(s);
    }
}
__global__ void linear_db_kernel(const float* part, int parts, int N, void* db) {
    pdl_wait_then_release();
    const int n = blockIdx.x * blockDim.x + threadIdx.x;
    if (n >= N) return;
    float s = 0.0f;
    for (int p = 0; p < parts; ++p) s += part[(int64_t)p * N + n];
    static_cast<__nv_bfloat16*>(db)[n] = __float2bfloat16_rn(s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
// parts of the rows whose column sums are taken separately: enough CTAs to fill the GPU, at least 64 rows each
int dz_parts(int rows, int N) {
    const int64_t cols = (N + 255) / 256;
    int64_t p = (4 * 148 + cols - 1) / cols;
    if (p > (rows + 63) / 64) p = (rows + 63) / 64;
    return (int)(p < 1 ? 1 : p);
}

int check_head(const void* hidden, int64_t hstride, const void* head, int64_t wstride, int H, int V, int rows,
               float temperature) {
    if (rows < 0 || V < 1 || H < 8 || H % 8 || hstride < H || hstride % 8 || wstride < H || wstride % 8)
        return B2S_ERR_INVALID;
    if (!lp_temperature_ok(temperature)) return B2S_ERR_INVALID;
    if (rows && (!hidden || !head || !aligned16(hidden) || !aligned16(head))) return B2S_ERR_INVALID;
    return B2S_OK;
}

}  // namespace
}  // namespace b2s

extern "C" {

int b2s_lmhead_logprobs_workspace(int32_t rows, int32_t vocab, int32_t hidden_dim, int64_t* bytes) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || hidden_dim < 8 || !bytes) return B2S_ERR_INVALID;
    const int tn = tile_cols(rows, vocab);
    *bytes = up((int64_t)rows * ((vocab + tn - 1) / tn) * 16 + (int64_t)rows * 4, 256);
    return B2S_OK;
}

int b2s_lmhead_logprobs(const b2s_lmhead_args* h, float* logprob, float* entropy, float* stats, void* stream) {
    using namespace b2s;
    if (!h) return B2S_ERR_INVALID;
    int rc = check_head(h->hidden, h->hidden_row_stride, h->head, h->head_row_stride, h->hidden_dim, h->vocab, h->rows,
                        h->temperature);
    if (rc != B2S_OK) return rc;
    if (h->rows == 0) return B2S_OK;
    int64_t need = 0;
    b2s_lmhead_logprobs_workspace(h->rows, h->vocab, h->hidden_dim, &need);
    if (!h->tokens || !h->workspace || h->workspace_bytes < need || !aligned16(h->workspace) || (stats && !aligned16(stats)))
        return B2S_ERR_INVALID;
    const int tn = tile_cols(h->rows, h->vocab);
    const int tiles = (h->vocab + tn - 1) / tn;
    GemmArgs a;
    memset(&a, 0, sizeof(a));
    a.M = h->rows;
    a.N = h->vocab;
    a.status = h->status;
    a.c = lp_scale(h->temperature);
    a.tokens = h->tokens;
    a.part = static_cast<float4*>(h->workspace);
    a.token_value = reinterpret_cast<float*>(a.part + (int64_t)h->rows * tiles);
    rc = gemm<false, false, EPI_LSE>({h->hidden, h->hidden_row_stride}, {h->head, h->head_row_stride}, h->hidden_dim, a,
                                     stream);
    if (rc != B2S_OK) return rc;
    const cudaError_t e = launch_pdl(lmhead_merge_kernel, dim3((unsigned)h->rows), LM_NT, 0, stream,
                                     (const float4*)a.part, tiles, (const float*)a.token_value, h->tokens,
                                     (int)h->vocab, a.c, logprob, entropy, reinterpret_cast<float4*>(stats), h->status);
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

int b2s_lmhead_logprobs_grad_workspace(int32_t rows, int32_t vocab, int32_t hidden_dim, int64_t* bytes) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || hidden_dim < 8 || !bytes) return B2S_ERR_INVALID;
    *bytes = up((int64_t)rows * up(vocab, 8) * 2, 256);
    return B2S_OK;
}

int b2s_lmhead_logprobs_grad(const b2s_lmhead_args* h, const float* stats, const float* grad_logprob,
                             const float* grad_entropy, void* grad_hidden, void* grad_head, void* stream) {
    using namespace b2s;
    if (!h) return B2S_ERR_INVALID;
    int rc = check_head(h->hidden, h->hidden_row_stride, h->head, h->head_row_stride, h->hidden_dim, h->vocab, h->rows,
                        h->temperature);
    if (rc != B2S_OK) return rc;
    if (grad_head && !aligned16(grad_head)) return B2S_ERR_INVALID;
    if (h->rows == 0) {
        if (!grad_head) return B2S_OK;
        const cudaError_t e = cudaMemsetAsync(grad_head, 0, (size_t)h->vocab * h->hidden_dim * 2, (cudaStream_t)stream);
        return e == cudaSuccess ? B2S_OK : cuda_fail(e);
    }
    int64_t need = 0;
    b2s_lmhead_logprobs_grad_workspace(h->rows, h->vocab, h->hidden_dim, &need);
    if (!h->tokens || !h->workspace || h->workspace_bytes < need || !aligned16(h->workspace) || !stats ||
        !aligned16(stats) || (grad_hidden && !aligned16(grad_hidden)))
        return B2S_ERR_INVALID;
    const int64_t ldz = up(h->vocab, 8);
    GemmArgs a;
    memset(&a, 0, sizeof(a));
    a.M = h->rows;
    a.N = h->vocab;
    a.status = h->status;
    a.c = lp_scale(h->temperature);
    a.inv_t = (float)(1.0 / (double)h->temperature);
    a.tokens = h->tokens;
    a.stats = reinterpret_cast<const float4*>(stats);
    a.g_lp = grad_logprob;
    a.g_h = grad_entropy;
    a.out = h->workspace;
    a.out_stride = ldz;
    a.out_vec = 1;
    rc = gemm<false, false, EPI_DZ>({h->hidden, h->hidden_row_stride}, {h->head, h->head_row_stride}, h->hidden_dim, a,
                                    stream);
    if (rc != B2S_OK) return rc;
    GemmArgs b;
    memset(&b, 0, sizeof(b));
    b.status = h->status;
    b.out_vec = 1;
    b.N = h->hidden_dim;
    b.out_stride = h->hidden_dim;
    if (grad_hidden) {
        b.M = h->rows;
        b.out = grad_hidden;
        rc = gemm<false, true, EPI_STORE>({h->workspace, ldz}, {h->head, h->head_row_stride}, h->vocab, b, stream);
        if (rc != B2S_OK) return rc;
    }
    if (grad_head) {
        b.M = h->vocab;
        b.out = grad_head;
        rc = gemm<true, true, EPI_STORE>({h->workspace, ldz}, {h->hidden, h->hidden_row_stride}, h->rows, b, stream);
    }
    return rc;
}

int b2s_linear_workspace(int32_t rows, int32_t in_features, int32_t out_features, int64_t* bytes) {
    if (rows < 0 || in_features < 8 || out_features < 1 || !bytes) return B2S_ERR_INVALID;
    *bytes = 0;
    return B2S_OK;
}

int b2s_linear(const b2s_linear_args* l, void* stream) {
    using namespace b2s;
    if (!l || l->rows < 0 || l->out_features < 1 || l->in_features < 8 || l->in_features % 8 || l->activation < 0 ||
        l->activation > B2S_ACT_SILU)
        return B2S_ERR_INVALID;
    if (l->rows == 0) return B2S_OK;
    if (!l->x || !l->weight || !l->out || !aligned16(l->x) || !aligned16(l->weight) || l->x_row_stride < l->in_features ||
        l->x_row_stride % 8 || l->weight_row_stride < l->in_features || l->weight_row_stride % 8 ||
        l->out_row_stride < l->out_features || (l->bias && !aligned16(l->bias)) ||
        (l->residual && l->residual_row_stride < l->out_features) ||
        (l->preact && (!aligned16(l->preact) || l->preact_row_stride < l->out_features || l->preact_row_stride % 8)) ||
        ((reinterpret_cast<uintptr_t>(l->out) | reinterpret_cast<uintptr_t>(l->residual)) & 1))
        return B2S_ERR_INVALID;
    GemmArgs a;
    memset(&a, 0, sizeof(a));
    a.M = l->rows;
    a.N = l->out_features;
    a.status = l->status;
    a.out = l->out;
    a.out_stride = l->out_row_stride;
    a.out_vec = aligned16(l->out) && l->out_row_stride % 8 == 0;
    a.bias = l->bias;
    a.residual = l->residual;
    a.res_stride = l->residual_row_stride;
    a.res_vec = aligned16(l->residual) && l->residual_row_stride % 8 == 0;
    a.act = l->activation;
    a.preact = l->preact;
    a.pre_stride = l->preact_row_stride;
    return gemm<false, false, EPI_LINEAR>({l->x, l->x_row_stride}, {l->weight, l->weight_row_stride}, l->in_features, a,
                                          stream);
}

int b2s_linear_grad_workspace(int32_t rows, int32_t in_features, int32_t out_features, int64_t* bytes) {
    using namespace b2s;
    if (rows < 0 || in_features < 8 || out_features < 1 || !bytes) return B2S_ERR_INVALID;
    *bytes = up((int64_t)rows * up(out_features, 8) * 2, 256) +
             up((int64_t)dz_parts(rows, out_features) * out_features * 4, 256);
    return B2S_OK;
}

int b2s_linear_grad(const b2s_linear_grad_args* l, void* stream) {
    using namespace b2s;
    if (!l || l->rows < 0 || l->out_features < 1 || l->in_features < 8 || l->in_features % 8 || l->activation < 0 ||
        l->activation > B2S_ACT_SILU || (l->grad_weight && !aligned16(l->grad_weight)))
        return B2S_ERR_INVALID;
    if (l->rows == 0) {  // sums over no rows
        cudaError_t e = cudaSuccess;
        if (l->grad_weight)
            e = cudaMemsetAsync(l->grad_weight, 0, (size_t)l->out_features * l->in_features * 2, (cudaStream_t)stream);
        if (e == cudaSuccess && l->grad_bias)
            e = cudaMemsetAsync(l->grad_bias, 0, (size_t)l->out_features * 2, (cudaStream_t)stream);
        return e == cudaSuccess ? B2S_OK : cuda_fail(e);
    }
    int64_t need = 0;
    b2s_linear_grad_workspace(l->rows, l->in_features, l->out_features, &need);
    if (!l->grad_out || l->grad_out_row_stride < l->out_features || (reinterpret_cast<uintptr_t>(l->grad_out) & 1) ||
        !l->workspace || !aligned16(l->workspace) || l->workspace_bytes < need ||
        (l->activation != B2S_ACT_NONE &&
         (!l->preact || !aligned16(l->preact) || l->preact_row_stride < l->out_features || l->preact_row_stride % 8)) ||
        (l->grad_x && (!l->weight || !aligned16(l->weight) || !aligned16(l->grad_x) ||
                       l->weight_row_stride < l->in_features || l->weight_row_stride % 8)) ||
        (l->grad_weight && (!l->x || !aligned16(l->x) || l->x_row_stride < l->in_features || l->x_row_stride % 8)))
        return B2S_ERR_INVALID;
    const int64_t ldz = up(l->out_features, 8);
    const bool dy_vec = aligned16(l->grad_out) && l->grad_out_row_stride % 8 == 0;
    // without an activation dz is dy itself, where the tensor maps can read it
    const bool direct = l->activation == B2S_ACT_NONE && dy_vec;
    const bool products = l->grad_x || l->grad_weight;
    Operand dz = {l->workspace, ldz};
    if (direct) dz = {l->grad_out, l->grad_out_row_stride};
    if ((products && !direct) || l->grad_bias) {
        const int parts = dz_parts(l->rows, l->out_features);
        float* part = reinterpret_cast<float*>(static_cast<unsigned char*>(l->workspace) + up((int64_t)l->rows * ldz * 2, 256));
        const int per = (l->rows + parts - 1) / parts;
        const bool two = l->grad_bias && parts > 1;
        cudaError_t e = launch_pdl(linear_dz_kernel, dim3((unsigned)((l->out_features + 255) / 256), (unsigned)parts),
                                   DZ_NT, 0, stream, l->grad_out, l->grad_out_row_stride, (int)dy_vec, l->preact,
                                   l->preact_row_stride, (int)l->activation, (int)l->rows, (int)l->out_features, per,
                                   products && !direct ? l->workspace : nullptr, ldz, two ? part : nullptr,
                                   two ? nullptr : l->grad_bias);
        if (e == cudaSuccess && two)
            e = launch_pdl(linear_db_kernel, dim3((unsigned)((l->out_features + 127) / 128)), 128, 0, stream,
                           (const float*)part, parts, (int)l->out_features, l->grad_bias);
        if (e != cudaSuccess) return cuda_fail(e);
    }
    GemmArgs b;
    memset(&b, 0, sizeof(b));
    b.status = l->status;
    b.out_vec = 1;
    b.N = l->in_features;
    b.out_stride = l->in_features;
    int rc = B2S_OK;
    if (l->grad_x) {
        b.M = l->rows;
        b.out = l->grad_x;
        rc = gemm<false, true, EPI_STORE>(dz, {l->weight, l->weight_row_stride}, l->out_features, b, stream);
        if (rc != B2S_OK) return rc;
    }
    if (l->grad_weight) {
        b.M = l->out_features;
        b.out = l->grad_weight;
        rc = gemm<true, true, EPI_STORE>(dz, {l->x, l->x_row_stride}, l->rows, b, stream);
    }
    return rc;
}

}  // extern "C"
