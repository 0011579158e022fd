// The product kernel and what is built on it: the head's log probabilities (logits never written), their gradient,
// the projection with bias, activation and residual in its epilogue, and its gradient.  No counterpart in the
// reference, whose call sites use F.linear.
#include <string.h>

#include <atomic>

#include "b2s_gemm.cuh"

namespace b2s {

int cuda_fail(cudaError_t e);
int tensor_map_2d(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int64_t outer_stride, int box_inner,
                  int box_outer);

namespace {

// Tile t (TM rows each) of the order that takes GM_GROUP x 128 rows at a time.
template <int TM>
__device__ __forceinline__ void tile_of(const GemmArgs& a, int64_t t, int* mt, int* nt) {
    constexpr int GROUP = GM_GROUP * GM_M / TM;
    const int64_t per = (int64_t)GROUP * a.tiles_n;
    const int g = (int)(t / per), in = (int)(t % per);
    const int gm = min(GROUP, a.tiles_m - g * GROUP);
    *mt = g * GROUP + in % gm;
    *nt = in / gm;
}

// The i-th piece of work of CTA (or pair) c of G: a tile and its k blocks [kb0, kb1); slot: where its sums go, -1 for a whole tile.
struct Piece {
    int64_t tile;
    int kb0, kb1, slot;
};
template <int CG>
__device__ __forceinline__ bool piece_at(const GemmArgs& a, int i, Piece* p) {
    const int c = (int)blockIdx.x / CG, G = (int)gridDim.x / CG;
    p->kb0 = 0;
    p->kb1 = a.nkb;
    p->slot = -1;
    if (i < a.waves) {
        p->tile = (int64_t)i * G + c;
        return true;
    }
    const int64_t u = (int64_t)(i - a.waves) * G + c;
    if (u >= (int64_t)a.rest * a.split) return false;
    p->tile = (int64_t)a.waves * G + u % a.rest;
    if (a.split > 1) {
        p->kb0 = (int)(u / a.rest) * a.chunk;
        p->kb1 = min(a.nkb, p->kb0 + a.chunk);
        p->slot = (int)u;
    }
    return true;
}

template <int N>
__device__ __forceinline__ void fill_nan(float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = __int_as_float(0x7fffffff);
}
// Whether a block of 32 columns from n is copied as 16-byte vectors.
__device__ __forceinline__ bool vec_block(const GemmArgs& a, int n, int aligned) { return aligned && n + 32 <= a.N; }
// The residual's block of 32 columns from n of the 32 rows from row0.
__device__ __forceinline__ void residual_fetch(const GemmArgs& a, uint32_t (&q)[16], int row0, int n) {
    if (a.residual && n < a.N)
        block_fetch(q, static_cast<const unsigned short*>(a.residual) + (int64_t)row0 * a.res_stride + n, a.res_stride,
                    a.M - row0, a.N - n, vec_block(a, n, a.res_vec));
}

// The epilogue of one warp: 32 rows of a tile, columns [n0, n0 + COLS) from tensor memory at `tm` (lane = row).  `rq`:
// the residual's first block.  Not `good`: the accumulator was given up, and NaN takes its place.
template <int TM, int TN, int EPI>
__device__ __forceinline__ void epilogue_rows(const GemmArgs& a, uint32_t tm, bool good, int row0, int n0, int nt, int slot,
                                              unsigned char* st, uint32_t (&rq)[16]) {
    constexpr int COLS = TN / 2;
    const int lane = threadIdx.x & 31;
    const int rows = min(32, a.M - row0);  // <= 0: a warp past the last row
    {
        if (slot >= 0) {  // a chunk of a split tile: its fp32 sums as they are
            const int held = min(a.M, TM);
            float* dst = a.partial + ((int64_t)slot * held + row0 % TM) * TN + n0 - nt * TN;
#pragma unroll 1
            for (int q = 0; q < COLS / 32; ++q) {
                float v[32];
                if (good) tmem_ld32(tm + 32u * q, v);
                else fill_nan(v);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *stage_at(st, lane, j) = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                                        __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 32; h += 16) {  // read before it is stored, as in block_store
                    uint4 u[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) u[i] = *stage_at(st, h + 4 * i + (lane >> 3), lane & 7);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = h + 4 * i + (lane >> 3);
                        if (r < rows) *reinterpret_cast<uint4*>(dst + (int64_t)r * TN + 32 * q + 4 * (lane & 7)) = u[i];
                    }
                }
                __syncwarp();
            }
            return;
        }
        unsigned short* out = static_cast<unsigned short*>(a.out) + (int64_t)row0 * a.out_stride;
        const bool with_res = EPI == EPI_LINEAR && a.residual;
#pragma unroll 1
        for (int q = 0; q < COLS / 32; ++q) {
            const int n = n0 + 32 * q, cols = a.N - n;
            if (cols <= 0) break;
            if (with_res) {
                block_put(st, rq, vec_block(a, n, a.res_vec));
                if (q + 1 < COLS / 32) residual_fetch(a, rq, row0, n + 32);  // in flight under this block
                __syncwarp();
            }
            float v[32];
            if (good) tmem_ld32(tm + 32u * q, v);
            else fill_nan(v);
            if constexpr (EPI == EPI_LINEAR) {
                if (a.bias) {
                    const float b = lane < cols ? bf16_bits_to_f(__ldg(static_cast<const unsigned short*>(a.bias) + n + lane)) : 0.0f;
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] += __shfl_sync(0xffffffffu, b, j);
                }
                if (a.preact) stage_preact(st, v);
                if (a.act == ACT_RELU) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = act_apply<ACT_RELU>(v[j]);
                } else if (a.act == ACT_GELU) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = act_apply<ACT_GELU>(v[j]);
                } else if (a.act == ACT_SILU) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = act_apply<ACT_SILU>(v[j]);
                }
                if (with_res) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 u = *stage_at(st, lane, j);
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            v[8 * j + 2 * k] += __uint_as_float(w[k] << 16);
                            v[8 * j + 2 * k + 1] += __uint_as_float(w[k] & 0xffff0000u);
                        }
                    }
                }
            }
            stage_row(st, 0, v);  // over this lane's own row of the residual
            __syncwarp();
            block_store(st, 0, out + n, a.out_stride, rows, cols, vec_block(a, n, a.out_vec));
            if (EPI == EPI_LINEAR && a.preact)
                block_store(st, 4, static_cast<unsigned short*>(a.preact) + (int64_t)row0 * a.pre_stride + n, a.pre_stride,
                            rows, cols, vec_block(a, n, 1));
            __syncwarp();
        }
    }
}

// The head's epilogues: this lane's row of COLS fp32 logits (before the temperature) from column n0.
template <int COLS, int EPI>
__device__ __forceinline__ void epilogue_logits(const GemmArgs& a, const float (&v)[COLS], int row0, int n0, int half, int nt,
                                                unsigned char* st) {
    const int lane = threadIdx.x & 31, row = row0 + lane;
    const bool live = row < a.M;
    const int64_t tok = live ? a.tokens[row] : -1;
    if constexpr (EPI == EPI_LSE) {
        LpState s;
        s.m = f_ninf();
        s.S = s.U = 0.0f;
        if (tok >= n0 && tok < min(n0 + COLS, a.N)) {
            float tv = v[0];
#pragma unroll
            for (int j = 1; j < COLS; ++j) tv = tok == n0 + j ? v[j] : tv;
            a.token_value[row] = tv;
        }
#pragma unroll
        for (int q = 0; q < COLS / 32; ++q) {
            const int n = n0 + 32 * q;
            if (n < a.N) {
                float x[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = n + j < a.N ? v[32 * q + j] : f_ninf();
                lp_add_any<32>(s, x, a.c);
            }
        }
        if (live) a.part[((int64_t)row * a.tiles_n + nt) * 2 + half] = make_float4(s.m, s.S, s.U, 0.0f);
    } else {
        const int rows = min(32, a.M - row0);
        const float4 stt = live ? a.stats[row] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const LpGrad g(stt, tok >= 0 && tok < a.N ? (int)tok : -1, live && a.g_lp ? a.g_lp[row] : 0.0f,
                       live && a.g_h ? a.g_h[row] : 0.0f, a.inv_t);
        unsigned short* out = static_cast<unsigned short*>(a.out) + (int64_t)row0 * a.out_stride;
#pragma unroll
        for (int q = 0; q < COLS / 32; ++q) {
            const int n = n0 + 32 * q, cols = a.N - n;
            if (cols > 0) {
                float x[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = g.at(v[32 * q + j], n + j, a.c);
                // dz is rounded to bf16 once: it is the tensor cores' operand in both gradient products
                stage_row(st, 0, x);
                __syncwarp();
                block_store(st, 0, out + n, a.out_stride, rows, cols, vec_block(a, n, 1));
                __syncwarp();
            }
        }
    }
}

template <int CG, int TN, bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(GM_THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                const __grid_constant__ GemmArgs a) {
    constexpr int TM = CG * GM_M, BN = TN / CG;  // rows of a tile; this CTA's columns of B
    constexpr int ST = gm_stages(CG, TN), SEGMENT = EPI == EPI_LSE || EPI == EPI_DZ ? GM_SEGMENT : 1 << 24;
    constexpr uint32_t STAGE = gm_stage_bytes(CG, TN);
    constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)AMN << 15) | ((uint32_t)BMN << 16) |
                               ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
    extern __shared__ __align__(128) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
    const uint32_t base_u = smem_u32(smem_raw);
    unsigned char* sm = smem_raw + (((base_u + 1023u) & ~1023u) - base_u);
    unsigned char* staging = sm + ST * STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + GM_STAGING);  // the first CTA's serves both
    uint64_t* empty = full + ST;
    uint64_t* tfull = empty + ST;   // [2] an accumulator is complete
    uint64_t* tempty = tfull + 2;   // [2] an accumulator has been read (the first CTA's, by both)
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
            mbar_init(&tempty[s], 32 * GM_EPI * CG);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
        *fail = 0;
        *issued = 0;
        *consumed = 0;
    }
    if (warp == GM_EPI + 1) {
        if constexpr (CG == 2) tmem_alloc_pair(tslot, 2 * TN);
        else tmem_alloc(tslot, 2 * TN);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) {  // the partner's mbarriers exist before anything signals them
        cluster_arrive_release();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem = *tslot;
    pdl_wait_then_release();

    // The loading and the issuing warp run their loops converged, one lane elected where something is issued: with the
    // loops inside a one-lane branch a k block cost the issuing thread 580 clocks, more than its MMAs' 512.
    if (warp == GM_EPI) {
        int s = 0, it = 0;
        uint32_t ph = 1;  // parity of `empty`'s last phase: the first round finds every stage free
        bool ok = a.wait > 0;
        const uint32_t bar0 = CG == 2 ? mapa_shared(smem_u32(full), 0) : smem_u32(full);
        Piece p;
        for (int i = 0; ok && piece_at<CG>(a, i, &p); ++i) {
            int mt, nt;
            tile_of<TM>(a, p.tile, &mt, &nt);
            const int m0 = mt * TM + (int)rank * GM_M, n0 = nt * TN + (int)rank * BN;
            for (int kb = p.kb0; kb < p.kb1; ++kb, ++it) {
                if (!__all_sync(0xffffffffu, gm_wait<false>(&empty[s], ph, a.wait))) {
                    *fail = 1;
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    unsigned char* sa = sm + s * STAGE;
                    unsigned char* sb = sa + GM_A_BYTES;
                    // parts outside the tensors are filled with zeros and count as bytes
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], CG * STAGE);
                    auto load = [&](unsigned char* dst, const CUtensorMap* map, int x, int y) {
                        if constexpr (CG == 2) tma_load_2d_pair(dst, map, x, y, bar0 + 8u * s);
                        else tma_load_2d(dst, map, x, y, &full[s]);
                    };
                    if constexpr (AMN) {
#pragma unroll
                        for (int j = 0; j < GM_M / 64; ++j) load(sa + 8192 * j, &amap, m0 + 64 * j, kb * GM_KB);
                    } else {
                        load(sa, &amap, kb * GM_KB, m0);
                    }
                    if constexpr (BMN) {
#pragma unroll
                        for (int j = 0; j < BN / 64; ++j) load(sb + 8192 * j, &bmap, n0 + 64 * j, kb * GM_KB);
                    } else {
                        load(sb, &bmap, kb * GM_KB, n0);
                    }
                }
                __syncwarp();
                if (++s == ST) {
                    s = 0;
                    ph ^= 1;
                }
            }
        }
        if (lane == 0) *issued = it;
        // the first CTA's last signals to this CTA's `empty` have landed before it leaves
        if (CG == 2 && ok)
            for (int k = it > ST ? it - ST : 0; k < it; ++k)
                if (!gm_wait<false>(&empty[k % ST], (uint32_t)(k / ST) & 1u, a.wait)) {
                    *fail = 1;
                    break;
                }
    } else if (warp == GM_EPI + 1) {
        if (rank == 0) {  // MMAs
            int s = 0, it = 0;
            uint32_t ph = 0;
            bool ok = a.wait > 0;
            const uint64_t da0 = AMN ? umma_desc_mn128(smem_u32(sm)) : umma_desc_sw128(smem_u32(sm));
            const uint64_t db0 = BMN ? umma_desc_mn128(smem_u32(sm) + GM_A_BYTES) : umma_desc_sw128(smem_u32(sm) + GM_A_BYTES);
            auto commit = [&](uint64_t* bar) {
                if constexpr (CG == 2) umma_commit_pair(bar);
                else umma_commit(bar);
            };
            Piece p;
            int g = 0;  // accumulators handed over
            for (int i = 0; ok && piece_at<CG>(a, i, &p); ++i) {
                for (int k0 = p.kb0; ok && k0 < p.kb1; k0 += SEGMENT, ++g) {
                    const int acc = g & 1, k1 = min(p.kb1, k0 + SEGMENT);
                    if (g >= 2 && !__all_sync(0xffffffffu, gm_wait<CG == 2>(&tempty[acc], (uint32_t)(g / 2 - 1) & 1u, a.wait))) {
                        *fail = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + (uint32_t)(acc * TN);
                    uint32_t more = 0;
                    for (int kb = k0; kb < k1; ++kb, ++it) {
                        if (!__all_sync(0xffffffffu, gm_wait<false>(&full[s], ph, a.wait))) {
                            *fail = 1;
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            // a stage is STAGE bytes on, a step of 16 k 32 bytes (k contiguous) or 2 KB, in units of 16
                            const uint64_t da = da0 + (uint32_t)s * (STAGE >> 4), db = db0 + (uint32_t)s * (STAGE >> 4);
#pragma unroll
                            for (int k = 0; k < GM_KB / 16; ++k) {
                                if constexpr (CG == 2)
                                    umma_bf16_pair(d, da + (AMN ? 128 : 2) * k, db + (BMN ? 128 : 2) * k, IDESC, more);
                                else
                                    umma_bf16(d, da + (AMN ? 128 : 2) * k, db + (BMN ? 128 : 2) * k, IDESC, more);
                                more = 1;
                            }
                            commit(&empty[s]);
                            if (kb + 1 == k1) commit(&tfull[acc]);
                        }
                        more = 1;
                        __syncwarp();
                        if (++s == ST) {
                            s = 0;
                            ph ^= 1;
                        }
                    }
                }
            }
            if (lane == 0) *consumed = it;
        }
    } else {
        Piece p;
        int g = 0;
        bool ok = a.wait > 0;
        if (!ok) *fail = 1;
        const int half = warp >> 2;
        const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * (TN / 2));
        auto take = [&]() {  // the next accumulator
            ok = ok && __all_sync(0xffffffffu, gm_wait<false>(&tfull[g & 1], (uint32_t)(g / 2) & 1u, a.wait) && !*fail);
            if (!ok) *fail = 1;
            tc_fence_after();
            return ok;
        };
        auto give = [&]() {
            if (!ok) return;
            tc_fence_before();
            if constexpr (CG == 2) mbar_arrive_remote(mapa_shared(smem_u32(&tempty[g & 1]), 0));
            else mbar_arrive(&tempty[g & 1]);
            ++g;
        };
        // once a wait gave up the pieces that are left take NaN without waiting
        for (int i = 0; piece_at<CG>(a, i, &p); ++i) {
            int mt, nt;
            tile_of<TM>(a, p.tile, &mt, &nt);
            const int row0 = mt * TM + (int)rank * GM_M + (warp & 3) * 32, n0 = nt * TN + half * (TN / 2);
            if constexpr (EPI == EPI_LSE || EPI == EPI_DZ) {
                float v[TN / 2];
                take();  // what was given up is read all the same: any values, replaced below
#pragma unroll
                for (int q = 0; q < TN / 64; ++q) tmem_ld32(tm + (uint32_t)((g & 1) * TN + 32 * q), v + 32 * q);
                give();
#pragma unroll 1
                for (int k0 = p.kb0 + SEGMENT; k0 < p.kb1; k0 += SEGMENT) {
                    take();
#pragma unroll
                    for (int q = 0; q < TN / 32; ++q) {
                        uint32_t x[16];
                        tmem_ld16(tm + (uint32_t)((g & 1) * TN + 16 * q), x);
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[16 * q + j] += __uint_as_float(x[j]);
                    }
                    give();
                }
                if (!ok) fill_nan(v);
                if (EPI == EPI_LSE && p.slot >= 0) {  // a chunk of a split tile: fp32 sums, for lmhead_merge_kernel
                    const int row = row0 + lane;
                    float4* dst = reinterpret_cast<float4*>(a.partial + ((int64_t)p.slot * min(a.M, TM) + row) * TN + half * (TN / 2));
                    if (row < a.M) {
#pragma unroll
                        for (int j = 0; j < TN / 8; ++j) dst[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                } else {
                    epilogue_logits<TN / 2, EPI>(a, v, row0, n0, half, nt, staging + warp * 4096);
                }
            } else {
                uint32_t rq[16];
                if (EPI == EPI_LINEAR && p.slot < 0) residual_fetch(a, rq, row0, n0);  // before the accumulator is there
                take();
                epilogue_rows<TM, TN, EPI>(a, tm + (uint32_t)((g & 1) * TN), ok, row0, n0, nt, p.slot, staging + warp * 4096, rq);
                give();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*fail && warp == GM_EPI + 1 && rank == 0) {  // every MMA issued has completed
        if (elect_one()) {
            if constexpr (CG == 2) umma_commit_pair(drain);
            else umma_commit(drain);
        }
        __syncwarp();
        gm_wait<false>(drain, 0u);
        tc_fence_before();
    }
    if (*fail && tid == 0) {
        if (a.status) atomicOr(a.status, B2S_STATUS_WAIT_TIMEOUT);
        // loads issued but not seen landing still write this CTA's shared memory: those that the first CTA counts are
        // waited for, any other for a millisecond, a thousand times what a load takes
        if (rank == 0)
            for (int it = *consumed; it < *issued; ++it)
                gm_wait<false>(&full[it % ST], (uint32_t)(it / ST) & 1u);
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {
        }
    }
    if (*fail) __syncthreads();  // the same for all: nothing writes it after the barrier above
    if constexpr (CG == 2) {  // neither CTA leaves while the other may signal it or its MMAs read its shared memory
        __syncwarp();
        cluster_arrive_release();
        cluster_wait();
    }
    if (warp == GM_EPI + 1) {
        tc_fence_after();
        if constexpr (CG == 2) tmem_dealloc_pair(tmem, 2 * TN);
        else tmem_dealloc(tmem, 2 * TN);
    }
}

template <typename... P, typename... A>
cudaError_t launch_cluster(void (*kernel)(P...), dim3 grid, int cluster, int threads, uint32_t smem, void* stream,
                           A... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
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
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, uint32_t smem, void* stream, A... args) {
    return launch_cluster(kernel, grid, 1, threads, smem, stream, args...);
}

// Adds a split tile's sums in k order and runs the epilogue: a thread per 4 columns of a row, grid.y = the split tiles.
constexpr int FIX_NT = 256;
template <int TM, int TN, int EPI>
__global__ void __launch_bounds__(FIX_NT) gemm_join_kernel(const __grid_constant__ GemmArgs a, int G) {
    pdl_wait_then_release();
    int mt, nt;
    tile_of<TM>(a, (int64_t)a.waves * G + blockIdx.y, &mt, &nt);
    const int held = min(a.M, TM), rows = min(TM, a.M - mt * TM);
    const int i = (int)blockIdx.x * FIX_NT + (int)threadIdx.x;
    const int lr = i / (TN / 4), n = nt * TN + (i % (TN / 4)) * 4, row = mt * TM + lr;
    if (lr >= rows || n >= a.N) return;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const float* part = a.partial + ((int64_t)blockIdx.y * held + lr) * TN + n - nt * TN;
    const int64_t step = (int64_t)a.rest * held * TN;
#pragma unroll 4
    for (int s = 0; s < a.split; ++s) {
        const float4 p = *reinterpret_cast<const float4*>(part + s * step);
        v[0] += p.x;
        v[1] += p.y;
        v[2] += p.z;
        v[3] += p.w;
    }
    unsigned short* out = static_cast<unsigned short*>(a.out) + (int64_t)row * a.out_stride + n;
    const int cols = min(4, a.N - n);
    if (EPI == EPI_LINEAR) {
        const unsigned short* bias = static_cast<const unsigned short*>(a.bias);
        const unsigned short* res = static_cast<const unsigned short*>(a.residual) + (int64_t)row * a.res_stride + n;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < cols) {
                if (bias) v[j] += bf16_bits_to_f(__ldg(bias + n + j));
                if (a.preact)
                    (static_cast<unsigned short*>(a.preact) + (int64_t)row * a.pre_stride + n)[j] = preact_bits(v[j]);
                v[j] = act_apply(v[j], a.act);
                if (a.residual) v[j] += bf16_bits_to_f(__ldg(res + j));
            }
        }
    }
    if (a.out_vec && cols == 4) {
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cols) out[j] = __bfloat16_as_ushort(__float2bfloat16_rn(v[j]));
    }
}

// An operand of a product: rows of `k` elements `stride` apart (k contiguous), or, transposed, k rows of `m` elements.
struct Operand {
    const void* base;
    int64_t stride;
};

// How a product is cut: CTAs per tile, columns per tile, CTAs (or pairs) at work, whole waves, the rest and the chunks
// along k that the rest is cut into.
struct Plan {
    int cg, tn, G, waves, rest, split, chunk;
    int64_t bytes;  // of the split's workspace
};
// The cheapest cut by estimated clocks.  A k block costs a CTA its MMAs (measured without loads: 530 clocks for 256 or
// 128 columns alike, 290 for 64) or its stage's way from L2 (64 bytes a clock; rows outside A are not fetched).  An
// epilogue costs 14 clocks a column where it only stores, 40 with the projection's bias, activation, residual and
// pre-activation, and is hidden under the next tile's k blocks except the last one's.  A split costs a second launch,
// about 9000 clocks with its wait, and its sums' way out and back, about 3000 bytes a clock over all SMs.
Plan plan_for(int M, int N, int64_t K, int epi, int sms) {
    const bool may_split = epi == EPI_LINEAR || epi == EPI_STORE;
    Plan best = {};
    int64_t best_cost = INT64_MAX;
    const int64_t nkb = (K + GM_KB - 1) / GM_KB;
    auto ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    for (int cg = 2; cg >= 1; --cg) {
        for (int tn = 256; tn >= (cg == 2 ? 128 : 64); tn >>= 1) {
            if (cg == 2 && M <= GM_M) continue;  // half of the pair would have no rows
            const int tm = cg * GM_M, U = sms / cg;
            const int64_t tiles = ceil_div(M, tm) * ceil_div(N, tn);
            const int64_t mma = tn == 64 ? 290 : 530, fill = 2 * ((M < GM_M ? M : GM_M) + tn / cg);
            const int64_t kb_cost = mma > fill ? mma : fill;
            Plan p = {};
            p.cg = cg;
            p.tn = tn;
            p.G = (int)(tiles < U ? tiles : U);
            p.waves = (int)(tiles / U);
            p.rest = (int)(tiles % U);
            p.split = 1;
            p.chunk = (int)nkb;
            const int64_t tail = (epi == EPI_LINEAR ? 40 : 14) * tn;
            auto tiles_cost = [&](int64_t rounds, int64_t nk) {
                const int64_t mine = nk * kb_cost;
                return rounds ? mine + (rounds - 1) * (mine > tail ? mine : tail) + tail : 0;
            };
            int64_t cost = tiles_cost(p.waves + (p.rest ? 1 : 0), nkb);
            // The head's states cannot be joined across k; but where whole waves leave a handful of column tiles over (a step's
            // 594 on 148 CTAs: two, which alone would stream their 4 MB at two SMs' rate), and one tile holds all rows,
            // those are split 8 ways and lmhead_merge_kernel adds their logits.  That saves a tile's way from HBM, which
            // grows with K, and costs the merge, which grows with the tiles and the rows.  Whole / split, us, 296 tiles and
            // `rest` on 148 CTAs: K = 1024, 16 rows, rest 1 41.7 / 40.4, 2 41.5 / 42.8, 8 41.7 / 54.3; K = 2048, 16 rows,
            // 2 70.6 / 68.4, 4 70.8 / 72.9; 128 rows, 1 67.1 / 66.2, 2 68.2 / 68.8; K = 4096, 16 rows, 2 126.5 / 111.1,
            // 6 127.5 / 120.2, 10 127.3 / 126.9; 128 rows, 3 129.2 / 120.1, 6 129.1 / 128.2, 8 128.9 / 131.7; K = 8192,
            // 16 rows, 10 243 / 223.
            if (epi == EPI_LSE && M <= GM_M && p.waves && p.rest && p.rest * (M > 64 ? 16 : 8) <= nkb - 16) {
                p.chunk = (int)ceil_div(nkb, 8);
                p.split = (int)ceil_div(nkb, p.chunk);
                p.bytes = (int64_t)p.split * p.rest * M * tn * 4;
                cost = tiles_cost(p.waves, nkb) + ceil_div(p.rest * p.split, U) * p.chunk * kb_cost;
            }
            if (may_split && p.rest) {
                const int64_t held = M < tm ? M : tm;
                for (int64_t want = 2; want <= nkb && want <= 64; want += want < 4 ? 1 : want / 2) {  // 2 3 4 6 9 13 19 28 42 63
                    const int64_t chunk = ceil_div(nkb, want), split = ceil_div(nkb, chunk);
                    const int64_t bytes = split * p.rest * held * tn * 4;
                    const int64_t c = tiles_cost(p.waves, nkb) + ceil_div(p.rest * split, U) * chunk * kb_cost + 14 * tn + 9000 +
                                      2 * bytes / 3000;
                    if (split > 1 && c < cost) {
                        cost = c;
                        p.split = (int)split;
                        p.chunk = (int)chunk;
                        p.bytes = bytes;
                        p.G = (int)(p.waves || p.rest * split >= U ? U : p.rest * split);
                    }
                }
            }
            if (cost < best_cost) {
                best_cost = cost;
                best = p;
            }
        }
    }
    return best;
}

// Multiprocessors of the current device (without one, where only sizes are asked for, a B200's 148).
int sms_here() {
    int sms = 0;
    return device_sms(&sms) == cudaSuccess && sms > 0 ? sms : 148;
}

// The plan on the current device.  A plan
// is a function of the sizes alone; each thread keeps its last few (making one takes the host about a microsecond, and a
// gradient asks for five).
Plan plan_here(int M, int N, int64_t K, int epi) {
    struct Kept {
        int M, N, epi, sms;
        int64_t K;
        Plan plan;
    };
    static thread_local Kept kept[16] = {};
    const int sms = sms_here();
    Kept& k = kept[((unsigned)M * 31u + (unsigned)N * 17u + (unsigned)K * 7u + (unsigned)epi) % 16u];
    if (k.M != M || k.N != N || k.K != K || k.epi != epi || k.sms != sms) {
        k.plan = plan_for(M, N, K, epi, sms);
        k.M = M;
        k.N = N;
        k.K = K;
        k.epi = epi;
        k.sms = sms;
    }
    return k.plan;
}

template <int CG, int TN, bool AMN, bool BMN, int EPI>
int gemm_tn(const Operand& A, const Operand& B, int64_t K, GemmArgs a, const Plan& p, void* stream) {
    constexpr int TM = CG * GM_M;
    a.wait = wait_limit();
    CUtensorMap amap, bmap;
    int rc = AMN ? tensor_map_2d(&amap, A.base, a.M, K, A.stride, 64, GM_KB)
                 : tensor_map_2d(&amap, A.base, K, a.M, A.stride, GM_KB, GM_M);
    if (rc == B2S_OK)
        rc = BMN ? tensor_map_2d(&bmap, B.base, a.N, K, B.stride, 64, GM_KB)
                 : tensor_map_2d(&bmap, B.base, K, a.N, B.stride, GM_KB, TN / CG);
    if (rc != B2S_OK) return rc;
    a.tiles_m = (a.M + TM - 1) / TM;
    a.tiles_n = (a.N + TN - 1) / TN;
    a.nkb = (int)((K + GM_KB - 1) / GM_KB);
    a.waves = p.waves;
    a.rest = p.rest;
    a.split = p.split;
    a.chunk = p.chunk;
    const auto kernel = gemm_kernel<CG, TN, AMN, BMN, EPI>;
    static std::atomic<bool> set[64];  // the attribute is set once per device; racing callers set the same
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e);
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gm_smem(CG, TN));
        if (e != cudaSuccess) return cuda_fail(e);
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    e = launch_cluster(kernel, dim3((unsigned)(p.G * CG)), CG, GM_THREADS, gm_smem(CG, TN), stream, amap, bmap, a);
    if constexpr (EPI == EPI_LINEAR || EPI == EPI_STORE) {
        if (e == cudaSuccess && p.split > 1) {
            const int held = a.M < TM ? a.M : TM;
            e = launch_pdl(gemm_join_kernel<TM, TN, EPI>,
                           dim3((unsigned)((held * (TN / 4) + FIX_NT - 1) / FIX_NT), (unsigned)p.rest), FIX_NT, 0, stream,
                           a, p.G);
        }
    }
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

template <bool AMN, bool BMN, int EPI>
int gemm(const Operand& A, const Operand& B, int64_t K, const GemmArgs& a, void* stream) {
    const Plan p = plan_here(a.M, a.N, K, EPI);
    if (p.cg == 2)
        return p.tn == 256 ? gemm_tn<2, 256, AMN, BMN, EPI>(A, B, K, a, p, stream)
                           : gemm_tn<2, 128, AMN, BMN, EPI>(A, B, K, a, p, stream);
    switch (p.tn) {
        case 256: return gemm_tn<1, 256, AMN, BMN, EPI>(A, B, K, a, p, stream);
        case 128: return gemm_tn<1, 128, AMN, BMN, EPI>(A, B, K, a, p, stream);
        default: return gemm_tn<1, 64, AMN, BMN, EPI>(A, B, K, a, p, stream);
    }
}

// ------------------------------------------------------------------ the head's log probabilities

constexpr int LM_NT = 256;
// One CTA per row: the column tiles' states into the row's outputs, and the logits of the last `rest` tiles where those
// were split along k (at most 128 rows): their chunks added in k order, then the columns' states like any other.
__global__ void __launch_bounds__(LM_NT) lmhead_merge_kernel(const float4* part, int states, int stride, const float* partial,
                                                             int rest, int split, int tn, int rows, const float* token_value,
                                                             const int64_t* tokens, int V, float c, float* logprob,
                                                             float* entropy, float4* stats, uint32_t* status) {
    pdl_wait_then_release();
    __shared__ LpState sw[LM_NT / 32];
    __shared__ float tv;
    const int r = blockIdx.x, tid = threadIdx.x;
    const int64_t tok = tokens[r];
    const bool has = tok >= 0 && tok < V;
    const int n0 = split > 1 ? (states / 2) * tn : V;  // first column of the split tiles
    LpState s;
    s.m = f_ninf();
    s.S = s.U = 0.0f;
    if (tid == 0 && has && tok < n0) tv = token_value[r];
    const int64_t step = (int64_t)rest * rows * tn;
    for (int n = n0 + tid; n < V; n += LM_NT) {
        const int i = n - n0;
        const float* p = partial + ((int64_t)(i / tn) * rows + r) * tn + i % tn;
        float x = 0.0f;
#pragma unroll 8
        for (int k = 0; k < split; ++k) x += p[k * step];
        if (n == tok) tv = x;
        const float one[1] = {x};
        lp_add_any<1>(s, one, c);
    }
    for (int i = tid; i < states; i += LM_NT) {
        const float4 p = part[(int64_t)r * stride + i];
        LpState o;
        o.m = p.x;
        o.S = p.y;
        o.U = p.z;
        s = lp_merge(s, o, c);
    }
    lp_warp_merge(s, c);
    if ((tid & 31) == 0) sw[tid >> 5] = s;
    __syncthreads();
    if (tid < 32) {
        s.m = f_ninf();
        s.S = s.U = 0.0f;
        if (tid < LM_NT / 32) s = sw[tid];
        lp_warp_merge(s, c);
        if (tid == 0) {
            const LpFinal f = lp_final(s, c);
            if (logprob) logprob[r] = has ? lp_value(tv, f, c) : 0.0f;
            if (entropy) entropy[r] = f.entropy;
            if (stats) stats[r] = make_float4(f.m, f.R, f.log2S, f.entropy);
            if (status && tok >= V) atomicOr(status, B2S_STATUS_TOKEN_RANGE);
        }
    }
}

// ------------------------------------------------------------------ the projection of few rows

// out = act(x w^T + bias) + residual for at most R rows: a CTA of 4 warps per F output features, which deal the k between
// them 8 at a time, every lane 16-byte loads of the weight (read once, past L1) and of the rows (from L1), fp32 sums joined
// by shuffles and through shared memory.  Bound by the weight's read: the tensor cores' path needs a split along k, two
// launches and 128-row tiles for the same bytes.
constexpr int ROWS_NT = 128;
template <int R, int F>
__global__ void __launch_bounds__(ROWS_NT) linear_rows_kernel(const __grid_constant__ GemmArgs a, const void* x,
                                                              int64_t x_stride, const void* w, int64_t w_stride, int K) {
    __shared__ float red[ROWS_NT / 32][R * F];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n0 = (int)blockIdx.x * F;
    pdl_wait_then_release();
    const uint4* wp[F];
    const uint4* xp[R];
#pragma unroll
    for (int f = 0; f < F; ++f)  // rows and features past the end repeat the last one; they are not stored
        wp[f] = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(w) + (int64_t)min(n0 + f, a.N - 1) * w_stride);
#pragma unroll
    for (int r = 0; r < R; ++r)
        xp[r] = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(x) + (int64_t)min(r, a.M - 1) * x_stride);
    float2 acc[R][F];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int f = 0; f < F; ++f) acc[r][f] = make_float2(0.0f, 0.0f);
    auto wide = [](uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); };
#pragma unroll 4
    for (int v = tid; v < K / 8; v += ROWS_NT) {
        uint4 q[F];
#pragma unroll
        for (int f = 0; f < F; ++f) q[f] = ldg_stream(wp[f] + v);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint4 u = __ldg(xp[r] + v);
            const float2 x0 = wide(u.x), x1 = wide(u.y), x2 = wide(u.z), x3 = wide(u.w);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                acc[r][f] = __ffma2_rn(x0, wide(q[f].x), acc[r][f]);
                acc[r][f] = __ffma2_rn(x1, wide(q[f].y), acc[r][f]);
                acc[r][f] = __ffma2_rn(x2, wide(q[f].z), acc[r][f]);
                acc[r][f] = __ffma2_rn(x3, wide(q[f].w), acc[r][f]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int f = 0; f < F; ++f) {
            float t = acc[r][f].x + acc[r][f].y;
#pragma unroll
            for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) red[warp][r * F + f] = t;
        }
    __syncthreads();
    if (tid < R * F) {
        const int r = tid / F, n = n0 + tid % F;
        if (r < a.M && n < a.N) {
            float t = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
            if (a.bias) t += bf16_bits_to_f(__ldg(static_cast<const unsigned short*>(a.bias) + n));
            if (a.preact) static_cast<unsigned short*>(a.preact)[(int64_t)r * a.pre_stride + n] = preact_bits(t);
            t = act_apply(t, a.act);
            if (a.residual) t += bf16_bits_to_f(__ldg(static_cast<const unsigned short*>(a.residual) + (int64_t)r * a.res_stride + n));
            static_cast<__nv_bfloat16*>(a.out)[(int64_t)r * a.out_stride + n] = __float2bfloat16_rn(t);
        }
    }
}
// Which projections take it.  Against the tensor cores' path (us): 1 x 768 x 4096 3.5 : 11.1, 1 x 4096 x 4096 7.7 : 13.0,
// 4 x 4096 x 4096 12.2 : 13.0, 8 x 768 x 4096 5.5 : 11.5, but 8 x 4096 x 4096 20.9 : 13.8 and 8 x 6562 x 768 14.2 : 10.2 (the
// rows are read from L1 and unpacked once per two features).
bool few_rows(int rows, int N, int64_t K) {
    return rows <= 2 || (rows <= 4 && N * K <= 1 << 24) || (rows <= 8 && N <= 2048 && N * K <= 1 << 22);
}
cudaError_t linear_rows(const GemmArgs& a, const void* x, int64_t xs, const void* w, int64_t ws, int K, void* stream) {
    auto go = [&](auto kernel, int F) {
        return launch_pdl(kernel, dim3((unsigned)((a.N + F - 1) / F)), ROWS_NT, 0, stream, a, x, xs, w, ws, K);
    };
    if (a.M == 1) return go(linear_rows_kernel<1, 1>, 1);
    if (a.M == 2) return go(linear_rows_kernel<2, 1>, 1);
    if (a.M <= 4) return go(linear_rows_kernel<4, 2>, 2);
    return go(linear_rows_kernel<8, 2>, 2);
}

// ------------------------------------------------------------------ the projection's elementwise gradient

// dz = dy act'(z) (bf16, rows dz_stride apart) and the sums of its columns over this CTA's rows, 8 columns of a row per
// thread (z's and dz's rows are padded to that).  VEC: dy's rows are 16-byte aligned; else a row starts on a whole word or
// half a word off, and a thread's 8 values are four words, or two halves and the three words between them.  32 threads
// cover 256 columns, the 8 warps take rows in turn; the sums (fp32, of the unrounded dz) go to part[blockIdx.y][n], or,
// with one part, straight to the bias gradient.
constexpr int DZ_NT = 256;
template <bool VEC, int ACT>
__global__ void __launch_bounds__(DZ_NT) linear_dz_kernel(const void* dy, int64_t dy_stride, const void* z,
                                                          int64_t z_stride, int rows, int N, int rows_per,
                                                          void* dz, int64_t dz_stride, float* part, void* db) {
    constexpr int E = 8;
    pdl_wait_then_release();
    __shared__ float red[8][32][E + 1];
    const int cg = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int n = (blockIdx.x * 32 + cg) * E;
    const int r0 = blockIdx.y * rows_per, r1 = min(rows, r0 + rows_per);
    float sum[E] = {};
    if (n < N) {
#pragma unroll 4
        for (int r = r0 + rl; r < r1; r += 8) {
            const unsigned short* gp = static_cast<const unsigned short*>(dy) + (int64_t)r * dy_stride + n;
            const unsigned short* zp = static_cast<const unsigned short*>(z) + (int64_t)r * z_stride + n;
            float g[E], x[E];
            if (VEC || n + E > N) {
                load8(gp, 0, N - n, VEC, g);
            } else {
                const bool half = reinterpret_cast<uintptr_t>(gp) & 2;
                const uint32_t* mid = reinterpret_cast<const uint32_t*>(gp + (half ? 1 : 0));
                uint32_t w[4] = {__ldg(mid), __ldg(mid + 1), __ldg(mid + 2), 0u};
                if (half) {
                    const uint32_t lo = __ldg(gp), hi = __ldg(gp + 7);
                    w[3] = w[2] >> 16 | hi << 16;
                    w[2] = __funnelshift_l(w[1], w[2], 16);
                    w[1] = __funnelshift_l(w[0], w[1], 16);
                    w[0] = lo | w[0] << 16;
                } else {
                    w[3] = __ldg(mid + 3);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    g[2 * j] = __uint_as_float(w[j] << 16);
                    g[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                }
            }
            if constexpr (ACT != ACT_NONE) {
                const uint4 q = __ldg(reinterpret_cast<const uint4*>(zp));
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < E; ++j) x[j] = preact_value((unsigned short)(w[j >> 1] >> (16 * (j & 1))));
#pragma unroll
                for (int j = 0; j < E; ++j) g[j] *= n + j < N ? act_slope<ACT>(x[j]) : 0.0f;
            }
            if (dz) store8(static_cast<unsigned short*>(dz) + (int64_t)r * dz_stride + n, 0, N - n, true, g);
#pragma unroll
            for (int j = 0; j < E; ++j) sum[j] += g[j];
        }
    }
    if (!part && !db) return;
#pragma unroll
    for (int j = 0; j < E; ++j) red[rl][cg][j] = sum[j];
    __syncthreads();
    const int i = threadIdx.x, c = i / E, j = i % E;  // one column per thread
    const int col = blockIdx.x * 32 * E + i;
    if (i >= 32 * E || col >= N) return;
    float s = red[0][c][j];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][c][j];
    if (part) part[(int64_t)blockIdx.y * N + col] = s;
    else static_cast<__nv_bfloat16*>(db)[col] = __float2bfloat16_rn(s);
}
// db = the sums of the parts' sums, each of 8 warps taking an eighth of the parts of 32 columns.
__global__ void __launch_bounds__(DZ_NT) linear_db_kernel(const float* part, int parts, int N, void* db) {
    pdl_wait_then_release();
    __shared__ float red[8][32];
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
    float s = 0.0f;
    if (n < N) {
#pragma unroll 8
        for (int p = w; p < parts; p += 8) s += part[(int64_t)p * N + n];
    }
    red[w][c] = s;
    __syncthreads();
    if (w || n >= N) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][c];
    static_cast<__nv_bfloat16*>(db)[n] = __float2bfloat16_rn(s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
// parts of the rows whose column sums are taken separately: one round of CTAs (four an SM), at least 32 rows each
int dz_parts(int rows, int N) {
    const int64_t cols = (N + 255) / 256;
    int64_t p = 4 * sms_here() / cols;
    if (p > (rows + 31) / 32) p = (rows + 31) / 32;
    return (int)(p < 1 ? 1 : p);
}

int check_head(const void* hidden, int64_t hstride, const void* head, int64_t wstride, int H, int V, int rows,
               float temperature) {
    if (rows < 0 || V < 1 || H < 8 || H % 8 || hstride < H || hstride % 8 || wstride < H || wstride % 8)
        return B2S_ERR_INVALID;
    if (!lp_temperature_ok(temperature)) return B2S_ERR_INVALID;
    if (rows > LP_MAX_SIZE || V > LP_MAX_SIZE || H > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
    if (rows && (!hidden || !head || !aligned16(hidden) || !aligned16(head))) return B2S_ERR_INVALID;
    return B2S_OK;
}

}  // namespace
}  // namespace b2s

extern "C" {

int b2s_lmhead_logprobs_workspace(int32_t rows, int32_t vocab, int32_t hidden_dim, int64_t* bytes) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || hidden_dim < 8 || !bytes) return B2S_ERR_INVALID;
    const Plan p = plan_here(rows > 0 ? rows : 1, vocab, hidden_dim, EPI_LSE);
    *bytes = up((int64_t)rows * ((vocab + p.tn - 1) / p.tn) * 32 + (int64_t)rows * 4, 256) + p.bytes;
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
    const Plan p = plan_here(h->rows, h->vocab, h->hidden_dim, EPI_LSE);
    const int tiles = (h->vocab + p.tn - 1) / p.tn, whole = p.split > 1 ? tiles - p.rest : tiles;
    GemmArgs a;
    memset(&a, 0, sizeof(a));
    a.M = h->rows;
    a.N = h->vocab;
    a.status = h->status;
    a.c = lp_scale(h->temperature);
    a.tokens = h->tokens;
    a.part = static_cast<float4*>(h->workspace);  // two states a row and column tile
    a.token_value = reinterpret_cast<float*>(a.part + (int64_t)h->rows * tiles * 2);
    a.partial = reinterpret_cast<float*>(static_cast<unsigned char*>(h->workspace) +
                                         up((int64_t)h->rows * tiles * 32 + (int64_t)h->rows * 4, 256));
    rc = gemm<false, false, EPI_LSE>({h->hidden, h->hidden_row_stride}, {h->head, h->head_row_stride}, h->hidden_dim, a,
                                     stream);
    if (rc != B2S_OK) return rc;
    const cudaError_t e = launch_pdl(lmhead_merge_kernel, dim3((unsigned)h->rows), LM_NT, 0, stream,
                                     (const float4*)a.part, 2 * whole, 2 * tiles, (const float*)a.partial, p.rest, p.split,
                                     p.tn, (int)h->rows, (const float*)a.token_value, h->tokens, (int)h->vocab, a.c, logprob,
                                     entropy, reinterpret_cast<float4*>(stats), h->status);
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

int b2s_lmhead_logprobs_grad_workspace(int32_t rows, int32_t vocab, int32_t hidden_dim, int64_t* bytes) {
    using namespace b2s;
    if (rows < 0 || vocab < 1 || hidden_dim < 8 || !bytes) return B2S_ERR_INVALID;
    const int64_t r = rows > 0 ? rows : 1;
    const int64_t dh = plan_here((int)r, hidden_dim, vocab, EPI_STORE).bytes, dw = plan_here(vocab, hidden_dim, r, EPI_STORE).bytes;
    *bytes = up(r * up(vocab, 8) * 2, 256) + up(dh > dw ? dh : dw, 256);
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
    b.partial = reinterpret_cast<float*>(static_cast<unsigned char*>(h->workspace) + up((int64_t)h->rows * ldz * 2, 256));
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
    using namespace b2s;
    if (rows < 0 || in_features < 8 || out_features < 1 || !bytes) return B2S_ERR_INVALID;
    *bytes = rows && !few_rows(rows, out_features, in_features) ? plan_here(rows, out_features, in_features, EPI_LINEAR).bytes : 0;
    return B2S_OK;
}

int b2s_linear(const b2s_linear_args* l, void* stream) {
    using namespace b2s;
    if (!l || l->rows < 0 || l->out_features < 1 || l->in_features < 8 || l->in_features % 8 || l->activation < 0 ||
        l->activation > B2S_ACT_SILU)
        return B2S_ERR_INVALID;
    if (l->rows > LP_MAX_SIZE || l->in_features > LP_MAX_SIZE || l->out_features > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
    if (l->rows == 0) return B2S_OK;
    if (!l->x || !l->weight || !l->out || !aligned16(l->x) || !aligned16(l->weight) || l->x_row_stride < l->in_features ||
        l->x_row_stride % 8 || l->weight_row_stride < l->in_features || l->weight_row_stride % 8 ||
        l->out_row_stride < l->out_features || (l->bias && !aligned16(l->bias)) ||
        (l->residual && l->residual_row_stride < l->out_features) ||
        (l->preact && (!aligned16(l->preact) || l->preact_row_stride < l->out_features || l->preact_row_stride % 8)) ||
        ((reinterpret_cast<uintptr_t>(l->out) | reinterpret_cast<uintptr_t>(l->residual)) & 1))
        return B2S_ERR_INVALID;
    int64_t need = 0;
    b2s_linear_workspace(l->rows, l->in_features, l->out_features, &need);
    if (need && (!l->workspace || l->workspace_bytes < need || !aligned16(l->workspace))) return B2S_ERR_INVALID;
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
    a.partial = static_cast<float*>(l->workspace);
    if (few_rows(l->rows, l->out_features, l->in_features)) {
        const cudaError_t e = linear_rows(a, l->x, l->x_row_stride, l->weight, l->weight_row_stride, l->in_features, stream);
        return e == cudaSuccess ? B2S_OK : cuda_fail(e);
    }
    return gemm<false, false, EPI_LINEAR>({l->x, l->x_row_stride}, {l->weight, l->weight_row_stride}, l->in_features, a,
                                          stream);
}

int b2s_linear_grad_workspace(int32_t rows, int32_t in_features, int32_t out_features, int64_t* bytes) {
    using namespace b2s;
    if (rows < 0 || in_features < 8 || out_features < 1 || !bytes) return B2S_ERR_INVALID;
    const int64_t r = rows > 0 ? rows : 1;
    const int64_t dx = plan_here((int)r, in_features, out_features, EPI_STORE).bytes;
    const int64_t dw = plan_here(out_features, in_features, r, EPI_STORE).bytes;
    *bytes = up(r * up(out_features, 8) * 2, 256) + up((int64_t)dz_parts((int)r, out_features) * out_features * 4, 256) +
             up(dx > dw ? dx : dw, 256);
    return B2S_OK;
}

int b2s_linear_grad(const b2s_linear_grad_args* l, void* stream) {
    using namespace b2s;
    if (!l || l->rows < 0 || l->out_features < 1 || l->in_features < 8 || l->in_features % 8 || l->activation < 0 ||
        l->activation > B2S_ACT_SILU || (l->grad_weight && !aligned16(l->grad_weight)))
        return B2S_ERR_INVALID;
    if (l->rows > LP_MAX_SIZE || l->in_features > LP_MAX_SIZE || l->out_features > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
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
    const int parts = dz_parts(l->rows, l->out_features);
    float* part = reinterpret_cast<float*>(static_cast<unsigned char*>(l->workspace) + up((int64_t)l->rows * ldz * 2, 256));
    if (direct) dz = {l->grad_out, l->grad_out_row_stride};
    if ((products && !direct) || l->grad_bias) {
        const int per = (l->rows + parts - 1) / parts;
        const bool two = l->grad_bias && parts > 1;
        static constexpr decltype(&linear_dz_kernel<true, ACT_NONE>) kernels[2][4] = {
            {linear_dz_kernel<false, ACT_NONE>, linear_dz_kernel<false, ACT_RELU>, linear_dz_kernel<false, ACT_GELU>,
             linear_dz_kernel<false, ACT_SILU>},
            {linear_dz_kernel<true, ACT_NONE>, linear_dz_kernel<true, ACT_RELU>, linear_dz_kernel<true, ACT_GELU>,
             linear_dz_kernel<true, ACT_SILU>}};
        cudaError_t e = launch_pdl(kernels[dy_vec][l->activation],
                                   dim3((unsigned)((l->out_features + 255) / 256), (unsigned)parts), DZ_NT, 0,
                                   stream, l->grad_out, l->grad_out_row_stride, l->preact, l->preact_row_stride,
                                   (int)l->rows, (int)l->out_features, per,
                                   products && !direct ? l->workspace : nullptr, ldz, two ? part : nullptr,
                                   two ? nullptr : l->grad_bias);
        if (e == cudaSuccess && two)
            e = launch_pdl(linear_db_kernel, dim3((unsigned)((l->out_features + 31) / 32)), DZ_NT, 0, stream,
                           (const float*)part, parts, (int)l->out_features, l->grad_bias);
        if (e != cudaSuccess) return cuda_fail(e);
    }
    GemmArgs b;
    memset(&b, 0, sizeof(b));
    b.status = l->status;
    b.out_vec = 1;
    b.N = l->in_features;
    b.out_stride = l->in_features;
    b.partial = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(part) +
                                         up((int64_t)parts * l->out_features * 4, 256));
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
