// The product of microscaled 4-bit operands on the tensor cores (sm_100a): D[m, n] = sum_k A[m, k] B[n, k] with
// tcgen05.mma kind::mxf4, whose blocks of 32 k carry their scales into the multiplication, at four times bf16's rate; fp32
// accumulation in tensor memory; bias, activation and residual in the epilogue.
//
// The shape is b2s_gemm.cuh's: persistent CTAs or pairs of them, a TMA ring (a stage of 256 k holds the 128 bytes a row that 64 k
// are in bf16), a loading and an issuing warp, tiles that do not fill a round split along k and joined by a second kernel.
// What is different:
// * A stage brings 1 KB of scales for each 128 rows, as the matrix's scale tiles lie, and the issuing warp has the tensor cores
//   copy them to tensor memory (tcgen05.cp: 512 bytes to 32 lanes x 4 columns, the same in all four lane quarters).  Each
//   stage of the ring has its own columns there: when a stage is full again, the MMAs that read its scales are done.
// * Two accumulators of 256 columns leave no room for scales beside them, so they share 128 columns: the epilogue takes those to
//   registers first and lets the next tile's MMAs begin, then the other 128 from where they lie.  (Taken whole, 128 columns a
//   thread, the registers spilled to a first-level cache that the ring leaves nothing of: 1000 x 4096 x 151936 993 us against
//   254 with shared columns.)
// * Sixteen epilogue warps instead of eight: the MMAs are four times as fast, the epilogue is what is left (8192 x 4096 x 4096
//   with gelu 105 against 84 us).
// A large product is bound by the way from L2 to the SMs: a pair's stage asks for 70 KB in 530 clocks, 66 bytes a clock and SM,
// and the output's way out comes on top (1000 x 4096 x 151936: 5.0 PFLOP/s; 5.7 without the epilogue, 6.6 without loads too).
#include <string.h>

#include <atomic>

#include "../../include/b2s_sampler.h"
#include "b2s_gemm.cuh"
#include "b2s_launch.cuh"
#include "b2s_mx.cuh"

namespace b2s {

int cuda_fail(cudaError_t e);
int tensor_map_2d(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int64_t outer_stride, int box_inner,
                  int box_outer);
int tensor_map_words(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int box_inner, int box_outer);

namespace {

constexpr int MXG_KB = 256;  // k per stage: one 128-byte row of the swizzle
constexpr int MXG_EPI = 16;  // epilogue warps: warp w has tensor-memory quarter w % 4 and part w / 4 of the columns
constexpr int MXG_THREADS = 32 * MXG_EPI + 64;
constexpr uint32_t MXG_STAGING = MXG_EPI * 2048;  // per epilogue warp: 32 rows of 32 bf16, or of 16 fp32
constexpr int MXG_PARTS = 4;  // of 32 columns, and again 32 of 256
__host__ __device__ constexpr int mxg_btiles(int tn) { return tn / 128; }  // scale tiles of B
// A stage of one CTA: 128 rows of A, its share of B, A's scales (1 KB) and all of the tile's B's.
__host__ __device__ constexpr uint32_t mxg_stage_bytes(int cg, int tn) {
    return GM_A_BYTES + (uint32_t)(tn / cg) * 128 + 1024 + 1024 * mxg_btiles(tn);
}
__host__ __device__ constexpr int mxg_stages(int cg, int tn) {
    return (int)(184u * 1024u / mxg_stage_bytes(cg, tn)) > 7 ? 7 : (int)(184u * 1024u / mxg_stage_bytes(cg, tn));
}
__host__ __device__ constexpr uint32_t mxg_smem(int cg, int tn) {
    return 1024 + mxg_stages(cg, tn) * mxg_stage_bytes(cg, tn) + MXG_STAGING + 256;
}
// Tensor memory: two accumulators, then each stage's scales: for each half of 128 k 4 columns of A's and 4 per tile of B's.
// Two times 256 columns of accumulator would leave none for the scales, so those share their middle: the second starts at
// column 128.
__host__ __device__ constexpr int mxg_acc_step(int tn) { return tn == 256 ? 128 : tn; }
__host__ __device__ constexpr int mxg_acc_cols(int tn) { return mxg_acc_step(tn) + tn; }
__host__ __device__ constexpr int mxg_free(int tn) { return tn == 256 ? 1 : 2; }  // accumulators handed back apart
__host__ __device__ constexpr int mxg_sf_cols(int tn) { return 8 + 8 * mxg_btiles(tn); }
constexpr uint32_t MXG_TMEM = 512;
static_assert(mxg_acc_cols(128) + mxg_stages(1, 128) * mxg_sf_cols(128) <= (int)MXG_TMEM &&
                  mxg_acc_cols(256) + mxg_stages(2, 256) * mxg_sf_cols(256) <= (int)MXG_TMEM,
              "accumulators and scales fit tensor memory");

// Shared-memory descriptor of 512 bytes of scales: 32 rows of 16 bytes, 8 rows at a time (128 bytes), no swizzle.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// To 4 columns of tensor memory, the same in each quarter of the lanes (of both CTAs, each from its own shared memory).
template <int CG>
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int CG>
__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
}

// An arrival on the first CTA's mbarrier that orders nothing but this CTA's: what it tells of, tensor memory read, is ordered by
// the tcgen05 fences.  (With the cluster's scope it waits for the warp's stores of the tile before: 1100 clocks a tile.)
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ------------------------------------------------------------------ the epilogue's blocks of 32 rows x 32 columns
// b2s_gemm.cuh's, but for twice as many warps: 64-byte rows of staging, two blocks' worth of which a 5th stage of the ring
// takes, the bias from broadcast loads and packed arithmetic.

// 16-byte chunk j of row r: conflict-free for a lane per row, and for 4 lanes a row.
__device__ __forceinline__ uint4* row_at(unsigned char* st, int r, int j) {
    return reinterpret_cast<uint4*>(st + r * 64 + ((j ^ ((r >> 1) & 3)) << 4));
}
// Pairs of 16-bit values, 32 of this lane's row, to global memory: rows `stride` elements apart.
__device__ __forceinline__ void put_rows(unsigned char* st, const uint32_t (&w)[16], unsigned short* out, int64_t stride, int rows,
                                         int cols, bool vec) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j) *row_at(st, lane, j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    __syncwarp();
    if (vec) {
        const int r = lane >> 2, c = lane & 3;
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *row_at(st, 8 * i + r, c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (8 * i + r < rows) *reinterpret_cast<uint4*>(out + (8 * i + r) * stride + 8 * c) = v[i];
    } else if (lane < cols) {
        out += lane;
#pragma unroll 1
        for (int r = 0; r < 32; r += 8) {
            unsigned short v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[k] = reinterpret_cast<const unsigned short*>(row_at(st, r + k, lane >> 3))[lane & 7];
#pragma unroll
            for (int k = 0; k < 8; ++k, out += stride)
                if (r + k < rows) *out = v[k];
        }
    }
    __syncwarp();
}
// A block of the residual into registers, in flight until it is wanted, and its row for this lane.
__device__ __forceinline__ void fetch_rows(const GemmArgs& a, uint32_t (&q)[16], int row0, int n) {
    if (!a.residual || n >= a.N) return;
    const int lane = threadIdx.x & 31, rows = a.M - row0, left = a.N - n;
    const unsigned short* p = static_cast<const unsigned short*>(a.residual) + (int64_t)row0 * a.res_stride + n;
    if (vec_block(a, n, a.res_vec)) {
        const int r = lane >> 2, c = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (8 * i + r < rows) u = __ldg(reinterpret_cast<const uint4*>(p + (8 * i + r) * a.res_stride + 8 * c));
            q[4 * i] = u.x;
            q[4 * i + 1] = u.y;
            q[4 * i + 2] = u.z;
            q[4 * i + 3] = u.w;
        }
    } else {
        const int w = 2 * (lane & 15);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = 2 * i + (lane >> 4);
            const unsigned short* g = p + r * a.res_stride + w;
            const uint32_t lo = r < rows && w < left ? __ldg(g) : 0, hi = r < rows && w + 1 < left ? __ldg(g + 1) : 0;
            q[i] = lo | hi << 16;
        }
    }
}
__device__ __forceinline__ void turn_rows(unsigned char* st, uint32_t (&q)[16], bool vec) {
    const int lane = threadIdx.x & 31;
    if (vec) {
        const int r = lane >> 2, c = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) *row_at(st, 8 * i + r, c) = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
    } else {
        const int w = lane & 15;
#pragma unroll
        for (int i = 0; i < 16; ++i) reinterpret_cast<uint32_t*>(row_at(st, 2 * i + (lane >> 4), w >> 2))[w & 3] = q[i];
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint4 u = *row_at(st, lane, j);
        q[4 * j] = u.x;
        q[4 * j + 1] = u.y;
        q[4 * j + 2] = u.z;
        q[4 * j + 3] = u.w;
    }
    __syncwarp();
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// The activations of pairs, act_apply's in packed arithmetic, in as few operations as they take: with gelu, bias and residual the
// epilogue's instructions are what a tile of 4096 k waits for.  gelu(z) = max(z, 0) - |z| q with act_apply's tail q = 1 - Phi(|z|)
// (its polynomial halved); silu as there, e^z by halves.
template <int ACT>
__device__ __forceinline__ float2 act_pair(float2 z) {
    // finite, so that infinity times the tail's zero is no NaN; NaN comes through z itself
    const float2 m = make_float2(fminf(fabsf(z.x), ACT_FAR), fminf(fabsf(z.y), ACT_FAR));
    if (ACT == ACT_RELU) return make_float2(fmax_nan(z.x, 0.0f), fmax_nan(z.y, 0.0f));
    if (ACT == ACT_GELU) {
        const float2 d = __ffma2_rn(both(GELU_T), m, both(1.0f)), t = make_float2(rcp(d.x), rcp(d.y));
        const float2 x = __fmul2_rn(__fmul2_rn(both(GELU_E), m), m);
        const float2 q = __fmul2_rn(__fmul2_rn(gelu_poly(t, 0.5f), t), make_float2(ex2(x.x), ex2(x.y)));
        return __ffma2_rn(make_float2(-m.x, -m.y), q, make_float2(fmax_nan(z.x, 0.0f), fmax_nan(z.y, 0.0f)));
    }
    if (ACT == ACT_SILU) {
        z = make_float2(fmax_nan(z.x, -ACT_FAR), fmax_nan(z.y, -ACT_FAR));
        const float2 x = __fmul2_rn(both(-0.72134752044448170f), m), h = make_float2(ex2(x.x), ex2(x.y));
        const float2 w = __fmul2_rn(__fmul2_rn(z, h), h), d = __ffma2_rn(h, h, both(1.0f));
        return __fmul2_rn(make_float2(z.x < 0.0f ? w.x : z.x, z.y < 0.0f ? w.y : z.y), make_float2(rcp(d.x), rcp(d.y)));
    }
    return z;
}
template <int ACT>
__device__ __forceinline__ void act_row(float2 (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = act_pair<ACT>(v[j]);
}
__device__ __forceinline__ float2 wide2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// This lane's row of 32 accumulated columns from n through the epilogue and to the output; rq: the residual's block.
__device__ __forceinline__ void finish_block(const GemmArgs& a, const float (&acc)[32], uint32_t (&rq)[16], int row0, int n,
                                             unsigned char* st) {
    const int lane = threadIdx.x & 31, rows = a.M - row0, cols = a.N - n;
    const unsigned short* bias = static_cast<const unsigned short*>(a.bias);
    float2 v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = make_float2(acc[2 * j], acc[2 * j + 1]);
    if (bias) {
        if (cols >= 32 && (reinterpret_cast<uintptr_t>(bias) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(bias + n) + j);
                v[4 * j] = __fadd2_rn(v[4 * j], wide2(u.x));
                v[4 * j + 1] = __fadd2_rn(v[4 * j + 1], wide2(u.y));
                v[4 * j + 2] = __fadd2_rn(v[4 * j + 2], wide2(u.z));
                v[4 * j + 3] = __fadd2_rn(v[4 * j + 3], wide2(u.w));
            }
        } else {
            const float b = lane < cols ? bf16_bits_to_f(__ldg(bias + n + lane)) : 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                v[j] = __fadd2_rn(v[j], make_float2(__shfl_sync(0xffffffffu, b, 2 * j), __shfl_sync(0xffffffffu, b, 2 * j + 1)));
        }
    }
    uint32_t w[16];
    if (a.preact) {
        // as preact_bits, whose smallest positive value is asked for by the rectifier's slope alone
        if (a.act == ACT_RELU) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = (uint32_t)preact_bits(v[j].x) | (uint32_t)preact_bits(v[j].y) << 16;
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const __half2 h = __floats2half2_rn(v[j].x, v[j].y);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        put_rows(st, w, static_cast<unsigned short*>(a.preact) + (int64_t)row0 * a.pre_stride + n, a.pre_stride, rows, cols,
                 vec_block(a, n, 1));
    }
    if (a.act == ACT_RELU) act_row<ACT_RELU>(v);
    else if (a.act == ACT_GELU) act_row<ACT_GELU>(v);
    else if (a.act == ACT_SILU) act_row<ACT_SILU>(v);
    if (a.residual) {
        turn_rows(st, rq, vec_block(a, n, a.res_vec));
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = __fadd2_rn(v[j], wide2(rq[j]));
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = pack_bf16(v[j].x, v[j].y);  // the output's one rounding
    put_rows(st, w, static_cast<unsigned short*>(a.out) + (int64_t)row0 * a.out_stride + n, a.out_stride, rows, cols,
             vec_block(a, n, a.out_vec));
}
// A chunk of a split tile: 32 columns of its fp32 sums as they are, 16 at a time.
template <int TM, int TN>
__device__ __forceinline__ void keep_sums(const GemmArgs& a, const float (&v)[32], int row0, int n, int nt, int slot, unsigned char* st) {
    const int lane = threadIdx.x & 31, rows = a.M - row0, r = lane >> 2, c = lane & 3;
    float* dst = a.partial + ((int64_t)slot * min(a.M, TM) + row0 % TM) * TN + n - nt * TN + 4 * c;
#pragma unroll
    for (int h = 0; h < 32; h += 16, dst += 16) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4*>(row_at(st, lane, j)) = make_float4(v[h + 4 * j], v[h + 4 * j + 1], v[h + 4 * j + 2], v[h + 4 * j + 3]);
        __syncwarp();
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = *row_at(st, 8 * i + r, c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (8 * i + r < rows) *reinterpret_cast<uint4*>(dst + (int64_t)(8 * i + r) * TN) = u[i];
        __syncwarp();
    }
}

template <int CG, int TN>
__global__ void __launch_bounds__(MXG_THREADS, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap atail,
                   const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap btail,
                   const __grid_constant__ CUtensorMap asmap, const __grid_constant__ CUtensorMap bsmap,
                   const __grid_constant__ GemmArgs a) {
    constexpr int TM = CG * GM_M, BN = TN / CG, ST = mxg_stages(CG, TN), BT = mxg_btiles(TN), ACCS = mxg_free(TN);
    constexpr uint32_t STAGE = mxg_stage_bytes(CG, TN), SFA = GM_A_BYTES + BN * 128, SFB = SFA + 1024;
    constexpr uint32_t SF0 = mxg_acc_cols(TN), SFC = mxg_sf_cols(TN);  // the scales' first column, columns a stage
    // E2M1 operands (bits 7-9, 10-11 = 1), both K-major, N >> 3 at bit 17, E8M0 scales (bit 23), M >> 4 at bit 24; which two
    // of a column's four scales A and B take at bits 29 and 4
    constexpr uint32_t IDESC = (1u << 7) | (1u << 10) | ((uint32_t)(TN >> 3) << 17) | (1u << 23) | ((uint32_t)(TM >> 4) << 24);
    extern __shared__ __align__(128) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
    const uint32_t base_u = smem_u32(smem_raw);
    unsigned char* sm = smem_raw + (((base_u + 1023u) & ~1023u) - base_u);
    unsigned char* staging = sm + ST * STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + MXG_STAGING);  // the first CTA's serves both
    uint64_t* empty = full + ST;
    uint64_t* tfull = empty + ST;      // [ACCS] an accumulator is complete
    uint64_t* tempty = tfull + ACCS;   // [ACCS] an accumulator has been read (the first CTA's, by both)
    uint64_t* drain = tempty + ACCS;   // every MMA issued has completed (only after a failure)
    uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tslot + 1);
    volatile int* issued = fail + 1;    // stage loads issued
    volatile int* consumed = fail + 2;  // stage loads seen to land

    if (tid == 0) {
        prefetch_tensormap(&amap);
        prefetch_tensormap(&bmap);
        prefetch_tensormap(&atail);
        prefetch_tensormap(&btail);
        prefetch_tensormap(&asmap);
        prefetch_tensormap(&bsmap);
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < ACCS; ++s) {
            mbar_init(&tfull[s], 1);
            mbar_init(&tempty[s], 4 * MXG_PARTS * CG);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
        *fail = 0;
        *issued = 0;
        *consumed = 0;
    }
    if (warp == MXG_EPI + 1) {
        if constexpr (CG == 2) tmem_alloc_pair(tslot, MXG_TMEM);
        else tmem_alloc(tslot, MXG_TMEM);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) {  // the partner's mbarriers exist before anything signals them
        cluster_arrive_release();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem = *tslot;
    if (warp != MXG_EPI) pdl_wait_then_release();

    if (warp == MXG_EPI) {
        int s = 0, it = 0;
        uint32_t ph = 1;  // parity of `empty`'s last phase: the first round finds every stage free
        bool ok = a.wait > 0;
        const uint32_t bar0 = CG == 2 ? mapa_shared(smem_u32(full), 0) : smem_u32(full);
        auto load = [&](int stage, uint32_t to, const CUtensorMap* map, int x, int y) {
            unsigned char* dst = sm + stage * STAGE + to;
            if constexpr (CG == 2) tma_load_2d_pair(dst, map, x, y, bar0 + 8u * stage);
            else tma_load_2d(dst, map, x, y, &full[stage]);
        };
        // A CTA's parts of a tile's operands, the rows that are there (by a map of the last part's height, rounded up to 8): rows
        // past the end cost a load as much as others (a tile of 16 rows that loads 128 takes 16 x 4096 x 151936 from 69 to 78
        // us).  What is not loaded is left as it was and not stored.
        const CUtensorMap *ma, *mb;  // null: no rows
        int m0, n0, nt;
        uint32_t bytes;
        auto tile = [&](int64_t t) {
            auto held = [](int first, int part, int end) { return end - first >= part ? part : end > first ? (end - first + 7) / 8 * 8 : 0; };
            int mt;
            tile_of<TM>(a, t, &mt, &nt);
            m0 = mt * TM + (int)rank * GM_M;
            n0 = nt * TN + (int)rank * BN;
            const int ra = held(m0, GM_M, a.M), rb = held(n0, BN, a.N);
            ma = ra == GM_M ? &amap : ra ? &atail : nullptr;
            mb = rb == BN ? &bmap : rb ? &btail : nullptr;
            bytes = CG * (STAGE - SFA) + 128u * (uint32_t)(ra + rb);
            if (CG == 2) bytes += 128u * (uint32_t)(held(m0 + GM_M, GM_M, a.M) + held(n0 + BN, BN, a.N));  // the first CTA counts both
        };
        auto load_b = [&](int stage, int kb) {
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
            if (mb) load(stage, GM_A_BYTES, mb, kb * (MXG_KB / 4), n0);  // in units of 2 bytes
            load(stage, SFB, &bsmap, kb * 256, nt * TN / 128);           // in words; tiles past the end are zeros and count as bytes
        };
        Piece p;
        int early = 0;  // stages whose B is on its way before the wait for the kernel that makes A
        if (ok && a.early) {
            for (int i = 0; early < ST && piece_at<CG>(a, i, &p); ++i) {
                tile(p.tile);
                for (int kb = p.kb0; kb < p.kb1 && early < ST; ++kb, ++early)
                    if (elect_one()) load_b(early, kb);
            }
            __syncwarp();
        }
        pdl_wait_then_release();
        for (int i = 0; ok && piece_at<CG>(a, i, &p); ++i) {
            tile(p.tile);
            for (int kb = p.kb0; kb < p.kb1; ++kb, ++it) {
                if (!__all_sync(0xffffffffu, gm_wait<false>(&empty[s], ph, a.wait))) {
                    *fail = 1;
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    if (it >= early) load_b(s, kb);
                    if (ma) load(s, 0, ma, kb * (MXG_KB / 4), m0);
                    load(s, SFA, &asmap, kb * 256, m0 / 128);
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
    } else if (warp == MXG_EPI + 1) {
        if (rank == 0) {  // MMAs
            int s = 0, it = 0;
            uint32_t ph = 0;
            bool ok = a.wait > 0;
            const uint64_t da0 = umma_desc_sw128(smem_u32(sm)), db0 = umma_desc_sw128(smem_u32(sm) + GM_A_BYTES);
            const uint64_t sf0 = scale_desc(smem_u32(sm) + SFA);
            auto commit = [&](uint64_t* bar) {
                if constexpr (CG == 2) umma_commit_pair(bar);
                else umma_commit(bar);
            };
            Piece p;
            int g = 0;  // accumulators handed over
            for (int i = 0; ok && piece_at<CG>(a, i, &p); ++i, ++g) {
                const int acc = g % ACCS;
                if (g >= ACCS &&
                    !__all_sync(0xffffffffu, gm_wait<CG == 2>(&tempty[acc], (uint32_t)(g / ACCS - 1) & 1u, a.wait))) {
                    *fail = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)((g & 1) * mxg_acc_step(TN));
                uint32_t more = 0;
                for (int kb = p.kb0; kb < p.kb1; ++kb, ++it) {
                    if (!__all_sync(0xffffffffu, gm_wait<false>(&full[s], ph, a.wait))) {
                        *fail = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t at = (uint32_t)s * (STAGE >> 4);  // a stage on, in units of 16
                        const uint32_t sa = tmem + SF0 + (uint32_t)s * SFC, sb = sa + 8;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            scales_to_tmem<CG>(sa + 4 * h, sf0 + at + 32 * h);
#pragma unroll
                            for (int t = 0; t < BT; ++t) scales_to_tmem<CG>(sb + 4 * BT * h + 4 * t, sf0 + at + 64 + 64 * t + 32 * h);
                        }
#pragma unroll
                        for (int k = 0; k < MXG_KB / 64; ++k) {  // 64 k: 32 bytes
                            const uint32_t id = IDESC | (uint32_t)(k & 1) << 30 | (uint32_t)(k & 1) << 5;
                            umma_mxf4<CG>(d, da0 + at + 2 * k, db0 + at + 2 * k, id, sa + 4 * (k >> 1), sb + 4 * BT * (k >> 1), more);
                            more = 1;
                        }
                        commit(&empty[s]);
                        if (kb + 1 == p.kb1) commit(&tfull[acc]);
                    }
                    more = 1;
                    __syncwarp();
                    if (++s == ST) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (lane == 0) *consumed = it;
        }
    } else if (warp < 4 * MXG_PARTS) {
        Piece p;
        int g = 0;
        bool ok = a.wait > 0;
        if (!ok) *fail = 1;
        // A warp takes its part of the accumulator's shared columns first (of all, where nothing is shared), to registers, gives
        // the accumulator back, and then its part of the others from where they lie.
        const uint32_t tq = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        unsigned char* st = staging + warp * 2048;
        // once a wait gave up the pieces that are left take NaN without waiting
        for (int i = 0; piece_at<CG>(a, i, &p); ++i) {
            int mt, nt;
            tile_of<TM>(a, p.tile, &mt, &nt);
            const int row0 = mt * TM + (int)rank * GM_M + (warp & 3) * 32, n0 = nt * TN;
            int c = (TN == 256 && !(g & 1) ? 128 : 0) + (warp >> 2) * 32;
            uint32_t rq[16];
            if (p.slot < 0) fetch_rows(a, rq, row0, n0 + c);  // before the accumulator is there
            const int acc = g % ACCS;
            const uint32_t tm = tq + (uint32_t)((g & 1) * mxg_acc_step(TN));
            ok = ok && __all_sync(0xffffffffu, gm_wait<false>(&tfull[acc], (uint32_t)(g / ACCS) & 1u, a.wait) && !*fail);
            if (!ok) *fail = 1;
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < (TN == 256 ? 2 : 1); ++q) {
                float v[32];
                if (ok) tmem_ld32(tm + (uint32_t)c, v);
                else fill_nan(v);
                if (q == 0 && ok) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (CG == 2) arrive_remote(mapa_shared(smem_u32(&tempty[acc]), 0));
                        else mbar_arrive(&tempty[acc]);
                    }
                    ++g;
                }
                const int n = n0 + c;
                c ^= 128;
                if (p.slot >= 0) {
                    keep_sums<TM, TN>(a, v, row0, n, nt, p.slot, st);
                } else {
                    if (n < a.N) finish_block(a, v, rq, row0, n, st);
                    if (TN == 256 && q == 0) fetch_rows(a, rq, row0, n0 + c);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*fail && warp == MXG_EPI + 1 && rank == 0) {  // every MMA issued has completed
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
    if (warp == MXG_EPI + 1) {
        tc_fence_after();
        if constexpr (CG == 2) tmem_dealloc_pair(tmem, MXG_TMEM);
        else tmem_dealloc(tmem, MXG_TMEM);
    }
}

template <int CG, int TN>
int mx_gemm_tn(const MxOperand& A, const MxOperand& B, int64_t K, GemmArgs a, const Plan& p, void* stream) {
    constexpr int TM = CG * GM_M;
    a.wait = wait_limit();
    CUtensorMap amap, atail, bmap, btail, asmap, bsmap;
    const int64_t row = mx_row_bytes(K) / 2, tiles = mx_tiles(K);  // a row's codes in units of 2 bytes
    constexpr int BN = TN / CG;
    auto tail = [](int all, int part) { return all % part ? (all % part + 7) / 8 * 8 : 8; };
    int rc = tensor_map_2d(&amap, A.codes, row, a.M, row, MXG_KB / 4, GM_M);
    if (rc == B2S_OK) rc = tensor_map_2d(&atail, A.codes, row, a.M, row, MXG_KB / 4, tail(a.M, GM_M));
    if (rc == B2S_OK) rc = tensor_map_2d(&bmap, B.codes, row, a.N, row, MXG_KB / 4, BN);
    if (rc == B2S_OK) rc = tensor_map_2d(&btail, B.codes, row, a.N, row, MXG_KB / 4, tail(a.N, BN));
    if (rc == B2S_OK) rc = tensor_map_words(&asmap, A.scales, tiles * 256, (a.M + 127) / 128, 256, 1);
    if (rc == B2S_OK) rc = tensor_map_words(&bsmap, B.scales, tiles * 256, (a.N + 127) / 128, 256, mxg_btiles(TN));
    if (rc != B2S_OK) return rc;
    a.tiles_m = (a.M + TM - 1) / TM;
    a.tiles_n = (a.N + TN - 1) / TN;
    a.nkb = (int)tiles;
    // Row tiles one after another where the weight stays in L2 meanwhile, a third of it at most (8192 x 14336 x 4096 168 us against
    // 174, 8192 x 4096 x 14336 146 against 149.5, but 8192 x 4096 x 4096 51.6 against 50.8); beyond, so many together that it is
    // read once for each 2048 rows (2048 x 28672 x 8192 164 against 200, 1000 x 75968 x 4096 125 against 151).
    a.group = a.N * row * 2 <= 40ll << 20 ? 1 : 0;
    a.waves = p.waves;
    a.rest = p.rest;
    a.split = p.split;
    a.chunk = p.chunk;
    const auto kernel = mx_gemm_kernel<CG, TN>;
    static std::atomic<bool> set[64];  // the attribute is set once per device; racing callers set the same
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e);
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)mxg_smem(CG, TN));
        if (e != cudaSuccess) return cuda_fail(e);
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    e = launch_cluster(kernel, dim3((unsigned)(p.G * CG)), CG, MXG_THREADS, mxg_smem(CG, TN), stream, amap, atail, bmap, btail,
                       asmap, bsmap, a);
    if (e == cudaSuccess && p.split > 1) {
        const int held = a.M < TM ? a.M : TM;
        e = launch_pdl(gemm_join_kernel<TM, TN, EPI_LINEAR>,
                       dim3((unsigned)((held * (TN / 4) + FIX_NT - 1) / FIX_NT), (unsigned)p.rest), FIX_NT, 0, stream, a, p.G);
    }
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

}  // namespace

// The cheaper of two cuts by estimated clocks: tiles of 128 x 128 by one CTA, 256 x 256 by a pair (128 x 64 was up to 1 us
// better for a few short products, 128 x 256 or a pair with 128 columns up to 4 % for a few others).  A stage costs its MMAs
// (530 clocks for 256 columns; 480 for 128, the issuing warp's pace) or its way from L2 (62 bytes a clock; rows outside A are
// not fetched), with a single tile of rows its weights' way from HBM (26 bytes a clock for each of all CTAs).  A pair's
// accumulators share columns, and its MMAs wait 1500 clocks a tile for the epilogue to take them.  The epilogue costs 4000
// clocks for 128 columns, hidden under the next tile's stages except the last one's.  Tiles that do not fill a round may be
// split along k, where the saving passes the second launch, 6000 clocks, and the sums' way there and back.
// Measured, us, 128 x 128 / 256 x 256: 300 x 4096 x 4096 13.8 / 15.9, 2000 x 4096 x 4096 33 / 28, 1000 x 4096 x 151936 345 / 248,
// 8192 x 768 x 768 15.9 / 18.7; 16 x 16384 x 256 23.7 whole, 14.3 in four.
Plan mx_plan(int M, int N, int64_t K) {
    auto ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    const int sms = sms_here();
    const int64_t nkb = mx_tiles(K);
    Plan best = {};
    int64_t best_cost = INT64_MAX;
    for (int cg = 1; cg <= 2; ++cg) {
        const int tn = 128 * cg, tm = GM_M * cg, U = sms / cg;
        if (cg == 2 && M <= GM_M) continue;  // half of the pair would have no rows
        const int64_t tiles = ceil_div(M, tm) * ceil_div(N, tn);
        const int64_t busy = tiles < U ? tiles : U, hbm = M <= GM_M ? tn * 136 * busy / (26 * U) : 0;
        int64_t stage = cg == 2 ? 530 : 480;
        const int64_t fill = ((M < GM_M ? M : GM_M) + tn / cg) * 136 / 62;
        if (stage < fill) stage = fill;
        if (stage < hbm) stage = hbm;
        const int64_t wait = cg == 2 ? 1500 : 300, tail = tn == 256 ? 8000 : 4000;
        Plan p = {};
        p.cg = cg;
        p.tn = tn;
        p.G = (int)busy;
        p.waves = (int)(tiles / U);
        p.rest = (int)(tiles % U);
        p.split = 1;
        p.chunk = (int)nkb;
        auto rounds_cost = [&](int64_t rounds) {
            const int64_t mine = nkb * stage + wait;
            return rounds ? mine + (rounds - 1) * (mine > tail ? mine : tail) + tail : 0;
        };
        int64_t cost = rounds_cost(p.waves + (p.rest ? 1 : 0));
        for (int64_t want = 2; p.rest && want <= nkb && want <= 64; want += want < 4 ? 1 : want / 2) {  // 2 3 4 6 9 13 19 28 42 63
            const int64_t chunk = ceil_div(nkb, want), split = ceil_div(nkb, chunk);
            const int64_t bytes = split * p.rest * (M < tm ? M : tm) * tn * 4;
            const int64_t c = rounds_cost(p.waves) + ceil_div(p.rest * split, U) * chunk * stage + tail + 6000 + 2 * bytes / 3000;
            if (split > 1 && c < cost) {
                cost = c;
                p.split = (int)split;
                p.chunk = (int)chunk;
                p.bytes = bytes;
                p.G = (int)(p.waves || p.rest * split >= U ? U : p.rest * split);
            }
        }
        if (cost < best_cost) {
            best_cost = cost;
            best = p;
        }
    }
    return best;
}

int mx_gemm(const MxOperand& A, const MxOperand& B, int64_t K, const GemmArgs& a, void* stream) {
    const Plan p = mx_plan(a.M, a.N, K);
    return p.cg == 2 ? mx_gemm_tn<2, 256>(A, B, K, a, p, stream) : mx_gemm_tn<1, 128>(A, B, K, a, p, stream);
}

}  // namespace b2s
