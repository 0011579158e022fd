// The tensor-core product behind the head's log probabilities and the projection (sm_100a): D[m, n] = sum_k A[m, k]
// B[n, k], bf16 operands, fp32 accumulation in tensor memory, with an epilogue that consumes the accumulator where it
// lies.  Either operand may be stored with k contiguous (rows of A or B as they are) or with m / n contiguous (a
// gradient's transposed operand), without a transposed copy: the 128-byte swizzled shared-memory layouts of both
// orders are fed to the same MMA through its descriptors.
//
// A persistent CTA, or a pair of them (a cluster of two on one tile, cta_group::2), takes tiles of 128 or 256 x TN in an
// order that keeps a group of row tiles together (so that a wave's operands stay in L2).  What bounds a large product is
// the way from L2 to the SMs, about 64 bytes a clock each: a 128 x 256 tile of one CTA asks for 96 while its MMAs run
// (48 KB per 512 clocks), so it keeps the tensor pipe 60 % busy; a pair holds 128 rows of A each and half of B's
// columns, and asks for 64.  Warp 8 fills a ring of stages by TMA, warp 9 issues the MMAs and eight warps run the
// epilogue of one tile on one half of tensor memory while the MMAs of the next fill the other half.  Tiles that do not
// fill a wave are split along k into equal chunks, all tiles' first chunks first (CTAs at work at the same time then
// read the same k range of both operands, once from HBM); a chunk's fp32 sums go to a workspace, and a second kernel
// adds them in k order and runs the epilogue, so the result does not depend on timing.  Rows go to and from global memory through a swizzled 4 KB block of shared memory per
// warp, whole 128-byte lines at a time.  The epilogues are loops over 32 columns with short bodies: unrolled over a
// tile, with every activation inlined per element, they ran from beyond the instruction cache and a 128 x 256 tile took
// 17 to 47 us.  Every wait is bounded; a wait that gives up ends the loads and the MMAs, makes NaN of every accumulator
// that was not complete (in the output, or in the sums and states that the following kernels read, which make NaN of them
// in turn), waits (bounded) for copies and MMAs in flight, and sets B2S_STATUS_WAIT_TIMEOUT.
#pragma once

#include <cuda_fp16.h>

#include "b2s_head.cuh"
#include "b2s_logprobs.cuh"

namespace b2s {

constexpr int GM_M = 128;        // rows of a tile: the MMA's M, one accumulator lane each
constexpr int GM_KB = 64;        // k per stage: one 128-byte row of the swizzle
constexpr int GM_EPI = 8;        // epilogue warps: warp w has tensor-memory quarter w % 4 and half w / 4 of the columns
constexpr int GM_THREADS = 32 * GM_EPI + 64;
constexpr int GM_GROUP = 16;     // row tiles taken together
constexpr uint32_t GM_A_BYTES = GM_M * GM_KB * 2;

// A stage of one CTA: its 128 rows of A and its 1 / CG of the TN columns of B.
__host__ __device__ constexpr uint32_t gm_stage_bytes(int cg, int tn) { return GM_A_BYTES + (uint32_t)(tn / cg) * GM_KB * 2; }
constexpr uint32_t GM_STAGING = GM_EPI * 4096;  // per epilogue warp: 32 rows x (64 bytes of output, 64 of pre-activation)
// as many stages as fit 192 KB, at most 8
__host__ __device__ constexpr int gm_stages(int cg, int tn) {
    return (int)(192u * 1024u / gm_stage_bytes(cg, tn)) > 8 ? 8 : (int)(192u * 1024u / gm_stage_bytes(cg, tn));
}
__host__ __device__ constexpr uint32_t gm_smem(int cg, int tn) {
    return 1024 + gm_stages(cg, tn) * gm_stage_bytes(cg, tn) + GM_STAGING + 256;
}

// The head's logits are handed over every 1024 k and added in registers: the tensor cores' fp32 accumulation loses about a
// truncation per MMA of what is summed so far, which over 4096 k put the log probabilities 1.6e-6 off (relative), and by
// quarters a quarter of that.
constexpr int GM_SEGMENT = 1024 / GM_KB;

enum { EPI_LINEAR = 0, EPI_LSE = 1, EPI_DZ = 2, EPI_STORE = 3 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

struct GemmArgs {
    int M, N, nkb, tiles_m, tiles_n;
    // full waves of whole tiles, then `rest` tiles in `split` chunks of `chunk` k blocks each (split 1: whole tiles)
    int waves, rest, split, chunk;
    long long wait;  // clocks a wait takes at most; 0: nothing is loaded or multiplied and the product counts as given up
    float* partial;  // split > 1: [split][rest][min(M, rows of a tile)][TN] fp32
    uint32_t* status;
    // EPI_LINEAR, EPI_STORE, EPI_DZ: the output [M, N] bf16
    void* out;
    int64_t out_stride;
    int out_vec;  // rows of `out` 16-byte aligned
    // EPI_LINEAR
    const void* bias;
    const void* residual;
    int64_t res_stride;
    int res_vec;
    int act;
    void* preact;
    int64_t pre_stride;
    // EPI_LSE: per row and half of a column tile (m, S, U), the token's value; EPI_DZ: the gradient's inputs
    float c, inv_t;
    const int64_t* tokens;
    float4* part;
    float* token_value;
    const float4* stats;
    const float* g_lp;
    const float* g_h;
};

// 2 (1 - Phi(|z|)) = erfc(|z| / sqrt 2), and e^(-z^2 / 2), which the slope needs too: the tail is t P(t) e^(-z^2 / 2) with
// t = 1 / (1 + 0.363 |z|) and P the polynomial of degree 6 whose largest relative error over |z| <= 14.5 is least (a linear
// program over a grid: 8e-7).  For negative z the result is z times the tail, so that the error has to be relative: with
// fp32's arithmetic it is below 2e-6 down to z = -5 and 8e-6 at -13 (the exponent's own rounding), where the result leaves
// fp32's normal range; a half step of bf16 is 2e-3 at least.
__device__ __forceinline__ float gelu_tail(float z, float* e) {
    const float a = fabsf(z), t = __fdividef(1.0f, __fmaf_rn(0.363f, a, 1.0f));
    *e = ex2(-0.72134752044448170f * a * a);
    float p = 0.096218183507f;
    p = __fmaf_rn(p, t, -0.358431707466f);
    p = __fmaf_rn(p, t, 0.346512311336f);
    p = __fmaf_rn(p, t, 0.061501895887f);
    p = __fmaf_rn(p, t, 0.278014403086f);
    p = __fmaf_rn(p, t, 0.286393762026f);
    p = __fmaf_rn(p, t, 0.289791861116f);
    return p * t * *e;
}
template <int ACT>
__device__ __forceinline__ float act_apply(float z) {
    if (ACT == ACT_RELU) return fmax_nan(z, 0.0f);
    if (ACT == ACT_GELU) {
        float e;
        const float q = 0.5f * gelu_tail(z, &e);
        return z * (z > 0.0f ? 1.0f - q : q);
    }
    if (ACT == ACT_SILU) {  // z / (1 + e^-z); below zero z e^z / (1 + e^z), e^z by halves, as it leaves the range before z e^z does
        const float h = ex2(-0.72134752044448170f * fabsf(z)), w = z < 0.0f ? z * h * h : z;
        return __fdividef(w, __fmaf_rn(h, h, 1.0f));
    }
    return z;
}
__device__ __forceinline__ float act_apply(float z, int act) {
    return act == ACT_RELU ? act_apply<ACT_RELU>(z)
                           : act == ACT_GELU ? act_apply<ACT_GELU>(z) : act == ACT_SILU ? act_apply<ACT_SILU>(z) : z;
}
// The slope of a pre-activation that came back from fp16: past 65504 (infinite there) it is what it is at 6e4.
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    z = fabsf(z) > 6.0e4f ? copysignf(6.0e4f, z) : z;
    if (ACT == ACT_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if (ACT == ACT_GELU) {
        float e;
        const float q = 0.5f * gelu_tail(z, &e);
        return __fmaf_rn(0.398942280401432678f * z, e, z > 0.0f ? 1.0f - q : q);
    }
    if (ACT == ACT_SILU) {
        const float s = __fdividef(1.0f, 1.0f + ex2(-1.44269504088896341f * z));
        return s * (1.0f + z * (1.0f - s));
    }
    return 1.0f;
}

// Shared-memory matrix descriptor of an operand with m (or n) contiguous, 128-byte swizzle: blocks of [64 k rows x 64
// m], 8 KB each; leading offset = the next block of 64 m (bits 16-29), stride offset = the next 8 k rows (bits 32-45).
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// 32 lanes x 32 columns of fp32 from tensor memory (this warp's lane quarter), waited for.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* f) {
    uint32_t v[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p)::"memory");
    return p != 0;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The pair's forms (cta_group::2): tensor memory allocated in both CTAs by a warp of each, MMAs issued by the first CTA
// over both CTAs' shared memory (the same offsets) into both CTAs' tensor memory, completion signalled to the same
// mbarrier in both, and loads into this CTA's shared memory that complete on an mbarrier of the first CTA.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void umma_bf16_pair(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(cluster_bar)
        : "memory");
}

// 16-byte chunk j of row r in a warp's staging block (chunks 0-3: the output or the residual, 4-7: the pre-activation):
// conflict-free for a lane per row, and for the copies below, whose 8 lanes of a phase hold rows r and r + 4.
__device__ __forceinline__ uint4* stage_at(unsigned char* st, int r, int j) {
    return reinterpret_cast<uint4*>(st + r * 128 + ((j ^ (r & 7)) << 4));
}
// The 4-byte word of columns 2 w, 2 w + 1 of row r.
__device__ __forceinline__ uint32_t* stage_word(unsigned char* st, int r, int w) {
    return reinterpret_cast<uint32_t*>(st + r * 128 + (((w >> 2) ^ (r & 7)) << 4)) + (w & 3);
}
// Copies between a staging block and 32 rows x 32 bf16 of global memory, rows `stride` elements apart.  `vec` (16-byte
// aligned rows, all 32 columns there): 4 lanes per row, 8 rows at a time; else a column per lane.  What is read from the
// block goes to registers before any of it is stored, as the compiler cannot tell that the two do not overlap and would wait
// for each read by itself (4099 rows of 1537 columns out of 768: 20.0 against 15.2 us).
__device__ __forceinline__ int vec_row(int i) {
    const int rr = (threadIdx.x & 31) >> 2;
    return 8 * i + (rr & 1) * 4 + (rr >> 1);
}
__device__ __forceinline__ void block_store(unsigned char* st, int base, void* out, int64_t stride, int rows, int cols,
                                            bool vec) {
    const int lane = threadIdx.x & 31;
    unsigned short* p = static_cast<unsigned short*>(out);
    if (vec) {
        const int c = lane & 3;
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *stage_at(st, vec_row(i), base + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = vec_row(i);
            if (r < rows) *reinterpret_cast<uint4*>(p + r * stride + 8 * c) = v[i];
        }
    } else if (lane < cols) {
        const unsigned char* column = st + 2 * (lane & 7);
        p += lane;
#pragma unroll 1
        for (int r = 0; r < 32; r += 8) {
            unsigned short v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[k] = *reinterpret_cast<const unsigned short*>(column + (r + k) * 128 + (((base + (lane >> 3)) ^ k) << 4));
#pragma unroll
            for (int k = 0; k < 8; ++k, p += stride)
                if (r + k < rows) *p = v[k];
        }
    }
}
// A block of the residual into registers, in flight until it is put into the staging block.
__device__ __forceinline__ void block_fetch(uint32_t (&q)[16], const void* in, int64_t stride, int rows, int cols, bool vec) {
    const int lane = threadIdx.x & 31;
    const unsigned short* p = static_cast<const unsigned short*>(in);
    if (vec) {
        const int c = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = vec_row(i);
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (r < rows) u = __ldg(reinterpret_cast<const uint4*>(p + r * stride + 8 * c));
            q[4 * i] = u.x;
            q[4 * i + 1] = u.y;
            q[4 * i + 2] = u.z;
            q[4 * i + 3] = u.w;
        }
    } else {
        const int w = lane & 15, left = cols - 2 * w;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = 2 * i + (lane >> 4);
            const unsigned short* g = p + r * stride + 2 * w;
            uint32_t lo = 0, hi = 0;
            if (r < rows && left >= 1) lo = __ldg(g);
            if (r < rows && left >= 2) hi = __ldg(g + 1);
            q[i] = lo | hi << 16;
        }
    }
}
__device__ __forceinline__ void block_put(unsigned char* st, const uint32_t (&q)[16], bool vec) {
    const int lane = threadIdx.x & 31;
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *stage_at(st, vec_row(i), lane & 3) = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) *stage_word(st, 2 * i + (lane >> 4), lane & 15) = q[i];
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// This lane's row of 32 values into chunks `base` .. base + 3, each rounded once to bf16 (the output's type).
__device__ __forceinline__ void stage_row(unsigned char* st, int base, const float (&v)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *stage_at(st, lane, base + j) =
            make_uint4(pack_bf16(v[8 * j], v[8 * j + 1]), pack_bf16(v[8 * j + 2], v[8 * j + 3]),
                       pack_bf16(v[8 * j + 4], v[8 * j + 5]), pack_bf16(v[8 * j + 6], v[8 * j + 7]));
}

// The saved pre-activation is fp16: the slope taken from it is off by 2^-12 of z times the activation's curvature, an
// eighth of what bf16 would add to dz's own rounding to the tensor cores' bf16, and slopes are flat long before fp16's
// range ends.  A positive value below its range stays positive (the rectifier's slope asks for the sign).
__device__ __forceinline__ unsigned short preact_bits(float z) {
    const unsigned short h = __half_as_ushort(__float2half_rn(z));
    return z > 0.0f && h == 0 ? 1 : h;
}
__device__ __forceinline__ float preact_value(unsigned short h) { return __half2float(__ushort_as_half(h)); }
__device__ __forceinline__ void stage_preact(unsigned char* st, const float (&v)[32]) {
    const int lane = threadIdx.x & 31;
    auto two = [](float a, float b) { return (uint32_t)preact_bits(a) | (uint32_t)preact_bits(b) << 16; };
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *stage_at(st, lane, 4 + j) = make_uint4(two(v[8 * j], v[8 * j + 1]), two(v[8 * j + 2], v[8 * j + 3]),
                                                two(v[8 * j + 4], v[8 * j + 5]), two(v[8 * j + 6], v[8 * j + 7]));
}

// Up to 8 bf16 of a row from column n (N columns), `vec`: the row is 16-byte aligned and n a multiple of 8.
__device__ __forceinline__ void load8(const void* row, int n, int N, bool vec, float (&x)[8]) {
    const unsigned short* p = static_cast<const unsigned short*>(row) + n;
    if (vec && n + 8 <= N) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = n + j < N ? bf16_bits_to_f(__ldg(p + j)) : 0.0f;
    }
}
// The same stored, each value rounded once to bf16 (the output's type).
__device__ __forceinline__ void store8(void* row, int n, int N, bool vec, const float* x) {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(row) + n;
    if (vec && n + 8 <= N) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < N) p[j] = __float2bfloat16_rn(x[j]);
    }
}

}  // namespace b2s
