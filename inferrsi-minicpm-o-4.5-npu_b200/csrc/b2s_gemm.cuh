// The tensor-core product behind the head's log probabilities and the projection (sm_100a): D[m, n] = sum_k A[m, k]
// B[n, k], bf16 operands, fp32 accumulation in tensor memory, with an epilogue that consumes the accumulator where it
// lies.  Either operand may be stored with k contiguous (rows of A or B as they are) or with m / n contiguous (a
// gradient's transposed operand), without a transposed copy: the 128-byte swizzled shared-memory layouts of both
// orders are fed to the same MMA through its descriptors.
//
// A persistent CTA takes tiles of 128 x TN in an order that keeps a group of row tiles together (so that a wave's
// operands stay in L2).  Warp 4 fills a ring of stages by TMA, warp 5 issues the MMAs and the other four warps run the
// epilogue of one tile on one half of tensor memory while the MMAs of the next fill the other half.  Every wait is
// bounded; a wait that gives up ends all roles, waits (bounded) for copies and MMAs in flight, and sets
// B2S_STATUS_WAIT_TIMEOUT.
#pragma once

#include "b2s_head.cuh"
#include "b2s_logprobs.cuh"

namespace b2s {

constexpr int GM_M = 128;        // rows of a tile: the MMA's M, one accumulator lane each
constexpr int GM_KB = 64;        // k per stage: one 128-byte row of the swizzle
constexpr int GM_THREADS = 192;  // warps 0-3: epilogue (their tensor-memory quarter), 4: loads, 5: MMAs
constexpr int GM_GROUP = 16;     // row tiles taken together
constexpr uint32_t GM_A_BYTES = GM_M * GM_KB * 2;

__host__ __device__ constexpr uint32_t gm_b_bytes(int tn) { return (uint32_t)tn * GM_KB * 2; }
__host__ __device__ constexpr uint32_t gm_stage_bytes(int tn) { return GM_A_BYTES + gm_b_bytes(tn); }
// as many stages as fit 200 KB, at most 8
__host__ __device__ constexpr int gm_stages(int tn) {
    return (int)(200u * 1024u / gm_stage_bytes(tn)) > 8 ? 8 : (int)(200u * 1024u / gm_stage_bytes(tn));
}
__host__ __device__ constexpr uint32_t gm_smem(int tn) { return 1024 + gm_stages(tn) * gm_stage_bytes(tn) + 256; }

enum { EPI_LINEAR = 0, EPI_LSE = 1, EPI_DZ = 2, EPI_STORE = 3 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

struct GemmArgs {
    int M, N, nkb, tiles_m, tiles_n;
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
    // EPI_LSE: per row and column tile (m, S, U), the token's value; EPI_DZ: the gradient's inputs
    float c, inv_t;
    const int64_t* tokens;
    float4* part;
    float* token_value;
    const float4* stats;
    const float* g_lp;
    const float* g_h;
};

__device__ __forceinline__ float act_apply(float z, int act) {
    if (act == ACT_RELU) return fmax_nan(z, 0.0f);
    if (act == ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.707106781186547524f));
    if (act == ACT_SILU) return __fdividef(z, 1.0f + ex2(-1.44269504088896341f * z));
    return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == ACT_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if (act == ACT_GELU)
        return 0.5f * (1.0f + erff(z * 0.707106781186547524f)) +
               0.398942280401432678f * z * ex2(-0.72134752044448170f * z * z);
    if (act == ACT_SILU) {
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
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&f)[32]) {
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

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
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
