// Microscaled 4-bit matrices (b2s_mx.cuh): quantisation, the way back, and the product of microscaled operands with bias,
// activation and residual in its epilogue.  No counterpart in the reference.
#include <string.h>

#include <type_traits>

#include "../../include/b2s_sampler.h"
#include "b2s_gemm.cuh"
#include "b2s_launch.cuh"
#include "b2s_mx.cuh"

namespace b2s {

int cuda_fail(cudaError_t e);
Plan mx_plan(int M, int N, int64_t K);
int mx_gemm(const MxOperand& A, const MxOperand& B, int64_t K, const GemmArgs& a, void* stream);

namespace {

// ------------------------------------------------------------------ quantisation and back

constexpr int MX_NT = 256;
// Of the kernels of 8-bit blocks, which run beside a product (`beside`: they read nothing that the kernel in front of them
// writes, nor write what it reads): 128 threads of 64 registers fit an SM that the product's CTA is on (2000 x 4096 x 4096 with
// silu: forward 54.5 us against 61.1 with the kernel in front, gradient 108.9 against 113.9; 1024 x 4096 x 768 23.4 against 28.2
// and 30.0 against 32.8; 8192 x 4096 x 4096, where the power cap binds, the same).
constexpr int MX8_NT = 128;
__host__ __device__ constexpr int mx_threads(bool eight) { return eight ? MX8_NT : MX_NT; }
constexpr int MX_SEG = 256;  // elements of a row that a warp takes at a time: 8 a lane, the 8 blocks of a scale tile
// A warp takes the same segment of PER rows, in flight together: of fp32 4, 32 bytes a lane each (2: 2000 x 4096 8.2 us, 4 7.4);
// of bf16 8, 16 bytes each, where that makes more warps than the SMs hold at once, 4 where they are fewer (4 against 8: 300 x 4096
// 2.9 us to 3.3, 2000 x 4095 7.5 to 8.9, but 4099 x 4096 10.4 to 9.9 and 32768 x 4096 67 to 60).  One row after another costs an
// addition or two for each address; segments taken as they come, with a division for each warp, were bound by instruction issue
// (32768 x 4096 bf16 86 against 60 us there, 76 against 59 back: 5.7 TB/s).
bool mx_many(int64_t rows, int64_t k) { return (rows + 7) / 8 * mx_tiles(k) > 32 * (int64_t)sms_here(); }
// A CTA's warps: `wide` of them (1, 2, 4, 8) on segments side by side, the others on further rows.
struct MxGrid {
    int64_t r0, tile, step;  // first row; first segment and the next one's distance
    __device__ __forceinline__ MxGrid(int threads, int wide, int per) {
        const int warp = threadIdx.x >> 5;
        r0 = ((int64_t)blockIdx.x * ((threads / 32) / wide) + warp / wide) * per;
        tile = (int64_t)blockIdx.y * wide + warp % wide;
        step = (int64_t)gridDim.y * wide;
    }
};

// 8 elements of a row as they lie: bf16 pairs or fp32 words.
template <typename T>
struct MxWords {
    uint32_t w[sizeof(T) * 2];
};
__device__ __forceinline__ MxWords<unsigned short> mx_words(const unsigned short* p) {
    const uint4 a = ldg_stream(reinterpret_cast<const uint4*>(p));
    return {{a.x, a.y, a.z, a.w}};
}
__device__ __forceinline__ MxWords<float> mx_words(const float* p) {
    const uint4 a = ldg_stream(reinterpret_cast<const uint4*>(p)), b = ldg_stream(reinterpret_cast<const uint4*>(p) + 1);
    return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
// The same past the first-level cache, for a kernel that has not waited for the one in front of it.
template <typename T>
__device__ __forceinline__ MxWords<T> mx_words_l2(const T* p) {
    MxWords<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint4 a = __ldcg(reinterpret_cast<const uint4*>(p) + i);
        r.w[4 * i] = a.x;
        r.w[4 * i + 1] = a.y;
        r.w[4 * i + 2] = a.z;
        r.w[4 * i + 3] = a.w;
    }
    return r;
}
// Element by element, zeros from n on.
template <typename T>
__device__ __forceinline__ MxWords<T> mx_words(const T* p, int64_t n) {
    MxWords<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 2; ++i) {
        if constexpr (sizeof(T) == 4) r.w[i] = i < n ? __float_as_uint(__ldg(p + i)) : 0u;
        else r.w[i] = (2 * i < n ? (uint32_t)__ldg(p + 2 * i) : 0u) | (2 * i + 1 < n ? (uint32_t)__ldg(p + 2 * i + 1) << 16 : 0u);
    }
    return r;
}
// The largest magnitude's bits as an fp32's (NaN above everything), and the values times `inv` as fp32.
__device__ __forceinline__ uint32_t mx_most(const MxWords<float>& x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, x.w[i] & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ uint32_t mx_most(const MxWords<unsigned short>& x) {
    auto larger = [](uint32_t a, uint32_t b) {  // of the magnitudes, NaN if one is; some sign
        uint32_t r;
        asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    };
    const uint32_t m = larger(larger(x.w[0], x.w[1]), larger(x.w[2], x.w[3])) & 0x7fff7fffu;
    return max(m & 0xffff0000u, m << 16);
}
__device__ __forceinline__ void mx_times(const MxWords<float>& x, float inv, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(x.w[i]) * inv;
}
__device__ __forceinline__ void mx_times(const MxWords<unsigned short>& x, float inv, float (&v)[8]) {
    const uint32_t f = mx_twice(inv);  // what the product takes below bf16's range is far below the smallest element
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = mx_scale2(x.w[i], f);
        v[2 * i] = __uint_as_float(w << 16);
        v[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    }
}
// A segment of an unaligned row, coalesced: elements (fp32) or whole words (bf16, but for the first element of a row that starts
// half a word off), zeros from n on; and through the warp's shared memory 8 consecutive elements a lane.
template <typename T>
struct MxRaw {
    uint32_t w[sizeof(T) * 2], first;
};
__device__ __forceinline__ MxRaw<float> mx_raw(const float* p, int n) {
    const int lane = threadIdx.x & 31;
    MxRaw<float> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = 32 * i + lane < n ? __float_as_uint(__ldg(p + 32 * i + lane)) : 0u;
    return r;
}
__device__ __forceinline__ int mx_half(const unsigned short* p) { return (int)(reinterpret_cast<uintptr_t>(p) >> 1) & 1; }
__device__ __forceinline__ MxRaw<unsigned short> mx_raw(const unsigned short* p, int n) {
    const int lane = threadIdx.x & 31, off = mx_half(p);
    MxRaw<unsigned short> r;
    r.first = off && lane == 0 && n > 0 ? (uint32_t)__ldg(p) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = off + 2 * (32 * i + lane);
        r.w[i] = e + 1 < n ? __ldg(reinterpret_cast<const uint32_t*>(p + e)) : e < n ? (uint32_t)__ldg(p + e) : 0u;
    }
    return r;
}
__device__ __forceinline__ MxWords<float> mx_turn_in(const MxRaw<float>& r, const float*, uint32_t* turn) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) turn[32 * i + lane] = r.w[i];
    __syncwarp();
    const uint4 a = *reinterpret_cast<const uint4*>(turn + 8 * lane), b = *reinterpret_cast<const uint4*>(turn + 8 * lane + 4);
    return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ MxWords<unsigned short> mx_turn_in(const MxRaw<unsigned short>& r, const unsigned short* p, uint32_t* turn) {
    const int lane = threadIdx.x & 31, off = mx_half(p);
    unsigned short* t = reinterpret_cast<unsigned short*>(turn);
    __syncwarp();
    if (off) {
        if (lane == 0) t[0] = (unsigned short)r.first;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 1 + 2 * (32 * i + lane);
            t[e] = (unsigned short)r.w[i];
            if (e + 1 < MX_SEG) t[e + 1] = (unsigned short)(r.w[i] >> 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) turn[32 * i + lane] = r.w[i];
    }
    __syncwarp();
    const uint4 a = *reinterpret_cast<const uint4*>(turn + 4 * lane);
    return {{a.x, a.y, a.z, a.w}};
}
// The way back: 8 consecutive elements a lane, as pairs, to n elements of an unaligned row.
__device__ __forceinline__ void mx_turn_out(unsigned short* p, int n, uint32_t* turn, const uint32_t (&w)[4]) {
    const int lane = threadIdx.x & 31;
    const unsigned short* t = reinterpret_cast<const unsigned short*>(turn);
    __syncwarp();
    *reinterpret_cast<uint4*>(turn + 4 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
    __syncwarp();
    const int off = mx_half(p);
    if (off && lane == 0 && n > 0) p[0] = t[0];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = off + 2 * (32 * i + lane);
        if (e + 1 < n) *reinterpret_cast<uint32_t*>(p + e) = t[e] | (uint32_t)t[e + 1] << 16;
        else if (e < n) p[e] = t[e];
    }
}

// VEC: 16-byte aligned rows.  EIGHT: E4M3 codes, a byte each, and scales [blocks][rows]; else the 4-bit layout, whose scale
// tiles' rows past the matrix get zeros.
template <typename T, bool VEC, bool EIGHT, int PER>
__global__ void __launch_bounds__(mx_threads(EIGHT)) mx_quantize_kernel(const T* x, int64_t row_stride, int64_t rows, int k,
                                                                        uint8_t* codes, uint8_t* scales, int wide, int beside) {
    static_assert(!EIGHT || (VEC && sizeof(T) == 2), "8 bits are a projection's x");
    constexpr int E = EIGHT ? 8 : 2, BYTES = EIGHT ? 8 : 4;  // of a lane's codes
    __shared__ __align__(16) uint32_t turn[VEC ? 1 : MX_NT / 32][VEC ? 4 : MX_SEG * sizeof(T) / 4];
    if (!EIGHT || !beside) pdl_wait_then_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t tiles = mx_tiles(k), nb = mx_blocks(k);
    const MxGrid g(mx_threads(EIGHT), wide, PER);
    if (g.r0 >= (EIGHT ? rows : (rows + 127) / 128 * 128)) return;
    const int live = (int)max((int64_t)0, min((int64_t)PER, rows - g.r0));  // rows of the matrix
    for (int64_t tile = g.tile; tile < tiles; tile += g.step) {
        const int64_t n = tile * MX_SEG + 8 * lane, block = tile * 8 + (lane >> 2);
        const T* p = x + g.r0 * row_stride + (VEC ? n : tile * MX_SEG);
        std::conditional_t<VEC, MxWords<T>, MxRaw<T>> in[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const T* q = p + j * row_stride;
            if constexpr (!VEC) in[j] = mx_raw(q, j < live ? (int)min((int64_t)MX_SEG, k - tile * MX_SEG) : 0);
            else if (j < live && n + 8 <= k) in[j] = EIGHT ? mx_words_l2(q) : mx_words(q);
            else in[j] = mx_words(q, j < live ? k - n : 0);
        }
        uint8_t* c = codes + g.r0 * nb * (4 * BYTES) + block * (4 * BYTES) + BYTES * (lane & 3);
        uint8_t* s = EIGHT ? scales + block * rows + g.r0 : scales + mx_scale_at(g.r0, tile * 8 + (lane >> 4) * 4, tiles);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            MxWords<T> v;
            if constexpr (VEC) v = in[j];
            else v = mx_turn_in(in[j], p + j * row_stride, turn[warp]);
            uint32_t most = mx_most(v);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const uint32_t code = mx_scale_code<E>(most);
            float u[8];
            mx_times(v, mx_inverse(code), u);
            if constexpr (EIGHT) {
                if (j < live && block < nb) {
                    *reinterpret_cast<uint2*>(c) =
                        make_uint2(mx_encode4_e4m3(u[0], u[1], u[2], u[3]), mx_encode4_e4m3(u[4], u[5], u[6], u[7]));
                    if ((lane & 3) == 0) s[j] = (uint8_t)code;
                }
            } else {
                uint32_t word = code | __shfl_down_sync(0xffffffffu, code, 4) << 8;  // four blocks' in every 16th lane
                word |= __shfl_down_sync(0xffffffffu, word, 8) << 16;
                if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(s + 16 * j) = word;
                if (j < live && block < nb) *reinterpret_cast<uint32_t*>(c) = mx_encode8(u);
            }
            c += nb * (4 * BYTES);
        }
    }
    if (EIGHT && beside && blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
}

// The way back, to bf16 or fp32.  A lane takes 8 elements, 16 bytes of bf16; to fp32 4 of either half of a segment, so that a
// store's lanes write one line after another (8 at once: 16384 x 4096 67 against 58 us).
template <typename T, bool VEC, bool EIGHT, int PER>
__global__ void __launch_bounds__(mx_threads(EIGHT)) mx_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                                                          int k, T* out, int64_t out_stride, int wide, int beside) {
    static_assert(!EIGHT || VEC, "8 bits are a projection's x");
    constexpr int H = sizeof(T) == 4 ? 2 : 1, N = 8 / H;  // loads a segment, elements of each
    static_assert(!EIGHT || H == 1, "8 bits come back as bf16");
    __shared__ __align__(16) uint32_t turn[VEC ? 1 : MX_NT / 32][VEC ? 4 : MX_SEG * sizeof(T) / 4];
    if (!EIGHT || !beside) pdl_wait_then_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t tiles = mx_tiles(k), nb = mx_blocks(k);
    const MxGrid g(mx_threads(EIGHT), wide, PER);
    const int live = (int)max((int64_t)0, min((int64_t)PER, rows - g.r0));
    for (int64_t tile = g.tile; tile < tiles; tile += g.step) {
        uint32_t c[PER][EIGHT ? 2 : H], f[PER][H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int n = 128 * h + N * lane;  // in the segment
            const int64_t block = tile * 8 + n / 32;
            const uint8_t* pc = codes + (g.r0 * nb + block) * (EIGHT ? 32 : 16) + (EIGHT ? n % 32 : n % 32 / 2);
            const uint8_t* ps = EIGHT ? scales + block * rows + g.r0 : scales + mx_scale_at(g.r0, block, tiles);
#pragma unroll
            for (int j = 0; j < PER; ++j, pc += nb * (EIGHT ? 32 : 16)) {
                c[j][h] = f[j][h] = 0;
                if (j < live && block < nb) {
                    if constexpr (EIGHT) {
                        const uint2 q = __ldcg(reinterpret_cast<const uint2*>(pc));
                        c[j][0] = q.x;
                        c[j][1] = q.y;
                        f[j][h] = __ldcg(ps + j);
                    } else {
                        if constexpr (H == 2) c[j][h] = __ldg(reinterpret_cast<const unsigned short*>(pc));
                        else c[j][h] = __ldg(reinterpret_cast<const uint32_t*>(pc));
                        f[j][h] = __ldg(ps + 16 * j);
                    }
                }
            }
        }
        T* p = out + g.r0 * out_stride + tile * MX_SEG;
        const int left = (int)min((int64_t)MX_SEG, k - tile * MX_SEG);
#pragma unroll
        for (int j = 0; j < PER; ++j, p += out_stride) {
            if (j >= live) break;
            if constexpr (sizeof(T) == 2) {
                const float s = mx_scale(f[j][0]);
                uint32_t w[4];
                if constexpr (EIGHT) {
                    float a[4], b[4];
                    mx_decode4_e4m3(c[j][0], a);
                    mx_decode4_e4m3(c[j][1], b);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        w[i] = pack_bf16(a[2 * i] * s, a[2 * i + 1] * s);
                        w[2 + i] = pack_bf16(b[2 * i] * s, b[2 * i + 1] * s);
                    }
                } else {
                    mx_decode8(c[j][0], w);
                    const uint32_t s2 = mx_twice(s);
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = mx_scale2(w[i], s2);
                }
                const int n = 8 * lane;
                if constexpr (!VEC) {
                    mx_turn_out(p, left, turn[warp], w);
                } else if (n + 8 <= left) {
                    __stcs(reinterpret_cast<uint4*>(p + n), make_uint4(w[0], w[1], w[2], w[3]));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (n + i < left) p[n + i] = (T)(w[i >> 1] >> (16 * (i & 1)));
                }
            } else {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const float s = mx_scale(f[j][h]);
                    uint32_t w[2];
                    mx_decode4(c[j][h], w);
                    const float4 v = make_float4(__uint_as_float(w[0] << 16) * s, __uint_as_float(w[0] & 0xffff0000u) * s,
                                                 __uint_as_float(w[1] << 16) * s, __uint_as_float(w[1] & 0xffff0000u) * s);
                    const int n = 128 * h + 4 * lane;
                    if (VEC && n + 4 <= left) {
                        __stcs(reinterpret_cast<float4*>(p + n), v);
                    } else if constexpr (VEC) {
                        if (n < left) p[n] = v.x;
                        if (n + 1 < left) p[n + 1] = v.y;
                        if (n + 2 < left) p[n + 2] = v.z;
                    } else {
                        *reinterpret_cast<float4*>(turn[warp] + n) = v;
                    }
                }
                if constexpr (!VEC) {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (32 * i + lane < left) p[32 * i + lane] = __uint_as_float(turn[warp][32 * i + lane]);
                    __syncwarp();
                }
            }
        }
    }
    if (EIGHT && beside && blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
}

// Rows of up to 128 elements, R of them side by side in a warp's 32 lanes (8 of up to 32 elements, 4 of 64, 2), MXN_PER times:
// 262,144 x 128 bf16 17.6 us there and 17.0 back, x 64 9.3, where the kernels above, a row a warp, take 43 and 34, 42 and 34.  Not
// back to unaligned rows, whose stores those put together (65536 x 100 23 against 11).
constexpr int MXN_PER = 4;
constexpr int MX_NARROW = 128;
template <typename T, bool VEC, int R>
__global__ void __launch_bounds__(MX_NT) mx_quantize_narrow_kernel(const T* x, int64_t row_stride, int64_t rows, int k,
                                                                   uint8_t* codes, uint8_t* scales) {
    constexpr int L = 32 / R;  // lanes of a row
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31, col = lane % L, n = 8 * col, block = col >> 2, nb = (int)mx_blocks(k);
    const int64_t all = (rows + 127) / 128 * 128;  // the scale tiles' rows past the matrix get zeros
    const int64_t r0 = ((int64_t)blockIdx.x * (MX_NT / 32) + (threadIdx.x >> 5)) * (R * MXN_PER) + lane / L;
    MxWords<T> in[MXN_PER];
#pragma unroll
    for (int j = 0; j < MXN_PER; ++j) {
        const int64_t r = r0 + j * R;
        const T* q = x + r * row_stride + n;
        if (VEC && r < rows && n + 8 <= k) in[j] = mx_words(q);
        else in[j] = mx_words(q, r < rows ? k - n : 0);
    }
#pragma unroll
    for (int j = 0; j < MXN_PER; ++j) {
        const int64_t r = r0 + j * R;
        uint32_t most = mx_most(in[j]);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const uint32_t code = mx_scale_code<2>(most);
        float u[8];
        mx_times(in[j], mx_inverse(code), u);
        uint32_t word = code;  // the row's blocks in its first lane
        if (L >= 8) word |= __shfl_down_sync(0xffffffffu, word, 4) << 8;
        if (L >= 16) word |= __shfl_down_sync(0xffffffffu, word, 8) << 16;
        if (col == 0 && r < all) {
            uint32_t* s = reinterpret_cast<uint32_t*>(scales + mx_scale_at(r, 0, 1));
            s[0] = word;
            s[128] = 0;  // blocks 4 to 7
        }
        if (r < rows && block < nb) *reinterpret_cast<uint32_t*>(codes + (r * nb + block) * 16 + 4 * (col & 3)) = mx_encode8(u);
    }
}
// 8 elements a lane to bf16, 4 to fp32, 16 bytes each.
template <typename T, int R>
__global__ void __launch_bounds__(MX_NT) mx_dequantize_narrow_kernel(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                                                     int k, T* out, int64_t out_stride) {
    constexpr int L = 32 / R, N = 16 / sizeof(T);
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31, n = N * (lane % L), block = n >> 5, nb = (int)mx_blocks(k);
    const int64_t r0 = ((int64_t)blockIdx.x * (MX_NT / 32) + (threadIdx.x >> 5)) * (R * MXN_PER) + lane / L;
    uint32_t c[MXN_PER], f[MXN_PER];
#pragma unroll
    for (int j = 0; j < MXN_PER; ++j) {
        const int64_t r = r0 + j * R;
        c[j] = f[j] = 0;
        if (r < rows && block < nb) {
            const uint8_t* p = codes + (r * nb + block) * 16 + n % 32 / 2;
            if constexpr (N == 8) c[j] = __ldg(reinterpret_cast<const uint32_t*>(p));
            else c[j] = __ldg(reinterpret_cast<const unsigned short*>(p));
            f[j] = __ldg(scales + mx_scale_at(r, block, 1));
        }
    }
#pragma unroll
    for (int j = 0; j < MXN_PER; ++j) {
        const int64_t r = r0 + j * R;
        if (r >= rows || n >= k) continue;
        float v[8];
        mx_decode8(c[j], v);
        const float s = mx_scale(f[j]);
        T* p = out + r * out_stride + n;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= s;
        if constexpr (N == 8) {
            mx_store8(p, min(8, k - n), true, v);
        } else if (n + 4 <= k) {
            __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < k) p[i] = v[i];
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Segments that a CTA's warps take side by side: as many as leave no warp without one where there are many (65536 x 768 bf16 24.2
// us against 26.2, x 576 27.6 against 30.8), else as many as leave each one (4099 x 768 3.9 against 4.3).
int mx_wide(int64_t k, int warps, bool many) {
    const int64_t t = mx_tiles(k), w = many ? t & -t : t > 4 ? 8 : t > 2 ? 4 : t;
    return w < warps ? (int)w : warps;
}
dim3 mx_grid(int64_t rows, int64_t k, int per, int warps, int wide) {
    const int64_t each = (int64_t)per * (warps / wide), y = (mx_tiles(k) + wide - 1) / wide;
    return dim3((unsigned)((rows + each - 1) / each), (unsigned)(y < 65535 ? y : 65535));
}
cudaError_t mx_quantize(const void* x, int dtype, int64_t rows, int k, int64_t row_stride, void* codes, void* scales,
                        void* stream) {
    const int64_t all = (rows + 127) / 128 * 128;
    const bool many = mx_many(all, k);
    const int wide = mx_wide(k, MX_NT / 32, many);
    auto narrow = [&](auto* p, bool vec) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        auto run = [&](auto kernel, int r) {
            const int64_t each = r * MXN_PER * (MX_NT / 32);
            return launch_pdl(kernel, dim3((unsigned)((all + each - 1) / each)), MX_NT, 0, stream, p, row_stride, rows, k,
                              static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
        };
        return k <= 32   ? run(vec ? mx_quantize_narrow_kernel<T, true, 8> : mx_quantize_narrow_kernel<T, false, 8>, 8)
               : k <= 64 ? run(vec ? mx_quantize_narrow_kernel<T, true, 4> : mx_quantize_narrow_kernel<T, false, 4>, 4)
                         : run(vec ? mx_quantize_narrow_kernel<T, true, 2> : mx_quantize_narrow_kernel<T, false, 2>, 2);
    };
    auto go = [&](auto kernel, auto* p, int per) {
        return launch_pdl(kernel, mx_grid(all, k, per, MX_NT / 32, wide), MX_NT, 0, stream, p, row_stride, rows, k,
                          static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), wide, 0);
    };
    const bool vec = aligned16(x) && row_stride * (dtype == B2S_DTYPE_F32 ? 4 : 2) % 16 == 0;
    if (dtype == B2S_DTYPE_F32) {
        const float* p = static_cast<const float*>(x);
        if (k <= MX_NARROW) return narrow(p, vec);
        return go(vec ? mx_quantize_kernel<float, true, false, 4> : mx_quantize_kernel<float, false, false, 4>, p, 4);
    }
    using T = unsigned short;
    const T* p = static_cast<const T*>(x);
    if (k <= MX_NARROW) return narrow(p, vec);
    return many ? go(vec ? mx_quantize_kernel<T, true, false, 8> : mx_quantize_kernel<T, false, false, 8>, p, 8)
                : go(vec ? mx_quantize_kernel<T, true, false, 4> : mx_quantize_kernel<T, false, false, 4>, p, 4);
}
cudaError_t mx_dequantize(const void* codes, const void* scales, int64_t rows, int k, int dtype, void* out, int64_t out_stride,
                          void* stream) {
    const bool many = mx_many(rows, k);
    const int wide = mx_wide(k, MX_NT / 32, many);
    auto narrow = [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        auto run = [&](auto kernel, int r) {
            const int64_t each = r * MXN_PER * (MX_NT / 32);
            return launch_pdl(kernel, dim3((unsigned)((rows + each - 1) / each)), MX_NT, 0, stream,
                              static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, k, p, out_stride);
        };
        constexpr int R = sizeof(T) == 2 ? 8 : 4;  // of rows of 32 elements
        return k <= 32   ? run(mx_dequantize_narrow_kernel<T, R>, R)
               : k <= 64 ? run(mx_dequantize_narrow_kernel<T, R / 2>, R / 2)
                         : run(mx_dequantize_narrow_kernel<T, R / 4>, R / 4);
    };
    auto go = [&](auto kernel, auto* p, int per) {
        return launch_pdl(kernel, mx_grid(rows, k, per, MX_NT / 32, wide), MX_NT, 0, stream, static_cast<const uint8_t*>(codes),
                          static_cast<const uint8_t*>(scales), rows, k, p, out_stride, wide, 0);
    };
    const bool vec = aligned16(out) && out_stride * (dtype == B2S_DTYPE_F32 ? 4 : 2) % 16 == 0;
    if (dtype == B2S_DTYPE_F32) {
        float* p = static_cast<float*>(out);
        if (k <= MX_NARROW && vec) return narrow(p);
        return go(vec ? mx_dequantize_kernel<float, true, false, 4> : mx_dequantize_kernel<float, false, false, 4>, p, 4);
    }
    using T = unsigned short;
    T* p = static_cast<T*>(out);
    if (k <= MX_NARROW && vec) return narrow(static_cast<__nv_bfloat16*>(out));
    return many ? go(vec ? mx_dequantize_kernel<T, true, false, 8> : mx_dequantize_kernel<T, false, false, 8>, p, 8)
                : go(vec ? mx_dequantize_kernel<T, true, false, 4> : mx_dequantize_kernel<T, false, false, 4>, p, 4);
}

// ------------------------------------------------------------------ the product of few rows

// Each 4-bit code of a word as a byte, twice its value: {0, 1, 2, 3, 4, 6, 8, 12}, negative where bit 3 is set.
__device__ __forceinline__ void mx_bytes(uint32_t c, int& lo, int& hi) {
    auto four = [](uint32_t n) {  // the low four codes
        const uint32_t pos = __byte_perm(0x03020100u, 0x0c080604u, n & 0x7777u);
        const uint32_t neg = __byte_perm(0xfdfeff00u, 0xf4f8fafcu, n & 0x7777u);
        const uint32_t mask = __byte_perm(0x0000ff00u, 0u, (n >> 3) & 0x1111u);
        return (int)((pos & ~mask) | (neg & mask));
    };
    lo = four(c);
    hi = four(c >> 16);
}
// The product of two scales: finite unless one is NaN, so that a block whose products are all zero adds zero.
__device__ __forceinline__ float mx_factor(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, 0f7F7FFFFF;" : "=f"(r) : "f"(a * b));
    return r;
}
struct MxRowsArgs {
    const unsigned short* x;  // bf16 rows, or null and the codes and scales of a quantised x
    int64_t x_stride;
    const uint8_t *xc, *xs;
    const uint8_t *wc, *ws;
    int M, N, K, act, x_vec;
    const unsigned short *bias, *residual;
    int64_t res_stride;
    __half* preact;
    int64_t pre_stride;
    __nv_bfloat16* out;
    int64_t out_stride;
};

// out = act(x^ w^T + b) + r for at most R rows.  A CTA quantises x itself (no launch of its own), to bytes in shared memory; then its
// warps take F features at a time: a lane has the blocks 32 apart, 16 bytes of codes each, turned to bytes, and integer dot
// products with x's, exact within a block; blocks are added in fp32.  (With x's blocks in registers and a group of threads per
// feature x was quantised once for every four features: 1 x 4096 x 4096 9.5 us against 6.2.)
constexpr int MXR_NT = 256;
constexpr int MXR_SMEM = 36 * 1024;  // of x: 32 bytes and a factor a block and row
template <int R, int F>
__global__ void __launch_bounds__(MXR_NT) mx_rows_kernel(const __grid_constant__ MxRowsArgs a) {
    constexpr int W = MXR_NT / 32, U = 4;  // warps; blocks of a lane in flight
    extern __shared__ __align__(16) unsigned char xsm[];
    pdl_wait_then_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nb = (int)mx_blocks(a.K);
    const int64_t tiles = mx_tiles(a.K), step = (int64_t)gridDim.x * W * F;
    const uint4* wp[F];
    const uint8_t* sp[F];
    auto at = [&](int64_t n0) {
#pragma unroll
        for (int f = 0; f < F; ++f) {  // a feature past the end repeats the last one
            const int64_t n = min(n0 + f, (int64_t)a.N - 1);
            wp[f] = reinterpret_cast<const uint4*>(a.wc) + n * nb;
            sp[f] = a.ws + mx_scale_at(n, 0, tiles);
        }
    };
    uint4 w[U][F];
    uint32_t ws[U][F];
    auto load = [&](int b0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int f = 0; f < F; ++f)
                if (b0 + 32 * u < nb) {
                    w[u][f] = ldg_stream(wp[f] + b0 + 32 * u);
                    ws[u][f] = __ldg(sp[f] + mx_scale_at(0, b0 + 32 * u, tiles));
                }
    };
    int64_t n0 = ((int64_t)blockIdx.x * W + warp) * F;
    if (n0 < a.N) {  // on their way while x is quantised
        at(n0);
        load(lane);
    }
    uint2* xb = reinterpret_cast<uint2*>(xsm);  // [R][nb][4]: a lane's 8 elements as bytes; the lanes' 16-byte reads are 32 apart
    float* xf = reinterpret_cast<float*>(xsm + (size_t)R * nb * 32);  // [R][nb]
    for (int i0 = warp * 32; i0 < 4 * R * nb; i0 += MXR_NT) {         // 8 elements a lane, a block four lanes
        const int i = i0 + lane, r = i / (4 * nb), e = i % (4 * nb);
        const bool in = i < 4 * R * nb;
        const int64_t m = min(r, a.M - 1);  // rows past the end repeat the last one; they are not stored
        uint32_t c = 0;
        float f = 0.0f;
        if (a.x) {
            const unsigned short* row = a.x + m * a.x_stride + 8 * e;
            const int left = in ? a.K - 8 * e : 0;
            const MxWords<unsigned short> v = a.x_vec && left >= 8 ? mx_words(row) : mx_words(row, left);
            uint32_t most = mx_most(v);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const uint32_t code = mx_scale_code<2>(most);
            float u[8];
            mx_times(v, mx_inverse(code), u);
            c = mx_encode8(u);
            f = mx_scale(code);
        } else if (in) {
            c = __ldg(reinterpret_cast<const uint32_t*>(a.xc) + m * nb * 4 + e);
            f = mx_scale(__ldg(a.xs + mx_scale_at(m, e >> 2, tiles)));
        }
        if (!in) continue;
        int lo, hi;
        mx_bytes(c, lo, hi);
        xb[i] = make_uint2((uint32_t)lo, (uint32_t)hi);
        if ((e & 3) == 0) xf[i >> 2] = f * 0.25f;  // both operands' bytes are doubled
    }
    __syncthreads();
    for (; n0 < a.N; n0 += step) {
        float acc[R][F] = {};
        for (int b0 = lane; b0 < nb; b0 += 32 * U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int b = b0 + 32 * u;
                if (b >= nb) break;
                int wb[F][8];
                float s[F];
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    mx_bytes(w[u][f].x, wb[f][0], wb[f][1]);
                    mx_bytes(w[u][f].y, wb[f][2], wb[f][3]);
                    mx_bytes(w[u][f].z, wb[f][4], wb[f][5]);
                    mx_bytes(w[u][f].w, wb[f][6], wb[f][7]);
                    s[f] = mx_scale(ws[u][f]);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int4* x = reinterpret_cast<const int4*>(xb) + 2 * (r * nb + b);
                    const int4 p = x[0], q = x[1];
                    const float xs = xf[r * nb + b];
#pragma unroll
                    for (int f = 0; f < F; ++f) {
                        int d = __dp4a(wb[f][0], p.x, 0);
                        d = __dp4a(wb[f][1], p.y, d);
                        d = __dp4a(wb[f][2], p.z, d);
                        d = __dp4a(wb[f][3], p.w, d);
                        d = __dp4a(wb[f][4], q.x, d);
                        d = __dp4a(wb[f][5], q.y, d);
                        d = __dp4a(wb[f][6], q.z, d);
                        d = __dp4a(wb[f][7], q.w, d);
                        acc[r][f] = __fmaf_rn((float)d, mx_factor(xs, s[f]), acc[r][f]);
                    }
                }
            }
            if (b0 + 32 * U < nb) load(b0 + 32 * U);
        }
        const int64_t done = n0;
        if (n0 + step < a.N) {  // the next features' on their way under the sums
            at(n0 + step);
            load(lane);
        }
        float mine = 0.0f;  // lane r F + f: the row's and feature's sum
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int f = 0; f < F; ++f) {
                float t = acc[r][f];
#pragma unroll
                for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
                mine = lane == r * F + f ? t : mine;
            }
        const int m = lane / F;
        const int64_t n = done + lane % F;
        if (lane < R * F && m < a.M && n < a.N) {
            float t = mine;
            if (a.bias) t += bf16_bits_to_f(__ldg(a.bias + n));
            if (a.preact) a.preact[(int64_t)m * a.pre_stride + n] = __ushort_as_half(preact_bits(t));
            t = act_apply(t, a.act);
            if (a.residual) t += bf16_bits_to_f(__ldg(a.residual + (int64_t)m * a.res_stride + n));
            a.out[(int64_t)m * a.out_stride + n] = __float2bfloat16_rn(t);
        }
    }
}

template <int R>
cudaError_t mx_rows(const MxRowsArgs& a, void* stream) {
    const int64_t most = 3 * (int64_t)sms_here(), one = ((int64_t)a.N + 7) / 8;  // blocks with a feature a warp
    auto go = [&](auto kernel, int64_t want) {
        return launch_pdl(kernel, dim3((unsigned)(want < most ? want : most)), MXR_NT, (uint32_t)(R * mx_blocks(a.K) * 36), stream, a);
    };
    return one <= most ? go(mx_rows_kernel<R, 1>, one) : go(mx_rows_kernel<R, 2>, (one + 1) / 2);
}
cudaError_t mx_rows(const MxRowsArgs& a, void* stream) {
    return a.M == 1 ? mx_rows<1>(a, stream) : a.M == 2 ? mx_rows<2>(a, stream) : mx_rows<4>(a, stream);
}
// Which products take it.  Against the tensor cores' path, us: 1 x 4096 x 768 3.7 : 11.0, 4 x 768 x 6562 6.1 : 8.4, 1 x 4096 x 4096
// 6.2 : 11.7, 4 rows of it 9.9 : 11.9, but 1 x 4096 x 8192 11.9 : 12.3 and 4 rows 20.5 : 12.3, 1 x 768 x 30000 14.0 : 11.3, 1 x
// 4096 x 151936 106 : 63 (turning codes to bytes takes two operations an element).
bool mx_few_rows(int rows, int N, int64_t K) {
    return rows <= 4 && N * K <= 1 << 24 && (rows < 3 ? rows : 4) * mx_blocks(K) * 36 <= MXR_SMEM;
}

// The workspace of the tensor cores' path: x's codes and scales, then the sums of tiles that are split.
struct MxWork {
    int64_t scales, partial;
};
MxWork mx_work(int64_t rows, int64_t k) {
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t s = up(rows * mx_row_bytes(k));
    return {s, s + (rows + 127) / 128 * mx_tiles(k) * 1024};
}

}  // namespace

// Whole rows of a multiple of 8 bf16, all 16-byte aligned.  `beside`: the kernel in front of this one is of the same call and
// waited for what came before it.
cudaError_t mx8_quantize(const void* x, int64_t rows, int k, int64_t row_stride, void* codes, void* scales, bool beside, void* stream) {
    using T = unsigned short;
    const int wide = mx_wide(k, MX8_NT / 32, false);
    return launch_pdl(mx_quantize_kernel<T, true, true, 8>, mx_grid(rows, k, 8, MX8_NT / 32, wide), MX8_NT, 0, stream,
                      static_cast<const T*>(x), row_stride, rows, k, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales),
                      wide, (int)beside);
}
cudaError_t mx8_dequantize(const void* codes, const void* scales, int64_t rows, int k, void* out, bool beside, void* stream) {
    using T = unsigned short;
    const int wide = mx_wide(k, MX8_NT / 32, false);
    return launch_pdl(mx_dequantize_kernel<T, true, true, 8>, mx_grid(rows, k, 8, MX8_NT / 32, wide), MX8_NT, 0, stream,
                      static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, k, static_cast<T*>(out),
                      (int64_t)k, wide, (int)beside);
}

}  // namespace b2s

extern "C" {

int b2s_mx_quantize(const void* x, int32_t dtype, int32_t rows, int32_t k, int64_t row_stride, void* codes, void* scales,
                    void* stream) {
    using namespace b2s;
    if (rows < 0 || k < 1 || row_stride < k || (dtype != B2S_DTYPE_F32 && dtype != B2S_DTYPE_BF16)) return B2S_ERR_INVALID;
    if (rows > LP_MAX_SIZE || k > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
    if (rows == 0) return B2S_OK;
    if (!x || !codes || !scales || !aligned16(codes) || !aligned16(scales) ||
        (reinterpret_cast<uintptr_t>(x) & (dtype == B2S_DTYPE_F32 ? 3 : 1)))
        return B2S_ERR_INVALID;
    const cudaError_t e = mx_quantize(x, dtype, rows, k, row_stride, codes, scales, stream);
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

int b2s_mx_dequantize(const void* codes, const void* scales, int32_t rows, int32_t k, int32_t dtype, void* out,
                      int64_t out_row_stride, void* stream) {
    using namespace b2s;
    if (rows < 0 || k < 1 || out_row_stride < k || (dtype != B2S_DTYPE_F32 && dtype != B2S_DTYPE_BF16)) return B2S_ERR_INVALID;
    if (rows > LP_MAX_SIZE || k > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
    if (rows == 0) return B2S_OK;
    if (!out || !codes || !scales || !aligned16(codes) || !aligned16(scales) ||
        (reinterpret_cast<uintptr_t>(out) & (dtype == B2S_DTYPE_F32 ? 3 : 1)))
        return B2S_ERR_INVALID;
    const cudaError_t e = mx_dequantize(codes, scales, rows, k, dtype, out, out_row_stride, stream);
    return e == cudaSuccess ? B2S_OK : cuda_fail(e);
}

int b2s_mx_linear_workspace(int32_t rows, int32_t in_features, int32_t out_features, int64_t* bytes) {
    using namespace b2s;
    if (rows < 0 || in_features < 1 || out_features < 1 || !bytes) return B2S_ERR_INVALID;
    *bytes = 0;
    if (rows && !mx_few_rows(rows, out_features, in_features)) {
        const MxWork w = mx_work(rows, in_features);
        *bytes = w.partial + mx_plan(rows, out_features, in_features).bytes;
    }
    return B2S_OK;
}

int b2s_mx_linear(const b2s_mx_linear_args* l, void* stream) {
    using namespace b2s;
    if (!l || l->rows < 0 || l->out_features < 1 || l->in_features < 1 || l->activation < 0 || l->activation > B2S_ACT_SILU)
        return B2S_ERR_INVALID;
    if (l->rows > LP_MAX_SIZE || l->in_features > LP_MAX_SIZE || l->out_features > LP_MAX_SIZE) return B2S_ERR_UNSUPPORTED;
    if (l->rows == 0) return B2S_OK;
    if (!l->x == !l->x_codes || !l->weight_codes || !l->weight_scales || !l->out || !aligned16(l->weight_codes) ||
        !aligned16(l->weight_scales) || (l->x && l->x_row_stride < l->in_features) ||
        (l->x_codes && (!l->x_scales || !aligned16(l->x_codes) || !aligned16(l->x_scales))) ||
        l->out_row_stride < l->out_features || (l->residual && l->residual_row_stride < l->out_features) ||
        (l->preact && (!aligned16(l->preact) || l->preact_row_stride < l->out_features || l->preact_row_stride % 8)) ||
        ((reinterpret_cast<uintptr_t>(l->x) | reinterpret_cast<uintptr_t>(l->out) | reinterpret_cast<uintptr_t>(l->bias) |
          reinterpret_cast<uintptr_t>(l->residual)) & 1))
        return B2S_ERR_INVALID;
    int64_t need = 0;
    b2s_mx_linear_workspace(l->rows, l->in_features, l->out_features, &need);
    if (need && (!l->workspace || l->workspace_bytes < need || !aligned16(l->workspace))) return B2S_ERR_INVALID;
    if (mx_few_rows(l->rows, l->out_features, l->in_features)) {
        MxRowsArgs a;
        memset(&a, 0, sizeof(a));
        a.x = static_cast<const unsigned short*>(l->x);
        a.x_stride = l->x_row_stride;
        a.x_vec = aligned16(l->x) && l->x_row_stride % 8 == 0;
        a.xc = static_cast<const uint8_t*>(l->x_codes);
        a.xs = static_cast<const uint8_t*>(l->x_scales);
        a.wc = static_cast<const uint8_t*>(l->weight_codes);
        a.ws = static_cast<const uint8_t*>(l->weight_scales);
        a.M = l->rows;
        a.N = l->out_features;
        a.K = l->in_features;
        a.act = l->activation;
        a.bias = static_cast<const unsigned short*>(l->bias);
        a.residual = static_cast<const unsigned short*>(l->residual);
        a.res_stride = l->residual_row_stride;
        a.preact = static_cast<__half*>(l->preact);
        a.pre_stride = l->preact_row_stride;
        a.out = static_cast<__nv_bfloat16*>(l->out);
        a.out_stride = l->out_row_stride;
        const cudaError_t e = mx_rows(a, stream);
        return e == cudaSuccess ? B2S_OK : cuda_fail(e);
    }
    const MxWork w = mx_work(l->rows, l->in_features);
    unsigned char* ws = static_cast<unsigned char*>(l->workspace);
    MxOperand x = {l->x_codes, l->x_scales};
    if (l->x) {
        x = {ws, ws + w.scales};
        const cudaError_t e = mx_quantize(l->x, B2S_DTYPE_BF16, l->rows, l->in_features, l->x_row_stride, ws, ws + w.scales, stream);
        if (e != cudaSuccess) return cuda_fail(e);
    }
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
    a.partial = reinterpret_cast<float*>(ws + w.partial);
    // The kernel in front of the product is the quantisation, which waits for everything before it: the weight is there.
    a.early = l->x != nullptr;
    return mx_gemm(x, {l->weight_codes, l->weight_scales}, l->in_features, a, stream);
}

}  // extern "C"
