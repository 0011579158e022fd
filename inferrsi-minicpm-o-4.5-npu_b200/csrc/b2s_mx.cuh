// Microscaled blocks (OCP MX): 32 consecutive elements of a row share a scale 2^e, kept as the byte e + 127 (E8M0; 255 is
// NaN), e = max(floor(log2 max|x|) - E, -127), and an element is x 2^-e rounded to the nearest E2M1 value (4 bits, E = 2, at
// most 6) or E4M3 value (8 bits, E = 8, at most 448), ties to even, saturated.  Scaling by a power of two is exact, so an
// element is rounded once.  A block that holds NaN or an infinity has the scale NaN.
//
// A 4-bit matrix lies as rows of 16 bytes a block (the first of two elements in the low half of a byte, elements past the
// row's end zero) and scales in tiles of 128 rows x 8 blocks, 1024 bytes each, rows of tiles one after another.  A tile is
// what the tensor cores take for 256 k: two halves of 4 blocks, in each 16 bytes for row % 32, in those 4 for row / 32.
#pragma once

#include <cuda_fp16.h>

#include "b2s_device.cuh"

namespace b2s {

constexpr int MX_BLOCK = 32;

// A 4-bit matrix.
struct MxOperand {
    const void* codes;
    const void* scales;
};

__host__ __device__ constexpr int64_t mx_blocks(int64_t k) { return (k + MX_BLOCK - 1) / MX_BLOCK; }
__host__ __device__ constexpr int64_t mx_row_bytes(int64_t k) { return mx_blocks(k) * 16; }
__host__ __device__ constexpr int64_t mx_tiles(int64_t k) { return (mx_blocks(k) + 7) / 8; }  // along a row
// Where the scale of a row's block lies, `tiles` = mx_tiles.
__host__ __device__ constexpr int64_t mx_scale_at(int64_t row, int64_t block, int64_t tiles) {
    return ((row >> 7) * tiles + (block >> 3)) * 1024 + ((block >> 2) & 1) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// The scale's byte for the largest magnitude of a block (its bits), and 2^-e for the byte.
template <int E>
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t most) {
    const int f = (int)(most >> 23);
    return f == 255 ? 255u : (uint32_t)max(f - E, 0);
}
__device__ __forceinline__ float mx_inverse(uint32_t code) { return __uint_as_float((254u - min(code, 253u)) << 23); }
// 2^e: a subnormal at 0, NaN at 255.
__device__ __forceinline__ float mx_scale(uint32_t code) {
    return __uint_as_float(code == 0 ? 0x00400000u : code == 255 ? 0x7fc00000u : code << 23);
}

// 8 values (already times 2^-e) as E2M1 codes, the first in the low bits.
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8]) {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t b;
        asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}"
            : "=r"(b)
            : "f"(v[2 * j]), "f"(v[2 * j + 1]));
        r |= b << (8 * j);
    }
    return r;
}
// The values of E2M1 codes as bf16 pairs: both bytes of a magnitude looked up by its code's low three bits, four codes at a
// time (a byte permutation takes its selectors where the codes lie), the sign put on top.
__device__ __forceinline__ void mx_decode4(uint32_t n, uint32_t* w) {
    const uint32_t lo = __byte_perm(0xc0800000u, 0xc0804000u, n & 0x7777u);
    const uint32_t hi = __byte_perm(0x3f3f3f00u, 0x40404040u, n & 0x7777u) | __byte_perm(0x00008000u, 0u, (n >> 3) & 0x1111u);
    w[0] = __byte_perm(lo, hi, 0x5140u);
    w[1] = __byte_perm(lo, hi, 0x7362u);
}
__device__ __forceinline__ void mx_decode8(uint32_t c, uint32_t (&w)[4]) {
    mx_decode4(c, w);
    mx_decode4(c >> 16, w + 2);
}
__device__ __forceinline__ void mx_decode8(uint32_t c, float (&v)[8]) {
    uint32_t w[4];
    mx_decode8(c, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
}
// Two bf16 times a power of two (a bf16): exact, but below the normal range.
__device__ __forceinline__ uint32_t mx_scale2(uint32_t w, uint32_t f) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(f));
    return r;
}
// 2^e, or 2^-e, twice as bf16.
__device__ __forceinline__ uint32_t mx_twice(float f) {
    const uint32_t b = __float_as_uint(f) >> 16;
    return b | b << 16;
}
// 4 values as E4M3, and back.
__device__ __forceinline__ uint32_t mx_encode4_e4m3(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
__device__ __forceinline__ void mx_decode4_e4m3(uint32_t c, float (&v)[4]) {
    uint32_t l, h;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(l), "=r"(h)
        : "r"(c));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&l)), y = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[0] = x.x;
    v[1] = x.y;
    v[2] = y.x;
    v[3] = y.y;
}

// Up to 8 values to bf16, each rounded once; `vec`: p is 16-byte aligned.
__device__ __forceinline__ void mx_store8(__nv_bfloat16* p, int n, bool vec, const float (&v)[8]) {
    if (vec && n == 8) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) p[j] = __float2bfloat16_rn(v[j]);
    }
}

}  // namespace b2s
