// The embedding lookup with a scale, out[i] = s T[t_i], and its gradient dT[v] = s sum of g[i] over the positions i with
// t_i = v, in ascending order of i.  Ids below 0 are padding: zeros, and no part in the gradient.  Ids past the table are
// taken as padding too and set B2S_STATUS_TOKEN_RANGE.  No counterpart in the reference, whose models call torch's own.
//
// Forward: a copy of rows.  A warp takes a piece of one row, 16 bytes a lane and load, as many loads in flight as the row's length
// wants (one, two or four; eight of single elements).  From a microscaled table a lane decodes 8 elements a load.
//
// Gradient: the whole table's gradient is written once, so what bounds it is that write (1.24 GB for the Thinker's table)
// and one read of the rows' gradients.  The positions are sorted by id without a sort of keys: a count per id (the atomic's
// old value is the position's place among its id's, in order of arrival), the counts' prefix sums, and then each id's
// positions put in ascending order, so that sums do not depend on who arrived first.  The sorted positions are summed in
// chunks of 8 to 32, whatever ids they hold, one chunk a warp and part of a row, in order, in fp32: an id inside a chunk is
// written at once, of one that goes on the sums are joined by whoever completes them, 16 neighbours at a time in a fixed tree.  Where
// chunks cut an id's positions depends on how many positions lower ids have: the same call gives the same bits, another list
// of tokens may add the same rows in another grouping.
#include <string.h>

#include <type_traits>

#include "../../include/b2s_sampler.h"
#include "b2s_device.cuh"
#include "b2s_gemm.cuh"
#include "b2s_launch.cuh"
#include "b2s_logprobs.cuh"
#include "b2s_mx.cuh"

namespace b2s {

int cuda_fail(cudaError_t e);

namespace {

constexpr int EM_NT = 256;
constexpr int EM_JOIN = 4;     // 2^4 sums joined at a time
constexpr int EM_SHORT = 64;   // positions of an id that are put in order by comparison with all of its others
constexpr int EM_MID = 512;    // ... that a CTA puts in order in shared memory; beyond, by bitmaps
constexpr int EM_HUGE = 4096;  // ... beyond which several CTAs do, EM_PARTS at most
constexpr int EM_BINS = 4096;  // at most, of ids counted together
constexpr int EM_UNITS = 64;   // 16-byte units of a row that a warp takes
constexpr int EM_ELEMENTS = 256;  // or single elements, of rows that are not aligned
// Where rows are summed, of single fp32 elements EM_WIDE (30001 x 1001 81 us with 64, 56 with 128, 52 with 256, but 300 x 33 9.9,
// 10.3 and 11.6), of bf16 64 (61; 77 with 256).
constexpr int EM_WIDE = 128;
__host__ __device__ constexpr int em_units(bool vec, int e) { return vec || e == 2 ? EM_UNITS : EM_WIDE; }
constexpr int EM_PARTS = 64;
constexpr int EM_WINDOW = 1 << 17;  // positions that a CTA's bitmap covers (16 KB)

// E: 4 (fp32) or 2 (bf16) bytes an element; a unit is 16 bytes of them (VEC) or a single one, as it lies and as fp32.
template <int E, bool VEC>
struct RawUnit {
    uint32_t w[VEC ? 4 : 1];
    __device__ __forceinline__ void take(const uint4& q) {
        w[0] = q.x;
        w[1] = q.y;
        w[2] = q.z;
        w[3] = q.w;
    }
    __device__ __forceinline__ void load(const void* row, int64_t u) {
        if constexpr (VEC) {
            take(ldg_stream(reinterpret_cast<const uint4*>(row) + u));
        } else if constexpr (E == 4) {
            w[0] = __ldg(static_cast<const uint32_t*>(row) + u);
        } else {
            w[0] = (uint32_t)__ldg(static_cast<const unsigned short*>(row) + u) << 16;
        }
    }
};
template <int E, bool VEC>
struct Unit {
    static constexpr int N = VEC ? 16 / E : 1;
    float v[N];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 0.0f;
    }
    __device__ __forceinline__ void add(const RawUnit<E, VEC>& o) {
        if constexpr (VEC && E == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] += __uint_as_float(o.w[j] << 16);
                v[2 * j + 1] += __uint_as_float(o.w[j] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] += __uint_as_float(o.w[j]);
        }
    }
    // each value times s, rounded to the element's type
    __device__ __forceinline__ void store(void* row, int64_t u, float s) const {
        if constexpr (VEC) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (E == 4) {
                    w[j] = __float_as_uint(v[j] * s);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j] * s, v[2 * j + 1] * s);
                    w[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            __stcs(reinterpret_cast<uint4*>(row) + u, make_uint4(w[0], w[1], w[2], w[3]));
        } else if constexpr (E == 4) {
            static_cast<float*>(row)[u] = v[0] * s;
        } else {
            static_cast<__nv_bfloat16*>(row)[u] = __float2bfloat16_rn(v[0] * s);
        }
    }
};

// The token of a position: -1 for padding and ids past the table.
__device__ __forceinline__ int64_t token_at(const int64_t* tokens, int64_t i, int64_t vocab, uint32_t* status) {
    const int64_t t = __ldg(tokens + i);
    if (t >= vocab) {
        if (status) atomicOr(status, B2S_STATUS_TOKEN_RANGE);
        return -1;
    }
    return t < 0 ? -1 : t;
}

// grid: a warp per row and part of U units, all in flight together.  U is the least that holds a row, up to 128 (131,072 x 768
// fp32 83 us against 98 with 64; 200,000 x 256 bf16 29.6 with 32 against 34 with 64 and 48 with 128), of unaligned rows 256
// elements (30001 x 1001 bf16 30 us; 64 with 64).
template <int E, bool VEC, int U>
__global__ void __launch_bounds__(EM_NT) embed_kernel(const int64_t* tokens, int64_t n, const void* table,
                                                      int64_t row_bytes, int64_t vocab, int64_t units, int64_t parts, float s,
                                                      void* out, uint32_t* status) {
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * (EM_NT / 32) + (threadIdx.x >> 5), i = w / parts, u0 = (w % parts) * U + lane;
    if (i >= n) return;
    const int64_t t = token_at(tokens, i, vocab, u0 == 0 ? status : nullptr);
    const unsigned char* src = static_cast<const unsigned char*>(table) + (t < 0 ? 0 : t) * row_bytes;
    unsigned char* dst = static_cast<unsigned char*>(out) + i * units * Unit<E, VEC>::N * E;
    RawUnit<E, VEC> q[U / 32];
#pragma unroll
    for (int j = 0; j < U / 32; ++j)
        if (t >= 0 && u0 + 32 * j < units) q[j].load(src, u0 + 32 * j);
#pragma unroll
    for (int j = 0; j < U / 32; ++j) {
        Unit<E, VEC> v;
        v.zero();
        if (t >= 0) v.add(q[j]);
        if (u0 + 32 * j < units) v.store(dst, u0 + 32 * j, t < 0 ? 1.0f : s);  // padding is +0 whatever the scale's sign
    }
}

// The same from a microscaled table: a unit is 8 elements, 4 bytes of codes.  U: 128 where that takes an aligned row at once
// (131,072 x 768 62.6 us against 72.6 with 64; 16000 x 1001 51 against 48), 64 of longer ones (2000 x 4096 7.5; 128: 7.8), 32 of
// short ones (100,000 x 256 22.0; 64: 23.5).
template <int U>
__global__ void __launch_bounds__(EM_NT) embed_mx_kernel(const int64_t* tokens, int64_t n, const uint8_t* codes,
                                                         const uint8_t* scales, int64_t vocab, int width, int64_t pieces, float s,
                                                         __nv_bfloat16* out, int vec, uint32_t* status) {
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31, units = (width + 7) / 8;
    const int64_t w = (int64_t)blockIdx.x * (EM_NT / 32) + (threadIdx.x >> 5), i = w / pieces;
    const int u0 = (int)(w % pieces) * U + lane;
    if (i >= n) return;
    const int64_t t = token_at(tokens, i, vocab, lane == 0 && u0 == 0 ? status : nullptr);
    const int64_t bytes = mx_row_bytes(width), tiles = mx_tiles(width);
    uint32_t c[U / 32];
    float f[U / 32];
#pragma unroll
    for (int j = 0; j < U / 32; ++j) {
        const int u = u0 + 32 * j;
        c[j] = 0;
        f[j] = 0.0f;
        if (t >= 0 && u < units) {
            c[j] = __ldg(reinterpret_cast<const uint32_t*>(codes + t * bytes) + u);
            f[j] = mx_scale(__ldg(scales + mx_scale_at(t, u >> 2, tiles)));
        }
    }
#pragma unroll
    for (int j = 0; j < U / 32; ++j) {
        const int u = u0 + 32 * j;
        if (u >= units) break;
        float v[8];
        mx_decode8(c[j], v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = t < 0 ? 0.0f : v[k] * f[j] * s;
        mx_store8(out + i * width + 8 * u, min(8, width - 8 * u), vec, v);
    }
}

// ------------------------------------------------------------------ gradient

// The workspace: words that start as zero, then the arrays that the kernels fill.
struct EmbedSort {
    int* count;    // [vocab] positions of an id
    int* bin;      // [bins] positions of 1 << shift ids
    int* arrived;  // [slots][parts] sums that are there, of those that are joined
    int* longs;    // how many parts the ids with more than EM_SHORT positions have
    int* total;    // positions that are not padding
    int2* long_id; // [2 n / EM_SHORT] which, and which part of its positions
    int* base;     // [vocab] where an id's positions start, sorted
    int* place;    // [n] among the id's positions in order of arrival; -1: none
    int* loose;    // [n] positions by id, in order of arrival
    int* order;    // [n] positions by id, ascending
    int* id;       // [n] their ids
    float* sums;   // [slots][width]: two for each chunk, of the id that came from the one before and of the last one, that goes on
    int slots, shift, bins, windows;
    int chunk;     // sorted positions that a warp sums, as a power of two: 8, 16 or 32
    // CTAs that put an id's positions in order, each in its share of the windows
    __device__ __forceinline__ int parts_of(int positions) const { return positions > EM_HUGE ? min(windows, EM_PARTS) : 1; }
};

// Zeros, as a kernel that starts under the end of the one before and lets the next one start (a memset does neither: the gradient
// of 30001 of 6562 x 768 36.4 us against 34.5, of 16 of 1000 x 256 8.2 against 6.6).
__global__ void __launch_bounds__(EM_NT) embed_clear_kernel(uint4* p, int64_t units) {
    pdl_wait_then_release();
    const int64_t step = (int64_t)gridDim.x * EM_NT;
    for (int64_t i = (int64_t)blockIdx.x * EM_NT + threadIdx.x; i < units; i += step) p[i] = make_uint4(0u, 0u, 0u, 0u);
}

// Counts per id and bin, an atomic for a warp's equal ids.  TABLE: a CTA's positions are counted in shared memory first, ids in a
// table (open addressing, never more than half full), so that an id or a bin that is much of the input costs an atomic a CTA: the
// gradient of 300,000 positions of 151,936 ids, 8 wide, takes 96 us against 125, a million Zipf-distributed 340 against 450, but
// 30001 of 6562 768 wide 30.9 against 28.8.
constexpr int EM_TABLE = 2 * EM_NT;
constexpr int EM_MANY = 1 << 16;  // positions from which on
template <bool TABLE>
__global__ void __launch_bounds__(EM_NT) embed_count_kernel(const int64_t* tokens, int n, int64_t vocab, EmbedSort e) {
    __shared__ int key[TABLE ? EM_TABLE : 1], num[TABLE ? EM_TABLE : 1], bin[TABLE ? EM_BINS : 1];
    const int tid = threadIdx.x, lane = tid & 31;
    if constexpr (TABLE) {
        for (int j = tid; j < EM_TABLE; j += EM_NT) {
            key[j] = -1;
            num[j] = 0;
        }
        for (int j = tid; j < e.bins; j += EM_NT) bin[j] = 0;
    }
    pdl_wait_then_release();
    const int i = blockIdx.x * EM_NT + tid;
    const int t = i < n ? (int)token_at(tokens, i, vocab, nullptr) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, t);
    const int leader = __ffs(same) - 1;
    const bool leads = t >= 0 && lane == leader;
    int at = 0;
    if constexpr (TABLE) {
        int slot = 0;
        bool first = false;  // of the CTA with this id
        __syncthreads();
        if (leads) {
            slot = (int)((uint32_t)t * 2654435761u >> 16) & (EM_TABLE - 1);
            for (;; slot = (slot + 1) & (EM_TABLE - 1)) {
                const int was = atomicCAS(&key[slot], -1, t);
                first = was == -1;
                if (first || was == t) break;
            }
            at = atomicAdd(&num[slot], __popc(same));
            atomicAdd(&bin[t >> e.shift], __popc(same));
        }
        __syncthreads();
        if (first) num[slot] = atomicAdd(e.count + t, num[slot]);
        for (int j = tid; j < e.bins; j += EM_NT)
            if (bin[j]) atomicAdd(e.bin + j, bin[j]);
        __syncthreads();
        if (leads) at += num[slot];
    } else {
        if (leads) at = atomicAdd(e.count + t, __popc(same));
        const uint32_t near = __match_any_sync(0xffffffffu, t < 0 ? -1 : t >> e.shift);
        if (t >= 0 && lane == __ffs(near) - 1) atomicAdd(e.bin + (t >> e.shift), __popc(near));
    }
    at = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1u));
    if (i < n) e.place[i] = t < 0 ? -1 : at;
}

// Exclusive prefix of v over the CTA's threads, and the sum.
__device__ __forceinline__ int em_scan(int v, int* total) {
    __shared__ int sums[EM_NT / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int at = incl - v, all = 0;
#pragma unroll
    for (int j = 0; j < EM_NT / 32; ++j) {
        if (j < warp) at += sums[j];
        all += sums[j];
    }
    __syncthreads();
    *total = all;
    return at;
}
// A CTA per bin: where its ids' positions start.
__global__ void __launch_bounds__(EM_NT) embed_scan_kernel(int64_t vocab, EmbedSort e) {
    pdl_wait_then_release();
    int mine = 0, start;
    for (int j = threadIdx.x; j < (int)blockIdx.x; j += EM_NT) mine += e.bin[j];
    em_scan(mine, &start);
    const int64_t first = (int64_t)blockIdx.x << e.shift, end = min(vocab, first + ((int64_t)1 << e.shift));
    for (int64_t v0 = first; v0 < end; v0 += 4 * EM_NT) {
        const int64_t v = v0 + 4 * threadIdx.x;  // count and base are padded to whole vectors
        int4 c = make_int4(0, 0, 0, 0);
        if (v < end) c = *reinterpret_cast<const int4*>(e.count + v);
        int all;
        const int at = start + em_scan(c.x + c.y + c.z + c.w, &all);
        if (v < end) *reinterpret_cast<int4*>(e.base + v) = make_int4(at, at + c.x, at + c.x + c.y, at + c.x + c.y + c.z);
        if (max(max(c.x, c.y), max(c.z, c.w)) > EM_SHORT) {  // in any order: each is put in order by itself
            const int k[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (k[j] <= EM_SHORT) continue;
                const int parts = e.parts_of(k[j]), f = atomicAdd(e.longs, parts);
                for (int p = 0; p < parts; ++p) e.long_id[f + p] = make_int2((int)v + j, p);
            }
        }
        start += all;
    }
    if ((int)blockIdx.x == e.bins - 1 && threadIdx.x == 0) *e.total = start;
}

__global__ void __launch_bounds__(EM_NT) embed_scatter_kernel(const int64_t* tokens, int n, EmbedSort e) {
    pdl_wait_then_release();
    const int i = blockIdx.x * EM_NT + threadIdx.x;
    if (i >= n || e.place[i] < 0) return;
    e.loose[e.base[tokens[i]] + e.place[i]] = i;
}

// All of that for up to EM_FEW positions in one launch: a position's place is how many come before it by (id, position), found by
// comparison with all, EM_RANK lanes a position (three launches instead of six: 1024 of 1000 x 256 12.4 us against 17.4, 2048 14.5
// against 17.2, 4096 20.8 against 18.5, but of 30,000 x 2048 33.6 against 37.6; with 8 lanes and an id at a time 14.4, 16.4, 22.3).
constexpr int EM_FEW = 4096;
constexpr int EM_RANK = 16;
__global__ void __launch_bounds__(EM_NT) embed_rank_kernel(const int64_t* tokens, int n, int64_t vocab, EmbedSort e) {
    __shared__ __align__(16) int ids[EM_FEW];
    pdl_wait_then_release();
    int real = 0;
    for (int j = threadIdx.x; j < n; j += EM_NT) {
        const int t = (int)token_at(tokens, j, vocab, nullptr);
        ids[j] = t < 0 ? 0x7fffffff : t;  // behind all others, equal to none
        real += t >= 0;
    }
    for (int j = n + threadIdx.x; j < (n + 3) / 4 * 4; j += EM_NT) ids[j] = 0x7fffffff;
    int all;
    em_scan(real, &all);
    if (blockIdx.x == 0 && threadIdx.x == 0) *e.total = all;
    const int i = blockIdx.x * (EM_NT / EM_RANK) + threadIdx.x / EM_RANK, t = i < n ? ids[i] : 0x7fffffff;
    int before = 0, lower = 0, same = 0;
#pragma unroll 4
    for (int j = 4 * (threadIdx.x % EM_RANK); j < n; j += 4 * EM_RANK) {
        const int4 q = *reinterpret_cast<const int4*>(ids + j);
        const int o[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            lower += o[k] < t;
            same += o[k] == t;
            before += o[k] == t && j + k < i;
        }
    }
#pragma unroll
    for (int o = 1; o < EM_RANK; o <<= 1) {
        lower += __shfl_xor_sync(0xffffffffu, lower, o);
        same += __shfl_xor_sync(0xffffffffu, same, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (threadIdx.x % EM_RANK || t == 0x7fffffff) return;
    e.order[lower + before] = i;
    e.id[lower + before] = t;
    if (before == 0) {
        e.base[t] = lower;
        e.count[t] = same;
    }
}

// Warp w of those that write zeros for the ids that do not occur: EM_ZERO bytes of a row each, `zeros` of them a row.
constexpr int EM_ZERO = 8192;
__device__ __forceinline__ void em_zero(int64_t w, int64_t vocab, int64_t row_bytes, int64_t zeros, unsigned char* out, int e_bytes,
                                        const EmbedSort& e) {
    const int lane = threadIdx.x & 31;
    const int64_t v = w / zeros;
    if (v >= vocab || e.count[v]) return;
    unsigned char* p = out + v * row_bytes + w % zeros * EM_ZERO;
    unsigned char* end = out + v * row_bytes + min(row_bytes, (w % zeros + 1) * EM_ZERO);
    unsigned char* a = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p) + 15) & ~(uintptr_t)15);
    unsigned char* z = reinterpret_cast<unsigned char*>(reinterpret_cast<uintptr_t>(end) & ~(uintptr_t)15);
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    if (a < z) {
#pragma unroll 4
        for (unsigned char* q = a + 16 * lane; q < z; q += 512) __stcs(reinterpret_cast<uint4*>(q), none);
    } else {
        a = z = end;
    }
    // the ends that are not whole vectors, in elements
    for (unsigned char* q = p + (int64_t)lane * e_bytes; q < a; q += 32 * e_bytes)
        if (e_bytes == 4) *reinterpret_cast<uint32_t*>(q) = 0;
        else *reinterpret_cast<unsigned short*>(q) = 0;
    for (unsigned char* q = z + (int64_t)lane * e_bytes; q < end; q += 32 * e_bytes)
        if (e_bytes == 4) *reinterpret_cast<uint32_t*>(q) = 0;
        else *reinterpret_cast<unsigned short*>(q) = 0;
}

// The first `longs` CTAs put the positions of the ids with more than EM_SHORT of them in ascending order.  Where one bitmap covers
// all positions they are marked in it and read back.  Of longer inputs, up to EM_MID by comparison in shared memory, more by bitmaps
// of EM_WINDOW positions, each behind as many as come before it; of an id with more than EM_HUGE several CTAs each do some of the
// windows (300,000 equal ids 8 wide 226 us against 483 by one CTA; a million Zipf-distributed 340 against 425, and 732 with
// bitmaps for up to EM_MID too; with one bitmap comparisons cost 30001 of 6562 40 against 37).  The next `orders` CTAs do the
// others', a place's rank by comparison with the id's other places.  The last ones write zeros for the ids that do not occur.
__global__ void __launch_bounds__(EM_NT) embed_order_kernel(const int64_t* tokens, int n, int64_t vocab, int64_t row_bytes,
                                                            int64_t zeros, int longs, int orders, unsigned char* out, int e_bytes,
                                                            EmbedSort e) {
    __shared__ __align__(16) uint32_t bits[EM_WINDOW / 32];
    pdl_wait_then_release();
    const int tid = threadIdx.x, warp = tid >> 5;
    if ((int)blockIdx.x >= longs + orders) {
        em_zero((int64_t)(blockIdx.x - longs - orders) * (EM_NT / 32) + warp, vocab, row_bytes, zeros, out, e_bytes, e);
        return;
    }
    if ((int)blockIdx.x >= longs) {
        const int64_t k = (int64_t)(blockIdx.x - longs) * EM_NT + tid;
        if (k >= *e.total) return;
        const int i = e.loose[k], t = (int)tokens[i], c = e.count[t], b = e.base[t];
        e.id[k] = t;
        if (c > EM_SHORT) return;
        int rank = 0;
#pragma unroll 16
        for (int j = 0; j < c; ++j) rank += e.loose[b + j] < i;
        e.order[b + rank] = i;
        return;
    }
    for (int f = blockIdx.x; f < *e.longs; f += longs) {
        const int t = e.long_id[f].x, c = e.count[t], b = e.base[t], parts = e.parts_of(c);
        const int* loose = e.loose + b;
        if (c <= EM_MID && e.windows > 1) {
            int* at = reinterpret_cast<int*>(bits);
            for (int j = tid; j < EM_MID; j += EM_NT) at[j] = j < c ? loose[j] : 0x7fffffff;
            __syncthreads();
            for (int j = tid; j < c; j += EM_NT) {
                const int i = at[j];
                int rank = 0;
#pragma unroll 4
                for (int k = 0; k < c; k += 4) {
                    const int4 q = *reinterpret_cast<const int4*>(at + k);
                    rank += (q.x < i) + (q.y < i) + (q.z < i) + (q.w < i);
                }
                e.order[b + rank] = i;
            }
            __syncthreads();
            continue;
        }
        for (int w = e.long_id[f].y; w < e.windows; w += parts) {
            const int w0 = w * EM_WINDOW, held = min(EM_WINDOW, n - w0);
            const int words = (held + 31) / 32, per = (words + EM_NT - 1) / EM_NT;
            for (int j = tid; j < words; j += EM_NT) bits[j] = 0;
            __syncthreads();
            int before = 0, mine = 0, start, all;
#pragma unroll 8
            for (int j = tid; j < c; j += EM_NT) {
                const int i = loose[j] - w0;
                before += i < 0;
                if (i >= 0 && i < held) atomicOr(&bits[i >> 5], 1u << (i & 31));
            }
            __syncthreads();
            if (e.windows > 1) em_scan(before, &start);
            else start = 0;
            for (int j = tid * per; j < min(words, (tid + 1) * per); ++j) mine += __popc(bits[j]);
            int at = b + start + em_scan(mine, &all);
            for (int j = tid * per; j < min(words, (tid + 1) * per); ++j)
                for (uint32_t m = bits[j]; m; m &= m - 1) e.order[at++] = w0 + 32 * j + __ffs(m) - 1;
            __syncthreads();
            if (start + all == c) break;
        }
    }
}

// A warp per chunk and part of a row.  Whole 16-byte units come by asynchronous copies, EM_AHEAD rows ahead of the sums and each
// lane its own: what bounds this is bytes in flight, and loads to registers, four rows at a time, left too few (30001 x 768 fp32
// of 6562 ids, with the sort, 45 us against 38.5, 32768 x 1024 bf16 of 20000 49 against 40; 8 rows ahead 40 and 46).  CTAs of two
// warps: their shares end more evenly than four warps' (38.5 against 42).  CTAs from `sums` on write zeros (em_zero).
constexpr int EM_SUM_NT = 64;
constexpr int EM_ROWS = 4;    // rows taken together
constexpr int EM_AHEAD = 12;  // rows in flight
template <int E, bool VEC>
__global__ void __launch_bounds__(EM_SUM_NT, 8) embed_sum_kernel(const void* grad, int64_t row_bytes, int64_t units, int parts,
                                                                 float s, void* out, EmbedSort e, unsigned sums, int64_t vocab,
                                                                 int64_t zeros) {
    constexpr int N = Unit<E, VEC>::N, W = em_units(VEC, E) / 32;
    pdl_wait_then_release();
    if (blockIdx.x >= sums) {
        em_zero((int64_t)(blockIdx.x - sums) * (EM_SUM_NT / 32) + (threadIdx.x >> 5), vocab, units * N * E, zeros,
                static_cast<unsigned char*>(out), E, e);
        return;
    }
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * (EM_SUM_NT / 32) + (threadIdx.x >> 5), chunk = w / parts;
    const int part = (int)(w % parts), total = *e.total;
    const int64_t u0 = (int64_t)part * em_units(VEC, E) + lane, width = units * N, k0 = chunk << e.chunk;
    if (k0 >= total) return;
    const int held = (int)min((int64_t)1 << e.chunk, total - k0);
    const int pos = lane < held ? e.order[k0 + lane] : 0, id = lane < held ? e.id[k0 + lane] : -1;
    const int before = k0 ? e.id[k0 - 1] : -1, after = k0 + held < total ? e.id[k0 + held] : -1;
    const int next = __shfl_down_sync(0xffffffffu, id, 1);
    const uint32_t ends = __ballot_sync(0xffffffffu, lane < held && (lane == held - 1 || next != id));  // last rows of ids
    const int first_id = __shfl_sync(0xffffffffu, id, 0), last_id = __shfl_sync(0xffffffffu, id, held - 1);
    const bool from = first_id == before, on = last_id == after;  // an id from the chunk before, one that goes on
    Unit<E, VEC> sum[W];
#pragma unroll
    for (int j = 0; j < W; ++j) sum[j].zero();
    auto write = [&](int64_t to) {
        unsigned char* dst = static_cast<unsigned char*>(out) + to * width * E;
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (u0 + 32 * j < units) sum[j].store(dst, u0 + 32 * j, s);
    };
    auto keep = [&](int64_t slot) {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (u0 + 32 * j < units) {
                float* q = e.sums + slot * width + (u0 + 32 * j) * N;
                if constexpr (VEC) {
#pragma unroll
                    for (int k = 0; k < N; k += 4)
                        __stcg(reinterpret_cast<float4*>(q + k),
                               make_float4(sum[j].v[k], sum[j].v[k + 1], sum[j].v[k + 2], sum[j].v[k + 3]));
                } else {
                    __stcg(q, sum[j].v[0]);
                }
            }
    };
    int start = 0;  // of the id being summed
    RawUnit<E, VEC> g[EM_ROWS][W];
    auto row = [&](int k) { return static_cast<const unsigned char*>(grad) + __shfl_sync(0xffffffffu, pos, k & 31) * row_bytes; };
    auto add_rows = [&](int k) {
#pragma unroll
        for (int r = 0; r < EM_ROWS; ++r) {
            if (k + r >= held) break;
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (u0 + 32 * j < units) sum[j].add(g[r][j]);
            if (ends >> (k + r) & 1) {
                const bool goes = on && k + r == held - 1, came = from && start == 0;
                if (goes || came) keep(2 * chunk + (came ? 0 : 1));
                else write(__shfl_sync(0xffffffffu, id, k + r));
#pragma unroll
                for (int j = 0; j < W; ++j) sum[j].zero();
                start = k + r + 1;
            }
        }
    };
    if constexpr (VEC) {
        __shared__ uint4 ring[EM_SUM_NT / 32][EM_AHEAD][EM_UNITS];
        uint4(*mine)[EM_UNITS] = ring[threadIdx.x >> 5];
        auto fetch = [&](int k, int slot) {
#pragma unroll
            for (int r = 0; r < EM_ROWS; ++r) {
                const uint4* src = reinterpret_cast<const uint4*>(row(k + r));
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (k + r < held && u0 + 32 * j < units) cp_async16(&mine[slot + r][32 * j + lane], src + u0 + 32 * j);
            }
            cp_async_commit();
        };
#pragma unroll
        for (int k = 0; k < EM_AHEAD; k += EM_ROWS) fetch(k, k);
        int slot = 0;
#pragma unroll 1
        for (int k = 0; k < held; k += EM_ROWS) {
            cp_async_wait<EM_AHEAD / EM_ROWS - 1>();
#pragma unroll
            for (int r = 0; r < EM_ROWS; ++r)
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (k + r < held && u0 + 32 * j < units) g[r][j].take(mine[slot + r][32 * j + lane]);
            __syncwarp();  // read, before the next rows are written there
            fetch(k + EM_AHEAD, slot);
            slot = slot + EM_ROWS == EM_AHEAD ? 0 : slot + EM_ROWS;
            add_rows(k);
        }
    } else {
#pragma unroll 1
        for (int k = 0; k < held; k += EM_ROWS) {
#pragma unroll
            for (int r = 0; r < EM_ROWS; ++r) {
                const unsigned char* src = row(k + r);
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (k + r < held && u0 + 32 * j < units) g[r][j].load(src, u0 + 32 * j);
            }
            add_rows(k);
        }
    }
    if (!from && !on) return;
    auto last = [&](int64_t counter, int of) {  // whether this warp is the last of `of` to get here
        __threadfence();
        __syncwarp();
        int there = 0;
        if (lane == 0) there = atomicAdd(e.arrived + counter * parts + part, 1);
        there = __shfl_sync(0xffffffffu, there, 0);
        __threadfence();
        return there == of - 1;
    };
    // An id's sums lie with its chunks from c0 on, in the first one's second place and the others' first.  They are added in
    // order, 2^EM_JOIN neighbours at a time, then as many of those sums, and so on, so that which warp it is that completes
    // them does not matter.  A sum replaces its first part; level l counts arrivals at its first part's l-th neighbour.
#pragma unroll 1
    for (int both = 0; both < 2; ++both) {
        if (both ? !on || (from && first_id == last_id) : !from) continue;  // a chunk of one id has one sum
        const int t = both ? last_id : first_id, b = e.base[t], c0 = b >> e.chunk, of = ((b + e.count[t] - 1) >> e.chunk) - c0 + 1;
        auto slot = [&](int j) { return 2 * (int64_t)(c0 + j) + (j ? 0 : 1); };
        auto join = [&](int j0, int count, int apart) {
#pragma unroll
            for (int j = 0; j < W; ++j) sum[j].zero();
#pragma unroll 4
            for (int k = 0; k < count; ++k) {
                const float* q = e.sums + slot(j0 + k * apart) * width;
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (u0 + 32 * j < units) {
                        if constexpr (VEC) {
#pragma unroll
                            for (int c = 0; c < N; c += 4) {
                                const float4 v = __ldcg(reinterpret_cast<const float4*>(q + (u0 + 32 * j) * N + c));
                                sum[j].v[c] += v.x;
                                sum[j].v[c + 1] += v.y;
                                sum[j].v[c + 2] += v.z;
                                sum[j].v[c + 3] += v.w;
                            }
                        } else {
                            sum[j].v[0] += __ldcg(q + u0 + 32 * j);
                        }
                    }
            }
        };
        bool whole = true;
        for (int level = 0, span = 0; (of - 1) >> span; ++level, span += EM_JOIN) {  // 2^span chunks in a sum
            const int group = ((int)chunk - c0) >> (span + EM_JOIN) << (span + EM_JOIN);
            const int in = min(1 << EM_JOIN, ((of - group - 1) >> span) + 1);
            if (in == 1) continue;  // the last sum of its level, as it is
            if (!last(slot(group + level), in)) {
                whole = false;
                break;
            }
            join(group, in, 1 << span);
            if ((of - 1) >> (span + EM_JOIN)) keep(slot(group));
        }
        if (whole) write(t);
    }
}

int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
int64_t parts_of(int64_t units, bool vec, int e) { return (units + em_units(vec, e) - 1) / em_units(vec, e); }
// The workspace's arrays, and its bytes, `zeroed` of them to be zero; the parts of a row are those of single elements, where rows
// may be unaligned.
int64_t embed_layout(int64_t n, int64_t vocab, int64_t width, unsigned char* at, EmbedSort* e, int64_t* zeroed) {
    int64_t used = 0;
    auto take = [&](int64_t bytes) {
        unsigned char* p = at ? at + used : nullptr;
        used += up(bytes, 256);
        return p;
    };
    // 32 positions a warp, fewer where there would be few warps (2048 x 768 of 6562 ids: 26 against 21 us)
    const int64_t shares = n * ((width + 511) / 512);
    e->chunk = shares <= 1 << 13 ? 3 : shares <= 1 << 15 ? 4 : 5;
    e->slots = (int)(2 * (((n - 1) >> e->chunk) + 1));
    e->shift = 10;  // bins of 1024 ids, or as many as make EM_BINS
    while ((vocab - 1) >> e->shift >= EM_BINS) ++e->shift;
    e->bins = (int)(((vocab - 1) >> e->shift) + 1);
    e->windows = (int)((n - 1) / EM_WINDOW + 1);
    e->count = reinterpret_cast<int*>(take(up(vocab, 4) * 4));
    e->bin = reinterpret_cast<int*>(take((int64_t)e->bins * 4));
    e->arrived = reinterpret_cast<int*>(take((int64_t)e->slots * parts_of(width, false, 2) * 4));
    e->longs = reinterpret_cast<int*>(take(4));
    *zeroed = used;
    e->total = reinterpret_cast<int*>(take(4));
    e->long_id = reinterpret_cast<int2*>(take(2 * (n / EM_SHORT) * 8));
    e->base = reinterpret_cast<int*>(take(up(vocab, 4) * 4));
    e->place = reinterpret_cast<int*>(take(n * 4));
    e->loose = reinterpret_cast<int*>(take(n * 4));
    e->order = reinterpret_cast<int*>(take(n * 4));
    e->id = reinterpret_cast<int*>(take(n * 4));
    e->sums = reinterpret_cast<float*>(take((int64_t)e->slots * width * 4));
    return used;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool embed_sizes_ok(int64_t n, int64_t vocab, int64_t width) {
    return n <= LP_MAX_SIZE && vocab <= LP_MAX_SIZE && width <= LP_MAX_SIZE;
}
// Blocks of a launch with `warps` warps, 0 where those are more than a grid holds.
unsigned blocks_of(int64_t warps, int threads = EM_NT) {
    const int64_t each = threads / 32, b = (warps + each - 1) / each;
    return b > 0x7fffffff ? 0u : (unsigned)b;
}

}  // namespace
}  // namespace b2s

extern "C" {

int b2s_embedding(const int64_t* tokens, int32_t n, const void* table, int32_t dtype, int32_t vocab, int32_t width,
                  int64_t row_stride, float scale, void* out, uint32_t* status, void* stream) {
    using namespace b2s;
    if (n < 0 || vocab < 1 || width < 1 || row_stride < width || (dtype != B2S_DTYPE_F32 && dtype != B2S_DTYPE_BF16) ||
        !(scale - scale == 0.0f))
        return B2S_ERR_INVALID;
    if (!embed_sizes_ok(n, vocab, width)) return B2S_ERR_UNSUPPORTED;
    if (n == 0) return B2S_OK;
    const int e = dtype == B2S_DTYPE_F32 ? 4 : 2;
    if (!tokens || !table || !out || ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out)) & (e - 1)))
        return B2S_ERR_INVALID;
    const bool vec = aligned16(table) && aligned16(out) && (int64_t)width * e % 16 == 0 && row_stride * e % 16 == 0;
    const int64_t units = vec ? (int64_t)width * e / 16 : width;
    const int64_t each = !vec ? EM_ELEMENTS : units <= 32 ? 32 : units <= 64 ? 64 : 128;
    const int64_t pieces = (units + each - 1) / each;
    const unsigned blocks = blocks_of(n * pieces);
    if (!blocks) return B2S_ERR_UNSUPPORTED;
    auto go = [&](auto kernel) {
        return launch_pdl(kernel, dim3(blocks), EM_NT, 0, stream, tokens, (int64_t)n, table, row_stride * e, (int64_t)vocab,
                          units, pieces, scale, out, status);
    };
    auto typed = [&](auto bytes) {
        constexpr int E = decltype(bytes)::value;
        if (!vec) return go(embed_kernel<E, false, EM_ELEMENTS>);
        return each == 32   ? go(embed_kernel<E, true, 32>)
               : each == 64 ? go(embed_kernel<E, true, 64>)
                            : go(embed_kernel<E, true, 128>);
    };
    const cudaError_t r = e == 4 ? typed(std::integral_constant<int, 4>()) : typed(std::integral_constant<int, 2>());
    return r == cudaSuccess ? B2S_OK : cuda_fail(r);
}

int b2s_embedding_mx(const int64_t* tokens, int32_t n, const void* codes, const void* scales, int32_t vocab, int32_t width,
                     float scale, void* out, uint32_t* status, void* stream) {
    using namespace b2s;
    if (n < 0 || vocab < 1 || width < 1 || !(scale - scale == 0.0f)) return B2S_ERR_INVALID;
    if (!embed_sizes_ok(n, vocab, width)) return B2S_ERR_UNSUPPORTED;
    if (n == 0) return B2S_OK;
    if (!tokens || !codes || !scales || !out || !aligned16(codes) || !aligned16(scales) || (reinterpret_cast<uintptr_t>(out) & 1))
        return B2S_ERR_INVALID;
    const bool vec = aligned16(out) && width % 8 == 0;
    const int64_t units = (width + 7) / 8, each = units <= 32 ? 32 : vec && units > 64 && units <= 128 ? 128 : 64;
    const int64_t pieces = (units + each - 1) / each;
    const unsigned blocks = blocks_of(n * pieces);
    if (!blocks) return B2S_ERR_UNSUPPORTED;
    auto go = [&](auto kernel) {
        return launch_pdl(kernel, dim3(blocks), EM_NT, 0, stream, tokens, (int64_t)n, static_cast<const uint8_t*>(codes),
                          static_cast<const uint8_t*>(scales), (int64_t)vocab, (int)width, pieces, scale,
                          static_cast<__nv_bfloat16*>(out), (int)vec, status);
    };
    const cudaError_t r = each == 32 ? go(embed_mx_kernel<32>) : each == 64 ? go(embed_mx_kernel<64>) : go(embed_mx_kernel<128>);
    return r == cudaSuccess ? B2S_OK : cuda_fail(r);
}

int b2s_embedding_grad_workspace(int32_t n, int32_t vocab, int32_t width, int64_t* bytes) {
    using namespace b2s;
    if (n < 0 || vocab < 1 || width < 1 || !bytes) return B2S_ERR_INVALID;
    EmbedSort e;
    int64_t zeroed;
    *bytes = n ? embed_layout(n, vocab, width, nullptr, &e, &zeroed) : 0;
    return B2S_OK;
}

int b2s_embedding_grad(const int64_t* tokens, int32_t n, const void* grad_out, int64_t grad_row_stride, int32_t dtype,
                       int32_t vocab, int32_t width, float scale, void* grad_table, void* workspace, int64_t workspace_bytes,
                       void* stream) {
    using namespace b2s;
    if (n < 0 || vocab < 1 || width < 1 || (dtype != B2S_DTYPE_F32 && dtype != B2S_DTYPE_BF16) || !(scale - scale == 0.0f) ||
        !grad_table)
        return B2S_ERR_INVALID;
    if (!embed_sizes_ok(n, vocab, width)) return B2S_ERR_UNSUPPORTED;
    const int e = dtype == B2S_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(grad_table) & (e - 1)) return B2S_ERR_INVALID;
    if (n == 0) {
        const cudaError_t r = cudaMemsetAsync(grad_table, 0, (size_t)vocab * width * e, (cudaStream_t)stream);
        return r == cudaSuccess ? B2S_OK : cuda_fail(r);
    }
    EmbedSort s;
    int64_t zeroed;
    if (!tokens || !grad_out || grad_row_stride < width || (reinterpret_cast<uintptr_t>(grad_out) & (e - 1)) || !workspace ||
        !aligned16(workspace) ||
        workspace_bytes < embed_layout(n, vocab, width, static_cast<unsigned char*>(workspace), &s, &zeroed))
        return B2S_ERR_INVALID;
    const bool vec = aligned16(grad_out) && aligned16(grad_table) && (int64_t)width * e % 16 == 0 && grad_row_stride * e % 16 == 0;
    const int64_t units = vec ? (int64_t)width * e / 16 : width, parts = parts_of(units, vec, e);
    const int64_t row_bytes = (int64_t)width * e, zeros = (row_bytes + EM_ZERO - 1) / EM_ZERO;
    const unsigned per = (unsigned)(((int64_t)n + EM_NT - 1) / EM_NT);
    const unsigned blocks = blocks_of((((int64_t)n - 1 >> s.chunk) + 1) * parts, EM_SUM_NT), zero_blocks = blocks_of(vocab * zeros);
    if (!blocks || !zero_blocks || (int64_t)zero_blocks + per + 1024 > 0x7fffffff) return B2S_ERR_UNSUPPORTED;
    const bool few = n <= EM_FEW;
    const unsigned late = few ? blocks_of(vocab * zeros, EM_SUM_NT) : 0u;  // CTAs of the last launch that write zeros then
    if (few && (!late || (int64_t)late + blocks > 0x7fffffff)) return B2S_ERR_UNSUPPORTED;
    const int64_t clear = zeroed / 16, clears = (clear + EM_NT - 1) / EM_NT, room = 8 * (int64_t)sms_here();
    cudaError_t r = launch_pdl(embed_clear_kernel, dim3((unsigned)(clears < room ? clears : room)), EM_NT, 0, stream,
                               static_cast<uint4*>(workspace), clear);
    if (few) {
        if (r == cudaSuccess)
            r = launch_pdl(embed_rank_kernel, dim3((unsigned)((n + EM_NT / EM_RANK - 1) / (EM_NT / EM_RANK))), EM_NT, 0, stream,
                           tokens, (int)n, (int64_t)vocab, s);
    } else {
        if (r == cudaSuccess)
            r = n < EM_MANY ? launch_pdl(embed_count_kernel<false>, dim3(per), EM_NT, 0, stream, tokens, (int)n, (int64_t)vocab, s)
                            : launch_pdl(embed_count_kernel<true>, dim3(per), EM_NT, 0, stream, tokens, (int)n, (int64_t)vocab, s);
        if (r == cudaSuccess) r = launch_pdl(embed_scan_kernel, dim3((unsigned)s.bins), EM_NT, 0, stream, (int64_t)vocab, s);
        if (r == cudaSuccess) r = launch_pdl(embed_scatter_kernel, dim3(per), EM_NT, 0, stream, tokens, (int)n, s);
    }
    if (r == cudaSuccess && !few) {
        // four CTAs an SM for ids with many positions (two: 524,288 of 6562 x 768 Zipf-distributed 356 us against 310)
        const unsigned most = 4 * (unsigned)sms_here(), longs = 2 * (n / EM_SHORT) < (int)most ? 2 * (n / EM_SHORT) : most;
        r = launch_pdl(embed_order_kernel, dim3(zero_blocks + per + longs), EM_NT, 0, stream, tokens, (int)n, (int64_t)vocab,
                       row_bytes, zeros, (int)longs, (int)per, static_cast<unsigned char*>(grad_table), e, s);
    }
    if (r != cudaSuccess) return cuda_fail(r);
    auto sum = [&](auto kernel) {
        return launch_pdl(kernel, dim3(blocks + late), EM_SUM_NT, 0, stream, grad_out, grad_row_stride * e, units, (int)parts,
                          scale, grad_table, s, blocks, (int64_t)vocab, zeros);
    };
    r = e == 4 ? (vec ? sum(embed_sum_kernel<4, true>) : sum(embed_sum_kernel<4, false>))
               : (vec ? sum(embed_sum_kernel<2, true>) : sum(embed_sum_kernel<2, false>));
    return r == cudaSuccess ? B2S_OK : cuda_fail(r);
}

}  // extern "C"
