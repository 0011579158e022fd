// The embedding lookup with a scale, out[i] = s T[t_i], and its gradient dT[v] = s sum of g[i] over the positions i with
// t_i = v, in ascending order of i.  Ids below 0 are padding: zeros, and no part in the gradient.  Ids past the table are
// taken as padding too and set B2S_STATUS_TOKEN_RANGE.  No counterpart in the reference, whose models call torch's own.
//
// Forward: a copy of rows.  A warp takes a piece of one row, 16 bytes a lane and four loads in flight.  From a
// microscaled table a lane decodes 8 elements.
//
// Gradient: the whole table's gradient is written once, so what bounds it is that write (1.24 GB for the Thinker's table)
// and one read of the rows' gradients.  The positions are sorted by id without a sort of keys: a count per id (the atomic's
// old value is the position's place among its id's, in order of arrival), ranges handed out to the ids that occur, and
// then each id's positions put in ascending order, so that sums do not depend on who arrived first.  An id's positions
// are summed in pieces of EM_PIECE, in order, in fp32; an id with several pieces leaves their sums in a workspace, and a
// last kernel adds them in order.
#include <string.h>

#include "../../include/b2s_sampler.h"
#include "b2s_device.cuh"
#include "b2s_launch.cuh"
#include "b2s_logprobs.cuh"
#include "b2s_mx.cuh"

namespace b2s {

int cuda_fail(cudaError_t e);

namespace {

constexpr int EM_NT = 256;
constexpr int EM_PIECE = 32;   // positions summed by one warp
constexpr int EM_UNITS = 128;  // 16-byte units (or elements) of a row that a warp takes
constexpr int EM_WINDOW = 1 << 17;  // positions that a CTA's bitmap covers (16 KB)

// E: 4 (fp32) or 2 (bf16) bytes an element; a unit is 16 bytes of them (VEC) or a single one.
template <int E, bool VEC>
struct Unit {
    static constexpr int N = VEC ? 16 / E : 1;
    float v[N];
    __device__ __forceinline__ void load(const void* row, int64_t u) {
        if constexpr (VEC) {
            const uint4 q = ldg_stream(reinterpret_cast<const uint4*>(row) + u);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (E == 4) {
                    v[j] = __uint_as_float(w[j]);
                } else {
                    v[2 * j] = __uint_as_float(w[j] << 16);
                    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                }
            }
        } else if constexpr (E == 4) {
            v[0] = __ldg(static_cast<const float*>(row) + u);
        } else {
            v[0] = bf16_bits_to_f(__ldg(static_cast<const unsigned short*>(row) + u));
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
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 0.0f;
    }
    __device__ __forceinline__ void add(const Unit& o) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += o.v[j];
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

// grid: a warp per row and piece of EM_UNITS units
template <int E, bool VEC>
__global__ void __launch_bounds__(EM_NT) embed_kernel(const int64_t* tokens, int64_t n, const void* table,
                                                      int64_t row_bytes, int64_t vocab, int64_t units, int64_t pieces, float s,
                                                      void* out, uint32_t* status) {
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * (EM_NT / 32) + (threadIdx.x >> 5), i = w / pieces, u0 = (w % pieces) * EM_UNITS + lane;
    if (i >= n) return;
    const int64_t t = token_at(tokens, i, vocab, lane == 0 && u0 == 0 ? status : nullptr);
    const unsigned char* src = static_cast<const unsigned char*>(table) + (t < 0 ? 0 : t) * row_bytes;
    unsigned char* dst = static_cast<unsigned char*>(out) + i * units * Unit<E, VEC>::N * E;
    Unit<E, VEC> v[EM_UNITS / 32];
#pragma unroll
    for (int j = 0; j < EM_UNITS / 32; ++j) {
        v[j].zero();
        if (t >= 0 && u0 + 32 * j < units) v[j].load(src, u0 + 32 * j);
    }
#pragma unroll
    for (int j = 0; j < EM_UNITS / 32; ++j)
        if (u0 + 32 * j < units) v[j].store(dst, u0 + 32 * j, s);
}

// The same from a microscaled table: a unit is 8 elements, 4 bytes of codes.
__global__ void __launch_bounds__(EM_NT) embed_mx_kernel(const int64_t* tokens, int64_t n, const uint8_t* codes,
                                                         const uint8_t* scales, int64_t vocab, int width, int64_t pieces, float s,
                                                         __nv_bfloat16* out, int vec, uint32_t* status) {
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31, units = (width + 7) / 8;
    const int64_t w = (int64_t)blockIdx.x * (EM_NT / 32) + (threadIdx.x >> 5), i = w / pieces;
    const int u0 = (int)(w % pieces) * EM_UNITS + lane;
    if (i >= n) return;
    const int64_t t = token_at(tokens, i, vocab, lane == 0 && u0 == 0 ? status : nullptr);
    const int64_t bytes = mx_row_bytes(width), tiles = mx_tiles(width);
    uint32_t c[EM_UNITS / 32];
    float f[EM_UNITS / 32];
#pragma unroll
    for (int j = 0; j < EM_UNITS / 32; ++j) {
        const int u = u0 + 32 * j;
        c[j] = 0;
        f[j] = 0.0f;
        if (t >= 0 && u < units) {
            c[j] = __ldg(reinterpret_cast<const uint32_t*>(codes + t * bytes) + u);
            f[j] = mx_scale(__ldg(scales + mx_scale_at(t, u >> 2, tiles)));
        }
    }
#pragma unroll
    for (int j = 0; j < EM_UNITS / 32; ++j) {
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

// The words that start as zero, then the arrays that the kernels fill.
struct EmbedSort {
    int* next;    // [4]: places, pieces, ids with several pieces, their sums
    int* count;   // [vocab] positions of an id
    int* base;    // [vocab] where they start, for the ids that occur
    int* place;   // [n] among the id's positions in order of arrival; -1: none
    int* loose;   // [n] positions by id, in order of arrival
    int* order;   // [n] positions by id, ascending
    int4* piece;  // [n] (id, start, length, sum's place or -1)
    int4* split;  // [n / EM_PIECE + 1] (id, first sum, sums)
    float* sums;  // [2 n / EM_PIECE][width]
};

__global__ void __launch_bounds__(EM_NT) embed_count_kernel(const int64_t* tokens, int n, int64_t vocab, EmbedSort e) {
    pdl_wait_then_release();
    const int i = blockIdx.x * EM_NT + threadIdx.x, lane = threadIdx.x & 31;
    const int t = i < n ? (int)token_at(tokens, i, vocab, nullptr) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, t);  // one atomic for a warp's equal ids
    const int leader = __ffs(same) - 1;
    int at = 0;
    if (t >= 0 && lane == leader) at = atomicAdd(e.count + t, __popc(same));
    at = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1u));
    if (i < n) e.place[i] = t < 0 ? -1 : at;
}

// The first arrival of each id takes a range of places and its pieces; which range an id gets does not matter.
__global__ void __launch_bounds__(EM_NT) embed_range_kernel(const int64_t* tokens, int n, EmbedSort e) {
    pdl_wait_then_release();
    const int i = blockIdx.x * EM_NT + threadIdx.x, lane = threadIdx.x & 31;
    const bool first = i < n && e.place[i] == 0;
    const int t = first ? (int)tokens[i] : 0, c = first ? e.count[t] : 0, p = (c + EM_PIECE - 1) / EM_PIECE;
    const int s = p > 1 ? p : 0;
    auto take = [&](int k, int want) {  // a warp's wants from a counter with one atomic
        int incl = want;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += u;
        }
        int at = 0;
        if (lane == 31 && incl) at = atomicAdd(e.next + k, incl);
        return __shfl_sync(0xffffffffu, at, 31) + incl - want;
    };
    const int base = take(0, c), piece = take(1, p), split = take(2, s ? 1 : 0), sum = take(3, s);
    if (first) e.base[t] = base;
    if (s) e.split[split] = make_int4(t, sum, s, 0);
    uint32_t todo = __ballot_sync(0xffffffffu, first);
    if (first && p == 1) e.piece[piece] = make_int4(t, base, c, -1);
    for (todo = __ballot_sync(0xffffffffu, p > 1); todo; todo &= todo - 1) {  // long ones by the whole warp
        const int l = __ffs(todo) - 1;
        const int lt = __shfl_sync(0xffffffffu, t, l), lb = __shfl_sync(0xffffffffu, base, l), lc = __shfl_sync(0xffffffffu, c, l);
        const int lp = __shfl_sync(0xffffffffu, piece, l), ls = __shfl_sync(0xffffffffu, sum, l);
        for (int k = lane; k * EM_PIECE < lc; k += 32)
            e.piece[lp + k] = make_int4(lt, lb + k * EM_PIECE, min(EM_PIECE, lc - k * EM_PIECE), ls + k);
    }
}

__global__ void __launch_bounds__(EM_NT) embed_scatter_kernel(const int64_t* tokens, int n, EmbedSort e) {
    pdl_wait_then_release();
    const int i = blockIdx.x * EM_NT + threadIdx.x;
    if (i >= n || e.place[i] < 0) return;
    e.loose[e.base[tokens[i]] + e.place[i]] = i;
}

// Each id's positions in ascending order.  Up to EM_SHORT of them: a place's rank by comparison with the others.  More: the
// CTA that has the range's first place marks them in a bitmap, EM_WINDOW positions at a time, and reads it in order.
constexpr int EM_SHORT = 64;
__global__ void __launch_bounds__(EM_NT) embed_order_kernel(const int64_t* tokens, int n, EmbedSort e) {
    __shared__ uint32_t bits[EM_WINDOW / 32];
    __shared__ int warp_sum[EM_NT / 32], longs[EM_NT / EM_SHORT + 1], found;
    pdl_wait_then_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int k = blockIdx.x * EM_NT + tid, all = e.next[0];
    if (tid == 0) found = 0;
    __syncthreads();
    if (k < all) {
        const int i = e.loose[k], t = (int)tokens[i], c = e.count[t], b = e.base[t];
        if (c <= EM_SHORT) {
            int rank = 0;
            for (int j = 0; j < c; ++j) rank += e.loose[b + j] < i;
            e.order[b + rank] = i;
        } else if (b == k) {
            longs[atomicAdd(&found, 1)] = t;
        }
    }
    __syncthreads();
    for (int f = 0; f < found; ++f) {
        const int t = longs[f], c = e.count[t], b = e.base[t];
        int done = 0;
        for (int64_t w0 = 0; w0 < n && done < c; w0 += EM_WINDOW) {
            const int words = ((int)min((int64_t)EM_WINDOW, n - w0) + 31) / 32, per = (words + EM_NT - 1) / EM_NT;
            for (int j = tid; j < words; j += EM_NT) bits[j] = 0;
            __syncthreads();
            for (int j = tid; j < c; j += EM_NT) {
                const int64_t i = e.loose[b + j] - w0;
                if (i >= 0 && i < EM_WINDOW) atomicOr(&bits[i >> 5], 1u << (i & 31));
            }
            __syncthreads();
            int mine = 0;
            for (int j = tid * per; j < min(words, (tid + 1) * per); ++j) mine += __popc(bits[j]);
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += u;
            }
            if (lane == 31) warp_sum[warp] = incl;
            __syncthreads();
            int at = b + done + incl - mine, total = 0;
            for (int j = 0; j < EM_NT / 32; ++j) {
                if (j < warp) at += warp_sum[j];
                total += warp_sum[j];
            }
            for (int j = tid * per; j < min(words, (tid + 1) * per); ++j)
                for (uint32_t m = bits[j]; m; m &= m - 1) e.order[at++] = (int)w0 + 32 * j + __ffs(m) - 1;
            done += total;
            __syncthreads();
        }
    }
}

// grid: first a warp per piece and part of a row (`warps` of them), then a warp per id and part that writes zeros for the
// ids that do not occur.
template <int E, bool VEC>
__global__ void __launch_bounds__(EM_NT) embed_sum_kernel(const void* grad, int64_t row_bytes, int n, int64_t vocab,
                                                          int64_t units, int64_t pieces, float s, void* out, EmbedSort e) {
    constexpr int N = Unit<E, VEC>::N, W = EM_UNITS / 32;
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31;
    int64_t w = (int64_t)blockIdx.x * (EM_NT / 32) + (threadIdx.x >> 5);
    const int64_t i = w / pieces, u0 = (w % pieces) * EM_UNITS + lane;
    Unit<E, VEC> sum[W];
#pragma unroll
    for (int j = 0; j < W; ++j) sum[j].zero();
    if (i >= n) {
        const int64_t v = i - n;
        if (v >= vocab || e.count[v]) return;
        unsigned char* dst = static_cast<unsigned char*>(out) + v * units * N * E;
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (u0 + 32 * j < units) sum[j].store(dst, u0 + 32 * j, 0.0f);
        return;
    }
    if (i >= e.next[1]) return;
    const int4 p = e.piece[i];
    const int mine = lane < p.z ? e.order[p.y + lane] : 0;
#pragma unroll 2
    for (int k = 0; k < p.z; ++k) {
        const unsigned char* src = static_cast<const unsigned char*>(grad) + __shfl_sync(0xffffffffu, mine, k) * row_bytes;
        Unit<E, VEC> g[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            g[j].zero();
            if (u0 + 32 * j < units) g[j].load(src, u0 + 32 * j);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) sum[j].add(g[j]);
    }
    if (p.w < 0) {
        unsigned char* dst = static_cast<unsigned char*>(out) + p.x * units * N * E;
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (u0 + 32 * j < units) sum[j].store(dst, u0 + 32 * j, s);
    } else {
        float* dst = e.sums + p.w * units * N;
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (u0 + 32 * j < units)
#pragma unroll
                for (int k = 0; k < N; ++k) dst[(u0 + 32 * j) * N + k] = sum[j].v[k];
    }
}

// The ids with several pieces: their sums added in order.  grid: (parts of a row of EM_NT columns, ids).
template <int E>
__global__ void __launch_bounds__(EM_NT) embed_join_kernel(int64_t width, float s, void* out, EmbedSort e) {
    pdl_wait_then_release();
    const int64_t col = (int64_t)blockIdx.x * EM_NT + threadIdx.x;
    const int ids = e.next[2];
    if (col >= width) return;
    for (int k = blockIdx.y; k < ids; k += gridDim.y) {
        const int4 p = e.split[k];
        float v = 0.0f;
#pragma unroll 8
        for (int j = 0; j < p.z; ++j) v += e.sums[(int64_t)(p.y + j) * width + col];
        const int64_t at = p.x * width + col;
        if (E == 4) static_cast<float*>(out)[at] = v * s;
        else static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v * s);
    }
}

int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// The workspace's arrays, and its bytes.
int64_t embed_layout(int64_t n, int64_t vocab, int64_t width, unsigned char* at, EmbedSort* e, int64_t* zeroed) {
    int64_t used = 0;
    auto take = [&](int64_t bytes) {
        unsigned char* p = at ? at + used : nullptr;
        used += up(bytes, 256);
        return p;
    };
    e->next = reinterpret_cast<int*>(take(16));
    e->count = reinterpret_cast<int*>(take(vocab * 4));
    *zeroed = used;
    e->base = reinterpret_cast<int*>(take(vocab * 4));
    e->place = reinterpret_cast<int*>(take(n * 4));
    e->loose = reinterpret_cast<int*>(take(n * 4));
    e->order = reinterpret_cast<int*>(take(n * 4));
    e->piece = reinterpret_cast<int4*>(take(n * 16));
    e->split = reinterpret_cast<int4*>(take((n / EM_PIECE + 1) * 16));
    e->sums = reinterpret_cast<float*>(take(2 * (n / EM_PIECE) * width * 4));
    return used;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool embed_sizes_ok(int64_t n, int64_t vocab, int64_t width) {
    return n <= LP_MAX_SIZE && vocab <= LP_MAX_SIZE && width <= LP_MAX_SIZE;
}
// Blocks of a launch with `warps` warps, 0 where those are more than a grid holds.
unsigned blocks_of(int64_t warps) {
    const int64_t b = (warps + EM_NT / 32 - 1) / (EM_NT / 32);
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
    const int64_t units = vec ? (int64_t)width * e / 16 : width, pieces = (units + EM_UNITS - 1) / EM_UNITS;
    const unsigned blocks = blocks_of(n * pieces);
    if (!blocks) return B2S_ERR_UNSUPPORTED;
    auto go = [&](auto kernel) {
        return launch_pdl(kernel, dim3(blocks), EM_NT, 0, stream, tokens, (int64_t)n, table, row_stride * e, (int64_t)vocab,
                          units, pieces, scale, out, status);
    };
    const cudaError_t r = e == 4 ? (vec ? go(embed_kernel<4, true>) : go(embed_kernel<4, false>))
                                 : (vec ? go(embed_kernel<2, true>) : go(embed_kernel<2, false>));
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
    const int64_t pieces = ((width + 7) / 8 + EM_UNITS - 1) / EM_UNITS;
    const unsigned blocks = blocks_of(n * pieces);
    if (!blocks) return B2S_ERR_UNSUPPORTED;
    const cudaError_t r = launch_pdl(embed_mx_kernel, dim3(blocks), EM_NT, 0, stream, tokens, (int64_t)n,
                                     static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), (int64_t)vocab,
                                     (int)width, pieces, scale, static_cast<__nv_bfloat16*>(out),
                                     (int)(aligned16(out) && width % 8 == 0), status);
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
    const int64_t units = vec ? (int64_t)width * e / 16 : width, pieces = (units + EM_UNITS - 1) / EM_UNITS;
    const unsigned blocks = blocks_of(((int64_t)n + vocab) * pieces), per = (unsigned)(((int64_t)n + EM_NT - 1) / EM_NT);
    if (!blocks) return B2S_ERR_UNSUPPORTED;
    cudaError_t r = cudaMemsetAsync(workspace, 0, (size_t)zeroed, (cudaStream_t)stream);
    if (r == cudaSuccess) r = launch_pdl(embed_count_kernel, dim3(per), EM_NT, 0, stream, tokens, (int)n, (int64_t)vocab, s);
    if (r == cudaSuccess) r = launch_pdl(embed_range_kernel, dim3(per), EM_NT, 0, stream, tokens, (int)n, s);
    if (r == cudaSuccess) r = launch_pdl(embed_scatter_kernel, dim3(per), EM_NT, 0, stream, tokens, (int)n, s);
    if (r == cudaSuccess) r = launch_pdl(embed_order_kernel, dim3(per), EM_NT, 0, stream, tokens, (int)n, s);
    if (r != cudaSuccess) return cuda_fail(r);
    auto sum = [&](auto kernel) {
        return launch_pdl(kernel, dim3(blocks), EM_NT, 0, stream, grad_out, grad_row_stride * e, (int)n, (int64_t)vocab, units,
                          pieces, scale, grad_table, s);
    };
    r = e == 4 ? (vec ? sum(embed_sum_kernel<4, true>) : sum(embed_sum_kernel<4, false>))
               : (vec ? sum(embed_sum_kernel<2, true>) : sum(embed_sum_kernel<2, false>));
    if (r == cudaSuccess && n > EM_PIECE) {
        const dim3 grid((unsigned)((width + EM_NT - 1) / EM_NT), (unsigned)(n / EM_PIECE < 64 ? n / EM_PIECE : 64));
        auto join = [&](auto kernel) { return launch_pdl(kernel, grid, EM_NT, 0, stream, (int64_t)width, scale, grad_table, s); };
        r = e == 4 ? join(embed_join_kernel<4>) : join(embed_join_kernel<2>);
    }
    return r == cudaSuccess ? B2S_OK : cuda_fail(r);
}

}  // extern "C"
