// What the log-probability kernels share (logits rows and the head's epilogue): the running softmax statistics and a
// bounded wait.  See b2s_logprobs.cu for the formulas; everything is in base 2, c = log2(e) / T.
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "b2s_device.cuh"

namespace b2s {

// Waits for the phase of `bar` with the given parity, for at most `limit` clocks (false then).  The bound is kept with
// the SM's own clock: a read of the global timer costs more than a k block's MMAs, and a wait per k block that took it
// held the products to 740 clocks per k block whatever the tile's width.
constexpr long long GM_WAIT = 500ll * 1000 * 1000;  // about a quarter of a second
template <bool CLUSTER>
__device__ __forceinline__ bool gm_try(uint64_t* bar, uint32_t parity) {
    if constexpr (!CLUSTER) return mbar_try_wait(bar, parity);
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
template <bool CLUSTER>
__device__ __forceinline__ bool gm_wait(uint64_t* bar, uint32_t parity, long long limit = GM_WAIT) {
    if (gm_try<CLUSTER>(bar, parity)) return true;
    const long long t0 = clock64();
    do {
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
            if (gm_try<CLUSTER>(bar, parity)) return true;
    } while (clock64() - t0 < limit);
    return false;
}

// m: maximum of the raw values (NaN once one was seen); S = sum 2^y, U = sum 2^y y with y relative to m (lp_y).
struct LpState {
    float m, S, U;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whether a reference R = fl(m c) is far from zero.  Near, y = fma(x, c, -R) is one rounding of x c - R, and R's own
// rounding, at most 2^-5, drops out of every difference.  Far, that rounding would be what 2^y is made of (it passes
// fp32's exponents from |R| about 2^31 on, and R overflows beyond), so y = (x - m) c there, whose maximum is exactly 0.
// Every user of a reference asks here, so that all of them take the same form.
__device__ __forceinline__ bool lp_far(float R) { return !(fabsf(R) <= 1048576.0f); }

// y of x against the maximum m; never below -200 (2^-200 is nothing beside the maximum's 1, and 0 * -inf would be NaN).
__device__ __forceinline__ float lp_y(float x, float m, float c) {
    const float R = __fmul_rn(m, c);
    const float y = lp_far(R) ? __fmul_rn(__fsub_rn(x, m), c) : __fmaf_rn(x, c, -R);
    return fmaxf(y, -200.0f);
}

// The shift of y when the maximum goes from `from` to `to` >= from (both finite), each with its own form.
__device__ __forceinline__ float lp_shift(float from, float to, float c) {
    const float Rf = __fmul_rn(from, c), Rt = __fmul_rn(to, c);
    const float d = lp_far(Rt) ? (lp_far(Rf) ? __fmul_rn(__fsub_rn(from, to), c) : -__fmaf_rn(to, c, -Rf))
                               : (lp_far(Rf) ? __fmaf_rn(from, c, -Rt) : __fsub_rn(Rf, Rt));
    return fmaxf(d, -400.0f);
}

// The state moved to the maximum m (s.m <= m, m neither NaN nor infinite).
__device__ __forceinline__ void lp_rescale(LpState& s, float m, float c) {
    if (s.m == f_ninf()) {
        s.m = m;
        return;  // S = U = 0
    }
    const float d = lp_shift(s.m, m, c), f = ex2(d);
    s.U = f * __fmaf_rn(d, s.S, s.U);
    s.S = f * s.S;
    s.m = m;
}

__device__ __forceinline__ LpState lp_merge(LpState a, LpState b, float c) {
    const float m = fmax_nan(a.m, b.m);
    LpState r;
    r.m = m;
    r.S = r.U = 0.0f;
    if (!(fabsf(m) <= 3.402823466e38f)) return r;  // NaN, +inf, or nothing but -inf
    if (a.m != f_ninf()) {
        lp_rescale(a, m, c);
        r.S += a.S;
        r.U += a.U;
    }
    if (b.m != f_ninf()) {
        lp_rescale(b, m, c);
        r.S += b.S;
        r.U += b.U;
    }
    return r;
}

__device__ __forceinline__ void lp_warp_merge(LpState& s, float c) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        LpState t;
        t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
        t.S = __shfl_xor_sync(0xffffffffu, s.S, o);
        t.U = __shfl_xor_sync(0xffffffffu, s.U, o);
        s = lp_merge(s, t, c);
    }
}

// N elements at once, any values: every y bounded below (a masked element adds 0), the form of y chosen per
// call.  Short code for the products' epilogue, whose arithmetic the MMAs hide.
template <int N>
__device__ __forceinline__ void lp_add_any(LpState& s, const float (&x)[N], float c) {
    float bm = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) bm = fmax_nan(bm, x[j]);
    const float m = fmax_nan(s.m, bm);
    if (!(fabsf(m) <= 3.402823466e38f)) {
        s.m = m;
        return;
    }
    if (m > s.m) lp_rescale(s, m, c);
    const float R = __fmul_rn(s.m, c);
    const bool far = lp_far(R);
    const float mul = c, off = far ? s.m : R, pre = far ? 1.0f : c, post = far ? mul : 1.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        // fma(x, c, -R), or (x - m) c
        const float y = fmaxf(__fmul_rn(__fmaf_rn(x[j], pre, -off), post), -200.0f), e = ex2(y);
        s.S += e;
        s.U = __fmaf_rn(e, y, s.U);
    }
}

// What the outputs need of a whole row.
struct LpFinal {
    float m, R, log2S, entropy;
};

__device__ __forceinline__ LpFinal lp_final(const LpState& s, float c) {
    LpFinal f;
    f.m = s.m;
    f.R = __fmul_rn(s.m, c);
    if (s.m == f_ninf()) {  // nothing left: probability 0 everywhere
        f.log2S = 0.0f;
        f.entropy = 0.0f;
    } else if (!(fabsf(s.m) <= 3.402823466e38f)) {
        f.m = f.log2S = f.entropy = __int_as_float(0x7fffffff);
    } else {
        f.log2S = log2f(s.S);
        f.entropy = fmax_nan((f.log2S - s.U / s.S) * 0.693147180559945309f, 0.0f);
    }
    return f;
}

// log p of the value x of a row.
__device__ __forceinline__ float lp_value(float x, const LpFinal& f, float c) {
    if (f.m != f.m) return f.m;
    if (x == f_ninf()) return x;
    const float y = lp_far(f.R) ? __fmul_rn(__fsub_rn(x, f.m), c) : __fmaf_rn(x, c, -f.R);
    if (fabsf(y) <= 3.0e38f) return (y - f.log2S) * 0.693147180559945309f;
    // a value so low that y overflows in base 2 may still be a number in base e (log2 S is nothing beside it), even where
    // x - m overflows
    const float ce = c * 0.693147180559945309f;
    return ce <= 1.0f ? __fmaf_rn(x, ce, -__fmul_rn(f.m, ce)) : __fmul_rn(__fsub_rn(x, f.m), ce);
}

// The gradient of g_lp logprob + g_h entropy with respect to one value of a row:
// (-p (g_lp + g_h H + g_h log p) + [id = token] g_lp) / T = p (scale + slope log2 p) + [id = token] bump.
struct LpGrad {
    float m, R, log2S, scale, slope, bump;
    bool far;
    int t;
    // st: the forward's (m, R, log2S, entropy); the row's token or -1 (no gradient through logprob)
    __device__ __forceinline__ LpGrad(float4 st, int tok, float g_lp, float g_h, float inv_t)
        : m(st.x), R(st.y), log2S(st.z), t(tok) {
        const bool none = m == f_ninf();  // nothing left: no gradient
        const float glp = tok >= 0 && !none ? g_lp : 0.0f, gh = none ? 0.0f : g_h;
        scale = -(glp + gh * st.w) * inv_t;
        slope = -gh * 0.693147180559945309f * inv_t;
        bump = glp * inv_t;
        far = lp_far(R) && !none;
        if (none) {
            R = 0.0f;
            log2S = 1000.0f;  // p = 0 for every value that is left: there is none
        }
    }
    // without the token's own part
    __device__ __forceinline__ float rest(float x, float c) const {
        float y = far ? __fmul_rn(__fsub_rn(x, m), c) : __fmaf_rn(x, c, -R);
        y = fmax_nan(y - log2S, -400.0f);  // log2 p, kept finite where p is 0
        return ex2(y) * __fmaf_rn(slope, y, scale);
    }
    __device__ __forceinline__ float at(float x, int id, float c) const { return rest(x, c) + (id == t ? bump : 0.0f); }
};

// Host side: the scale log2(e) / T rounded once.
inline float lp_scale(float temperature) { return (float)(1.4426950408889634 / (double)temperature); }
// Temperatures whose scale is a normal number well inside fp32.
inline bool lp_temperature_ok(float t) { return t >= 1e-6f && t <= 1e6f; }

// Rows, ids and features of a call: indices rounded up to a tile stay within 32 bits.
constexpr int LP_MAX_SIZE = 0x7fffffff - 4096;

cudaError_t device_sms(int* sms);  // multiprocessors of the current device
long long wait_limit();            // of the kernels' waits, in clocks (b2s_wait_limit); 0: they give up before they start

}  // namespace b2s
