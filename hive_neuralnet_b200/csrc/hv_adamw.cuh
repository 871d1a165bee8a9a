// hv_adamw.cuh -- one AdamW step over many tensors in one launch.
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every product and sum is rounded by itself (no contraction), so a step is
// the same on every path.  The moments live in two flat arrays; a tensor's
// part begins at a multiple of 256 values.
//
// 8-bit moments: a scale for each 256 values (largest magnitude / largest
// code).  m is stored as sign + 4 exponent + 3 mantissa bits; of v the root is
// stored, 4 exponent + 4 mantissa bits, which halves the range it has to span
// (the step divides by the root anyway).  A code's value is the float whose
// bits are code << 20 (<< 19) times 2^120, so subnormal codes need no case of
// their own.  Rounding is stochastic: a running mean that moves by 1 - b2 =
// 0.1 % a step would never leave a code 6 % wide if it were rounded to the
// nearest, and v would stay where its first steps left it.  The random bits
// are a hash of (position, step, seed), so a step can be repeated.  A positive
// root is never rounded to zero: the next step would divide by eps alone.
#pragma once

#include "hv_elem.cuh"

namespace hv {

constexpr int kAdamBlock = 256;  // values of one 8-bit scale; one warp's unit of work
constexpr int kAdamWarps = 8;
constexpr float kCodeMaxM = 480.f, kCodeMaxR = 496.f;

struct AdamScalars {
    float b1, one_b1, b2, one_b2, eps, decay, step_size, inv_root_bc2;
    uint32_t key;  // of the stochastic rounding
};

// Tensor table of one launch, passed as a kernel argument.
template <int CAP>
struct AdamTable {
    void* p[CAP];
    const void* g[CAP];
    int64_t n[CAP];
    int32_t first[CAP + 1];  // first 256-value unit of each tensor
    int32_t tensors;
};

__device__ __forceinline__ uint32_t adam_hash(uint64_t i, uint32_t key) {
    uint32_t h = (uint32_t)i * 0x9E3779B1u + (uint32_t)(i >> 32) * 0x3C6EF372u + key;
    h = (h ^ (h >> 16)) * 0x6A09E667u;
    h = (h ^ (h >> 13)) * 0xBB67AE85u;
    return h ^ (h >> 16);
}

__device__ __forceinline__ float code_value_m(uint32_t c) {
    const float y = __uint_as_float((c & 127u) << 20) * 0x1p120f;
    return c & 128u ? -y : y;
}

__device__ __forceinline__ float code_value_r(uint32_t c) { return __uint_as_float(c << 19) * 0x1p120f; }

__device__ __forceinline__ uint32_t encode(float y, uint32_t noise, int shift, uint32_t top) {
    const uint32_t c = (__float_as_uint(__fmul_rn(y, 0x1p-120f)) + noise) >> shift;
    return c < top ? c : top;
}

__device__ __forceinline__ void adam_value(float& p, float g, float& m, float& v, const AdamScalars& s) {
    m = __fadd_rn(__fmul_rn(m, s.b1), __fmul_rn(g, s.one_b1));
    v = __fadd_rn(__fmul_rn(v, s.b2), __fmul_rn(__fmul_rn(g, g), s.one_b2));
    const float denom = __fadd_rn(__fmul_rn(__fsqrt_rn(v), s.inv_root_bc2), s.eps);
    p = __fsub_rn(__fmul_rn(p, s.decay), __fmul_rn(__fdiv_rn(m, denom), s.step_size));
}

// 4 values at p + i of a tensor of n values; whole vectors where they fit.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t i, int64_t n, bool vec, float* x) {
    if (vec && i + 4 <= n) {
        load_vec<T, 4>(p + i, x);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = i + j < n ? to_f32(p[i + j]) : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, bool vec, const float* x) {
    if (vec && i + 4 <= n) {
        store_vec<T, 4>(p + i, x);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < n) p[i + j] = from_f32<T>(x[j]);
    }
}

// One warp takes 256 values, 4 + 4 a lane.  unit0: the table's first unit in
// the flat states.
template <typename T, bool SMALL, int CAP>
__global__ void __launch_bounds__(kAdamWarps * 32) k_adamw(const __grid_constant__ AdamTable<CAP> t, void* m_all,
                                                           void* v_all, float* m_scale, float* v_scale,
                                                           int64_t unit0, const AdamScalars s) {
    const int unit = blockIdx.x * kAdamWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (unit >= t.first[t.tensors]) return;
    int lo = 0, hi = t.tensors;  // the last tensor whose first unit is <= unit
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= unit)
            lo = mid;
        else
            hi = mid;
    }
    T* p = static_cast<T*>(t.p[lo]);
    const T* g = static_cast<const T*>(t.g[lo]);
    const int64_t n = t.n[lo], at = (int64_t)(unit - t.first[lo]) * kAdamBlock;
    const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & (4 * sizeof(T) - 1)) == 0;
    const int64_t u = unit0 + unit, flat = u * kAdamBlock;
    float P[8], M[8], R[8], Gr[8];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        load4<T>(p, at + h * 128 + lane * 4, n, vec, P + h * 4);
        load4<T>(g, at + h * 128 + lane * 4, n, vec, Gr + h * 4);
    }
    if (!SMALL) {
        float* m = static_cast<float*>(m_all) + flat;
        float* v = static_cast<float*>(v_all) + flat;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            load_vec<float, 4>(m + h * 128 + lane * 4, M + h * 4);
            load_vec<float, 4>(v + h * 128 + lane * 4, R + h * 4);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) adam_value(P[i], Gr[i], M[i], R[i], s);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            store_vec<float, 4>(m + h * 128 + lane * 4, M + h * 4);
            store_vec<float, 4>(v + h * 128 + lane * 4, R + h * 4);
        }
    } else {
        uint32_t* mc = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(m_all) + flat);
        uint32_t* vc = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(v_all) + flat);
        const float ms = m_scale[u], vs = v_scale[u];
        float top_m = 0.f, top_r = 0.f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t a = mc[h * 32 + lane], b = vc[h * 32 + lane];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = h * 4 + j;
                M[i] = __fmul_rn(code_value_m((a >> (8 * j)) & 255u), ms);
                const float r = __fmul_rn(code_value_r((b >> (8 * j)) & 255u), vs);
                R[i] = __fmul_rn(r, r);
                adam_value(P[i], Gr[i], M[i], R[i], s);
                R[i] = __fsqrt_rn(R[i]);
                top_m = fmaxf(top_m, fabsf(M[i]));
                top_r = fmaxf(top_r, R[i]);
            }
        }
        // non-negative floats order as their bits do
        top_m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_m)));
        top_r = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_r)));
        const bool live_m = top_m >= 0x1p-100f, live_r = top_r >= 0x1p-100f;  // below: no scale is kept
        const float inv_m = __fdiv_rn(kCodeMaxM, top_m), inv_r = __fdiv_rn(kCodeMaxR, top_r);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t a = 0, b = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = h * 4 + j;
                const uint32_t noise = adam_hash((uint64_t)(flat + h * 128 + lane * 4 + j), s.key);
                uint32_t c = encode(__fmul_rn(fabsf(M[i]), inv_m), noise & 0xFFFFFu, 20, 127u) | (M[i] < 0.f ? 128u : 0u);
                a |= (live_m ? c : 0u) << (8 * j);
                c = encode(__fmul_rn(R[i], inv_r), noise >> 13, 19, 255u);
                c = R[i] > 0.f && c == 0u ? 1u : c;
                b |= (live_r ? c : 0u) << (8 * j);
            }
            mc[h * 32 + lane] = a;
            vc[h * 32 + lane] = b;
        }
        if (lane == 0) {
            m_scale[u] = live_m ? __fdiv_rn(top_m, kCodeMaxM) : 0.f;
            v_scale[u] = live_r ? __fdiv_rn(top_r, kCodeMaxR) : 0.f;
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) store4<T>(p, at + h * 128 + lane * 4, n, vec, P + h * 4);
}

// The values that 8-bit states stand for, 4 a thread.
template <bool SECOND>
__global__ void __launch_bounds__(256) k_adamw_values(const uint32_t* __restrict__ codes,
                                                      const float* __restrict__ scale, int64_t words, float* out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= words) return;
    const uint32_t c = codes[i];
    const float s = scale[i / (kAdamBlock / 4)];
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t b = (c >> (8 * j)) & 255u;
        x[j] = __fmul_rn(SECOND ? code_value_r(b) : code_value_m(b), s);
        if (SECOND) x[j] = __fmul_rn(x[j], x[j]);
    }
    store_vec<float, 4>(out + i * 4, x);
}

}  // namespace hv
