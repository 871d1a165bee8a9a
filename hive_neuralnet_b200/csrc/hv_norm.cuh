// hv_norm.cuh -- layer norm over the last axis, with an optional residual
// added first, and its backward pass.
//
//   s = x + r (kept in the stored type)      mean = sum s / C
//   y = (s - mean) rstd w + b                rstd = 1 / sqrt(sum (s - mean)^2 / C + eps)
//
//   xh = (s - mean) rstd,  g = dy w
//   dx = rstd (g - mean(g) - xh mean(g xh)) + ds
//   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// A row is held in the registers of G threads (a power of two; within a warp,
// or the whole block for wide rows), K vectors of V values each, so it is read
// once and the variance is that of the centred values.  All arithmetic is fp32.
#pragma once

#include "hv_elem.cuh"

namespace hv {

constexpr int kNormThreads = 256;     // rows within a warp
constexpr int kNormMaxThreads = 512;  // a row in a block
constexpr int kNormValues = 16;       // values of a row a thread holds at most

struct NormArgs {
    const void *x, *r, *w, *b;  // b: forward only
    void *s, *y;                // forward outputs; s NULL without a residual
    float *mean, *rstd;
    const void *dy, *ds;  // backward
    void *dx, *dw, *db;
    float* partial;  // [grid][2][C]; not used by a single block
    int64_t rows;
    int C, G, w_f32;
    float eps;
};

// Sum of a pair of values over the G threads of a row, in all of them.
__device__ __forceinline__ float2 row_sum(float2 v, int G, float2* scratch) {
    const int w = G < 32 ? G : 32;
    for (int o = w >> 1; o; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (G > 32) {
        __syncthreads();  // the previous sum's readers are done
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        v = scratch[0];
        for (int i = 1; i < (int)(blockDim.x >> 5); i++) v.x += scratch[i].x, v.y += scratch[i].y;
    }
    return v;
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kNormMaxThreads) k_norm_forward(const NormArgs a) {
    __shared__ float2 scratch[32];
    const int G = a.G, lane = threadIdx.x & (G - 1), groups = blockDim.x / G, group = threadIdx.x / G;
    float w[K][V], b[K][V];
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = (k * G + lane) * V + i;
            w[k][i] = c < a.C ? load_param<T>(a.w, c, a.w_f32) : 0.f;
            b[k][i] = c < a.C ? load_param<T>(a.b, c, a.w_f32) : 0.f;
        }
    const float inv_c = 1.f / (float)a.C;
    // whole groups of rows, so that every thread of a warp reaches the shuffles
    const int64_t step = (int64_t)gridDim.x * groups;
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += step) {
        const int64_t row = r0 + group;
        const bool live = row < a.rows;
        const T* x = static_cast<const T*>(a.x) + row * a.C;
        float v[K][V];
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * G + lane) * V;
            const bool in = live && c < a.C;
#pragma unroll
            for (int i = 0; i < V; i++) v[k][i] = 0.f;
            if (in) {
                load_vec<T, V>(x + c, v[k]);
                if (a.r) {
                    float r[V];
                    load_vec<T, V>(static_cast<const T*>(a.r) + row * a.C + c, r);
#pragma unroll
                    for (int i = 0; i < V; i++) v[k][i] = to_f32(from_f32<T>(v[k][i] + r[i]));
                    store_vec<T, V>(static_cast<T*>(a.s) + row * a.C + c, v[k]);
                }
            }
#pragma unroll
            for (int i = 0; i < V; i++) sum.x += v[k][i];
        }
        const float mean = row_sum(sum, G, scratch).x * inv_c;
        sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[k][i] = (k * G + lane) * V + i < a.C ? v[k][i] - mean : 0.f;
                sum.x = fmaf(v[k][i], v[k][i], sum.x);
            }
        const float rstd = 1.f / sqrtf(row_sum(sum, G, scratch).x * inv_c + a.eps);
        if (!live) continue;
        T* y = static_cast<T*>(a.y) + row * a.C;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * G + lane) * V;
            if (c >= a.C) continue;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; i++) o[i] = fmaf(v[k][i] * rstd, w[k][i], b[k][i]);
            store_vec<T, V>(y + c, o);
        }
        if (lane == 0 && a.mean) a.mean[row] = mean, a.rstd[row] = rstd;
    }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kNormMaxThreads) k_norm_backward(const NormArgs a) {
    __shared__ float2 scratch[32];
    __shared__ float part[kNormThreads * V];
    const int G = a.G, lane = threadIdx.x & (G - 1), groups = blockDim.x / G, group = threadIdx.x / G;
    float w[K][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = (k * G + lane) * V + i;
            w[k][i] = c < a.C ? load_param<T>(a.w, c, a.w_f32) : 0.f;
            dw[k][i] = db[k][i] = 0.f;
        }
    const float inv_c = 1.f / (float)a.C;
    const int64_t step = (int64_t)gridDim.x * groups;
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += step) {
        const int64_t row = r0 + group;
        const bool live = row < a.rows;
        const float mean = live ? a.mean[row] : 0.f, rstd = live ? a.rstd[row] : 0.f;
        float xh[K][V], g[K][V];
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * G + lane) * V;
            if (live && c < a.C) {
                load_vec<T, V>(static_cast<const T*>(a.x) + row * a.C + c, xh[k]);
                load_vec<T, V>(static_cast<const T*>(a.dy) + row * a.C + c, g[k]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) xh[k][i] = mean, g[k][i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                xh[k][i] = (xh[k][i] - mean) * rstd;
                db[k][i] += g[k][i];
                dw[k][i] = fmaf(g[k][i], xh[k][i], dw[k][i]);
                g[k][i] *= w[k][i];
                sum.x += g[k][i];
                sum.y = fmaf(g[k][i], xh[k][i], sum.y);
            }
        }
        sum = row_sum(sum, G, scratch);
        const float mg = sum.x * inv_c, mgx = sum.y * inv_c;
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * G + lane) * V;
            if (c >= a.C) continue;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; i++) o[i] = rstd * (g[k][i] - mg - xh[k][i] * mgx);
            if (a.ds) {
                float d[V];
                load_vec<T, V>(static_cast<const T*>(a.ds) + row * a.C + c, d);
#pragma unroll
                for (int i = 0; i < V; i++) o[i] += d[i];
            }
            store_vec<T, V>(static_cast<T*>(a.dx) + row * a.C + c, o);
        }
    }
    // this block's sums over its rows, in a fixed order: over the groups of a
    // warp by shuffles, over the warps through shared memory
    // (a single block's are the results)
    float* out = a.partial + (int64_t)blockIdx.x * 2 * a.C;
    auto put = [&](int which, int c, float x) {
        if (gridDim.x == 1)
            store_param<T>(which ? a.db : a.dw, c, a.w_f32, x);
        else
            out[which * a.C + c] = x;
    };
    const int span = G < 32 ? G : 32, warp = threadIdx.x >> 5, l = threadIdx.x & 31;
#pragma unroll
    for (int which = 0; which < 2; which++)
#pragma unroll
        for (int k = 0; k < K; k++) {
            float v[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[i] = which ? db[k][i] : dw[k][i];
                for (int o = span; o < 32; o <<= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
            }
            if (G > 32) {  // one row a block: its threads own their columns
                const int c = (k * G + lane) * V;
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (c + i < a.C) put(which, c + i, v[i]);
                continue;
            }
            __syncthreads();
            if (l < G)
#pragma unroll
                for (int i = 0; i < V; i++) part[(warp * G + l) * V + i] = v[i];
            __syncthreads();
            for (int j = threadIdx.x; j < G * V; j += blockDim.x) {
                float t = 0.f;
                for (int q = 0; q < (int)(blockDim.x >> 5); q++) t += part[q * G * V + j];
                const int c = k * G * V + j;
                if (c < a.C) put(which, c, t);
            }
        }
}

// Sums the blocks' partial rows [n][2][C] into dw and db: 32 columns a block,
// 32 threads down each column.
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_reduce(const float* __restrict__ partial, int n, int C, void* dw,
                                                      void* db, int w_f32) {
    __shared__ float t[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float v = 0.f;
    if (col < 2 * C)
        for (int i = part; i < n; i += 32) v += partial[(int64_t)i * 2 * C + col];
    t[part][threadIdx.x & 31] = v;
    __syncthreads();
    v = t[threadIdx.x & 31][part];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int c = blockIdx.x * 32 + part;
    if ((threadIdx.x & 31) == 0 && c < 2 * C) store_param<T>(c < C ? dw : db, c < C ? c : c - C, w_f32, v);
}

}  // namespace hv
