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
constexpr int kNormValues = 16;       // values of a row a thread holds at most ...
constexpr int kNormValuesWarp = 8;    // ... where a row lies within a warp

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

// Sum of a pair of values over the G threads of a row, in all of them.  WIDE:
// over the block; its warps meet once, two scratch rows take turns.
template <bool WIDE>
struct RowSum {
    float2 (*scratch)[kNormMaxThreads / 32];
    int G, turn;
    __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (WIDE || o < G) {
                v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
                v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
            }
        if (WIDE) {
            float2* s = scratch[turn];
            turn ^= 1;
            if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
            __syncthreads();
            const int warps = blockDim.x >> 5;  // a power of two, at most 16
            v = s[threadIdx.x & (warps - 1)];
#pragma unroll
            for (int o = kNormMaxThreads / 64; o; o >>= 1)
                if (o < warps) {
                    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
                    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
                }
        }
        return v;
    }
    __device__ __forceinline__ float operator()(float x) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (WIDE || o < G) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (WIDE) {
            float2* s = scratch[turn];
            turn ^= 1;
            if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5].x = x;
            __syncthreads();
            const int warps = blockDim.x >> 5;
            x = s[threadIdx.x & (warps - 1)].x;
#pragma unroll
            for (int o = kNormMaxThreads / 64; o; o >>= 1)
                if (o < warps) x += __shfl_xor_sync(0xffffffffu, x, o);
        }
        return x;
    }
};

// A thread's vectors of a row, K of V values; at: the element offset of the first.
template <typename T, int V, int K>
struct RowOf {
    Vec<T, V> x[K];
    __device__ __forceinline__ void load(const void* base, int64_t at, int step, int left) {
        const T* p = static_cast<const T*>(base) + at;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (k * step < left) x[k] = *reinterpret_cast<const Vec<T, V>*>(p + k * step);
    }
    __device__ __forceinline__ float at(int k, int i) const { return to_f32(x[k].x[i]); }
};

// Registers: rows within a warp are held to 64, four blocks an SM; wide rows
// to 128.
#define HV_NORM_BOUNDS __launch_bounds__(WIDE ? kNormMaxThreads : kNormThreads, WIDE ? 1 : 4)

template <typename T, int V, int K, bool WIDE, bool RES>
__global__ void HV_NORM_BOUNDS k_norm_forward(const NormArgs a) {
    __shared__ float2 scratch[2][kNormMaxThreads / 32];
    const int G = WIDE ? blockDim.x : a.G, lane = threadIdx.x & (G - 1), groups = blockDim.x / G, group = threadIdx.x / G;
    const int C = a.C, vstep = G * V, left = C - lane * V;  // vector k of a thread is in its row if k vstep < left
    RowSum<WIDE> row_sum = {scratch, G, 0};
    float w[K][V], b[K][V];
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = k * vstep + lane * V + i;
            w[k][i] = c < C ? load_param<T>(a.w, c, a.w_f32) : 0.f;
            b[k][i] = c < C ? load_param<T>(a.b, c, a.w_f32) : 0.f;
        }
    const float inv_c = 1.f / (float)C;
    const int64_t step = (int64_t)gridDim.x * groups, astep = step * C;
    int64_t row = (int64_t)blockIdx.x * groups + group, at = row * C + lane * V;
    RowOf<T, V, K> x, r;
    if (row < a.rows) {
        x.load(a.x, at, vstep, left);
        if (RES) r.load(a.r, at, vstep, left);
    }
    // whole groups of rows, so that every thread of a warp reaches the shuffles
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += step) {
        const bool live = row < a.rows;
        float v[K][V], sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool in = live && k * vstep < left;
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[k][i] = x.at(k, i);
                if (RES) v[k][i] = to_f32(from_f32<T>(v[k][i] + r.at(k, i)));
                v[k][i] = in ? v[k][i] : 0.f;
                sum += v[k][i];
            }
            if (RES && in) store_vec<T, V>(static_cast<T*>(a.s) + at + k * vstep, v[k]);
        }
        if (row + step < a.rows) {  // the next row's, a turn ahead
            x.load(a.x, at + astep, vstep, left);
            if (RES) r.load(a.r, at + astep, vstep, left);
        }
        const float mean = row_sum(sum) * inv_c;
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[k][i] = k * vstep < left ? v[k][i] - mean : 0.f;
                sum = fmaf(v[k][i], v[k][i], sum);
            }
        const float rstd = rsqrtf(row_sum(sum) * inv_c + a.eps);
        if (live) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (k * vstep >= left) continue;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; i++) o[i] = fmaf(v[k][i] * rstd, w[k][i], b[k][i]);
                store_vec<T, V>(static_cast<T*>(a.y) + at + k * vstep, o);
            }
            if (lane == 0 && a.mean) a.mean[row] = mean, a.rstd[row] = rstd;
        }
        row += step, at += astep;
    }
}

template <typename T, int V, int K, bool WIDE, bool RES>
__global__ void HV_NORM_BOUNDS k_norm_backward(const NormArgs a) {
    __shared__ float2 scratch[2][kNormMaxThreads / 32];
    __shared__ float part[WIDE ? 1 : kNormThreads * V];
    const int G = WIDE ? blockDim.x : a.G, lane = threadIdx.x & (G - 1), groups = blockDim.x / G, group = threadIdx.x / G;
    const int C = a.C, vstep = G * V, left = C - lane * V;
    RowSum<WIDE> row_sum = {scratch, G, 0};
    float w[K][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = k * vstep + lane * V + i;
            w[k][i] = c < C ? load_param<T>(a.w, c, a.w_f32) : 0.f;
            dw[k][i] = db[k][i] = 0.f;
        }
    const float inv_c = 1.f / (float)C;
    const int64_t step = (int64_t)gridDim.x * groups, astep = step * C;
    int64_t row = (int64_t)blockIdx.x * groups + group, at = row * C + lane * V;
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += step) {
        const bool live = row < a.rows;
        RowOf<T, V, K> x, dy, ds;
        float mean = 0.f, rstd = 0.f;
        if (live) {
            x.load(a.x, at, vstep, left);
            dy.load(a.dy, at, vstep, left);
            if (RES) ds.load(a.ds, at, vstep, left);
            mean = a.mean[row], rstd = a.rstd[row];
        }
        float xh[K][V], g[K][V];
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool in = live && k * vstep < left;
#pragma unroll
            for (int i = 0; i < V; i++) {
                xh[k][i] = in ? (x.at(k, i) - mean) * rstd : 0.f;
                g[k][i] = in ? dy.at(k, i) : 0.f;
                db[k][i] += g[k][i];
                dw[k][i] = fmaf(g[k][i], xh[k][i], dw[k][i]);
                g[k][i] *= w[k][i];
                sum.x += g[k][i];
                sum.y = fmaf(g[k][i], xh[k][i], sum.y);
            }
        }
        sum = row_sum(sum);
        const float mg = sum.x * inv_c, mgx = sum.y * inv_c;
        if (live)
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (k * vstep >= left) continue;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    o[i] = rstd * (g[k][i] - mg - xh[k][i] * mgx);
                    if (RES) o[i] += ds.at(k, i);
                }
                store_vec<T, V>(static_cast<T*>(a.dx) + at + k * vstep, o);
            }
        row += step, at += astep;
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
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
#pragma unroll
    for (int which = 0; which < 2; which++)
#pragma unroll
        for (int k = 0; k < K; k++) {
            float v[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[i] = which ? db[k][i] : dw[k][i];
                if (!WIDE)
                    for (int o = G; o < 32; o <<= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
            }
            if (WIDE) {  // one row a block: its threads own their columns
                const int c = k * vstep + lane * V;
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (c + i < C) put(which, c + i, v[i]);
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
                if (c < C) put(which, c, t);
            }
        }
}

#undef HV_NORM_BOUNDS

// Sums the blocks' partial rows [n][2][C] into dw and db: 32 columns a block,
// 32 threads down each column.
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_reduce(const float* __restrict__ partial, int n, int C, void* dw,
                                                      void* db, int w_f32) {
    __shared__ float t[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float v = 0.f;
    if (col < 2 * C)
#pragma unroll 8
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
