// hv_attn.cuh -- self-attention with a learned (dq, dr, dz) offset bias per
// head, and its backward pass, which recomputes the probabilities.
//
//   s_ij = scale q_i . k_j + Tq[clip(q_j - q_i)] + Tr[clip(r_j - r_i)] + Tz[clip(z_j - z_i)]
//   p_i  = softmax of s_i over the valid tokens j,      o_i = sum_j p_ij v_j
//
//   dv_j = sum_i p_ij do_i        dp_ij = do_i . v_j       ds_ij = p_ij (dp_ij - sum_k p_ik dp_ik)
//   dq_i = scale sum_j ds_ij k_j  dk_j = scale sum_i ds_ij q_i
//   dT[c] = sum of ds_ij over the pairs whose clipped offset is c
//
// A masked token takes no part: its key and value are never read into a sum,
// its output row and its gradients are zero.
#pragma once

#include "hv_elem.cuh"

namespace hv {

constexpr int kCoordMax = 1 << 19;  // coordinates are clamped to this first, so that offsets cannot overflow

struct AttnArgs {
    const void *q, *k, *v, *dout;
    int64_t qs[3], ks[3], vs[3], os[3], gs[3], gks[3];  // batch, token, head strides: q, k, v, dout, dq, dk and dv
    void* out;                                  // [B, Nq, H, D]
    void *dq, *dk, *dv;
    const int32_t *tq, *tr, *tz;
    int64_t tqs, trs, tzs, ms;
    const uint8_t* mask;
    const void *bq, *br, *bz;
    void *dbq, *dbr, *dbz;
    float* p;   // workspace [B, H, Nq, N]
    float* ds;  // workspace [B, H, Nq, N]
    float* partial;
    int64_t B;
    int N, Nq, H, D, clip, clip_z, t_f32;
    float scale;
};

__device__ __forceinline__ int clip_offset(int a, int b, int c) { return min(max(a - b, -c), c) + c; }
__device__ __forceinline__ int coord(int x) { return min(max(x, -kCoordMax), kCoordMax); }

// One warp per (batch, head, query).  BACK: recomputes p, writes p and ds, and dq.
template <typename T, bool BACK>
__global__ void __launch_bounds__(128) k_attn_row(const AttnArgs a) {
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (w >= a.B * a.H * a.Nq) return;
    const int i = (int)(w % a.Nq), h = (int)(w / a.Nq % a.H);
    const int64_t b = w / a.Nq / a.H;
    const uint8_t* mask = a.mask + b * a.ms;
    const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
    const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + h * a.ks[2];
    const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + h * a.vs[2];
    const T* go = static_cast<const T*>(a.dout) + b * a.os[0] + i * a.os[1] + h * a.os[2];
    float* p = a.p + w * a.N;
    float* ds = BACK ? a.ds + w * a.N : nullptr;
    T* out = BACK ? static_cast<T*>(a.dq) + b * a.gs[0] + i * a.gs[1] + h * a.gs[2]
                  : static_cast<T*>(a.out) + ((b * a.Nq + i) * a.H + h) * a.D;
    if (!mask[i]) {
        for (int d = lane; d < a.D; d += 32) out[d] = from_f32<T>(0.f);
        if (BACK)
            for (int j = lane; j < a.N; j += 32) p[j] = ds[j] = 0.f;
        return;
    }
    const int qi = coord(a.tq[b * a.tqs + i]), ri = coord(a.tr[b * a.trs + i]), zi = coord(a.tz[b * a.tzs + i]);
    float top = -INFINITY;
    for (int j = lane; j < a.N; j += 32) {
        float s = -INFINITY;
        if (mask[j]) {
            s = 0.f;
            for (int d = 0; d < a.D; d++) s = fmaf(to_f32(q[d]), to_f32(k[j * a.ks[1] + d]), s);
            const int cq = clip_offset(coord(a.tq[b * a.tqs + j]), qi, a.clip);
            const int cr = clip_offset(coord(a.tr[b * a.trs + j]), ri, a.clip);
            const int cz = clip_offset(coord(a.tz[b * a.tzs + j]), zi, a.clip_z);
            s = s * a.scale + load_param<T>(a.bq, cq * a.H + h, a.t_f32) + load_param<T>(a.br, cr * a.H + h, a.t_f32) +
                load_param<T>(a.bz, cz * a.H + h, a.t_f32);
        }
        p[j] = s;
        top = fmaxf(top, s);
    }
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.f;
    for (int j = lane; j < a.N; j += 32) {
        const float e = mask[j] ? expf(p[j] - top) : 0.f;
        p[j] = e;
        sum += e;
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float delta = 0.f;
    for (int j = lane; j < a.N; j += 32) {
        p[j] /= sum;
        if (BACK) {
            float dp = 0.f;
            if (mask[j])
                for (int d = 0; d < a.D; d++) dp = fmaf(to_f32(go[d]), to_f32(v[j * a.vs[1] + d]), dp);
            ds[j] = dp;
            delta = fmaf(p[j], dp, delta);
        }
    }
    for (int o = 16; o; o >>= 1) delta += __shfl_xor_sync(0xffffffffu, delta, o);
    if (BACK)
        for (int j = lane; j < a.N; j += 32) ds[j] = p[j] * (ds[j] - delta);
    __syncwarp();
    for (int d = lane; d < a.D; d += 32) {
        float o = 0.f;
        for (int j = 0; j < a.N; j++)
            if (mask[j]) o = BACK ? fmaf(ds[j], to_f32(k[j * a.ks[1] + d]), o) : fmaf(p[j], to_f32(v[j * a.vs[1] + d]), o);
        out[d] = from_f32<T>(BACK ? o * a.scale : o);
    }
}

// One warp per (batch, head, key): dk and dv from the stored p and ds.
template <typename T>
__global__ void __launch_bounds__(128) k_attn_key(const AttnArgs a) {
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (w >= a.B * a.H * a.N) return;
    const int j = (int)(w % a.N), h = (int)(w / a.N % a.H);
    const int64_t b = w / a.N / a.H;
    const uint8_t* mask = a.mask + b * a.ms;
    const float* p = a.p + (b * a.H + h) * a.Nq * (int64_t)a.N + j;
    const float* ds = a.ds + (b * a.H + h) * a.Nq * (int64_t)a.N + j;
    const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[2];
    const T* go = static_cast<const T*>(a.dout) + b * a.os[0] + h * a.os[2];
    const int64_t at = b * a.gks[0] + j * a.gks[1] + h * a.gks[2];
    for (int d = lane; d < a.D; d += 32) {
        float gk = 0.f, gv = 0.f;
        if (mask[j])
            for (int i = 0; i < a.Nq; i++)
                if (mask[i]) {
                    gk = fmaf(ds[(int64_t)i * a.N], to_f32(q[i * a.qs[1] + d]), gk);
                    gv = fmaf(p[(int64_t)i * a.N], to_f32(go[i * a.os[1] + d]), gv);
                }
        static_cast<T*>(a.dk)[at + d] = from_f32<T>(gk * a.scale);
        static_cast<T*>(a.dv)[at + d] = from_f32<T>(gv);
    }
}

// Bias-table gradients: one warp per (head, share of the rows).  Each lane
// keeps its own sums in shared memory, [class][lane], so no two lanes meet on
// an address and the order of the sums is fixed.
constexpr int kHistShares = 1024;

__global__ void __launch_bounds__(32) k_attn_table(const AttnArgs a) {
    extern __shared__ float hist[];
    const int lane = threadIdx.x, h = blockIdx.y, W = 2 * a.clip + 1, classes = 2 * W + 2 * a.clip_z + 1;
    for (int c = 0; c < classes; c++) hist[c * 32 + lane] = 0.f;
    for (int64_t row = blockIdx.x; row < a.B * a.Nq; row += gridDim.x) {
        const int64_t b = row / a.Nq;
        const int i = (int)(row % a.Nq);
        const int qi = coord(a.tq[b * a.tqs + i]), ri = coord(a.tr[b * a.trs + i]), zi = coord(a.tz[b * a.tzs + i]);
        const float* ds = a.ds + ((b * a.H + h) * a.Nq + i) * (int64_t)a.N;
        for (int j = lane; j < a.N; j += 32) {
            const float x = ds[j];
            hist[clip_offset(coord(a.tq[b * a.tqs + j]), qi, a.clip) * 32 + lane] += x;
            hist[(W + clip_offset(coord(a.tr[b * a.trs + j]), ri, a.clip)) * 32 + lane] += x;
            hist[(2 * W + clip_offset(coord(a.tz[b * a.tzs + j]), zi, a.clip_z)) * 32 + lane] += x;
        }
    }
    for (int c = 0; c < classes; c++) {
        float x = hist[c * 32 + lane];
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (lane == 0) a.partial[((int64_t)blockIdx.x * classes + c) * a.H + h] = x;
    }
}

// Sums n partial tables [n][classes][H]; one warp per value.
template <typename T>
__global__ void __launch_bounds__(128) k_attn_table_sum(const float* __restrict__ partial, int n, int W, int classes,
                                                        int H, void* dbq, void* dbr, void* dbz, int t_f32) {
    const int w = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (w >= classes * H) return;
    float x = 0.f;
    for (int i = lane; i < n; i += 32) x += partial[(int64_t)i * classes * H + w];
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane) return;
    if (w < W * H)
        store_param<T>(dbq, w, t_f32, x);
    else if (w < 2 * W * H)
        store_param<T>(dbr, w - W * H, t_f32, x);
    else
        store_param<T>(dbz, w - 2 * W * H, t_f32, x);
}

}  // namespace hv
