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

#include "../../include/hive_b200.h"
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
    float* partial;  // sums of ds by class, for each block: [blocks][classes][H]
    int64_t B;
    int N, Nq, H, D, clip, clip_z, t_f32;
    float scale;
};

__device__ __forceinline__ int coord(int x) { return min(max(x, -kCoordMax), kCoordMax); }

// A pair's classes, times 4: from 4 x the key's coordinates and 4 x (clip less
// the query's).
struct Classes {
    int top, top_z, W, q, r, z;
    __device__ explicit Classes(const AttnArgs& a) : top(8 * a.clip), top_z(8 * a.clip_z), W(2 * a.clip + 1), q(0), r(0), z(0) {}
    __device__ __forceinline__ void of(int kq, int kr, int kz, int qq, int qr, int qz) {
        q = __viaddmin_s32_relu(kq, qq, top), r = __viaddmin_s32_relu(kr, qr, top), z = __viaddmin_s32_relu(kz, qz, top_z);
    }
};

// The bias in two terms: dz and dq from one table [dz][dq], dr from another
// (one lookup less than three tables; all three joined would be 1445 entries a
// head, to be built by every block, with bank conflicts at every lookup).
__device__ __forceinline__ float2 bias_of(const char* joined, const char* dr, const Classes& c) {
    return make_float2(*reinterpret_cast<const float*>(joined + (c.z * c.W + c.q)), *reinterpret_cast<const float*>(dr + c.r));
}

// A value that all lanes of a warp have, as one that the compiler knows to be so.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Sums n partial tables [n][classes][H] in a fixed order: a block takes 8
// values, 128 threads down each.
template <typename T>
__global__ void __launch_bounds__(1024) k_attn_table_sum(const float* __restrict__ partial, int64_t n, int W, int classes,
                                                         int H, void* dbq, void* dbr, void* dbz, int t_f32) {
    __shared__ float sums[32][8];
    after_previous();
    const int v = threadIdx.x & 7, part = threadIdx.x >> 3, at = blockIdx.x * 8 + v, values = classes * H;
    float x = 0.f;
    if (at < values)
#pragma unroll 4
        for (int64_t i = part; i < n; i += 128) x += partial[i * values + at];
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    x += __shfl_xor_sync(0xffffffffu, x, 16);
    if ((threadIdx.x & 31) < 8) sums[threadIdx.x >> 5][v] = x;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    // warp c: value c's 32 sums
    x = sums[threadIdx.x & 31][threadIdx.x >> 5];
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    const int c = blockIdx.x * 8 + (threadIdx.x >> 5);
    if ((threadIdx.x & 31) || c >= values) return;
    if (c < W * H)
        store_param<T>(dbq, c, t_f32, x);
    else if (c < 2 * W * H)
        store_param<T>(dbr, c - W * H, t_f32, x);
    else
        store_param<T>(dbz, c - 2 * W * H, t_f32, x);
}

}  // namespace hv
