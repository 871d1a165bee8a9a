// hv_attn_short.cuh -- the attention of hv_attn.cuh for up to 32 tokens, the
// network's own case (28 piece tokens and CLS).
//
// A block takes one position and a group of heads at a time, a warp one head:
// the position's rows come into shared memory once, coalesced over the heads,
// while the position before is computed.  Masked tokens are left out when the
// rows are stored, so a position costs what its valid tokens cost (an opening
// position has a few of its 28).  A head's scores (two 16 x 32 tiles at most)
// stay in registers from the first product to the last; the backward pass
// recomputes them from q and k, so nothing is kept between the passes.
// Results overwrite the operands they no longer need and leave in whole rows.
//
// Bias-table gradients: every lane adds into its own column of a [class][lane]
// table in shared memory for all positions its block takes; the columns are
// summed once at the end, in a fixed order.
#pragma once

#include "hv_attn.cuh"
#include "hv_mma.cuh"

namespace hv {

constexpr int kSlots = 32;  // tokens of a position after compaction

struct ShortPlan {
    int HG, groups;            // heads a block, groups of heads
    int row;                   // bytes of a row of one operand in shared memory
    int stage, tables, total;  // bytes: one stage, the tables before the stages, all
    int vec_in, vec_out;       // 16-byte copies
    int per_group;             // blocks for each group of heads
};

// The copies between global memory and the slots.  A unit is half the rows
// (16) of one operand, and a warp's: 16-byte pieces, each lane at its own
// place in a row, 32 / pieces rows at a time.
template <typename T, int DP>
struct RowCopy {
    int D, row, width;
    bool vec;
    int r0, rows, at, lane, head, piece;  // 16-byte pieces: the lane's first row, rows at a time, its bytes in a slot

    __device__ void init(int heads, int D_, int row_, bool vec_) {
        D = D_, row = row_, vec = vec_, width = heads * D_, lane = threadIdx.x & 31;
        const int per_head = D * (int)sizeof(T) / 16, pieces = heads * per_head;
        if (vec) {
            rows = 32 / pieces, r0 = lane / pieces;
            const int x = lane - r0 * pieces;
            head = x / per_head, piece = x - head * per_head;
            at = head * DP * (int)sizeof(T) + piece * 16;
            if (r0 >= rows) r0 = kSlots;  // lanes past the last whole row
        }
    }
    __device__ static int slot(uint32_t valid, int r) { return __popc(valid & ((1u << r) - 1)); }

    // half 0, 1: rows 16 half .. of the n tokens
    __device__ void load(char* dst, const void* src, const int64_t* s, int64_t b, int h0, int n, int half,
                         uint32_t valid) const {
        const T* base = static_cast<const T*>(src) + b * s[0] + h0 * s[2];
        const int end = min(n, 16 * half + 16);
        if (vec) {
            const T* p = base + head * s[2] + piece * (16 / (int)sizeof(T));
            for (int r = 16 * half + r0; r < end; r += rows)
                if (valid >> r & 1) cp_async16(dst + slot(valid, r) * row + at, p + r * s[1]);
        } else {
            for (int i = 16 * half * width + lane; i < end * width; i += 32) {
                const int r = i / width, c = i - r * width, h = c / D, d = c - h * D;
                if (valid >> r & 1)
                    reinterpret_cast<T*>(dst + slot(valid, r) * row)[h * DP + d] = base[r * s[1] + h * s[2] + d];
            }
        }
        if (half == 0) {  // the slots up to the next multiple of 16 count as zero rows
            const int c = __popc(valid & (n < 32 ? (1u << n) - 1 : 0xffffffffu));
            uint4* z = reinterpret_cast<uint4*>(dst + c * row);
            for (int i = lane; i < (-c & 15) * (row >> 4); i += 32) z[i] = make_uint4(0, 0, 0, 0);
        }
    }
    __device__ void store(const char* src, void* dst, const int64_t* s, int64_t b, int h0, int n, int half,
                          uint32_t valid) const {
        T* base = static_cast<T*>(dst) + b * s[0] + h0 * s[2];
        const int end = min(n, 16 * half + 16);
        if (vec) {
            T* p = base + head * s[2] + piece * (16 / (int)sizeof(T));
            for (int r = 16 * half + r0; r < end; r += rows) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (valid >> r & 1) v = *reinterpret_cast<const uint4*>(src + slot(valid, r) * row + at);
                *reinterpret_cast<uint4*>(p + r * s[1]) = v;
            }
        } else {
            for (int i = 16 * half * width + lane; i < end * width; i += 32) {
                const int r = i / width, c = i - r * width, h = c / D, d = c - h * D;
                T v = from_f32<T>(0.f);
                if (valid >> r & 1) v = reinterpret_cast<const T*>(src + slot(valid, r) * row)[h * DP + d];
                base[r * s[1] + h * s[2] + d] = v;
            }
        }
    }
};

// Byte offsets (4 x class) of a pair's three classes; the coordinates are
// multiplied by 4 and the query's are negated with 4 clip added.
struct ClassOf {
    int top, top_z;
    __device__ __forceinline__ int q(int key, int query) const { return __viaddmin_s32_relu(key, query, top); }
    __device__ __forceinline__ int z(int key, int query) const { return __viaddmin_s32_relu(key, query, top_z); }
};

template <typename T, int DP, bool BACK>
__global__ void __launch_bounds__(256) k_attn_short(const AttnArgs a, const ShortPlan p) {
    using Op = Tile<T, DP == 8>;
    constexpr int NC = DP / 8, CB = NC < 4 ? NC : 4, PARTS = kParts<T>;  // 8-value chunks of a head
    constexpr bool F32 = sizeof(T) == 4;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = blockIdx.x % p.groups, h0 = group * p.HG, heads = min(p.HG, a.H - h0);
    const int W = 2 * a.clip + 1, Z = 2 * a.clip_z + 1, classes = 2 * W + Z;
    const int ld = p.row / (int)sizeof(T);
    constexpr float kLog2e = 1.4426950408889634f;

    // the transposes' room (float2 words: first, where it is aligned), bias
    // (times log2 e) [head][class], the lanes' sums
    float* scratch = reinterpret_cast<float*>(smem);
    float* tab = scratch + (BACK && F32 ? p.HG * 16 * kTransposeLd : 0);
    float* hist = tab + p.HG * classes;
    char* stages = smem + p.tables;
    for (int i = threadIdx.x; i < p.HG * classes; i += blockDim.x) {
        const int h = i / classes, c = i - h * classes;
        float v = 0.f;
        if (h < heads) {
            const void* src = c < W ? a.bq : c < 2 * W ? a.br : a.bz;
            v = load_param<T>(src, (int64_t)(c < W ? c : c < 2 * W ? c - W : c - 2 * W) * a.H + h0 + h, a.t_f32);
        }
        tab[i] = v * kLog2e;
    }
    if (BACK)
        for (int i = threadIdx.x; i < p.HG * classes * 32; i += blockDim.x) hist[i] = 0.f;
    // columns past D stay zero: no copy writes them, and results there are zero
    for (int i = threadIdx.x; i < 2 * p.stage / 16; i += blockDim.x)
        reinterpret_cast<uint4*>(stages)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();

    RowCopy<T, DP> in, out;
    in.init(heads, a.D, p.row, p.vec_in);
    out.init(heads, a.D, p.row, p.vec_out);
    const uint32_t queries = a.Nq < 32 ? (1u << a.Nq) - 1 : 0xffffffffu;
    const int64_t step = gridDim.x / p.groups;
    const int operand = kSlots * p.row;

    // a position's mask (in every warp) and coordinates (in warp 0), held from
    // one turn to the next so that their loads are not waited for
    struct Tokens {
        int alive;
        int c[3];
    };
    auto fetch = [&](int64_t b) {
        Tokens k = {0, {0, 0, 0}};
        if (b < a.B && lane < a.N) {
            k.alive = a.mask[b * a.ms + lane];
            if (warp == 0) k.c[0] = a.tq[b * a.tqs + lane], k.c[1] = a.tr[b * a.trs + lane], k.c[2] = a.tz[b * a.tzs + lane];
        }
        return k;
    };
    auto issue = [&](int64_t b, char* st, const Tokens& k) -> uint32_t {
        const uint32_t valid = __ballot_sync(0xffffffffu, k.alive != 0);
        if (b < a.B) {
            if (warp == 0 && k.alive) {
                int* c = reinterpret_cast<int*>(st) + __popc(valid & ((1u << lane) - 1));
#pragma unroll
                for (int i = 0; i < 3; i++) c[i * kSlots] = coord(k.c[i]) * 4;
            }
            char* x = st + 3 * kSlots * 4;
            for (int u = warp; u < (BACK ? 8 : 6); u += warps) {
                const int o = u >> 1;
                const void* src = o == 0 ? a.q : o == 1 ? a.k : o == 2 ? a.v : a.dout;
                const int64_t* s = o == 0 ? a.qs : o == 1 ? a.ks : o == 2 ? a.vs : a.os;
                in.load(x + o * operand, src, s, b, h0, o == 0 || o == 3 ? a.Nq : a.N, u & 1, valid);
            }
        }
        cp_async_commit();
        return valid;
    };

    int64_t b = blockIdx.x / p.groups;
    Tokens next = fetch(b);
    uint32_t valid = issue(b, stages, next);
    next = fetch(b + step);
    const float scale2 = a.scale * kLog2e;
    const ClassOf cls = {8 * a.clip, 8 * a.clip_z};
    for (int turn = 0; b < a.B; b += step, turn ^= 1) {
        char* st = stages + turn * p.stage;
        const uint32_t valid_next = issue(b + step, stages + (turn ^ 1) * p.stage, next);
        next = fetch(b + 2 * step);
        cp_async_wait<1>();
        __syncthreads();
        char* x = st + 3 * kSlots * 4;
        if (warp < heads && valid) {
            const int n = __popc(valid), nq = __popc(valid & queries);
            const int* co = reinterpret_cast<const int*>(st);
            T* Q = reinterpret_cast<T*>(x) + warp * DP;
            T* K = reinterpret_cast<T*>(x + operand) + warp * DP;
            T* V = reinterpret_cast<T*>(x + 2 * operand) + warp * DP;
            T* G = reinterpret_cast<T*>(x + 3 * operand) + warp * DP;
            const char* bias = reinterpret_cast<const char*>(tab + warp * classes);
            const char* bias_r = bias + W * 4;
            const char* bias_z = bias + 2 * W * 4;
            const uint32_t hq = smem_addr(hist + warp * classes * 32 + lane), hr = hq + W * 128, hz = hr + W * 128;
            float dk[2][NC][4], dv[2][NC][4];
            if (BACK)
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++) dk[m][c][e] = dv[m][c][e] = 0.f;
#pragma unroll 1
            for (int m0 = 0; m0 < nq; m0 += 16) {
                float s[4][4], dp[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[i][e] = dp[i][e] = 0.f;
#pragma unroll
                for (int d = 0; d < DP; d += Op::KD) {
                    typename Op::A qa[1];
                    typename Op::B kb[2];
                    Op::load_a(qa[0], Q + m0 * ld + d, ld, lane);
                    Op::load_bn(kb, K + d, ld, lane);
                    Op::template product_d<false>(s, qa, kb);
                    if (n > 16) {
                        Op::load_bn(kb, K + 16 * ld + d, ld, lane);
                        Op::template product_d<false>(s + 2, qa, kb);
                    }
                    if (BACK) {
                        Op::load_a(qa[0], G + m0 * ld + d, ld, lane);
                        Op::load_bn(kb, V + d, ld, lane);
                        Op::template product_d<false>(dp, qa, kb);
                        if (n > 16) {
                            Op::load_bn(kb, V + 16 * ld + d, ld, lane);
                            Op::template product_d<false>(dp + 2, qa, kb);
                        }
                    }
                }
                int q4[2][3];
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int i = 0; i < 3; i++)
                        q4[r][i] = 4 * (i < 2 ? a.clip : a.clip_z) - co[i * kSlots + m0 + g + 8 * r];
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (8 * i >= n) continue;
                    const int j = 8 * i + 2 * t;
                    const int2 kq = *reinterpret_cast<const int2*>(co + j), kr = *reinterpret_cast<const int2*>(co + kSlots + j),
                               kz = *reinterpret_cast<const int2*>(co + 2 * kSlots + j);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = e >> 1;
                        const int cq = cls.q(e & 1 ? kq.y : kq.x, q4[r][0]), cr = cls.q(e & 1 ? kr.y : kr.x, q4[r][1]),
                                  cz = cls.z(e & 1 ? kz.y : kz.x, q4[r][2]);
                        const float add = *reinterpret_cast<const float*>(bias + cq) +
                                          *reinterpret_cast<const float*>(bias_r + cr) +
                                          *reinterpret_cast<const float*>(bias_z + cz);
                        s[i][e] = j + (e & 1) < n ? fmaf(s[i][e], scale2, add) : -INFINITY;
                        top[r] = fmaxf(top[r], s[i][e]);
                    }
                }
                float sum[2] = {0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (8 * i >= n) continue;  // s stays 0 there
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s[i][e] = exp2_approx(s[i][e] - top[e >> 1]);
                        sum[e >> 1] += s[i][e];
                    }
                }
                float delta[2] = {0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                    sum[r] = rcp_approx(sum[r]);
                }
                if constexpr (!BACK) {
                    // o = p v; the division by the sum comes last
                    float o[NC][4];
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[c][e] = 0.f;
#pragma unroll
                    for (int k = 0; k < kSlots; k += Op::KK) {
                        if (k >= n) continue;
                        typename Op::A pa[PARTS];
                        Op::a_from_c(pa, s + k / 8);
#pragma unroll
                        for (int c = 0; c < NC; c += CB) {
                            typename Op::B vb[CB];
                            Op::load_bk(vb, V + k * ld + 8 * c, ld, lane);
                            Op::template product<false>(o + c, pa, vb);
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        float lo[2] = {o[c][0] * sum[0], o[c][1] * sum[0]}, hi[2] = {o[c][2] * sum[1], o[c][3] * sum[1]};
                        store_vec<T, 2>(Q + (m0 + g) * ld + 8 * c + 2 * t, lo);
                        store_vec<T, 2>(Q + (m0 + g + 8) * ld + 8 * c + 2 * t, hi);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (8 * i >= n) continue;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            s[i][e] *= sum[e >> 1];
                            delta[e >> 1] = fmaf(s[i][e], dp[i][e], delta[e >> 1]);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        delta[r] += __shfl_xor_sync(0xffffffffu, delta[r], 1);
                        delta[r] += __shfl_xor_sync(0xffffffffu, delta[r], 2);
                    }
                    // dp becomes ds; its sums by class
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (8 * i >= n) continue;
#pragma unroll
                        for (int e = 0; e < 4; e++) dp[i][e] = s[i][e] * (dp[i][e] - delta[e >> 1]);
                        const int j = 8 * i + 2 * t;
                        const int2 kq = *reinterpret_cast<const int2*>(co + j), kr = *reinterpret_cast<const int2*>(co + kSlots + j),
                                   kz = *reinterpret_cast<const int2*>(co + 2 * kSlots + j);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int r = e >> 1;
                            add_at(hq + cls.q(e & 1 ? kq.y : kq.x, q4[r][0]) * 32, hr + cls.q(e & 1 ? kr.y : kr.x, q4[r][1]) * 32,
                                   hz + cls.z(e & 1 ? kz.y : kz.x, q4[r][2]) * 32, dp[i][e]);
                        }
                    }
                    typename Op::A pt[2][16 / Op::KK][PARTS];
                    float* room = scratch + (F32 ? warp * 16 * kTransposeLd : 0);
                    transpose_c<T, DP == 8>(pt, s, room, lane);
#pragma unroll
                    for (int k = 0; k < 16 / Op::KK; k++)
#pragma unroll
                        for (int c = 0; c < NC; c += CB) {
                            typename Op::B gb[CB];
                            Op::load_bk(gb, G + (m0 + k * Op::KK) * ld + 8 * c, ld, lane);
                            Op::template product<false>(dv[0] + c, pt[0][k], gb);
                            if (n > 16) Op::template product<false>(dv[1] + c, pt[1][k], gb);
                        }
                    transpose_c<T, DP == 8>(pt, dp, room, lane);
#pragma unroll
                    for (int k = 0; k < 16 / Op::KK; k++)
#pragma unroll
                        for (int c = 0; c < NC; c += CB) {
                            typename Op::B qb[CB];
                            Op::load_bk(qb, Q + (m0 + k * Op::KK) * ld + 8 * c, ld, lane);
                            Op::template product<false>(dk[0] + c, pt[0][k], qb);
                            if (n > 16) Op::template product<false>(dk[1] + c, pt[1][k], qb);
                        }
                    __syncwarp();  // this tile's rows of Q are done with: dq takes their place
#pragma unroll
                    for (int c = 0; c < NC; c += CB) {
                        float o[CB][4];
#pragma unroll
                        for (int z = 0; z < CB; z++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[z][e] = 0.f;
#pragma unroll
                        for (int k = 0; k < kSlots; k += Op::KK) {
                            if (k >= n) continue;
                            typename Op::A da[PARTS];
                            typename Op::B kb[CB];
                            Op::a_from_c(da, dp + k / 8);
                            Op::load_bk(kb, K + k * ld + 8 * c, ld, lane);
                            Op::template product<false>(o, da, kb);
                        }
#pragma unroll
                        for (int z = 0; z < CB; z++) {
                            float lo[2] = {o[z][0] * a.scale, o[z][1] * a.scale}, hi[2] = {o[z][2] * a.scale, o[z][3] * a.scale};
                            store_vec<T, 2>(Q + (m0 + g) * ld + 8 * (c + z) + 2 * t, lo);
                            store_vec<T, 2>(Q + (m0 + g + 8) * ld + 8 * (c + z) + 2 * t, hi);
                        }
                    }
                }
            }
            if constexpr (BACK) {
                __syncwarp();
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        if (16 * m >= n) continue;
                        const int at = (16 * m + g) * ld + 8 * c + 2 * t;
                        float lo[2] = {dk[m][c][0] * a.scale, dk[m][c][1] * a.scale},
                              hi[2] = {dk[m][c][2] * a.scale, dk[m][c][3] * a.scale};
                        store_vec<T, 2>(K + at, lo);
                        store_vec<T, 2>(K + at + 8 * ld, hi);
                        store_vec<T, 2>(V + at, dv[m][c]);
                        store_vec<T, 2>(V + at + 8 * ld, dv[m][c] + 2);
                    }
            }
        }
        __syncthreads();
        for (int u = warp; u < (BACK ? 6 : 2); u += warps) {
            const int o = u >> 1;
            void* dst = !BACK ? a.out : o == 0 ? a.dq : o == 1 ? a.dk : a.dv;
            out.store(x + o * operand, dst, o == 0 ? a.gs : a.gks, b, h0, o == 0 ? a.Nq : a.N, u & 1, valid);
        }
        __syncthreads();
        valid = valid_next;
    }
    cp_async_wait<0>();
    if (BACK && warp < heads) {
        // this block's sums: a lane takes a class and adds up its 32 columns
        float* part = a.partial + (int64_t)(blockIdx.x / p.groups) * classes * a.H + h0 + warp;
        for (int c = lane; c < classes; c += 32) {
            const float* col = hist + (warp * classes + c) * 32;
            float v = 0.f;
            for (int i = 0; i < 32; i++) v += col[(i + lane) & 31];
            part[(int64_t)c * a.H] = v;
        }
    }
}

}  // namespace hv
