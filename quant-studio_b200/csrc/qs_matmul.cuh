// Shared pieces of the packed products (qs_matmul_few.cu, qs_matmul_tile.cu).
//
// y[slot, n] = sum over the 32-value units u of a row of
//   dx[slot, u] * (dl[n, u] * sum lw * lx  -  ml[n, u] * sum lx)
// with lw, lx the 8-bit levels of weight row n and of the slot's Q8_0 row. The level sums are
// exact integers; the scales and the running sum are float32.
//
// Slots: row i of the activations, or (token, j) when every token asks for several experts.
// Slots are grouped by weight matrix: `order` lists them group by group, group e is
// [offsets[e], offsets[e + 1]); the last group (index n_exp) has no expert, and its output rows
// are zero. Without `order` there is one group of all slots in their own order. A CTA's share
// of the slots is a chunk: up to C slots of one group. Chunks are numbered over the groups, and
// each warp finds its own from the offsets.
#pragma once

#include "qs_levels.cuh"

namespace qs {

struct MmArgs {
    const uint8_t* w;
    int64_t w_row, w_exp;  // bytes between weight rows / matrices
    const uint8_t* x;      // Q8_0 rows
    int64_t x_row;         // bytes
    int x_div;             // activation row of slot s: s / x_div
    int n, units;          // weight rows; 32-value units of a row
    int slots;
    const int* order;
    const int* offsets;
    int n_exp;
    void* out;             // slot s, column c at s * out_stride + c
    int64_t out_stride;
    int out_type;
    float* part;           // float32 results [slot][n] instead of out, or null
    int splits;            // CTAs that share a tile's rows (tiles only)
    const uint16_t* kgrid;
};

struct Chunk {
    int group;   // -1: no such chunk
    int lo, hi;  // positions in `order`
};

// chunk c of the numbering (all 32 lanes call it)
template <int C>
__device__ __forceinline__ Chunk find_chunk(const MmArgs& a, int c) {
    Chunk r{-1, 0, 0};
    if (!a.order) {
        r.lo = c * C;
        r.hi = min(r.lo + C, a.slots);
        r.group = r.lo < a.slots ? 0 : -1;
        return r;
    }
    const int lane = threadIdx.x & 31;
    int run = 0;
    for (int base = 0; base <= a.n_exp; base += 32) {
        const int e = base + lane;
        int lo = 0, hi = 0;
        if (e <= a.n_exp) {
            lo = __ldg(a.offsets + e);
            hi = e < a.n_exp ? __ldg(a.offsets + e + 1) : a.slots;
        }
        const int cnt = (hi - lo + C - 1) / C;
        int inc = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        const int first = run + inc - cnt;
        const unsigned hit = __ballot_sync(0xffffffffu, c >= first && c < first + cnt);
        if (hit) {
            const int l = __ffs(hit) - 1;
            const int g_first = __shfl_sync(0xffffffffu, first, l);
            r.group = base + l;
            r.lo = __shfl_sync(0xffffffffu, lo, l) + (c - g_first) * C;
            r.hi = min(r.lo + C, __shfl_sync(0xffffffffu, hi, l));
            return r;
        }
        run += __shfl_sync(0xffffffffu, inc, 31);
    }
    return r;
}

// the number of chunks is at most this (it depends on the offsets, which the host does not read)
inline int64_t max_chunks(const MmArgs& a, int c) {
    if (!a.order) return ((int64_t)a.slots + c - 1) / c;
    const int64_t groups = a.n_exp + 1 < a.slots ? a.n_exp + 1 : a.slots;
    return c == 1 ? a.slots : a.slots / c + groups;
}

__device__ __forceinline__ void store_val(void* p, int64_t i, int type, float v) {
    if (type == SRC_F32) static_cast<float*>(p)[i] = v;
    else if (type == SRC_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// 16 bytes at any address
__device__ __forceinline__ uint4 ld_16b(const uint8_t* p) {
    uint32_t w[4];
    ld_words<4, 1>(p, w);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ int sum16(const uint4& v) {
    const int one = 0x01010101;
    return __dp4a((int)v.x, one, __dp4a((int)v.y, one, __dp4a((int)v.z, one, __dp4a((int)v.w, one, 0))));
}

// shared memory that the kernel for few slots may use: (32 levels, a scale, up to 2 sums) per unit
// and slot, for up to 8 slots
constexpr int FEW_SMEM_MAX = 200 * 1024, FEW_SLOTS = 8, FEW_UNIT_MAX = 44;
cudaError_t launch_mm_few(int type, const MmArgs& a, const LaunchCtx& ctx);
cudaError_t launch_mm_tile(int type, const MmArgs& a, int bn, const LaunchCtx& ctx);
// out[token] = sum over its per_out slots that have an expert of weight * part
cudaError_t launch_mm_sum(const MmArgs& a, int per_out, const float* weights, const int* ids, const LaunchCtx& ctx);

#define QS_FOR_TYPES(X)                                                                                     \
    X(QS_Q4_0) X(QS_Q4_1) X(QS_Q5_0) X(QS_Q5_1) X(QS_Q8_0) X(QS_Q2_K) X(QS_Q3_K) X(QS_Q4_K) X(QS_Q5_K)      \
    X(QS_Q6_K) X(QS_IQ2_XXS) X(QS_IQ2_XS) X(QS_IQ2_S) X(QS_IQ3_XXS) X(QS_IQ3_S) X(QS_IQ4_XS)

}  // namespace qs
