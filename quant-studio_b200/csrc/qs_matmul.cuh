// Shared pieces of the packed products (qs_matmul_few.cu, qs_matmul_mid.cu, qs_matmul_tc.cuh).
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

#include <atomic>

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
    unsigned int* fault;   // the device's fault word
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
    constexpr int W = 4;  // windows of 32 groups whose offsets are on their way together
    for (int base = 0; base <= a.n_exp; base += 32 * W) {
        int lo[W], hi[W];
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int e = base + 32 * j + lane;
            lo[j] = e <= a.n_exp ? __ldg(a.offsets + e) : 0;
            hi[j] = e < a.n_exp ? __ldg(a.offsets + e + 1) : e == a.n_exp ? a.slots : 0;
        }
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int cnt = (hi[j] - lo[j] + C - 1) / C;
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
                r.group = base + 32 * j + l;
                r.lo = __shfl_sync(0xffffffffu, lo[j], l) + (c - g_first) * C;
                r.hi = min(r.lo + C, __shfl_sync(0xffffffffu, hi[j], l));
                return r;
            }
            run += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    return r;
}

// the number of chunks is at most this (it depends on the offsets, which the host does not read)
inline int64_t max_chunks(bool ordered, int64_t slots, int64_t n_exp, int c) {
    if (!ordered) return (slots + c - 1) / c;
    const int64_t groups = n_exp + 1 < slots ? n_exp + 1 : slots;
    return c == 1 ? slots : slots / c + groups;
}
inline int64_t max_chunks(const MmArgs& a, int c) { return max_chunks(a.order != nullptr, a.slots, a.n_exp, c); }

__device__ __forceinline__ void store_val(void* p, int64_t i, int type, float v) {
    if (type == SRC_F32) static_cast<float*>(p)[i] = v;
    else if (type == SRC_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// A slot's 128 columns from n0 on, 4 per lane, to element `at` of out; vec: all exist, 4-element aligned.
__device__ __forceinline__ void store_row4(void* out, int64_t at, int type, float4 v, int lane, int n0, int n, bool vec) {
    if (vec) {
        if (type == SRC_F32) {
            reinterpret_cast<float4*>(static_cast<float*>(out) + at)[lane] = v;
        } else if (type == SRC_F16) {
            const __half2 p = __floats2half2_rn(v.x, v.y), q = __floats2half2_rn(v.z, v.w);
            reinterpret_cast<uint2*>(static_cast<__half*>(out) + at)[lane] =
                make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
        } else {
            const __nv_bfloat162 p = __floats2bfloat162_rn(v.x, v.y), q = __floats2bfloat162_rn(v.z, v.w);
            reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + at)[lane] =
                make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
        }
    } else {
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (n0 + 4 * lane + c < n) store_val(out, at + 4 * lane + c, type, e[c]);
    }
}

// Dynamic shared memory beyond 48 KB for a kernel, asked for once per device (`asked`: bits of the
// devices, one word per kernel).
inline cudaError_t allow_smem(const void* kernel, int bytes, int device, std::atomic<unsigned long long>& asked) {
    if (device >= 0 && device < 64 && (asked.load(std::memory_order_relaxed) >> device) & 1ull) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device >= 0 && device < 64) asked.fetch_or(1ull << device, std::memory_order_relaxed);
    return e;
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
// and slot, for up to 4 slots
constexpr int FEW_SMEM_MAX = 200 * 1024, FEW_SLOTS = 4, FEW_UNIT_MAX = 44;
cudaError_t launch_mm_few(int type, const MmArgs& a, const LaunchCtx& ctx);
// up to 64 slots a matrix, for bfloat16 results 32 with superblocks (qs_matmul_mid.cu): tiles of bn = 8, 16, 32 or 64 slots; ws: mm_mid_workspace
// bytes; rows: activation rows
inline int64_t mm_mid_workspace(int64_t units, int64_t rows, int sums) { return rows * ((units + 3) / 4 * 4) * (32 + 4 * (1 + sums)); }
cudaError_t launch_mm_mid(int type, const MmArgs& a, int bn, int rows, void* ws, const LaunchCtx& ctx);
// tcgen05 tiles (qs_matmul_tc.cuh): tiles of bn slots; lo: both float16 parts of the activations. ws:
// mm_tc_workspace bytes for `chunks` chunks (the rows' powers of two lead); sums: sums of activations per unit
// (1 with minima, 2 with minima per 16 values, else 0), 32 to a stage
inline int64_t xs_bytes(int64_t chunks, int bn) { return (chunks * bn * 4 + 255) / 256 * 256; }
inline int64_t mm_tc_workspace(int64_t units, int64_t chunks, int bn, bool lo, int sums) {
    return xs_bytes(chunks, bn) + chunks * ((units + 1) / 2 + (units * sums + 31) / 32) * (int64_t)bn * 128 * (lo ? 2 : 1);
}
// by the file that holds the type
cudaError_t launch_mm_tc_legacy(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx);
cudaError_t launch_mm_tc_k(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx);
cudaError_t launch_mm_tc_k2(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx);
cudaError_t launch_mm_tc_iq(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx);
inline cudaError_t launch_mm_tc(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx) {
    switch (type) {
    case QS_Q4_0: case QS_Q4_1: case QS_Q5_0: case QS_Q5_1: case QS_Q8_0: return launch_mm_tc_legacy(type, a, bn, lo, ws, ctx);
    case QS_Q2_K: case QS_Q3_K: case QS_Q4_K: return launch_mm_tc_k(type, a, bn, lo, ws, ctx);
    case QS_Q5_K: case QS_Q6_K: case QS_IQ4_XS: return launch_mm_tc_k2(type, a, bn, lo, ws, ctx);
    default: return launch_mm_tc_iq(type, a, bn, lo, ws, ctx);
    }
}
// out[token] = sum over its per_out slots that have an expert of weight * part
cudaError_t launch_mm_sum(const MmArgs& a, int per_out, const float* weights, const int* ids, const LaunchCtx& ctx);

#define QS_FOR_TYPES(X)                                                                                     \
    X(QS_Q4_0) X(QS_Q4_1) X(QS_Q5_0) X(QS_Q5_1) X(QS_Q8_0) X(QS_Q2_K) X(QS_Q3_K) X(QS_Q4_K) X(QS_Q5_K)      \
    X(QS_Q6_K) X(QS_IQ2_XXS) X(QS_IQ2_XS) X(QS_IQ2_S) X(QS_IQ3_XXS) X(QS_IQ3_S) X(QS_IQ4_XS)

}  // namespace qs
