// Packed products for many slots on the 5th-generation tensor cores (tcgen05, float16 operands,
// float32 sums in tensor memory).
//
// Weights: integer levels are exact in float16, and so is level * sub-scale of the formats with one
// scale per superblock (at most 2048): for those D sums W' x over a superblock of 256 values (LO: half of it), and
//   acc[n, t] += d[n, superblock] * D[n, t]
// in float32 registers. Formats with a scale per 32 values are scaled and added every 32. Q6_K's
// level * sub-scale (up to 4096) is float16 hi + lo, exact together.
// Activations: scale * level has 19 bits; times a power of two per row (that takes the largest scale to 2^7 ..
// 2^8, values below 2^15) it is float16 hi + lo, exact together but for 2^-25, which is at most 2^-39 of 128 times the
// row's largest scale. LO: the
// products use both parts (Q6_K: hi hi, hi lo, lo hi), for float32 and float16 results. For
// bfloat16 results hi alone is multiplied: that rounds the activations to 11 bits, by at most 2^-11 of a value
// (or those 2^-25), 1/8 of the result's own rounding where the terms
// are of both signs (in the 2-norm 2.1e-4 and 1.66e-3). Q6_K's level * sub-scale above 2048 (5 % of the weights with
// sub-scales of 40 to 127) is rounded to 11 bits there as well.
// Minima: - ml[n, unit] * (sum of the unit's activations)[t, unit] is a product of its own, with K / 32 (K / 16
// for Q2_K) terms; it follows the levels as further stages of 32 terms, the weights' side times a power of two
// per row and stage. It nearly cancels the levels' product where the activations have one sign, so both sides are
// hi + lo for every result (22 bits; the hi parts are the stage's first 32 columns, the lo parts the others, and
// all four pairs are multiplied), and the sums are those of the activations as they are multiplied. With 11 bits
// of either, the error of Q4_K with 4096 values was 6e-4 of the result for normal activations and 3e-3 for
// equal ones.
//
// A pass over K = 32 of a 128 x 256 tile is 271 cycles of the matrix unit (540 with LO). Scaling every 32
// values by both operands' scales instead, with exact integers in D, was built first and took 1235 us
// for 2048 slots of Q4_K 14336 x 4096: three float32 operations per value and unit are 768 cycles
// (a packed f32x2 operation takes two), an SM has no more than 128 lanes.
//
// Roles in a CTA (one per SM, 20 warps):
//   warps 0-7    own the tile's sums: lane = weight row, each warp half of the columns
//   warps 8-15   unpack the weights, warps 8-11 the even stages, 12-15 the odd ones (thread = row, both
//                units of the stage: a stage's unpacking is mostly latency, so two are under way)
//   warp 16      issues the matrix products (and owns the tensor memory)
//   warp 17      copies the activations' stage (one bulk copy: float16 rows as the matrix unit reads
//                them), laid out beforehand by xpack_kernel
//   warps 18, 19 copy the weights' bytes (cp.async) in steps of RS stages: the 16-byte pieces that
//                cover a row's share wherever it starts, adjacent lanes adjacent pieces
// Stages are a ring in shared memory (full: unpacked + copied, empty: products done); the
// accumulators are a ring in tensor memory; the weights' scales are a longer ring of their own, which
// the unpacking can not lap: stage i waits for the products of stage i - NS, these for their accumulator,
// which the sums released NB accumulators ago. With GROUP stages to an accumulator the oldest scale that is
// still to be read is at most NS + (NB - 1) GROUP stages old (16 for tiles of 128 with GROUP = 4, else 10 at
// most), less than the ring's length. Every wait is bounded: one that runs out records bit 0 of the fault
// word and its role leaves; the roles behind it run out in turn, and the sums store a tile of NaN.
// Measured: 2048 slots of Q4_K 14336 x 4096 to bfloat16 344 us with xpack_kernel (11 us), 700 TFLOP/s, 42 % of the
// measured bf16 rate (338 us with minima of 11 bits); 4096 slots of 4096 x 4096 208 us; 1024 to float32 (LO) 99 us.
// The matrix unit is active for 43 % of the time. Without any unpacking or copying the loop took 247 us: a stage
// moves 105 KB through shared memory (operands read by the matrix unit, unpacked and copied data), 820 cycles at
// 128 bytes each, against 512 of products. Tiles of
// 256 columns halve what a column costs in unpacking. Pairs of CTAs that hold half of the columns' operand
// each (cta_group::2) move 74 KB per stage, but took 452 us: every stage then waits for arrivals from
// the other CTA.
// The order of the 32 values within a unit does not matter to the sum; both operands use the one
// that unpacks cheapest (word_halves).
#pragma once

#include <algorithm>
#include <cooperative_groups.h>

#include "qs_matmul.cuh"

namespace qs {

namespace {

namespace cg = cooperative_groups;

constexpr int TC_M = 128, TC_THREADS = 640;
constexpr int TC_SMEM = 227 * 1024;

template <int T, int BN, bool LO>
struct TcCfg {
    using L = Lv<T>;
    static constexpr bool SPLIT = LO && T == QS_Q6_K;
    static constexpr int SUMS = !L::HASMIN ? 0 : L::G16 ? 2 : 1;  // minima per unit
    // stages that share an accumulator (0: one per unit). The matrix unit adds with truncation: over 256
    // values that cost 4.6e-7 of a result, half of it over 128
    static constexpr int GROUP = !L::FOLD ? 0 : LO ? 2 : 4;
    static constexpr int A_BYTES = TC_M * 128, A_ALL = A_BYTES * (SPLIT ? 2 : 1), B_BYTES = BN * 128, X_BYTES = B_BYTES * (LO ? 2 : 1);
    static constexpr int STAGE = A_ALL + X_BYTES;
    // packed bytes: steps of RS stages (a superblock, or 4 blocks of 32), the bytes of a row's step and
    // the pitch of the pieces that cover them, an odd number of pieces against bank conflicts
    static constexpr int RS = L::QK == 256 ? 4 : 2, WB = RS * 64 / L::QK * L::BB;
    static constexpr int COVER = L::MAXAL >= 16 ? WB : (WB + 16 - L::MAXAL + 15) / 16 * 16, WP = COVER / 16 % 2 ? COVER : COVER + 16;
    static constexpr int RAW = TC_M * WP, RR = 2 * RAW <= 24 * 1024 ? 4 : 2;  // steps in the ring
    static constexpr int NB = BN == 256 ? 2 : 4;       // accumulators in tensor memory
    static constexpr int COLS = NB * BN;
    static constexpr int NS_MAX = 4;
    // ring of scales, [slot][unit][128]: longer than the stages that unpacking may be ahead of the sums
    static constexpr int LEAD = NS_MAX + (NB - 1) * (GROUP ? GROUP : 1), DR = LEAD < 16 ? 16 : 32;
    static constexpr int D_BYTES = DR * 2 * TC_M * 4;
    static constexpr int FIT = (TC_SMEM - 1024 - 512 - BN * 8 - D_BYTES - RR * RAW) / STAGE, NS = FIT > NS_MAX ? NS_MAX : FIT;
    // the sums of 256 columns are 128 registers a thread: registers move to their two warpgroups
    // (160, 160, 64, 64, 32 a thread of the 96 at launch)
    static constexpr int R_SUM = 160, R_UNPACK = 64, R_REST = 32, R_LAUNCH = 96;
    static_assert(2 * R_SUM + 2 * R_UNPACK + R_REST <= 5 * R_LAUNCH, "the shares are what the launch has");
    static constexpr int OUT_PITCH = TC_M + 4;
    static constexpr int BYTES = NS * STAGE + D_BYTES + RR * RAW + 1024;  // 1024 to align the ring
    static_assert(NS >= 2 && DR > NS + (NB - 1) * (GROUP ? GROUP : 1), "ring lengths");
    static_assert(BN * OUT_PITCH * 4 <= NS * STAGE, "the tile leaves through the same memory");
    // further stages with the minima of `units` units: 32 terms each
    __host__ __device__ static int min_blocks(int units) { return (units * SUMS + 31) / 32; }
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("{ .reg .b64 st; mbarrier.arrive.shared::cta.b64 st, [%0]; }" ::"r"(bar) : "memory");
}
// Completion of the phase of that parity; false (and the fault recorded) after a bounded number of
// polls, seconds beyond anything a running product needs.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, unsigned int* fault) {
    for (int it = 0; it < (1 << 20); it++) {
        uint32_t ok;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (it > 64) __nanosleep(64);
    }
    atomicOr(fault, 1u);
    return false;
}
// `bytes` from global to shared memory, completing on the barrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "{ .reg .b64 st; mbarrier.arrive.expect_tx.shared::cta.b64 st, [%3], %2; }\n"
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <class L>
__device__ __forceinline__ float base_of(const uint32_t* r) {
    if constexpr (L::FOLD) return L::base(r);
    else return 0.0f;
}
// Shared-memory operands K-major, rows of 128 bytes in the 128-byte swizzle: 8-row groups 1024
// bytes apart. a, b: addresses in 16-byte units
__device__ __forceinline__ void mma_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    constexpr uint32_t HI = (1024 >> 4) | (1u << 14) | (2u << 29);
    asm volatile(
        "{ .reg .pred p; .reg .b64 x, y; mov.b64 x, {%1, %5}; mov.b64 y, {%2, %5}; setp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p; }"
        ::"r"(d), "r"(a | 0x10000u), "r"(b | 0x10000u), "r"(idesc), "r"((uint32_t)add), "r"(HI) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr) : "memory");
}
// the loads' registers pass through the wait, so that nothing reads them before it
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}

// 4 byte levels as 4 float16, in the order b0 b2 b1 b3: a byte behind 0x64 is 1024 + byte
__device__ __forceinline__ void word_halves(uint32_t w, __half2 bias, __half2* h) {
    const uint32_t a = (w & 0x00FF00FFu) | 0x64006400u, b = ((w >> 8) & 0x00FF00FFu) | 0x64006400u;
    h[0] = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    h[1] = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
}
// the same, times sc plus less
__device__ __forceinline__ void word_fma(uint32_t w, __half2 sc, __half2 less, __half2* h) {
    const uint32_t a = (w & 0x00FF00FFu) | 0x64006400u, b = ((w >> 8) & 0x00FF00FFu) | 0x64006400u;
    h[0] = __hfma2(*reinterpret_cast<const __half2*>(&a), sc, less);
    h[1] = __hfma2(*reinterpret_cast<const __half2*>(&b), sc, less);
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// The slots' Q8_0 rows as the matrix unit reads them, [chunk][stage]: BN rows of 64 float16 values
// (two units) in the 128-byte swizzle, with LO the rows' low parts behind them; then as many stages as
// hold 32 sums of a unit's values each (or of its halves'), times 2^-7, their hi parts, then their lo parts.
// All times the row's power of two, whose inverse goes to xs[chunk][slot]. Rows without a slot stay as they
// are: their columns of the product are not stored. gridDim.z warps per row: each finds the largest scale, then
// takes every gridDim.z-th run of 32 units.
template <int BN, int SUMS, bool LO>
__global__ void __launch_bounds__(256) xpack_kernel(MmArgs a, uint8_t* out, float* xs) {
    constexpr int B_BYTES = BN * 128, X_BYTES = B_BYTES * (LO ? 2 : 1);
    const Chunk ch = find_chunk<BN>(a, blockIdx.y);
    if (ch.group < 0 || (a.order && ch.group == a.n_exp)) return;
    const int lane = threadIdx.x & 31, t = blockIdx.x * 8 + (threadIdx.x >> 5), stages = (a.units + 1) / 2;
    const int blocks = (a.units * SUMS + 31) / 32;
    if (ch.lo + t >= ch.hi) return;
    const int slot = a.order ? __ldg(a.order + ch.lo + t) : ch.lo + t;
    const uint8_t* row = a.x + (int64_t)(slot / a.x_div) * a.x_row;
    uint32_t top = 0;  // largest |scale| as float16 bits; above 0x7BFF: inf or NaN
    for (int u0 = lane; u0 < a.units; u0 += 32 * 8) {  // 8 loads under way
        uint32_t d[8];
#pragma unroll
        for (int j = 0; j < 8; j++) d[j] = u0 + 32 * j < a.units ? ld_u16<1>(row + (int64_t)(u0 + 32 * j) * 34) & 0x7FFFu : 0u;
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, d[j]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    // 2^(7 - exponent): scales below 2^8, values at most 2^15
    float up = 1.0f;
    if (top > 0 && top <= 0x7BFFu) up = __uint_as_float((uint32_t)(127 + 7 + 127 - (int)(__float_as_uint(h2f(top)) >> 23)) << 23);
    if (lane == 0 && blockIdx.z == 0) xs[(int64_t)blockIdx.y * BN + t] = 1.0f / up;
    uint8_t* o = out + (int64_t)blockIdx.y * (stages + blocks) * X_BYTES;
    auto put_sum = [&](int p, float v) {  // term p of the sums
        const int c = (p & 31) >> 3;
        uint8_t* at = o + (int64_t)(stages + (p >> 5)) * X_BYTES + t * 128 + (p & 7) * 2;
        const __half h = __float2half_rn(v);
        *reinterpret_cast<__half*>(at + ((c ^ (t & 7)) << 4)) = h;
        *reinterpret_cast<__half*>(at + (((4 + c) ^ (t & 7)) << 4)) = __float2half_rn(v - __half2float(h));
    };
    const int last = max(2 * stages, SUMS ? blocks * 32 / SUMS : 0);
    uint32_t next[9];  // the next unit's levels and scale
    auto load = [&](int u) {
#pragma unroll
        for (int e = 0; e < 9; e++) next[e] = 0;
        if (u < a.units) {
            ld_words<8, 1>(row + (int64_t)u * 34 + 2, next);
            next[8] = ld_u16<1>(row + (int64_t)u * 34);
        }
    };
    const int hop = 32 * gridDim.z;
    load(blockIdx.z * 32 + lane);
    for (int u = blockIdx.z * 32 + lane; u < last; u += hop) {
        uint32_t q[8];
#pragma unroll
        for (int e = 0; e < 8; e++) q[e] = next[e];
        const float d = h2f(next[8]) * up;
        load(u + hop);
        float half_sum[2] = {0.0f, 0.0f};  // of the values as they are multiplied (multiples of one small step: exact)
        if (u < 2 * stages) {
            uint8_t* st = o + (int64_t)(u >> 1) * X_BYTES;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    // halves of word 2 c + e / 2: bytes 0, 2 or 1, 3
                    const uint32_t w = q[2 * c + (e >> 1)] >> (8 * (e & 1));
                    const float v0 = d * (float)(int8_t)w, v1 = d * (float)(int8_t)(w >> 16);
                    const __half2 h = __floats2half2_rn(v0, v1);
                    const float2 f = __half22float2(h);
                    hi[e] = h2_bits(h);
                    if constexpr (SUMS > 0 && !LO) half_sum[c >> 1] += f.x + f.y;
                    if constexpr (LO) lo[e] = h2_bits(__floats2half2_rn(v0 - f.x, v1 - f.y));
                }
                uint8_t* p = st + t * 128 + (((4 * (u & 1) + c) ^ (t & 7)) << 4);
                *reinterpret_cast<uint4*>(p) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (LO) *reinterpret_cast<uint4*>(p + B_BYTES) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        if constexpr (SUMS > 0) {
            if constexpr (LO) {
                half_sum[0] = d * (float)sum16(make_uint4(q[0], q[1], q[2], q[3]));
                half_sum[1] = d * (float)sum16(make_uint4(q[4], q[5], q[6], q[7]));
            }
            if (u < blocks * 32 / SUMS) {
                if constexpr (SUMS == 1) put_sum(u, 0.0078125f * (half_sum[0] + half_sum[1]));
                else {
                    put_sum(2 * u, 0.0078125f * half_sum[0]);
                    put_sum(2 * u + 1, 0.0078125f * half_sum[1]);
                }
            }
        }
    }
}

template <int T, int BN, bool LO>
__global__ void __launch_bounds__(TC_THREADS, 1) tc_kernel(MmArgs a, const uint8_t* xp, const float* xs) {
    using L = Lv<T>;
    using C = TcCfg<T, BN, LO>;
    constexpr int UPB = L::QK / 32, SUMS = C::SUMS, NS = C::NS, NB = C::NB, GROUP = C::GROUP, RS = C::RS, RR = C::RR;
    constexpr int HALF = BN / 2;  // columns of a warp
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * NS + 2 * NB + 2 * RR];
    __shared__ uint32_t s_tmem;
    __shared__ int s_slot[BN];   // the tile's slots and their rows' powers of two
    __shared__ float s_up[BN];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Chunk ch = find_chunk<BN>(a, blockIdx.y);
    if (ch.group < 0) return;  // the CTAs of a cluster share the chunk
    const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
    uint8_t* const ring_p = smem_raw + (ring - smem_u32(smem_raw));
    float* const scales = reinterpret_cast<float*>(ring_p + NS * C::STAGE);
    const uint8_t* const bytes_p = ring_p + NS * C::STAGE + C::D_BYTES;
    const uint32_t full = smem_u32(bars), empty = full + 8 * NS, acc_full = empty + 8 * NS, acc_empty = acc_full + 8 * NB,
                   raw_full = acc_empty + 8 * NB, raw_empty = raw_full + 8 * RR;
    if (tid == 0) {
        for (int s = 0; s < NS; s++) {
            mbar_init(full + 8 * s, 4 + 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < NB; b++) {
            mbar_init(acc_full + 8 * b, 2);
            mbar_init(acc_empty + 8 * b, 8);
        }
        for (int r = 0; r < RR; r++) {
            mbar_init(raw_full + 8 * r, 64);
            mbar_init(raw_empty + 8 * r, 8);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    {
        const bool some = !a.order || ch.group < a.n_exp;
        for (int t = tid; t < BN; t += TC_THREADS) {
            s_slot[t] = ch.lo + t < ch.hi ? (a.order ? __ldg(a.order + ch.lo + t) : ch.lo + t) : 0;
            s_up[t] = some && ch.lo + t < ch.hi ? __ldg(xs + (int64_t)blockIdx.y * BN + t) : 1.0f;
        }
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "n"(C::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;

    const int n0 = blockIdx.x * TC_M, cnt = ch.hi - ch.lo;
    const int stages = (a.units + 1) / 2, per = ((stages + a.splits - 1) / a.splits + 3) & ~3;  // whole superblocks
    const int blocks = C::min_blocks(a.units);
    const bool real = !a.order || ch.group < a.n_exp;
    // this CTA's stages: k0 .. of the levels (`main` of them), then its share of the minima's blocks
    const int k0 = min((int)blockIdx.z * per, stages), main = real ? min(per, stages - k0) : 0;
    const int e0 = blocks * (int)blockIdx.z / a.splits, extra = real ? blocks * ((int)blockIdx.z + 1) / a.splits - e0 : 0;
    const int total = main + extra;
    // whether unit uu of stage i begins / ends an accumulator
    auto begins = [&](int i, int uu) { return i >= main ? uu == 0 : !GROUP || (uu == 0 && i % (GROUP ? GROUP : 1) == 0); };
    auto ends = [&](int i, int uu) { return i >= main ? uu == 1 : !GROUP || (uu == 1 && (i % (GROUP ? GROUP : 1) == GROUP - 1 || i + 1 == main)); };

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_REST));
        if (warp == 16) {
            // the whole warp runs the loop, so that addresses stay in uniform registers; one lane issues
            const bool leader = elect_one();
            // D float32, A and B float16 K-major, N = BN, M = 128
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TC_M >> 4) << 24);
            int b = 0, b_ph = 1;  // accumulator, parity of its last release
            int s = 0, ph = 0;
            for (int i = 0; i < total; i++) {
                if (!mbar_wait(full + 8 * s, ph, a.fault)) break;
                const uint32_t st = (ring + s * C::STAGE) >> 4;
                bool ok = true;
#pragma unroll
                for (int uu = 0; uu < 2; uu++) {
                    const bool first = begins(i, uu);
                    if (first && !(ok = mbar_wait(acc_empty + 8 * b, b_ph, a.fault))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < 2; kk++) {
                            constexpr uint32_t X = C::A_ALL >> 4;
                            const uint32_t at = st + uu * 4 + kk * 2;
                            if (SUMS > 0 && i >= main) {  // one part of the minima with both of the sums
                                mma_f16(tmem + b * BN, at, st + kk * 2 + X, idesc, !first || kk > 0);
                                mma_f16(tmem + b * BN, at, st + kk * 2 + X + 4, idesc, true);
                                continue;
                            }
                            mma_f16(tmem + b * BN, at, at + X, idesc, !first || kk > 0);
                            if constexpr (LO) mma_f16(tmem + b * BN, at, at + X + (C::B_BYTES >> 4), idesc, true);
                            if constexpr (C::SPLIT) mma_f16(tmem + b * BN, at + (C::A_BYTES >> 4), at + X, idesc, true);
                        }
                    }
                    if (ends(i, uu)) {
                        // the products' end, and a release of its own for the scales that came with `full`
                        if (leader) {
                            mma_commit(acc_full + 8 * b);
                            mbar_arrive(acc_full + 8 * b);
                        }
                        if (++b == NB) {
                            b = 0;
                            b_ph ^= 1;
                        }
                    }
                }
                if (!ok) break;
                if (leader) mma_commit(empty + 8 * s);
                if (++s == NS) {
                    s = 0;
                    ph ^= 1;
                }
            }
            __syncwarp();
            asm volatile("bar.sync 1, 288;" ::: "memory");  // the sums' warps have read their last accumulator
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::COLS));
        } else if (warp >= 18) {
            // one warp half of the rows each; adjacent lanes take adjacent pieces of a row
            constexpr int P = C::COVER / 16, HALF_ROWS = TC_M / 2;
            const int first = (warp - 18) * HALF_ROWS, rows = min(HALF_ROWS, a.n - n0 - first), steps = (main + RS - 1) / RS;
            const uint8_t* w = a.w + (real ? ch.group * a.w_exp : 0) + (int64_t)(n0 + first) * a.w_row;
            const int64_t len = (int64_t)a.units / UPB * L::BB;
            for (int k = 0; k < steps; k++) {
                const int r = k % RR;
                if (!mbar_wait(raw_empty + 8 * r, ((k / RR) & 1) ^ 1, a.fault)) break;
                const int64_t lo = (int64_t)(k0 / RS + k) * C::WB, hi = min(lo + C::WB, len);
                const uint32_t dst = smem_u32(bytes_p) + r * C::RAW + first * C::WP;
#pragma unroll 4
                for (int i = lane; i < HALF_ROWS * P; i += 32) {
                    const int t = i / P, piece = i - t * P;
                    const uint8_t* row = w + t * a.w_row;
                    const uint8_t* q = (const uint8_t*)((uintptr_t)(row + lo) & ~(uintptr_t)15) + piece * 16;
                    if (t < rows && q < row + hi) cp16(dst + t * C::WP + piece * 16, q);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(raw_full + 8 * r) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else if (warp == 17 && lane == 0) {
            const uint8_t* src = xp + (int64_t)blockIdx.y * (stages + blocks) * C::X_BYTES;
            int i = 0;
            for (; i < total; i++) {
                const int s = i % NS;
                if (!mbar_wait(empty + 8 * s, ((i / NS) & 1) ^ 1, a.fault)) break;
                const int k = i < main ? k0 + i : stages + e0 + i - main;
                bulk_load(ring + s * C::STAGE + C::A_ALL, src + (int64_t)k * C::X_BYTES, i < main ? C::X_BYTES : C::B_BYTES, full + 8 * s);
            }
            // no copy outlives the CTA
            for (int j = max(0, i - NS); j < i; j++) mbar_wait(full + 8 * (j % NS), (j / NS) & 1, a.fault);
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_UNPACK));
        const int row = tid & 127, odd = (warp - 8) >> 2;  // weight row of the tile, stages 2 j + odd
        const bool mine = n0 + row < a.n;
        const uint8_t* w = a.w + (real ? ch.group * a.w_exp : 0) + (int64_t)(mine ? n0 + row : 0) * a.w_row;
        auto put = [&](uint8_t* st, int c, const __half2* h) {  // piece c of the row
            *reinterpret_cast<uint4*>(st + row * 128 + ((c ^ (row & 7)) << 4)) = make_uint4(h2_bits(h[0]), h2_bits(h[1]), h2_bits(h[2]), h2_bits(h[3]));
        };
        // k0 is a whole number of steps, so stage i is stage i % RS of step i / RS
        auto unpack = [&](int i, uint8_t* st, const uint8_t* bytes) {
            const uint32_t off = L::MAXAL >= 16 ? 0 : (uint32_t)(uintptr_t)(w + (int64_t)(k0 / RS + i / RS) * C::WB) & 15;
            uint32_t r[2][L::WORDS];
#pragma unroll
            for (int uu = 0; uu < 2; uu++) {
                const int in = 2 * (i % RS) + uu;
                if (mine && 2 * (k0 + i) + uu < a.units) {
                    L::template load<L::MAXAL, true>(bytes + row * C::WP + off + in / UPB * L::BB, in % UPB, r[uu]);
                } else {
#pragma unroll
                    for (int e = 0; e < L::WORDS; e++) r[uu][e] = 0;  // zero scales
                }
            }
#pragma unroll
            for (int uu = 0; uu < 2; uu++) {
                const int j = (2 * (i % RS) + uu) % UPB;
                uint32_t q[8];
                float dl[2], ml[2];
                L::levels(r[uu], j, a.kgrid, q, dl, ml);
                // the bytes' float16 is 1024 + byte; less the bias, times the sub-scale: one exact operation
                // where bias * sub-scale is a float16 (not for Q6_K's factors of up to 128)
                constexpr float BIAS = L::SIGNED ? 1152.0f : 1024.0f;
                constexpr uint32_t FLIP = L::SIGNED ? 0x80808080u : 0u;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    __half2 h[4];
                    if constexpr (L::FOLD && T != QS_Q6_K) {
                        const float sub = (float)L::sub(r[uu], j, c >> 1);
                        const __half2 sc = __float2half2_rn(sub), less = __float2half2_rn(-BIAS * sub);
                        word_fma(q[2 * c] ^ FLIP, sc, less, h);
                        word_fma(q[2 * c + 1] ^ FLIP, sc, less, h + 2);
                    } else {
                        const __half2 bias = __float2half2_rn(BIAS);
                        word_halves(q[2 * c] ^ FLIP, bias, h);
                        word_halves(q[2 * c + 1] ^ FLIP, bias, h + 2);
                        if constexpr (L::FOLD) {
                            const __half2 sc = __float2half2_rn((float)L::sub(r[uu], j, c >> 1));
                            __half2 p[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) p[e] = __hmul2(h[e], sc);
                            if constexpr (C::SPLIT) {  // the product's rounding error, exact in float16
#pragma unroll
                                for (int e = 0; e < 4; e++) h[e] = __hfma2(h[e], sc, __hneg2(p[e]));
                                put(st + C::A_BYTES, 4 * uu + c, h);
                            }
#pragma unroll
                            for (int e = 0; e < 4; e++) h[e] = p[e];
                        }
                    }
                    put(st, 4 * uu + c, h);
                }
                scales[((i % C::DR) * 2 + uu) * TC_M + row] = L::FOLD ? base_of<L>(r[uu]) : dl[0];
            }
        };
        // 32 minima of the row (negated) times a power of two, hi and lo parts; its inverse (and the sums' 2^7)
        // as the scale
        auto unpack_minima = [&](int i, uint8_t* st) {
            if constexpr (SUMS > 0) {
                constexpr int PER = UPB * SUMS;  // minima of a block
                const int p0 = (e0 + i - main) * 32;
                float m[32], top = 0.0f;
#pragma unroll
                for (int p = 0; p < 32; p += PER) {
                    const bool in = mine && p0 + p < a.units * SUMS;
#pragma unroll
                    for (int j = 0; j < PER; j++) m[p + j] = 0.0f;
                    if (in) L::template minima<L::MAXAL>(w + (int64_t)((p0 + p) / PER) * L::BB, m + p);
                }
#pragma unroll
                for (int p = 0; p < 32; p++) top = fmaxf(top, fabsf(m[p]));
                float up = 1.0f;  // the largest below 2^11
                if (top > 0.0f && top < INFINITY) up = __uint_as_float((uint32_t)(127 + 10 + 127 - (int)(__float_as_uint(top) >> 23)) << 23);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    __half2 h[4], l[4];
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const float v0 = -m[8 * c + 2 * x] * up, v1 = -m[8 * c + 2 * x + 1] * up;
                        h[x] = __floats2half2_rn(v0, v1);
                        const float2 f = __half22float2(h[x]);
                        l[x] = __floats2half2_rn(v0 - f.x, v1 - f.y);
                    }
                    put(st, c, h);
                    put(st, 4 + c, l);
                }
                scales[((i % C::DR) * 2 + 1) * TC_M + row] = 128.0f / up;
            }
        };
        int s = odd % NS, ph = odd / NS & 1 ? 0 : 1;  // stage of the ring, the parity that its last use ended with
        for (int i = odd; i < total; i += 2) {
            if (!mbar_wait(empty + 8 * s, ph, a.fault)) break;
            uint8_t* st = ring_p + s * C::STAGE;
            if (i < main) {
                const int k = i / RS, r = k % RR;
                if (i % RS == odd && !mbar_wait(raw_full + 8 * r, (k / RR) & 1, a.fault)) break;
                unpack(i, st, bytes_p + r * C::RAW);
                if (i % RS == RS - 2 + odd) {  // this half's last stage of the step
                    __syncwarp();
                    if (lane == 0) mbar_arrive(raw_empty + 8 * r);
                }
            } else {
                unpack_minima(i, st);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * s);
            s += 2;
            if (s >= NS) {
                s -= NS;
                ph ^= 1;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::R_SUM));
        const int row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * HALF;
        constexpr int NBT = HALF / 16;
        f32x2 acc[HALF / 2];
#pragma unroll
        for (int i = 0; i < HALF / 2; i++) acc[i] = 0ull;
        int b = 0, b_ph = 0;  // accumulator to read, its parity
        bool ok = true;
        for (int i = 0; i < total && ok; i++) {
            for (int uu = 0; uu < 2; uu++) {
                if (!ends(i, uu)) continue;
                if (!(ok = mbar_wait(acc_full + 8 * b, b_ph, a.fault))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const f32x2 dl = f2_splat(*(volatile float*)&scales[((i % C::DR) * 2 + uu) * TC_M + row]);
                const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + b * BN + c0;
#pragma unroll
                for (int bt = 0; bt < NBT; bt++) {
                    uint32_t r[16];
                    tmem_ld16(at + 16 * bt, r);
                    tmem_wait_ld(r);
                    if (bt == NBT - 1) {  // the last loads are in registers
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_empty + 8 * b);
                    }
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        acc[bt * 8 + c] = f2_fma(dl, f2_pack(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), acc[bt * 8 + c]);
                }
                if (++b == NB) {
                    b = 0;
                    b_ph ^= 1;
                }
            }
        }
        if (!ok) {  // no sums: the result must not pass for one
#pragma unroll
            for (int i = 0; i < HALF / 2; i++) acc[i] = f2_splat(NAN);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.sync 1, 288;" ::: "memory");

        // the tile through shared memory (all copies and products have been waited for), so that a
        // slot's columns leave in whole rows
        float* o = reinterpret_cast<float*>(ring_p);
#pragma unroll
        for (int i = 0; i < HALF / 2; i++) {
            float x0, x1;
            f2_unpack(acc[i], x0, x1);
            o[(c0 + 2 * i) * C::OUT_PITCH + row] = x0;
            o[(c0 + 2 * i + 1) * C::OUT_PITCH + row] = x1;
        }
        const int rank = blockIdx.z, ranks = a.splits;
        if (ranks > 1) cg::this_cluster().sync();
        else asm volatile("bar.sync 2, 256;" ::: "memory");
        void* out = a.part ? (void*)a.part : a.out;
        const int type = a.part ? (int)SRC_F32 : a.out_type;
        const int64_t stride = a.part ? a.n : a.out_stride;
        const bool vec = n0 + TC_M <= a.n && stride % 4 == 0 && ((uintptr_t)out & 15) == 0;
        if (ranks == 1) {
#pragma unroll 4
            for (int t = warp; t < cnt; t += 8) {
                const float4 v = *reinterpret_cast<const float4*>(o + t * C::OUT_PITCH + 4 * lane);
                const float u = s_up[t];
                store_row4(out, (int64_t)s_slot[t] * stride + n0, type, make_float4(v.x * u, v.y * u, v.z * u, v.w * u), lane, n0, a.n, vec);
            }
        } else {
            for (int t = warp * ranks + rank; t < cnt; t += 8 * ranks) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                for (int r = 0; r < ranks; r++) {
                    const float4 f = *reinterpret_cast<const float4*>(cg::this_cluster().map_shared_rank(o, r) + t * C::OUT_PITCH + 4 * lane);
                    v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
                }
                const float u = s_up[t];
                store_row4(out, (int64_t)s_slot[t] * stride + n0, type, make_float4(v.x * u, v.y * u, v.z * u, v.w * u), lane, n0, a.n, vec);
            }
        }
    }
    __syncwarp();
    if (a.splits > 1) {
        if (warp >= 8) cg::this_cluster().sync();  // the sums' warps have met the others' already
        cg::this_cluster().sync();  // the others may still read this tile
    }
}

template <int T, int BN, bool LO>
cudaError_t launch_tc_t(const MmArgs& a, void* ws, const LaunchCtx& ctx) {
    using C = TcCfg<T, BN, LO>;
    const int64_t chunks = max_chunks(a, BN);
    if (chunks > 65535) return cudaErrorInvalidConfiguration;
    float* xs = static_cast<float*>(ws);
    uint8_t* xp = static_cast<uint8_t*>(ws) + xs_bytes(chunks, BN);
    // warps per row: up to four CTAs per SM in all, each warp with a run of 32 units at least
    const int64_t rows8 = BN / 8 * chunks, runs = (a.units + 31) / 32, z = std::max<int64_t>(1, std::min(runs, 4 * 148 / rows8));
    xpack_kernel<BN, C::SUMS, LO><<<dim3(BN / 8, (unsigned)chunks, (unsigned)z), 256, 0, ctx.stream>>>(a, xp, xs);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    auto kernel = tc_kernel<T, BN, LO>;
    static std::atomic<unsigned long long> asked{0};
    if ((e = allow_smem((const void*)kernel, C::BYTES, ctx.device, asked)) != cudaSuccess) return e;
    // the warpgroups' shares must be there at launch
    static const int regs = [] {
        cudaFuncAttributes f;
        return cudaFuncGetAttributes(&f, tc_kernel<T, BN, LO>) == cudaSuccess ? f.numRegs : 0;
    }();
    if (regs < C::R_LAUNCH) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((a.n + TC_M - 1) / TC_M), (unsigned)chunks, (unsigned)a.splits);
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = C::BYTES;
    cfg.stream = ctx.stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = (unsigned)a.splits;
    cfg.attrs = at;
    cfg.numAttrs = a.splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, static_cast<const uint8_t*>(xp), static_cast<const float*>(xs));
}

template <int T>
cudaError_t launch_tc(const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx) {
    if (lo) return launch_tc_t<T, 128, true>(a, ws, ctx);
    return bn == 128 ? launch_tc_t<T, 128, false>(a, ws, ctx) : launch_tc_t<T, 256, false>(a, ws, ctx);
}

}  // namespace

}  // namespace qs
