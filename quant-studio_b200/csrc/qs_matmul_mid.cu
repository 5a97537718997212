// Packed products for up to 64 slots per weight matrix (32 for bfloat16 results from superblocks): 16
// weight rows per warp on the integer tensor cores (mma.sync s8).
//
// Both operands are 8-bit levels, so a unit's 32 products sum exactly in the s32 accumulator; the
// accumulator starts at the bit pattern of 1.5 * 2^23 and its result is that float plus the sum
// (|sum| <= 32 * 128 * 128 < 2^22). Scaled by dl * dx it is added to the float32 sums in
// registers: three float operations per value and unit, four with minima. With so few slots the weights'
// bytes and their unpacking are the work, not these operations.
//
// Each warp runs by itself over its 16 rows: the packed bytes come by cp.async, 16-byte pieces that
// cover a row's share of a step wherever it starts, into the warp's own ring; 4 units at a time are unpacked
// into the warp's own 16 x 128 levels and multiplied. The warps of a CTA share only the activations'
// levels and scales (laid out by pack_kernel), SL units of all slots at a time. A long row of few
// tiles is split over the CTAs of a cluster, which add their tiles through distributed shared memory in
// rank order.
//
// Measured (with pack_kernel, 3 us): Q4_0 4096 x 4096 10.7 us for 5 slots, 19 us for 64; Q6_K 4096 x 14336 35 us
// for 7. Of the 15 us of a CTA with 64 slots and 16 units of Q4_0, set-up is 1.5 us, staging 1.5 us, unpacking
// 2 us, products 5 us (the float operations, 12 cycles per 16 x 8 product), joining the cluster's tiles 3 us;
// fewer CTAs per cluster, or one per SM, are slower (24 against 21 us). For Q6_K
// shared memory is what is busiest (66 % of its cycles, 37 % of them conflicts of the unpacking's words at unaligned
// addresses), the issue slots are at 49 % with 16 warps per SM; pieces of 8 bytes, which halve the bank conflicts, cost more
// copies than they save (38 us), and 16-byte loads without conflicts more selects (36 us).
#include <cooperative_groups.h>

#include "qs_matmul.cuh"

namespace qs {

namespace {

namespace cg = cooperative_groups;

constexpr int MID_WARPS = 8, MID_ROWS = 16 * MID_WARPS, MID_THREADS = 32 * MID_WARPS;
constexpr int MID_SMEM = 111 * 1024;  // two CTAs per SM

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4_or_zero(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
constexpr int MAGIC_BITS = 0x4B400000;  // 12582912.0f = 1.5 * 2^23
// 16 x 8 products over 32 (16) levels; c0, c1: row g, columns 2t, 2t + 1; c2, c3: row g + 8
__device__ __forceinline__ void mma32(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(MAGIC_BITS));
}
__device__ __forceinline__ void mma16(int* c, uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(b0), "r"(MAGIC_BITS));
}

template <int T, int NT>
struct MidCfg {
    using L = Lv<T>;
    static constexpr int BN = 8 * NT, H = L::G16 ? 2 : 1, SUMS = L::HASMIN ? H : 0;
    // a step: one superblock, or 4 blocks of 32; a row's bytes and the pitch of the pieces that cover
    // them, an odd number of pieces against bank conflicts
    static constexpr int RU = L::QK == 256 ? 8 : 4, WB = RU * 32 / L::QK * L::BB;
    static constexpr int COVER = L::MAXAL >= 16 ? WB : (WB + 16 - L::MAXAL + 15) / 16 * 16, WP = COVER / 16 % 2 ? COVER : COVER + 16;
    static constexpr int RAW = 16 * WP, RR = RAW <= 2048 ? 3 : 2;  // bytes of a step, steps in the ring
    // a warp's own memory: ring, levels of 4 units, scales [unit][half][16] each twice (a packed
    // pair), minima alike
    static constexpr int LEVELS = 16 * 128, SC = 4 * H * 16 * 8;
    static constexpr int OWN = RR * RAW + LEVELS + SC * (SUMS ? 2 : 1);
    // activations per unit of all slots: levels, planes [scale, sums][slot]; the slots' level rows are
    // 16 bytes longer than their units
    static constexpr int UNIT_X = BN * 32 + (1 + SUMS) * BN * 4;
    static constexpr int FIT = (MID_SMEM - MID_WARPS * OWN - BN * 16) / UNIT_X / 8 * 8, SL = FIT > 128 ? 128 : FIT;
    static constexpr int PITCH = SL * 32 + 16, OFF_XD = BN * PITCH, OFF_OWN = OFF_XD + (1 + SUMS) * SL * BN * 4;
    // the two units of 4 that half warp x unpacks: neighbours share their bytes in most formats, Q6_K's
    // low nibbles belong to units j and j + 2
    __device__ static int item(int x, int h) { return T == QS_Q6_K ? x + 2 * h : 2 * x + h; }
    static constexpr int OUT_PITCH = MID_ROWS + 4;
    static constexpr int BYTES = OFF_OWN + MID_WARPS * OWN;
    static_assert(SL >= 8, "a superblock of activations");
    static_assert(BN * OUT_PITCH * 4 <= BYTES, "the tile leaves through the same memory");
};

template <int T, int NT>
__global__ void __launch_bounds__(MID_THREADS, 2) mid_kernel(MmArgs a, const int8_t* xq, const float* xd, int64_t x_plane, int units_pad) {
    using L = Lv<T>;
    using C = MidCfg<T, NT>;
    constexpr int UPB = L::QK / 32, H = C::H, SUMS = C::SUMS, BN = C::BN, RU = C::RU, RR = C::RR, SL = C::SL;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_slot[BN], s_row[BN];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tg = lane & 3;
    const Chunk ch = find_chunk<BN>(a, blockIdx.y);
    if (ch.group < 0) return;  // the CTAs of a cluster share the chunk
    const int n0 = blockIdx.x * MID_ROWS, nw = n0 + warp * 16, cnt = ch.hi - ch.lo;
    for (int i = tid; i < BN; i += MID_THREADS) {
        const int slot = i < cnt ? (a.order ? __ldg(a.order + ch.lo + i) : ch.lo + i) : -1;
        s_slot[i] = slot;
        s_row[i] = slot < 0 ? -1 : slot / a.x_div;
    }
    const int eights = (a.units + 7) / 8, per = (eights + a.splits - 1) / a.splits;
    const bool real = !a.order || ch.group < a.n_exp;
    const int u0 = min((int)blockIdx.z * per * 8, a.units), u1 = real ? min(u0 + per * 8, a.units) : u0;
    const int wrows = min(16, a.n - nw);  // may be <= 0
    const uint8_t* w = a.w + (real ? ch.group * a.w_exp : 0) + (int64_t)nw * a.w_row;
    const int64_t w_len = (int64_t)a.units / UPB * L::BB;
    uint8_t* const own = smem + C::OFF_OWN + warp * C::OWN;
    uint8_t* const lev = own + RR * C::RAW;
    f32x2* const sdl = reinterpret_cast<f32x2*>(lev + C::LEVELS);
    f32x2* const sml = sdl + 4 * H * 16;
    const uint32_t own_a = smem_u32(own), lev_a = smem_u32(lev), x_a = smem_u32(smem);

    const int steps = (u1 - u0 + RU - 1) / RU;
    auto fetch = [&](int k) {
        if (k < steps) {
            constexpr int P = C::COVER / 16;
            const int64_t lo = (int64_t)(u0 / RU + k) * C::WB, hi = min(lo + C::WB, w_len);
            const uint32_t dst = own_a + k % RR * C::RAW;
#pragma unroll
            for (int i0 = 0; i0 < 16 * P; i0 += 32) {
                const int i = i0 + lane, t = i / P, piece = i - t * P;
                const uint8_t* row = w + t * a.w_row;
                const uint8_t* q = (const uint8_t*)((uintptr_t)(row + lo) & ~(uintptr_t)15) + piece * 16;
                if (t < wrows && q < row + hi) cp16(dst + t * C::WP + piece * 16, q);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int k = 0; k < RR; k++) fetch(k);

    f32x2 acc[NT][2];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = 0ull;
    const f32x2 nmagic = f2_splat(-12582912.0f);
    const int ir = lane & 15;  // the row that this lane unpacks

    int k = 0;
    for (int us = u0; us < u1; us += SL) {
        const int nu = min(SL, u1 - us);
        __syncthreads();  // the last slice is used up
        // all copies under way at once; rows without a slot are filled with zeros
#pragma unroll 8
        for (int i = tid; i < BN * SL * 2; i += MID_THREADS) {
            const int t = i / (SL * 2), c = i % (SL * 2), row = s_row[t];
            if (c < nu * 2) cp16_or_zero(x_a + t * C::PITCH + c * 16, xq + ((int64_t)max(row, 0) * units_pad + us) * 32 + c * 16, row >= 0);
        }
#pragma unroll 4
        for (int i = tid; i < (1 + SUMS) * BN * SL; i += MID_THREADS) {
            const int u = i % SL, t = i / SL % BN, p = i / (SL * BN), row = s_row[t];
            if (u < nu) cp4_or_zero(x_a + C::OFF_XD + ((p * SL + u) * BN + t) * 4, xd + p * x_plane + (int64_t)max(row, 0) * units_pad + us + u, row >= 0);
        }
        cp_commit();
        cp_wait<0>();
        __syncthreads();
        for (int su = 0; su < nu; su += RU, k++) {
            cp_wait<RR - 1>();
            __syncwarp();
            const uint8_t* raw = own + k % RR * C::RAW;
            const int live = min(RU, nu - su);
            const uint32_t off = L::MAXAL >= 16 ? 0 : (uint32_t)(uintptr_t)(w + ir * a.w_row + (int64_t)(u0 / RU + k) * C::WB) & 15;
#pragma unroll
            for (int q4 = 0; q4 < RU; q4 += 4) {
                if (RU > 4 && q4 >= live) break;
                // both units' bytes first: units that share bytes load them once
                uint32_t r[2][L::WORDS];
#pragma unroll
                for (int h2 = 0; h2 < 2; h2++) {
                    const int in = q4 + C::item(lane >> 4, h2);
                    if (ir < wrows && in < live) {
                        L::template load<L::MAXAL, true>(raw + ir * C::WP + off + in / UPB * L::BB, in % UPB, r[h2]);
                    } else {
#pragma unroll
                        for (int e = 0; e < L::WORDS; e++) r[h2][e] = 0;  // zero scales
                    }
                }
                __syncwarp();  // the last 4 units are used up
#pragma unroll
                for (int h2 = 0; h2 < 2; h2++) {
                    const int u = C::item(lane >> 4, h2);
                    uint32_t q[8];
                    float dl[2], ml[2];
                    L::levels(r[h2], (q4 + u) % UPB, a.kgrid, q, dl, ml);
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        *reinterpret_cast<uint4*>(lev + ir * 128 + (((2 * u + h) ^ (ir & 7)) << 4)) = make_uint4(q[4 * h], q[4 * h + 1], q[4 * h + 2], q[4 * h + 3]);
                    const int pos = ((ir & 7) << 1) | (ir >> 3);  // rows g and g + 8 side by side
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        sdl[(u * H + h) * 16 + pos] = f2_splat(dl[h]);
                        if constexpr (SUMS > 0) sml[(u * H + h) * 16 + pos] = f2_splat(-ml[h]);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    if (q4 + u >= live) break;
                    const int ux = su + q4 + u;  // unit of the slice
                    uint32_t ar[4];
                    ldsm4(lev_a + (lane & 15) * 128 + (((2 * u + (lane >> 4)) ^ (lane & 7)) << 4), ar);
                    f32x2 dl[H][2], ml[H][2];
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(sdl + (u * H + h) * 16 + 2 * g);
                        dl[h][0] = v.x;
                        dl[h][1] = v.y;
                        if constexpr (SUMS > 0) {
                            const ulonglong2 m = *reinterpret_cast<const ulonglong2*>(sml + (u * H + h) * 16 + 2 * g);
                            ml[h][0] = m.x;
                            ml[h][1] = m.y;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NT; j += 2) {
                        // lanes 0-7: slots j, first half; 8-15: second half; 16-31: slots j + 1 (of one tile: again)
                        uint32_t b[4];
                        ldsm4(x_a + ((NT > 1 ? (j + (lane >> 4)) * 8 : 0) + (lane & 7)) * C::PITCH + ux * 32 + ((lane >> 3) & 1) * 16, b);
#pragma unroll
                        for (int jj = 0; jj < (NT > 1 ? 2 : 1); jj++) {
                            const float* xp = reinterpret_cast<const float*>(smem + C::OFF_XD) + ux * BN + (j + jj) * 8 + 2 * tg;
                            const f32x2 x0 = *reinterpret_cast<const f32x2*>(xp);
#pragma unroll
                            for (int h = 0; h < H; h++) {
                                int c4[4];
                                if constexpr (H == 1) mma32(c4, ar, b[2 * jj], b[2 * jj + 1]);
                                else mma16(c4, ar[2 * h], ar[2 * h + 1], b[2 * jj + h]);
                                f32x2 xs = 0ull;
                                if constexpr (SUMS > 0) xs = *reinterpret_cast<const f32x2*>(xp + (1 + h) * SL * BN);
#pragma unroll
                                for (int v = 0; v < 2; v++) {
                                    const f32x2 s = f2_add(f2_pack(__int_as_float(c4[2 * v]), __int_as_float(c4[2 * v + 1])), nmagic);
                                    acc[j + jj][v] = f2_fma(s, f2_mul_z(dl[h][v], x0), acc[j + jj][v]);
                                    if constexpr (SUMS > 0) acc[j + jj][v] = f2_fma(ml[h][v], xs, acc[j + jj][v]);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();  // all lanes have read this step's bytes
            fetch(k + RR);
        }
    }
    cp_wait<0>();
    __syncthreads();

    // the tile through shared memory, so that a slot's columns leave in whole rows
    float* o = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int v = 0; v < 2; v++) {
            float x0, x1;
            f2_unpack(acc[j][v], x0, x1);
            o[(j * 8 + 2 * tg) * C::OUT_PITCH + warp * 16 + v * 8 + g] = x0;
            o[(j * 8 + 2 * tg + 1) * C::OUT_PITCH + warp * 16 + v * 8 + g] = x1;
        }
    const int rank = blockIdx.z, ranks = a.splits;
    if (ranks > 1) cg::this_cluster().sync();
    else __syncthreads();
    void* out = a.part ? (void*)a.part : a.out;
    const int type = a.part ? (int)SRC_F32 : a.out_type;
    const int64_t stride = a.part ? a.n : a.out_stride;
    const bool vec = n0 + MID_ROWS <= a.n && stride % 4 == 0 && ((uintptr_t)out & 15) == 0;
    for (int t = warp * ranks + rank; t < cnt; t += MID_WARPS * ranks) {
        float4 v = *reinterpret_cast<const float4*>(o + t * C::OUT_PITCH + 4 * lane);
        if (ranks > 1) {
            v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int r = 0; r < ranks; r++) {
                const float4 f = *reinterpret_cast<const float4*>(cg::this_cluster().map_shared_rank(o, r) + t * C::OUT_PITCH + 4 * lane);
                v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
            }
        }
        store_row4(out, (int64_t)s_slot[t] * stride + n0, type, v, lane, n0, a.n, vec);
    }
    if (ranks > 1) cg::this_cluster().sync();  // the others may still read this tile
}

// Q8_0 rows -> 16-byte aligned levels [row][units_pad] and planes [scale, scale * sum of levels (of a
// half)][row][units_pad]. One thread per half unit.
__global__ void __launch_bounds__(256) pack_kernel(const uint8_t* x, int64_t x_row, int rows, int units, int units_pad, int8_t* xq, float* xd,
                                                   int64_t plane, int planes) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t unit = i >> 1;
    const int h = (int)(i & 1);
    const bool live = unit < (int64_t)rows * units_pad;
    const int64_t row = live ? unit / units_pad : 0;
    const int u = (int)(unit - row * units_pad);
    uint4 q = make_uint4(0, 0, 0, 0);
    float d = 0.0f;
    if (live && u < units) {
        const uint8_t* b = x + row * x_row + (int64_t)u * 34;
        q = ld_16b(b + 2 + 16 * h);
        d = h2f(ld_u16<1>(b));
    }
    const int s = sum16(q), o = __shfl_xor_sync(0xffffffffu, s, 1);
    if (!live) return;
    reinterpret_cast<uint4*>(xq)[unit * 2 + h] = q;
    if (h == 0) xd[unit] = d;
    if (planes == 2 && h == 0) xd[plane + unit] = d * (float)(s + o);
    if (planes == 3) xd[(1 + h) * plane + unit] = d * (float)s;
}

template <int T, int NT>
cudaError_t launch_mid_t(const MmArgs& a, const int8_t* xq, const float* xd, int64_t plane, int units_pad, const LaunchCtx& ctx) {
    using C = MidCfg<T, NT>;
    const int64_t chunks = max_chunks(a, C::BN);
    if (chunks > 65535) return cudaErrorInvalidConfiguration;
    static std::atomic<unsigned long long> asked{0};
    const cudaError_t e = allow_smem((const void*)mid_kernel<T, NT>, C::BYTES, ctx.device, asked);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((a.n + MID_ROWS - 1) / MID_ROWS), (unsigned)chunks, (unsigned)a.splits);
    cfg.blockDim = dim3(MID_THREADS);
    cfg.dynamicSmemBytes = C::BYTES;
    cfg.stream = ctx.stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = (unsigned)a.splits;
    cfg.attrs = at;
    cfg.numAttrs = a.splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, mid_kernel<T, NT>, a, xq, xd, plane, units_pad);
}

template <int T>
cudaError_t launch_mid(const MmArgs& a, int bn, int rows, void* ws, const LaunchCtx& ctx) {
    const int units_pad = (a.units + 3) / 4 * 4;
    int8_t* xq = static_cast<int8_t*>(ws);
    const int64_t plane = (int64_t)rows * units_pad;
    float* xd = reinterpret_cast<float*>(xq + plane * 32);
    const int64_t threads = plane * 2;
    pack_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, ctx.stream>>>(a.x, a.x_row, rows, a.units, units_pad, xq, xd, plane, 1 + MidCfg<T, 1>::SUMS);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return bn == 8    ? launch_mid_t<T, 1>(a, xq, xd, plane, units_pad, ctx)
           : bn == 16 ? launch_mid_t<T, 2>(a, xq, xd, plane, units_pad, ctx)
           : bn == 32 ? launch_mid_t<T, 4>(a, xq, xd, plane, units_pad, ctx)
                      : launch_mid_t<T, 8>(a, xq, xd, plane, units_pad, ctx);
}

}  // namespace

cudaError_t launch_mm_mid(int type, const MmArgs& a, int bn, int rows, void* ws, const LaunchCtx& ctx) {
    switch (type) {
#define X(T) case T: return launch_mid<T>(a, bn, rows, ws, ctx);
        QS_FOR_TYPES(X)
#undef X
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qs
