// Packed products for many slots: tiles of 128 weight rows x BN slots on the integer tensor
// cores (mma.sync s8).
//
// Both operands are 8-bit levels, so a unit's 32 products sum exactly in the s32 accumulator;
// the accumulator starts at the bit pattern of 1.5 * 2^23 and its result is that float plus the
// sum (|sum| <= 32 * 128 * 128 < 2^22), so one packed add gives two sums as floats. They are
// scaled by dl * dx and added to the float32 tile in registers: per 16 x 8 x 32 product three
// pairs of packed float operations (add, scale product, fused multiply-add), plus one pair for
// formats with minima. A tensor-memory accumulator can not take this sum: its scale changes
// every 32 values in both operands, and reading it back that often costs more than the
// register form (an s32 tile of 128 x 256 is 256 cycles of tensor-memory reads against 128 of
// products). Measured alone, product and scaling together run at 1387 TOP/s, 83 % of the bf16
// matrix rate of this GPU.
//
// A CTA of 16 warps walks the row in steps of 256 values (8 units). The packed bytes of both
// operands come by cp.async, 16-byte pieces that cover a row's share of a step wherever it starts,
// into a ring of stages; each step they are unpacked once (levels with 16-byte pieces swizzled
// by the row, scales and scaled level sums), and then multiplied. All global latency hides in the
// ring, so the two phases run from shared memory. A long row of few tiles is split over the CTAs of
// a cluster, which add their tiles through distributed shared memory in rank order.
#include <cooperative_groups.h>

#include "qs_matmul.cuh"

namespace qs {

namespace {

namespace cg = cooperative_groups;

constexpr int TM = 128, TU = 8, TILE_THREADS = 512;  // weight rows, units per step
constexpr int SMEM_MAX = 227 * 1024;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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

template <int T, int BN>
struct TileCfg {
    using L = Lv<T>;
    static constexpr int H = L::G16 ? 2 : 1, SUMS = L::HASMIN ? H : 0;
    static constexpr int WM = BN == 32 ? 8 : 4, WN = 16 / WM;  // warps along the rows / the slots
    static constexpr int MT = TM / WM / 16, NT = BN / WN / 8;  // 16 x 8 products of a warp
    // packed bytes of a step per row, and the pitch of the pieces that cover them
    static constexpr int WB = TU * 32 / L::QK * L::BB, XB = TU * 34;
    static constexpr int WP = (WB + 15 + 15) / 16 * 16, XP = (XB + 15 + 15) / 16 * 16;
    // unpacked: levels of the weights and the slots (256 bytes a row), weight scales
    // [unit][half][128] each twice (a packed pair), minima alike, slot planes [scale, sums][unit][BN]
    static constexpr int OFF_X = TM * 256, OFF_DL = OFF_X + BN * 256, OFF_ML = OFF_DL + TU * H * TM * 8;
    static constexpr int OFF_XD = OFF_ML + (SUMS ? TU * H * TM * 8 : 0), OFF_RAW = OFF_XD + (1 + SUMS) * TU * BN * 4;
    static constexpr int STAGE = TM * WP + BN * XP;
    static constexpr int FIT = (SMEM_MAX - OFF_RAW - 2 * BN * 8 - 64) / STAGE, NS = FIT > 5 ? 5 : FIT;
    static constexpr int OUT_PITCH = TM + 4;
    static constexpr int BYTES = OFF_RAW + NS * STAGE;
    static_assert(NS >= 2, "two stages at least");
    static_assert(BN * OUT_PITCH * 4 <= BYTES, "the tile leaves through the same memory");
};

// place of a weight row's scale: rows g and g + 8 of a 16-row product side by side
__device__ __forceinline__ int scale_pos(int row) { return (row & ~15) | ((row & 7) << 1) | ((row >> 3) & 1); }

template <int T, int BN>
__global__ void __launch_bounds__(TILE_THREADS, 1) tile_kernel(MmArgs a) {
    using L = Lv<T>;
    using C = TileCfg<T, BN>;
    constexpr int UPB = L::QK / 32, H = C::H, SUMS = C::SUMS, MT = C::MT, NT = C::NT, NS = C::NS;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_slot[BN];
    __shared__ const uint8_t* s_x[BN];  // the slots' activation rows
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Chunk ch = find_chunk<BN>(a, blockIdx.y);
    if (ch.group < 0) return;  // the CTAs of a cluster share the chunk
    const int n0 = blockIdx.x * TM, cnt = ch.hi - ch.lo;
    for (int i = tid; i < BN; i += TILE_THREADS) {
        const int slot = i < cnt ? (a.order ? __ldg(a.order + ch.lo + i) : ch.lo + i) : -1;
        s_slot[i] = slot;
        s_x[i] = slot < 0 ? nullptr : a.x + (int64_t)(slot / a.x_div) * a.x_row;
    }
    __syncthreads();
    const int steps = (a.units + TU - 1) / TU, per = (steps + a.splits - 1) / a.splits;
    const int k0 = blockIdx.z * per;
    const bool real = !a.order || ch.group < a.n_exp;
    const int k1 = real ? min(k0 + per, steps) : k0;
    const uint8_t* w = a.w + (real ? ch.group * a.w_exp : 0) + (int64_t)n0 * a.w_row;
    const int wrows = min(TM, a.n - n0);
    const int wm = warp % C::WM, wn = warp / C::WM, g = lane >> 2, tg = lane & 3;

    // the 16-byte pieces that hold bytes [lo, hi) of a row
    auto cover = [&](const uint8_t* row, int64_t lo, int64_t hi, uint32_t dst, int piece) {
        const uint8_t* p = row + lo;
        const uint8_t* q = p - ((uintptr_t)p & 15) + piece * 16;
        if (q < row + hi) cp16(dst + piece * 16, q);
    };
    const int64_t w_len = (int64_t)a.units / UPB * L::BB, x_len = (int64_t)a.units * 34;
    auto fetch = [&](int k) {
        if (k < k1) {
            const uint32_t st = smem_u32(smem) + C::OFF_RAW + (k - k0) % NS * C::STAGE;
            for (int i = tid; i < TM * (C::WP / 16); i += TILE_THREADS) {
                const int row = i / (C::WP / 16), piece = i % (C::WP / 16);
                if (row < wrows) cover(w + row * a.w_row, (int64_t)k * C::WB, min((int64_t)(k + 1) * C::WB, w_len), st + row * C::WP, piece);
            }
            for (int i = tid; i < BN * (C::XP / 16); i += TILE_THREADS) {
                const int t = i / (C::XP / 16), piece = i % (C::XP / 16);
                if (t < cnt) cover(s_x[t], (int64_t)k * C::XB, min((int64_t)(k + 1) * C::XB, x_len), st + TM * C::WP + t * C::XP, piece);
            }
        }
        cp_commit();
    };

    f32x2 acc[MT][NT][2];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j][0] = acc[i][j][1] = 0ull;
#pragma unroll
    for (int s = 0; s < NS; s++) fetch(k0 + s);
    const f32x2 nmagic = f2_splat(-12582912.0f);
    const uint32_t base = smem_u32(smem);

    for (int k = k0; k < k1; k++) {
        cp_wait<NS - 1>();
        __syncthreads();  // this step's bytes are there, the last step's levels are used up
        const uint8_t* st = smem + C::OFF_RAW + (k - k0) % NS * C::STAGE;
        const int live = min(TU, a.units - k * TU);
#pragma unroll
        for (int i = 0; i < TM * TU / TILE_THREADS; i++) {
            const int item = tid + i * TILE_THREADS, row = item / TU, u = item % TU;
            uint32_t q[8];
            float dl[2], ml[2];
            if (row < wrows && u < live) {
                const uint8_t* p = w + row * a.w_row + (int64_t)k * C::WB;
                uint32_t raw[L::WORDS];
                L::template load<L::MAXAL, true>(st + row * C::WP + ((uintptr_t)p & 15) + u / UPB * L::BB, u % UPB, raw);
                L::levels(raw, u % UPB, a.kgrid, q, dl, ml);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) q[j] = 0;
                dl[0] = dl[1] = ml[0] = ml[1] = 0.0f;
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
                *reinterpret_cast<uint4*>(smem + row * 256 + (((2 * u + h) ^ (row & 7)) << 4)) = make_uint4(q[4 * h], q[4 * h + 1], q[4 * h + 2], q[4 * h + 3]);
#pragma unroll
            for (int h = 0; h < H; h++) {
                reinterpret_cast<f32x2*>(smem + C::OFF_DL)[(u * H + h) * TM + scale_pos(row)] = f2_splat(dl[h]);
                if constexpr (SUMS > 0) reinterpret_cast<f32x2*>(smem + C::OFF_ML)[(u * H + h) * TM + scale_pos(row)] = f2_splat(-ml[h]);
            }
        }
        for (int item = tid; item < BN * TU; item += TILE_THREADS) {
            const int t = item / TU, u = item % TU;
            uint32_t q[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            float d = 0.0f;
            if (t < cnt && u < live) {
                const uint8_t* p = st + TM * C::WP + t * C::XP + ((uintptr_t)(s_x[t] + (int64_t)k * C::XB) & 15) + u * 34;
                ld_words<8, 1, true>(p + 2, q);
                d = h2f(ld_u16<1, true>(p));
            }
            const uint4 qa = make_uint4(q[0], q[1], q[2], q[3]), qb = make_uint4(q[4], q[5], q[6], q[7]);
            *reinterpret_cast<uint4*>(smem + C::OFF_X + t * 256 + (((2 * u) ^ (t & 7)) << 4)) = qa;
            *reinterpret_cast<uint4*>(smem + C::OFF_X + t * 256 + (((2 * u + 1) ^ (t & 7)) << 4)) = qb;
            float* xd = reinterpret_cast<float*>(smem + C::OFF_XD) + u * BN + t;
            xd[0] = d;
            if constexpr (SUMS == 1) xd[TU * BN] = d * (float)(sum16(qa) + sum16(qb));
            if constexpr (SUMS == 2) {
                xd[TU * BN] = d * (float)sum16(qa);
                xd[2 * TU * BN] = d * (float)sum16(qb);
            }
        }
        __syncthreads();
        fetch(k + NS);
#pragma unroll
        for (int u = 0; u < TU; u++) {
            uint32_t b[NT][2];
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
                // lanes 0-7: slots j, first half; 8-15: second half; 16-31: slots j + 1
                const int t = wn * (BN / C::WN) + (j + (lane >> 4)) * 8 + (lane & 7), c = 2 * u + ((lane >> 3) & 1);
                uint32_t r[4];
                ldsm4(base + C::OFF_X + t * 256 + ((c ^ (t & 7)) << 4), r);
                b[j][0] = r[0]; b[j][1] = r[1];
                b[j + 1][0] = r[2]; b[j + 1][1] = r[3];
            }
            f32x2 xd[1 + SUMS][NT];
#pragma unroll
            for (int p = 0; p < 1 + SUMS; p++)
#pragma unroll
                for (int j = 0; j < NT; j++)
                    xd[p][j] = *reinterpret_cast<const f32x2*>(smem + C::OFF_XD + ((p * TU + u) * BN + wn * (BN / C::WN) + j * 8 + 2 * tg) * 4);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const int row = wm * (TM / C::WM) + i * 16 + (lane & 15), c = 2 * u + (lane >> 4);
                uint32_t ar[4];
                ldsm4(base + row * 256 + ((c ^ (row & 7)) << 4), ar);
                f32x2 dl[H][2], ml[H][2];
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const int o = ((u * H + h) * TM + wm * (TM / C::WM) + i * 16 + 2 * g) * 8;
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(smem + C::OFF_DL + o);
                    dl[h][0] = v.x;
                    dl[h][1] = v.y;
                    if constexpr (SUMS > 0) {
                        const ulonglong2 m = *reinterpret_cast<const ulonglong2*>(smem + C::OFF_ML + o);
                        ml[h][0] = m.x;
                        ml[h][1] = m.y;
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        int c4[4];
                        if constexpr (H == 1) mma32(c4, ar, b[j][0], b[j][1]);
                        else mma16(c4, ar[2 * h], ar[2 * h + 1], b[j][h]);
#pragma unroll
                        for (int v = 0; v < 2; v++) {
                            const f32x2 s = f2_add(f2_pack(__int_as_float(c4[2 * v]), __int_as_float(c4[2 * v + 1])), nmagic);
                            acc[i][j][v] = f2_fma(s, f2_mul_z(dl[h][v], xd[0][j]), acc[i][j][v]);
                            if constexpr (SUMS > 0) acc[i][j][v] = f2_fma(ml[h][v], xd[1 + h][j], acc[i][j][v]);
                        }
                    }
            }
        }
    }
    cp_wait<0>();
    __syncthreads();

    // the tile through shared memory, so that a slot's columns leave in whole rows
    float* o = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int v = 0; v < 2; v++) {
                const int row = wm * (TM / C::WM) + i * 16 + v * 8 + g, t = wn * (BN / C::WN) + j * 8 + 2 * tg;
                float x0, x1;
                f2_unpack(acc[i][j][v], x0, x1);
                o[t * C::OUT_PITCH + row] = x0;
                o[(t + 1) * C::OUT_PITCH + row] = x1;
            }
    const int rank = blockIdx.z, ranks = a.splits;
    if (ranks > 1) cg::this_cluster().sync();
    else __syncthreads();
    void* out = a.part ? (void*)a.part : a.out;
    const int type = a.part ? (int)SRC_F32 : a.out_type;
    const int64_t stride = a.part ? a.n : a.out_stride;
    const bool vec = n0 + TM <= a.n && stride % 4 == 0 && ((uintptr_t)out & 15) == 0;
    for (int t = warp * ranks + rank; t < cnt; t += TILE_THREADS / 32 * ranks) {
        const int64_t at = (int64_t)s_slot[t] * stride + n0;
        float4 v = *reinterpret_cast<const float4*>(o + t * C::OUT_PITCH + 4 * lane);
        if (ranks > 1) {
            v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int r = 0; r < ranks; r++) {
                const float4 f = *reinterpret_cast<const float4*>(cg::this_cluster().map_shared_rank(o, r) + t * C::OUT_PITCH + 4 * lane);
                v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
            }
        }
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
                if (n0 + 4 * lane + c < a.n) store_val(out, at + 4 * lane + c, type, e[c]);
        }
    }
    if (ranks > 1) cg::this_cluster().sync();  // the others may still read this tile
}

// One thread per VEC columns of an output row: the slots in order.
template <int VEC>
__global__ void __launch_bounds__(256) sum_kernel(MmArgs a, int per_out, const float* weights, const int* ids, int n_vec) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, outs = a.slots / per_out;
    if (i >= outs * n_vec) return;
    const int64_t r = i / n_vec;
    const int c = (int)(i - r * n_vec) * VEC;
    float sum[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) sum[v] = 0.0f;
    constexpr int B = 4;  // slots whose loads are in flight together
    for (int j0 = 0; j0 < per_out; j0 += B) {
        float p[B][VEC], wt[B];
        bool use[B];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int64_t slot = r * per_out + j0 + b;
            const bool in = j0 + b < per_out;
            use[b] = in && (unsigned)__ldg(ids + (in ? slot : 0)) < (unsigned)a.n_exp;
            wt[b] = in ? __ldg(weights + slot) : 0.0f;
            const float* q = a.part + (in ? slot : 0) * a.n + c;
            if constexpr (VEC == 4) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(q));
                p[b][0] = f.x; p[b][1] = f.y; p[b][2] = f.z; p[b][3] = f.w;
            } else {
                p[b][0] = __ldg(q);
            }
        }
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int v = 0; v < VEC; v++)
                if (use[b]) sum[v] = __fmaf_rn(wt[b], p[b][v], sum[v]);
    }
#pragma unroll
    for (int v = 0; v < VEC; v++) store_val(a.out, r * a.out_stride + c + v, a.out_type, sum[v]);
}

template <int T, int BN>
cudaError_t launch_tile_t(const MmArgs& a, const LaunchCtx& ctx) {
    using C = TileCfg<T, BN>;
    const int64_t chunks = max_chunks(a, BN);
    if (chunks > 65535) return cudaErrorInvalidConfiguration;
    cudaError_t e = cudaFuncSetAttribute(tile_kernel<T, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((a.n + TM - 1) / TM), (unsigned)chunks, (unsigned)a.splits);
    cfg.blockDim = dim3(TILE_THREADS);
    cfg.dynamicSmemBytes = C::BYTES;
    cfg.stream = ctx.stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = (unsigned)a.splits;
    cfg.attrs = at;
    cfg.numAttrs = a.splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, tile_kernel<T, BN>, a);
}

template <int T>
cudaError_t launch_tile(const MmArgs& a, int bn, const LaunchCtx& ctx) {
    return bn == 32 ? launch_tile_t<T, 32>(a, ctx) : bn == 64 ? launch_tile_t<T, 64>(a, ctx) : launch_tile_t<T, 128>(a, ctx);
}

}  // namespace

cudaError_t launch_mm_tile(int type, const MmArgs& a, int bn, const LaunchCtx& ctx) {
    switch (type) {
#define X(T) case T: return launch_tile<T>(a, bn, ctx);
        QS_FOR_TYPES(X)
#undef X
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_mm_sum(const MmArgs& a, int per_out, const float* weights, const int* ids, const LaunchCtx& ctx) {
    const bool v4 = a.n % 4 == 0;
    const int n_vec = v4 ? a.n / 4 : a.n;
    const int64_t threads = (int64_t)(a.slots / per_out) * n_vec;
    const unsigned blocks = (unsigned)((threads + 255) / 256);
    if (v4) sum_kernel<4><<<blocks, 256, 0, ctx.stream>>>(a, per_out, weights, ids, n_vec);
    else sum_kernel<1><<<blocks, 256, 0, ctx.stream>>>(a, per_out, weights, ids, n_vec);
    return cudaGetLastError();
}

}  // namespace qs
