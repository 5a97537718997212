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
// A CTA of 8 warps walks the row in steps of 128 values (4 units), two stages in shared memory:
// the next step's levels are unpacked from the blocks to registers, and its activations are
// copied (cp.async), before this step's products.
#include "qs_matmul.cuh"

namespace qs {

namespace {

constexpr int TM = 128, TU = 4, TILE_THREADS = 256;  // weight rows, units per step

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
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
    static constexpr int WM = BN == 128 ? 2 : 4, WN = 8 / WM;  // warps along the rows / the slots
    static constexpr int MT = TM / WM / 16, NT = BN / WN / 8;  // 16 x 8 products of a warp
    // one stage: levels of the weights and the slots (128-byte rows, 16-byte pieces swizzled by
    // the row), weight scales [unit][half][128] each twice (a packed pair), minima alike, slot
    // planes [plane][unit][BN]
    static constexpr int OFF_X = TM * 128, OFF_DL = OFF_X + BN * 128, OFF_ML = OFF_DL + TU * H * TM * 8;
    static constexpr int OFF_XD = OFF_ML + (SUMS ? TU * H * TM * 8 : 0);
    static constexpr int STAGE = OFF_XD + (1 + SUMS) * TU * BN * 4;
    static constexpr int OUT_PITCH = TM + 4;
    static constexpr int BYTES = 2 * STAGE > BN * OUT_PITCH * 4 ? 2 * STAGE : BN * OUT_PITCH * 4;
};

// place of a weight row's scale: rows g and g + 8 of a 16-row product side by side
__device__ __forceinline__ int scale_pos(int row) { return (row & ~15) | ((row & 7) << 1) | ((row >> 3) & 1); }

template <int T, int BN>
__global__ void __launch_bounds__(TILE_THREADS, BN == 128 ? 1 : 2) tile_kernel(MmArgs a) {
    using L = Lv<T>;
    using C = TileCfg<T, BN>;
    constexpr int UPB = L::QK / 32, H = C::H, SUMS = C::SUMS, MT = C::MT, NT = C::NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_slot[BN], s_row[BN];  // output slots and activation rows of the tile
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Chunk ch = find_chunk<BN>(a, blockIdx.y);
    if (ch.group < 0) return;
    const int n0 = blockIdx.x * TM, cnt = ch.hi - ch.lo;
    for (int i = tid; i < BN; i += TILE_THREADS) {
        const int slot = i < cnt ? (a.order ? __ldg(a.order + ch.lo + i) : ch.lo + i) : -1;
        s_slot[i] = slot;
        s_row[i] = slot < 0 ? -1 : slot / a.x_div;
    }
    __syncthreads();
    const int steps = a.units_pad / TU, per = (steps + a.splits - 1) / a.splits;
    const int k0 = blockIdx.z * per, k1 = min(k0 + per, steps);
    const bool real = !a.order || ch.group < a.n_exp;
    const uint8_t* w = a.w + (real ? ch.group * a.w_exp : 0);
    const int wm = warp % C::WM, wn = warp / C::WM, g = lane >> 2, tg = lane & 3;

    f32x2 acc[MT][NT][2];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j][0] = acc[i][j][1] = 0ull;

    // weight items of a step: (row, unit), 2 per thread; 4 adjacent lanes one row. The block
    // bytes are loaded a step ahead and unpacked behind the products that cover their latency.
    uint32_t raw[2][L::WORDS];
    auto load_w = [&](int step) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int item = tid + i * TILE_THREADS, row = item >> 2, u = step * TU + (item & 3);
            if (n0 + row < a.n && u < a.units)
                L::template load<L::MAXAL>(w + (int64_t)(n0 + row) * a.w_row + (int64_t)(u / UPB) * L::BB, u % UPB, raw[i]);
            else
#pragma unroll
                for (int j = 0; j < L::WORDS; j++) raw[i][j] = 0;  // zero scales
        }
    };
    auto put_w = [&](int step, uint8_t* st) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int item = tid + i * TILE_THREADS, row = item >> 2, u = item & 3;
            uint32_t q[8];
            float dl[2], ml[2];
            L::levels(raw[i], (step * TU + u) % UPB, a.kgrid, q, dl, ml);
#pragma unroll
            for (int h = 0; h < 2; h++)
                *reinterpret_cast<uint4*>(st + row * 128 + (((2 * u + h) ^ (row & 7)) << 4)) = make_uint4(q[4 * h], q[4 * h + 1], q[4 * h + 2], q[4 * h + 3]);
#pragma unroll
            for (int h = 0; h < H; h++) {
                reinterpret_cast<f32x2*>(st + C::OFF_DL)[(u * H + h) * TM + scale_pos(row)] = f2_splat(dl[h]);
                if constexpr (SUMS > 0) reinterpret_cast<f32x2*>(st + C::OFF_ML)[(u * H + h) * TM + scale_pos(row)] = f2_splat(-ml[h]);
            }
        }
    };
    // a thread's copies: piece tid & 7 of the levels of slots tid / 8, tid / 8 + 32, ...; the planes
    // by (plane, slot, unit). The sources advance by one step's bytes.
    constexpr int XC = BN * 8 / TILE_THREADS, DC = ((1 + SUMS) * TU * BN + TILE_THREADS - 1) / TILE_THREADS;
    int xrow[XC];
#pragma unroll
    for (int i = 0; i < XC; i++) xrow[i] = s_row[(tid >> 3) + i * (TILE_THREADS / 8)];
    int drow[DC];
#pragma unroll
    for (int i = 0; i < DC; i++) drow[i] = s_row[((tid + i * TILE_THREADS) >> 2) % BN];
    const int xpitch = a.units_pad * 32;
    auto copy_x = [&](int step, uint8_t* st) {
        const uint32_t base = smem_u32(st);
#pragma unroll
        for (int i = 0; i < XC; i++) {
            const int t = (tid >> 3) + i * (TILE_THREADS / 8), c = tid & 7;
            cp16(base + C::OFF_X + t * 128 + ((c ^ (t & 7)) << 4), a.xq + (int64_t)max(xrow[i], 0) * xpitch + (step * 128 + c * 16), xrow[i] >= 0);
        }
#pragma unroll
        for (int i = 0; i < DC; i++) {
            const int j = tid + i * TILE_THREADS, u = j & 3, t = (j >> 2) % BN, p = (j >> 2) / BN;
            if (DC * TILE_THREADS == (1 + SUMS) * TU * BN || j < (1 + SUMS) * TU * BN)
                cp4(base + C::OFF_XD + ((p * TU + u) * BN + t) * 4, a.xd + p * a.x_plane + (int64_t)max(drow[i], 0) * a.units_pad + (step * TU + u), drow[i] >= 0);
        }
        cp_commit();
    };

    if (real && k0 < k1) {
        copy_x(k0, smem);
        load_w(k0);
        put_w(k0, smem);
        cp_wait_all();
        __syncthreads();
        const f32x2 nmagic = f2_splat(-12582912.0f);
        for (int k = k0; k < k1; k++) {
            uint8_t* st = smem + ((k - k0) & 1) * C::STAGE;
            uint8_t* nx = smem + ((k - k0 + 1) & 1) * C::STAGE;
            const bool more = k + 1 < k1;
            if (more) {
                copy_x(k + 1, nx);
                load_w(k + 1);
            }
            const uint32_t base = smem_u32(st);
#pragma unroll
            for (int u = 0; u < TU; u++) {
                uint32_t b[NT][2];
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    // lanes 0-7: slots j, first half; 8-15: second half; 16-31: slots j + 1
                    const int t = wn * (BN / C::WN) + (j + (lane >> 4)) * 8 + (lane & 7), c = 2 * u + ((lane >> 3) & 1);
                    uint32_t r[4];
                    ldsm4(base + C::OFF_X + t * 128 + ((c ^ (t & 7)) << 4), r);
                    b[j][0] = r[0]; b[j][1] = r[1];
                    b[j + 1][0] = r[2]; b[j + 1][1] = r[3];
                }
                f32x2 xd[1 + SUMS][NT];
#pragma unroll
                for (int p = 0; p < 1 + SUMS; p++)
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        xd[p][j] = *reinterpret_cast<const f32x2*>(st + C::OFF_XD + ((p * TU + u) * BN + wn * (BN / C::WN) + j * 8 + 2 * tg) * 4);
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const int row = wm * (TM / C::WM) + i * 16 + (lane & 15), c = 2 * u + (lane >> 4);
                    uint32_t ar[4];
                    ldsm4(base + row * 128 + ((c ^ (row & 7)) << 4), ar);
                    f32x2 dl[H][2], ml[H][2];
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const int o = ((u * H + h) * TM + wm * (TM / C::WM) + i * 16 + 2 * g) * 8;
                        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(st + C::OFF_DL + o);
                        dl[h][0] = v.x;
                        dl[h][1] = v.y;
                        if constexpr (SUMS > 0) {
                            const ulonglong2 m = *reinterpret_cast<const ulonglong2*>(st + C::OFF_ML + o);
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
            if (more) put_w(k + 1, nx);
            cp_wait_all();
            __syncthreads();
        }
    }

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
    __syncthreads();
    void* out = a.part ? (void*)(a.part + (int64_t)blockIdx.z * a.slots * a.n) : a.out;
    const int type = a.part ? (int)SRC_F32 : a.out_type;
    const int64_t stride = a.part ? a.n : a.out_stride;
    const bool vec = n0 + TM <= a.n && stride % 4 == 0 && ((uintptr_t)out & 15) == 0;
    for (int t = warp; t < cnt; t += TILE_THREADS / 32) {
        const int64_t at = (int64_t)s_slot[t] * stride + n0;
        const float* r = o + t * C::OUT_PITCH;
        if (vec) {
            const float4 v = *reinterpret_cast<const float4*>(r + 4 * lane);
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
            for (int c = lane; c < TM && n0 + c < a.n; c += 32) store_val(out, at + c, type, r[c]);
        }
    }
}

// Q8_0 rows -> 16-byte aligned levels and float planes; units beyond the row are zero. One thread
// per half unit.
__global__ void __launch_bounds__(256) pack_kernel(const uint8_t* x, int64_t x_row, int rows, int units, int units_pad,
                                                   int8_t* xq, float* xd, int64_t plane, int planes) {
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

// One thread per VEC columns of an output row: slots in order, splits in order.
template <int VEC>
__global__ void __launch_bounds__(256) finish_kernel(MmArgs a, int per_out, const float* weights, const int* ids, int n_vec) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, outs = a.slots / per_out;
    if (i >= outs * n_vec) return;
    const int64_t r = i / n_vec;
    const int c = (int)(i - r * n_vec) * VEC;
    float sum[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) sum[v] = 0.0f;
    for (int j = 0; j < per_out; j++) {
        const int64_t slot = r * per_out + j;
        if (ids && (unsigned)__ldg(ids + slot) >= (unsigned)a.n_exp) continue;
        float p[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) p[v] = 0.0f;
        for (int s = 0; s < a.splits; s++) {
            const float* q = a.part + ((int64_t)s * a.slots + slot) * a.n + c;
            if constexpr (VEC == 4) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(q));
                p[0] += f.x; p[1] += f.y; p[2] += f.z; p[3] += f.w;
            } else {
                p[0] += __ldg(q);
            }
        }
        const float wt = weights ? __ldg(weights + slot) : 1.0f;
#pragma unroll
        for (int v = 0; v < VEC; v++) sum[v] = weights ? __fmaf_rn(wt, p[v], sum[v]) : sum[v] + p[v];
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
    const dim3 grid((unsigned)((a.n + TM - 1) / TM), (unsigned)chunks, (unsigned)a.splits);
    tile_kernel<T, BN><<<grid, TILE_THREADS, C::BYTES, ctx.stream>>>(a);
    return cudaGetLastError();
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

cudaError_t launch_mm_pack(const MmArgs& a, int rows, int8_t* xq, float* xd, int planes, const LaunchCtx& ctx) {
    const int64_t threads = (int64_t)rows * a.units_pad * 2;
    pack_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, ctx.stream>>>(a.x, a.x_row, rows, a.units, a.units_pad, xq, xd, a.x_plane, planes);
    return cudaGetLastError();
}

cudaError_t launch_mm_finish(const MmArgs& a, int per_out, const float* weights, const int* ids, const LaunchCtx& ctx) {
    const bool v4 = a.n % 4 == 0;
    const int n_vec = v4 ? a.n / 4 : a.n;
    const int64_t threads = (int64_t)(a.slots / per_out) * n_vec;
    const unsigned blocks = (unsigned)((threads + 255) / 256);
    if (v4) finish_kernel<4><<<blocks, 256, 0, ctx.stream>>>(a, per_out, weights, ids, n_vec);
    else finish_kernel<1><<<blocks, 256, 0, ctx.stream>>>(a, per_out, weights, ids, n_vec);
    return cudaGetLastError();
}

}  // namespace qs
