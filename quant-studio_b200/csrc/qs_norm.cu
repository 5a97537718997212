// RMS norm of rows, with the residual's addition, into Q8_0 blocks (sm_100a).
//
//   t = x + residual (float32 sum rounded to the rows' type; t = x without a residual)
//   r = 1 / sqrt(mean(t^2) + eps),  p = t * weight
//   per 32 values: m = max |p|, levels sign(p) floor(127 |p| / m + 1/2), scale f16(m r / 127)
//
// The levels do not depend on r, and |p| / m is compared with the borders between two levels as in 64
// bits: in float32 first, where a level's error is below 4.6e-5 of a step (two units of __fdividef's last
// place and the roundings of p and m, 3.6e-7 of up to 127.5) and a scale's below 2.4e-7; blocks with a value within
// 5e-5 of a border, or a scale within 3e-7 of a float16 border, are done again in double by their warp (about
// one warp pass of 8 blocks in 20). The sum of squares is in double throughout. A row holding inf or NaN gets
// NaN scales and zero levels.
//
// Neither bound is met: device memory (read x and the residual, write their sum and 34 bytes per 32 values)
// runs at half its rate, the some 33 instructions per value take 59 % of the issue slots, since a CTA loads, sums and
// stores in turn and registers admit 32 warps per SM (the part before the row's sum alone runs at the memory's
// pace). One row per CTA, two chunks of 8 values per thread in registers between the passes; of rows beyond 8192
// values an SM holds one CTA. Measured: 4096 rows of 4096 bfloat16 with a residual 35.3 us, 3.4 TB/s (four chunks
// per thread, fewer warps: 45 us; every border in double by the full formula: 38 us); 333 float32 rows of 14336
// 13.8 us, in three waves; one row of 4096 3 us.
#include "qs_kernels.h"

namespace qs {

namespace {

struct NormArgs {
    const void* x;
    const void* res;   // or null
    void* total;       // null without a residual; may be x or res
    const float* w;
    uint8_t* dst;
    int64_t x_stride, res_stride, total_stride;  // elements
    int64_t dst_stride;                          // bytes
    int k;
    double eps, inv_k;
};

// float32 remainders of levels below SURE, and scales that NEAR does not take across a float16 border, are
// as in exact arithmetic
constexpr float SURE = 0.49995f, NEAR = 4e-7f;

// 1 / sqrt(x) to about one step: two Newton steps from the float32 approximation (2^-22, squared twice)
__device__ __forceinline__ double rsqrt64(double x) {
    if (!(x > 1e-30 && x < 1e30)) return 1.0 / sqrt(x);
    double y = (double)rsqrtf((float)x);
#pragma unroll
    for (int i = 0; i < 2; i++) y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
    return y;
}

// 127 x - h m, of the right sign for products x and m of two float32 values and h of 8 bits: next to the border
// both differences are exact
__device__ __forceinline__ double over_border(double x, double m, double h) {
    const double y = 127.0 * x;
    return fma(-h, m, y) + fma(127.0, x, -y);
}

// Levels (x, y) and scale (z) of 8 values of a block, whose 4 lanes call it together, for products of any size. Rarely
// needed, and kept out of the kernel's registers (inlined: 36.6 us for 4096 rows of 4096).
__device__ __noinline__ uint3 in_double(const float* t, const float* w, double r127) {
    double m = 0.0;
#pragma unroll 1
    for (int i = 0; i < 8; i++) m = fmax(m, fabs((double)t[i] * (double)w[i]));
    m = fmax(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmax(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (!(m <= 1.7e308)) return make_uint3(0, 0, 0x7E00);
    unsigned long long q = 0;
#pragma unroll 1
    for (int i = 0; i < 8 && m > 0.0; i++) {
        const double x = (double)t[i] * (double)w[i], h = floor(127.0 * (fabs(x) / m)) + 0.5;
        const int l = (int)(over_border(fabs(x), m, h) >= 0.0 ? h + 0.5 : h - 0.5);
        q |= (unsigned long long)((uint32_t)(x < 0.0 ? -l : l) & 0xFFu) << (8 * i);
    }
    return make_uint3((uint32_t)q, (uint32_t)(q >> 32), f16_bits((float)(m * r127)));
}

__device__ __forceinline__ double block_sum(double v, double* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();  // red may still be read from an earlier sum
    if (lane == 0) red[warp] = v;
    __syncthreads();
    double s = lane < nw ? red[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// 8 values of chunk c of the row: t; with a residual it is also written to `total`
template <int SRC, bool RES>
__device__ __forceinline__ void load_chunk(const NormArgs& a, int64_t row, int c, float* v) {
    load_row<8>(a.x, row * a.x_stride + 8 * (int64_t)c, SRC, v);
    if constexpr (RES) {
        float r[8];
        load_row<8>(a.res, row * a.res_stride + 8 * (int64_t)c, SRC, r);
        const int64_t o = row * a.total_stride + 8 * (int64_t)c;
        if constexpr (SRC == SRC_F32) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __fadd_rn(v[i], r[i]);
            {
                float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.total) + o);
                p[0] = make_float4(v[0], v[1], v[2], v[3]);
                p[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t h[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float s = __fadd_rn(v[2 * i + j], r[2 * i + j]);
                    if constexpr (SRC == SRC_BF16) {
                        h[j] = __bfloat16_as_ushort(__float2bfloat16_rn(s));
                        v[2 * i + j] = __uint_as_float(h[j] << 16);
                    } else {
                        h[j] = f16_bits(s);
                        v[2 * i + j] = f16_val((uint16_t)h[j]);
                    }
                }
                b[i] = h[0] | (h[1] << 16);
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.total) + o) = make_uint4(b[0], b[1], b[2], b[3]);
        }
    }
}

// The same values a second time. `total` may be x or the residual, so with a residual this is
// what the thread itself stored (a coherent load).
template <int SRC, bool RES>
__device__ __forceinline__ void reload_chunk(const NormArgs& a, int64_t row, int c, float* v) {
    if constexpr (!RES) {
        load_row<8>(a.x, row * a.x_stride + 8 * (int64_t)c, SRC, v);
    } else {
        const int64_t o = row * a.total_stride + 8 * (int64_t)c;
        if constexpr (SRC == SRC_F32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.total) + o);
            const float4 b0 = __ldcg(p), b1 = __ldcg(p + 1);
            v[0] = b0.x; v[1] = b0.y; v[2] = b0.z; v[3] = b0.w;
            v[4] = b1.x; v[5] = b1.y; v[6] = b1.z; v[7] = b1.w;
        } else {
            const uint4 b = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.total) + o));
            const uint32_t w4[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t h = (w4[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
                v[j] = SRC == SRC_BF16 ? __uint_as_float(h << 16) : f16_val((uint16_t)h);
            }
        }
    }
}

// One row per CTA; a thread owns chunks of 8 values, 4 adjacent lanes one block. CH: chunks a
// thread keeps in registers between the two passes over the row; CH = 0: rows longer than the
// registers hold, read twice (the second time from L2).
template <int SRC, bool RES, int CH>
__global__ void __launch_bounds__(1024) norm_kernel(NormArgs a) {
    __shared__ double red[32];
    __shared__ __align__(16) uint8_t stage[32][272];  // 8 blocks per warp
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nchunk = a.k >> 3;
    const int64_t row = blockIdx.x;
    constexpr int NC = CH == 0 ? 1 : CH;
    float v[NC][8];
    double s0 = 0.0, s1 = 0.0;
    auto add_squares = [&](const float* t) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const double x = (double)t[i], y = (double)t[i + 1];
            s0 = fma(x, x, s0);
            s1 = fma(y, y, s1);
        }
    };
    if constexpr (CH == 0) {
        for (int c = tid; c < nchunk; c += blockDim.x) {
            load_chunk<SRC, RES>(a, row, c, v[0]);
            add_squares(v[0]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = tid + j * blockDim.x;
            if (c < nchunk) load_chunk<SRC, RES>(a, row, c, v[j]);
        }
#pragma unroll
        for (int j = 0; j < NC; j++)
            if (tid + j * (int)blockDim.x < nchunk) add_squares(v[j]);
    }
    // the first weights are on their way during the sum
    float w[8];
    if (tid < nchunk) load_f32<8>(a.w + 8 * (int64_t)tid, w);
    const double sum = block_sum(s0 + s1, red);
    const bool bad = !(sum <= 1.7e308);
    const double r127 = rsqrt64(fma(sum, a.inv_k, a.eps)) * (1.0 / 127.0);
    const float r127f = (float)r127;
    uint8_t* out = a.dst + row * a.dst_stride;
    const int rounds = (nchunk + blockDim.x - 1) / blockDim.x;
#pragma unroll
    for (int j = 0; j < (CH == 0 ? rounds : NC); j++) {
        const int c0 = j * (int)blockDim.x + warp * 32, c = c0 + lane;
        if (CH != 0 && j >= rounds) break;
        if (c0 >= nchunk) break;  // whole warps leave together
        float* t = v[CH == 0 ? 0 : j];
        const bool live = c < nchunk;  // nchunk is a multiple of 4: the 4 lanes of a block agree
        if (live) {
            if constexpr (CH == 0) reload_chunk<SRC, RES>(a, row, c, t);
            if (j > 0) load_f32<8>(a.w + 8 * (int64_t)c, w);
        }
        float mh = 0.0f, p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[i] = live ? __fmul_rn(t[i], w[i]) : 0.0f;
            mh = fmaxf(mh, fabsf(p[i]));
        }
        mh = fmaxf(mh, __shfl_xor_sync(0xffffffffu, mh, 1));
        mh = fmaxf(mh, __shfl_xor_sync(0xffffffffu, mh, 2));
        // 127 p / m plus 1.5 * 2^23: the level is the low byte
        const float inv = __fdividef(127.0f, mh);
        float off = 0.0f;
        uint32_t z[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = __fmaf_rn(p[i], inv, 12582912.0f);
            off = fmaxf(off, fabsf(__fmaf_rn(p[i], inv, -__fadd_rn(y, -12582912.0f))));
            z[i] = __float_as_uint(y);
        }
        uint32_t q[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
            q[i] = __byte_perm(__byte_perm(z[4 * i], z[4 * i + 1], 0x0040u), __byte_perm(z[4 * i + 2], z[4 * i + 3], 0x0040u), 0x5410u);
        const float ds = __fmul_rn(mh, r127f);
        uint16_t d = f16_bits(ds);
        const bool normal = mh > 1e-25f && mh < 1e37f;  // products and their remainders are normal numbers
        // (r / 127 below the normal range, in rows of values beyond 6e35, has few bits)
        const bool sure = off < SURE && r127f >= 1.1754944e-38f && f16_bits(__fmul_rn(ds, 1.0f - NEAR)) == f16_bits(__fmul_rn(ds, 1.0f + NEAR));
        if (!__all_sync(0xffffffffu, (normal && sure) || !live || bad)) {
            if (__all_sync(0xffffffffu, normal || !live || bad)) {
                // the block's exact largest product: the largest remainder among the largest products
                float me = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (live && fabsf(p[i]) == mh) me = fmaxf(me, __fmaf_rn(fabsf(t[i]), fabsf(w[i]), -fabsf(p[i])));
                me = fmaxf(me, __shfl_xor_sync(0xffffffffu, me, 1));
                me = fmaxf(me, __shfl_xor_sync(0xffffffffu, me, 2));
                const double m = (double)mh + (double)me;
                d = f16_bits((float)(m * r127));
                // a value next to a border: on which side 127 x lies of m times the border (a half; on it,
                // away from zero)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float n = __fadd_rn(__uint_as_float(z[i]), -12582912.0f), f = __fmaf_rn(p[i], inv, -n);
                    if (live && fabsf(f) >= SURE) {
                        const double h = (double)n + (f > 0.0f ? 0.5 : -0.5), over = over_border((double)t[i] * (double)w[i], m, h);
                        const int level = (int)(over > 0.0 || (over == 0.0 && h > 0.0) ? h + 0.5 : h - 0.5);
                        const int sh = 8 * (i & 3);
                        q[i >> 2] = (q[i >> 2] & ~(0xFFu << sh)) | (((uint32_t)level & 0xFFu) << sh);
                    }
                }
            } else {
                float copy[16];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    copy[i] = live ? t[i] : 0.0f;
                    copy[8 + i] = live ? w[i] : 0.0f;
                }
                const uint3 r = in_double(copy, copy + 8, r127);
                q[0] = r.x;
                q[1] = r.y;
                d = (uint16_t)r.z;
            }
        }
        if (bad) {
            q[0] = q[1] = 0;
            d = 0x7E00;
        }
        // 34-byte blocks: staged per warp, then whole 16-byte pieces where they line up
        uint8_t* sb = stage[warp] + (lane >> 2) * 34;
        const int o = 2 + 8 * (lane & 3);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; i++) {
            *reinterpret_cast<uint16_t*>(sb + o + 4 * i) = (uint16_t)q[i];
            *reinterpret_cast<uint16_t*>(sb + o + 4 * i + 2) = (uint16_t)(q[i] >> 16);
        }
        if ((lane & 3) == 0) *reinterpret_cast<uint16_t*>(sb) = d;
        __syncwarp();
        uint8_t* g = out + (int64_t)(c0 >> 2) * 34;
        const int nb = min(8, (nchunk - c0) >> 2) * 34;
        if (nb == 272 && ((uintptr_t)g & 15) == 0) {
            if (lane < 17) reinterpret_cast<uint4*>(g)[lane] = reinterpret_cast<const uint4*>(stage[warp])[lane];
        } else if (((uintptr_t)g & 1) == 0) {
            for (int i = lane; i < nb / 2; i += 32) reinterpret_cast<uint16_t*>(g)[i] = reinterpret_cast<const uint16_t*>(stage[warp])[i];
        } else {
            for (int i = lane; i < nb; i += 32) g[i] = stage[warp][i];
        }
    }
}

template <int SRC, bool RES>
cudaError_t launch_t(const NormArgs& a, int64_t rows, const LaunchCtx& ctx) {
    const int nchunk = a.k / 8;
    const int whole = (nchunk + 31) / 32 * 32;
    // Few rows: as many threads per row as it has chunks (latency). Many: 2 chunks a thread.
    const bool few = rows < 4 * (int64_t)ctx.num_sms;
    if (few && whole <= 1024) norm_kernel<SRC, RES, 1><<<(unsigned)rows, whole, 0, ctx.stream>>>(a);
    else if (nchunk <= 2 * 1024) norm_kernel<SRC, RES, 2><<<(unsigned)rows, ((nchunk + 1) / 2 + 31) / 32 * 32, 0, ctx.stream>>>(a);
    else norm_kernel<SRC, RES, 0><<<(unsigned)rows, 1024, 0, ctx.stream>>>(a);
    return cudaGetLastError();
}

template <int SRC>
cudaError_t launch_s(const NormArgs& a, int64_t rows, const LaunchCtx& ctx) {
    return a.res ? launch_t<SRC, true>(a, rows, ctx) : launch_t<SRC, false>(a, rows, ctx);
}

}  // namespace

cudaError_t launch_rms_norm_q8(const NormCall& c, const LaunchCtx& ctx) {
    NormArgs a;
    a.x = c.x;
    a.res = c.residual;
    a.total = c.total;
    a.w = c.weight;
    a.dst = static_cast<uint8_t*>(c.dst);
    a.x_stride = c.x_stride;
    a.res_stride = c.residual_stride;
    a.total_stride = c.total_stride;
    a.dst_stride = c.dst_row_bytes;
    a.k = (int)c.k;
    a.eps = c.eps;
    a.inv_k = 1.0 / (double)c.k;
    switch (c.x_type) {
    case SRC_F32: return launch_s<SRC_F32>(a, c.n_rows, ctx);
    case SRC_F16: return launch_s<SRC_F16>(a, c.n_rows, ctx);
    default: return launch_s<SRC_BF16>(a, c.n_rows, ctx);
    }
}

}  // namespace qs
