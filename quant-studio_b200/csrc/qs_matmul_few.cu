// Packed products for few slots per weight matrix (one decoded token, a small batch).
//
// The weights' bytes are the work: each is read once, a warp takes whole weight rows, lane l the
// units l, l + 32, ... of a row, and the levels meet those of up to NT slots in 4-way integer
// dot products (dp4a). The slots' Q8_0 rows are staged in shared memory once per CTA, in
// slices of 128 units.
#include "qs_matmul.cuh"

namespace qs {

namespace {

constexpr int FEW_WARPS = 8, FEW_ROWS = 2, SLICE = 128;  // warps, weight rows per warp, units per slice

template <int T, int NT>
struct FewSmem {
    static constexpr int SUMS = !Lv<T>::HASMIN ? 0 : Lv<T>::G16 ? 2 : 1;
    uint4 q[NT][2][SLICE];  // halves of 16 levels: adjacent lanes read adjacent 16 bytes
    float d[NT][SLICE];
    float s[SUMS ? SUMS : 1][NT][SUMS ? SLICE : 1];  // scale * sum of levels (of a half)
};

template <int T, int NT>
__global__ void __launch_bounds__(32 * FEW_WARPS) few_kernel(MmArgs a) {
    using L = Lv<T>;
    constexpr int UPB = L::QK / 32, SUMS = FewSmem<T, NT>::SUMS;
    __shared__ FewSmem<T, NT> sm;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Chunk ch = find_chunk<NT>(a, blockIdx.y);
    if (ch.group < 0) return;
    const int n0 = (blockIdx.x * FEW_WARPS + warp) * FEW_ROWS, cnt = ch.hi - ch.lo;
    float acc[FEW_ROWS][NT];
#pragma unroll
    for (int r = 0; r < FEW_ROWS; r++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[r][t] = 0.0f;
    if (!a.order || ch.group < a.n_exp) {
        const uint8_t* w = a.w + ch.group * a.w_exp;
        for (int u0 = 0; u0 < a.units; u0 += SLICE) {
            const int nu = min(SLICE, a.units - u0);
            if (u0) __syncthreads();
            for (int i = tid; i < NT * 2 * SLICE; i += 32 * FEW_WARPS) {
                const int t = i / (2 * SLICE), u = (i / 2) % SLICE, h = i & 1;
                uint4 q = make_uint4(0, 0, 0, 0);
                float d = 0.0f;
                if (t < cnt && u < nu) {
                    const int slot = a.order ? __ldg(a.order + ch.lo + t) : ch.lo + t;
                    const uint8_t* b = a.x + (slot / a.x_div) * a.x_row + (int64_t)(u0 + u) * 34;
                    q = ld_16b(b + 2 + 16 * h);
                    d = h2f(ld_u16<1>(b));
                }
                sm.q[t][h][u] = q;
                if (h == 0) sm.d[t][u] = d;
                if constexpr (SUMS == 2) sm.s[h][t][u] = d * (float)sum16(q);
                if constexpr (SUMS == 1) {
                    const int s = sum16(q), o = __shfl_xor_sync(0xffffffffu, s, 1);
                    if (h == 0) sm.s[0][t][u] = d * (float)(s + o);
                }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < FEW_ROWS; r++) {
                if (n0 + r >= a.n) break;
                const uint8_t* wr = w + (n0 + r) * a.w_row;
#pragma unroll
                for (int i = 0; i < SLICE / 32; i++) {
                    const int u = lane + 32 * i;
                    if (u >= nu) break;
                    uint32_t q[8];
                    float dl[2], ml[2];
                    L::template unit<L::MAXAL>(wr + (int64_t)((u0 + u) / UPB) * L::BB, (u0 + u) % UPB, a.kgrid, q, dl, ml);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const uint4 xa = sm.q[t][0][u], xb = sm.q[t][1][u];
                        const float d = sm.d[t][u];
                        int s0 = __dp4a((int)q[0], (int)xa.x, 0), s1 = 0;
                        s0 = __dp4a((int)q[1], (int)xa.y, s0);
                        s0 = __dp4a((int)q[2], (int)xa.z, s0);
                        s0 = __dp4a((int)q[3], (int)xa.w, s0);
                        if (!L::G16) s1 = s0;
                        s1 = __dp4a((int)q[4], (int)xb.x, s1);
                        s1 = __dp4a((int)q[5], (int)xb.y, s1);
                        s1 = __dp4a((int)q[6], (int)xb.z, s1);
                        s1 = __dp4a((int)q[7], (int)xb.w, s1);
                        if (L::G16) acc[r][t] = __fmaf_rn(dl[0] * d, (float)s0, acc[r][t]);
                        acc[r][t] = __fmaf_rn(dl[1] * d, (float)s1, acc[r][t]);
                        if constexpr (SUMS >= 1) acc[r][t] = __fmaf_rn(-ml[0], sm.s[0][t][u], acc[r][t]);
                        if constexpr (SUMS == 2) acc[r][t] = __fmaf_rn(-ml[1], sm.s[1][t][u], acc[r][t]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < FEW_ROWS; r++) {
        if (n0 + r >= a.n) break;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float v = acc[r][t];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == 0 && t < cnt) {
                const int64_t slot = a.order ? __ldg(a.order + ch.lo + t) : ch.lo + t;
                if (a.part) a.part[slot * a.n + n0 + r] = v;
                else store_val(a.out, slot * a.out_stride + n0 + r, a.out_type, v);
            }
        }
    }
}

template <int T, int NT>
cudaError_t launch_few_t(const MmArgs& a, const LaunchCtx& ctx) {
    const int64_t chunks = max_chunks(a, NT);
    if (chunks > 65535) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)((a.n + FEW_WARPS * FEW_ROWS - 1) / (FEW_WARPS * FEW_ROWS)), (unsigned)chunks);
    few_kernel<T, NT><<<grid, 32 * FEW_WARPS, 0, ctx.stream>>>(a);
    return cudaGetLastError();
}

template <int T>
cudaError_t launch_few(const MmArgs& a, const LaunchCtx& ctx) {
    // one slot per expert is the rule when a few tokens share many experts
    if (a.slots == 1 || (a.order && a.slots <= a.n_exp)) return launch_few_t<T, 1>(a, ctx);
    if (!a.order && a.slots <= 4) return launch_few_t<T, 4>(a, ctx);
    return launch_few_t<T, 8>(a, ctx);
}

}  // namespace

cudaError_t launch_mm_few(int type, const MmArgs& a, const LaunchCtx& ctx) {
    switch (type) {
#define X(T) case T: return launch_few<T>(a, ctx);
        QS_FOR_TYPES(X)
#undef X
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qs
