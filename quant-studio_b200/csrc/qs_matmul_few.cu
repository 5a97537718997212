// Packed products for few slots per weight matrix (one decoded token, a small batch).
//
// The weights' bytes are the work: each is read once, and the levels meet those of up to NT slots in
// 4-way integer dot products (dp4a). A lane takes two units at a time, a pair that shares its bytes
// where the format has such pairs (both nibbles of the same 32 bytes). LPR lanes share a weight row (all
// 32, fewer for short rows); lane l takes the pairs l, l + LPR, ... The slots' Q8_0 rows are staged in
// shared memory once per CTA. A warp's (rows, pair) steps form one sequence, loaded PF steps ahead, so
// that loads are in flight across row ends too. The CTAs run in one wave and take rows in turn.
//
// Measured for one slot: Q4_K 14336 x 4096 (33 MB) 13.4 us, 2.5 TB/s (15.0 us with one run of rows per warp, whose
// last warps idle); Q4_K / Q4_0 / Q8_0 4096 x 4096 6.5 / 6.7 / 6.8 us, of which about 3 us are launch, staging and first loads. Neither memory nor
// the issue slots are full: 280 instructions per pair step of a warp are 60 % of the slots, and 24 warps per SM (79
// registers) wait for their loads and for one another's results in between. With more than a few slots the dot products (half rate on this GPU) take
// over: 4 slots 12 us, and from 5 on the tensor cores' kernel is faster.
#include <algorithm>

#include "qs_matmul.cuh"

namespace qs {

namespace {

template <int T, int NT>
struct FewCfg {
    using L = Lv<T>;
    static constexpr int SUMS = !L::HASMIN ? 0 : L::G16 ? 2 : 1;
    static constexpr int PF = L::WORDS <= 6 ? 3 : 2;  // steps loaded ahead
    static constexpr int PPB = L::QK == 256 ? 4 : 1;  // pairs of a superblock
    // unit h of pair p: neighbours, but Q6_K's low nibbles belong to units j and j + 2
    __host__ __device__ static int unit(int p, int h) { return T == QS_Q6_K ? 4 * (p >> 1) + (p & 1) + 2 * h : 2 * p + h; }
    // bytes per unit of a slot: levels as two planes of 16 bytes, scale, scale * sums of levels
    static constexpr int UNIT = 32 + 4 + 4 * SUMS;
    static int bytes(int units) { return NT * (units + 1) / 2 * 2 * UNIT; }
};

template <int T, int NT>
__global__ void __launch_bounds__(512) few_kernel(MmArgs a, int lpr) {
    using L = Lv<T>;
    using C = FewCfg<T, NT>;
    constexpr int UPB = L::QK / 32, SUMS = C::SUMS, PF = C::PF, PPB = C::PPB;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, units = a.units, pairs = (units + 1) >> 1;
    uint4* const xq = reinterpret_cast<uint4*>(smem);                                // [slot][unit of pair][half][pair]
    float* const xd = reinterpret_cast<float*>(smem + NT * pairs * 64);              // [slot][unit of pair][pair]
    float* const xs = xd + NT * pairs * 2;                                           // [half][slot][unit of pair][pair]
    const Chunk ch = find_chunk<NT>(a, blockIdx.y);
    if (ch.group < 0) return;
    const int cnt = ch.hi - ch.lo;
    auto put = [&](int64_t r, int t, float v) {
        const int64_t slot = a.order ? __ldg(a.order + ch.lo + t) : ch.lo + t;
        if (a.part) a.part[slot * a.n + r] = v;
        else store_val(a.out, slot * a.out_stride + r, a.out_type, v);
    };
    if (a.order && ch.group == a.n_exp) {  // slots without an expert
        for (int64_t r = (int64_t)blockIdx.x * blockDim.x + tid; r < a.n; r += (int64_t)gridDim.x * blockDim.x)
            for (int t = 0; t < cnt; t++) put(r, t, 0.0f);
        return;
    }
    // lpr is a multiple of PPB, so lane l's pairs l + lpr i lie at the same place of their blocks
    const int l = lane & (lpr - 1), sub = lane / lpr, at_once = 32 / lpr;  // lane of the row, row of the pass
    const int iters = (pairs + lpr - 1) / lpr, hop = lpr / PPB * (UPB == 1 ? 2 : 1) * L::BB;
    const int place = l % PPB;
    // passes over at_once rows, dealt to the warps of all CTAs in turn
    const int64_t first = ((int64_t)blockIdx.x * (blockDim.x >> 5) + warp) * at_once, turn = (int64_t)gridDim.x * (blockDim.x >> 5) * at_once;
    const uint8_t* row_at = a.w + ch.group * a.w_exp + (first + sub) * a.w_row + (UPB == 1 ? 2 * l : l / PPB) * L::BB;
    const uint8_t* at = row_at;
    uint32_t raw[PF][2][L::WORDS];
    int64_t lr = first + sub;  // row and pair of the next load
    int lp = l;
    auto load = [&](uint32_t (*r)[L::WORDS]) {
        if (lr < a.n && lp < pairs) {
            if constexpr (UPB == 1) {
                L::template load<L::MAXAL>(at, 0, r[0]);
                if (2 * lp + 1 < units) {
                    L::template load<L::MAXAL>(at + L::BB, 0, r[1]);
                } else {
#pragma unroll
                    for (int e = 0; e < L::WORDS; e++) r[1][e] = 0;  // zero scale
                }
            } else {
                L::template load<L::MAXAL>(at, C::unit(place, 0), r[0]);
                L::template load<L::MAXAL>(at, C::unit(place, 1), r[1]);
            }
        }
        at += hop;
        lp += lpr;
        if (lp - l >= iters * lpr) {
            lp = l;
            lr += turn;
            at = row_at += a.w_row * turn;
        }
    };
#pragma unroll
    for (int p = 0; p < PF; p++) load(raw[p]);

    for (int i = tid; i < NT * 2 * pairs * 2; i += blockDim.x) {
        const int h = i & 1, k = i >> 1, t = k / (2 * pairs), u = k - t * 2 * pairs;
        const int p = T == QS_Q6_K ? 2 * (u >> 2) + (u & 1) : u >> 1, e = T == QS_Q6_K ? (u >> 1) & 1 : u & 1;
        uint4 q = make_uint4(0, 0, 0, 0);
        float d = 0.0f;
        int s = 0, other = 0;
        if (t < cnt && u < units) {
            const int slot = a.order ? __ldg(a.order + ch.lo + t) : ch.lo + t;
            const uint8_t* b = a.x + (slot / a.x_div) * a.x_row + (int64_t)u * 34;
            q = ld_16b(b + 2 + 16 * h);
            d = h2f(ld_u16<1>(b));
            if constexpr (SUMS > 0) s = sum16(q);
            // the other half's sum, computed again rather than exchanged: lanes may have left the loop
            if constexpr (SUMS == 1) other = sum16(ld_16b(b + 2 + 16 * (h ^ 1)));
        }
        xq[((t * 2 + e) * 2 + h) * pairs + p] = q;
        if (h == 0) xd[(t * 2 + e) * pairs + p] = d;
        if constexpr (SUMS == 2) xs[((h * NT + t) * 2 + e) * pairs + p] = d * (float)s;
        if constexpr (SUMS == 1)
            if (h == 0) xs[(t * 2 + e) * pairs + p] = d * (float)(s + other);
    }
    __syncthreads();

    float acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = 0.0f;
    int64_t cr = first + sub;  // row and pair at hand
    int cp = l;
    const int64_t passes = first < a.n ? (a.n - first + turn - 1) / turn : 0, steps = passes * iters;
    for (int64_t s = 0; s < steps; s += PF) {
#pragma unroll
        for (int p = 0; p < PF; p++) {
            if (s + p >= steps) break;
            const bool live = cp < pairs && cr < a.n;
            if (live) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    uint32_t q[8];
                    float dl[2], ml[2];
                    L::levels(raw[p][e], UPB == 1 ? 0 : C::unit(place, e), a.kgrid, q, dl, ml);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const uint4 xa = xq[((t * 2 + e) * 2) * pairs + cp], xb = xq[((t * 2 + e) * 2 + 1) * pairs + cp];
                        const float d = xd[(t * 2 + e) * pairs + cp];
                        int s0 = __dp4a((int)q[0], (int)xa.x, 0), s1 = 0;
                        s0 = __dp4a((int)q[1], (int)xa.y, s0);
                        s0 = __dp4a((int)q[2], (int)xa.z, s0);
                        s0 = __dp4a((int)q[3], (int)xa.w, s0);
                        if (!L::G16) s1 = s0;
                        s1 = __dp4a((int)q[4], (int)xb.x, s1);
                        s1 = __dp4a((int)q[5], (int)xb.y, s1);
                        s1 = __dp4a((int)q[6], (int)xb.z, s1);
                        s1 = __dp4a((int)q[7], (int)xb.w, s1);
                        if (L::G16) acc[t] = __fmaf_rn(dl[0] * d, (float)s0, acc[t]);
                        acc[t] = __fmaf_rn(dl[1] * d, (float)s1, acc[t]);
                        if constexpr (SUMS >= 1) acc[t] = __fmaf_rn(-ml[0], xs[(t * 2 + e) * pairs + cp], acc[t]);
                        if constexpr (SUMS == 2) acc[t] = __fmaf_rn(-ml[1], xs[((NT + t) * 2 + e) * pairs + cp], acc[t]);
                    }
                }
            }
            load(raw[p]);
            cp += lpr;
            if (cp - l >= iters * lpr) {  // the rows' end
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float v = acc[t];
                    for (int o = lpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    if (l == 0 && t < cnt && cr < a.n) put(cr, t, v);
                    acc[t] = 0.0f;
                }
                cp = l;
                cr += turn;
            }
        }
    }
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

template <int T, int NT>
cudaError_t launch_few_t(const MmArgs& a, const LaunchCtx& ctx) {
    const int64_t chunks = max_chunks(a, NT);
    const int bytes = FewCfg<T, NT>::bytes(a.units);
    if (chunks > 65535 || bytes > FEW_SMEM_MAX) return cudaErrorInvalidConfiguration;
    static std::atomic<unsigned long long> asked{0};
    if (bytes > 48 * 1024) {
        const cudaError_t e = allow_smem((const void*)few_kernel<T, NT>, FEW_SMEM_MAX, ctx.device, asked);
        if (e != cudaSuccess) return e;
    }
    const int pairs = (a.units + 1) / 2;
    int lpr = 32;  // lanes of a row: no more than it has pairs (at least a superblock's 4)
    while (lpr > 4 && lpr / 2 >= pairs) lpr /= 2;
    // Activations beyond a quarter of an SM's shared memory: fewer CTAs fit, with 16 warps each.
    const int warps = bytes <= 48 * 1024 ? 8 : 16;
    static const int regs = [] {
        cudaFuncAttributes f;
        return cudaFuncGetAttributes(&f, few_kernel<T, NT>) == cudaSuccess ? (f.numRegs + 7) / 8 * 8 : 128;
    }();
    const int per_sm = std::max(1, std::min({65536 / (regs * 32 * warps), 64 / warps, 227 * 1024 / (bytes + 1024)}));
    // CTAs per chunk: what fits the SMs at once in one wave or in a few, by the steps of a warp over all waves
    // and 4 for a wave's start and end. Q4_K, one wave / two: 8 chunks of 8192 x 4096 46 / 63 us; 64 of them
    // (256 CTAs of 296 / 576 of 592) 359 / 309 us.
    const int64_t at_once = (int64_t)per_sm * ctx.num_sms, most = ((a.n + 32 / lpr - 1) / (32 / lpr) + warps - 1) / warps;
    const int64_t iters = (pairs + lpr - 1) / lpr;
    int64_t ctas = 1, best = INT64_MAX;
    for (int w = 1; w <= 8; w++) {
        const int64_t c = std::min(most, std::max<int64_t>(1, at_once * w / chunks));
        const int64_t waves = (chunks * c + at_once - 1) / at_once, steps = waves * ((most + c - 1) / c * iters + 4);
        if (steps < best) best = steps, ctas = c;
    }
    const dim3 grid((unsigned)ctas, (unsigned)chunks);
    few_kernel<T, NT><<<grid, 32 * warps, bytes, ctx.stream>>>(a, lpr);
    return cudaGetLastError();
}

template <int T>
cudaError_t launch_few(const MmArgs& a, const LaunchCtx& ctx) {
    // one slot per expert is the rule when a few tokens share many experts
    return a.slots == 1 || a.order ? launch_few_t<T, 1>(a, ctx) : launch_few_t<T, 4>(a, ctx);
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
