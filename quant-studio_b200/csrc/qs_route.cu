// Routing of tokens to experts, and the plan that groups the chosen slots by expert (sm_100a).
#include "qs_kernels.h"

namespace qs {

namespace {

struct RouteArgs {
    const void* logits;
    int64_t stride;  // elements
    const float* bias;
    int* ids;
    float* weights;
    int64_t rows;
    int n_exp, top_k, n_groups, kept;
    int sigmoid, top2, renorm;
    float scale;
    int src;
};

__device__ __forceinline__ float logit_at(const RouteArgs& a, int64_t i) {
    if (a.src == SRC_F32) return __ldg(static_cast<const float*>(a.logits) + i);
    const uint16_t b = __ldg(static_cast<const uint16_t*>(a.logits) + i);
    return a.src == SRC_BF16 ? __uint_as_float((uint32_t)b << 16) : f16_val(b);
}

// Selection values as unsigned words of the same order: larger value, larger word; 0 for what can not
// be chosen (-inf and NaN). -0 counts as +0.
struct Key32 {
    typedef uint32_t K;
    __device__ static K of(float v) {
        if (!(v > -INFINITY)) return 0u;
        const uint32_t b = __float_as_uint(v + 0.0f);
        return (b >> 31) ? ~b : b | 0x80000000u;
    }
    __device__ static float value(K k) { return k == 0u ? -INFINITY : __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k); }
    __device__ static K warp_max(K v) { return __reduce_max_sync(0xffffffffu, v); }
};
struct Key64 {
    typedef unsigned long long K;
    __device__ static K of(double v) {
        if (!(v > -INFINITY)) return 0ull;
        const K b = (K)__double_as_longlong(v + 0.0);
        return (b >> 63) ? ~b : b | 0x8000000000000000ull;
    }
    __device__ static double value(K k) { return k == 0ull ? -INFINITY : __longlong_as_double((long long)((k >> 63) ? k & 0x7FFFFFFFFFFFFFFFull : ~k)); }
    __device__ static K warp_max(K v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const K u = __shfl_xor_sync(0xffffffffu, v, o);
            v = u > v ? u : v;
        }
        return v;
    }
};

constexpr int ROUTE_WARPS = 4;

// The top_k experts by key, lane r keeps the r-th (-1: none is left); lane l holds the keys of experts
// l, l + 32, ... gap: the smallest difference between two values whose order decided something
// (sums of two count half).
template <class W, int EPL>
__device__ __forceinline__ int choose(const RouteArgs& a, typename W::K* key, int lane, float& gap) {
    typedef typename W::K K;
    gap = INFINITY;
    if (a.n_groups > 1) {
        // group scores; lane g (and g + 32) keeps those of its group
        const int gs = a.n_exp / a.n_groups;
        K gk[2] = {0, 0};
        auto score = [&](K best, K second, int g) {
            const K m1 = W::warp_max(best);
            K v = m1;
            if (a.top2) {  // one holder of the largest gives its second
                const unsigned who = __ballot_sync(0xffffffffu, best == m1);
                const K m2 = W::warp_max(lane == __ffs(who) - 1 ? second : best);
                v = W::of(W::value(m1) + W::value(m2));
            }
            if ((g & 31) == lane) gk[g >> 5] = v;
        };
        if (gs % 32 == 0) {  // whole registers belong to one group: a single pass
            K best = 0, second = 0;
            int g = 0, left = gs;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                const K k = key[i];
                second = k > best ? best : (k > second ? k : second);
                best = k > best ? k : best;
                left -= 32;
                if (left == 0) {
                    if (g < a.n_groups) score(best, second, g);
                    g++;
                    left = gs;
                    best = second = 0;
                }
            }
        } else {
            for (int g = 0; g < a.n_groups; g++) {
                K best = 0, second = 0;
                const int lo = g * gs - lane, hi = lo + gs;  // of 32 i
#pragma unroll
                for (int i = 0; i < EPL; i++)
                    if (32 * i >= lo && 32 * i < hi) {
                        const K k = key[i];
                        second = k > best ? best : (k > second ? k : second);
                        best = k > best ? k : best;
                    }
                score(best, second, g);
            }
        }
        // keep the best groups, ties to the lowest; a group without a usable score comes last
        unsigned long long keep = 0ull;  // bit g
        float before = INFINITY;
        for (int r = 0; r <= a.kept && r < a.n_groups; r++) {
            K b = 0;
            int bg = 0x7FFFFFFF;
#pragma unroll
            for (int h = 1; h >= 0; h--) {
                const int g = lane + 32 * h;
                if (g < a.n_groups && !((keep >> g) & 1ull) && gk[h] >= b) { b = gk[h]; bg = g; }
            }
            const K m = W::warp_max(b);
            if (r == a.kept) {  // the best of the rest
                if (m) gap = (before - (float)W::value(m)) * (a.top2 ? 0.5f : 1.0f);
                break;
            }
            if (b != m) bg = 0x7FFFFFFF;
            keep |= 1ull << __reduce_min_sync(0xffffffffu, bg);
            before = (float)W::value(m);
        }
        if (gs % 32 == 0) {
            int g = 0, left = gs;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                if (g >= a.n_groups || !((keep >> g) & 1ull)) key[i] = 0;
                left -= 32;
                if (left == 0) {
                    g++;
                    left = gs;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                const int e = lane + 32 * i;
                if (e < a.n_exp && !((keep >> (e / gs)) & 1ull)) key[i] = 0;
            }
        }
    }
    // the k largest, one after the other, ties to the lowest expert
    int my_id = -1;
    float before = INFINITY;
    for (int r = 0; r <= a.top_k; r++) {
        K b = key[0];
#pragma unroll
        for (int i = 1; i < EPL; i++) b = key[i] > b ? key[i] : b;
        const K m = W::warp_max(b);
        if (m == 0) break;  // nothing usable is left
        const float v = (float)W::value(m);
        gap = fminf(gap, before - v);
        before = v;
        if (r == a.top_k) break;
        int be = EPL;  // this lane's first holder
#pragma unroll
        for (int i = EPL - 1; i >= 0; i--)
            if (key[i] == m) be = i;
        const int mine = be < EPL ? lane + 32 * be : 0x7FFFFFFF, e = __reduce_min_sync(0xffffffffu, mine);
        if (lane == r) my_id = e;
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (mine == e && be == i) key[i] = 0;
    }
    return my_id;
}

// One warp per token. Without a bias (and without sums over groups) scores are monotone in the
// logits, whose float32 values are compared as they are. Otherwise the selection values are
// computed in float32, each within `err` of its exact value; where two of them that decide come
// within 2 err of one another the row is done again in double, so that near ties fall as in
// exact arithmetic (a few rows in 1000 for 256 experts). About 1700 instructions per row of 256 experts in 8 groups,
// most of them in the k + 1 rounds of the choice, which wait for one another: 79 registers admit 24 warps per SM, and
// the issue slots are at 55 %. 8192 such rows take 27.6 us (43 us with doubles throughout; 31.0 us with groups by
// their two best), one row 2.5 us.
template <int EPL>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) route_kernel(RouteArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const bool direct = !a.bias && !(a.n_groups > 1 && a.top2);
    float z[EPL], zmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        const int e = lane + 32 * i;
        z[i] = e < a.n_exp ? logit_at(a, row * a.stride + e) : NAN;
        zmax = fmaxf(zmax, z[i]);  // NaN is passed over
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) zmax = fmaxf(zmax, __shfl_xor_sync(0xffffffffu, zmax, o));
    // exp(z - zmax); the largest (+inf too) gives 1
    auto soft = [&](float v) { return v == zmax ? 1.0 : exp((double)v - (double)zmax); };
    auto sigm = [&](float v) { return 1.0 / (1.0 + exp(-(double)v)); };
    auto bias = [&](int i) { return a.bias && lane + 32 * i < a.n_exp ? __ldg(a.bias + lane + 32 * i) : 0.0f; };
    double sum = 1.0;  // of all softmax scores, where it is needed
    int my_id;
    float gap;
    {
        uint32_t key[EPL];
        if (direct) {
#pragma unroll
            for (int i = 0; i < EPL; i++) key[i] = Key32::of(z[i]);
            my_id = choose<Key32, EPL>(a, key, lane, gap);
        } else {
            float s[EPL], total = 0.0f, top = 0.0f;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                const bool can = z[i] > -INFINITY;
                s[i] = !can ? 0.0f : a.sigmoid ? __fdividef(1.0f, 1.0f + expf(-z[i])) : z[i] == zmax ? 1.0f : expf(z[i] - zmax);
                total += s[i];
            }
            float inv = 1.0f;
            if (!a.sigmoid) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
                inv = total > 0.0f ? __frcp_rn(total) : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                const float b = bias(i);
                if (fabsf(b) < INFINITY) top = fmaxf(top, fabsf(b));
                key[i] = z[i] > -INFINITY ? Key32::of(s[i] * inv + b) : 0u;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            my_id = choose<Key32, EPL>(a, key, lane, gap);
            // scores are at most 1 and good to 24 + EPL float32 steps of it (the exponential, its rounded
            // argument, the sum and the reciprocal), the sum with the bias to one of 1 + |bias|
            const float err = (1.0f + top) * (24.0f + EPL) * 5.9604645e-8f;
            if (!(gap > 2.0f * err)) {
                unsigned long long wide[EPL];
                double d[EPL];
                double all = 0.0;
#pragma unroll
                for (int i = 0; i < EPL; i++) {
                    d[i] = !(z[i] > -INFINITY) ? 0.0 : a.sigmoid ? sigm(z[i]) : soft(z[i]);
                    all += d[i];
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
#pragma unroll
                for (int i = 0; i < EPL; i++) wide[i] = z[i] > -INFINITY ? Key64::of((a.sigmoid ? d[i] : d[i] / all) + (double)bias(i)) : 0ull;
                my_id = choose<Key64, EPL>(a, wide, lane, gap);
            }
        }
    }
    if (!a.sigmoid && !a.renorm) {
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (z[i] > -INFINITY) sum += soft(z[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float v = my_id >= 0 ? logit_at(a, row * a.stride + my_id) : -INFINITY;
    if (a.renorm && !a.sigmoid) {  // any common factor cancels: the largest chosen one is 1
        zmax = v;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) zmax = fmaxf(zmax, __shfl_xor_sync(0xffffffffu, zmax, o));
    }
    double w = my_id < 0 ? 0.0 : a.sigmoid ? sigm(v) : soft(v);
    if (a.renorm) {
        sum = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane < a.top_k) {
        a.ids[row * a.top_k + lane] = my_id;
        a.weights[row * a.top_k + lane] = my_id >= 0 && sum > 0.0 ? (float)(w / sum * (double)a.scale) : 0.0f;
    }
}

// The slots (token, j) grouped by expert, in the order of the slots: a stable counting sort
// without atomics. CTA e counts the ids below e and equal to e, and writes its own slots behind
// the former; CTA n_exp takes the slots without an expert (ids outside [0, n_exp)) to the end.
// Each thread owns one contiguous run of the slots. Every CTA reads all ids, so the work grows with slots times
// experts: 2.0 us for 8 slots of 64 experts, 3.7 us for 6000 of 32, 100 us for 65536 of 256.
constexpr int PLAN_THREADS = 512;

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const int* ids, int n, int n_exp, int* order, int* offsets) {
    __shared__ int s_less[PLAN_THREADS / 32], s_same[PLAN_THREADS / 32];
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS;
    const int lo = (int)min((int64_t)tid * per, (int64_t)n), hi = (int)min((int64_t)lo + per, (int64_t)n);
    int less = 0, same = 0;
    for (int i = lo; i < hi; i++) {
        const int v = __ldg(ids + i), c = (unsigned)v < (unsigned)n_exp ? v : n_exp;
        less += c < e;
        same += c == e;
    }
    int inc = same;  // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
        less += __shfl_xor_sync(0xffffffffu, less, o);
    }
    if (lane == 31) s_same[warp] = inc;
    if (lane == 0) s_less[warp] = less;
    __syncthreads();
    int start = 0;
    for (int w = 0; w < PLAN_THREADS / 32; w++) start += s_less[w];
    int at = start + inc - same;
    for (int w = 0; w < warp; w++) at += s_same[w];
    if (tid == 0) offsets[e] = start;
    for (int i = lo; same > 0 && i < hi; i++) {
        const int v = __ldg(ids + i), c = (unsigned)v < (unsigned)n_exp ? v : n_exp;
        if (c == e) order[at++] = i;
    }
}

template <int EPL>
cudaError_t launch_route_t(const RouteArgs& a, const LaunchCtx& ctx) {
    route_kernel<EPL><<<(unsigned)((a.rows + ROUTE_WARPS - 1) / ROUTE_WARPS), 32 * ROUTE_WARPS, 0, ctx.stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_route(const RouteCall& c, const LaunchCtx& ctx) {
    RouteArgs a;
    a.logits = c.logits;
    a.stride = c.logits_stride;
    a.bias = c.bias;
    a.ids = c.ids;
    a.weights = c.weights;
    a.rows = c.n_rows;
    a.n_exp = c.n_experts;
    a.top_k = c.top_k;
    a.n_groups = c.n_groups;
    a.kept = c.groups_kept;
    a.sigmoid = c.sigmoid;
    a.top2 = c.group_top2;
    a.renorm = c.renormalize;
    a.scale = c.scale;
    a.src = c.logits_type;
    if (c.n_experts <= 32) return launch_route_t<1>(a, ctx);
    if (c.n_experts <= 64) return launch_route_t<2>(a, ctx);
    if (c.n_experts <= 128) return launch_route_t<4>(a, ctx);
    if (c.n_experts <= 256) return launch_route_t<8>(a, ctx);
    if (c.n_experts <= 512) return launch_route_t<16>(a, ctx);
    return launch_route_t<32>(a, ctx);
}

cudaError_t launch_expert_plan(const int* ids, int n, int n_experts, int* order, int* offsets, const LaunchCtx& ctx) {
    plan_kernel<<<n_experts + 1, PLAN_THREADS, 0, ctx.stream>>>(ids, n, n_experts, order, offsets);
    return cudaGetLastError();
}

}  // namespace qs
