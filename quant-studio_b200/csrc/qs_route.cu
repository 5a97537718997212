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

// Order of the selection values as unsigned words: larger value, larger word; 0 for what can
// not be chosen (-inf and NaN). -0 counts as +0.
__device__ __forceinline__ unsigned long long order_key(double v) {
    if (!(v > -INFINITY)) return 0ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_value(unsigned long long k) {
    if (k == 0ull) return -INFINITY;
    return __longlong_as_double((long long)((k >> 63) ? k & 0x7FFFFFFFFFFFFFFFull : ~k));
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
        v = u > v ? u : v;
    }
    return v;
}

constexpr int ROUTE_WARPS = 4;

// One warp per token; lane l holds experts l, l + 32, ... (EPL of them). The selection values
// are doubles, so that near ties fall as in exact arithmetic; without a bias (and without sums
// over groups) scores are monotone in the logits, and the logits themselves are compared.
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
    double sum = 1.0;
    unsigned long long key[EPL];
    if (direct) {
#pragma unroll
        for (int i = 0; i < EPL; i++) key[i] = order_key((double)z[i]);
        if (!a.sigmoid && !a.renorm) {
            sum = 0.0;
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (key[i]) sum += soft(z[i]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
    } else {
        double s[EPL];
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            s[i] = !(z[i] > -INFINITY) ? 0.0 : a.sigmoid ? sigm(z[i]) : soft(z[i]);
            sum += s[i];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (a.sigmoid) sum = 1.0;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = lane + 32 * i;
            const bool can = z[i] > -INFINITY;
            key[i] = can ? order_key((a.sigmoid ? s[i] : s[i] / sum) + (a.bias ? (double)__ldg(a.bias + e) : 0.0)) : 0ull;
        }
    }
    if (a.n_groups > 1) {
        // group scores; lane g (and g + 32) keeps those of its group
        const int gs = a.n_exp / a.n_groups;
        unsigned long long gk[2] = {0ull, 0ull};
        for (int g = 0; g < a.n_groups; g++) {
            unsigned long long best = 0ull;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                const int e = lane + 32 * i;
                if (e / gs == g && key[i] > best) best = key[i];
            }
            const unsigned long long m1 = warp_max(best);
            unsigned long long score = m1;
            if (a.top2) {
                // the second largest: the first one's lowest-numbered holder steps aside
                int mine = 0x7FFFFFFF;
#pragma unroll
                for (int i = EPL - 1; i >= 0; i--) {
                    const int e = lane + 32 * i;
                    if (e / gs == g && key[i] == m1) mine = e;
                }
                const int first = __reduce_min_sync(0xffffffffu, mine);
                best = 0ull;
#pragma unroll
                for (int i = 0; i < EPL; i++) {
                    const int e = lane + 32 * i;
                    if (e / gs == g && e != first && key[i] > best) best = key[i];
                }
                score = order_key(key_value(m1) + key_value(warp_max(best)));
            }
            if ((g & 31) == lane) gk[g >> 5] = score;
        }
        // keep the best groups, ties to the lowest; a group without a usable score comes last
        unsigned long long keep = 0ull;  // bit g
        for (int r = 0; r < a.kept; r++) {
            unsigned long long b = 0ull;
            int bg = 0x7FFFFFFF;
#pragma unroll
            for (int h = 1; h >= 0; h--) {
                const int g = lane + 32 * h;
                if (g < a.n_groups && !((keep >> g) & 1ull) && gk[h] >= b) { b = gk[h]; bg = g; }
            }
            const unsigned long long m = warp_max(b);
            if (b != m) bg = 0x7FFFFFFF;
            keep |= 1ull << __reduce_min_sync(0xffffffffu, bg);
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = lane + 32 * i;
            if (e < a.n_exp && !((keep >> (e / gs)) & 1ull)) key[i] = 0ull;
        }
    }
    // the k largest, one after the other, ties to the lowest expert; lane r keeps the r-th
    int my_id = -1;
    for (int r = 0; r < a.top_k; r++) {
        unsigned long long b = 0ull;
        int be = 0x7FFFFFFF;
#pragma unroll
        for (int i = EPL - 1; i >= 0; i--)
            if (key[i] >= b && key[i]) { b = key[i]; be = lane + 32 * i; }
        const unsigned long long m = warp_max(b);
        if (m == 0ull) break;  // nothing usable is left
        if (b != m) be = 0x7FFFFFFF;
        const int e = __reduce_min_sync(0xffffffffu, be);
        if (lane == r) my_id = e;
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (lane + 32 * i == e) key[i] = 0ull;
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
// Each thread owns one contiguous run of the slots.
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
