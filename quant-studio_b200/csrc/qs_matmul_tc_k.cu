// tcgen05 tiles (qs_matmul_tc.cuh) of Q2_K, Q3_K, Q4_K.
#include "qs_matmul_tc.cuh"

namespace qs {

cudaError_t launch_mm_tc_k(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx) {
    switch (type) {
    case QS_Q2_K: return launch_tc<QS_Q2_K>(a, bn, lo, ws, ctx);
    case QS_Q3_K: return launch_tc<QS_Q3_K>(a, bn, lo, ws, ctx);
    case QS_Q4_K: return launch_tc<QS_Q4_K>(a, bn, lo, ws, ctx);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qs
