// tcgen05 tiles (qs_matmul_tc.cuh) of Q4_0, Q4_1, Q5_0, Q5_1, Q8_0.
#include "qs_matmul_tc.cuh"

namespace qs {

cudaError_t launch_mm_tc_legacy(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx) {
    switch (type) {
    case QS_Q4_0: return launch_tc<QS_Q4_0>(a, bn, lo, ws, ctx);
    case QS_Q4_1: return launch_tc<QS_Q4_1>(a, bn, lo, ws, ctx);
    case QS_Q5_0: return launch_tc<QS_Q5_0>(a, bn, lo, ws, ctx);
    case QS_Q5_1: return launch_tc<QS_Q5_1>(a, bn, lo, ws, ctx);
    case QS_Q8_0: return launch_tc<QS_Q8_0>(a, bn, lo, ws, ctx);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qs
