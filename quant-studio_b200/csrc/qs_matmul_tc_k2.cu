// tcgen05 tiles (qs_matmul_tc.cuh) of Q5_K, Q6_K, IQ4_XS.
#include "qs_matmul_tc.cuh"

namespace qs {

cudaError_t launch_mm_tc_k2(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx) {
    switch (type) {
    case QS_Q5_K: return launch_tc<QS_Q5_K>(a, bn, lo, ws, ctx);
    case QS_Q6_K: return launch_tc<QS_Q6_K>(a, bn, lo, ws, ctx);
    case QS_IQ4_XS: return launch_tc<QS_IQ4_XS>(a, bn, lo, ws, ctx);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qs
