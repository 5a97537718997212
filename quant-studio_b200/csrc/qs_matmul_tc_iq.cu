// tcgen05 tiles (qs_matmul_tc.cuh) of IQ2_XXS, IQ2_XS, IQ2_S, IQ3_XXS, IQ3_S.
#include "qs_matmul_tc.cuh"

namespace qs {

cudaError_t launch_mm_tc_iq(int type, const MmArgs& a, int bn, bool lo, void* ws, const LaunchCtx& ctx) {
    switch (type) {
    case QS_IQ2_XXS: return launch_tc<QS_IQ2_XXS>(a, bn, lo, ws, ctx);
    case QS_IQ2_XS: return launch_tc<QS_IQ2_XS>(a, bn, lo, ws, ctx);
    case QS_IQ2_S: return launch_tc<QS_IQ2_S>(a, bn, lo, ws, ctx);
    case QS_IQ3_XXS: return launch_tc<QS_IQ3_XXS>(a, bn, lo, ws, ctx);
    case QS_IQ3_S: return launch_tc<QS_IQ3_S>(a, bn, lo, ws, ctx);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qs
