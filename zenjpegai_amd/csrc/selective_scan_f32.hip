// Selective state-space scan: the kernels of whole sequences of f32 (gfx950 / CDNA4, wave64).
#include "selective_scan.h"

namespace zjai {

template <>
hipError_t launch_scan_kernels<float>(const ScanArgs& a, const ScanPlan& p, bool outputs, float* scratch, hipStream_t s) {
    return outputs ? scan<float, true>(a, p, scratch, s) : scan<float, false>(a, p, scratch, s);
}

}  // namespace zjai
