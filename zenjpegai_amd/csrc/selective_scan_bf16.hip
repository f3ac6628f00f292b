// Selective state-space scan: the kernels of whole sequences of bf16 (gfx950 / CDNA4, wave64).
#include "selective_scan.h"

namespace zjai {

template <>
hipError_t launch_scan_kernels<__bf16>(const ScanArgs& a, const ScanPlan& p, bool outputs, float* scratch, hipStream_t s) {
    return outputs ? scan<__bf16, true>(a, p, scratch, s) : scan<__bf16, false>(a, p, scratch, s);
}

}  // namespace zjai
