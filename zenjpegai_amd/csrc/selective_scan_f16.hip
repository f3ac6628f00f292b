// Selective state-space scan: the kernels of whole sequences of f16 (gfx950 / CDNA4, wave64).
#include "selective_scan.h"

namespace zjai {

template <>
hipError_t launch_scan_kernels<_Float16>(const ScanArgs& a, const ScanPlan& p, bool outputs, float* scratch, hipStream_t s) {
    return outputs ? scan<_Float16, true>(a, p, scratch, s) : scan<_Float16, false>(a, p, scratch, s);
}

}  // namespace zjai
