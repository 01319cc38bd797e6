// The recurrence on fp16 data (a translation unit of its own: the kernels of a type compile in parallel to the others').
#include "scan.cuh"

namespace tsb {
namespace scan {

int launch_f16(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream) {
  if (gate_dtype == TSB_F32) return backward ? launch<__half, float, true>(p, stream) : launch<__half, float, false>(p, stream);
  return backward ? launch<__half, __half, true>(p, stream) : launch<__half, __half, false>(p, stream);
}

}  // namespace scan
}  // namespace tsb
