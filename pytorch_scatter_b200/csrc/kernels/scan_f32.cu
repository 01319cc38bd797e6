// The recurrence on fp32 data (a translation unit of its own: the kernels of a type compile in parallel to the others').
#include "scan.cuh"

namespace tsb {
namespace scan {

int launch_f32(const ScanParams &p, int, bool backward, cudaStream_t stream) {
  return backward ? launch<float, float, true>(p, stream) : launch<float, float, false>(p, stream);
}

}  // namespace scan
}  // namespace tsb
