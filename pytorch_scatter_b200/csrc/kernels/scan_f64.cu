// The recurrence on fp64 data (a translation unit of its own: the kernels of a type compile in parallel to the others').
#include "scan.cuh"

namespace tsb {
namespace scan {

int launch_f64(const ScanParams &p, int, bool backward, cudaStream_t stream) {
  return backward ? launch<double, double, true>(p, stream) : launch<double, double, false>(p, stream);
}

}  // namespace scan
}  // namespace tsb
