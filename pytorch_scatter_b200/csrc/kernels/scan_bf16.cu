// The recurrence on bf16 data (a translation unit of its own: the kernels of a type compile in parallel to the others').
#include "scan.cuh"

namespace tsb {
namespace scan {

int launch_bf16(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream) {
  if (gate_dtype == TSB_F32) return backward ? launch<__nv_bfloat16, float, true>(p, stream) : launch<__nv_bfloat16, float, false>(p, stream);
  return backward ? launch<__nv_bfloat16, __nv_bfloat16, true>(p, stream) : launch<__nv_bfloat16, __nv_bfloat16, false>(p, stream);
}

}  // namespace scan
}  // namespace tsb
