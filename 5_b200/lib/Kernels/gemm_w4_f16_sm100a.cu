// The 4-bit products of gemm_w4.cuh for float16 rows (a source of its own, to compile beside the other type's).
#include "gemm_w4.cuh"

namespace hc {
namespace sm100 {

cudaError_t launch_gemm_w4_f16(const CUtensorMap *tmap_q, const CUtensorMap &tmap_a, const W4 &p, int *status,
                               cudaStream_t stream) {
  return w4::launch_w4<false>(tmap_q, tmap_a, p, status, stream);
}

}  // namespace sm100
}  // namespace hc
