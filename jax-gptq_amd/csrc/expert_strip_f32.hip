// The strip kernels of the experts' product for one type of activations (a translation unit each: they compile side by
// side).
#include "expert_strip.h"

int expert_strip_f32(hipStream_t s, const ExpertArgs &a, int row_blocks) {
  if (row_blocks == 1) return xqmm::strip_launch<GPTQ_HIP_F32, 1, 8>(s, a);
  return xqmm::strip_launch<GPTQ_HIP_F32, 2, 8>(s, a);
}
