// The tile kernels of the experts' product for one type of activations (a translation unit each: they compile side by
// side).
#include "expert_tile.h"

int expert_tile_f16(hipStream_t s, const ExpertArgs &a, int shape, void *ws) {
  return xqmm::tile_launch<GPTQ_HIP_F16>(s, a, shape, ws);
}
