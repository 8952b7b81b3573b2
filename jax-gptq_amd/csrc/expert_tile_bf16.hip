// The tile kernels of the experts' product for one type of activations (a translation unit each: they compile side by
// side).
#include "expert_tile.h"

int expert_tile_bf16(hipStream_t s, const ExpertArgs &a, int shape, void *ws) {
  return xqmm::tile_launch<GPTQ_HIP_BF16>(s, a, shape, ws);
}
