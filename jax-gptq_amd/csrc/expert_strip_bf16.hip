// The strip kernels of the experts' product for one type of activations (a translation unit each: they compile side by
// side).
#include "expert_strip.h"

int expert_strip_bf16(hipStream_t s, const ExpertArgs &a) { return xqmm::strip_launch<GPTQ_HIP_BF16>(s, a); }
