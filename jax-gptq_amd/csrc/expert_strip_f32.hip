// The strip kernels of the experts' product for one type of activations (a translation unit each: they compile side by
// side).
#include "expert_strip.h"

int expert_strip_f32(hipStream_t s, const ExpertArgs &a) { return xqmm::strip_launch<GPTQ_HIP_F32>(s, a); }
