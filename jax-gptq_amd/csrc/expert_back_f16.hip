// The transposed kernels of the experts' product for one type of activations (a translation unit each: they compile
// side by side).
#include "expert_back.h"

int expert_back_f16(hipStream_t s, const ExpertArgs &a, void *ws) { return xqmm::back_launch<GPTQ_HIP_F16>(s, a, ws); }
