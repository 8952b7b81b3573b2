// The transposed kernels of the experts' product for one type of activations (a translation unit each: they compile
// side by side).
#include "expert_back.h"

int expert_back_bf16(hipStream_t s, const ExpertArgs &a, void *ws) { return xqmm::back_launch<GPTQ_HIP_BF16>(s, a, ws); }
