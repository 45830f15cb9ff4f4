#include "attention_grad_kernels.h"

namespace lattice {

template int attend_grad<float>(const lattice_attention&, const GradLayout&, const void*, const void*, const float*,
                                const void*, void*, void*, void*, float2*, const FirstParts&, hipStream_t);

}  // namespace lattice
