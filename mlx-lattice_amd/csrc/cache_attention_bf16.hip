// Attention over an 8-bit cache with queries in __bf16.
#include "cache_attention_kernels.h"

int lattice::cache_attend_bf16(const CacheCall& call, const CacheLayout& layout, const CachePart& part, void* out,
                             hipStream_t stream) {
    return launch_cache<__bf16>(call, layout, part, out, stream);
}
