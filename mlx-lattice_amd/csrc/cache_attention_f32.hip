// Attention over an 8-bit cache with queries in float.
#include "cache_attention_kernels.h"

int lattice::cache_attend_f32(const CacheCall& call, const CacheLayout& layout, const CachePart& part, void* out,
                             hipStream_t stream) {
    return launch_cache<float>(call, layout, part, out, stream);
}
