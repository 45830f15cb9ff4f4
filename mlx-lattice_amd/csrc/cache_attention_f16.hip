// Attention over an 8-bit cache with queries in _Float16.
#include "cache_attention_kernels.h"

int lattice::cache_attend_f16(const CacheCall& call, const CacheLayout& layout, const CachePart& part, void* out,
                             hipStream_t stream) {
    return launch_cache<_Float16>(call, layout, part, out, stream);
}
