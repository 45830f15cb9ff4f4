// Attention over an 8-bit cache: what its units of translation share.
#pragma once

#include "cache.h"

namespace lattice {

// A part of a row's softmax, over some of its tokens: the largest score (log2),
// the sum of exp2(score - top), and the average of v by those shares.
struct CachePart {
    float* values;   // [splits][queries * heads][dim]
    float2* states;  // [splits][queries * heads]: (top, sum)
};

// How a call is laid out.
struct CacheLayout {
    bool share;       // the waves of a block share their pairs and split the tokens, or have pairs of their own
    int tiles;        // tiles of 16 (query, head) pairs a wave
    int splits;       // blocks that split a pair's tokens
    long long slots;  // blocks of pairs at most
    int rows() const { return 16 * tiles * (share ? 1 : kAttnWaves); }
};

// Most tiles of pairs that fit a wave's registers.  2 x 2048 queries of 16 heads
// in float32 over 8192 tokens, us with one and two: 469 and 409 at 64 channels, 786
// and 671 at 128, where some 70 bytes a lane no longer fit.
template <typename T> constexpr int cache_most_tiles(int width) {
    return sizeof(T) == 4 ? (width == 32 ? 4 : 2) : width <= 64 ? 4 : width == 96 ? 3 : 2;
}
// Where widening a block's codes once for four waves, by way of LDS, is faster: 2
// x 2048 queries of 16 heads over 16384 tokens take 588 us against 679 with two
// tiles that widen their own in bfloat16, 4096 queries 597 against 680 from int8
// in half precision.  Narrower heads have three or four tiles to a widening.
template <typename T> constexpr bool cache_many(int width) { return width == 128 && sizeof(T) == 2; }

// Both structures, with bounds that keep positions inside 32 bits.
struct CacheCall {
    lattice_cache cache;
    lattice_cache_attention args;
};

int cache_attend_f32(const CacheCall& call, const CacheLayout& layout, const CachePart& part, void* out,
                     hipStream_t stream);
int cache_attend_f16(const CacheCall& call, const CacheLayout& layout, const CachePart& part, void* out,
                     hipStream_t stream);
int cache_attend_bf16(const CacheCall& call, const CacheLayout& layout, const CachePart& part, void* out,
                      hipStream_t stream);

}  // namespace lattice
