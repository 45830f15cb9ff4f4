// Attention over an 8-bit cache: how a call is laid out, and its entry.

#include "cache_attention.h"

namespace lattice {
namespace {

// What the entry checks; NULL, or what is wrong.
const char* cache_attention_fault(const lattice_cache* c, const lattice_cache_attention* a) {
    if (const char* fault = cache_fault(c)) return fault;
    if (!a) return "attention arguments must be non-null.";
    if (a->dtype != LATTICE_F32 && a->dtype != LATTICE_F16 && a->dtype != LATTICE_BF16)
        return "attention supports float32, float16 and bfloat16.";
    if (a->queries < 0 || a->queries >= 1 << 28) return "cache attention takes up to 2^28 - 1 rows of queries.";
    if (a->heads < 1 || a->heads % c->kv_heads != 0)
        return "the number of heads must be a multiple of the number of key heads.";
    if (static_cast<long long>(a->queries) * a->heads >= 1ll << 31)
        return "attention takes up to 2^31 - 1 rows of heads.";
    if (a->left < 0 || a->right < 0 || a->sinks < 0) return "left, right and sinks must be non-negative.";
    if (a->queries == 0) return nullptr;
    if (!a->q || !a->offsets || (c->sequences > 0 && !a->lengths)) return "attention pointers must be non-null.";
    const long long piece = 16 / (a->dtype == LATTICE_F32 ? 4 : 2);
    if (a->q_row_stride < 0 || a->q_head_stride < 0 || a->q_row_stride % piece != 0 || a->q_head_stride % piece != 0)
        return "attention strides must be whole 16-byte pieces.";
    if (c->dim % piece != 0) return "attention rows must be whole 16-byte pieces.";
    if (reinterpret_cast<uintptr_t>(a->q) % 16 != 0) return "attention rows must lie on 16-byte boundaries.";
    return nullptr;
}

constexpr int kUnits = 512;  // blocks that fill the chip, two a unit

CacheCall cache_call(const lattice_cache& c, const lattice_cache_attention& a) {
    CacheCall call{c, a};
    // Positions stay below 2^29 + 2^28, the sums with these inside 32 bits.
    constexpr int kFar = 1 << 30;
    static_assert(kCacheLongest <= 1 << 29);
    call.args.left = std::min(a.left, kFar);
    call.args.right = std::min(a.right, kFar);
    call.args.sinks = std::min(a.sinks, c.blocks * kCacheBlock);
    return call;
}

CacheLayout cache_layout(const CacheCall& call) {
    const lattice_cache& c = call.cache;
    const lattice_cache_attention& a = call.args;
    const int group = a.heads / c.kv_heads, width = cache_width(c);
    const long long pairs = static_cast<long long>(a.queries) * group;
    const int sequences = std::max(1, c.sequences);
    // Blocks that have rows.
    const auto blocks = [&](int rows) {
        return std::max<long long>((pairs + rows - 1) / rows, std::min<long long>(sequences, a.queries)) * c.kv_heads;
    };
    const auto filled = [&](int rows) { return 2 * pairs > static_cast<long long>(rows) * sequences; };
    CacheLayout l{true, 1, 1, 0};
    // Rows of their own for the waves where that fills the chip.  One sequence of
    // 16 heads over 4 key heads in bfloat16 over 16384 tokens, us with and without,
    // by blocks of 128 pairs: 64 404 and 122, 128 407 and 197, 256 408 and 355, 352
    // 542 and 502, 512 564 and 636, 752 808 and 886, 1024 950 and 1098.  In a window
    // of 1024: 128 36 and 23, 256 37 and 43, 512 55 and 81; prompts that see only
    // themselves, whose last rows are the longest: 256 59 and 45, 512 133 and 125.
    const bool f32 = a.dtype == LATTICE_F32;
    if ((f32 ? cache_many<float>(width) : cache_many<_Float16>(width)) && filled(32 * kAttnWaves) &&
        blocks(32 * kAttnWaves) >= kUnits) {
        l.share = false;
        l.tiles = 2;
    } else {
        // Tiles that share the codes' reads and widening, if the chip stays full.
        // Queries of 8 heads over 2 key heads in bfloat16, us with one, two and the
        // most tiles: 4 x 512 over 4096 tokens 27, 28, 33 at 32 channels, 43, 40, 44
        // at 96; 4 x 333 of 8 key heads in a window of 1024 12, 14, 16 at 32 and 30,
        // 25 at 128; 2 x 2048 of 16 heads over 16384 tokens 548, 362, 323 at 64.
        // 128 queries over 8192 tokens, split in its best way, 14.5 and 15.0 at 32,
        // 30 and 24 at 128.
        const int most = f32 ? cache_most_tiles<float>(width) : cache_most_tiles<_Float16>(width);
        const int pair_blocks = f32 || width <= 64 ? kUnits : kUnits / 4;
        const long long seen = std::min<long long>(
            static_cast<long long>(a.left) + a.right + a.sinks + std::min(a.queries, 16),
            static_cast<long long>(c.blocks) * kCacheBlock);
        const auto parts = [&](int tiles) { return std::max(1ll, std::min<long long>(64, seen / (tiles > 1 ? 2048 : 1024))); };
        if (most > 2 && filled(16 * most) && blocks(16 * most) >= kUnits) {
            l.tiles = most;
        } else if (filled(32) && blocks(32) * parts(2) >= pair_blocks) {
            l.tiles = 2;
        }
        // Parts of 1024 tokens or more, 256 a wave, since each is joined in a
        // launch of its own.  One query of 16 heads over 4 key heads of 32 caches,
        // us in 1, 4, 8 and 16 parts: 8000 tokens of 64 channels 27, 24, 25, 26,
        // 32768 of 128 -, 192, 169, 165.
        const long long own = blocks(16 * l.tiles);
        if (own < kUnits) {
            const long long wanted = (l.tiles > 1 ? 2 : 4) * kUnits;
            l.splits = static_cast<int>(std::min(parts(l.tiles), (wanted + own - 1) / own));
        }
    }
    l.slots = pairs / l.rows() + c.sequences + 2;
    return l;
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" size_t lattice_hip_cache_attention_workspace_bytes(const lattice_cache* cache,
                                                              const lattice_cache_attention* args) {
    if (cache_attention_fault(cache, args) || args->queries == 0) return 0;
    const CacheLayout l = cache_layout(cache_call(*cache, *args));
    if (l.splits == 1) return 0;
    const size_t rows = static_cast<size_t>(l.splits) * args->queries * args->heads;
    return aligned_bytes(rows * cache->dim * sizeof(float)) + aligned_bytes(rows * sizeof(float2));
}

extern "C" int lattice_hip_cache_attention_layout(const lattice_cache* cache, const lattice_cache_attention* args,
                                                  int* share, int* tiles, int* splits) {
    if (const char* fault = cache_attention_fault(cache, args)) {
        set_error(fault);
        return LATTICE_ERROR_INVALID_ARGUMENT;
    }
    LATTICE_REQUIRE(share && tiles && splits, "attention pointers must be non-null.");
    const CacheLayout l = cache_layout(cache_call(*cache, *args));
    *share = l.share;
    *tiles = l.tiles;
    *splits = l.splits;
    return LATTICE_OK;
}

extern "C" int lattice_hip_cache_attention(const lattice_cache* cache, const lattice_cache_attention* args, void* out,
                                           void* workspace, size_t workspace_bytes, void* stream_ptr) {
    if (const char* fault = cache_attention_fault(cache, args)) {
        set_error(fault);
        return LATTICE_ERROR_INVALID_ARGUMENT;
    }
    if (args->queries == 0) return LATTICE_OK;
    LATTICE_REQUIRE(out, "attention pointers must be non-null.");
    const CacheCall call = cache_call(*cache, *args);
    const CacheLayout l = cache_layout(call);
    LATTICE_REQUIRE(l.slots * cache->kv_heads * l.splits < 1ll << 36, "the cache has too many sequences and heads.");
    CachePart part{nullptr, nullptr};
    if (l.splits > 1) {
        Workspace ws{static_cast<char*>(workspace), workspace ? workspace_bytes : 0};
        const size_t rows = static_cast<size_t>(l.splits) * args->queries * args->heads;
        part.values = ws.take<float>(rows * cache->dim);
        part.states = ws.take<float2>(rows);
        LATTICE_REQUIRE(part.values && part.states, "attention workspace is too small.");
    }
    hipStream_t stream = as_stream(stream_ptr);
    if (args->dtype == LATTICE_F32) return cache_attend_f32(call, l, part, out, stream);
    if (args->dtype == LATTICE_F16) return cache_attend_f16(call, l, part, out, stream);
    return cache_attend_bf16(call, l, part, out, stream);
}
