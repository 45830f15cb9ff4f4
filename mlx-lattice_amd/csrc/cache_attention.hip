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
    const bool f32 = a.dtype == LATTICE_F32;
    if ((f32 ? cache_many<float>(width) : cache_many<_Float16>(width)) && filled(32 * kAttnWaves) &&
        blocks(32 * kAttnWaves) >= kUnits) {
        l.share = false;
        l.tiles = 2;
    } else {
        // The largest tiles that are mostly filled and, their tokens split, give
        // every unit its blocks.
        const long long seen = std::min<long long>(
            static_cast<long long>(a.left) + a.right + a.sinks + std::min(a.queries, 16),
            static_cast<long long>(c.blocks) * kCacheBlock);
        const int most = f32 ? cache_most_tiles<float>(width) : cache_most_tiles<_Float16>(width);
        for (int tiles : {most, 2, 1}) {
            const long long own = blocks(16 * tiles), parts = std::min<long long>(64, seen / (tiles > 1 ? 2048 : 512));
            if (tiles > 1 && (!filled(16 * tiles) || own * std::max(1ll, parts) < kUnits / 2)) continue;
            l.tiles = tiles;
            if (own < kUnits) {
                const long long wanted = (tiles > 1 ? 2 : 4) * kUnits;
                l.splits = static_cast<int>(std::max(1ll, std::min(parts, (wanted + own - 1) / own)));
            }
            break;
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
