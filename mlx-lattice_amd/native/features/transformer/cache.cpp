#include <ATen/DeviceGuard.h>

#include <algorithm>
#include <stdexcept>

#include "features/transformer/api.h"
#include "features/transformer/checks.h"

namespace lattice_native {

namespace {

constexpr int64_t kCacheBlock = 32;

void require_part(const at::Tensor& t, const at::Tensor& keys, at::ScalarType type, at::IntArrayRef shape,
                  const char* message) {
    if (t.scalar_type() != type || t.sizes() != shape) throw std::invalid_argument(message);
    require_device(t, "cache");
    if (t.device() != keys.device()) throw std::invalid_argument("the parts of a cache must be on one device.");
    if (!t.is_contiguous()) throw std::invalid_argument("the parts of a cache must be contiguous.");
}

lattice_cache cache_of(const CacheParts& parts, int64_t dim) {
    const auto& [keys, values, key_exponents, value_exponents] = parts;
    if (keys.dim() != 4) throw std::invalid_argument("cache keys must have shape (B, kv_heads, capacity, width).");
    const at::ScalarType type = keys.scalar_type();
    if (type != at::kFloat8_e4m3fn && type != at::kChar) {
        throw std::invalid_argument("cache codes must be float8_e4m3fn or int8.");
    }
    if (dim < 1 || dim > 128) throw std::invalid_argument("cache heads must have between 1 and 128 channels.");
    const int64_t b = keys.size(0), heads = keys.size(1), capacity = keys.size(2), width = keys.size(3);
    if (heads < 1) throw std::invalid_argument("a cache must have a key head.");
    if (capacity % kCacheBlock != 0) throw std::invalid_argument("a cache's capacity must be a multiple of 32.");
    if (width != (dim + 31) / 32 * 32) {
        throw std::invalid_argument("cache rows must be the head's channels rounded up to a multiple of 32.");
    }
    const int64_t blocks = capacity / kCacheBlock;
    require_part(keys, keys, type, {b, heads, capacity, width}, "");
    require_part(values, keys, type, {b, heads, blocks, width, kCacheBlock},
                 "cache values must have shape (B, kv_heads, capacity / 32, width, 32) and the keys' dtype.");
    for (const at::Tensor& e : {key_exponents, value_exponents}) {
        require_part(e, keys, at::kChar, {b, heads, blocks},
                     "cache exponents must have shape (B, kv_heads, capacity / 32) and int8 dtype.");
    }
    lattice_cache c;
    c.code = type == at::kChar ? LATTICE_CODE_INT8 : LATTICE_CODE_E4M3;
    if (b > kMost || heads > kMost || blocks > kMost) throw std::invalid_argument("the cache is too large.");
    c.sequences = static_cast<int>(b);
    c.kv_heads = static_cast<int>(heads);
    c.blocks = static_cast<int>(blocks);
    c.dim = static_cast<int>(dim);
    c.keys = keys.data_ptr();
    c.values = values.data_ptr();
    c.key_exponents = key_exponents.data_ptr<int8_t>();
    c.value_exponents = value_exponents.data_ptr<int8_t>();
    return c;
}

void require_layout(const at::Tensor& offsets, const at::Tensor& lengths, const at::Tensor& like, int64_t sequences) {
    require_index(offsets, like, sequences + 1, "offsets must have shape (B + 1,) and int32 dtype.");
    require_index(lengths, like, sequences, "lengths must have shape (B,) and int32 dtype.");
    if (!offsets.is_contiguous() || !lengths.is_contiguous()) {
        throw std::invalid_argument("offsets and lengths must be contiguous.");
    }
}

void refuse_grad(const at::Tensor& t) {
    if (at::GradMode::is_enabled() && t.requires_grad()) {
        throw std::runtime_error("an 8-bit cache has no gradient: use it under torch.no_grad().");
    }
}

// Rows of heads with unit stride in the channels, or a copy.
at::Tensor unit_heads(const at::Tensor& t) { return t.size(2) == 1 || t.stride(2) == 1 ? t : t.contiguous(); }
long long head_stride(const at::Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; }

}  // namespace

void cache_write(const CacheParts& parts, int64_t dim, const at::Tensor& k_in, const at::Tensor& v_in,
                 const at::Tensor& offsets, const at::Tensor& lengths) {
    refuse_tangents({k_in, v_in});
    const lattice_cache c = cache_of(parts, dim);
    if (k_in.dim() != 3 || k_in.size(1) != c.kv_heads || k_in.size(2) != dim || v_in.sizes() != k_in.sizes()) {
        throw std::invalid_argument("k and v must have shape (N, kv_heads, dim) of the cache.");
    }
    const int dtype = dtype_code(k_in, "k and v");
    require_device(k_in, "k");
    require_same(v_in, k_in, "v");
    if (k_in.device() != std::get<0>(parts).device()) {
        throw std::invalid_argument("the cache must be on the same device.");
    }
    require_layout(offsets, lengths, k_in, c.sequences);
    refuse_grad(k_in);
    refuse_grad(v_in);
    const at::DeviceGuard guard(k_in.device());
    const at::Tensor k = unit_heads(k_in), v = unit_heads(v_in);
    check_status(lattice_hip_cache_write(&c, dtype, k.data_ptr(), row_stride(k), head_stride(k), v.data_ptr(),
                                         row_stride(v), head_stride(v), row_count(k, "k"), ci32(offsets),
                                         ci32(lengths), current_stream(k)));
    const auto& [keys, values, key_exponents, value_exponents] = parts;
    for (const at::Tensor& t : {keys, values, key_exponents, value_exponents})
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

std::tuple<at::Tensor, at::Tensor> cache_read(const CacheParts& parts, int64_t dim, const at::Tensor& lengths,
                                              at::ScalarType type) {
    const lattice_cache c = cache_of(parts, dim);
    const at::Tensor& keys = std::get<0>(parts);
    require_index(lengths, keys, c.sequences, "lengths must have shape (B,) and int32 dtype.");
    if (!lengths.is_contiguous()) throw std::invalid_argument("lengths must be contiguous.");
    const at::DeviceGuard guard(keys.device());
    const auto options = keys.options().dtype(type);
    at::Tensor k = at::empty({c.sequences, keys.size(2), c.kv_heads, dim}, options);
    at::Tensor v = at::empty(k.sizes(), options);
    check_status(lattice_hip_cache_read(&c, dtype_code(k, "rows of a cache"), ci32(lengths), k.data_ptr(),
                                        v.data_ptr(), current_stream(k)));
    return {k, v};
}

at::Tensor cache_attention(const at::Tensor& q_in, const CacheParts& parts, int64_t dim, const at::Tensor& offsets,
                           const at::Tensor& lengths, int64_t left, int64_t right, int64_t sinks, double scale) {
    refuse_tangents({q_in});
    lattice_cache c = cache_of(parts, dim);
    if (q_in.dim() != 3 || q_in.size(2) != dim) {
        throw std::invalid_argument("q must have shape (N, heads, dim) of the cache.");
    }
    lattice_cache_attention a;
    a.dtype = dtype_code(q_in, "q");
    require_row_values(q_in.size(1), dim, "q");
    if (q_in.size(1) < 1 || q_in.size(1) % c.kv_heads != 0) {
        throw std::invalid_argument("the number of heads must be a multiple of the number of key heads.");
    }
    if (left < 0 || right < 0 || sinks < 0) {
        throw std::invalid_argument("left, right and sinks must be non-negative.");
    }
    require_device(q_in, "q");
    if (q_in.device() != std::get<0>(parts).device()) {
        throw std::invalid_argument("the cache must be on the same device.");
    }
    require_layout(offsets, lengths, q_in, c.sequences);
    refuse_grad(q_in);
    const at::DeviceGuard guard(q_in.device());
    const at::Tensor q = pieces(q_in, q_in.size(1) / c.kv_heads);
    // Channels up to whole 16-byte pieces: the cache's are zeros.
    c.dim = static_cast<int>(q.size(2));
    a.queries = row_count(q, "q");
    a.heads = static_cast<int>(q.size(1));
    a.left = static_cast<int>(std::min(left, kMost));
    a.right = static_cast<int>(std::min(right, kMost));
    a.sinks = static_cast<int>(std::min(sinks, kMost));
    a.scale = static_cast<float>(scale);
    a.q = q.data_ptr();
    a.q_row_stride = row_stride(q);
    a.q_head_stride = head_stride(q);
    a.offsets = ci32(offsets);
    a.lengths = ci32(lengths);
    at::Tensor out = at::empty(q.sizes(), q.options());
    const size_t bytes = lattice_hip_cache_attention_workspace_bytes(&c, &a);
    at::Tensor ws;
    if (bytes) ws = workspace(bytes, q);
    check_status(lattice_hip_cache_attention(&c, &a, out.data_ptr(), or_null(ws), bytes, current_stream(q)));
    return unpadded(out, dim);
}

}  // namespace lattice_native
