// Checks and layouts that the transformer operators share.
#pragma once

#include <torch/extension.h>

#include <algorithm>
#include <initializer_list>
#include <limits>
#include <stdexcept>
#include <string>

#include "foundation/runtime.h"

namespace lattice_native {

inline int dtype_code(const at::Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return LATTICE_F32;
        case at::kHalf: return LATTICE_F16;
        case at::kBFloat16: return LATTICE_BF16;
        default: throw std::invalid_argument(std::string(what) + " must be float32, float16 or bfloat16.");
    }
}

inline constexpr int64_t kMost = std::numeric_limits<int32_t>::max();

inline int row_count(const at::Tensor& t, const char* what) {
    if (t.size(0) > kMost) throw std::invalid_argument(std::string(what) + " has too many rows.");
    return static_cast<int>(t.size(0));
}

// The kernels count the values of a row in 32 bits.
inline void require_row_values(int64_t heads, int64_t dim, const char* what) {
    if (dim > 0 && heads > (kMost - 64) / dim) throw std::invalid_argument(std::string(what) + " are too wide.");
}

// A tangent of forward-mode differentiation would be lost.
inline void refuse_tangents(std::initializer_list<at::Tensor> tensors) {
    for (const at::Tensor& t : tensors) {
        if (t.defined() && t._fw_grad(/*level=*/0).defined())
            throw std::runtime_error("the transformer operators have no forward-mode derivatives.");
    }
}

inline at::Tensor or_undefined(const c10::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); }

inline void require_same(const at::Tensor& t, const at::Tensor& like, const char* what) {
    require_device(t, what);
    if (t.device() != like.device()) throw std::invalid_argument(std::string(what) + " must be on the same device.");
    if (t.scalar_type() != like.scalar_type()) throw std::invalid_argument(std::string(what) + " must share a dtype.");
}

inline void require_index(const at::Tensor& t, const at::Tensor& like, int64_t size, const char* message) {
    if (t.dim() != 1 || t.size(0) != size || t.scalar_type() != at::kInt) throw std::invalid_argument(message);
    require_device(t, "offsets");
    if (t.device() != like.device()) throw std::invalid_argument("offsets must be on the same device.");
}

// Rows of unit stride (any row stride), or a copy.
inline at::Tensor unit_rows(const at::Tensor& t) {
    return t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous();
}
inline long long row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }

inline const void* data_or_null(const c10::optional<at::Tensor>& t) {
    return t && t->defined() ? t->data_ptr() : nullptr;
}

inline const int32_t* active_or_null(const c10::optional<at::Tensor>& t, const at::Tensor& like) {
    if (!t || !t->defined()) return nullptr;
    require_index(*t, like, 1, "active_rows must have shape (1,) and int32 dtype.");
    return ci32(*t);
}

inline at::Tensor channel_vector(const c10::optional<at::Tensor>& t, const at::Tensor& x, const char* what) {
    if (!t || !t->defined()) return {};
    require_same(*t, x, what);
    if (t->dim() != 1 || t->size(0) != x.size(1)) {
        throw std::invalid_argument(std::string(what) + " must have shape (C,).");
    }
    return t->contiguous();
}

inline void* or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

inline int64_t piece_of(const at::Tensor& t) { return 16 / t.element_size(); }

// group: heads that are read together.
inline bool in_pieces(const at::Tensor& t, int64_t group) {
    const int64_t piece = piece_of(t);
    return t.stride(2) == 1 && (t.size(0) <= 1 || (t.stride(0) % piece == 0 && t.stride(0) < piece << 18)) &&
           (t.size(1) <= 1 || (t.stride(1) % piece == 0 && t.stride(1) < (piece << 25) / group)) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// Heads of whole 16-byte pieces on 16-byte boundaries, not too far apart: `t`
// itself, or a copy with the channels padded by zeros, which add nothing to a
// product.
inline at::Tensor pieces(const at::Tensor& t, int64_t group = 1) {
    const int64_t piece = piece_of(t), dim = t.size(2), padded = (dim + piece - 1) / piece * piece;
    if (padded != dim) return at::constant_pad_nd(t, {0, padded - dim}).contiguous();
    if (in_pieces(t, group)) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

// The first `dim` channels of padded heads.
inline at::Tensor unpadded(const at::Tensor& t, int64_t dim) {
    return t.size(2) == dim ? t : t.narrow(2, 0, dim).contiguous();
}

}  // namespace lattice_native
