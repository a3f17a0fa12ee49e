// Helpers shared by the translation units of the compiled module `torchsplinekan_b200._C`.
#pragma once
#include <torch/extension.h>

#include <string>

#include "../../include/kan_b200.h"

namespace kan_ext {

using at::Tensor;

inline bool has(const Tensor& t) { return t.defined() && t.numel() > 0; }
inline const void* cptr(const Tensor& t) { return has(t) ? t.data_ptr() : nullptr; }
inline void* mptr(Tensor& t) { return has(t) ? t.data_ptr() : nullptr; }

inline void check_rc(int rc) {
    if (rc == KANB200_OK) return;
    const std::string msg = kanb200_last_error();
    if (rc == KANB200_EINVAL) TORCH_CHECK(false, msg);
    TORCH_CHECK(false, "kan_b200 error ", rc, ": ", msg);
}

// An activation [rows, width] as 8-bit codes with one scale per 128 columns of a row (kan_block_ext.cpp); format:
// KANB200_PACK_INT8 or _E4M3.
struct Packed {
    Tensor codes, scales;
};
Packed pack_rows(const Tensor& x, int format);
Tensor unpack_rows(const Tensor& codes, const Tensor& scales, at::ScalarType dtype);

void bind_block_operators(pybind11::module_& m);

}  // namespace kan_ext
