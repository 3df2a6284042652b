// What the operators on sequences share: their element types and 16-byte access.
#pragma once
#include <algorithm>

#include "common.hpp"

namespace cpde {

using bf16 = __bf16;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <class T, int N>
using vec = T __attribute__((ext_vector_type(N)));

inline size_t type_bytes(int dtype) { return dtype == CPDE_F32 ? 4 : 2; }
inline void check_dtype(int dtype) {
    require(dtype == CPDE_F32 || dtype == CPDE_F16 || dtype == CPDE_BF16, "unknown element type");
}
// Calls body with a value of the element type.
template <class F>
void with_type(int dtype, F body) {
    if (dtype == CPDE_F32) body(float{});
    else if (dtype == CPDE_F16) body(_Float16{});
    else body(bf16{});
}

// Whether an address and an element stride are whole multiples of 16 bytes.
inline bool wide(const void* p, int64_t stride, size_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * int64_t(size) % 16 == 0;
}


}  // namespace cpde
