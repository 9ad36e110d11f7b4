// Element types of the catalogue operators (NCF_F32 / NCF_BF16 / NCF_F16) and their loads and stores.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "movierec_ncf.h"

namespace ncf {

typedef float vf32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t vu32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes, element aligned
    static constexpr int kVec = 4;
};
template <>
struct Elem<__bf16> {
    typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
    static constexpr int kVec = 8;
};
template <>
struct Elem<_Float16> {
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
    static constexpr int kVec = 8;
};

// 16 bytes at any byte address (one global_load_dwordx4: MI355X loads unaligned vectors)
__device__ __forceinline__ vu32x4 load16(const void* p) {
    typedef uint32_t u __attribute__((ext_vector_type(4), aligned(1)));
    return *reinterpret_cast<const u*>(p);
}

}  // namespace ncf
