// 16-bit floats in and out of registers, by the QM_IN_* type they are stored in.
#pragma once
#include "qm_common.hpp"
#include "../../include/qm_abi.h"

namespace qm {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

static_assert(QM_IN_F16 == (int)OUT_F16 && QM_IN_BF16 == (int)OUT_BF16, "one number for a 16-bit type, in or out");

template <int T>
__device__ __forceinline__ float float_of(uint16_t bits)
{
    if constexpr (T == QM_IN_F16) return (float)__builtin_bit_cast(_Float16, bits);
    else return __builtin_bit_cast(float, (uint32_t)bits << 16);
}
// element i of an array of type T (QM_IN_F16, QM_IN_BF16 or QM_IN_F32)
template <int T>
__device__ __forceinline__ float element(const void *p, size_t i)
{
    if constexpr (T == QM_IN_F32) return static_cast<const float *>(p)[i];
    else return float_of<T>(static_cast<const uint16_t *>(p)[i]);
}

}  // namespace qm
