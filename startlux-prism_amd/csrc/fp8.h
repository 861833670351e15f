// e4m3 weights with block scales: what the GEMM (fp8.hip) and the experts (moe.hip) share.
#pragma once

#include "common.h"

namespace prism {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr float kE4m3Max = 448.f, kAmaxMin = 1e-10f;
constexpr int64_t kFp8MaxDim = 1 << 20;      // inputs and outputs of a weight: a 16-row tile stays far below 2^31 bytes
constexpr int64_t kFp8MaxLd = 1 << 22;       // row strides of activations: 64 rows stay below 2^30 bytes

}  // namespace prism
