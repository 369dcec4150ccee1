// ffn_dev.h -- what the kernels between and inside the linears share: element types and activations.
#pragma once
#include "rt4_dev.h"

namespace rt4 {

// Element types and activations as the ABI numbers them (RT4_F32, RT4_BF16, RT4_F16; RT4_SILU, RT4_GELU_TANH).
enum { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum { kSilu = 0, kGeluTanh = 1 };
typedef __bf16 bf16;
typedef _Float16 f16;

// x / (1 + exp(-x)) or, by tanh's own definition, 0.5 x (1 + tanh z) = x / (1 + exp(-2 z)): one
// exponential to the base 2 and one reciprocal (1 ulp each).  The exponent's roundings are the largest
// error.  With u = 2^-24, relative to the result: silu 2 u |x| (the constant, the product), 1e-6 at
// x = -8; gelu 5 u |2 z| (a square, two constants, a fused sum, a product), 1.5e-5 at x = -8, where the
// result is 2e-21.  For x > 0 the exponential is the small term of the sum and so is its error.
// Where 1 / (1 + e) is below 2^-126 the reciprocal gives 0, and so does this function.
__device__ __forceinline__ float activate(float x, int act) {
    constexpr float log2e = 1.44269504088896341f, z = 2.0f * log2e * 0.79788456080286536f;
    const float e = x * (act == kSilu ? -log2e : fmaf(x * x, -z * 0.044715f, -z));
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(e));
}

}  // namespace rt4
