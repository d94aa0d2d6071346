// Device pieces shared by the operators that end in an MX operand or in an activation: the padded
// blocked scale layout, the block quantiser on f32 values, and the activations with their
// derivatives.
#pragma once

#include <cstddef>
#include <cstdint>

#include "common.cuh"
#include "data_types.cuh"

namespace ptxstd {

// ---- programmatic dependent launch ---------------------------------------------------------
__device__ __forceinline__ void pdl_launch_dependents() {
    asm volatile("griddepcontrol.launch_dependents;");
}
__device__ __forceinline__ void pdl_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

namespace mx {

// ---- blocked scales, padded ------------------------------------------------------------------
// Tiles of 128 rows x 4 scale columns, 512 bytes each, row-tile major, as the block-scaled GEMMs
// read them; rows and scale columns are padded up to whole tiles.
__host__ __device__ __forceinline__ size_t tiles_k(size_t sf_cols) { return (sf_cols + 3) >> 2; }
__host__ __device__ __forceinline__ size_t padded_rows(size_t rows) {
    return (rows + 127) & ~static_cast<size_t>(127);
}
// Offset of the four scales of row r, scale columns 4 t .. 4 t + 3 (4-byte aligned).
__host__ __device__ __forceinline__ size_t word_offset(size_t r, size_t t, size_t k_tiles) {
    return ((r >> 7) * k_tiles + t) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// ---- block quantiser on f32 ------------------------------------------------------------------
// Element types an operator can write: the one-byte ones, by their F8f6f4ElementType code.
constexpr uint32_t kE4m3 = 0, kE5m2 = 1;

// |x| and |y| folded into a running block maximum of magnitude bits: for non-negative f32
// patterns the integer order is the float order and every NaN sorts above infinity, so the
// maximum propagates NaN as the quantisers of bf16 do.
__device__ __forceinline__ uint32_t amax_bits(uint32_t m, float x) {
    return max(m, __float_as_uint(x) & 0x7FFFFFFFu);
}
// Scale code of a block from its magnitude bits: floor-pow2 (TowardZero, SaturateFinite) minus
// the format's emax (E4M3 8, E5M2 15), clamped at 0; NaN stays NaN.
__device__ __forceinline__ uint32_t scale_code(uint32_t bits, uint32_t emax) {
    const uint32_t u = data_types::ue8m0_from_f32<false, true>(__uint_as_float(bits));
    return u == 0xFFu ? 0xFFu : (u > emax ? u - emax : 0u);
}
// Two values times 2^-(code-127) (exact but for subnormal results) as a code pair.
template <uint32_t T>
__device__ __forceinline__ uint32_t pack2(float a, float b, float inv) {
    return T == kE4m3 ? data_types::e4m3x2_from_f32<false>(a * inv, b * inv)
                      : data_types::e5m2x2_from_f32<false>(a * inv, b * inv);
}
__device__ __forceinline__ uint32_t pack4(uint32_t type, float a, float b, float c, float d,
                                          float inv) {
    return type == kE4m3 ? pack2<kE4m3>(a, b, inv) | (pack2<kE4m3>(c, d, inv) << 16)
                         : pack2<kE5m2>(a, b, inv) | (pack2<kE5m2>(c, d, inv) << 16);
}
__host__ __device__ __forceinline__ uint32_t emax_of(uint32_t type) {
    return type == kE4m3 ? 8u : 15u;
}

// ---- activations ------------------------------------------------------------------------------
// sigmoid with the fast exponential and divide (each within a few ulp of f32; every caller rounds
// the result to bf16 or to an 8-bit float). z -> -inf gives 0 through 1 / inf.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// 2 sqrt(2 / pi) and its product with 3 * 0.044715: gelu_tanh(x) = x sigmoid(kG (x + c x^3)).
constexpr float kG = 1.5957691216057308f;
constexpr float kC = 0.044715f;

// Normal distribution function, accurate in the lower tail (1 + erf would cancel there).
__device__ __forceinline__ float phi_cdf(float x) {
    return 0.5f * erfcf(-0.7071067811865476f * x);
}

__device__ __forceinline__ float act(uint32_t kind, float x) {
    switch (kind) {
    case PTXSTD_ACT_RELU: return x < 0.0f ? 0.0f : x;  // a NaN stays NaN
    case PTXSTD_ACT_SILU: return x * sigmoid(x);
    case PTXSTD_ACT_GELU: return x * phi_cdf(x);
    case PTXSTD_ACT_GELU_TANH: return x * sigmoid(kG * x * (1.0f + kC * x * x));
    default: return x;
    }
}
// f(x) and f'(x) together (they share the exponential).
__device__ __forceinline__ void act_grad(uint32_t kind, float x, float& f, float& df) {
    switch (kind) {
    case PTXSTD_ACT_RELU:
        f = x < 0.0f ? 0.0f : x;
        df = x > 0.0f ? 1.0f : 0.0f;
        break;
    case PTXSTD_ACT_SILU: {
        const float t = sigmoid(x);
        f = x * t;
        df = t * (1.0f + x * (1.0f - t));
        break;
    }
    case PTXSTD_ACT_GELU: {
        const float t = phi_cdf(x);
        f = x * t;
        df = t + x * (0.3989422804014327f * __expf(-0.5f * x * x));
        break;
    }
    case PTXSTD_ACT_GELU_TANH: {
        const float x2 = fminf(x * x, 1.0e6f);  // t is 0 or 1 long before; keeps 0 * inf out
        const float t = sigmoid(kG * x * (1.0f + kC * x2));
        f = x * t;
        df = t + f * (1.0f - t) * (kG * (1.0f + 3.0f * kC * x2));
        break;
    }
    default:
        f = x;
        df = 1.0f;
    }
}

}  // namespace mx
}  // namespace ptxstd
