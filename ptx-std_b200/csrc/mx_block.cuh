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

// ---- packed f32 pairs --------------------------------------------------------------------------
// sm_100's two-wide f32 instructions (two IEEE operations per issue slot); element 0 in the low
// half.
using f32x2 = uint64_t;
__device__ __forceinline__ f32x2 pack2f(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float hsum2(f32x2 v) {
    const float2 f = unpack2(v);
    return f.x + f.y;
}
// Eight bf16 values of a 16-byte vector as four pairs, and back (round to nearest even).
struct Oct {
    f32x2 v[4];
};
__device__ __forceinline__ Oct widen(const uint4& w) {
    Oct o;
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        o.v[k] = pack2f(data_types::bf16_lo(x[k]), data_types::bf16_hi(x[k]));
    return o;
}
__device__ __forceinline__ uint4 narrow(const Oct& o) {
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2(o.v[k]);
        x[k] = data_types::bf16x2_from_f32(f.x, f.y);
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
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

// Running block maximum of magnitudes, NaN-propagating like the quantisers of bf16; the pair form
// is one three-input maximum.
__device__ __forceinline__ float amax(float m, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
    return r;
}
__device__ __forceinline__ float amax(float m, float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(x)), "f"(fabsf(y)));
    return r;
}
template <uint32_t L>
__device__ __forceinline__ float amax_of(const float (&v)[L]) {
    float m = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < L; i += 2) m = amax(m, v[i], v[i + 1]);
    return m;
}
// The maximum over the four lanes that hold a block of 32 (eight values each).
__device__ __forceinline__ float amax_quad(float m) {
    m = amax(m, __shfl_xor_sync(0xffffffffu, m, 1));
    return amax(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
// Scale of a block from its largest magnitude: code = floor(log2 amax) + 127 - emax (E4M3 8,
// E5M2 15), clamped at 0, and inv = 2^-(code-127). The exponent field is the floor-pow2
// (TowardZero) code already; an infinite amax takes the largest finite exponent
// (SaturateFinite), a NaN gives the NaN code and a NaN factor. The code is at most 246, so inv is
// a normal number.
struct Scale {
    uint32_t code;
    float inv;
};
__device__ __forceinline__ Scale scale_of(float amax, uint32_t emax) {
    const uint32_t bits = __float_as_uint(amax);
    const uint32_t e = max(bits >> 23, emax);
    Scale s = {e - emax, __uint_as_float((254u + emax - e) << 23)};
    if (bits >= 0x7F800000u) {
        const bool nan = bits > 0x7F800000u;
        s.code = nan ? 0xFFu : 254u - emax;
        s.inv = __uint_as_float(nan ? 0x7FFFFFFFu : emax << 23);
    }
    return s;
}
// Two values times 2^-(code-127) (exact but for subnormal results) as a code pair.
template <uint32_t T>
__device__ __forceinline__ uint32_t pack2(float a, float b, float inv) {
    const float2 v = unpack2(mul2(pack2f(a, b), pack2f(inv, inv)));
    return T == kE4m3 ? data_types::e4m3x2_from_f32<false>(v.x, v.y)
                      : data_types::e5m2x2_from_f32<false>(v.x, v.y);
}
// Eight values as eight codes.
template <uint32_t T>
__device__ __forceinline__ uint2 pack8(const float* v, float inv) {
    return make_uint2(pack2<T>(v[0], v[1], inv) | (pack2<T>(v[2], v[3], inv) << 16),
                      pack2<T>(v[4], v[5], inv) | (pack2<T>(v[6], v[7], inv) << 16));
}
__device__ __forceinline__ uint2 pack8(uint32_t type, const float* v, float inv) {
    return type == kE4m3 ? pack8<kE4m3>(v, inv) : pack8<kE5m2>(v, inv);
}
__host__ __device__ __forceinline__ uint32_t emax_of(uint32_t type) {
    return type == kE4m3 ? 8u : 15u;
}

// ---- activations ------------------------------------------------------------------------------
// Hardware reciprocal (1 ulp): 1 / inf is 0.
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// sigmoid with the fast exponential and reciprocal (each within a few ulp of f32; every caller
// rounds the result to bf16 or to an 8-bit float). z -> -inf gives 0 through 1 / inf.
__device__ __forceinline__ float sigmoid(float z) { return rcp(1.0f + __expf(-z)); }

// 2 sqrt(2 / pi) and the cubic's factor: gelu_tanh(x) = x sigmoid(kG (x + kC x^3)).
constexpr float kG = 1.5957691216057308f;
constexpr float kC = 0.044715f;

// Normal distribution function Phi(x) and exp(-x^2 / 2). For x <= 0,
// Phi(x) = 0.5 erfcx(|x| / sqrt(2)) exp(-x^2 / 2), which keeps the lower tail's relative accuracy
// (1 + erf would cancel there). erfcx(z) = exp(z^2) erfc(z) is a degree-8 polynomial without
// constant term in t = 1 / (1 + 0.33 z) (the form of Abramowitz and Stegun 7.1.26), its
// coefficients fitted here for the least largest relative error on 0 <= z <= 9.6: 8.2e-8. Beyond,
// the exponential is below the smallest normal float. erfcf instead took act_backward_mx with
// GELU from 79 to 192 us at 4096 x 16384.
__device__ __forceinline__ float phi_cdf(float x, float& e) {
    const float t = rcp(fmaf(fabsf(x), 0.33f * 0.70710678f, 1.0f));
    e = __expf(-0.5f * x * x);
    float p = -0.067971688f;
    p = fmaf(p, t, 0.23137758f);
    p = fmaf(p, t, -0.17778363f);
    p = fmaf(p, t, 0.20633723f);
    p = fmaf(p, t, 0.022465308f);
    p = fmaf(p, t, 0.10097591f);
    p = fmaf(p, t, 0.091415916f);
    p = fmaf(p, t, 0.093183258f);
    const float q = p * t * e;
    return x > 0.0f ? 1.0f - q : q;
}
__device__ __forceinline__ float phi_cdf(float x) {
    float e;
    return phi_cdf(x, e);
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
        float e;
        const float t = phi_cdf(x, e);
        f = x * t;
        df = fmaf(x * 0.3989422804014327f, e, t);
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
