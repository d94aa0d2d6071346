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
__device__ __forceinline__ void flatten(const Oct& o, float (&a)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2(o.v[k]);
        a[2 * k] = f.x;
        a[2 * k + 1] = f.y;
    }
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
// On pairs: the multiplies and adds are packed, the exponential and the reciprocal are one hardware
// instruction per element (2 and 1 ulp). Results are rounded to bf16 or to an 8-bit float, but for
// the f32 column sums of act_backward_mx. Far out in the lower tails the exponential's argument is
// large and its f32 rounding shows: up to 3e-5 of the result (z near 128), still well below bf16's
// 2^-9. Where even the tail is out of range the result is zero: below logistic2's 2^-128, and with
// GELU where the density is below 2^-126 (|x| > 13.15, the result is then subnormal).
__device__ __forceinline__ f32x2 splat(float a) { return pack2f(a, a); }
__device__ __forceinline__ f32x2 exp2_2(f32x2 v) {
    const float2 f = unpack2(v);
    float a, b;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(f.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(f.y));
    return pack2f(a, b);
}
__device__ __forceinline__ f32x2 rcp2(f32x2 v) {  // 1 / inf is 0
    const float2 f = unpack2(v);
    float a, b;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(f.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(f.y));
    return pack2f(a, b);
}
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + 2^z): with z = -x log2(e) the logistic function of x. x -> -inf gives 1 / inf = 0.
// The reciprocal is taken of the denominator times 2^-8 (an fma instead of an add), because the
// instruction flushes results below 2^-126 to zero: without that SiLU is zero from x = -87.3 on,
// where it is -1e-36. With it a result is zero only where 2^z overflows (z >= 128: x < -88.7, the
// logistic function below 2^-128). Scaling z instead would reach further and round small z coarser.
// It costs act_backward_mx about 1 % (SiLU, 2048 x 4096: 13.4 -> 13.7 us; 4096 x 16384 within the
// noise of the clock); the instruction that keeps subnormal results cost 12 to 17 %.
__device__ __forceinline__ f32x2 logistic2(f32x2 z) {
    const f32x2 c = splat(0.00390625f);
    return mul2(rcp2(fma2(exp2_2(z), c, c)), c);
}

// gelu_tanh(x) = x sigmoid(kG (x + kC x^3)), kG = 2 sqrt(2 / pi).
constexpr float kG = 1.5957691216057308f;
constexpr float kC = 0.044715f;

// The normal distribution: with a = |x|, phi its density and M(a) = Phi(-a) / phi(a) (Mills' ratio),
//   Phi(x) = s + (1 - 2 s) phi M,   Phi(x) + x phi(x) = s + (1 - 2 s) phi (M - a),   s = [x > 0],
// which keeps the lower tail's relative accuracy (1 + erf would cancel there). M is a degree-8
// polynomial without constant term in t = 1 / (1 + 0.33 a / sqrt(2)) (the form of Abramowitz and
// Stegun 7.1.26), its coefficients fitted here for the least largest relative error on 0 <= a <=
// 13.5: 1.3e-7, and 9e-8 of the result on average with the f32 arithmetic. (Degree 7 would save 1 %
// of act_backward_mx's time, but its 8e-7 moves 8-bit codes off the exact value's rounding, a dozen
// in a million.) Beyond 13.5, phi is below the smallest normal float. act_backward_mx with GELU,
// 4096 x 16384, took 192 us with CUDA's erfcf when it took 120 us with a polynomial for erfcx, and
// 91 us with that, 1 - q and a choice for each element where it takes 89 us in this form.
struct Normal2 {
    f32x2 na, t, p, phi;  // -a; M = p t
    f32x2 s, sign;        // s and 1 - 2 s
};
__device__ __forceinline__ Normal2 normal2(f32x2 x) {
    const float2 v = unpack2(x);
    Normal2 n;
    n.na = pack2f(-fabsf(v.x), -fabsf(v.y));
    n.t = rcp2(fma2(n.na, splat(-0.23334524f), splat(1.0f)));
    n.phi = exp2_2(fma2(mul2(x, x), splat(-0.5f * kLog2e), splat(-1.3257481f)));  // log2 phi(0)
    f32x2 p = splat(-0.17008568f);
    p = fma2(p, n.t, splat(0.57873446f));
    p = fma2(p, n.t, splat(-0.4434476f));
    p = fma2(p, n.t, splat(0.51513124f));
    p = fma2(p, n.t, splat(0.05745955f));
    p = fma2(p, n.t, splat(0.2527419f));
    p = fma2(p, n.t, splat(0.22920893f));
    n.p = fma2(p, n.t, splat(0.23357132f));
    float a, b;
    asm("set.gt.f32.f32 %0, %1, 0f00000000;" : "=f"(a) : "f"(v.x));
    asm("set.gt.f32.f32 %0, %1, 0f00000000;" : "=f"(b) : "f"(v.y));
    n.s = pack2f(a, b);
    n.sign = fma2(n.s, splat(-2.0f), splat(1.0f));
    return n;
}
__device__ __forceinline__ f32x2 gelu2(f32x2 x, const Normal2& n) {
    return mul2(x, fma2(mul2(mul2(n.p, n.t), n.phi), n.sign, n.s));
}

// f(x) of a pair.
template <uint32_t KIND>
__device__ __forceinline__ f32x2 act2(f32x2 x) {
    if constexpr (KIND == PTXSTD_ACT_RELU) {
        const float2 v = unpack2(x);
        return pack2f(v.x < 0.0f ? 0.0f : v.x, v.y < 0.0f ? 0.0f : v.y);  // a NaN stays NaN
    } else if constexpr (KIND == PTXSTD_ACT_SILU) {
        return mul2(x, logistic2(mul2(x, splat(-kLog2e))));
    } else if constexpr (KIND == PTXSTD_ACT_GELU) {
        return gelu2(x, normal2(x));
    } else if constexpr (KIND == PTXSTD_ACT_GELU_TANH) {
        const f32x2 u = mul2(x, fma2(mul2(x, x), splat(-kG * kC * kLog2e), splat(-kG * kLog2e)));
        return mul2(x, logistic2(u));
    } else {
        return x;
    }
}
// f(x) and f'(x) of a pair (they share the exponential).
template <uint32_t KIND>
__device__ __forceinline__ void act_grad2(f32x2 x, f32x2& f, f32x2& df) {
    if constexpr (KIND == PTXSTD_ACT_RELU) {
        const float2 v = unpack2(x);
        f = act2<KIND>(x);
        df = pack2f(v.x > 0.0f ? 1.0f : 0.0f, v.y > 0.0f ? 1.0f : 0.0f);
    } else if constexpr (KIND == PTXSTD_ACT_SILU) {
        // t + x t (1 - t)
        const f32x2 t = logistic2(mul2(x, splat(-kLog2e)));
        f = mul2(x, t);
        df = fma2(f, fma2(t, splat(-1.0f), splat(1.0f)), t);
    } else if constexpr (KIND == PTXSTD_ACT_GELU) {
        const Normal2 n = normal2(x);
        f = gelu2(x, n);
        df = fma2(mul2(n.phi, fma2(n.p, n.t, n.na)), n.sign, n.s);
    } else if constexpr (KIND == PTXSTD_ACT_GELU_TANH) {
        // the square is capped: t is 0 or 1 long before, and 0 * inf stays out
        const float2 v = unpack2(mul2(x, x));
        const f32x2 x2 = pack2f(fminf(v.x, 1.0e6f), fminf(v.y, 1.0e6f));
        const f32x2 t =
            logistic2(mul2(x, fma2(x2, splat(-kG * kC * kLog2e), splat(-kG * kLog2e))));
        f = mul2(x, t);
        const f32x2 du = fma2(x2, splat(3.0f * kG * kC), splat(kG));
        df = fma2(mul2(f, fma2(t, splat(-1.0f), splat(1.0f))), du, t);
    } else {
        f = x;
        df = splat(1.0f);
    }
}
// Calls body(Act<KIND>{}) for the activation `kind`: the choice is made once, outside the loops
// over elements.
template <uint32_t KIND>
struct Act {
    static constexpr uint32_t value = KIND;
};
template <class Body>
__device__ __forceinline__ void with_act(uint32_t kind, Body&& body) {
    switch (kind) {
    case PTXSTD_ACT_RELU: body(Act<PTXSTD_ACT_RELU>{}); break;
    case PTXSTD_ACT_SILU: body(Act<PTXSTD_ACT_SILU>{}); break;
    case PTXSTD_ACT_GELU: body(Act<PTXSTD_ACT_GELU>{}); break;
    case PTXSTD_ACT_GELU_TANH: body(Act<PTXSTD_ACT_GELU_TANH>{}); break;
    default: body(Act<PTXSTD_ACT_NONE>{});
    }
}

}  // namespace mx
}  // namespace ptxstd
