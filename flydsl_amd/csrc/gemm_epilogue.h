// The fused epilogue: out = round(act(v + bias[n]) + residual[m][n]), v the product with its scales
// applied, everything in fp32 and one rounding at the end.
//
// Activations (x the value behind the bias), each from the hardware's exp2 and reciprocal (1 ulp):
//   relu       x < 0 ? 0 : x (a NaN stays)
//   silu       x s(x), s(x) = 1 / (1 + 2^(-x log2 e))
//   gelu_tanh  0.5 x (1 + tanh(u)), u = sqrt(2/pi) (x + 0.044715 x^3), as x s(2u): no cancellation for
//              negative x, and x^2 past the largest float still gives x or 0
//   gelu       0.5 x erfc(-x / sqrt 2).  For z >= 0 erfc(z) / 2 = t P(t) exp(-z^2) with t = 1 / (1 + 0.46 z):
//              erfcx(z) / t is smooth over t in (0, 1], and P its polynomial of degree 7, fitted in the relative error
//              (7e-7; degree 8 reaches 1.3e-7 for one more instruction a value, behind which exp2's argument and the
//              reciprocal leave 1e-6 all the same).  With h = erfc(|x| / sqrt 2) / 2, x < 0 takes x h and x >= 0
//              x (1 - h), so neither side cancels.  In fp32 within 2.2e-6 of the value for |x| < 6 and 9e-6 to
//              |x| = 13 (the exponent's rounding), against 2.4e-4, half a step of an fp16 output.  From x = -13.05 the
//              value is below the smallest normal number, and from -13.2 exp2 gives 0 for it (5e-39 off at most).
// Which activation is a wave-uniform branch on a kernel argument, around all of a tile's values (or half of
// them): five kernels in its place would be five times the library.  Branching per four values inside the
// unrolled code cost more than most activations: the path taken hopped through 60 KB of instructions.
#pragma once
#include "gemm_common.h"

namespace flygemm {

enum Act : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// x / (1 + exp(-y))
__device__ __forceinline__ float times_sigmoid(float x, float y) {
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y * -1.4426950408889634f));
}

__device__ __forceinline__ float gelu_erf(float x) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.32526913f, __builtin_fabsf(x), 1.f));
  float p = 0.03385719f;
  p = __builtin_fmaf(p, t, -0.11331469f);
  p = __builtin_fmaf(p, t, 0.084595546f);
  p = __builtin_fmaf(p, t, 0.026305294f);
  p = __builtin_fmaf(p, t, 0.093423896f);
  p = __builtin_fmaf(p, t, 0.115590945f);
  p = __builtin_fmaf(p, t, 0.12977864f);
  p = __builtin_fmaf(p, t, 0.12976353f);
  const float h = t * p * __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
  return x * (x < 0.f ? h : 1.f - h);
}

// ACT_SILU and ACT_GELU_TANH are one formula with y = x (c1 + c3 x^2)
enum ActCode : int { CODE_NONE = 0, CODE_RELU = 1, CODE_GELU = 2, CODE_SIGMOID = 3 };

template <int CODE>
__device__ __forceinline__ void activate4(float (&v)[4], bool silu) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float x = v[q];
    if constexpr (CODE == CODE_RELU) v[q] = x < 0.f ? 0.f : x;
    if constexpr (CODE == CODE_GELU) v[q] = gelu_erf(x);
    if constexpr (CODE == CODE_SIGMOID) {
      // silu: c3 = 0 with x^2 = 0 (0 * inf would be NaN)
      const float c1 = silu ? 1.f : 1.5957691216057308f, c3 = silu ? 0.f : 0.071354816272600244f;
      v[q] = times_sigmoid(x, x * __builtin_fmaf(c3, silu ? 0.f : x * x, c1));
    }
  }
}

// calls f with the code of activation act as a compile-time constant
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
  if (act == ACT_NONE) f(std::integral_constant<int, CODE_NONE>{});
  else if (act == ACT_RELU) f(std::integral_constant<int, CODE_RELU>{});
  else if (act == ACT_GELU) f(std::integral_constant<int, CODE_GELU>{});
  else f(std::integral_constant<int, CODE_SIGMOID>{});
}

// The epilogue's kernel arguments, read where the epilogue begins: held in scalar registers from the kernel's
// start, they push the main loop's own out of them (its loop got 11 instructions longer).
struct FusedArgs {
  const void* bias;
  const void* res;
  int bias_f32, act;
};
__device__ __forceinline__ FusedArgs late_args() {
  typedef const __attribute__((address_space(4))) GemmArgs* ArgPtr;
  ArgPtr k = (ArgPtr)__builtin_amdgcn_kernarg_segment_ptr();   // GemmArgs is the only argument
  asm volatile("" : "+s"(k));
  return FusedArgs{k->bias, k->res, k->bias_f32, k->act};
}

// Four consecutive biases from column col, as fp32 (0 without a bias)
template <bool BF16>
__device__ __forceinline__ f32x4 load_bias4(const FusedArgs& p, int col) {
  typedef typename OutT<BF16>::type OT4 __attribute__((ext_vector_type(4)));
  if (!p.bias) return f32x4{0.f, 0.f, 0.f, 0.f};
  if (p.bias_f32) return *(const f32x4*)((const float*)p.bias + col);
  const OT4 b = *(const OT4*)((const typename OutT<BF16>::type*)p.bias + col);
  return f32x4{(float)b.x, (float)b.y, (float)b.z, (float)b.w};
}

// Four residual values held in two dwords
template <bool BF16>
__device__ __forceinline__ f32x4 widen4(const i32x2& r) {
  typedef typename OutT<BF16>::type OT4 __attribute__((ext_vector_type(4)));
  const OT4 b = __builtin_bit_cast(OT4, r);
  return f32x4{(float)b.x, (float)b.y, (float)b.z, (float)b.w};
}

// v -> act(v + bias) + residual
template <int CODE>
__device__ __forceinline__ void finish4(float (&v)[4], const f32x4& bias, const f32x4& res, bool silu) {
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] += bias[q];
  activate4<CODE>(v, silu);
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] += res[q];
}

}  // namespace flygemm
