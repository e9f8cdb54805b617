// The gated activations with their partial derivatives, for the epilogues of gated_gemm.cu and gated_small.cu.
#pragma once

#include "common.cuh"

namespace fmoe {

namespace {

__device__ __forceinline__ uint32_t pack_bf16(float low, float high) {
  const __nv_bfloat162 pair = __floats2bfloat162_rn(low, high);
  return *reinterpret_cast<const uint32_t*>(&pair);
}

// The derivatives that a forward pass keeps lie in blocks of 32 rows x 32 channels, each as 2 sides (by gate, by up) x 8 groups of four
// channels x 32 rows of 16 bytes: the lane of an epilogue warp that holds a row then loads and stores next to its neighbours.  (Read as
// rows, 16 bytes of 32 rows at a time, the epilogue behind 256 rows of dy W2 took 18 us longer.)  First float4 of the block of row0 and channel0.
__host__ __device__ __forceinline__ int64_t derivative_block(int64_t row0, int channel0, int channels) {
  return ((row0 >> 5) * ((channels + 31) >> 5) + (channel0 >> 5)) * 512;
}

// h and its partial derivatives (common: gate * act'(gate) forms; NaN stays NaN through the limits).
template <typename Tag>
__device__ __forceinline__ void gated_with_derivatives(Tag, float gate, float up, float limit, float* h, float* by_gate, float* by_up) {
  if constexpr (Tag::value == FMOE_ACT_GELU) {
    // Phi(-a) = e^(-a^2/2) Q(a) for a >= 0, with Q(a) = erfcx(a / sqrt 2) / 2 fitted here (least squares, reweighted towards the largest relative error) by a polynomial in
    // t = 1 / (1 + 0.36 a): within 1e-6 of its value on [0, 14.5], behind which e^(-a^2/2) is 0 in 32 bits.  The left tail keeps its relative precision, which
    // 0.5 (1 + erf) loses, and the one exponential serves the density too (forward and backward of 1333 rows of 2048 x 1024: 97 us with normcdff, 75 like this).
    const float a = fabsf(gate);
    const float e = __expf(-0.5f * a * a);
    const float t = __fdividef(1.0f, fmaf(0.36f, a, 1.0f));
    float q = fmaf(0.046782233718879906f, t, -0.17882609622498481f);
    q = fmaf(q, t, 0.1796773446277012f);
    q = fmaf(q, t, 0.027426644660340928f);
    q = fmaf(q, t, 0.13940009972259584f);
    q = fmaf(q, t, 0.14183037149665473f);
    q = fmaf(q, t, 0.14370896987904766f);
    const float tail = e * q * t;
    const float cdf = gate < 0.0f ? tail : 1.0f - tail;
    const float density = 0.39894228040143267794f * e;
    *h = gate * cdf * up;
    *by_gate = up * (cdf + gate * density);
    *by_up = gate * cdf;
  } else {
    constexpr bool kOai = Tag::value == FMOE_ACT_SWIGLUOAI;
    const float bound = kOai ? 7.0f : (limit > 0.0f ? limit : __int_as_float(0x7f800000));
    constexpr float kAlpha = kOai ? 1.702f : 1.0f;
    const bool gate_cut = gate > bound;
    const bool up_cut = fabsf(up) > bound;
    const float g = gate_cut ? bound : gate;
    const float u = (up_cut ? copysignf(bound, up) : up) + (kOai ? 1.0f : 0.0f);
    const float s = __fdividef(1.0f, 1.0f + __expf(-kAlpha * g));  // e^-g = inf divides to 0
    const float gs = g * s;
    *h = gs * u;
    *by_gate = gate_cut ? 0.0f : u * s * (1.0f + kAlpha * g * (1.0f - s));
    *by_up = up_cut ? 0.0f : gs;
  }
}

}  // namespace

}  // namespace fmoe
