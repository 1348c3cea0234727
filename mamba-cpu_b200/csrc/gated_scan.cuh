// gated_scan.cuh -- gated linear recurrence: argument block, launchers and the gate arithmetic.
//
//   a_t = exp(A s_r),  m_t = sqrt(1 - a_t^2),  h_t = a_t h_{t-1} + m_t s_i u_t
//   with s_r = sigmoid(decay_gate), s_i = sigmoid(input_gate), A <= 0 per channel.
#pragma once

#include "common.cuh"

namespace mb200 {

constexpr int kGatedItems = 8;                      // consecutive steps a lane holds
constexpr int kGatedChunk = MB200_GATED_SCAN_CHUNK;  // steps a warp covers at once: 32 lanes x kGatedItems
static_assert(kGatedChunk == 32 * kGatedItems, "a warp's chunk");
constexpr int kGatedHeader = 4;
constexpr int kGatedMaxWarps = 32;  // warps that may share a row (CTA warps x CTAs of the cluster)

struct GatedScanArgs {
  const void *u, *r, *i;
  const float *A, *h0;
  const int32_t* ids;
  void* out;
  float* last;
  float* states;
  int64_t batch, dim, L;
  int64_t sub, sud, srb, srd, sib, sid, sqb;
  int64_t u_elements, r_elements, i_elements;  // from a tensor's first element to behind its last
  int chunks;  // room for a row's states, which begin kGatedHeader floats into `states`
  // The chunks of row (b, d) begin (phase + b phase_b + d phase_d) mod kGatedItems steps before its
  // first step: u's misalignment there, so that every lane's steps are aligned in memory. The forward
  // leaves the three in front of the states, and the backward goes by them: the u that it gets may be
  // a copy at another address.
  int phase, phase_b, phase_d;
  // backward
  const void* dout;
  const float* dlast;
  void *du, *dr, *di;
  float* part;  // (batch, dim) sums of dA
  float* dh0;
};

struct GatedStepArgs {
  const void* state;
  void* new_state;
  const void *u, *r, *i;
  const float* A;
  void* out;
  int64_t batch, dim;
  int64_t ss, sn, su, sr, si;  // row strides; out is dense
  int vec;
};

cudaError_t launch_gated_scan_fwd(const GatedScanArgs& a, int dtype, cudaStream_t stream);
cudaError_t launch_gated_scan_bwd(const GatedScanArgs& a, int dtype, float* dA, cudaStream_t stream);
cudaError_t launch_gated_step(const GatedStepArgs& a, int dtype, int state_dtype, cudaStream_t stream);

// 1 / sqrt(x) on the SFU, to about one unit in the last place.
__device__ __forceinline__ float rsqrt_f(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / (1 + e^-x): 0 and 1 at infinite gates, where e^-x is infinite or 0.
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  float2 t = mul2(x, two(-kLog2e));
  t = add2(make_float2(ex2(t.x), ex2(t.y)), two(1.f));
  return make_float2(rcp_f(t.x), rcp_f(t.y));
}

// a = e^-y and q = 1 - a^2 for y = -A s >= 0. Slow decays (a near 1) are what long memories are made
// of: there p = 1 - e^-y comes from a polynomial and keeps its relative accuracy, and so does
// q = p (2 - p) = p + p a, the square of the input's factor. The decay a = 1 - p is the float32 nearest to that:
// off by 2^-25 at most, so 1 - a, which sets how long a channel remembers, is off by 0.3% at p = 1e-5 and 3% at
// 1e-6, and below p = 2^-25 a is 1. The polynomial is the one of degree 5 nearest to (1 - e^-y) / y on [0, 1] in relative error (2^-23 with these coefficients).
//
// `rate` is -A. A channel with A >= -1 (SLOW: one branch for a whole row) never leaves the polynomial's
// range and needs no exponential from the SFU; others take e^-y where y > 1.
template <bool SLOW>
__device__ __forceinline__ void decay2(float2 rate, float2 s, float2& a, float2& q) {
  const float2 y = mul2(s, rate);
  float2 c = fma2(y, two(-0.0009071574313566089f), two(0.007823704741895199f));
  c = fma2(c, y, two(-0.04140659421682358f));
  c = fma2(c, y, two(0.16660521924495697f));
  c = fma2(c, y, two(-0.49999457597732544f));
  c = fma2(c, y, two(0.9999999403953552f));
  float2 p = mul2(c, y);
  if (SLOW) {
    a = fma2(p, two(-1.f), two(1.f));
  } else {
    const float2 t = mul2(y, two(-kLog2e));
    const float2 e = make_float2(ex2(t.x), ex2(t.y));
    a.x = y.x <= 1.f ? 1.f - p.x : e.x;
    a.y = y.y <= 1.f ? 1.f - p.y : e.y;
    p.x = y.x <= 1.f ? p.x : 1.f - e.x;
    p.y = y.y <= 1.f ? p.y : 1.f - e.y;
  }
  q = fma2(p, a, p);
}

// sqrt(q) sigmoid(x) = q / sqrt(q d^2) with d = 1 + e^-x: one special function instead of two. The
// small number added under the root makes 0 of q = 0 and is lost in any other q that counts; a gate
// below -44, where d^2 overflows and the sigmoid is below 1e-19, gives 0, as a shut one does.
__device__ __forceinline__ float2 gated_root2(float2 q, float2 x) {
  const float2 t = mul2(x, two(-kLog2e));
  const float2 d = add2(make_float2(ex2(t.x), ex2(t.y)), two(1.f));
  const float2 s = mul2(mul2(add2(q, two(1e-37f)), d), d);
  return mul2(q, make_float2(rsqrt_f(s.x), rsqrt_f(s.y)));
}

// A positive A has no real root: NaN, as the formula gives.
__device__ __forceinline__ float checked_decay(float A) { return A > 0.f ? __int_as_float(0x7fffffff) : A; }

}  // namespace mb200
