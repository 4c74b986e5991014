// What the kernels of the gated projections share: the activations, and the launch for a few rows.
#pragma once
#include "../../include/ksana_b200.h"
#include "common.cuh"

namespace ksb {
namespace gated {

// Both activations are v s with s = sigmoid(w(v)): SiLU w = v; GELU (tanh form) w = 2 sqrt(2 / pi) (v + 0.044715 v^3), since
// (1 + tanh z) / 2 = sigmoid(2 z).
constexpr float GELU_C = 1.5957691216057308f, GELU_K = 0.044715f, NEG_LOG2E = -1.4426950408889634f;
__device__ __forceinline__ float sigmoid_of(float w) {
  float s;  // subnormal results kept: v s is a normal number where s is not any more
  asm("rcp.approx.f32 %0, %1;" : "=f"(s) : "f"(1.f + fast_exp2(w * NEG_LOG2E)));
  return s;
}
__device__ __forceinline__ float act_sigmoid(float v, int act) { return sigmoid_of(act == KSB_ACT_SILU ? v : GELU_C * fmaf(GELU_K * v * v, v, v)); }
// act'(v) = s + v s (1 - s) w'(v); far out s (1 - s) is 0, and w' is kept finite
__device__ __forceinline__ float act_slope(float v, float s, int act) {
  const float c = fminf(fmaxf(v, -64.f), 64.f);
  const float w = act == KSB_ACT_SILU ? 1.f : GELU_C * fmaf(3.f * GELU_K * c, c, 1.f);
  return fmaf(c * s * (1.f - s), w, s);
}

// h = act(x Wg^T + bg) * (x Wu^T + bu) for up to MAX_ROWS rows of x.
constexpr int MAX_ROWS = 16;
struct RowsCall {
  const void* x;
  const void* w_gate;
  const void* w_up;
  const void* b_gate;  // or null
  const void* b_up;
  void* h;
  int64_t ldx, ldg, ldu;
  int M, F, K, act;
};
int run_rows(const RowsCall& call, int dtype, cudaStream_t st);

}  // namespace gated
}  // namespace ksb
