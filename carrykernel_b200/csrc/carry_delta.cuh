// The gated delta rule over whole sequences: what its kernels share.
//
//   alpha = exp(-exp(A_log) softplus(a + dt_bias)),  beta = sigmoid(b)
//   S <- alpha S;  u = beta (v - S k);  S <- S + u k^T;  o = S (scale q)          S [V, K], for every value head
#pragma once

#include "carry_hybrid.cuh"

namespace carry {

constexpr float kL2Eps = 1e-6f;

// What makes a key or query with this sum of squares one of length `by`.  Of one whose squares pass fp32 nothing is known: NaN, and not the 0 that a
// division by infinity gives.
__device__ __forceinline__ float norm_factor(float squares, float by) { return squares < INFINITY ? __fdiv_rn(by, sqrtf(squares + kL2Eps)) : __builtin_nanf(""); }

// A request's rows, brought into bounds.
struct PrefillRequest {
  int first, count;
};
__device__ __forceinline__ PrefillRequest prefill_request(const CarryGdnPrefillArgs& a, int b, int* status) {
  PrefillRequest r;
  if (a.query_start) {
    const int from = a.query_start[b], to = a.query_start[b + 1];
    r.first = min(max(from, 0), a.N);
    r.count = min(max(min(to, a.N), r.first) - r.first, a.max_query);   // no difference that 32 bits do not hold
    if (status && (r.first != from || r.first + r.count != to)) atomicOr(status, CARRY_GDN_STATUS_BAD_RANGE);
  } else {
    r.first = b * a.max_query;
    r.count = a.max_query;
  }
  return r;
}

// What a token's gates are made of, and log alpha and beta.  The softplus of a large negative number is that number's exponential, of which
// log(1 + x) would leave few bits; steps of 0.001 are where models begin.
struct GateInputs {
  float a, b, A_log, dt_bias;
};
__device__ __forceinline__ GateInputs gate_inputs(const CarryGdnPrefillArgs& a, long long row, int hv) {
  return {load_as_float(a.a, row * a.stride_a_tok + hv, a.ab_dtype), load_as_float(a.b, row * a.stride_b_tok + hv, a.ab_dtype),
          load_as_float(a.A_log, hv, a.A_log_dtype), load_as_float(a.dt_bias, hv, a.dt_bias_dtype)};
}
__device__ __forceinline__ void gates_of(const GateInputs& g, float& log_alpha, float& beta) {
  const float x = g.a + g.dt_bias;
  const float softplus = x <= kSoftplusThreshold ? log1pf(expf(x)) : x;
  log_alpha = -expf(g.A_log) * softplus;
  beta = __fdiv_rn(1.0f, 1.0f + expf(-g.b));
}
__device__ __forceinline__ void prefill_gates(const CarryGdnPrefillArgs& a, long long row, int hv, float& log_alpha, float& beta) {
  gates_of(gate_inputs(a, row, hv), log_alpha, beta);
}

int64_t delta_workspace(const CarryGdnPrefillArgs& a);
int launch_delta(const CarryGdnPrefillArgs& a, cudaStream_t stream);
bool delta_rows_alone(const CarryGdnPrefillArgs& a);
int launch_delta_recurrent(const CarryGdnPrefillArgs& a, cudaStream_t stream);

}  // namespace carry
