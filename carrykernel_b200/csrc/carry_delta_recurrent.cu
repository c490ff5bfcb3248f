// The gated delta rule token by token, in fp32: few tokens of a request, from a floating-point state.
//
// Rows of the state do not depend on one another, so a CTA has some of a head's rows, in registers: eight lanes to a row, each with
// every eighth run of four numbers, so that the state comes and goes in whole lines.  What a token costs is a chain: the products of
// the state with key and query (formed together from the state as it was, for o = alpha S q + u (k . q)), their sum over eight
// lanes, and the row that is added.  The next token's numbers are asked for ahead of it.
#include "carry_delta.cuh"

namespace carry {
namespace {

constexpr int kThreads = 128, kLanes = 8;

template <int DTYPE>
struct Four;
template <>
struct Four<CARRY_F32> {
  float4 u;
};
template <>
struct Four<CARRY_BF16> {
  uint2 u;
};
template <>
struct Four<CARRY_F16> {
  uint2 u;
};
template <int DTYPE>
__device__ __forceinline__ Four<DTYPE> load_four(const void* base, long long at, bool aligned) {
  Four<DTYPE> f;
  if constexpr (DTYPE == CARRY_F32) {
    const float* p = reinterpret_cast<const float*>(base) + at;
    f.u = aligned ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
    f.u = aligned ? *reinterpret_cast<const uint2*>(p) : make_uint2(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16);
  }
  return f;
}
template <int DTYPE>
__device__ __forceinline__ void unpack_four(const Four<DTYPE>& f, float2 (&x)[2]) {
  if constexpr (DTYPE == CARRY_F32) {
    x[0] = make_float2(f.u.x, f.u.y);
    x[1] = make_float2(f.u.z, f.u.w);
  } else {
    const uint32_t w[2] = {f.u.x, f.u.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (DTYPE == CARRY_BF16) x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      else x[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
  }
}
__device__ __forceinline__ float over_lanes(float x) {
#pragma unroll
  for (int d = kLanes / 2; d > 0; d /= 2) x += __shfl_xor_sync(~0u, x, d);
  return x;
}

// ROWS of the state to a group of eight lanes
template <int DTYPE, int K, int ROWS>
__global__ void __launch_bounds__(kThreads) recurrent_kernel(const __grid_constant__ CarryGdnPrefillArgs a, bool aligned) {
  constexpr int kFours = K / 32;
  depend_release();
  depend_wait();
  const int b = blockIdx.z, hv = blockIdx.y, lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, h = hv / (a.HV / a.H);
  const int row0 = blockIdx.x * (kThreads / kLanes * ROWS) + group * ROWS;
  const PrefillRequest r = prefill_request(a, b, threadIdx.x == 0 && hv == 0 && blockIdx.x == 0 ? a.status : nullptr);
  const long long head = (long long)hv * a.V * K;
  float2 S[ROWS][kFours][2];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int f = 0; f < kFours; ++f) {
      float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (a.initial_state) u = *reinterpret_cast<const float4*>(a.initial_state + b * a.stride_initial_req + head + (long long)(row0 + i) * K + f * 32 + lane * 4);
      S[i][f][0] = make_float2(u.x, u.y);
      S[i][f][1] = make_float2(u.z, u.w);
    }

  struct Token {
    Four<DTYPE> q[kFours], k[kFours];
    float v[ROWS];
  };
  auto fetch = [&](int t, Token& x) {
    const long long at = (long long)(r.first + t) * a.stride_mixed_tok;
#pragma unroll
    for (int f = 0; f < kFours; ++f) {
      x.q[f] = load_four<DTYPE>(a.mixed_qkv, at + h * K + f * 32 + lane * 4, aligned);
      x.k[f] = load_four<DTYPE>(a.mixed_qkv, at + (a.H + h) * K + f * 32 + lane * 4, aligned);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) x.v[i] = load_as_float(a.mixed_qkv, at + 2LL * a.H * K + (long long)hv * a.V + row0 + i, DTYPE);
  };
  Token next;
  float log_alpha = 0.0f, beta_of = 0.0f;         // of token (t / 32) * 32 + this lane of the warp
  if (r.count > 0) fetch(0, next);
  for (int t = 0; t < r.count; ++t) {
    const Token now = next;
    if (t % 32 == 0 && t + (int)threadIdx.x % 32 < r.count) {
      prefill_gates(a, r.first + t + threadIdx.x % 32, hv, log_alpha, beta_of);
      log_alpha = expf(log_alpha);
    }
    if (t + 1 < r.count) fetch(t + 1, next);
    const float alpha = __shfl_sync(~0u, log_alpha, t % 32), beta = __shfl_sync(~0u, beta_of, t % 32);
    float2 q[kFours][2], k[kFours][2];
    float2 qq = make_float2(0.0f, 0.0f), kk = qq, kq = qq;
#pragma unroll
    for (int f = 0; f < kFours; ++f) {
      unpack_four<DTYPE>(now.q[f], q[f]);
      unpack_four<DTYPE>(now.k[f], k[f]);
    }
    float by_q = a.scale, by_k = 1.0f;
    if (a.use_qk_l2norm) {
#pragma unroll
      for (int f = 0; f < kFours; ++f)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qq = fma2(q[f][e], q[f][e], qq);
          kk = fma2(k[f][e], k[f][e], kk);
        }
      by_q = __fdiv_rn(a.scale, sqrtf(over_lanes(qq.x + qq.y) + kL2Eps));
      by_k = __fdiv_rn(1.0f, sqrtf(over_lanes(kk.x + kk.y) + kL2Eps));
    }
#pragma unroll
    for (int f = 0; f < kFours; ++f)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        q[f][e] = mul2(q[f][e], make_float2(by_q, by_q));
        k[f][e] = mul2(k[f][e], make_float2(by_k, by_k));
        kq = fma2(k[f][e], q[f][e], kq);
      }
    const float k_dot_q = over_lanes(kq.x + kq.y);
    float out[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      float2 sk = make_float2(0.0f, 0.0f), sq = sk;
#pragma unroll
      for (int f = 0; f < kFours; ++f)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sk = fma2(S[i][f][e], k[f][e], sk);
          sq = fma2(S[i][f][e], q[f][e], sq);
        }
      const float u = beta * fmaf(-alpha, over_lanes(sk.x + sk.y), now.v[i]);
      out[i] = fmaf(u, k_dot_q, alpha * over_lanes(sq.x + sq.y));
#pragma unroll
      for (int f = 0; f < kFours; ++f)
#pragma unroll
        for (int e = 0; e < 2; ++e) S[i][f][e] = fma2(make_float2(u, u), k[f][e], mul2(make_float2(alpha, alpha), S[i][f][e]));
    }
    const long long at = (long long)(r.first + t) * a.stride_out_tok + (long long)hv * a.V + row0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (lane == i) store_from_float(a.out, at + i, a.out_dtype, out[i]);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int f = 0; f < kFours; ++f)
      *reinterpret_cast<float4*>(a.final_state + b * a.stride_final_req + head + (long long)(row0 + i) * K + f * 32 + lane * 4) =
          make_float4(S[i][f][0].x, S[i][f][0].y, S[i][f][1].x, S[i][f][1].y);
}

template <int DTYPE, int K, int ROWS>
int launch_rows(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  constexpr int kSize = DTYPE == CARRY_F32 ? 4 : 2;
  const bool aligned = reinterpret_cast<uintptr_t>(a.mixed_qkv) % (4 * kSize) == 0 && a.stride_mixed_tok % 4 == 0;
  const dim3 grid((unsigned)(a.V / (kThreads / kLanes * ROWS)), (unsigned)a.HV, (unsigned)a.B);
  return launch_dependent(recurrent_kernel<DTYPE, K, ROWS>, grid, kThreads, 0, stream, a, aligned);
}

template <int DTYPE, int K>
int launch_heads(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  // one row to a group of lanes while that does not fill the processors with four warps to a scheduler
  return (long long)a.B * a.HV * a.V / 16 <= 4LL * sm_count() ? launch_rows<DTYPE, K, 1>(a, stream) : launch_rows<DTYPE, K, 4>(a, stream);
}

template <int DTYPE>
int launch_width(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  return a.K == 64 ? launch_heads<DTYPE, 64>(a, stream) : launch_heads<DTYPE, 128>(a, stream);
}

}  // namespace

int launch_delta_recurrent(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  return a.qkv_dtype == CARRY_F32 ? launch_width<CARRY_F32>(a, stream)
         : a.qkv_dtype == CARRY_BF16 ? launch_width<CARRY_BF16>(a, stream) : launch_width<CARRY_F16>(a, stream);
}

}  // namespace carry
