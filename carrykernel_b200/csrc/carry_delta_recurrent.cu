// The gated delta rule token by token, in fp32: few tokens of a request, from a floating-point state.
//
// Rows of the state do not depend on one another, so a CTA has some of a head's rows, in registers: eight lanes to a row, each with
// every eighth run of four numbers, so that the state comes and goes in whole lines.  What a token costs is a chain: the products of
// the state with key and query (formed together from the state as it was, for o = alpha S q + u (k . q)), their sum over eight
// lanes, and the row that is added.  Norms are formed for a block of tokens at a time, and the next block's numbers are asked for ahead of it.
//
// What bounds it, for 32 heads of 128 in bf16: the state's way in and out for one token (64 requests 46 us and more, 128 requests 83 us, which is the
// rate of a plain copy), a few tokens' chains beside it (32 requests of 5 tokens 35 to 38 us, of which the state is 21), and the chain for
// many: 0.35 us a token where every row has lanes of its own.  Two rows to eight lanes, and more warps, are slower for few tokens (56 us and
// 46): what a CTA does for a token once comes twice as often.
#include <cuda_pipeline_primitives.h>

#include <type_traits>

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

// Tokens come into shared memory a block at a time, a block ahead.
constexpr int kTokens = 16;
template <int DTYPE, int K, int ROWS>
struct Block {
  using Number = typename std::conditional<DTYPE == CARRY_F32, float, uint16_t>::type;
  static constexpr int kRows = kThreads / kLanes * ROWS;      // of the state to a CTA
  alignas(16) Number q[kTokens][K], k[kTokens][K], v[kTokens][kRows];
};
struct alignas(16) Factors {
  float alpha, beta, query, key;        // query and key: what their numbers are multiplied by
  float key_query, pad[3];              // product of the two as they are in memory, times both
};

// ROWS of the state to a group of eight lanes
template <int DTYPE, int K, int ROWS>
__global__ void __launch_bounds__(kThreads, ROWS == 4 || DTYPE == CARRY_F32 ? 4 : 6) recurrent_kernel(const __grid_constant__ CarryGdnPrefillArgs a, bool aligned) {
  using Tokens = Block<DTYPE, K, ROWS>;
  using Number = typename Tokens::Number;
  constexpr int kFours = K / 32, kRows = Tokens::kRows;
  __shared__ Tokens block[2];
  __shared__ Factors factors[kTokens];
  depend_release();
  depend_wait();
  const int b = blockIdx.z, hv = blockIdx.y, tid = threadIdx.x, lane = tid % kLanes, group = tid / kLanes, h = hv / (a.HV / a.H);
  const int row0 = blockIdx.x * kRows + group * ROWS;
  const long long head = (long long)hv * a.V * K;
  // the state first: nothing has to be known for it
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
  const PrefillRequest r = prefill_request(a, b, tid == 0 && hv == 0 && blockIdx.x == 0 ? a.status : nullptr);

  auto fetch = [&](int t0) {
    Tokens& to = block[t0 / kTokens & 1];
    const int n = min(r.count - t0, kTokens);
    const Number* rows = reinterpret_cast<const Number*>(a.mixed_qkv) + (long long)(r.first + t0) * a.stride_mixed_tok;
    auto bring = [&](Number* dst, int stride, const Number* src, int width) {
      if (aligned) {
        constexpr int kEach = 16 / sizeof(Number);
        for (int i = tid; i < n * width / kEach; i += kThreads) {
          const int t = i / (width / kEach), at = i % (width / kEach) * kEach;
          __pipeline_memcpy_async(dst + t * stride + at, src + t * a.stride_mixed_tok + at, 16);
        }
      } else {
        for (int i = tid; i < n * width; i += kThreads) dst[i / width * stride + i % width] = src[i / width * a.stride_mixed_tok + i % width];
      }
    };
    bring(to.q[0], K, rows + h * K, K);
    bring(to.k[0], K, rows + (a.H + h) * K, K);
    bring(to.v[0], kRows, rows + 2LL * a.H * K + (long long)hv * a.V + blockIdx.x * kRows, kRows);
  };
  float log_alpha = 0.0f, beta_of = 0.0f;         // of token tid of the block to come
  auto gates = [&](int t0) {
    if (tid < kTokens && t0 + tid < r.count) prefill_gates(a, r.first + t0 + tid, hv, log_alpha, beta_of);
  };
  if (r.count > 0) fetch(0);
  __pipeline_commit();
  if (r.count > kTokens) fetch(kTokens);
  __pipeline_commit();
  gates(0);

  for (int t0 = 0; t0 < r.count; t0 += kTokens) {
    const Tokens& now = block[t0 / kTokens & 1];
    const int n = min(r.count - t0, kTokens);
    __pipeline_wait_prior(1);
    if (tid < kTokens) {
      factors[tid].alpha = expf(log_alpha);
      factors[tid].beta = beta_of;
    }
    __syncthreads();
    // norms, and the product of query and key: a token to eight lanes
    for (int t = group; t < kTokens; t += kThreads / kLanes) {
      float2 qq = make_float2(0.0f, 0.0f), kk = qq, kq = qq;
#pragma unroll
      for (int f = 0; f < kFours; ++f) {
        float2 q[2], k[2];
        unpack_four<DTYPE>(load_four<DTYPE>(now.q[t], f * 32 + lane * 4, true), q);
        unpack_four<DTYPE>(load_four<DTYPE>(now.k[t], f * 32 + lane * 4, true), k);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qq = fma2(q[e], q[e], qq);
          kk = fma2(k[e], k[e], kk);
          kq = fma2(k[e], q[e], kq);
        }
      }
      const float query = a.use_qk_l2norm ? norm_factor(over_lanes(qq.x + qq.y), a.scale) : a.scale;
      const float key = a.use_qk_l2norm ? norm_factor(over_lanes(kk.x + kk.y), 1.0f) : 1.0f;
      const float product = over_lanes(kq.x + kq.y) * query * key;
      if (lane == 0) {
        factors[t].query = query;
        factors[t].key = key;
        factors[t].key_query = product;
      }
    }
    __syncthreads();
    gates(t0 + kTokens);
    long long at = (long long)(r.first + t0) * a.stride_out_tok + (long long)hv * a.V + row0;
    Four<DTYPE> next_q[kFours], next_k[kFours];
    auto ahead = [&](int t) {
#pragma unroll
      for (int f = 0; f < kFours; ++f) {
        next_q[f] = load_four<DTYPE>(now.q[t], f * 32 + lane * 4, true);
        next_k[f] = load_four<DTYPE>(now.k[t], f * 32 + lane * 4, true);
      }
    };
    ahead(0);
    for (int t = 0; t < n; ++t, at += a.stride_out_tok) {
      const float4 w = *reinterpret_cast<const float4*>(&factors[t]);
      const float alpha = w.x, beta = w.y, by_q = w.z, by_k = w.w, k_dot_q = factors[t].key_query;
      float2 q[kFours][2], k[kFours][2];
#pragma unroll
      for (int f = 0; f < kFours; ++f) {
        unpack_four<DTYPE>(next_q[f], q[f]);
        unpack_four<DTYPE>(next_k[f], k[f]);
      }
      ahead(min(t + 1, kTokens - 1));
      float sk[ROWS], sq[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        float2 x[2] = {}, y[2] = {};
#pragma unroll
        for (int f = 0; f < kFours; ++f)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            x[e] = fma2(S[i][f][e], k[f][e], x[e]);
            y[e] = fma2(S[i][f][e], q[f][e], y[e]);
          }
        const float2 z = add2(x[0], x[1]), o = add2(y[0], y[1]);
        sk[i] = z.x + z.y;
        sq[i] = o.x + o.y;
      }
      float u[ROWS];
      if constexpr (ROWS == 4) {
        // eight sums over eight lanes: lane i is left with row i's product with the key, lane 4 + i with the one with the query
        const bool second = lane & 4, odd_pair = lane & 2, odd = lane & 1;
        float four[4], two[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) four[i] = (second ? sq[i] : sk[i]) + __shfl_xor_sync(~0u, second ? sk[i] : sq[i], 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) two[i] = (odd_pair ? four[2 + i] : four[i]) + __shfl_xor_sync(~0u, odd_pair ? four[i] : four[2 + i], 2);
        const float one = (odd ? two[1] : two[0]) + __shfl_xor_sync(~0u, odd ? two[0] : two[1], 1);
        const float v = load_as_float(now.v[t], group * ROWS + lane % 4, DTYPE);
        const float added = beta * fmaf(-alpha * by_k, one, v);                   // of use in lanes 0 .. 3
        const float given = __shfl_xor_sync(~0u, added, 4);
        if (second) store_from_float(a.out, at + lane % 4, a.out_dtype, fmaf(given, k_dot_q, alpha * by_q * one));
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __shfl_sync(~0u, added, i, kLanes) * by_k;
      } else {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const float added = beta * fmaf(-alpha * by_k, over_lanes(sk[i]), load_as_float(now.v[t], group * ROWS + i, DTYPE));
          const float out = fmaf(added, k_dot_q, alpha * by_q * over_lanes(sq[i]));
          if (lane == i) store_from_float(a.out, at + i, a.out_dtype, out);
          u[i] = added * by_k;
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int f = 0; f < kFours; ++f)
#pragma unroll
          for (int e = 0; e < 2; ++e) S[i][f][e] = fma2(make_float2(u[i], u[i]), k[f][e], mul2(make_float2(alpha, alpha), S[i][f][e]));
    }
    __syncthreads();
    if (t0 + 2 * kTokens < r.count) fetch(t0 + 2 * kTokens);
    __pipeline_commit();
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
  const bool aligned = reinterpret_cast<uintptr_t>(a.mixed_qkv) % 16 == 0 && a.stride_mixed_tok * kSize % 16 == 0;
  const dim3 grid((unsigned)(a.V / (kThreads / kLanes * ROWS)), (unsigned)a.HV, (unsigned)a.B);
  return launch_dependent(recurrent_kernel<DTYPE, K, ROWS>, grid, kThreads, 0, stream, a, aligned);
}

template <int DTYPE, int K>
int launch_heads(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  return delta_rows_alone(a) ? launch_rows<DTYPE, K, 1>(a, stream) : launch_rows<DTYPE, K, 4>(a, stream);
}

template <int DTYPE>
int launch_width(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  return a.K == 64 ? launch_heads<DTYPE, 64>(a, stream) : launch_heads<DTYPE, 128>(a, stream);
}

}  // namespace

// A row of a state to eight lanes, while that fills the processors with no more than four warps to a scheduler; four rows otherwise.  40 tokens of
// 1, 2, 4 and 8 requests with 32 heads of 128: 19.7, 21.4, 33.7 and 62 us with a row, 19.9, 29.7, 35.5 and 46 with four.
bool delta_rows_alone(const CarryGdnPrefillArgs& a) { return (int64_t)a.B * a.HV * a.V / 16 <= 4LL * sm_count(); }

int launch_delta_recurrent(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  return a.qkv_dtype == CARRY_F32 ? launch_width<CARRY_F32>(a, stream)
         : a.qkv_dtype == CARRY_BF16 ? launch_width<CARRY_BF16>(a, stream) : launch_width<CARRY_F16>(a, stream);
}

}  // namespace carry
