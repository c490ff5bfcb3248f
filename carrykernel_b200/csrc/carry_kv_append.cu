// New tokens' keys and values into the 8-bit cache: one CTA for each (request, block of tokens, head) that the
// call touches, the keys on its first half and the values on its second.
//
// A block's scale is the smallest power of two that brings its largest magnitude within e4m3's 448.  Powers of two
// cost a float format no precision (only the exponent shifts), and they make a later growth of the scale exact: the
// codes of the block's earlier tokens move by whole binades, so a block filled token by token ends with the codes of
// one filled at once, subnormals apart.
#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr int kThreads = 256, kHalf = kThreads / 2, kMaxBlock = 128;
constexpr uint32_t kNotFinite = 0x7f800000u;      // bits of |x| from here on: infinities and NaNs

// eight consecutive elements as floats
template <class T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
  alignas(16) T raw[8];
  if (vec) {
    constexpr int n = sizeof(raw) / 16;
#pragma unroll
    for (int i = 0; i < n; ++i) reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(raw[i]);
}

__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | hi << 16;
  }
  return make_uint2(w[0], w[1]);
}

template <class T>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ CarryGdnKvAppendArgs a, const bool vec) {
  __shared__ uint32_t token_top[2][kMaxBlock];    // bits of each new token's largest magnitude
  __shared__ uint32_t top[2][kHalf / 32];
  depend_release();
  depend_wait();
  const CarryGdnKvCache& c = a.cache;
  const int b = blockIdx.z, h = blockIdx.y;
  const KvRequest r = kv_request(c, a.rows, b, blockIdx.x == 0 && h == 0 && threadIdx.x == 0 ? a.status : nullptr);
  const int origin = r.length - r.count;          // position of the request's row 0
  const int from = max(origin, 0), to = min(r.length, origin + r.todo);
  const int blk = from / c.block + blockIdx.x;
  const int start = blk * c.block, t0 = max(start, from), t1 = min(start + c.block, to);
  if (t0 >= t1) return;
  const int page = kv_page(c, b, start / c.page, h == 0 && threadIdx.x == 0 ? a.status : nullptr);
  if (page == 0) return;

  const bool is_v = threadIdx.x >= kHalf;
  const int tid = threadIdx.x % kHalf, offset = start % c.page;
  const int per_token = c.D / 8, items = (t1 - t0) * per_token;   // 8 or 16 neighbouring lanes have one token
  const long long stride_tok = is_v ? a.stride_v_tok : a.stride_k_tok;
  const T* x = reinterpret_cast<const T*>(is_v ? a.v : a.k) + (r.first + (t0 - origin)) * stride_tok +
               h * (is_v ? a.stride_v_head : a.stride_k_head);
  uint8_t* codes = (is_v ? c.v_codes + page * c.stride_v_page : c.k_codes + page * c.stride_k_page) +
                   ((long long)h * c.page + offset) * c.D;
  float* scale = (is_v ? c.v_scale + page * c.stride_vs_page : c.k_scale + page * c.stride_ks_page) +
                 h * (c.page / c.block) + offset / c.block;

  for (int base = 0; base < items; base += kHalf) {
    const int i = base + tid;
    uint32_t t = 0;
    if (i < items) {
      float e[8];
      load8(x + (i / per_token) * stride_tok + i % per_token * 8, vec, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) t = max(t, __float_as_uint(e[j]) & 0x7fffffffu);
    }
    for (int s = per_token / 2; s > 0; s /= 2) t = max(t, __shfl_xor_sync(~0u, t, s));
    if (i < items && i % per_token == 0) token_top[is_v][i / per_token] = t;
  }
  __syncthreads();
  uint32_t t = 0;
  if (tid < t1 - t0 && token_top[!is_v][tid] < kNotFinite && token_top[is_v][tid] < kNotFinite) t = token_top[is_v][tid];
  t = __reduce_max_sync(~0u, t);
  if (tid % 32 == 0) top[is_v][tid / 32] = t;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kHalf / 32; ++i) t = max(t, top[is_v][i]);

  float now = power_of_two_scale(__uint_as_float(t));
  if (t0 > start) {
    const float old = *scale;
    if (old < now) {
      const float shift = __fdiv_rn(old, now);
      uint8_t* early = codes;
      for (int i = tid; i < (t0 - start) * per_token; i += kHalf) {
        const uint2 w = reinterpret_cast<const uint2*>(early)[i];
        float e[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t half = j < 2 ? w.x : w.y;
          const __half2 v(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(half >> (j % 2 * 16)), __NV_E4M3));
          e[2 * j] = __low2float(v);
          e[2 * j + 1] = __high2float(v);
        }
        reinterpret_cast<uint2*>(early)[i] = codes8(e, shift);
      }
    } else {
      now = old;
    }
  }
  const float inv = __fdiv_rn(1.0f, now);
  uint8_t* to_codes = codes + (long long)(t0 - start) * c.D;
  for (int i = tid; i < items; i += kHalf) {
    const int token = i / per_token;
    float e[8];
    load8(x + token * stride_tok + i % per_token * 8, vec, e);
    uint2 w = codes8(e, inv);
    if (token_top[0][token] >= kNotFinite || token_top[1][token] >= kNotFinite)
      w = is_v ? make_uint2(0, 0) : make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    reinterpret_cast<uint2*>(to_codes)[i] = w;
  }
  __syncthreads();                                // every thread has read the old scale
  if (tid == 0) *scale = now;
}

}  // namespace

int launch_kv_append(const CarryGdnKvAppendArgs& a, cudaStream_t stream) {
  const CarryGdnKvCache& c = a.cache;
  const int blocks = (a.rows.max_query + 2 * c.block - 2) / c.block;   // that many blocks can a request's rows touch
  const int size = a.dtype == CARRY_F32 ? 4 : 2;
  bool vec = true;
  for (long long v : {(long long)reinterpret_cast<uintptr_t>(a.k), (long long)reinterpret_cast<uintptr_t>(a.v),
                      (long long)a.stride_k_tok * size, (long long)a.stride_k_head * size,
                      (long long)a.stride_v_tok * size, (long long)a.stride_v_head * size})
    vec = vec && v % 16 == 0;
  const dim3 grid(blocks, c.HKV, a.rows.B);
  if (a.dtype == CARRY_F32) return launch_dependent(kv_append_kernel<float>, grid, kThreads, 0, stream, a, vec);
  if (a.dtype == CARRY_BF16) return launch_dependent(kv_append_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, a, vec);
  return launch_dependent(kv_append_kernel<__half>, grid, kThreads, 0, stream, a, vec);
}

}  // namespace carry
