// What surrounds the recurrent step in a hybrid model's decoder layer: the 8-bit key/value cache of its
// full-attention layers and the norm at every layer's entry.  Shared helpers and launchers.
#pragma once

#include "carry_gdn_common.cuh"

namespace carry {

constexpr float kF8Max = 448.0f;                  // largest e4m3 value
constexpr long long kMaxTokens = 1 << 30;         // of one request
constexpr int kMinScaleExp = -100, kMaxScaleExp = 119;

// The smallest power of two s with amax / s <= 448 = 1.75 * 2^8, read off amax's bits.
__device__ __forceinline__ float power_of_two_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, kMinScaleExp), kMaxScaleExp);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}

// Eight neighbouring numbers of a type: as they lie in memory, and as fp32.
template <int DTYPE>
struct Raw {
  uint4 w[DTYPE == CARRY_F32 ? 2 : 1];
};
struct Eight {
  float2 x[4];
};
template <int DTYPE>
__device__ __forceinline__ Raw<DTYPE> load_raw(const void* p, long long at) {
  Raw<DTYPE> r;
  if constexpr (DTYPE == CARRY_F32) {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + at);
    r.w[0] = q[0];
    r.w[1] = q[1];
  } else {
    r.w[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + at);
  }
  return r;
}
template <int DTYPE>
__device__ __forceinline__ Eight unpack(const Raw<DTYPE>& r) {
  Eight e;
  const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
  if constexpr (DTYPE == CARRY_F32) {
    const uint32_t v[4] = {r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e.x[i] = make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
      e.x[i + 2] = make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      e.x[i] = DTYPE == CARRY_BF16 ? make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u))
                                   : __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
  }
  return e;
}

// Shift that stands for a division by x, or -1.
inline int shift_of(int x) {
  for (int s = 0; s < 31; ++s)
    if (1 << s == x) return s;
  return -1;
}
__device__ __forceinline__ int divide(int x, int by, int shift) { return shift >= 0 ? x >> shift : x / by; }

// A request's share of a call, with everything that comes from device memory brought into bounds.
struct KvRequest {
  int first, count;   // its rows: first .. first + count - 1
  int todo;           // how many of them the call covers (count <= max_query where the caller kept to that)
  int length;         // tokens in the cache, the new ones among them
};
__device__ __forceinline__ KvRequest kv_request(const CarryGdnKvCache& c, const CarryGdnKvRows& r, int b, int* status) {
  KvRequest q;
  const long long cap = min((long long)c.max_pages * c.page, kMaxTokens);
  const int given = c.lengths[b];
  q.length = (int)min((long long)max(given, 0), cap);
  bool bad = given != q.length;
  if (r.query_start) {
    const int from = r.query_start[b], to = r.query_start[b + 1];
    q.first = min(max(from, 0), r.N);
    q.count = max(min(to, r.N) - q.first, 0);
    q.todo = min(q.count, r.max_query);
    bad = bad || q.first != from || q.first + q.todo != to;
  } else {
    q.first = b * r.max_query;
    q.count = q.todo = r.max_query;
  }
  if (bad && status) atomicOr(status, CARRY_GDN_STATUS_BAD_RANGE);
  return q;
}

// Page of a token, or 0 (the padding page) where the table's id is no page of the cache.
__device__ __forceinline__ int kv_page(const CarryGdnKvCache& c, int b, int index, int* status) {
  const int id = c.block_table[b * c.stride_table + index];
  if (id >= c.num_pages && status) atomicOr(status, CARRY_GDN_STATUS_BAD_RANGE);
  return id > 0 && id < c.num_pages ? id : 0;
}

int launch_kv_append(const CarryGdnKvAppendArgs& a, cudaStream_t stream);
int launch_kv_attention(const CarryGdnKvAttentionArgs& a, cudaStream_t stream);
int64_t kv_attention_workspace(const CarryGdnKvAttentionArgs& a);
int launch_norm(const CarryGdnNormArgs& a, cudaStream_t stream);

}  // namespace carry
