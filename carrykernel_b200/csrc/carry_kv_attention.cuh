// What the kernels of the key/value attention share: parameters, pages, rows to memory.
#pragma once

#include <cuda_pipeline_primitives.h>

#include "carry_hybrid.cuh"

namespace carry {

constexpr int kGranule = 16;                      // tokens: no page and no block of a scale begins or ends inside
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoTokens = -1.0f;                // in a key scale's place: a padding page, or past the end

struct AttnParams {
  CarryGdnKvAttentionArgs a;
  int group, group_shift;         // query heads per key/value head, and its logarithm or -1
  int page_granules, page_shift;  // granules in a page, and its logarithm or -1
  int block_granules, block_shift;
  int rows;                       // rows of a (request, head): most that may be in use
  int splits, padded;             // parts that a context is cut into where the rows alone are few; rows from the first that are cut
};

// What a part of a context leaves for the joining kernel, by part, (request, head) and row: largest score and sum of
// weights, then the outputs, normalised.  A part whose waits ran out leaves kNoPart as the sum, and the row stays as it was.
constexpr float kNoPart = -1.0f;
struct Parts {
  float *top, *sum, *o;
};
__device__ __forceinline__ Parts parts_of(const AttnParams& p, int part, long long pair) {
  const long long pairs = (long long)p.a.rows.B * p.a.cache.HKV, all = p.splits * pairs * p.padded, first = (part * pairs + pair) * p.padded;
  float* base = reinterpret_cast<float*>(p.a.workspace);
  return {base + first, base + all + first, base + 2 * all + first * p.a.cache.D};
}
inline int64_t parts_bytes(const CarryGdnKvAttentionArgs& a, int splits, int padded) {
  return splits > 1 ? 4LL * splits * a.rows.B * a.cache.HKV * padded * (a.cache.D + 2) : 0;
}
// With fewer CTAs than processors a context is cut, into parts of eight steps of 64 tokens or more: a part costs some five
// microseconds of its own, four steps' worth.
inline int split_count(const CarryGdnKvAttentionArgs& a, long long ctas) {
  const long long steps = ((long long)a.cache.max_pages * a.cache.page + 63) / 64;
  const long long n = sm_count() / (ctas < 1 ? 1 : ctas), most = steps / 8;
  return (int)(n < most ? (n < 1 ? 1 : n > 32 ? 32 : n) : most < 1 ? 1 : most > 32 ? 32 : most);
}
// Parts and pieces of a row are joined by sums of their weights, which count up to a request's tokens: less this in the exponent, so that
// values at fp32's end times the sums stay within it.
constexpr float kJoinDown = 30.0f;
int launch_join_parts(const AttnParams& p, cudaStream_t stream);

__device__ __forceinline__ uint32_t pack_half2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }
// Where products are formed in registers, weights count with the value scales of their blocks, in a unit that is a power of two;
// what is kept is `up`, 2^15 over it.  As long as the scales that a warp meets lie within 2^4 of its first ones, the unit is the
// largest of them, for all rows: a weight then has all its bits down to 2^-21 of the row's largest weight times scale, and to 2^-29
// where the scales are the same.  From then on every row has a unit of its own, not below its largest weight times scale and looked
// at again with every step: blocks that a row does not see, or hardly weighs, cost it no bits (weights below 2^-126 are none).
constexpr float kUpStart = 0x1p-104f;             // of the largest scale
// 2^15 over a power of two, both ways
__device__ __forceinline__ float up_of(float unit) { return __uint_as_float((269u << 23) - __float_as_uint(unit)); }
// 2^15 over the power of two that is not below x
__device__ __forceinline__ float up_above(float x) { return up_of(__uint_as_float((__float_as_uint(fmaxf(x, 0x1p-100f)) + 0x7fffffu) & 0x7f800000u)); }
// what outputs are multiplied by when the unit grows; there are none yet where it would be more than 1
__device__ __forceinline__ float rescale(float up, float now) { return fminf(now * up_of(up) * 0x1p-15f, 1.0f); }
struct Scales {
  float most;                     // 2^4 times the first ones; infinite before them, and -1 once rows have their own units
  __device__ __forceinline__ bool fresh() const { return most == INFINITY; }
  // whether a step's scales may stand with the others; the same in every lane
  __device__ __forceinline__ bool alike(float vs_top, float vs_low) {
    if (fresh()) most = 16.0f * vs_top;
    if (most > 0.0f && vs_top <= most && vs_low * 256.0f >= most) return true;
    most = -1.0f;
    return false;
  }
  // larger ones are looked at
  __device__ __forceinline__ float limit(float up) const { return most < 0.0f ? -1.0f : up_of(up); }
};
// two weights with their values' scale, the scale first: a weight is at most 1, and together they are at most a unit
__device__ __forceinline__ float2 scaled(float2 weights, float vs, float2 up) { return mul2(mul2(weights, make_float2(vs, vs)), up); }
// four e4m3 codes as fp16 numbers, two to a word
__device__ __forceinline__ void halves_of(uint32_t codes, uint32_t& low, uint32_t& high) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(low), "=r"(high) : "r"(codes));
}
// results below 2^-126 are zero (without .ftz every call is four instructions)
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// a (request, head)'s row: number of its query token, and where it lies in q or out
__device__ __forceinline__ int token_of(const AttnParams& p, int row) { return divide(row, p.group, p.group_shift); }
__device__ __forceinline__ long long row_place(const AttnParams& p, const KvRequest& r, int h, int row, int token, long long stride_tok, long long stride_head) {
  return (r.first + token) * stride_tok + (h * p.group + row - token * p.group) * stride_head;
}
__device__ __forceinline__ int page_index(const AttnParams& p, int granule) { return divide(granule, p.page_granules, p.page_shift); }
__device__ __forceinline__ int page_id(const AttnParams& p, int b, int granule, int length) {
  if (granule * kGranule >= length) return 0;
  return kv_page(p.a.cache, b, page_index(p, granule), p.a.status);
}

// The power of two that a query row is divided by, from the bits of its largest magnitude: what is left is below 2^15.
__device__ __forceinline__ int up_exponent(uint32_t top) { return min(max(static_cast<int>(top >> 23) - 127, -100), 127) - 14; }

// eight neighbouring fp32 results to out's type
__device__ __forceinline__ void store8(void* out, long long at, int dtype, const float* x) {
  const long long byte = at * (dtype == CARRY_F32 ? 4 : 2);
  if ((reinterpret_cast<uintptr_t>(out) + byte) % 16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) store_from_float(out, at + i, dtype, x[i]);
    return;
  }
  uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out) + byte);
  if (dtype == CARRY_F32) {
    to[0] = *reinterpret_cast<const uint4*>(x);
    to[1] = *reinterpret_cast<const uint4*>(x + 4);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == CARRY_BF16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      w[i] = pack_half2(x[2 * i], x[2 * i + 1]);
    }
  }
  *to = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void mma_fp16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
  return fmaxf(x, __shfl_xor_sync(~0u, x, 2));
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
  return x;
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(~0u, x, 1);
  return x + __shfl_xor_sync(~0u, x, 2);
}

// Where the 16-byte chunk `chunk` of token `row` lies in a tile.  The lanes that read together then fall into different
// banks both ways: a quad of lanes reads one token's chunks (keys), or the same chunk of every second token (values).
template <int D>
__device__ __forceinline__ int tile_at(int row, int chunk) {
  if constexpr (D == 128) return (row * 8 + (chunk ^ (row & 6) ^ (row & 1) << 2)) * 16;
  const int line = row >> 1;
  return (line * 8 + (((row & 1) << 2 | chunk) ^ (line & 3) << 1)) * 16;
}

// This lane's share of a query row, in one trip to memory: of every 64 columns the 16 from 16 c on.  (One element at a
// time, with its type asked for each, every load would wait for the conversion of the one before.)
template <int D, int PARTS>
__device__ __forceinline__ void load_share(const AttnParams& p, long long at, bool there, float (&x)[D / 4]) {
  const int c = threadIdx.x % 4;
  if constexpr (PARTS == 2) {
    const float* q = reinterpret_cast<const float*>(p.a.q) + at + c * 16;
#pragma unroll
    for (int e = 0; e < D / 4; ++e) x[e] = there ? q[e / 16 * 64 + e % 16] : 0.0f;
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p.a.q) + at + c * 16;
    uint32_t w[D / 8] = {};
    if (there && reinterpret_cast<uintptr_t>(q) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(q + i / 2 * 64 + i % 2 * 8);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    } else if (there) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) w[i] = q[i / 8 * 64 + i % 8 * 2] | static_cast<uint32_t>(q[i / 8 * 64 + i % 8 * 2 + 1]) << 16;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float2 f = p.a.dtype == CARRY_BF16 ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)) : unpack_half2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// Lets a kernel use `smem` bytes of shared memory: asked for once per device and thread.
template <class K>
int prepare(K kernel, size_t smem, bool (&ready)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev < 64 && ready[dev]) return CARRY_GDN_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    cudaGetLastError();
    return CARRY_GDN_ERR_LAUNCH;
  }
  if (dev < 64) ready[dev] = true;
  return CARRY_GDN_OK;
}

// few rows of a request; many; many fp32 rows
bool few_rows(const CarryGdnKvAttentionArgs& a);
int launch_kv_decode(const AttnParams& p, cudaStream_t stream);
int64_t kv_decode_workspace(const CarryGdnKvAttentionArgs& a);
int launch_kv_chunk(AttnParams p, cudaStream_t stream);
int64_t kv_chunk_workspace(const CarryGdnKvAttentionArgs& a);
int launch_kv_prefill(AttnParams p, cudaStream_t stream);
int64_t kv_prefill_workspace(const CarryGdnKvAttentionArgs& a);

}  // namespace carry
