// New tokens' keys and values into the 8-bit cache: one CTA for each (request, block of tokens, head) that the
// call touches, the keys on its first half and the values on its second.
//
// A block's scale is the smallest power of two that brings its largest magnitude within e4m3's 448.  Powers of two
// cost a float format no precision (only the exponent shifts), and they make a later growth of the scale exact: the
// codes of the block's earlier tokens move by whole binades, so a block filled token by token ends with the codes of
// one filled at once, subnormals apart.
//
// A CTA lives for three trips to memory (lengths, page id, rows) and one block, so what counts is how many are on an SM.  With blocks
// of 32 tokens of 128 numbers and 16-bit rows (four items of eight numbers to a thread) six of 40 registers a thread write 8192
// tokens of 8 heads (50 MB) in 11.3 us, 4.4 TB/s, where the calls before have left them in L2, and 12.9 where not; five took 13.2, and
// reading the rows a second time for the codes 25.  Blocks of 64 and 128 take the kernel of 16 items (124 registers, two CTAs): 18.4
// and 13.0 us.  fp32 rows: 15.1 in blocks of 32 (70 registers, three CTAs), 31.3 and 21.9 in the others (190, one).
#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr int kThreads = 256, kHalf = kThreads / 2, kMaxBlock = 128;
constexpr uint32_t kNotFinite = 0x7f800000u;      // bits of |x| from here on: infinities and NaNs

struct AppendParams {
  CarryGdnKvAppendArgs a;
  int page_shift, block_shift;
  bool vec;                       // every row of k and v starts on a 16-byte boundary
};

// bits of the largest magnitude among eight numbers
template <int DTYPE>
__device__ __forceinline__ uint32_t top_bits(const Raw<DTYPE>& r) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
  uint32_t t = 0;
  if constexpr (DTYPE == CARRY_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, w[i] & 0x7fffffffu);
    return t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __vmaxu2(t, w[i] & 0x7fff7fffu);
    t = max(t >> 16, t & 0xffffu);
    if constexpr (DTYPE == CARRY_BF16) return t << 16;
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(t))));
  }
}

__device__ __forceinline__ uint2 codes8(const Eight& e, float inv) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __nv_cvt_float2_to_fp8x2(mul2(e.x[i], make_float2(inv, inv)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

// A block that already holds tokens may have them under any scale (a cache that was filled elsewhere), and only of a power of two
// with one in fp32's normal numbers is the reciprocal exact in fp32.  Of others it is taken in 64 bits, by Newton's iteration, so
// that a quotient halfway between two codes is found to be that.  (A division would be a call, and take the kernel's registers.)
__device__ __forceinline__ bool exact_inverse(float scale) {
  const uint32_t u = __float_as_uint(scale);
  return (u & 0x7fffffu) == 0 && u - 1 < (254u << 23) - 1;
}
__device__ __forceinline__ double inverse64(float scale) {
  const double d = scale;
  const long long u = __double_as_longlong(d);
  const double part = __longlong_as_double((u & 0xfffffffffffffll) | 1023ll << 52);       // of [1, 2)
  double r = __fdividef(1.0f, static_cast<float>(part));
  r = r * (2.0 - part * r);
  r = r * (2.0 - part * r);
  return r * __longlong_as_double((2046ll << 52) - (u & 0x7ff0000000000000ll));
}
__device__ __forceinline__ uint2 codes8(const Eight& e, double inv) {
  Eight y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y.x[i] = make_float2(static_cast<float>(e.x[i].x * inv), static_cast<float>(e.x[i].y * inv));
  return codes8(y, 1.0f);
}

// ITEMS: a thread's share of a block's new tokens, eight numbers each, held in registers from the maximum to the codes.
template <int D, int DTYPE, int ITEMS>
__global__ void __launch_bounds__(kThreads, ITEMS <= 4 && DTYPE != CARRY_F32 ? 6 : 1) kv_append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ uint32_t token_top[2][kMaxBlock];    // bits of each new token's largest magnitude
  __shared__ uint32_t top[2][kHalf / 32];
  constexpr int kPer = D / 8;                     // that many neighbouring lanes have a token
  depend_release();
  depend_wait();
  const CarryGdnKvAppendArgs& a = p.a;
  const CarryGdnKvCache& c = a.cache;
  const int b = blockIdx.z, h = blockIdx.y;
  const KvRequest r = kv_request(c, a.rows, b, blockIdx.x == 0 && h == 0 && threadIdx.x == 0 ? a.status : nullptr);
  const int origin = r.length - r.count;          // position of the request's row 0
  const int from = max(origin, 0), to = min(r.length, origin + r.todo);
  const int start = (divide(from, c.block, p.block_shift) + blockIdx.x) * c.block;
  const int t0 = max(start, from), t1 = min(start + c.block, to);
  if (t0 >= t1) return;
  const int index = divide(start, c.page, p.page_shift), offset = start - index * c.page;
  const int page = kv_page(c, b, index, h == 0 && threadIdx.x == 0 ? a.status : nullptr);
  if (page == 0) return;

  const bool is_v = threadIdx.x >= kHalf;
  const int tid = threadIdx.x % kHalf, items = (t1 - t0) * kPer;
  const long long stride_tok = is_v ? a.stride_v_tok : a.stride_k_tok;
  const long long row = (r.first + (t0 - origin) + tid / kPer) * stride_tok + h * (is_v ? a.stride_v_head : a.stride_k_head) + tid % kPer * 8;
  const void* x = is_v ? a.v : a.k;
  uint8_t* codes = (is_v ? c.v_codes + page * c.stride_v_page : c.k_codes + page * c.stride_k_page) +
                   ((long long)h * c.page + offset) * D;
  float* scale = (is_v ? c.v_scale + page * c.stride_vs_page : c.k_scale + page * c.stride_ks_page) +
                 h * divide(c.page, c.block, p.block_shift) + divide(offset, c.block, p.block_shift);

  Raw<DTYPE> e[ITEMS];
#pragma unroll
  for (int n = 0; n < ITEMS; ++n) {
    if (n * kHalf + tid >= items) continue;
    const long long at = row + n * (kHalf / kPer) * stride_tok;
    if (p.vec) {
      e[n] = load_raw<DTYPE>(x, at);
    } else if constexpr (DTYPE == CARRY_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<uint32_t*>(&e[n])[i] = reinterpret_cast<const uint32_t*>(x)[at + i];
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(x) + at;
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(&e[n])[i] = q[2 * i] | static_cast<uint32_t>(q[2 * i + 1]) << 16;
    }
  }
  const float old = t0 > start ? *scale : 0.0f;
#pragma unroll
  for (int n = 0; n < ITEMS; ++n) {
    uint32_t t = n * kHalf + tid < items ? top_bits<DTYPE>(e[n]) : 0;
#pragma unroll
    for (int s = kPer / 2; s > 0; s /= 2) t = max(t, __shfl_xor_sync(~0u, t, s));
    if (n * kHalf + tid < items && tid % kPer == 0) token_top[is_v][(n * kHalf + tid) / kPer] = t;
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
    if (old < now) {
      const float shift = __fdiv_rn(old, now);
      for (int i = tid; i < (t0 - start) * kPer; i += kHalf) {
        const uint2 w = reinterpret_cast<const uint2*>(codes)[i];
        Eight early;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          early.x[j] = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((j < 2 ? w.x : w.y) >> (j % 2 * 16)), __NV_E4M3)));
        reinterpret_cast<uint2*>(codes)[i] = codes8(early, shift);
      }
    } else {
      now = old;
    }
  }
  uint2* to_codes = reinterpret_cast<uint2*>(codes + (long long)(t0 - start) * D);
  auto store = [&](auto by) {
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
      const int i = n * kHalf + tid;
      if (i >= items) continue;
      uint2 w = codes8(unpack<DTYPE>(e[n]), by);
      if (max(token_top[0][i / kPer], token_top[1][i / kPer]) >= kNotFinite)
        w = is_v ? make_uint2(0, 0) : make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
      to_codes[i] = w;
    }
  };
  if (__builtin_expect(exact_inverse(now), 1)) store(__uint_as_float((254u << 23) - __float_as_uint(now)));
  else store(inverse64(now));
  if (tid == 0 && now != old) *scale = now;       // every thread read the old one before the first barrier
}

template <int D, int DTYPE>
int launch_items(const AppendParams& p, dim3 grid, cudaStream_t stream) {
  const int tokens = p.a.rows.max_query < p.a.cache.block ? p.a.rows.max_query : p.a.cache.block;
  const int items = (tokens * D / 8 + kHalf - 1) / kHalf;               // 16 at most
  if (items <= 1) return launch_dependent(kv_append_kernel<D, DTYPE, 1>, grid, kThreads, 0, stream, p);
  if (items <= 4) return launch_dependent(kv_append_kernel<D, DTYPE, 4>, grid, kThreads, 0, stream, p);
  return launch_dependent(kv_append_kernel<D, DTYPE, 16>, grid, kThreads, 0, stream, p);
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
  const AppendParams p = {a, shift_of(c.page), shift_of(c.block), vec};
  const dim3 grid(blocks, c.HKV, a.rows.B);
  if (a.dtype == CARRY_F32) return c.D == 64 ? launch_items<64, CARRY_F32>(p, grid, stream) : launch_items<128, CARRY_F32>(p, grid, stream);
  if (a.dtype == CARRY_BF16) return c.D == 64 ? launch_items<64, CARRY_BF16>(p, grid, stream) : launch_items<128, CARRY_BF16>(p, grid, stream);
  return c.D == 64 ? launch_items<64, CARRY_F16>(p, grid, stream) : launch_items<128, CARRY_F16>(p, grid, stream);
}

}  // namespace carry
