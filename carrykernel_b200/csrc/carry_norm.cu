// The entry of a layer: residual addition, root-mean-square norm, e4m3 codes with scales.  A CTA takes a row at a time.
//
// The row is read once and held in registers, and the CTA's next row is on its way while the present one is reduced.
// With t = h * weight the normed row is t * rstd, and its largest magnitude is rstd times t's, so the sum of squares and
// the maximum come out of one pass and one reduction.
#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr float kAmaxFloor = 1e-12f;
constexpr int kGroup = 128, kMaxWarps = 16;

// Squares from here on are summed times 2^-128: those of numbers that fp32 holds need not fit it.
constexpr float kLarge = 0x1p100f;

struct NormParams {
  CarryGdnNormArgs a;
  float inv_width;
};

template <int DTYPE>
__device__ __forceinline__ void store(void* p, long long at, const Eight& e) {
  if constexpr (DTYPE == CARRY_F32) {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at);
    q[0] = make_float4(e.x[0].x, e.x[0].y, e.x[1].x, e.x[1].y);
    q[1] = make_float4(e.x[2].x, e.x[2].y, e.x[3].x, e.x[3].y);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DTYPE == CARRY_BF16) {
        const __nv_bfloat162 v = __float22bfloat162_rn(e.x[i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __float22half2_rn(e.x[i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// the same an element at a time, for rows that are not aligned, or of types that have no kernel of their own
__device__ __forceinline__ Eight load_slow(const void* p, long long at, int n, int dtype) {
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e.x[i].x = 2 * i < n ? load_as_float(p, at + 2 * i, dtype) : 0.0f;
    e.x[i].y = 2 * i + 1 < n ? load_as_float(p, at + 2 * i + 1, dtype) : 0.0f;
  }
  return e;
}

// How rows are spread: a warp's share of a row's reduction costs as much as a chunk or two of its own work, so lanes have
// two chunks where that still leaves warps enough, four where a row is wide.  The next row's loads are in flight all the
// time: 1024 threads of two chunks of 2 x 16 bytes are 64 KB on an SM, and 40 KB hide the latency of the memory.
__host__ __device__ constexpr int max_threads(int C) { return C == 1 ? 128 : 512; }
__host__ __device__ constexpr int min_ctas(int C) { return C == 1 ? 8 : C == 2 ? 2 : 1; }

// C chunks of 8 columns per thread, chunk j of thread t being number j * blockDim + t of the row.  VEC: x is of type X,
// the residual of type R, every row starts on a 16-byte boundary and W is a multiple of 8; otherwise X and R say nothing.
template <int C, bool VEC, int X, int R>
__global__ void __launch_bounds__(max_threads(C), min_ctas(C)) norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float sums[2][kMaxWarps], larges[2][kMaxWarps], tops[2][kMaxWarps];
  constexpr bool kAhead = C <= 4;                 // more would not fit the registers
  depend_release();
  depend_wait();
  const CarryGdnNormArgs& a = p.a;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32, groups = (a.W + kGroup - 1) / kGroup;
  const bool has_residual = a.residual != nullptr;
  Raw<X> next_x[C];
  Raw<R> next_r[C];
  auto fetch = [&](long long row) {
    if (!VEC || row >= a.N) return;
    const long long x_row = row * a.stride_x, r_row = row * a.stride_residual;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int at = (j * blockDim.x + threadIdx.x) * 8;
      if (at >= a.W) continue;
      next_x[j] = load_raw<X>(a.x, x_row + at);
      if (has_residual) next_r[j] = load_raw<R>(a.residual, r_row + at);
    }
  };
  if (kAhead) fetch(blockIdx.x);
  int turn = 0;
  for (long long row = blockIdx.x; row < a.N; row += gridDim.x, turn ^= 1) {
    Eight t[C];
    float2 ss = make_float2(0.0f, 0.0f);
    float large = 0.0f, top[C], all = 0.0f;
    if (!kAhead) fetch(row);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int at = (j * blockDim.x + threadIdx.x) * 8, n = min(a.W - at, 8);
      if (n <= 0) continue;
      if constexpr (VEC) t[j] = unpack<X>(next_x[j]);
      else t[j] = load_slow(a.x, row * a.stride_x + at, n, a.x_dtype);
      if (has_residual) {
        Eight r;
        if constexpr (VEC) r = unpack<R>(next_r[j]);
        else r = load_slow(a.residual, row * a.stride_residual + at, n, a.residual_dtype);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[j].x[i] = add2(t[j].x[i], r.x[i]);
      }
    }
    if (kAhead) fetch(row + gridDim.x);           // in flight while this row is reduced
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int at = (j * blockDim.x + threadIdx.x) * 8, n = min(a.W - at, 8);
      top[j] = 0.0f;
      if (n <= 0) continue;
      Eight w;
      if constexpr (VEC) {
        if (a.residual_out) store<R>(a.residual_out, row * a.stride_residual_out + at, t[j]);
        if (a.weight_dtype == X) w = unpack<X>(load_raw<X>(a.weight, at));
        else if (a.weight_dtype == CARRY_F32) w = unpack<CARRY_F32>(load_raw<CARRY_F32>(a.weight, at));
        else w = load_slow(a.weight, at, 8, a.weight_dtype);
      } else {
        w = load_slow(a.weight, at, n, a.weight_dtype);
        if (a.residual_out) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < n) store_from_float(a.residual_out, row * a.stride_residual_out + at + i, a.residual_dtype, i % 2 ? t[j].x[i / 2].y : t[j].x[i / 2].x);
        }
      }
      float2 part = mul2(t[j].x[0], t[j].x[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) part = fma2(t[j].x[i], t[j].x[i], part);
      if (part.x + part.y < kLarge) {
        ss = add2(ss, part);
      } else {                                    // NaNs come here too
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = t[j].x[i].x * 0x1p-64f, v = t[j].x[i].y * 0x1p-64f;
          large += u * u + v * v;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[j].x[i] = mul2(t[j].x[i], w.x[i]);
        top[j] = fmaxf(top[j], fmaxf(fabsf(t[j].x[i].x), fabsf(t[j].x[i].y)));
      }
      all = fmaxf(all, top[j]);
    }
    float sum = ss.x + ss.y;
#pragma unroll
    for (int s = 16; s > 0; s /= 2) sum += __shfl_xor_sync(~0u, sum, s);
    all = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(all)));   // no NaNs, not negative: ordered as whole numbers
    if (__any_sync(~0u, large != 0.0f)) {
#pragma unroll
      for (int s = 16; s > 0; s /= 2) large += __shfl_xor_sync(~0u, large, s);
    }
    if (lane == 0) { sums[turn][warp] = sum; larges[turn][warp] = large; tops[turn][warp] = all; }
    __syncthreads();              // the next row has the other half: one barrier a row
    sum = large = 0.0f;
    for (int i = 0; i < warps; ++i) { sum += sums[turn][i]; large += larges[turn][i]; all = fmaxf(all, tops[turn][i]); }
    const bool finite = large < INFINITY && all < INFINITY;
    float rstd = large == 0.0f ? rsqrtf(fmaf(sum, p.inv_width, a.eps)) : rsqrtf(fmaf(sum, 0x1p-128f, large) * p.inv_width) * 0x1p-64f;
    if (!finite) rstd = __uint_as_float(0x7fffffffu);
    float scale = fmaxf(all * rstd, kAmaxFloor) * (1.0f / kF8Max), mul = __fdividef(rstd, scale);
    if (a.group == 0 && threadIdx.x == 0) a.scale[row] = finite ? scale : rstd;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int at = (j * blockDim.x + threadIdx.x) * 8, n = min(a.W - at, 8);
      if (a.group) {              // 16 neighbouring lanes have a group
#pragma unroll
        for (int s = 8; s > 0; s /= 2) top[j] = fmaxf(top[j], __shfl_xor_sync(~0u, top[j], s));
        scale = fmaxf(top[j] * rstd, kAmaxFloor) * (1.0f / kF8Max);
        mul = __fdividef(rstd, scale);
        if (n > 0 && lane % 16 == 0) a.scale[row * groups + at / kGroup] = finite ? scale : rstd;
      }
      if (n <= 0) continue;
      const float2 by = finite ? make_float2(mul, mul) : make_float2(rstd, rstd);
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = __nv_cvt_float2_to_fp8x2(mul2(t[j].x[i], by), __NV_SATFINITE, __NV_E4M3);
      uint8_t* to = a.codes + row * a.stride_codes + at;
      if constexpr (VEC) {
        *reinterpret_cast<uint2*>(to) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) to[i] = static_cast<uint8_t>(c[i / 2] >> (i % 2 * 8));
      }
    }
  }
}

template <bool VEC, int X, int R>
int launch_typed(const NormParams& p, cudaStream_t stream) {
  const int chunks = (p.a.W + 7) / 8;
  auto launch = [&](auto kernel, int c) {
    const unsigned threads = (chunks + 32 * c - 1) / (32 * c) * 32;
    const long long resident = (long long)sm_count() * (max_threads(c) * min_ctas(c) / threads);
    return launch_dependent(kernel, dim3((unsigned)(p.a.N < resident ? p.a.N : resident)), threads, 0, stream, p);
  };
  if (chunks <= 128) return launch(norm_kernel<1, VEC, X, R>, 1);
  if (chunks <= 1024) return launch(norm_kernel<2, VEC, X, R>, 2);
  if (chunks <= 2048) return launch(norm_kernel<4, VEC, X, R>, 4);
  return launch(norm_kernel<8, VEC, X, R>, 8);
}

}  // namespace

int launch_norm(const CarryGdnNormArgs& a, cudaStream_t stream) {
  if (sm_count() == 0) return CARRY_GDN_ERR_NO_DEVICE;
  const NormParams p = {a, 1.0f / a.W};
  bool vec = a.W % 8 == 0;
  auto size = [](int dtype) { return dtype == CARRY_F32 ? 4 : 2; };
  auto rows = [&](const void* q, long long stride, int bytes, int to) {
    if (q) vec = vec && reinterpret_cast<uintptr_t>(q) % to == 0 && stride * bytes % to == 0;
  };
  rows(a.x, a.stride_x, size(a.x_dtype), 16);
  rows(a.residual, a.stride_residual, size(a.residual_dtype), 16);
  rows(a.residual_out, a.stride_residual_out, size(a.residual_dtype), 16);
  rows(a.weight, 0, size(a.weight_dtype), 16);
  rows(a.codes, a.stride_codes, 1, 8);
  // the residual stream has x's type or is fp32; other pairs go an element at a time
  const int xd = a.x_dtype, rd = a.residual_dtype;
  if (vec && xd == CARRY_BF16 && rd == CARRY_BF16) return launch_typed<true, CARRY_BF16, CARRY_BF16>(p, stream);
  if (vec && xd == CARRY_F16 && rd == CARRY_F16) return launch_typed<true, CARRY_F16, CARRY_F16>(p, stream);
  if (vec && xd == CARRY_F32 && rd == CARRY_F32) return launch_typed<true, CARRY_F32, CARRY_F32>(p, stream);
  if (vec && xd == CARRY_BF16 && rd == CARRY_F32) return launch_typed<true, CARRY_BF16, CARRY_F32>(p, stream);
  if (vec && xd == CARRY_F16 && rd == CARRY_F32) return launch_typed<true, CARRY_F16, CARRY_F32>(p, stream);
  return launch_typed<false, CARRY_F32, CARRY_F32>(p, stream);
}

}  // namespace carry
