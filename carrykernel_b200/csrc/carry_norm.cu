// The entry of a layer: residual addition, root-mean-square norm, e4m3 codes with scales.  One CTA per row.
//
// The row is read once and held in registers.  With t = h * weight the normed row is t * rstd, and its largest
// magnitude is rstd times t's, so the sum of squares and the maximum come out of one pass and one reduction.
#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr float kAmaxFloor = 1e-12f;
constexpr int kGroup = 128;

struct NormParams {
  CarryGdnNormArgs a;
  double inv_width;
  bool vec;                       // every row starts on a 16-byte boundary and W is a multiple of 8
};

__device__ __forceinline__ void load8(const void* p, long long at, int n, int dtype, bool vec, float (&x)[8]) {
  if (vec && dtype == CARRY_F32) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
    const float4 u = q[0], v = q[1];
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
  } else if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (dtype == CARRY_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? load_as_float(p, at + i, dtype) : 0.0f;
  }
}

__device__ __forceinline__ void store8(void* p, long long at, int n, int dtype, bool vec, const float (&x)[8]) {
  if (vec && dtype == CARRY_F32) {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at);
    q[0] = make_float4(x[0], x[1], x[2], x[3]);
    q[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else if (vec) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (dtype == CARRY_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) store_from_float(p, at + i, dtype, x[i]);
  }
}

// C chunks of 8 columns per thread, chunk j of thread t being number j * blockDim + t of the row
template <int C>
__global__ void __launch_bounds__(512) norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ double sums[32];
  __shared__ uint32_t tops[32];
  depend_release();
  depend_wait();
  const CarryGdnNormArgs& a = p.a;
  const long long row = blockIdx.x;
  float t[C][8];
  double ss = 0.0;                // the sum of squares of numbers that fp32 holds need not fit it
  uint32_t top[C], all = 0;       // bits of the largest |t|: NaNs compare above infinities, and those above numbers
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int at = (j * blockDim.x + threadIdx.x) * 8, n = min(a.W - at, 8);
    top[j] = 0;
    if (n <= 0) continue;
    load8(a.x, row * a.stride_x + at, n, a.x_dtype, p.vec, t[j]);
    if (a.residual) {
      float r[8];
      load8(a.residual, row * a.stride_residual + at, n, a.residual_dtype, p.vec, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[j][i] += r[i];
    }
    if (a.residual_out) store8(a.residual_out, row * a.stride_residual_out + at, n, a.residual_dtype, p.vec, t[j]);
    float w[8];
    load8(a.weight, at, n, a.weight_dtype, p.vec, w);
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) part = fmaf(t[j][i], t[j][i], part);
    if (part < 0x1p126f) {
      ss += part;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += (double)t[j][i] * t[j][i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[j][i] *= w[i];
      top[j] = max(top[j], __float_as_uint(t[j][i]) & 0x7fffffffu);
    }
    all = max(all, top[j]);
  }
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
#pragma unroll
  for (int s = 16; s > 0; s /= 2) ss += __shfl_xor_sync(~0u, ss, s);
  all = __reduce_max_sync(~0u, all);
  if (lane == 0) { sums[warp] = ss; tops[warp] = all; }
  __syncthreads();
  ss = 0.0;
  for (int i = 0; i < warps; ++i) { ss += sums[i]; all = max(all, tops[i]); }
  const bool finite = all < 0x7f800000u;
  const double mean = ss * p.inv_width + a.eps;
  const float root = mean < 0x1p126 ? rsqrtf((float)mean) : rsqrtf((float)(mean * 0x1p-130)) * 0x1p-65f;
  const float rstd = finite ? root : __uint_as_float(0x7fffffffu);
  float scale = __fdiv_rn(fmaxf(__uint_as_float(all) * rstd, kAmaxFloor), kF8Max);
  if (a.group == 0 && threadIdx.x == 0) a.scale[row] = finite ? scale : rstd;
  const int groups = (a.W + kGroup - 1) / kGroup;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int at = (j * blockDim.x + threadIdx.x) * 8, n = min(a.W - at, 8);
    if (a.group) {                // 16 neighbouring lanes have a group
#pragma unroll
      for (int s = 8; s > 0; s /= 2) top[j] = max(top[j], __shfl_xor_sync(~0u, top[j], s));
      scale = __fdiv_rn(fmaxf(__uint_as_float(top[j]) * rstd, kAmaxFloor), kF8Max);
      if (n > 0 && lane % 16 == 0) a.scale[row * groups + at / kGroup] = finite ? scale : rstd;
    }
    if (n <= 0) continue;
    const float mul = finite ? __fdiv_rn(rstd, scale) : rstd;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __nv_cvt_float2_to_fp8x2(make_float2(t[j][2 * i] * mul, t[j][2 * i + 1] * mul), __NV_SATFINITE, __NV_E4M3);
    uint8_t* to = a.codes + row * a.stride_codes + at;
    if (p.vec) {
      *reinterpret_cast<uint2*>(to) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) to[i] = static_cast<uint8_t>(w[i / 2] >> (i % 2 * 8));
    }
  }
}

}  // namespace

int launch_norm(const CarryGdnNormArgs& a, cudaStream_t stream) {
  NormParams p = {a, 1.0 / a.W, a.W % 8 == 0};
  auto size = [](int dtype) { return dtype == CARRY_F32 ? 4 : 2; };
  auto rows = [&](const void* q, long long stride, int bytes, int to) {
    if (q) p.vec = p.vec && reinterpret_cast<uintptr_t>(q) % to == 0 && stride * bytes % to == 0;
  };
  rows(a.x, a.stride_x, size(a.x_dtype), 16);
  rows(a.residual, a.stride_residual, size(a.residual_dtype), 16);
  rows(a.residual_out, a.stride_residual_out, size(a.residual_dtype), 16);
  rows(a.weight, 0, size(a.weight_dtype), 16);
  rows(a.codes, a.stride_codes, 1, 8);
  const int chunks = (a.W + 7) / 8;
  auto threads = [&](int c) { return static_cast<unsigned>((chunks + 32 * c - 1) / (32 * c) * 32); };
  if (chunks <= 512) return launch_dependent(norm_kernel<1>, dim3(a.N), threads(1), 0, stream, p);
  if (chunks <= 1024) return launch_dependent(norm_kernel<2>, dim3(a.N), threads(2), 0, stream, p);
  if (chunks <= 2048) return launch_dependent(norm_kernel<4>, dim3(a.N), threads(4), 0, stream, p);
  return launch_dependent(norm_kernel<8>, dim3(a.N), threads(8), 0, stream, p);
}

}  // namespace carry
