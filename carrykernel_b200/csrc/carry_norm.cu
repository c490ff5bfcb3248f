// The entry of a layer: residual addition, root-mean-square norm, e4m3 codes with scales.  A CTA takes a row at a time.
//
// The row is read once and held in registers, and the CTA's next row is on its way while the present one is reduced.
// With t = h * weight the normed row is t * rstd, and its largest magnitude is rstd times t's, so the sum of squares and
// the maximum come out of one pass and one reduction.
//
// What bounds it: 16384 rows of 4096 in bf16 take 83 us, 5.7 TB/s, 87 % of the copy rate; 256 rows take 3.8 us, of which the
// launch and one trip to memory are most.  A row is
// 440 instructions of a warp; with 533 they were the bound (92 us).
#include <type_traits>

#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr float kAmaxFloor = 1e-12f;
constexpr int kGroup = 128, kMaxWarps = 16;

// Squares from here on are summed times 2^-160: those of numbers that fp32 holds need not fit it, and 32768 of the largest, times
// that, do.
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
// an element at a time: weights of another type than x
__device__ __forceinline__ Eight load_slow(const void* p, long long at, int dtype) {
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) e.x[i] = make_float2(load_as_float(p, at + 2 * i, dtype), load_as_float(p, at + 2 * i + 1, dtype));
  return e;
}

// How rows are spread: a warp's share of a row's reduction costs as much as a chunk or two of its own work, so lanes have
// two chunks where that still leaves warps enough, four where a row is wide.  The next row's loads are in flight all the
// time: 1024 threads of two chunks of 2 x 16 bytes are 64 KB on an SM, and 40 KB hide the latency of the memory.
__host__ __device__ constexpr int max_threads(int C) { return C == 1 ? 128 : 512; }
__host__ __device__ constexpr int min_ctas(int C) { return C == 1 ? 8 : C == 2 ? 2 : 1; }

// The reduction of a row across its warps, and what comes of it.
struct RowSums {
  float2 part[2][kMaxWarps];      // sum of squares and largest |t| of a warp; the sum is NaN where squares left its range
  float sum[2][kMaxWarps], large[2][kMaxWarps];
};
struct RowScale {
  float rstd, top;                // rstd is NaN where a number of the row is not finite
};
__device__ __forceinline__ RowScale reduce_row(const NormParams& p, RowSums& sh, int turn, float sum, float large, float top) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
#pragma unroll
  for (int s = 16; s > 0; s /= 2) sum += __shfl_xor_sync(~0u, sum, s);
  top = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top)));  // no NaNs, not negative: ordered as whole numbers
  const bool out = __any_sync(~0u, large != 0.0f);
  if (out) {
#pragma unroll
    for (int s = 16; s > 0; s /= 2) large += __shfl_xor_sync(~0u, large, s);
  }
  if (lane == 0) {
    sh.part[turn][warp] = make_float2(out ? NAN : sum, top);
    sh.sum[turn][warp] = sum;
    sh.large[turn][warp] = large;
  }
  __syncthreads();                // the next row has the other half: one barrier a row
  sum = 0.0f;
  for (int i = 0; i < warps; ++i) {
    const float2 x = sh.part[turn][i];
    sum += x.x;
    top = fmaxf(top, x.y);
  }
  float rstd = rsqrtf(fmaf(sum, p.inv_width, p.a.eps));
  if (sum != sum) {
    sum = large = 0.0f;
    for (int i = 0; i < warps; ++i) {
      sum += sh.sum[turn][i];
      large += sh.large[turn][i];
    }
    rstd = large < INFINITY ? rsqrtf(fmaf(sum * 0x1p-80f, 0x1p-80f, large) * p.inv_width) * 0x1p-80f : NAN;
  }
  return {top < INFINITY ? rstd : NAN, top};
}

// Sum of the squares of 2 N numbers; from kLarge on it counts in `large`, times 2^-160 (NaNs do, too).
template <int N>
__device__ __forceinline__ void add_squares(const float2 (&t)[N], float2& ss, float& large) {
  float2 part = mul2(t[0], t[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) part = fma2(t[i], t[i], part);
  if (part.x + part.y < kLarge) {
    ss = add2(ss, part);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float u = t[i].x * 0x1p-80f, v = t[i].y * 0x1p-80f;
      large += u * u + v * v;
    }
  }
}
// t * weight, and its largest magnitude
__device__ __forceinline__ float weigh(Eight& t, const Eight& w) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t.x[i] = mul2(t.x[i], w.x[i]);
    top = fmaxf(top, fmaxf(fabsf(t.x[i].x), fabsf(t.x[i].y)));
  }
  return top;
}
__device__ __forceinline__ uint2 codes_of(const Eight& t, float by) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __nv_cvt_float2_to_fp8x2(mul2(t.x[i], make_float2(by, by)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}
// The scale of a row or a group, whose largest |t| is `top`, and what t is multiplied by.
__device__ __forceinline__ float scale_of(const RowScale& r, float top, float& by) {
  const float scale = fmaxf(top * r.rstd, kAmaxFloor) * (1.0f / kF8Max);      // fmaxf drops a NaN
  by = r.rstd == r.rstd ? __fdividef(r.rstd, scale) : NAN;
  return r.rstd == r.rstd ? scale : NAN;
}
__device__ __forceinline__ float group_max(float top) {                       // 16 neighbouring lanes have a group
#pragma unroll
  for (int s = 8; s > 0; s /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
  return top;
}

// C chunks of 8 columns per thread, chunk j of thread t being number j * blockDim + t of the row; x is of type X, the
// residual of type R, every row starts on a 16-byte boundary and W is a multiple of 8.
template <int C, int X, int R>
__global__ void __launch_bounds__(max_threads(C), min_ctas(C)) norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ RowSums sums;
  constexpr bool kAhead = C <= 4;                 // more would not fit the registers
  constexpr int kX = X == CARRY_F32 ? 4 : 2, kR = R == CARRY_F32 ? 4 : 2;
  depend_release();
  depend_wait();
  const CarryGdnNormArgs& a = p.a;
  const int lane = threadIdx.x % 32, groups = (a.W + kGroup - 1) / kGroup, first = threadIdx.x * 8, jump = blockDim.x * 8;
  const bool has_residual = a.residual != nullptr;
  // this thread's first chunk of the CTA's next row to load, and of the present one
  const long long row0 = blockIdx.x, rows = gridDim.x;
  const char* x = static_cast<const char*>(a.x) + (row0 * a.stride_x + first) * kX;
  const char* r = static_cast<const char*>(a.residual) + (row0 * a.stride_residual + first) * kR;
  char* out = static_cast<char*>(a.residual_out) + (row0 * a.stride_residual_out + first) * kR;
  uint8_t* codes = a.codes + row0 * a.stride_codes + first;
  float* scales = a.scale + row0 * (a.group ? groups : 1);
  Raw<X> next_x[C];
  Raw<R> next_r[C];
  auto fetch = [&](bool there) {
    if (there) {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (first + j * jump >= a.W) continue;
        next_x[j] = load_raw<X>(x, j * jump);
        if (has_residual) next_r[j] = load_raw<R>(r, j * jump);
      }
    }
    x += rows * a.stride_x * kX;
    r += rows * a.stride_residual * kR;
  };
  if (kAhead) fetch(row0 < a.N);
  int turn = 0;
  for (long long row = row0; row < a.N; row += rows, turn ^= 1) {
    Eight t[C];
    float2 ss = make_float2(0.0f, 0.0f);
    float large = 0.0f, top[C], all = 0.0f;
    if (!kAhead) fetch(true);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      t[j] = unpack<X>(next_x[j]);
      if (has_residual) {
        const Eight add = unpack<R>(next_r[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[j].x[i] = add2(t[j].x[i], add.x[i]);
      }
    }
    if (kAhead) fetch(row + rows < a.N);          // in flight while this row is reduced
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int at = first + j * jump;
      top[j] = 0.0f;
      if (at >= a.W) continue;
      if (a.residual_out) store<R>(out, j * jump, t[j]);
      add_squares(t[j].x, ss, large);
      if (a.weight_dtype == X) top[j] = weigh(t[j], unpack<X>(load_raw<X>(a.weight, at)));
      else if (a.weight_dtype == CARRY_F32) top[j] = weigh(t[j], unpack<CARRY_F32>(load_raw<CARRY_F32>(a.weight, at)));
      else top[j] = weigh(t[j], load_slow(a.weight, at, a.weight_dtype));
      all = fmaxf(all, top[j]);
    }
    const RowScale s = reduce_row(p, sums, turn, ss.x + ss.y, large, all);
    if (a.group == 0) {
      float by;
      const float scale = scale_of(s, s.top, by);
      if (threadIdx.x == 0) *scales = scale;
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (first + j * jump < a.W) *reinterpret_cast<uint2*>(codes + j * jump) = codes_of(t[j], by);
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int at = first + j * jump;
        float by;
        const float scale = scale_of(s, group_max(top[j]), by);
        if (at >= a.W) continue;
        if (lane % 16 == 0) scales[at / kGroup] = scale;
        *reinterpret_cast<uint2*>(codes + j * jump) = codes_of(t[j], by);
      }
    }
    out += rows * a.stride_residual_out * kR;
    codes += rows * a.stride_codes;
    scales += rows * (a.group ? groups : 1);
  }
}

// ---- any rows: odd widths, rows off the 16-byte grid, other pairs of types ---------------------------------------------

template <int DTYPE>
struct Number {
  using type = uint16_t;
};
template <>
struct Number<CARRY_F32> {
  using type = float;
};
template <int DTYPE>
__device__ __forceinline__ float value_of(typename Number<DTYPE>::type u) {
  if constexpr (DTYPE == CARRY_F32) return u;
  else if constexpr (DTYPE == CARRY_BF16) return __uint_as_float(static_cast<uint32_t>(u) << 16);
  else return __half2float(__ushort_as_half(u));
}
template <int DTYPE>
__device__ __forceinline__ void round_two(float2 v, typename Number<DTYPE>::type& low, typename Number<DTYPE>::type& high) {
  if constexpr (DTYPE == CARRY_F32) {
    low = v.x;
    high = v.y;
  } else {
    uint32_t u;
    if constexpr (DTYPE == CARRY_BF16) {
      const __nv_bfloat162 h = __float22bfloat162_rn(v);
      u = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __float22half2_rn(v);
      u = *reinterpret_cast<const uint32_t*>(&h);
    }
    low = static_cast<uint16_t>(u);
    high = static_cast<uint16_t>(u >> 16);
  }
}

// A warp takes C runs of 128 columns, lane l the numbers l, 32 + l, 64 + l and 96 + l of each: neighbouring lanes have
// neighbouring numbers, so a warp's access is one or two lines wherever the row begins, and a group's maximum is a
// warp's.  Only a row's last warp asks of its numbers whether they are there.  16384 rows of 4095 in bf16 take 128 us, 3.7 TB/s, bound
// by instructions for lanes of 2 bytes (a lane with eight neighbouring numbers 351; four, from the boundary that its
// tensors share, with edges by themselves, 170), in fp32 144 us, 92 % of the copy rate.
__host__ __device__ constexpr int any_ctas(int C) { return C <= 4 ? 2 : 1; }
template <int C, int X, int R>
__global__ void __launch_bounds__(512, any_ctas(C)) norm_any_kernel(const __grid_constant__ NormParams p) {
  __shared__ RowSums sums;
  depend_release();
  depend_wait();
  using XT = typename Number<X>::type;
  using RT = typename Number<R>::type;
  const CarryGdnNormArgs& a = p.a;
  const int lane = threadIdx.x % 32, groups = (a.W + kGroup - 1) / kGroup, run0 = threadIdx.x / 32 * C;
  const int first = run0 * kGroup + lane, left = a.W - first;      // columns from this lane's first on
  const bool whole = (run0 + C) * kGroup <= a.W;
  // Where a row's numbers leave the registers for it, the next row's are asked for while it is reduced, and the weights stay.
  constexpr bool kAhead = C <= 2;
  XT u[C][4];
  RT v[C][4];
  float weights[kAhead ? C : 1][4];
  auto fetch = [&](long long row) {
    auto get = [&](auto w) {
      constexpr bool kWhole = decltype(w)::value;
      const XT* x = static_cast<const XT*>(a.x) + row * a.stride_x + first;
      const RT* r = static_cast<const RT*>(a.residual) + row * a.stride_residual + first;
#pragma unroll
      for (int i = 0; i < 4 * C; ++i) u[i / 4][i % 4] = kWhole || i * 32 < left ? x[i * 32] : XT(0);
      if (a.residual) {
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) v[i / 4][i % 4] = kWhole || i * 32 < left ? r[i * 32] : RT(0);
      }
    };
    if (row >= a.N) return;
    if (whole) get(std::true_type());
    else get(std::false_type());
  };
  if constexpr (kAhead) {
    fetch(blockIdx.x);
#pragma unroll
    for (int i = 0; i < 4 * C; ++i) weights[i / 4][i % 4] = i * 32 < left ? load_as_float(a.weight, first + i * 32, a.weight_dtype) : 0.0f;
  }
  int turn = 0;
  for (long long row = blockIdx.x; row < a.N; row += gridDim.x, turn ^= 1) {
    float2 t[C][2], ss = make_float2(0.0f, 0.0f);
    float large = 0.0f, top[C], all = 0.0f;
    auto sum_up = [&] {
#pragma unroll
      for (int i = 0; i < 2 * C; ++i) {
        t[i / 2][i % 2] = make_float2(value_of<X>(u[i / 2][i % 2 * 2]), value_of<X>(u[i / 2][i % 2 * 2 + 1]));
        if (a.residual)
          t[i / 2][i % 2] = add2(t[i / 2][i % 2], make_float2(value_of<R>(v[i / 2][i % 2 * 2]), value_of<R>(v[i / 2][i % 2 * 2 + 1])));
      }
    };
    if constexpr (kAhead) {
      sum_up();
      fetch(row + gridDim.x);
    }
    auto enter = [&](auto w) {
      constexpr bool kWhole = decltype(w)::value;
      RT* out = static_cast<RT*>(a.residual_out) + row * a.stride_residual_out + first;
      auto there = [&](int at) { return kWhole || at < left; };
      if constexpr (!kAhead) {
        const XT* x = static_cast<const XT*>(a.x) + row * a.stride_x + first;
        const RT* r = static_cast<const RT*>(a.residual) + row * a.stride_residual + first;
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) u[i / 4][i % 4] = there(i * 32) ? x[i * 32] : XT(0);
        if (a.residual) {
#pragma unroll
          for (int i = 0; i < 4 * C; ++i) v[i / 4][i % 4] = there(i * 32) ? r[i * 32] : RT(0);
        }
        sum_up();
      }
      if (a.residual_out) {
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) {
          RT low, high;
          round_two<R>(t[i / 2][i % 2], low, high);
          if (there(i * 64)) out[i * 64] = low;
          if (there(i * 64 + 32)) out[i * 64 + 32] = high;
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j) add_squares(t[j], ss, large);
      auto weigh_all = [&](auto tag) {
        constexpr int T = decltype(tag)::value;
        const typename Number<T>::type* weight = static_cast<const typename Number<T>::type*>(a.weight) + first;
#pragma unroll
        for (int i = 0; i < 2 * C; ++i)
          t[i / 2][i % 2] = mul2(t[i / 2][i % 2], make_float2(there(i * 64) ? value_of<T>(weight[i * 64]) : 0.0f,
                                                              there(i * 64 + 32) ? value_of<T>(weight[i * 64 + 32]) : 0.0f));
      };
      if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) t[i / 2][i % 2] = mul2(t[i / 2][i % 2], make_float2(weights[i / 2][i % 2 * 2], weights[i / 2][i % 2 * 2 + 1]));
      } else if (a.weight_dtype == CARRY_BF16) weigh_all(std::integral_constant<int, CARRY_BF16>());
      else if (a.weight_dtype == CARRY_F16) weigh_all(std::integral_constant<int, CARRY_F16>());
      else weigh_all(std::integral_constant<int, CARRY_F32>());
    };
    if (whole) enter(std::true_type());
    else enter(std::false_type());
#pragma unroll
    for (int j = 0; j < C; ++j) {
      top[j] = fmaxf(fmaxf(fabsf(t[j][0].x), fabsf(t[j][0].y)), fmaxf(fabsf(t[j][1].x), fabsf(t[j][1].y)));
      all = fmaxf(all, top[j]);
    }
    const RowScale s = reduce_row(p, sums, turn, ss.x + ss.y, large, all);
    float by = 0.0f;
    if (a.group == 0) {
      const float scale = scale_of(s, s.top, by);
      if (threadIdx.x == 0) a.scale[row] = scale;
    }
    auto leave = [&](auto w) {
      constexpr bool kWhole = decltype(w)::value;
      uint8_t* codes = a.codes + row * a.stride_codes + first;
      auto there = [&](int at) { return kWhole || at < left; };
#pragma unroll
      for (int i = 0; i < 2 * C; ++i) {
        if (a.group && i % 2 == 0) {
          const float scale = scale_of(s, __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top[i / 2]))), by);
          if (lane == 0 && there(i * 64)) a.scale[row * groups + run0 + i / 2] = scale;
        }
        const uint32_t c = __nv_cvt_float2_to_fp8x2(mul2(t[i / 2][i % 2], make_float2(by, by)), __NV_SATFINITE, __NV_E4M3);
        if (there(i * 64)) codes[i * 64] = static_cast<uint8_t>(c);
        if (there(i * 64 + 32)) codes[i * 64 + 32] = static_cast<uint8_t>(c >> 8);
      }
    };
    if (whole) leave(std::true_type());
    else leave(std::false_type());
  }
}

template <class K>
int launch_rows(K kernel, const NormParams& p, int c, cudaStream_t stream) {
  const int chunks = (p.a.W + 7) / 8;
  const unsigned threads = (chunks + 32 * c - 1) / (32 * c) * 32;
  const long long resident = (long long)sm_count() * (max_threads(c) * min_ctas(c) / threads);
  return launch_dependent(kernel, dim3((unsigned)(p.a.N < resident ? p.a.N : resident)), threads, 0, stream, p);
}
template <int X, int R>
int launch_typed(const NormParams& p, cudaStream_t stream) {
  if (p.a.W <= 1024) return launch_rows(norm_kernel<1, X, R>, p, 1, stream);
  if (p.a.W <= 8192) return launch_rows(norm_kernel<2, X, R>, p, 2, stream);
  if (p.a.W <= 16384) return launch_rows(norm_kernel<4, X, R>, p, 4, stream);
  return launch_rows(norm_kernel<8, X, R>, p, 8, stream);
}
template <int C, int X, int R>
int launch_any(const NormParams& p, cudaStream_t stream) {
  const int runs = (p.a.W + kGroup - 1) / kGroup, warps = (runs + C - 1) / C;
  const long long resident = (long long)sm_count() * (16 * any_ctas(C) / warps);
  return launch_dependent(norm_any_kernel<C, X, R>, dim3((unsigned)(p.a.N < resident ? p.a.N : resident)), warps * 32, 0, stream, p);
}
template <int X, int R>
int launch_any(const NormParams& p, cudaStream_t stream) {
  // A row of 256 is a warp or two, which would wait for memory row by row (220 us for 2^26 numbers; 175 ahead of it); few rows
  // have all warps at work, and the weights on their way with the rest (one of 4097 3.4 us, 4.2 the other way).
  if (p.a.W <= 256 || (p.a.W <= 2048 && p.a.N <= sm_count())) return launch_any<1, X, R>(p, stream);
  if (p.a.W <= 4096 && p.a.N <= sm_count()) return launch_any<2, X, R>(p, stream);
  if (p.a.W <= 8192) return launch_any<4, X, R>(p, stream);
  return p.a.W <= 16384 ? launch_any<8, X, R>(p, stream) : launch_any<16, X, R>(p, stream);
}
template <int X>
int launch_any(const NormParams& p, cudaStream_t stream) {
  if (p.a.residual_dtype == CARRY_F32) return launch_any<X, CARRY_F32>(p, stream);
  return p.a.residual_dtype == CARRY_BF16 ? launch_any<X, CARRY_BF16>(p, stream) : launch_any<X, CARRY_F16>(p, stream);
}
int launch_any(const NormParams& p, cudaStream_t stream) {
  if (p.a.x_dtype == CARRY_F32) return launch_any<CARRY_F32>(p, stream);
  return p.a.x_dtype == CARRY_BF16 ? launch_any<CARRY_BF16>(p, stream) : launch_any<CARRY_F16>(p, stream);
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
  // the residual stream has x's type or is fp32; other pairs go a number at a time
  const int xd = a.x_dtype, rd = a.residual_dtype;
  if (vec && xd == CARRY_BF16 && rd == CARRY_BF16) return launch_typed<CARRY_BF16, CARRY_BF16>(p, stream);
  if (vec && xd == CARRY_F16 && rd == CARRY_F16) return launch_typed<CARRY_F16, CARRY_F16>(p, stream);
  // fp32 rows fill whole lines a number to a lane as well, and hold fewer registers so: 16384 rows of 4096 144 us, eight
  // numbers to a lane 172.  Few rows wait for one trip to memory less the other way (200 of 4096 3.5 us, 5.0).
  if (vec && xd == CARRY_F32 && rd == CARRY_F32 && (a.W <= 256 || a.N <= 4 * sm_count())) return launch_typed<CARRY_F32, CARRY_F32>(p, stream);
  if (vec && xd == CARRY_BF16 && rd == CARRY_F32) return launch_typed<CARRY_BF16, CARRY_F32>(p, stream);
  if (vec && xd == CARRY_F16 && rd == CARRY_F32) return launch_typed<CARRY_F16, CARRY_F32>(p, stream);
  return launch_any(p, stream);
}

}  // namespace carry
