// RMS norm of every query and key head and the rotation by the token's position, in one pass, in front of the key/value
// cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * (weight + weight_offset);   (y1, y2) -> (y1 cos - y2 sin, y2 cos + y1 sin)
//
// over pairs of the first `rotary` numbers: neighbours, or number i with i + rotary / 2.  Frequency i takes its angle from the
// table's row of the token's position on the frequency's axis.
//
// A lane has both numbers of its pairs: four neighbouring numbers and the four that are half the rotated width further on
// (or the four next to them, where pairs are neighbours or nothing is rotated), so that a row is read once, its sum is a few
// shuffles, and nothing is exchanged for the rotation.  A warp keeps its token's angles and walks over the token's heads, two rows of 128
// or four of 64 at a time: the table is read once a token and not once a head.  Few tokens are spread over more warps.
#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr int kThreads = 128, kMaxAxes = 4;

struct Params {
  CarryGdnRotateArgs a;
  int parts;                      // warps to a token
  float inv_width;
  int ends[kMaxAxes];             // first frequency beyond each axis
};

template <int DTYPE, int VE>
__device__ __forceinline__ void load_numbers(const void* base, long long at, float (&x)[VE]) {
  if constexpr (VE == 1) {
    x[0] = load_as_float(base, at, DTYPE);
  } else if constexpr (DTYPE == CARRY_F32) {
    const float4 u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(base) + at);
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (DTYPE == CARRY_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
}
template <int DTYPE, int VE>
__device__ __forceinline__ void store_numbers(void* base, long long at, const float (&x)[VE]) {
  if constexpr (VE == 1) {
    store_from_float(base, at, DTYPE, x[0]);
  } else if constexpr (DTYPE == CARRY_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + at) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (DTYPE == CARRY_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(base) + at) = make_uint2(w[0], w[1]);
  }
}

template <int LANES>
__device__ __forceinline__ float sum_over(float x) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d /= 2) x += __shfl_xor_sync(~0u, x, d);
  return x;
}

// LANES to a row, each with UNITS times two runs of VE numbers.  VE is 4, or 1 where widths, strides or addresses are off the grid of
// four numbers.
template <int DTYPE, int VE, int LANES, int UNITS>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = 32 / LANES;               // of a warp, at a time
  const CarryGdnRotateArgs& a = p.a;
  depend_release();
  depend_wait();
  const long long item = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  const int token = (int)(item / p.parts), part = (int)(item % p.parts);
  if (token >= a.N) return;
  const int lane = threadIdx.x % LANES, group = threadIdx.x % 32 / LANES, half = a.rotary / 2, units = a.D / (2 * VE), turned = half / VE;

  // the token's place on each axis; one without a place is left alone
  long long place[kMaxAxes];
  bool there = true, bad = false;
#pragma unroll
  for (int i = 0; i < kMaxAxes; ++i) {
    place[i] = 0;
    if (i >= a.axes) continue;
    const long long at = i * a.stride_positions + token;
    place[i] = a.positions_64 ? reinterpret_cast<const long long*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
    bad = bad || place[i] >= a.table_rows;
    there = there && place[i] >= 0 && place[i] < a.table_rows;
  }
  if (bad && a.status && part == 0 && threadIdx.x % 32 == 0) atomicOr(a.status, CARRY_GDN_STATUS_BAD_RANGE);
  if (!there) return;

  int first[UNITS], second[UNITS];                // where this lane's runs begin
  float cosine[UNITS][VE], sine[UNITS][VE];       // of its pairs; 1 and 0 where nothing is turned
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int unit = lane + u * LANES;
    const bool turns = unit < turned;
    const bool apart = turns && !a.interleaved;
    first[u] = apart ? unit * VE : unit * 2 * VE;
    second[u] = apart ? half + unit * VE : unit * 2 * VE + VE;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      cosine[u][e] = 1.0f;
      sine[u][e] = 0.0f;
      if (!turns) continue;
      const int f = unit * VE + e;
      long long row = place[0];
#pragma unroll
      for (int i = 1; i < kMaxAxes; ++i)
        if (i < a.axes && f >= p.ends[i - 1]) row = place[i];
      cosine[u][e] = load_as_float(a.cos_sin, row * a.stride_table + f, a.table_dtype);
      sine[u][e] = load_as_float(a.cos_sin, row * a.stride_table + half + f, a.table_dtype);
    }
  }

#pragma unroll
  for (int which = 0; which < 2; ++which) {       // queries, then keys
    const void* in = which ? a.k : a.q;
    void* out = which ? a.k_out : a.q_out;
    const void* weight = which ? a.k_weight : a.q_weight;
    const int heads = which ? a.HK : a.HQ, each = (heads + p.parts - 1) / p.parts, from = part * each, to = min(from + each, heads);
    const long long in_tok = which ? a.stride_k_tok : a.stride_q_tok, in_head = which ? a.stride_k_head : a.stride_q_head;
    const long long out_tok = which ? a.stride_k_out_tok : a.stride_q_out_tok, out_head = which ? a.stride_k_out_head : a.stride_q_out_head;
    if (from >= to) continue;
    float w[UNITS][2][VE];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (lane + u * LANES >= units) continue;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        w[u][0][e] = load_as_float(weight, first[u] + e, a.weight_dtype) + a.weight_offset;
        w[u][1][e] = load_as_float(weight, second[u] + e, a.weight_dtype) + a.weight_offset;
      }
    }
#pragma unroll 4
    for (int h0 = from; h0 < to; h0 += kRows) {
      const int h = h0 + group;
      const bool mine = h < to;
      float x[UNITS][2][VE], sum = 0.0f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[u][0][e] = x[u][1][e] = 0.0f;
        if (!mine || lane + u * LANES >= units) continue;
        const long long at = token * in_tok + h * in_head;
        load_numbers<DTYPE, VE>(in, at + first[u], x[u][0]);
        load_numbers<DTYPE, VE>(in, at + second[u], x[u][1]);
#pragma unroll
        for (int e = 0; e < VE; ++e) sum = fmaf(x[u][1][e], x[u][1][e], fmaf(x[u][0][e], x[u][0][e], sum));
      }
      sum = sum_over<LANES>(sum);
      float by = rsqrtf(fmaf(sum, p.inv_width, a.eps)), unit = 1.0f;
      if (__any_sync(~0u, sum == INFINITY)) {
        // squares beyond fp32: once more, in units of 2^100 (an infinity among the numbers makes the row NaN)
        float less = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float s = x[u][0][e] * 0x1p-100f, t = x[u][1][e] * 0x1p-100f;
            less = fmaf(t, t, fmaf(s, s, less));
          }
        less = sum_over<LANES>(less);
        if (sum == INFINITY) {
          by = less == INFINITY ? NAN : rsqrtf(less * p.inv_width);
          unit = 0x1p-100f;
        }
      }
      if (!mine) continue;
      const long long to_at = token * out_tok + h * out_head;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        if (lane + u * LANES >= units) continue;
        float y[2][VE], z[2][VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          y[0][e] = x[u][0][e] * unit * by * w[u][0][e];
          y[1][e] = x[u][1][e] * unit * by * w[u][1][e];
        }
        if (lane + u * LANES >= turned) {
#pragma unroll
          for (int e = 0; e < VE; ++e) { z[0][e] = y[0][e]; z[1][e] = y[1][e]; }
        } else if (a.interleaved && VE > 1) {     // the run's numbers 2i and 2i + 1 are pair i, over both runs
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float one = y[2 * e / VE][2 * e % VE], two = y[2 * e / VE][(2 * e + 1) % VE];
            z[2 * e / VE][2 * e % VE] = one * cosine[u][e] - two * sine[u][e];
            z[2 * e / VE][(2 * e + 1) % VE] = two * cosine[u][e] + one * sine[u][e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            z[0][e] = y[0][e] * cosine[u][e] - y[1][e] * sine[u][e];
            z[1][e] = y[1][e] * cosine[u][e] + y[0][e] * sine[u][e];
          }
        }
        store_numbers<DTYPE, VE>(out, to_at + first[u], z[0]);
        store_numbers<DTYPE, VE>(out, to_at + second[u], z[1]);
      }
    }
  }
}

template <int DTYPE, int VE, int LANES, int UNITS>
int launch(Params p, cudaStream_t stream) {
  // warps to a token: enough for twelve on a processor, a row at a time at least
  const int most = (p.a.HQ + 32 / LANES - 1) / (32 / LANES);
  const long long wanted = (12LL * sm_count() + p.a.N - 1) / p.a.N;
  p.parts = (int)(wanted < most ? wanted : most);
  if (p.parts < 1) p.parts = 1;
  const long long ctas = ((long long)p.a.N * p.parts + kThreads / 32 - 1) / (kThreads / 32);
  if (ctas > 0x7fffffff) return CARRY_GDN_ERR_TOO_LARGE;
  return launch_dependent(rotate_kernel<DTYPE, VE, LANES, UNITS>, dim3((unsigned)ctas), kThreads, 0, stream, p);
}

template <int DTYPE>
int launch_width(const Params& p, cudaStream_t stream) {
  const CarryGdnRotateArgs& a = p.a;
  constexpr int kSize = DTYPE == CARRY_F32 ? 4 : 2;
  bool grid = a.D % 8 == 0 && a.rotary % 8 == 0;
  for (const void* t : {a.q, a.k, (const void*)a.q_out, (const void*)a.k_out}) grid = grid && reinterpret_cast<uintptr_t>(t) % (4 * kSize) == 0;
  for (int64_t s : {a.stride_q_tok, a.stride_q_head, a.stride_k_tok, a.stride_k_head, a.stride_q_out_tok, a.stride_q_out_head, a.stride_k_out_tok,
                    a.stride_k_out_head})
    grid = grid && s % 4 == 0;
  if (!grid) return launch<DTYPE, 1, 32, 8>(p, stream);
  if (a.D <= 64) return launch<DTYPE, 4, 8, 1>(p, stream);
  if (a.D <= 128) return launch<DTYPE, 4, 16, 1>(p, stream);
  if (a.D <= 256) return launch<DTYPE, 4, 32, 1>(p, stream);
  return launch<DTYPE, 4, 32, 2>(p, stream);
}

}  // namespace

int launch_rotate(const CarryGdnRotateArgs& a, cudaStream_t stream) {
  Params p = {a, 1, 1.0f / a.D, {}};
  for (int i = 0, end = 0; i < kMaxAxes; ++i) p.ends[i] = end += i < a.axes ? a.sections[i] : 0;
  return a.dtype == CARRY_F32 ? launch_width<CARRY_F32>(p, stream)
         : a.dtype == CARRY_BF16 ? launch_width<CARRY_BF16>(p, stream) : launch_width<CARRY_F16>(p, stream);
}

}  // namespace carry
