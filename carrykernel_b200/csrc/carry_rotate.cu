// RMS norm of every query and key head and the rotation by the token's position, in one pass, in front of the key/value
// cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * (weight + weight_offset);   (y1, y2) -> (y1 cos - y2 sin, y2 cos + y1 sin)
//
// over pairs of the first `rotary` numbers: neighbours, or number i with i + rotary / 2.  Frequency i takes its angle from the
// table's row of the token's position on the frequency's axis.
//
// A lane has both numbers of its pairs: a run of four or eight neighbouring numbers and the run that is half the rotated width further on
// (or the one next to it, where pairs are neighbours or nothing is rotated), so that a row is read once, its sum is a few
// shuffles, and nothing is exchanged for the rotation.  A warp keeps its token's angles and walks over the token's heads, four rows of 128
// or eight of 64 at a time: the table is read once a token and not once a head.  Few tokens are spread over more warps.
//
// What bounds it: memory, behind it instructions (13 for a number; two numbers to one where the arithmetic allows).  16384 tokens of
// 32 and 8 heads of 128: 62 us in bf16, 85 % of a plain copy's rate (68 with eight rows at a time and none ahead), 106 in fp32, 96 %.  One token: 3.6 us,
// which is the host's call.
#include <type_traits>

#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr int kThreads = 128, kMaxAxes = 4;

struct Params {
  CarryGdnRotateArgs a;
  int parts;                      // warps to a token
  float inv_width;
  int runs_whole, table_whole, weights_whole;     // the runs' frequencies are of one axis; tables and weights can be read a run at a time
  int ends[kMaxAxes];             // first frequency beyond each axis
};

// VE numbers as they lie in memory, and as fp32
template <int DTYPE, int VE>
struct Run {
  typename std::conditional<VE == 1, float, typename std::conditional<DTYPE == CARRY_F32, float4, typename std::conditional<VE == 8, uint4, uint2>::type>::type>::type u;
};
template <int DTYPE, int VE>
__device__ __forceinline__ Run<DTYPE, VE> load_run(const void* base, long long at) {
  Run<DTYPE, VE> r;
  if constexpr (VE == 1) r.u = load_as_float(base, at, DTYPE);
  else if constexpr (DTYPE == CARRY_F32) r.u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
  else r.u = *reinterpret_cast<const decltype(r.u)*>(reinterpret_cast<const uint16_t*>(base) + at);
  return r;
}
template <int DTYPE, int VE>
__device__ __forceinline__ void numbers_of(const Run<DTYPE, VE>& r, float (&x)[VE]) {
  if constexpr (VE == 1) {
    x[0] = r.u;
  } else if constexpr (DTYPE == CARRY_F32) {
    x[0] = r.u.x; x[1] = r.u.y; x[2] = r.u.z; x[3] = r.u.w;
  } else {
    uint32_t w[VE / 2];
    memcpy(w, &r.u, sizeof(w));
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
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
    uint32_t w[VE / 2];
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      if constexpr (DTYPE == CARRY_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    if constexpr (VE == 8) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(base) + at) = make_uint2(w[0], w[1]);
  }
}

// VE numbers of a table or a weight, whose type is the call's; `whole`: on the grid of VE numbers
template <int VE>
__device__ __forceinline__ void load_factors(const void* base, long long at, int dtype, bool whole, float (&x)[VE]) {
  if (VE == 1 || !whole) {
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = load_as_float(base, at + e, dtype);
  } else if (dtype == CARRY_F32) {
#pragma unroll
    for (int e = 0; e < VE; e += 4) {
      const Run<CARRY_F32, 4> r = load_run<CARRY_F32, 4>(base, at + e);
      x[e] = r.u.x; x[e + 1] = r.u.y; x[e + 2] = r.u.z; x[e + 3] = r.u.w;
    }
  } else if (dtype == CARRY_BF16) {
    numbers_of<CARRY_BF16, VE>(load_run<CARRY_BF16, VE>(base, at), x);
  } else {
    numbers_of<CARRY_F16, VE>(load_run<CARRY_F16, VE>(base, at), x);
  }
}

// two numbers to an instruction, where a run has them
template <int VE, class Two, class One>
__device__ __forceinline__ void over_run(Two two, One one) {
  if constexpr (VE == 1) {
    one(0);
  } else {
#pragma unroll
    for (int e = 0; e < VE; e += 2) two(e);
  }
}
template <int VE>
__device__ __forceinline__ float2& pair(float (&x)[VE], int e) { return *reinterpret_cast<float2*>(&x[e]); }
template <int VE>
__device__ __forceinline__ float2 pair(const float (&x)[VE], int e) { return make_float2(x[e], x[e + 1]); }

template <int LANES>
__device__ __forceinline__ float sum_over(float x) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d /= 2) x += __shfl_xor_sync(~0u, x, d);
  return x;
}

// LANES to a row, each with UNITS times two runs of VE numbers: of 16 bytes, of four numbers or of one, as widths, strides and addresses allow.
template <int DTYPE, int VE, int LANES, int UNITS>
__global__ void __launch_bounds__(kThreads, VE == 8 ? 7 : VE == 1 || UNITS > 1 ? 1 : DTYPE == CARRY_F32 ? 5 : 6) rotate_kernel(const __grid_constant__ Params p) {
  // 16-bit rows: a row's registers take the next one as soon as its numbers have been unpacked, which leaves room for 24 to 28 warps on a
  // processor (62 us for the tokens above; with four times as many rows under way and 20 warps 65 to 68).  fp32 rows are as many registers as
  // their numbers, and come four at a time, for 20 warps (106 us; one ahead and 24 warps 112).
  constexpr bool kAhead = VE > 1 && DTYPE != CARRY_F32;
  constexpr int kRows = 32 / LANES, kBatch = VE > 1 && !kAhead ? 4 / UNITS : 1;    // rows of a warp at a time; how many times
  const CarryGdnRotateArgs& a = p.a;
  depend_release();
  depend_wait();
  const long long item = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  const int token = (int)item, part = blockIdx.y;
  if (item >= a.N) return;
  const int lane = threadIdx.x % LANES, group = threadIdx.x % 32 / LANES, half = a.rotary / 2, units = a.D / (2 * VE), turned = half / VE;

  int first[UNITS], second[UNITS];                // where this lane's runs begin
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int unit = lane + u * LANES;
    const bool apart = unit < turned && !a.interleaved;
    first[u] = apart ? unit * VE : unit * 2 * VE;
    second[u] = apart ? half + unit * VE : unit * 2 * VE + VE;
  }
  // the warp's share of the heads, and a batch of rows under way; the first one does not wait for the angles
  struct Heads {
    const void *in, *weight;
    void* out;
    int from, to;
    long long in_tok, in_head, out_tok, out_head;
  };
  const int each_q = (a.HQ + p.parts - 1) / p.parts, each_k = (a.HK + p.parts - 1) / p.parts;
  const Heads side[2] = {{a.q, a.q_weight, a.q_out, part * each_q, min((part + 1) * each_q, a.HQ), a.stride_q_tok, a.stride_q_head, a.stride_q_out_tok, a.stride_q_out_head},
                         {a.k, a.k_weight, a.k_out, part * each_k, min((part + 1) * each_k, a.HK), a.stride_k_tok, a.stride_k_head, a.stride_k_out_tok, a.stride_k_out_head}};
  Run<DTYPE, VE> rows[kBatch][UNITS][2];
  auto bring = [&](const Heads& s, int h, Run<DTYPE, VE> (&to)[UNITS][2]) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (h >= s.to || lane + u * LANES >= units) continue;
      const long long at = token * s.in_tok + h * s.in_head;
      to[u][0] = load_run<DTYPE, VE>(s.in, at + first[u]);
      to[u][1] = load_run<DTYPE, VE>(s.in, at + second[u]);
    }
  };
#pragma unroll
  for (int n = 0; n < kBatch; ++n) {
    if (!kAhead || side[0].from < side[0].to) bring(side[0], side[0].from + n * kRows + group, rows[n]);
    else bring(side[1], side[1].from + group, rows[n]);
  }

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

  alignas(8) float cosine[UNITS][VE], sine[UNITS][VE];       // of its pairs; 1 and 0 where nothing is turned
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int unit = lane + u * LANES;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      cosine[u][e] = 1.0f;
      sine[u][e] = 0.0f;
    }
    if (unit >= turned) continue;
    auto row_of = [&](int f) {
      long long row = place[0];
#pragma unroll
      for (int i = 1; i < kMaxAxes; ++i)
        if (i < a.axes && f >= p.ends[i - 1]) row = place[i];
      return row * a.stride_table;
    };
    if (p.runs_whole) {                           // a run's frequencies are of one axis
      const long long at = row_of(unit * VE) + unit * VE;
      load_factors<VE>(a.cos_sin, at, a.table_dtype, p.table_whole, cosine[u]);
      load_factors<VE>(a.cos_sin, at + half, a.table_dtype, p.table_whole, sine[u]);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const int f = unit * VE + e;
        const long long at = row_of(f) + f;
        cosine[u][e] = load_as_float(a.cos_sin, at, a.table_dtype);
        sine[u][e] = load_as_float(a.cos_sin, at + half, a.table_dtype);
      }
    }
  }

#pragma unroll
  for (int which = 0; which < 2; ++which) {       // queries, then keys
    const Heads& s = side[which];
    if (s.from >= s.to) continue;
    alignas(8) float w[UNITS][2][VE];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (lane + u * LANES >= units) continue;
      load_factors<VE>(s.weight, first[u], a.weight_dtype, p.weights_whole, w[u][0]);
      load_factors<VE>(s.weight, second[u], a.weight_dtype, p.weights_whole, w[u][1]);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        w[u][0][e] += a.weight_offset;
        w[u][1][e] += a.weight_offset;
      }
    }
    for (int h0 = s.from; h0 < s.to; h0 += kRows * kBatch) {
      if (!kAhead && (which > 0 || h0 > s.from)) {
#pragma unroll
        for (int n = 0; n < kBatch; ++n) bring(s, h0 + n * kRows + group, rows[n]);
      }
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int h = h0 + n * kRows + group;
        const bool mine = h < s.to;
        alignas(8) float x[UNITS][2][VE];
        float sum = 0.0f;
        float2 sums = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          numbers_of<DTYPE, VE>(rows[n][u][0], x[u][0]);
          numbers_of<DTYPE, VE>(rows[n][u][1], x[u][1]);
        }
        if (kAhead) {                             // of the same heads, or the keys' first one
          if (h0 + kRows < s.to) bring(s, h0 + kRows + group, rows[n]);
          else if (which == 0) bring(side[1], side[1].from + group, rows[n]);
        }
        if (h0 + n * kRows >= s.to) break;        // the same for all lanes
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          if (!mine || lane + u * LANES >= units) continue;
          over_run<VE>([&](int e) { sums = fma2(pair(x[u][1], e), pair(x[u][1], e), fma2(pair(x[u][0], e), pair(x[u][0], e), sums)); },
                       [&](int e) { sum = fmaf(x[u][1][e], x[u][1][e], fmaf(x[u][0][e], x[u][0][e], sum)); });
        }
        if (VE > 1) sum = sums.x + sums.y;
        sum = sum_over<LANES>(sum);
        float by = rsqrtf(fmaf(sum, p.inv_width, a.eps));
        if (__any_sync(~0u, sum == INFINITY)) {
          // squares beyond fp32: once more, in units of 2^100 (an infinity among the numbers makes the row NaN)
          float less = 0.0f;
#pragma unroll
          for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              if (lane + u * LANES >= units) continue;
              if (sum == INFINITY) {
                x[u][0][e] *= 0x1p-100f;
                x[u][1][e] *= 0x1p-100f;
              }
              less = fmaf(x[u][1][e], x[u][1][e], fmaf(x[u][0][e], x[u][0][e], less));
            }
          less = sum_over<LANES>(less);
          if (sum == INFINITY) by = less == INFINITY ? NAN : rsqrtf(less * p.inv_width);
        }
        if (!mine) continue;
        const long long to_at = token * s.out_tok + h * s.out_head;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          if (lane + u * LANES >= units) continue;
          alignas(8) float y[2][VE], z[2][VE];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            over_run<VE>([&](int e) { pair(y[i], e) = mul2(mul2(pair(x[u][i], e), make_float2(by, by)), pair(w[u][i], e)); },
                         [&](int e) { y[i][e] = x[u][i][e] * by * w[u][i][e]; });
          if (lane + u * LANES >= turned) {
#pragma unroll
            for (int e = 0; e < VE; ++e) { z[0][e] = y[0][e]; z[1][e] = y[1][e]; }
          } else if (a.interleaved && VE > 1) {   // the run's numbers 2i and 2i + 1 are pair i, over both runs
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const float one = y[2 * e / VE][2 * e % VE], two = y[2 * e / VE][(2 * e + 1) % VE];
              z[2 * e / VE][2 * e % VE] = one * cosine[u][e] - two * sine[u][e];
              z[2 * e / VE][(2 * e + 1) % VE] = two * cosine[u][e] + one * sine[u][e];
            }
          } else {
            over_run<VE>(
                [&](int e) {
                  const float2 c = pair(cosine[u], e), s = pair(sine[u], e), one = pair(y[0], e), two = pair(y[1], e);
                  pair(z[0], e) = sub2(mul2(one, c), mul2(two, s));
                  pair(z[1], e) = fma2(two, c, mul2(one, s));
                },
                [&](int e) {
                  z[0][e] = y[0][e] * cosine[u][e] - y[1][e] * sine[u][e];
                  z[1][e] = y[1][e] * cosine[u][e] + y[0][e] * sine[u][e];
                });
          }
          store_numbers<DTYPE, VE>(s.out, to_at + first[u], z[0]);
          store_numbers<DTYPE, VE>(s.out, to_at + second[u], z[1]);
        }
      }
    }
  }
}

template <int DTYPE, int VE, int LANES, int UNITS>
int launch(Params p, cudaStream_t stream) {
  const auto whole = [](const void* t, int64_t stride, int dtype) {
    const int n = dtype == CARRY_F32 && VE > 4 ? 4 : VE, size = dtype == CARRY_F32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(t) % (n * size) == 0 && stride % n == 0;
  };
  p.runs_whole = 1;
  for (int i = 0; i < p.a.axes; ++i) p.runs_whole = p.runs_whole && p.ends[i] % VE == 0;
  p.table_whole = whole(p.a.cos_sin, p.a.stride_table, p.a.table_dtype);
  p.weights_whole = whole(p.a.q_weight, 0, p.a.weight_dtype) && whole(p.a.k_weight, 0, p.a.weight_dtype);
  // warps to a token: enough for 64 on a processor, a row at a time at least
  const int most = (p.a.HQ + 32 / LANES - 1) / (32 / LANES);
  const long long wanted = (64LL * sm_count() + p.a.N - 1) / p.a.N;
  p.parts = (int)(wanted < most ? wanted : most);
  if (p.parts < 1) p.parts = 1;
  const long long ctas = ((long long)p.a.N + kThreads / 32 - 1) / (kThreads / 32);
  return launch_dependent(rotate_kernel<DTYPE, VE, LANES, UNITS>, dim3((unsigned)ctas, (unsigned)p.parts), kThreads, 0, stream, p);
}

template <int DTYPE>
int launch_width(const Params& p, cudaStream_t stream) {
  const CarryGdnRotateArgs& a = p.a;
  constexpr int kSize = DTYPE == CARRY_F32 ? 4 : 2;
  // runs of `n` numbers: 16 bytes, or 8 where widths, strides or addresses do not allow it
  auto fits = [&](int n) {
    bool yes = a.D % (2 * n) == 0 && a.rotary % (2 * n) == 0;
    for (const void* t : {a.q, a.k, (const void*)a.q_out, (const void*)a.k_out}) yes = yes && reinterpret_cast<uintptr_t>(t) % (n * kSize) == 0;
    for (int64_t s : {a.stride_q_tok, a.stride_q_head, a.stride_k_tok, a.stride_k_head, a.stride_q_out_tok, a.stride_q_out_head, a.stride_k_out_tok,
                      a.stride_k_out_head})
      yes = yes && s % n == 0;
    return yes;
  };
  if constexpr (kSize == 2) {
    if (fits(8)) {
      if (a.D <= 64) return launch<DTYPE, 8, 4, 1>(p, stream);
      if (a.D <= 128) return launch<DTYPE, 8, 8, 1>(p, stream);
      if (a.D <= 256) return launch<DTYPE, 8, 16, 1>(p, stream);
      return launch<DTYPE, 8, 32, 1>(p, stream);
    }
  }
  if (!fits(4)) return launch<DTYPE, 1, 32, 8>(p, stream);
  if (a.D <= 64) return launch<DTYPE, 4, 8, 1>(p, stream);
  if (a.D <= 128) return launch<DTYPE, 4, 16, 1>(p, stream);
  if (a.D <= 256) return launch<DTYPE, 4, 32, 1>(p, stream);
  return launch<DTYPE, 4, 32, 2>(p, stream);
}

}  // namespace

int launch_rotate(const CarryGdnRotateArgs& a, cudaStream_t stream) {
  Params p = {a, 1, 1.0f / a.D, 0, 0, 0, {}};
  for (int i = 0, end = 0; i < kMaxAxes; ++i) p.ends[i] = end += i < a.axes ? a.sections[i] : 0;
  return a.dtype == CARRY_F32 ? launch_width<CARRY_F32>(p, stream)
         : a.dtype == CARRY_BF16 ? launch_width<CARRY_BF16>(p, stream) : launch_width<CARRY_F16>(p, stream);
}

}  // namespace carry
