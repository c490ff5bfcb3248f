// Attention over the 8-bit key/value cache for few query rows of a request: one token, or some speculated ones.
//
// What a call reads is the cache, once.  The matrix products have 16 tokens (keys) or 16 columns (values) as the
// instruction's rows, and as its eight columns eight query rows: the query heads of a key/value head, so that the tokens
// are read once for all of them.  A warp has all query rows and every fourth run of 32 tokens, so that a code is converted
// once; its copies, its stages and its softmax are its own, and the warps meet only where a request ends.
//
// Two ways.  The tokens of all requests and heads are one line of tiles, cut evenly over the CTAs that fit the GPU, whatever
// the lengths are; where a cut falls inside a (request, head), pieces are joined by a second kernel.  Short contexts of few
// (request, head)s have a cluster each and no second kernel.
//
// What bounds it: 128 requests of 8192 tokens (8 heads of 128, 2.15 GB) take 350 to 400 us from box to box, 82 to 93 % of the copy
// rate; 64 of 1 to 8192 tokens 120 us, 4.6 TB/s, some 15 us of it the way in and out.  A run is about 700 instructions of a warp, half of them
// conversions and byte permutations at two cycles each; twelve warps an SM issue two instructions a cycle.  Tried and slower:
// e4m3 matrix instructions on unconverted keys (131 us for the 64 requests: twice the registers), runs of 64 tokens, two CTAs
// an SM with more stages (146).
#include <cooperative_groups.h>

#include "carry_kv_attention.cuh"

namespace carry {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kRun = 32, kLine = kRun * kWarps;   // tokens of a warp's step, and of a tile of the line

// What a CTA leaves for the joining kernel: at most one piece of a (request, head) that began in an earlier CTA (slot 0)
// and one that goes on in later ones (slot 1).
struct alignas(16) Piece {
  int first, rows, head, last;    // the request's first row and number of rows; last CTA with a piece of the same, or -1: none began here
};

template <int D>
struct RunStage {
  alignas(128) uint8_t k[kRun * D];
  uint8_t v[kRun * D];
  float ks[kRun / kGranule], vs[kRun / kGranule];
};
// CTAs of the decode kernel on an SM, by their registers, and stages of a warp, by the memory that this leaves.
__host__ __device__ constexpr int resident(int D, int NT, int PARTS) { return NT == 1 && PARTS == 1 ? (D == 128 ? 3 : 4) : 2; }
// Four leave the joining kernel some registers to wait in beside them: a call behind such a one starts when all its CTAs have
// (two requests of 8344 tokens, 32 heads over 4 of 64, one after another 11.5 us, 13.0 with 121 registers a thread).
__host__ __device__ constexpr int registers(int D, int NT, int PARTS) {
  return resident(D, NT, PARTS) == 4 ? 120 : resident(D, NT, PARTS) == 3 ? 168 : 255;
}
__host__ __device__ constexpr int stages(int D, int NT, int PARTS) { return D == 128 ? (resident(D, NT, PARTS) == 3 ? 2 : 3) : 3; }

template <int D, int NT, int PARTS>
struct DecodeShared {
  RunStage<D> stage[kWarps][stages(D, NT, PARTS)];
  float merge[NT * 8][D + 4];
  float top[kWarps][NT * 8], sum[kWarps][NT * 8];
};

__host__ __device__ constexpr long long slot_floats(int rows, int D) { return (long long)rows * (D + 2); }

__device__ __forceinline__ int tiles_of(const AttnParams& p, int b) {
  const long long cap = min((long long)p.a.cache.max_pages * p.a.cache.page, kMaxTokens);
  const int length = (int)min((long long)max(p.a.cache.lengths[b], 0), cap);
  return (length + kLine - 1) / kLine;
}

// Sum of x over the CTA, and over the threads before this one.
__device__ __forceinline__ long long block_scan(long long x, long long* scratch, long long& before) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  long long up = x;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long y = __shfl_up_sync(~0u, up, d);
    if (lane >= d) up += y;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = up;
  __syncthreads();
  long long total = 0;
  before = up - x;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  return total;
}

// A place on the line of tiles.
struct Cursor {
  int b, h, tile, tiles, length;
};
__device__ __forceinline__ void open_request(const AttnParams& p, Cursor& at) {
  while (at.b < p.a.rows.B && (at.tiles = tiles_of(p, at.b)) == 0) ++at.b;
  if (at.b < p.a.rows.B) at.length = kv_request(p.a.cache, p.a.rows, at.b, nullptr).length;
}
__device__ __forceinline__ void advance(const AttnParams& p, Cursor& at) {
  if (++at.tile < at.tiles) return;
  at.tile = 0;
  if (++at.h < p.a.cache.HKV) return;
  at.h = 0;
  ++at.b;
  open_request(p, at);
}

// Page ids of a warp's run of tokens, fetched a step ahead of its copies.
struct RunPages {
  int id[kRun / kGranule];
};
__device__ __forceinline__ RunPages fetch_run(const AttnParams& p, const Cursor& at) {
  RunPages r;
#pragma unroll
  for (int i = 0; i < kRun / kGranule; ++i)
    r.id[i] = page_id(p, at.b, at.tile * (kLine / kGranule) + threadIdx.x / 32 * (kRun / kGranule) + i, at.length);
  return r;
}

// The copies of a run.  Tokens at or beyond the request's length and tokens of padding pages are filled with zeros,
// whatever memory holds there.
template <int D>
__device__ __forceinline__ void load_run(const AttnParams& p, RunStage<D>& s, const Cursor& at, const RunPages& pages) {
  const CarryGdnKvCache& c = p.a.cache;
  constexpr int kChunks = D / 16, kCopies = kGranule * kChunks / 32;   // 16-byte copies of a granule, per lane
  const int lane = threadIdx.x % 32, first = at.tile * (kLine / kGranule) + threadIdx.x / 32 * (kRun / kGranule);
#pragma unroll
  for (int i = 0; i < kRun / kGranule; ++i) {
    const int granule = first + i, id = pages.id[i], left = id > 0 ? at.length - granule * kGranule : 0;
    const int in_page = granule - page_index(p, granule) * p.page_granules;
    const int off = (at.h * c.page + in_page * kGranule) * D + lane * 16;   // a page is below 2^31 bytes
    const uint8_t *k = c.k_codes + id * c.stride_k_page + off, *v = c.v_codes + id * c.stride_v_page + off;
    int to[kCopies];
#pragma unroll
    for (int x = 0; x < kCopies; ++x) to[x] = tile_at<D>(i * kGranule + lane / kChunks + x * (32 / kChunks), lane % kChunks);
    if (left >= kGranule) {
#pragma unroll
      for (int x = 0; x < kCopies; ++x) {
        __pipeline_memcpy_async(s.k + to[x], k + x * 512, 16);
        __pipeline_memcpy_async(s.v + to[x], v + x * 512, 16);
      }
    } else {
#pragma unroll
      for (int x = 0; x < kCopies; ++x) {
        const bool there = lane / kChunks + x * (32 / kChunks) < left;
        __pipeline_memcpy_async(s.k + to[x], there ? k + x * 512 : c.k_codes, 16, there ? 0 : 16);
        __pipeline_memcpy_async(s.v + to[x], there ? v + x * 512 : c.v_codes, 16, there ? 0 : 16);
      }
    }
    if (lane < 2) {
      const int block = at.h * (p.page_granules / p.block_granules) + divide(in_page, p.block_granules, p.block_shift);
      float* to_scale = lane == 0 ? &s.ks[i] : &s.vs[i];
      if (id > 0) __pipeline_memcpy_async(to_scale, lane == 0 ? c.k_scale + id * c.stride_ks_page + block : c.v_scale + id * c.stride_vs_page + block, 4);
      else *to_scale = lane == 0 ? kNoTokens : 0.0f;
    }
  }
}

// Query rows as the second operand: lane (g, c) has row 8 n + g, of every 64 columns the 16 from 16 c on.
template <int D, int NT, int PARTS>
struct Columns {
  uint32_t x[NT][PARTS][D / 16][2];
  float unit[NT][2];              // of rows 8 n + 2 c and 8 n + 2 c + 1: what a product counts in log2's scale; not negative
};
template <int D, int NT, int PARTS>
__device__ __forceinline__ void load_columns(const AttnParams& p, const KvRequest& r, int h, Columns<D, NT, PARTS>& q) {
  const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = 8 * n + g, i = token_of(p, row);
    const bool there = i < r.todo;
    const long long at = there ? row_place(p, r, h, row, i, p.a.stride_q_tok, p.a.stride_q_head) : 0;
    float x[D / 4];
    uint32_t top = 0;
    load_share<D, PARTS>(p, at, there, x);
#pragma unroll
    for (int e = 0; e < D / 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    top = max(top, __shfl_xor_sync(~0u, top, 2));
    const int e = up_exponent(top);
    const float up = copysignf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), p.a.scale);
    const float unit = fabsf(p.a.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    q.unit[n][0] = __shfl_sync(~0u, unit, c * 8);
    q.unit[n][1] = __shfl_sync(~0u, unit, c * 8 + 4);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
        float u = x[k * 4 + pair * 2] * up, v = x[k * 4 + pair * 2 + 1] * up;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t w = pack_half2(u, v);
          q.x[n][part][k][pair] = w;
          const float2 kept = unpack_half2(w);
          u -= kept.x;
          v -= kept.y;
        }
      }
  }
}

// Running softmax over a warp's tokens.  o: lane (g, c) has columns g D/8 + 2 m and + 1 of rows 8 n + 2 c and + 1.
template <int D, int NT>
struct Running {
  float o[NT][D / 16][4];
  float top[NT][2], sum[NT][2];   // the sums are this lane's share
  float up[NT][2];                // 2^15 over the unit that the row's outputs count in: o is that many times too large
  Scales scales;
  float limit;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int m = 0; m < D / 16; ++m) o[n][m][0] = o[n][m][1] = o[n][m][2] = o[n][m][3] = 0.0f;
      top[n][0] = top[n][1] = -INFINITY;
      sum[n][0] = sum[n][1] = 0.0f;
      up[n][0] = up[n][1] = kUpStart;
    }
    scales.most = INFINITY;
    limit = scales.limit(kUpStart);
  }
};

// A run of tokens.  `limit`: how many of the run's tokens rows 8 n + 2 c and + 1 see; `all`: every row of the warp sees
// every one that is there.
template <int D, int NT, int PARTS>
__device__ __forceinline__ void attend_run(const RunStage<D>& s, const Columns<D, NT, PARTS>& q, const int (&limit)[NT][2], bool all, Running<D, NT>& r) {
  const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  constexpr int kBlocks = kRun / kGranule;
  float score[kBlocks][NT][4] = {};               // tokens g (0, 1) and g + 8 (2, 3) of a block, rows 2c and 2c + 1
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const uint4 u = *reinterpret_cast<const uint4*>(s.k + tile_at<D>(b * kGranule + g, j * 4 + c));
      const uint4 v = *reinterpret_cast<const uint4*>(s.k + tile_at<D>(b * kGranule + g + 8, j * 4 + c));
      const uint32_t near[4] = {u.x, u.y, u.z, u.w}, far[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a[4];
        halves_of(near[k], a[0], a[2]);
        halves_of(far[k], a[1], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            mma_fp16(score[b][n], a, q.x[n][part][j * 4 + k][0], q.x[n][part][j * 4 + k][1]);
      }
    }
  float now[NT][2], count[kBlocks][NT][2];     // count: what a product of the block counts
  float vs_top = 0.0f;
#pragma unroll
  for (int n = 0; n < NT; ++n) now[n][0] = now[n][1] = -INFINITY;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const float ks = s.ks[b];
    vs_top = fmaxf(vs_top, s.vs[b]);
    if (!all || ks == kNoTokens) {
      const int t = ks == kNoTokens ? 1 << 30 : b * kGranule + g;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) score[b][n][i] = t + i / 2 * 8 < limit[n][i % 2] ? score[b][n][i] : -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        count[b][n][i] = fmaxf(q.unit[n][i] * ks, 0x1p-126f);
        now[n][i] = fmaxf(now[n][i], fmaxf(score[b][n][i], score[b][n][i + 2]) * count[b][n][i]);
      }
  }
  bool more = vs_top > r.limit;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 4; d < 32; d *= 2) now[n][i] = fmaxf(now[n][i], __shfl_xor_sync(~0u, now[n][i], d));
      more = more || now[n][i] > r.top[n][i];
    }
  if (__any_sync(~0u, more)) {
    float vs_low = vs_top, keep[NT][2];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) vs_low = fminf(vs_low, s.ks[b] == kNoTokens ? vs_top : s.vs[b]);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float high = fmaxf(now[n][i], r.top[n][i]);
        keep[n][i] = high == -INFINITY ? 1.0f : exp2_fast(r.top[n][i] - high);
        r.sum[n][i] *= keep[n][i];
        r.top[n][i] = high;
      }
    const bool fresh = r.scales.fresh();
    if (__builtin_expect(r.scales.alike(vs_top, vs_low), 1)) {
      if (fresh || vs_top > r.limit) {
        const float up = up_above(vs_top), less = rescale(r.up[0][0], up);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            r.up[n][i] = up;
            keep[n][i] *= less;
          }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float zero = r.top[n][i] == -INFINITY ? 0.0f : r.top[n][i], had = fresh ? 0.0f : up_of(r.up[n][i]) * keep[n][i];
          float met = 0.0f;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            float m = fmaxf(score[b][n][i], score[b][n][i + 2]) * count[b][n][i];
#pragma unroll
            for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
            met = fmaxf(met, exp2_fast(m - zero) * s.vs[b]);
          }
          r.up[n][i] = up_above(fmaxf(had, met));
          keep[n][i] = had * r.up[n][i] * 0x1p-15f;
        }
    }
    r.limit = r.scales.limit(r.up[0][0]);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) r.o[n][m][i] *= keep[n][i % 2];
  }
  float base[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) base[n][i] = r.top[n][i] == -INFINITY ? 0.0f : r.top[n][i];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const float vs = s.vs[b];
    uint32_t w[NT][PARTS][2];     // weights of tokens 2c, 2c + 1 and 2c + 8, 2c + 9, row 8 n + g
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float2 x = make_float2(exp2_fast(fmaf(score[b][n][half * 2], count[b][n][0], -base[n][0])),
                               exp2_fast(fmaf(score[b][n][half * 2 + 1], count[b][n][1], -base[n][1])));
        r.sum[n][0] += x.x;
        r.sum[n][1] += x.y;
        x = scaled(x, vs, make_float2(r.up[n][0], r.up[n][1]));
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t h = pack_half2(x.x, x.y);
          asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(w[n][part][half]) : "r"(h));
          const float2 kept = unpack_half2(h);
          x.x -= kept.x;
          x.y -= kept.y;
        }
      }
    constexpr int kWords = D / 32;                // this lane's columns of tokens 2c, 2c + 1, 2c + 8, 2c + 9
    uint32_t v[4][kWords];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = b * kGranule + 2 * c + i % 2 + i / 2 * 8;
      if constexpr (D == 128) {
        const uint4 u = *reinterpret_cast<const uint4*>(s.v + tile_at<D>(row, g));
        v[i][0] = u.x; v[i][1] = u.y; v[i][2] = u.z; v[i][3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(s.v + tile_at<D>(row, g / 2) + g % 2 * 8);
        v[i][0] = u.x; v[i][1] = u.y;
      }
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t a[4];
        halves_of(__byte_perm(v[0][k], v[1][k], e ? 0x7362 : 0x5140), a[0], a[1]);
        halves_of(__byte_perm(v[2][k], v[3][k], e ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int part = 0; part < PARTS; ++part) mma_fp16(r.o[n][k * 2 + e], a, w[n][part][0], w[n][part][1]);
      }
  }
}

// The warps' softmaxes into one: weights first, then the outputs in turn, normalised, in sh.merge.  top and sum are of rows
// 8 n + 2 c and + 1.
template <int D, int NT, int PARTS>
__device__ __forceinline__ void merge_warps(DecodeShared<D, NT, PARTS>& sh, Running<D, NT>& r, float (&top)[NT][2], float (&sum)[NT][2]) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, cc = lane % 4;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float share = r.sum[n][i];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) share += __shfl_xor_sync(~0u, share, d);
      if (g == 0) {
        sh.top[warp][8 * n + 2 * cc + i] = r.top[n][i];
        sh.sum[warp][8 * n + 2 * cc + i] = share;
      }
    }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 8 * n + 2 * cc + i;
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) m = fmaxf(m, sh.top[x][row]);
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) l += sh.sum[x][row] * exp2_fast(sh.top[x][row] - base);
      const float w = l == 0.0f ? 0.0f : __fdiv_rn(exp2_fast(r.top[n][i] - base), l), unit = up_of(r.up[n][i]) * 0x1p-15f;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        r.o[n][x][i] = r.o[n][x][i] * w * unit;
        r.o[n][x][i + 2] = r.o[n][x][i + 2] * w * unit;
      }
      top[n][i] = m;
      sum[n][i] = l;
    }
#pragma unroll
  for (int x = 0; x < kWarps; ++x) {
    if (x > 0) __syncthreads();
    if (x != warp) continue;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < D / 16; m += 2) {
          float4* cell = reinterpret_cast<float4*>(&sh.merge[8 * n + 2 * cc + i][g * (D / 8) + 2 * m]);
          float4 mine = make_float4(r.o[n][m][i], r.o[n][m][i + 2], r.o[n][m + 1][i], r.o[n][m + 1][i + 2]);
          if (x > 0) {
            const float4 had = *cell;
            mine.x += had.x; mine.y += had.y; mine.z += had.z; mine.w += had.w;
          }
          *cell = mine;
        }
  }
  __syncthreads();
}

// A (request, head) to a cluster of CL CTAs: one launch, where the line's way takes two.  For short contexts.  A CL-th of
// the columns is each CTA's to join: all warps of the cluster put what they have of it, normalised, into its shared memory, and
// one barrier later it is done.  (Joining the warps of a CTA first and reading the others' results afterwards took 2 us longer,
// of 7.6 for one token over 16.)
__host__ __device__ constexpr int pair_stages(int D) { return D == 128 ? 2 : 3; }       // two CTAs to an SM
template <int D, int NT, int PARTS, int CL>
struct PairShared {
  RunStage<D> stage[kWarps][pair_stages(D)];
  alignas(16) float o[CL * kWarps][NT * 8][D / CL];
  float top[CL * kWarps][NT * 8], sum[CL * kWarps][NT * 8];
};

template <int D, int NT, int PARTS, int CL>
__global__ void __launch_bounds__(kThreads, 2) kv_pair_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ __align__(128) uint8_t raw[];
  PairShared<D, NT, PARTS, CL>& sh = *reinterpret_cast<PairShared<D, NT, PARTS, CL>*>(raw);
  constexpr int kStages = pair_stages(D), kSources = CL * kWarps, kColumns = D / CL;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  depend_release();
  depend_wait();
  const CarryGdnKvCache& c = p.a.cache;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, cc = lane % 4;
  const int rank = blockIdx.x % CL, pair = blockIdx.x / CL;
  Cursor use;
  use.b = pair / c.HKV;
  use.h = pair % c.HKV;
  const KvRequest request = kv_request(c, p.a.rows, use.b, use.h == 0 && rank == 0 && threadIdx.x == 0 ? p.a.status : nullptr);
  use.length = request.length;
  use.tiles = (use.length + kLine - 1) / kLine;
  use.tile = rank;                                // tiles go round the cluster: neighbours read neighbouring pages
  Cursor load = use;
  RunPages pages = fetch_run(p, load);
  Columns<D, NT, PARTS> q;                        // while the page ids are on their way
  load_columns<D, NT, PARTS>(p, request, use.h, q);
  auto next_load = [&](int stage) {
    if (load.tile < load.tiles) {
      load_run<D>(p, sh.stage[warp][stage], load, pages);
      load.tile += CL;
      if (load.tile < load.tiles) pages = fetch_run(p, load);
    }
    __pipeline_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) next_load(s);
  Running<D, NT> r;
  r.clear();
  int stage = 0;
  for (; use.tile < use.tiles; use.tile += CL) {
    __pipeline_wait_prior(kStages - 2);
    __syncwarp();
    next_load(stage == 0 ? kStages - 1 : stage - 1);
    const int start = use.tile * kLine + warp * kRun;
    if (start < request.length) {
      int limit[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int x = token_of(p, 8 * n + 2 * cc + i);
          limit[n][i] = (x < request.todo ? request.length - request.count + x + 1 : 0) - start;
        }
      attend_run<D, NT, PARTS>(sh.stage[warp][stage], q, limit, start + kRun <= request.length - request.count + 1, r);
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  // lane (g, c) has the g-th eighth of the columns, of rows 8 n + 2 c and + 1
  const auto cluster = cooperative_groups::this_cluster();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");        // every CTA has started
  PairShared<D, NT, PARTS, CL>& theirs = *cluster.map_shared_rank(&sh, g * CL / 8);
  const int source = rank * kWarps + warp;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 8 * n + 2 * cc + i;
      float sum = r.sum[n][i];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(~0u, sum, d);
      theirs.top[source][row] = r.top[n][i];
      theirs.sum[source][row] = sum;
      const float w = sum == 0.0f ? 0.0f : __fdiv_rn(up_of(r.up[n][i]), sum) * 0x1p-15f;
      float4* to = reinterpret_cast<float4*>(theirs.o[source][row] + g % (8 / CL) * (D / 8));
#pragma unroll
      for (int m = 0; m < D / 16; m += 2)
        to[m / 2] = make_float4(r.o[n][m][i] * w, r.o[n][m][i + 2] * w, r.o[n][m + 1][i] * w, r.o[n][m + 1][i + 2] * w);
    }
  cluster.sync();
  for (int i = threadIdx.x; i < request.todo * p.group * kColumns; i += kThreads) {
    const int row = i / kColumns, col = i % kColumns;
    float top = -INFINITY, total = 0.0f, x = 0.0f;
#pragma unroll
    for (int n = 0; n < kSources; ++n) top = fmaxf(top, sh.top[n][row]);
    const float base = (top == -INFINITY ? 0.0f : top) + kJoinDown;
#pragma unroll 8
    for (int n = 0; n < kSources; ++n) {
      const float w = sh.sum[n][row] * exp2_fast(sh.top[n][row] - base);
      total += w;
      x = fmaf(w, sh.o[n][row][col], x);
    }
    store_from_float(p.a.out, row_place(p, request, use.h, row, token_of(p, row), p.a.stride_out_tok, p.a.stride_out_head) + rank * kColumns + col,
                     p.a.dtype, total == 0.0f ? 0.0f : __fdiv_rn(x, total));
  }
}

template <int D, int NT, int PARTS>
__global__ void __maxnreg__(registers(D, NT, PARTS)) kv_decode_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ __align__(128) uint8_t raw[];
  DecodeShared<D, NT, PARTS>& sh = *reinterpret_cast<DecodeShared<D, NT, PARTS>*>(raw);
  __shared__ long long scratch[kWarps];
  __shared__ int found[2];
  constexpr int kRows = NT * 8, kStages = stages(D, NT, PARTS);
  depend_release();
  depend_wait();
  const CarryGdnKvCache& c = p.a.cache;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, cc = lane % 4;
  Piece* pieces = reinterpret_cast<Piece*>(p.a.workspace);
  float* slots = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.a.workspace) + sizeof(Piece) * gridDim.x);

  // the line's length, and where on it this CTA begins
  long long total = 0, before;
  for (int b0 = 0; b0 < p.a.rows.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    total += block_scan(b < p.a.rows.B ? (long long)tiles_of(p, b) * c.HKV : 0, scratch, before);
  }
  const long long share = (total + gridDim.x - 1) / gridDim.x;
  const long long from = min(share * blockIdx.x, total), to = min(from + share, total);
  // requests without tokens have no tiles: their rows are zero
  for (int b = blockIdx.x; b < p.a.rows.B; b += gridDim.x) {
    const KvRequest q = kv_request(c, p.a.rows, b, threadIdx.x == 0 ? p.a.status : nullptr);
    if (q.length > 0) continue;
    for (int i = threadIdx.x; i < q.todo * p.a.HQ * D; i += kThreads)
      store_from_float(p.a.out, (q.first + i / (p.a.HQ * D)) * p.a.stride_out_tok + i / D % p.a.HQ * p.a.stride_out_head + i % D, p.a.dtype, 0.0f);
  }
  if (threadIdx.x == 0) pieces[blockIdx.x].last = -1;
  if (from == to) return;
  long long seen = 0;
  for (int b0 = 0; b0 < p.a.rows.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const long long mine = b < p.a.rows.B ? (long long)tiles_of(p, b) * c.HKV : 0;
    const long long all = p.a.rows.B <= kThreads ? total : block_scan(mine, scratch, before);   // else `before` is still right
    if (mine > 0 && from >= seen + before && from < seen + before + mine) {
      found[0] = b;
      found[1] = (int)(from - seen - before);
    }
    seen += all;
    if (from < seen) break;
  }
  __syncthreads();
  Cursor use;
  use.b = found[0];
  use.tiles = 1;
  open_request(p, use);
  use.h = found[1] / use.tiles;
  use.tile = found[1] % use.tiles;
  Cursor load = use;
  long long to_load = to - from;
  RunPages pages = fetch_run(p, load);
  auto next_load = [&](int stage) {
    if (to_load > 0) {
      load_run<D>(p, sh.stage[warp][stage], load, pages);
      advance(p, load);
      if (--to_load > 0) pages = fetch_run(p, load);
    }
    __pipeline_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) next_load(s);

  Columns<D, NT, PARTS> q;
  Running<D, NT> r;
  KvRequest request;
  bool begin = true;
  int first_tile = 0, stage = 0, sees[NT][2];     // tokens that rows 8 n + 2 c and + 1 see
  for (long long at = from; at < to; ++at) {
    if (begin) {
      request = kv_request(c, p.a.rows, use.b, nullptr);
      load_columns<D, NT, PARTS>(p, request, use.h, q);
      r.clear();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int x = token_of(p, 8 * n + 2 * cc + i);
          sees[n][i] = x < request.todo ? request.length - request.count + x + 1 : 0;
        }
      first_tile = use.tile;
      begin = false;
    }
    __pipeline_wait_prior(kStages - 2);
    __syncwarp();                                 // this run has landed, and every lane is done with the one before
    next_load(stage == 0 ? kStages - 1 : stage - 1);
    const int start = use.tile * kLine + warp * kRun;
    if (start < request.length) {
      int limit[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        limit[n][0] = sees[n][0] - start;
        limit[n][1] = sees[n][1] - start;
      }
      attend_run<D, NT, PARTS>(sh.stage[warp][stage], q, limit, start + kRun <= request.length - request.count + 1, r);
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
    const bool ends = use.tile + 1 == use.tiles;
    if (ends || at + 1 == to) {
      float top[NT][2], sum[NT][2];
      merge_warps(sh, r, top, sum);
      const bool whole = ends && first_tile == 0;
      float* slot = slots + (2 * blockIdx.x + (first_tile == 0)) * slot_floats(kRows, D);
      if (!whole && warp == 0 && g == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            slot[8 * n + 2 * cc + i] = top[n][i];
            slot[kRows + 8 * n + 2 * cc + i] = sum[n][i];
          }
      }
      for (int i = threadIdx.x; i < request.todo * p.group * (D / 8); i += kThreads) {
        const int row = i / (D / 8), col = i % (D / 8) * 8;
        alignas(16) float x[8];
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(&sh.merge[row][col]);
        *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(&sh.merge[row][col + 4]);
        if (whole) {
          store8(p.a.out, row_place(p, request, use.h, row, token_of(p, row), p.a.stride_out_tok, p.a.stride_out_head) + col,
                 p.a.dtype, x);
        } else {
          store8(slot, 2 * kRows + row * D + col, CARRY_F32, x);
        }
      }
      if (!ends && first_tile == 0 && threadIdx.x == 0) {
        // the rest of its tiles: the CTAs up to the one with its last tile
        const long long last = at + (use.tiles - 1 - use.tile);
        pieces[blockIdx.x] = {request.first, request.todo * p.group, use.h, (int)(last / share)};
      }
      __syncthreads();
      begin = true;
    }
    advance(p, use);
  }
}

// Pieces first, first + step, ... of the `count` of a (request, head) that began in CTA `cta` of the kernel above, for one
// row, by one warp.  Eight of them come in one trip to memory, with their weights.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kBatch = 8;

template <int D>
struct Joined {
  float top, sum, o[D / 32];
};
template <int D>
__device__ __forceinline__ void join_pieces(const float* slots, int rows, int row, int cta, int first, int step, int count, Joined<D>& r) {
  const int lane = threadIdx.x % 32;
  r.top = -INFINITY;
  r.sum = 0.0f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) r.o[e] = 0.0f;
  for (int i0 = first; i0 < count; i0 += kBatch * step) {
    float top[kBatch], sum[kBatch], o[kBatch][D / 32], most = r.top;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * step;
      top[k] = -INFINITY;
      sum[k] = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) o[k][e] = 0.0f;
      if (i >= count) continue;
      const float* s = slots + (2LL * (cta + i) + (i == 0)) * slot_floats(rows, D);
      top[k] = s[row];
      sum[k] = s[rows + row];
#pragma unroll
      for (int e = 0; e < D / 32; ++e) o[k][e] = s[2 * rows + row * D + e * 32 + lane];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) most = fmaxf(most, top[k]);
    const float base = most == -INFINITY ? 0.0f : most, keep = exp2_fast(r.top - base);
    r.top = most;
    r.sum *= keep;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) r.o[e] *= keep;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float w = sum[k] * exp2_fast(top[k] - base - kJoinDown);
      r.sum += w;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) r.o[e] = fmaf(w, o[k][e], r.o[e]);
    }
  }
}

// One warp to a row, for (request, head)s in few pieces: CTA by CTA of the kernel above, those where one began.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_few_kernel(const __grid_constant__ AttnParams p, const int kRows) {
  depend_release();
  depend_wait();
  const int4 word = *reinterpret_cast<const int4*>(reinterpret_cast<const Piece*>(p.a.workspace) + blockIdx.x);
  const Piece piece = {word.x, word.y, word.z, word.w};
  if (piece.last < 0) return;
  const float* slots = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(p.a.workspace) + sizeof(Piece) * gridDim.x);
  const int lane = threadIdx.x % 32;
  Joined<D> r;
  for (int row = threadIdx.x / 32; row < piece.rows; row += kJoinWarps) {
    join_pieces<D>(slots, kRows, row, blockIdx.x, 0, 1, piece.last - blockIdx.x + 1, r);
    const long long at = (piece.first + row / p.group) * p.a.stride_out_tok + (piece.head * p.group + row % p.group) * p.a.stride_out_head;
#pragma unroll
    for (int e = 0; e < D / 32; ++e)
      store_from_float(p.a.out, at + e * 32 + lane, p.a.dtype, r.sum == 0.0f ? 0.0f : __fdiv_rn(r.o[e], r.sum));
  }
}

// One CTA to a row, for (request, head)s in many pieces: there are few of them then, so each finds its CTAs by counting
// the tiles ahead of it on the line.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_many_kernel(const __grid_constant__ AttnParams p, const int kRows, const int ctas) {
  __shared__ float tops[kJoinWarps], sums[kJoinWarps], part_o[kJoinWarps][D];
  depend_release();
  depend_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, HKV = p.a.cache.HKV, b = blockIdx.x / HKV, h = blockIdx.x % HKV;
  long long total = 0, ahead = 0;
  int mine = 0;
  for (int x = lane; x < p.a.rows.B; x += 32) {
    const int tiles = tiles_of(p, x);
    total += tiles;
    if (x < b) ahead += tiles;
    if (x == b) mine = tiles;
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) {
    total += __shfl_xor_sync(~0u, total, d);
    ahead += __shfl_xor_sync(~0u, ahead, d);
    mine += __shfl_xor_sync(~0u, mine, d);
  }
  if (mine == 0) return;
  const long long share = (total * HKV + ctas - 1) / ctas, from = ahead * HKV + (long long)h * mine;
  const int first = (int)(from / share), count = (int)((from + mine - 1) / share) - first + 1;
  if (count == 1) return;                         // one CTA had all of it, and has written the output
  const KvRequest q = kv_request(p.a.cache, p.a.rows, b, nullptr);
  const int row = blockIdx.y;
  if (row >= q.todo * p.group) return;
  const float* slots = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(p.a.workspace) + sizeof(Piece) * ctas);
  Joined<D> r;
  join_pieces<D>(slots, kRows, row, first, warp, kJoinWarps, count, r);
  if (lane == 0) {
    tops[warp] = r.top;
    sums[warp] = r.sum;
  }
#pragma unroll
  for (int e = 0; e < D / 32; ++e) part_o[warp][e * 32 + lane] = r.o[e];
  __syncthreads();
  float top = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, tops[w]);
  const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    const float by = exp2_fast(tops[w] - base);
    sum += sums[w] * by;
    o = fmaf(part_o[w][threadIdx.x % D], by, o);
  }
  if (threadIdx.x < D)
    store_from_float(p.a.out, row_place(p, q, h, row, token_of(p, row), p.a.stride_out_tok, p.a.stride_out_head) + threadIdx.x, p.a.dtype,
                     sum == 0.0f ? 0.0f : __fdiv_rn(o, sum));
}

// Tiles of eight query rows that a warp of the decode kernel holds, or 0 where the rows are too many for its registers.
int column_tiles(const CarryGdnKvAttentionArgs& a) {
  const long long rows = (long long)a.rows.max_query * (a.HQ / a.cache.HKV);
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 0;
}

// CTAs of the decode kernel: all that are resident at a time, or one per tile where there cannot be as many.
long long decode_ctas(const CarryGdnKvAttentionArgs& a) {
  const long long tokens = (long long)a.cache.max_pages * a.cache.page;
  const long long most = (tokens + kLine - 1) / kLine * a.cache.HKV * a.rows.B;
  const long long fit = (long long)sm_count() * resident(a.cache.D, column_tiles(a), a.dtype == CARRY_F32 ? 2 : 1);
  return most < 1 ? 1 : most < fit ? most : fit;
}

// launch_dependent() with clusters of so many CTAs.
template <class K, class... A>
int launch_clusters(K kernel, int clusters, int size, size_t smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)clusters * size);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return CARRY_GDN_OK;
  cudaGetLastError();
  return CARRY_GDN_ERR_LAUNCH;
}

// CTAs of the clusters that take a call, or 0: as many as leave all clusters resident, two CTAs to an SM but for what the
// groups of SMs that a cluster has to fit in leave over; no more than a context has tiles, and four tiles for each CTA at most.
// One request of 1500 tokens and 8 heads takes 8.2 us so (clusters of eight), 11.4 by the line, four of 4096 16 and 18.2; 16 of
// 128 6.4 and 11.8, 32 of 300 (one CTA each) 10.1 and 14.7.  With more than are resident at a time the line is as good: 56 requests
// of 120 and 16 heads 18.1 and 19.5, of 500 38.6 and 35.8.
int cluster_size(const CarryGdnKvAttentionArgs& a) {
  const long long tokens = (long long)a.cache.max_pages * a.cache.page, pairs = (long long)a.rows.B * a.cache.HKV;
  for (int size = 8; size > 0; size /= 2)
    if (4 * pairs * size <= 7LL * sm_count() && (size == 1 || 2 * tokens > size * kLine))
      return tokens <= 4LL * size * kLine ? size : 0;
  return 0;
}

template <int D, int NT, int PARTS, int CL>
int launch_pairs(const AttnParams& p, cudaStream_t stream) {
  constexpr size_t smem = sizeof(PairShared<D, NT, PARTS, CL>);
  static thread_local bool ready[64];
  const int rc = prepare(kv_pair_kernel<D, NT, PARTS, CL>, smem, ready);
  return rc == CARRY_GDN_OK ? launch_clusters(kv_pair_kernel<D, NT, PARTS, CL>, p.a.rows.B * p.a.cache.HKV, CL, smem, stream, p) : rc;
}

template <int D, int NT, int PARTS>
int launch_decode(const AttnParams& p, cudaStream_t stream) {
  constexpr size_t smem = sizeof(DecodeShared<D, NT, PARTS>);
  static thread_local bool ready[64];
  switch (cluster_size(p.a)) {
    case 8: return launch_pairs<D, NT, PARTS, 8>(p, stream);
    case 4: return launch_pairs<D, NT, PARTS, 4>(p, stream);
    case 2: return launch_pairs<D, NT, PARTS, 2>(p, stream);
    case 1: return launch_pairs<D, NT, PARTS, 1>(p, stream);
  }
  const unsigned ctas = (unsigned)decode_ctas(p.a);
  int rc = prepare(kv_decode_kernel<D, NT, PARTS>, smem, ready);
  if (rc == CARRY_GDN_OK) rc = launch_dependent(kv_decode_kernel<D, NT, PARTS>, dim3(ctas), kThreads, smem, stream, p);
  if (rc != CARRY_GDN_OK) return rc;
  const long long pairs = (long long)p.a.rows.B * p.a.cache.HKV;
  if (ctas <= kBatch * pairs) return launch_dependent(kv_join_few_kernel<D>, dim3(ctas), kJoinThreads, 0, stream, p, NT * 8);
  return launch_dependent(kv_join_many_kernel<D>, dim3((unsigned)pairs, p.rows), kJoinThreads, 0, stream, p, NT * 8, (int)ctas);
}

template <int D, int PARTS>
int launch_tiles(const AttnParams& p, cudaStream_t stream) {
  return column_tiles(p.a) == 1 ? launch_decode<D, 1, PARTS>(p, stream) : launch_decode<D, 2, PARTS>(p, stream);
}

}  // namespace

bool few_rows(const CarryGdnKvAttentionArgs& a) { return column_tiles(a) > 0; }

int64_t kv_decode_workspace(const CarryGdnKvAttentionArgs& a) {
  if (cluster_size(a)) return 0;
  const long long ctas = decode_ctas(a);
  return sizeof(Piece) * ctas + 2 * ctas * slot_floats(column_tiles(a) * 8, a.cache.D) * 4;
}

int launch_kv_decode(const AttnParams& p, cudaStream_t stream) {
  if (p.a.cache.D == 64) return p.a.dtype == CARRY_F32 ? launch_tiles<64, 2>(p, stream) : launch_tiles<64, 1>(p, stream);
  return p.a.dtype == CARRY_F32 ? launch_tiles<128, 2>(p, stream) : launch_tiles<128, 1>(p, stream);
}

}  // namespace carry
