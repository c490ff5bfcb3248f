// Attention over the 8-bit key/value cache for many fp32 query rows of a request.  (16-bit rows go to the tensor-memory
// kernel, whose operands an fp32 row does not fit.)
//
// A CTA has 64 rows, 16 to a warp, and walks the tokens in tiles of 64; every warp converts the tile's codes for itself.
// Each number of q and each weight is two fp16 numbers, so products cost twice.  512 tokens of a prompt, 32 heads over 8 of 128:
// 41 us.
#include "carry_kv_attention.cuh"

namespace carry {
namespace {

constexpr int kTile = 64, kWarps = 4, kThreads = kWarps * 32;
constexpr int kRowsPerWarp = 16;
constexpr int PARTS = 2;                          // fp16 numbers to a number of q, and to a weight

template <int D>
struct Stage {
  alignas(128) uint8_t k[kTile * D];
  uint8_t v[kTile * D];
  float ks[kTile / kGranule], vs[kTile / kGranule];
};

// ---- tiles into shared memory ----------------------------------------------------------------------------------------

// The page ids that this thread's copies of a tile need, fetched a tile ahead of the copies.
template <int D>
struct Pages {
  int chunk[D / 32], scale;
};
template <int D>
__device__ __forceinline__ int granule_of(int i) {       // of this thread's i-th chunk of a tile
  return D == 128 ? i : 2 * i + (threadIdx.x >> 6);
}
template <int D>
__device__ __forceinline__ void fetch_pages(const AttnParams& p, int b, int tile, int length, Pages<D>& ids) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) ids.chunk[i] = page_id(p, b, tile * 4 + granule_of<D>(i), length);
  ids.scale = threadIdx.x < 8 ? page_id(p, b, tile * 4 + threadIdx.x % 4, length) : 0;
}

// Tokens at or beyond `length` and tokens of padding pages are filled with zeros, whatever memory holds there.
template <int D>
__device__ __forceinline__ void load_tile(const AttnParams& p, Stage<D>& s, int h, int tile, int length, const Pages<D>& ids) {
  const CarryGdnKvCache& c = p.a.cache;
  constexpr int kChunks = D / 16, kStep = kThreads / kChunks;
  const int chunk = threadIdx.x % kChunks;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int row = threadIdx.x / kChunks + i * kStep, granule = tile * 4 + granule_of<D>(i), id = ids.chunk[i];
    const int in_page = (granule - page_index(p, granule) * p.page_granules) * kGranule + row % kGranule;
    const long long at = ((long long)h * c.page + in_page) * D + chunk * 16;
    const size_t zero = id > 0 && tile * kTile + row < length ? 0 : 16;
    const int to = tile_at<D>(row, chunk);
    __pipeline_memcpy_async(s.k + to, zero ? c.k_codes : c.k_codes + id * c.stride_k_page + at, 16, zero);
    __pipeline_memcpy_async(s.v + to, zero ? c.v_codes : c.v_codes + id * c.stride_v_page + at, 16, zero);
  }
  if (threadIdx.x < 8) {
    const int i = threadIdx.x % 4, granule = tile * 4 + i, id = ids.scale;
    const int at = h * (p.page_granules / p.block_granules) + (granule - page_index(p, granule) * p.page_granules) / p.block_granules;
    float* to = threadIdx.x < 4 ? &s.ks[i] : &s.vs[i];
    if (id > 0) __pipeline_memcpy_async(to, threadIdx.x < 4 ? c.k_scale + id * c.stride_ks_page + at : c.v_scale + id * c.stride_vs_page + at, 4);
    else *to = threadIdx.x < 4 ? kNoTokens : 0.0f;
  }
}

// ---- one warp's rows -------------------------------------------------------------------------------------------------

// 16 query rows of a warp as operands of the matrix instructions.  Lane (g, c) = (lane / 4, lane % 4) has rows g and
// g + 8; the product sums over the columns in an order of its own, in which the lane's share of every 64 columns is 16
// neighbouring ones from 16 c on: those that one 16-byte load of key codes brings.
template <int D>
struct Query {
  uint32_t x[PARTS][D / 16][4];
  float unit[2];                  // scale * log2(e) over the power of two that the row was multiplied by
};

template <int D>
__device__ __forceinline__ void load_query(const AttnParams& p, const KvRequest& r, int h, int row0, Query<D>& q) {
  const int lane = threadIdx.x % 32, g = lane / 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + g + half * 8, i = token_of(p, row);
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
    const float up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    q.unit[half] = p.a.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
        float u = x[k * 4 + pair * 2] * up, v = x[k * 4 + pair * 2 + 1] * up;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t w = pack_half2(u, v);
          q.x[part][k][pair * 2 + half] = w;
          const float2 kept = unpack_half2(w);
          u -= kept.x;
          v -= kept.y;
        }
      }
  }
}

// Running softmax of a warp's rows over the tokens that it has seen.
template <int D>
struct Rows {
  float o[D / 8][4];              // lane (g, c): row g columns 2c (D/8) + n and (2c + 1) D/8 + n, then row g + 8's
  float top[2], sum[2];           // of rows g and g + 8; the sums are this lane's share
  float up[2];                    // 2^15 over the unit that a row's outputs count in: o is that many times too large
  Scales scales;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    top[0] = top[1] = -INFINITY;
    sum[0] = sum[1] = 0.0f;
    up[0] = up[1] = kUpStart;
    scales.most = INFINITY;
  }
};

// A tile of tokens.  `limit` says how many of the tile's tokens rows g and g + 8 see.
template <int D>
__device__ __forceinline__ void attend(const Stage<D>& s, const Query<D>& q, const int (&limit)[2], Rows<D>& r) {
  const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  float score[kTile / 8][4];
#pragma unroll
  for (int n = 0; n < kTile / 8; ++n) {
    float acc[4] = {};
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const uint4 w = *reinterpret_cast<const uint4*>(s.k + tile_at<D>(n * 8 + g, j * 4 + c));
      const uint32_t codes[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t b0, b1;
        halves_of(codes[k], b0, b1);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) mma_fp16(acc, q.x[part][j * 4 + k], b0, b1);
      }
    }
    const float ks = s.ks[(n * 8) / kGranule];
    const int t = ks == kNoTokens ? 1 << 30 : n * 8 + 2 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) score[n][i] = t + i % 2 < limit[i / 2] ? acc[i] * (q.unit[i / 2] * ks) : -INFINITY;
  }

  float now[2], vs_top = 0.0f;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float m = -INFINITY;
#pragma unroll
    for (int n = 0; n < kTile / 8; ++n) m = fmaxf(m, fmaxf(score[n][2 * half], score[n][2 * half + 1]));
    now[half] = fmaxf(r.top[half], quad_max(m));
  }
#pragma unroll
  for (int b = 0; b < kTile / kGranule; ++b) vs_top = fmaxf(vs_top, s.vs[b]);
  if (__any_sync(~0u, now[0] > r.top[0] || now[1] > r.top[1]) || vs_top * r.up[0] > 0x1p15f || r.scales.most < 0.0f) {
    float keep[2], vs_low = vs_top;
#pragma unroll
    for (int b = 0; b < kTile / kGranule; ++b) vs_low = fminf(vs_low, s.ks[b] == kNoTokens ? vs_top : s.vs[b]);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      keep[half] = now[half] == -INFINITY ? 1.0f : exp2_fast(r.top[half] - now[half]);
      r.sum[half] *= keep[half];
      r.top[half] = now[half];
    }
    const bool fresh = r.scales.fresh();
    if (__builtin_expect(r.scales.alike(vs_top, vs_low), 1)) {
      if (fresh || vs_top * r.up[0] > 0x1p15f) {
        const float up = up_above(vs_top), less = rescale(r.up[0], up);
        r.up[0] = r.up[1] = up;
        keep[0] *= less;
        keep[1] *= less;
      }
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float zero = now[half] == -INFINITY ? 0.0f : now[half], had = fresh ? 0.0f : up_of(r.up[half]) * keep[half];
        float met = 0.0f;
#pragma unroll
        for (int b = 0; b < kTile / kGranule; ++b) {
          const float m = fmaxf(fmaxf(score[2 * b][2 * half], score[2 * b][2 * half + 1]), fmaxf(score[2 * b + 1][2 * half], score[2 * b + 1][2 * half + 1]));
          met = fmaxf(met, exp2_fast(quad_max(m) - zero) * s.vs[b]);
        }
        r.up[half] = up_above(fmaxf(had, met));
        keep[half] = had * r.up[half] * 0x1p-15f;
      }
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) r.o[n][i] *= keep[i / 2];
  }
  const float base[2] = {now[0] == -INFINITY ? 0.0f : now[0], now[1] == -INFINITY ? 0.0f : now[1]};

#pragma unroll
  for (int b = 0; b < kTile / kGranule; ++b) {
    uint32_t w[PARTS][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {                  // rows g, g + 8 of the first eight tokens, then of the other eight
      const int half = x % 2, n = 2 * b + x / 2;
      float2 y = make_float2(exp2_fast(score[n][2 * half] - base[half]), exp2_fast(score[n][2 * half + 1] - base[half]));
      r.sum[half] += y.x + y.y;
      y = scaled(y, s.vs[b], make_float2(r.up[half], r.up[half]));
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        w[part][x] = pack_half2(y.x, y.y);
        const float2 kept = unpack_half2(w[part][x]);
        y.x -= kept.x;
        y.y -= kept.y;
      }
    }
    // values: this lane's columns of tokens 2c, 2c + 1, 2c + 8, 2c + 9
    const int t = b * kGranule + 2 * c;
    constexpr int kWords = D / 32;                // words of D / 8 codes
    uint32_t v[4][kWords];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = t + i % 2 + i / 2 * 8;
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
        uint32_t b0[2], b1[2];
        halves_of(__byte_perm(v[0][k], v[1][k], e ? 0x7362 : 0x5140), b0[0], b0[1]);
        halves_of(__byte_perm(v[2][k], v[3][k], e ? 0x7362 : 0x5140), b1[0], b1[1]);
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int part = 0; part < PARTS; ++part) mma_fp16(r.o[k * 4 + e * 2 + f], w[part], b0[f], b1[f]);
      }
  }
}

// A finished row's columns of this lane, normalised, to the output.
template <int D>
__device__ __forceinline__ void store_rows(const AttnParams& p, const KvRequest& q, int h, int row0, const Rows<D>& r) {
  const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + g + half * 8, i = token_of(p, row);
    if (i >= q.todo) continue;
    const long long at = row_place(p, q, h, row, i, p.a.stride_out_tok, p.a.stride_out_head) + c * (D / 4);
#pragma unroll
    for (int e = 0; e < D / 4; e += 8) {
      alignas(16) float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = r.o[(e + k) % (D / 8)][2 * half + (e + k) / (D / 8)];
      store8(p.a.out, at + e, p.a.dtype, x);
    }
  }
}

// How many of a tile's tokens the lane's rows see.
__device__ __forceinline__ void row_limits(const AttnParams& p, const KvRequest& q, int row0, int tile, int (&limit)[2]) {
  const int g = threadIdx.x % 32 / 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = token_of(p, row0 + g + half * 8);
    limit[half] = i < q.todo ? q.length - q.count + i + 1 - tile * kTile : 0;
  }
}

constexpr int kChunkStages = 3, kChunkRows = kWarps * kRowsPerWarp;

// Two CTAs to an SM.  At D = 64 the compiler is told so, or it fits the registers of three: few or ragged CTAs come uneven then (four
// requests of 32 rows over 4096 tokens 49 us, 65 in threes; three prompts of 1 to 1968 tokens and 8 heads 97 and 122; four prompts
// of 900 tokens, of which six come to an SM, are faster in threes, 122 against 137).
template <int D>
__global__ void __launch_bounds__(kThreads, D == 64 ? 2 : 0) kv_chunk_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ __align__(128) uint8_t raw[];
  Stage<D>* stages = reinterpret_cast<Stage<D>*>(raw);
  depend_release();
  depend_wait();
  const CarryGdnKvCache& c = p.a.cache;
  const int b = blockIdx.x / c.HKV, h = blockIdx.x % c.HKV, first_row = (gridDim.y - 1 - blockIdx.y) * kChunkRows;   // the longest of all go first
  const KvRequest q = kv_request(c, p.a.rows, b, first_row == 0 && h == 0 && threadIdx.x == 0 ? p.a.status : nullptr);
  if (first_row >= q.todo * p.group) return;
  const int row0 = first_row + threadIdx.x / 32 * kRowsPerWarp;
  const int last = min(token_of(p, first_row + kChunkRows - 1), q.todo - 1);
  const int length = max(min(q.length, q.length - q.count + last + 1), 0), all_tiles = (length + kTile - 1) / kTile;
  const int share = (all_tiles + p.splits - 1) / p.splits, tile0 = min(share * (int)blockIdx.z, all_tiles), tiles = min(share, all_tiles - tile0);
  Pages<D> ids;
  fetch_pages<D>(p, b, tile0, length, ids);
  auto next_load = [&](int tile) {
    if (tile < tiles) {
      load_tile<D>(p, stages[tile % kChunkStages], h, tile0 + tile, length, ids);
      if (tile + 1 < tiles) fetch_pages<D>(p, b, tile0 + tile + 1, length, ids);
    }
    __pipeline_commit();
  };
#pragma unroll
  for (int s = 0; s < kChunkStages - 1; ++s) next_load(s);
  Query<D> query;
  Rows<D> r;
  load_query<D>(p, q, h, row0, query);
  r.clear();
  for (int tile = 0; tile < tiles; ++tile) {
    __pipeline_wait_prior(kChunkStages - 2);
    __syncthreads();
    next_load(tile + kChunkStages - 1);
    int limit[2];
    row_limits(p, q, row0, tile0 + tile, limit);
    attend<D>(stages[tile % kChunkStages], query, limit, r);
  }
  float sum[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    sum[half] = quad_sum(r.sum[half]);
    const float w = sum[half] == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum[half]), unit = up_of(r.up[half]) * 0x1p-15f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      r.o[n][2 * half] = r.o[n][2 * half] * w * unit;
      r.o[n][2 * half + 1] = r.o[n][2 * half + 1] * w * unit;
    }
  }
  if (p.splits == 1) {
    store_rows<D>(p, q, h, row0, r);
    return;
  }
  const Parts part = parts_of(p, blockIdx.z, blockIdx.x);
  const int g = threadIdx.x % 32 / 4, cc = threadIdx.x % 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + g + half * 8;
    if (cc == 0) {
      part.top[row] = r.top[half];
      part.sum[row] = sum[half];
    }
    float4* o = reinterpret_cast<float4*>(part.o + (long long)row * D + cc * (D / 4));
#pragma unroll
    for (int e = 0; e < D / 4; e += 4) {
      const int i = 2 * half + e / (D / 8), n = e % (D / 8);
      o[e / 4] = make_float4(r.o[n][i], r.o[n + 1][i], r.o[n + 2][i], r.o[n + 3][i]);
    }
  }
}

// splits and padded rows of the kernel for many fp32 rows
void lay_out(const CarryGdnKvAttentionArgs& a, int& splits, int& padded) {
  const long long rows = (long long)a.rows.max_query * (a.HQ / a.cache.HKV), tiles = (rows + kChunkRows - 1) / kChunkRows;
  padded = tiles > 65535 ? -1 : (int)tiles * kChunkRows;
  splits = split_count(a, (tiles * a.cache.HKV * a.rows.B + 1) / 2);             // an SM holds two of its CTAs
}

template <int D>
int launch_chunk(AttnParams p, cudaStream_t stream) {
  lay_out(p.a, p.splits, p.padded);
  constexpr size_t smem = sizeof(Stage<D>) * kChunkStages;
  static thread_local bool ready[64];
  int rc = prepare(kv_chunk_kernel<D>, smem, ready);
  if (rc != CARRY_GDN_OK) return rc;
  const dim3 grid((unsigned)p.a.cache.HKV * p.a.rows.B, (unsigned)p.padded / kChunkRows, (unsigned)p.splits);
  rc = launch_dependent(kv_chunk_kernel<D>, grid, kThreads, smem, stream, p);
  return rc == CARRY_GDN_OK && p.splits > 1 ? launch_join_parts(p, stream) : rc;
}

}  // namespace

int64_t kv_chunk_workspace(const CarryGdnKvAttentionArgs& a) {
  int splits, padded;
  lay_out(a, splits, padded);
  return padded < 0 ? CARRY_GDN_ERR_TOO_LARGE : parts_bytes(a, splits, padded);
}

int launch_kv_chunk(AttnParams p, cudaStream_t stream) {
  return p.a.cache.D == 64 ? launch_chunk<64>(p, stream) : launch_chunk<128>(p, stream);
}

}  // namespace carry
