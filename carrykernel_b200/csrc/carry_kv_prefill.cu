// Attention over the 8-bit key/value cache for many query rows of a request: chunks of a prompt.
//
// A CTA has 256 rows (query tokens times the query heads of one key/value head) as two tiles of 128, and walks the
// request's tokens 128 at a time.  The work is in four places that run side by side:
//  * eight warps turn a tile's codes into fp16, keys and values, into shared memory (e4m3 is a subset of fp16; codes of
//    the tile after it wait in registers);
//  * one thread issues the matrix products on the fifth-generation tensor cores: S = Q K^T, operands in shared memory,
//    and O += P V with the weights P in tensor memory;
//  * eight warps for each row tile take its scores out of tensor memory, half a row to a thread, and put the weights back
//    in their place.  While one tile's weights are formed, the other's products run.
// What bounds it: 2 x 128 x 128 exponentials a step take 2048 cycles of the special function units, and the products as
// many of the tensor cores.
//
// A row's weights are relative to a maximum that is replaced, and O rescaled, only when it is outgrown by 2^4; values
// likewise count in the largest value scale until one is 2^4 larger.  A weight is formed times 2^7, so it stays below
// fp16's 2^16, and has all its bits down to 2^-21 of the row's largest.
#include "carry_kv_attention.cuh"

namespace carry {
namespace {

constexpr int kTokens = 128, kTileRows = 128, kCtaRows = 2 * kTileRows, kPlane = 128 * 128;   // a plane: 128 rows of 64 columns
constexpr int kTileThreads = 256, kSoftmaxThreads = 2 * kTileThreads, kConvertThreads = 256, kAllThreads = kSoftmaxThreads + kConvertThreads + 32;
constexpr int kBlocks = kTokens / kGranule;
constexpr float kUp = 7.0f, kSlack = 4.0f;

template <int D>
struct Shared {
  uint8_t q[2][D / 64][kPlane], k[2][D / 64][kPlane], v[2][D / 64][kPlane];
  // of a step's blocks: key scale, log2 of the value scale in the running unit plus kUp, and what a weight so formed
  // counts in the row's sum
  float ks[2][kBlocks], bias[2][kBlocks], counts[2][kBlocks];
  float rescale[2], unit;
  float top[2][2][2][kTileRows];                  // by step, tile and half of a step: largest score of a row
  float unit_q[2][kTileRows];
  uint64_t k_full[2], v_full[2], free[2], s_full[2], top_full[2], p_full[2], o_done[2];
  uint32_t tmem;
  int poison;
};

// ---- waiting ---------------------------------------------------------------------------------------------------------

constexpr int kSpinLimit = 1 << 20;               // polls of a barrier, each of which the hardware may hold for a while

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrier_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.b32 %0, 1, 0, p;\n}"
               : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
  return done;
}
// Waits for a phase of a barrier, within a limit; false when it ran out here or at another waiter.
__device__ __forceinline__ bool barrier_wait(uint64_t* bar, uint32_t parity, volatile int* poison, int* status) {
  if (barrier_try(bar, parity)) return true;
  for (int i = 0; i < kSpinLimit; ++i) {
    if (barrier_try(bar, parity)) return true;
    if (*poison) return false;
  }
  *poison = 1;
  if (status) atomicOr(status, CARRY_GDN_STATUS_TIMEOUT);
  return false;
}

// ---- tensor cores ----------------------------------------------------------------------------------------------------

// Operand in shared memory, rows of 128 bytes in groups of eight (1024 bytes), 16-byte chunks exchanged by the row's
// number in its group.  `step`: bytes between groups; `lead`: between planes of 64 columns, where columns are contiguous
// along the side that is not summed over.
__device__ __forceinline__ uint64_t descriptor(const void* p, uint32_t lead, uint32_t step) {
  return static_cast<uint64_t>((smem_addr(p) & 0x3ffff) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 |
         static_cast<uint64_t>(step >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// fp16 operands, fp32 sums, 128 rows, N columns; `across`: the second operand is contiguous along N
__host__ __device__ constexpr uint32_t instruction(int N, bool across) {
  return 1u << 4 | (across ? 1u << 16 : 0u) | static_cast<uint32_t>(N / 8) << 17 | static_cast<uint32_t>(128 / 16) << 24;
}
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
               "r"(what), "r"(static_cast<uint32_t>(add)) : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b),
               "r"(what), "r"(static_cast<uint32_t>(add)) : "memory");
}
// the barrier's phase ends when every product issued so far has
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of a warp's 32 rows, a row to a lane
__device__ __forceinline__ void tmem_load(uint32_t at, float (&x)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t at, const float (&x)[32]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(x);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
      "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// ---- tiles in shared memory ------------------------------------------------------------------------------------------

// where the 16-byte chunk `chunk` (eight numbers) of a row of a plane lies
__device__ __forceinline__ int plane_at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// A query row as fp16, scaled by a power of two, into its tile; what a product of it counts, in log2's scale.
template <int D>
__device__ __forceinline__ float stage_query(const AttnParams& p, const KvRequest& r, int h, int row, uint8_t (*tile)[kPlane], int tile_row) {
  const int i = row / p.group;
  const bool there = i < r.todo;
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p.a.q) +
                      (there ? (r.first + i) * p.a.stride_q_tok + (h * p.group + row % p.group) * p.a.stride_q_head : 0);
  const bool vec = reinterpret_cast<uintptr_t>(q) % 16 == 0;
  const bool bf16 = p.a.dtype == CARRY_BF16;
  uint32_t top = 0, w[D / 2];
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (there && vec) {
      u = *reinterpret_cast<const uint4*>(q + c * 8);
    } else if (there) {
      auto two = [&](int e) { return q[c * 8 + e] | static_cast<uint32_t>(q[c * 8 + e + 1]) << 16; };
      u = make_uint4(two(0), two(2), two(4), two(6));
    }
    w[4 * c] = u.x; w[4 * c + 1] = u.y; w[4 * c + 2] = u.z; w[4 * c + 3] = u.w;
  }
  auto numbers = [&](uint32_t u) { return bf16 ? make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)) : unpack_half2(u); };
#pragma unroll
  for (int c = 0; c < D / 2; ++c) {
    const float2 x = numbers(w[c]);
    top = max(top, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
  }
  const int e = up_exponent(top);
  const float up = copysignf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), p.a.scale);
#pragma unroll
  for (int c = 0; c < D / 2; ++c) {
    const float2 x = numbers(w[c]);
    w[c] = pack_half2(x.x * up, x.y * up);
  }
#pragma unroll
  for (int c = 0; c < D / 8; ++c)
    *reinterpret_cast<uint4*>(tile[c / 8] + plane_at(tile_row, c % 8)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  return fabsf(p.a.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// A step's granules, as the converting warps hold them: lane l < 8 has granule l's place in the codes (-1: no tokens) and
// in the scales.  They are fetched a step before the codes that they lead to.
struct StepPages {
  long long k, v;
  int id, block;
};
template <int D>
__device__ __forceinline__ StepPages fetch_pages(const AttnParams& p, int b, int h, int step, int length) {
  const CarryGdnKvCache& c = p.a.cache;
  const int granule = step * kBlocks + threadIdx.x % 32;
  StepPages x = {-1, -1, 0, 0};
  if (threadIdx.x % 32 < kBlocks) x.id = page_id(p, b, granule, length);
  if (x.id > 0) {
    const int in_page = granule - page_index(p, granule) * p.page_granules, at = (h * c.page + in_page * kGranule) * D;
    x.k = x.id * c.stride_k_page + at;
    x.v = x.id * c.stride_v_page + at;
    x.block = h * (p.page_granules / p.block_granules) + divide(in_page, p.block_granules, p.block_shift);
  }
  return x;
}
// A converting thread's codes of a step: chunk tid % (D / 16) of tokens tid / (D / 16) + i * kStride.  Tokens at or beyond
// the length and those of padding pages are zeros, whatever memory holds there.
template <int D>
constexpr int kCodes = kTokens * (D / 16) / kConvertThreads;
template <int D>
__device__ __forceinline__ void fetch_codes(const uint8_t* codes, long long place, int left, int tid, uint4 (&x)[kCodes<D>]) {
  constexpr int kChunks = D / 16, kStride = kConvertThreads / kChunks;
  const uint8_t* mine = codes + tid / kChunks % kGranule * D + tid % kChunks * 16;
  const int first = tid / kChunks;
  const bool whole = left >= kTokens && __all_sync(~0u, place >= 0 || threadIdx.x % 32 >= kBlocks);
#pragma unroll
  for (int i = 0; i < kCodes<D>; ++i) {
    const long long at = __shfl_sync(~0u, place, (first + i * kStride) / kGranule);
    if (whole) {
      x[i] = *reinterpret_cast<const uint4*>(mine + at);
    } else {
      x[i] = make_uint4(0, 0, 0, 0);
      if (at >= 0 && first + i * kStride < left) x[i] = *reinterpret_cast<const uint4*>(mine + at);
    }
  }
}
template <int D>
__device__ __forceinline__ void store_codes(const uint4 (&x)[kCodes<D>], uint8_t (*tile)[kPlane], int tid) {
  constexpr int kChunks = D / 16, kStride = kConvertThreads / kChunks;
  const int chunk = tid % kChunks, turn = chunk / 4;         // the planes' stores take turns, or they would meet in the banks
  // rows differ by a multiple of eight, so they lie alike in their groups
  uint8_t* first = tile[chunk / 4] + plane_at(tid / kChunks, chunk % 4 * 2 + turn);
  uint8_t* second = tile[chunk / 4] + plane_at(tid / kChunks, chunk % 4 * 2 + 1 - turn);
#pragma unroll
  for (int i = 0; i < kCodes<D>; ++i) {
    uint4 lo, hi;
    halves_of(x[i].x, lo.x, lo.y);
    halves_of(x[i].y, lo.z, lo.w);
    halves_of(x[i].z, hi.x, hi.y);
    halves_of(x[i].w, hi.z, hi.w);
    *reinterpret_cast<uint4*>(first + i * kStride * 128) = turn ? hi : lo;
    *reinterpret_cast<uint4*>(second + i * kStride * 128) = turn ? lo : hi;
  }
}

template <int D>
__global__ void __launch_bounds__(kAllThreads, 1) kv_prefill_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ uint8_t raw[];
  Shared<D>& sh = *reinterpret_cast<Shared<D>*>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
  depend_release();
  depend_wait();
  const CarryGdnKvCache& c = p.a.cache;
  const int b = blockIdx.z, h = blockIdx.y, first_row = (gridDim.x - 1 - blockIdx.x) * kCtaRows;     // the longest go first
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const KvRequest r = kv_request(c, p.a.rows, b, first_row == 0 && h == 0 && threadIdx.x == 0 ? p.a.status : nullptr);
  if (first_row >= r.todo * p.group) return;
  const int last = min((first_row + kCtaRows - 1) / p.group, r.todo - 1);
  const int length = max(min(r.length, r.length - r.count + last + 1), 0), steps = (length + kTokens - 1) / kTokens;

  if (threadIdx.x == 0) {
    sh.poison = 0;
    sh.unit = 1.0f;
    for (int i = 0; i < 2; ++i) {
      barrier_init(&sh.k_full[i], kConvertThreads);
      barrier_init(&sh.v_full[i], kConvertThreads);
      barrier_init(&sh.free[i], 1);
      barrier_init(&sh.s_full[i], 1);
      barrier_init(&sh.top_full[i], kTileThreads);
      barrier_init(&sh.p_full[i], kTileThreads);
      barrier_init(&sh.o_done[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kAllThreads / 32 - 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x < kCtaRows) {
    const int tile = threadIdx.x / kTileRows, row = threadIdx.x % kTileRows;
    sh.unit_q[tile][row] = stage_query<D>(p, r, h, first_row + threadIdx.x, sh.q[tile], row);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;                  // columns 0, 128: scores of the two tiles; 256, 384: outputs
  volatile int* poison = &sh.poison;

  if (threadIdx.x < kSoftmaxThreads) {
    // ---- half a row's scores to a thread ----
    const int tile = threadIdx.x / kTileThreads, part = threadIdx.x / kTileRows % 2, tile_row = threadIdx.x % kTileRows;
    const int row = first_row + tile * kTileRows + tile_row, i = row / p.group;
    const int sees = (i < r.todo ? r.length - r.count + i + 1 : 0) - part * 64;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t s_at = tmem + lanes + tile * 128 + part * 64, o_at = tmem + lanes + 256 + tile * 128 + part * (D / 2);
    const float unit_q = sh.unit_q[tile][tile_row];
    float top = -INFINITY, sum = 0.0f;
    bool healthy = true;
    for (int step = 0; step < steps; ++step) {
      const int stage = step & 1, parity = step / 2 & 1;
      healthy = barrier_wait(&sh.k_full[stage], parity, poison, p.a.status) && barrier_wait(&sh.s_full[tile], step & 1, poison, p.a.status);
      if (!healthy) break;
      fence_after();
      const int limit = sees - step * kTokens;
      const bool all = __all_sync(~0u, limit >= 64);
      float x[32], now = top;
#pragma unroll 1
      for (int n = 0; n < 2; ++n) {
        tmem_load(s_at + n * 32, x);
        wait_loads();
        if (!all) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = n * 32 + e < limit ? x[e] : -INFINITY;
        }
#pragma unroll
        for (int block = 0; block < 2; ++block) {
          const float ks = sh.ks[stage][part * 4 + n * 2 + block];
          float m = -INFINITY;
#pragma unroll
          for (int e = 0; e < 16; e += 2) m = fmaxf(m, fmaxf(x[block * 16 + e], x[block * 16 + e + 1]));
          if (ks != kNoTokens) now = fmaxf(now, m * fmaxf(unit_q * ks, 0x1p-126f));
        }
      }
      sh.top[stage][tile][part][tile_row] = now;
      barrier_arrive(&sh.top_full[tile]);
      healthy = barrier_wait(&sh.top_full[tile], step & 1, poison, p.a.status);
      if (!healthy) break;
      now = fmaxf(now, sh.top[stage][tile][part ^ 1][tile_row]);
      const float values = sh.rescale[stage];
      if (__any_sync(~0u, now > top + kSlack) || values != 1.0f) {   // alike in both halves of a row
        const float keep = now == -INFINITY ? 1.0f : exp2_fast(top - now);
        sum *= keep;
        top = now;
        if (step > 0) {
          healthy = barrier_wait(&sh.o_done[tile], (step - 1) & 1, poison, p.a.status);
          if (!healthy) break;
          fence_after();
#pragma unroll 1
          for (int n = 0; n < D / 64; ++n) {
            tmem_load(o_at + n * 32, x);
            wait_loads();
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] *= keep * values;
            tmem_store(o_at + n * 32, x);
          }
          wait_stores();
        }
      }
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll 1
      for (int n = 0; n < 2; ++n) {
        tmem_load(s_at + n * 32, x);
        wait_loads();
        uint32_t w[16];
#pragma unroll
        for (int block = 0; block < 2; ++block) {
          const int at = part * 4 + n * 2 + block;
          const float ks = sh.ks[stage][at], by = fmaxf(unit_q * ks, 0x1p-126f), bias = sh.bias[stage][at] - base;
          float2 total = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float2 y = fma2(make_float2(x[block * 16 + e], x[block * 16 + e + 1]), make_float2(by, by), make_float2(bias, bias));
            x[block * 16 + e] = exp2_fast(y.x);
            x[block * 16 + e + 1] = exp2_fast(y.y);
          }
          if (!all || ks == kNoTokens) {
            const int t = ks == kNoTokens ? 1 << 30 : n * 32 + block * 16;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[block * 16 + e] = t + e < limit ? x[block * 16 + e] : 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            total = add2(total, make_float2(x[block * 16 + e], x[block * 16 + e + 1]));
            w[block * 8 + e / 2] = pack_half2(x[block * 16 + e], x[block * 16 + e + 1]);
          }
          sum = fmaf(total.x + total.y, sh.counts[stage][at], sum);
        }
        tmem_store16(s_at + n * 16, w);           // over scores that this warp has read
      }
      wait_stores();
      fence_before();
      barrier_arrive(&sh.p_full[tile]);
    }
    if (healthy && steps > 0) {
      healthy = barrier_wait(&sh.o_done[tile], (steps - 1) & 1, poison, p.a.status);
      fence_after();
    }
    if (healthy) {
      sh.top[steps & 1][tile][part][tile_row] = sum;             // the halves of a row's sum meet
      barrier_arrive(&sh.top_full[tile]);
      healthy = barrier_wait(&sh.top_full[tile], steps & 1, poison, p.a.status);
    }
    if (healthy) {
      sum += sh.top[steps & 1][tile][part ^ 1][tile_row];
      const float by = sum == 0.0f ? 0.0f : __fdiv_rn(exp2f(-kUp), sum);
      const float unit = steps > 0 ? *reinterpret_cast<volatile float*>(&sh.unit) : 1.0f;
      const long long at = (r.first + i) * p.a.stride_out_tok + (h * p.group + row % p.group) * p.a.stride_out_head + part * (D / 2);
#pragma unroll 1
      for (int n = 0; n < D / 64; ++n) {
        alignas(16) float x[32];
        if (steps > 0) {
          tmem_load(o_at + n * 32, x);
          wait_loads();
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = sum == 0.0f ? 0.0f : x[e] * by * unit;
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = 0.0f;
        }
        if (i < r.todo) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) store8(p.a.out, at + n * 32 + e, p.a.dtype, x + e);
        }
      }
    }
  } else if (threadIdx.x < kSoftmaxThreads + kConvertThreads) {
    // ---- codes to operands ----
    const int tid = threadIdx.x - kSoftmaxThreads;
    float unit = 0.0f, ks = kNoTokens, vs = 0.0f;
    uint4 k[kCodes<D>], v[kCodes<D>];
    StepPages pages = fetch_pages<D>(p, b, h, 0, length);
    auto fetch_scales = [&]() {
      ks = pages.id > 0 ? c.k_scale[pages.id * c.stride_ks_page + pages.block] : kNoTokens;
      vs = pages.id > 0 ? c.v_scale[pages.id * c.stride_vs_page + pages.block] : 0.0f;
    };
    fetch_codes<D>(c.k_codes, pages.k, length, tid, k);
    fetch_codes<D>(c.v_codes, pages.v, length, tid, v);
    if (tid < 32) fetch_scales();
    pages = fetch_pages<D>(p, b, h, 1, length);
    for (int step = 0; step < steps; ++step) {
      const int stage = step & 1, parity = step / 2 & 1, left = length - (step + 1) * kTokens;
      if (step >= 2 && !barrier_wait(&sh.free[stage], parity ^ 1, poison, p.a.status)) break;
      if (tid < 32) {
        float most = vs;
#pragma unroll
        for (int d = 4; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
        most = fmaxf(__shfl_sync(~0u, most, 0), 0x1p-100f);
        float rescale = 1.0f;
        if (step == 0) {
          unit = most;
        } else if (most > unit * exp2f(kSlack)) {
          rescale = __fdiv_rn(unit, most);
          unit = most;
        }
        if (tid < kBlocks) {
          sh.ks[stage][tid] = ks;
          sh.bias[stage][tid] = vs > 0.0f ? __log2f(__fdiv_rn(vs, unit)) + kUp : 0.0f;
          sh.counts[stage][tid] = vs > 0.0f ? __fdiv_rn(unit, vs) * exp2f(-kUp) : exp2f(-kUp);
        }
        if (tid == 0) {
          sh.rescale[stage] = rescale;
          sh.unit = unit;
        }
      }
      store_codes<D>(k, sh.k[stage], tid);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      barrier_arrive(&sh.k_full[stage]);
      fetch_codes<D>(c.k_codes, pages.k, left, tid, k);
      if (tid < 32) fetch_scales();
      store_codes<D>(v, sh.v[stage], tid);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      barrier_arrive(&sh.v_full[stage]);
      fetch_codes<D>(c.v_codes, pages.v, left, tid, v);
      pages = fetch_pages<D>(p, b, h, step + 2, length);
    }
  } else if (lane == 0) {
    // ---- products ----
    auto scores = [&](int tile, int stage) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        mma_shared(tmem + tile * 128, descriptor(sh.q[tile][k / 4], 16, 1024) + k % 4 * 2, descriptor(sh.k[stage][k / 4], 16, 1024) + k % 4 * 2,
                   instruction(kTokens, false), k > 0);
      mma_commit(&sh.s_full[tile]);
    };
    bool healthy = steps > 0 && barrier_wait(&sh.k_full[0], 0, poison, p.a.status);
    if (healthy) {
      fence_after();
      scores(0, 0);
      scores(1, 0);
    }
    for (int step = 0; healthy && step < steps; ++step) {
      const int stage = step & 1, parity = step / 2 & 1;
      for (int tile = 0; tile < 2 && healthy; ++tile) {
        healthy = (tile > 0 || barrier_wait(&sh.v_full[stage], parity, poison, p.a.status)) &&
                  barrier_wait(&sh.p_full[tile], step & 1, poison, p.a.status);
        if (!healthy) break;
        fence_after();
#pragma unroll
        for (int k = 0; k < kTokens / 16; ++k)
          mma_tensor(tmem + 256 + tile * 128, tmem + tile * 128 + k / 4 * 64 + k % 4 * 8, descriptor(sh.v[stage][0] + k * 2048, kPlane, 1024), instruction(D, true),
                     step > 0 || k > 0);
        mma_commit(&sh.o_done[tile]);
        if (tile == 1) mma_commit(&sh.free[stage]);
        if (step + 1 < steps) {
          healthy = tile > 0 || barrier_wait(&sh.k_full[stage ^ 1], (step + 1) / 2 & 1, poison, p.a.status);
          if (!healthy) break;
          fence_after();
          scores(tile, stage ^ 1);
        }
      }
    }
    if (!healthy) {
      // products in flight still use shared and tensor memory: a bounded time for them to end
      for (int i = 0; i < 1 << 12; ++i) __nanosleep(64);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kAllThreads / 32 - 1) {
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int D>
int launch(const AttnParams& p, cudaStream_t stream) {
  constexpr size_t smem = sizeof(Shared<D>) + 1024;
  static thread_local bool ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(kv_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
      cudaGetLastError();
      return CARRY_GDN_ERR_LAUNCH;
    }
    if (dev < 64) ready[dev] = true;
  }
  const long long rows = (long long)p.a.rows.max_query * p.group;
  const dim3 grid((unsigned)((rows + kCtaRows - 1) / kCtaRows), p.a.cache.HKV, p.a.rows.B);
  return launch_dependent(kv_prefill_kernel<D>, grid, kAllThreads, smem, stream, p);
}

}  // namespace

int launch_kv_prefill(const AttnParams& p, cudaStream_t stream) {
  return p.a.cache.D == 64 ? launch<64>(p, stream) : launch<128>(p, stream);
}

}  // namespace carry
