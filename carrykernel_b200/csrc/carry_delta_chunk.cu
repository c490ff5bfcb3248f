// The gated delta rule in chunks of 64 tokens, on the fifth-generation tensor cores.
//
// With G_i the running sum of log alpha within a chunk and S the state at its start (as [K, V]), the rows u_i that a chunk adds
// are the solution of a triangular system,
//   (I + L) U = R,   R = diag(beta) (V - diag(exp G) K S),   L_ij = beta_i exp(G_i - G_j) k_i . k_j  for j < i,
// and with T = (I + L)^-1 and P_ij = exp(G_i - G_j) (scale q_i) . k_j for j <= i:
//   U = T R,   O = diag(exp G) (scale Q) S + (P T) R,   S' = exp(G_64) S + K^T diag(exp(G_64 - G)) U.
//
// T and P T do not depend on the state: unit_kernel (prepare_kernel for fp32) forms them for every chunk and head side by side.  sequence_kernel
// then walks a request's chunks, a CTA for 32 or 64 columns of a head's state, with three products to a chunk that wait for one another:
//   [K; Q] S  (128 x 32, over K),   [T; P T] R  (128 x 32, over 64 tokens),   K^T U  (K x 32, over 64 tokens).
// The state itself stays in registers, in fp32; its products take it as a sum of bf16 numbers.
//
// What bounds it.  One prompt of 8192 tokens, 32 heads of 128 over 16: 400 us, of which unit_kernel takes some 120 and the 128 steps of sequence_kernel
// 2.2 us each.  A step is a chain: its products take 1.7 of 3.9 thousand cycles (a left side of 128 rows is 4 KB of shared memory for 16 steps of the
// sum, whatever the columns, so a product of 32 columns times three terms runs at 60 % of the rate of one of 128), and between them a row's numbers
// go from tensor memory through the registers of the two schedulers that own the keys' lanes, as three bf16 numbers each, into shared memory.  With
// two CTAs to a processor (sixteen prompts of 4096: 2.4 to 2.5 ms from box to box, 96 to 99 TFLOP/s of the recurrence's own operations) the chains overlap, and the same
// traffic of shared memory bounds: 240 KB a chunk, 1900 cycles of 3300.  Two chains in one CTA that share its tiles came out no faster, nor did
// truncated terms, stores by a warp of their own, or workspaces that the second-level cache holds (400 us -> 530, for every launch has its own start).
//
// Precision.  Keys and queries in bf16 are operands as they are (norms and decays multiply rows of the products, in fp32); in fp16 they are
// the sum of two bf16 numbers, in fp32 of three.  What is computed is split too: S, R and U into three, of whose products the terms below 2^-18 of the
// largest are left out, and T and P T into two, or three with fp32 operands.  Two are a choice: a third would be 16 KB more to a chunk, for
// which two CTAs do not fit a processor, and an entry is 2.4e-6 off in the mean, all of it behind a diagonal that is exact.  P T's products
// take two terms as well: with all of them outputs are 1.7e-6 off ahead of their rounding and not 2.7e-6 (of bf16 ones 1.3 of a thousand fall to the
// other side and not 1.9; in plain fp32 arithmetic 0.2), for 27 us more of 8192 tokens.  Beyond that, decays are good to 2^-22 (ex2.approx, of differences
// that two fp32 numbers hold) and sums on the tensor cores are cut to fp32, not rounded.  The final state is 5e-7 to 7e-7 off the
// recurrence in 64 bits, in fp32 5e-7 (outputs too; in plain fp32 arithmetic 1.5e-7 to 1.9e-7); behind strong decays among slow ones 6e-7 at most.
// Two terms throughout would leave it 3.5e-6 off, and one (plain bf16 products) 2.4e-3.
#include <cuda_pipeline_primitives.h>

#include "carry_delta.cuh"
#include "carry_tensor.cuh"

namespace carry {
namespace {

// of a chunk's factors: its decay, and behind it a number that is not 0 where a wait ran out before T was there
constexpr int kChunk = 64, kPlane = 128 * 128, kDecayAt = 4 * kChunk, kVec = kDecayAt + 8, kTerms = 3;
constexpr float kLn2 = 0.69314718055994531f, kLeastLog = -200.0f;

struct ChunkParams {
  CarryGdnPrefillArgs a;
  int b0, chunk0, chunks;   // the launch's requests begin at b0; its chunks are chunk0 .. chunk0 + chunks - 1 of every request
  int packed;               // places in the workspace follow the rows (a launch that covers everything), or requests times chunks
  int aligned, out_aligned; // rows are on the grid of 16 bytes
  uint8_t *kq, *t;          // workspace: [place][H] tiles of keys and queries, [place][HV] tiles of T and P T,
  float* vec;               // [place][HV] factors of a chunk's rows
  int* lost;                // [request of the launch][HV][D / 32] whether a wait ran out for these columns in the launches before; NULL where there is one launch
};

// A token with a key or a gate that is not a number makes the state so, from there on; products over a whole chunk must not carry that back to
// the tokens ahead of it.  So from the first such token of a chunk on (`live` are the tokens ahead of it) keys and gates count as absent, and the
// factors of its outputs and of the state are NaN.  Values are looked after column by column, where they are used.
constexpr float kNotANumber = __builtin_nanf("");

struct Place {
  int first, count;         // the request's rows
  long long slot0;          // of its chunk chunk0
};
__device__ __forceinline__ Place place_of(const ChunkParams& p, int z, int* status) {
  const int b = p.b0 + z;
  const PrefillRequest r = prefill_request(p.a, b, status);
  return {r.first, r.count, p.packed ? r.first / kChunk + b : (long long)z * p.chunks};
}

// In the test-only build warps of every kind come late to some of their chunks, by more than the others' work on one: results must not depend on
// it.  A workspace is at most 64 MiB, so that calls are worked off in turns sooner.  And there, of three value heads, the first copies of head 1's first
// chunk announce 16 bytes more than they bring: a wait runs out, and the head's rows and state are left as they were.  Of five value heads in fp32, nothing announces the end of the first product of head 1's second chunk,
// of the second one of head 2's and of the third one of head 3's,
// and some warps hold the others up for longer than a poll takes.
#ifdef CARRY_TEST_WAIT_EXPIRY
__device__ __forceinline__ void test_come_late(int warp, int c) {
  if (warp % 4 == c % 4 || (warp + c) % 5 == 0) __nanosleep(4000);
}
__device__ __forceinline__ uint32_t test_extra_bytes(int heads, int hv, int c) { return heads == 3 && hv == 1 && c == 0 ? 16 : 0; }
__device__ __forceinline__ bool test_no_commit(int heads, int hv, int chunk, int product) { return heads == 5 && hv == 1 + product && chunk == 1; }
__device__ __forceinline__ void test_hold_up(int heads, int warp) {
  if (heads == 5 && warp % 4 == 1) __nanosleep(500000);
}
#else
__device__ __forceinline__ void test_come_late(int, int) {}
__device__ __forceinline__ uint32_t test_extra_bytes(int, int, int) { return 0; }
__device__ __forceinline__ bool test_no_commit(int, int, int, int) { return false; }
__device__ __forceinline__ void test_hold_up(int, int) {}
#endif

// bf16 numbers that a key's or query's numbers come as, and those of T
template <int DTYPE>
constexpr int kTermsX = DTYPE == CARRY_BF16 ? 1 : DTYPE == CARRY_F16 ? 2 : 3;
template <int DTYPE>
constexpr int kTermsT = DTYPE == CARRY_F32 ? 3 : 2;

// two numbers' next bf16 term, which is taken off them
__device__ __forceinline__ uint32_t take_term(float2& x) {
  const uint32_t u = pack_bf16(x.x, x.y);
  x = sub2(x, make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)));
  return u;
}
// eight numbers as TERMS chunks of 16 bytes, `apart` bytes from one another
template <int TERMS>
__device__ __forceinline__ void store_terms(uint8_t* to, int apart, float2 (&x)[4]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = take_term(x[e]);
    *reinterpret_cast<uint4*>(to + t * apart) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Eight numbers of a row, in whole 16 bytes or, off that grid, one by one.
template <int DTYPE>
__device__ __forceinline__ Raw<DTYPE> load_row(const void* base, long long at, bool aligned) {
  if (aligned) return load_raw<DTYPE>(base, at);
  Raw<DTYPE> r;
  if constexpr (DTYPE == CARRY_F32) {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(base) + at;
    r.w[0] = make_uint4(q[0], q[1], q[2], q[3]);
    r.w[1] = make_uint4(q[4], q[5], q[6], q[7]);
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(base) + at;
    r.w[0] = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
  }
  return r;
}

// ---- what does not depend on the state -------------------------------------------------------------------------------
//
// For fp32 keys and queries, three bf16 numbers each, which are too many for a warp's registers.
// With D the inverses of I + L's two 32 x 32 blocks on the diagonal, N its block below them, and Y = N D (of which the first half's columns are
// not zero): T = D - D Y and P T = P D - (P D) Y.  So two products with 128 rows, [N; P] D and [D; P D] Y, finish both.

constexpr int kRowWarps = 8, kPrepareThreads = (kRowWarps + 1) * 32, kHalf = kChunk / 2, kPad = 36;

template <int D>
struct PrepareShared {
  union {
    uint8_t kq[kTermsX<CARRY_F32>][D / 64][kPlane];   // rows 0 .. 63 keys, 64 .. 127 queries
    uint8_t np[kTerms][kPlane];           // when they are multiplied: rows 0 .. 63 N, then Y; 64 .. 127 P
  };
  uint8_t t[kTerms][kPlane];              // rows 0 .. 63 D, then T; 64 .. 127 P D, then P T
  alignas(16) float L[2][kHalf][kPad];    // the blocks of L on the diagonal
  // of a token: running sum of log2 alpha within its half, as two numbers; decay from the first half's token to that half's end, or from there to the
  // second half's token; decays from the chunk's start to the token and from there to the chunk's end; beta
  alignas(16) float G[kChunk], G_less[kChunk], to_middle[kChunk], from_start[kChunk], to_end[kChunk], beta[kChunk];
  alignas(16) float norm[2 * kChunk];     // what makes a key a unit one, and a query one times `scale`
  int live_keys[kRowWarps], live_gates;
  float decay;                            // of the chunk
  uint64_t done[3];
  uint32_t tmem;
  int poison;
};

__device__ __forceinline__ float exp2_quick(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_of(double x) {
  const float hi = (float)x;
  return exp2_quick(hi) * fmaf((float)(x - hi), kLn2, 1.0f);
}

// A running sum of log2 alpha as two fp32 numbers, some 48 bits.  A decay is the exponential of a difference of two such sums, and a strong decay
// ahead of both tokens makes the sums large without changing the difference: with one number each, of sums near 1000, it would be 6e-5 off.
__device__ __forceinline__ void two_numbers(double x, float& hi, float& lo) {
  hi = (float)x;
  lo = (float)(x - hi);
}

// A chunk's gates, by one warp; lane l has tokens 2 l and 2 l + 1.  Sums of decays are formed in 64 bits; what is kept of them, for
// differences, is the sum within half a chunk.
template <class Shared>
__device__ __forceinline__ void chunk_gates(const ChunkParams& p, Shared& sh, long long row, int n, int hv) {
  const int lane = threadIdx.x % 32;
  float log_alpha[2] = {}, beta[2] = {};
  int bad = n;
#pragma unroll
  for (int e = 1; e >= 0; --e) {
    if (2 * lane + e < n) prefill_gates(p.a, row + 2 * lane + e, hv, log_alpha[e], beta[e]);
    if (isnan(log_alpha[e]) || isnan(beta[e])) bad = 2 * lane + e;
  }
  const int live = __reduce_min_sync(~0u, bad);
  if (lane == 0) sh.live_gates = live;
  double g[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool there = 2 * lane + e < live;
    g[e] = there ? (double)(log_alpha[e] < kLeastLog ? kLeastLog : log_alpha[e]) * 1.4426950408889634 : 0.0;     // exp(-200) is 0, and sums stay finite
    sh.beta[2 * lane + e] = there ? beta[e] : 0.0f;
  }
  double sum = g[0] + g[1];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const double below = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += below;
  }
  const double G[2] = {sum - g[1], sum}, middle = __shfl_sync(~0u, sum, kHalf / 2 - 1), last = __shfl_sync(~0u, sum, 31);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    two_numbers(i < kHalf ? G[e] : G[e] - middle, sh.G[i], sh.G_less[i]);
    sh.to_middle[i] = exp2_of(i < kHalf ? middle - G[e] : G[e] - middle);
    sh.from_start[i] = exp2_of(G[e]);
    sh.to_end[i] = exp2_of(last - G[e]);
  }
  if (lane == 0) sh.decay = exp2_of(last);
}

// The inverse of a 32 x 32 block of I + L on the diagonal by substitution, a column to a lane, in fp32; its terms go into the tile of D.
template <class Shared>
__device__ __forceinline__ void invert_block(Shared& sh, int block) {
  const int lane = threadIdx.x % 32;
  float x[kHalf];
#pragma unroll
  for (int i = 0; i < kHalf; ++i) {
    float s[4] = {i == lane ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < i; k += 4) {
      const float4 l = *reinterpret_cast<const float4*>(&sh.L[block][i][k]);
      s[0] = fmaf(-l.x, x[k], s[0]);
      if (k + 1 < i) s[1] = fmaf(-l.y, x[k + 1], s[1]);
      if (k + 2 < i) s[2] = fmaf(-l.z, x[k + 2], s[2]);
      if (k + 3 < i) s[3] = fmaf(-l.w, x[k + 3], s[3]);
    }
    x[i] = (s[0] + s[1]) + (s[2] + s[3]);
  }
  const int chunk = block * kHalf / 8 + lane / 8;
  uint8_t* to = sh.t[0] + block * kHalf * 128 + lane % 8 * 2;
#pragma unroll
  for (int i = 0; i < kHalf; i += 2) {
    float2 y = make_float2(x[i], x[i + 1]);
#pragma unroll
    for (int t = 0; t < kTerms; ++t) {
      const uint32_t w = take_term(y);
      *reinterpret_cast<uint16_t*>(to + t * kPlane + plane_at(i, chunk)) = (uint16_t)w;
      *reinterpret_cast<uint16_t*>(to + t * kPlane + plane_at(i + 1, chunk)) = (uint16_t)(w >> 16);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kPrepareThreads, 2) prepare_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kX = kTermsX<CARRY_F32>, kT = kTermsT<CARRY_F32>, kPlanes = D / 64;
  static_assert(kT == kTerms, "T is left in the terms that it is worked out in");
  using Shared = PrepareShared<D>;
  extern __shared__ uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
  depend_release();
  depend_wait();
  const CarryGdnPrefillArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hv = blockIdx.y, group = a.HV / a.H, h = hv / group, c = blockIdx.x;
  const Place place = place_of(p, blockIdx.z, tid == 0 && hv == 0 && c == 0 && p.chunk0 == 0 ? a.status : nullptr);
  const int from = (p.chunk0 + c) * kChunk, n = min(place.count - from, kChunk);
  if (n <= 0) return;
  const long long row0 = place.first + from, slot = place.slot0 + c;

  if (warp < kRowWarps) {
    // keys and queries as operands; rows behind the last token are zeros, whatever memory holds there
    constexpr int kLanes = D / 8, kRows = 32 / kLanes, kTurns = 2 * kChunk / (kRowWarps * kRows), kBatch = 4;
    const int chunk = lane % kLanes, first = warp * kRows + lane / kLanes;
    int bad = n;
#pragma unroll
    for (int t0 = 0; t0 < kTurns; t0 += kBatch) {
      Raw<CARRY_F32> x[kBatch];
#pragma unroll
      for (int t = 0; t < kBatch; ++t) {
        const int row = first + (t0 + t) * kRowWarps * kRows, token = row % kChunk;
        x[t] = {};
        if (token < n) x[t] = load_row<CARRY_F32>(a.mixed_qkv, (row0 + token) * a.stride_mixed_tok + (row < kChunk ? a.H + h : h) * D + chunk * 8, p.aligned);
      }
#pragma unroll
      for (int t = 0; t < kBatch; ++t) {
        const int row = first + (t0 + t) * kRowWarps * kRows;
        Eight e = unpack<CARRY_F32>(x[t]);
        if (row < kChunk) {
          const float2 zero = make_float2(0.0f, 0.0f), none = fma2(e.x[0], zero, fma2(e.x[1], zero, fma2(e.x[2], zero, mul2(e.x[3], zero))));
          if (!(none.x + none.y == 0.0f)) bad = min(bad, row);
        }
        store_terms<kX>(sh.kq[0][chunk / 8] + plane_at(row, chunk % 8), kPlanes * kPlane, e.x);
      }
    }
    bad = __reduce_min_sync(~0u, bad);
    if (lane == 0) sh.live_keys[warp] = bad;
    fence_proxy();
  } else {
    if (lane == 0) {
      sh.poison = 0;
      for (int i = 0; i < 3; ++i) barrier_init(&sh.done[i], 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 128;" ::"r"(smem_addr(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    chunk_gates(p, sh, row0, n, hv);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* poison = &sh.poison;
  // the whole CTA goes on, or none of it
  auto wait = [&](int i) { return !__syncthreads_or(!barrier_wait(&sh.done[i], 0, poison, a.status)); };
  const uint32_t elected = warp == kRowWarps ? elect() : 0, base = __shfl_sync(~0u, tmem, 0);
  int live = n;
#pragma unroll
  for (int i = 0; i < kRowWarps; ++i) live = min(live, sh.live_keys[i]);
  if (live < n) {                                 // the same for all
    if (warp == kRowWarps) chunk_gates(p, sh, row0, live, hv);
    for (int i = tid; i < kX * kPlanes * kChunk * 8; i += kPrepareThreads)
      if (i / 8 % kChunk >= live) *reinterpret_cast<uint4*>(sh.kq[0][0] + i / (kChunk * 8) * kPlane + i % (kChunk * 8) * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy();
    fence_before();
    __syncthreads();
    fence_after();
  }
  live = min(live, sh.live_gates);

  // Sums on the tensor cores are cut to fp32, not rounded, after every product of sixteen columns, so that errors add up to one side: the products
  // of the smallest terms go first, and only those of the largest are cut at the sum's own size (the other way round a norm of 128 numbers was 1.7e-6 off).
  if (warp == kRowWarps) {                        // [K; Q] [K; Q]^T: the norms are on its diagonal
#pragma unroll
    for (int terms = 2 * kX - 2; terms >= 0; --terms)
#pragma unroll
      for (int x = terms < kX ? 0 : terms - kX + 1; x < kX && x <= terms; ++x)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t step = k / 4 * (kPlane / 16) + k % 4 * 2;
          mma_shared(elected, base, operand(sh.kq[x], 16) + step, operand(sh.kq[terms - x], 16) + step, instruction_bf16(2 * kChunk, false, false),
                     terms < 2 * kX - 2 || k > 0);
        }
    if (!test_no_commit(a.HV, hv, p.chunk0 + c, 0)) mma_commit(elected, &sh.done[0]);
    if (lane == 0 && hv % group == 0) {
      bulk_store(p.kq + (slot * a.H + h) * (kX * kPlanes * kPlane), sh.kq, kX * kPlanes * kPlane);
      bulk_commit();
      bulk_wait_read();
    }
    __syncwarp();
  } else {                                        // zeros beside the blocks of D
#pragma unroll
    for (int t = 0; t < kTerms; ++t) {
      const int row = tid / 4;
      *reinterpret_cast<uint4*>(sh.t[t] + plane_at(row, (row < kHalf ? 4 : 0) + tid % 4)) = make_uint4(0, 0, 0, 0);
    }
  }
  float* const vec = p.vec + (slot * a.HV + hv) * kVec;
  if (!wait(0)) {
    if (tid == 0) vec[kDecayAt + 1] = 1.0f;
    if (*poison)
      for (int k = 0; k < 1 << 12; ++k) __nanosleep(64);    // products in flight still use shared and tensor memory
    __syncthreads();
    if (warp == kRowWarps) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 128;" ::"r"(tmem) : "memory");
    return;
  }
  fence_after();
  // a row to a thread, half of its columns
  const int quarter = warp % 4, row = quarter * 32 + lane, i = row % kChunk, first = warp / 4 * kHalf;
  const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const bool key = row < kChunk;
  if (warp < 4) {
    float x[32], square = 0.0f;
    tmem_load(at + quarter * 32, x);
    wait_loads();
#pragma unroll
    for (int j = 0; j < 32; ++j) square = j == lane ? x[j] : square;
    sh.norm[row] = (a.use_qk_l2norm ? norm_factor(square, 1.0f) : 1.0f) * (key ? 1.0f : a.scale);
  }
  __syncthreads();
  if (warp < kRowWarps) {
    // L and P.  Between the halves of a chunk a decay is a product of two that end in the middle; both are at most 1.
    const float G = sh.G[i], G_less = sh.G_less[i], by = key ? sh.beta[i] * sh.norm[i] : sh.norm[row];
    const bool below = first < i / kHalf * kHalf, diagonal = first == i / kHalf * kHalf;    // the same for all lanes
    float2 x[16];
    if (below || diagonal) {
      tmem_load(at + first, *reinterpret_cast<float(*)[32]>(x));
      wait_loads();
    }
    if (diagonal) {
      const int most = (key ? i - 1 : i) - first;
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 g = *reinterpret_cast<const float4*>(&sh.G[first + j]), m = *reinterpret_cast<const float4*>(&sh.norm[first + j]);
        const float4 l = *reinterpret_cast<const float4*>(&sh.G_less[first + j]);
        const float2 d[2] = {make_float2(exp2_quick(G - g.x + (G_less - l.x)), exp2_quick(G - g.y + (G_less - l.y))),
                             make_float2(exp2_quick(G - g.z + (G_less - l.z)), exp2_quick(G - g.w + (G_less - l.w)))};
        const float2 f[2] = {make_float2(m.x, m.y), make_float2(m.z, m.w)};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 y = mul2(mul2(x[j / 2 + e], mul2(f[e], make_float2(by, by))), d[e]);
          x[j / 2 + e] = make_float2(j + 2 * e <= most ? y.x : 0.0f, j + 2 * e + 1 <= most ? y.y : 0.0f);
        }
      }
    } else if (below) {
      const float f = by * sh.to_middle[i];
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 d = *reinterpret_cast<const float4*>(&sh.to_middle[j]), m = *reinterpret_cast<const float4*>(&sh.norm[j]);
        x[j / 2] = mul2(mul2(x[j / 2], make_float2(f, f)), make_float2(m.x * d.x, m.y * d.y));
        x[j / 2 + 1] = mul2(mul2(x[j / 2 + 1], make_float2(f, f)), make_float2(m.z * d.z, m.w * d.w));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = make_float2(0.0f, 0.0f);
    }
    auto tile = [&](int to_row, int column) {     // the thread's numbers into the tile of N and P
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        float2 y[4] = {x[j], x[j + 1], x[j + 2], x[j + 3]};
        store_terms<kTerms>(sh.np[0] + plane_at(to_row, column / 8 + j / 4), kPlane, y);
      }
    };
    if (!key) {
      tile(row, first);
    } else if (diagonal) {
#pragma unroll
      for (int j = 0; j < 16; j += 2) *reinterpret_cast<float4*>(&sh.L[i / kHalf][lane][2 * j]) = make_float4(x[j].x, x[j].y, x[j + 1].x, x[j + 1].y);
    } else if (below) {
      tile(row, 0);
    } else {                                      // N's other places
      tile(lane, 0);
      tile(lane, kHalf);
      tile(lane + kHalf, kHalf);
    }
  }
  __syncthreads();
  if (warp < 2) {
    invert_block(sh, warp);
  } else if (warp < 4) {                          // the factors of the chunk's rows
    const int i = tid - 64;
    const bool there = i < live;
    vec[i] = there ? sh.beta[i] * sh.from_start[i] * sh.norm[i] : 0.0f;
    vec[kChunk + i] = sh.beta[i];
    vec[2 * kChunk + i] = there ? sh.to_end[i] * sh.norm[i] : 0.0f;
    vec[3 * kChunk + i] = there ? sh.from_start[i] * sh.norm[kChunk + i] : i < n ? kNotANumber : 0.0f;
    if (i < 8) vec[kDecayAt + i] = i > 0 ? 0.0f : live < n ? kNotANumber : sh.decay;
  }
  fence_proxy();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kRowWarps) {                        // [N; P] D
#pragma unroll
    for (int terms = kTerms - 1; terms >= 0; --terms)
#pragma unroll
      for (int x = 0; x <= terms; ++x)
#pragma unroll
        for (int k = 0; k < kChunk / 16; ++k)
          mma_shared(elected, base, operand(sh.np[x], 16) + k * 2, operand(sh.t[terms - x], 16) + k * 128, instruction_bf16(kChunk, false, true),
                     terms < kTerms - 1 || x + k > 0);
    if (!test_no_commit(a.HV, hv, p.chunk0 + c, 1)) mma_commit(elected, &sh.done[1]);
  }
  bool healthy = wait(1);
  float2 pd[16];
  if (healthy && warp < kRowWarps && (!key || (quarter == 1 && first == 0))) {
    fence_after();
    tmem_load(at + first, *reinterpret_cast<float(*)[32]>(pd));
    wait_loads();
    uint8_t* tile = key ? sh.np[0] : sh.t[0];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      float2 y[4] = {pd[j], pd[j + 1], pd[j + 2], pd[j + 3]};
      store_terms<kTerms>(tile + plane_at(row, first / 8 + j / 4), kPlane, y);
    }
    fence_proxy();
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kRowWarps) {                        // [D; P D] Y, over the second half
#pragma unroll
    for (int terms = kTerms - 1; terms >= 0; --terms)
#pragma unroll
      for (int x = 0; x <= terms; ++x)
#pragma unroll
        for (int k = kHalf / 16; k < kChunk / 16; ++k)
          mma_shared(elected, base + kChunk, operand(sh.t[x], 16) + k * 2, operand(sh.np[terms - x], 16) + k * 128, instruction_bf16(kHalf, false, true),
                     terms < kTerms - 1 || x > 0 || k > kHalf / 16);
    if (!test_no_commit(a.HV, hv, p.chunk0 + c, 2)) mma_commit(elected, &sh.done[2]);
  }
  healthy = wait(2) && healthy;
  if (healthy && warp < 4 && quarter > 0) {       // the first half's columns of T's rows below the middle, and of P T
    fence_after();
    float2 y[16];
    tmem_load(at + kChunk, *reinterpret_cast<float(*)[32]>(y));
    wait_loads();
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      float2 z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = sub2(key ? make_float2(0.0f, 0.0f) : pd[j + e], y[j + e]);
      store_terms<kT>(sh.t[0] + plane_at(row, j / 4), kPlane, z);
    }
    fence_proxy();
  }
  if (*poison)
    for (int k = 0; k < 1 << 12; ++k) __nanosleep(64);
  fence_before();
  __syncthreads();
  fence_after();
  if (tid == 0 && !healthy) vec[kDecayAt + 1] = 1.0f;
  if (warp == kRowWarps) {
    if (lane == 0 && healthy) {
      bulk_store(p.t + (slot * a.HV + hv) * (kT * kPlane), sh.t, kT * kPlane);
      bulk_commit();
      bulk_wait_read();
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 128;" ::"r"(tmem) : "memory");
  }
}

// ---- the same, a chunk and head to a warp ----------------------------------------------------------------------------
//
// For 16-bit keys and queries; 6300 instructions a warp, two warps to a scheduler (keys alone take half of a thread's registers), 29 ns a chunk and
// head over the whole GPU.  What bounds it is latency: an instruction in 4.4 cycles.  The form by tensor memory that fp32 has takes 44 ns.
// Everything is a product of 16 x 16 blocks whose operands are registers: a lane's part of a product's result
// is its part of the next one's left side, or of its right side transposed, so T^T and (P T)^T are built block by block,
//   W_jj = D_j^T,   W_jb = -(sum over j <= k < b of W_jk L_bk^T) D_b^T  (T_bj = W_jb^T),   (P T)_ij = (sum over j <= k <= i of W_jk P_ik^T)^T,
// and only the 16 x 16 inverses D_b go through shared memory.  No warp waits for another.  Keys and queries come from memory as they
// are: a lane has a quarter of a row, and which numbers of a row stand for which step of the sum is the same on both sides.

constexpr int kBlock = 16, kBlocks = kChunk / kBlock, kUnitWarps = 4;
__host__ __device__ constexpr int pair_of(int i, int k) { return i * (i + 1) / 2 + k; }        // of blocks, k <= i

struct alignas(16) Unit {
  float2 L[6][4][32], P[10][4][32];       // a lane's numbers of the blocks below the diagonal, and of all
  float D[kBlocks][kBlock][20];           // the blocks of L on the diagonal, then their inverses
  uint8_t rows[2][kBlock * 128];          // sixteen rows of a tile on their way out
  // of a token: running sum of log2 alpha within its block, as two numbers, decay from the block's start, decay to the block's end, decays from the
  // chunk's start and to its end, beta, norms of key and query
  float G[kChunk], G_less[kChunk], from_block[kChunk], to_block[kChunk], from_start[kChunk], to_end[kChunk], beta[kChunk], key[kChunk], query[kChunk];
};

template <bool HALF>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A lane's part of a 16 x 16 block, of which it has numbers (g, 2t), (g, 2t+1), (g+8, 2t), .. and the same eight columns on: for g = lane / 4,
// t = lane % 4.
struct Part {
  float x[2][4];
};
struct Split {
  uint32_t w[kTerms][4];                  // pairs (g, 2t), (g + 8, 2t), (g, 2t + 8), (g + 8, 2t + 8)
};
__device__ __forceinline__ Split split(const Part& p) {
  Split s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 y = make_float2(p.x[i / 2][i % 2 * 2], p.x[i / 2][i % 2 * 2 + 1]);
#pragma unroll
    for (int t = 0; t < kTerms; ++t) s.w[t][i] = take_term(y);
  }
  return s;
}
// c += a b^T, of terms whose numbers add up to less than TERMS: what is left out is 2^-27 of it with three, 2^-18 with two
template <int TERMS>
__device__ __forceinline__ void multiply(Part& c, const Split& a, const Split& b) {
#pragma unroll
  for (int x = TERMS - 1; x >= 0; --x)
#pragma unroll
    for (int y = TERMS - 1 - x; y >= 0; --y) {
      mma16<false>(c.x[0], a.w[x][0], a.w[x][1], a.w[x][2], a.w[x][3], b.w[y][0], b.w[y][2]);
      mma16<false>(c.x[1], a.w[x][0], a.w[x][1], a.w[x][2], a.w[x][3], b.w[y][1], b.w[y][3]);
    }
}
__device__ __forceinline__ void store_transposed(uint32_t to, const uint32_t (&w)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

// Gates of a chunk: lane l has tokens 2 l and 2 l + 1, whose inputs it has read.  Sums of decays are formed in 64 bits; what is kept of
// them, for differences, is the sum within a block.  `live`: tokens that count; less, when a gate among them is no number.  Returns the decays over
// the second block, over the third, and over the chunk.
__device__ __forceinline__ float3 unit_gates(Unit& sh, const GateInputs (&in)[2], int& live) {
  const int lane = threadIdx.x % 32;
  float log_alpha[2], beta[2];
  int bad = live;
#pragma unroll
  for (int e = 1; e >= 0; --e) {
    gates_of(in[e], log_alpha[e], beta[e]);
    if (2 * lane + e < live && (isnan(log_alpha[e]) || isnan(beta[e]))) bad = 2 * lane + e;
  }
  live = __reduce_min_sync(~0u, bad);
  double g[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool there = 2 * lane + e < live;
    g[e] = there ? (double)(log_alpha[e] < kLeastLog ? kLeastLog : log_alpha[e]) * 1.4426950408889634 : 0.0;     // exp(-200) is 0, and sums stay finite
    sh.beta[2 * lane + e] = there ? beta[e] : 0.0f;
  }
  double sum = g[0] + g[1];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const double below = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += below;
  }
  const double G[2] = {sum - g[1], sum}, last = __shfl_sync(~0u, sum, 31), end = __shfl_sync(~0u, sum, lane | 7);
  const double before = __shfl_sync(~0u, sum, (lane & 24) - 1 & 31), start = lane < 8 ? 0.0 : before;
  const double ends[3] = {__shfl_sync(~0u, sum, 7), __shfl_sync(~0u, sum, 15), __shfl_sync(~0u, sum, 23)};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    two_numbers(G[e] - start, sh.G[i], sh.G_less[i]);
    sh.from_block[i] = exp2_of(G[e] - start);
    sh.to_block[i] = exp2_of(end - G[e]);
    sh.from_start[i] = exp2_of(G[e]);
    sh.to_end[i] = exp2_of(last - G[e]);
  }
  return make_float3(exp2_of(ends[1] - ends[0]), exp2_of(ends[2] - ends[1]), exp2_of(last));
}

// Rows of keys or queries, for a lane a quarter of row first + 8 r + lane / 4 (r < ROWS), D / 4 numbers as they lie in memory; rows behind the
// last token are zeros, whatever memory holds there.
template <int D, int ROWS>
__device__ __forceinline__ void load_quarters(const ChunkParams& p, long long row0, int n, int first, long long column, uint32_t (&x)[ROWS][D / 8]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int token = first + 8 * r + lane / 4;
    const long long at = (row0 + token) * p.a.stride_mixed_tok + column + lane % 4 * (D / 4);
#pragma unroll
    for (int q = 0; q < D / 32; ++q) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (token < n) u = load_row<CARRY_BF16>(p.a.mixed_qkv, at + q * 8, p.aligned).w[0];
      x[r][4 * q] = u.x;
      x[r][4 * q + 1] = u.y;
      x[r][4 * q + 2] = u.z;
      x[r][4 * q + 3] = u.w;
    }
  }
}
// them as operand rows in the workspace; row: of the tile
template <int DTYPE, int D>
__device__ __forceinline__ void store_quarter(uint8_t* tile, int row, const uint32_t (&x)[D / 8]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int q = 0; q < D / 32; ++q) {
    const int chunk = lane % 4 * (D / 32) + q;
    uint8_t* to = tile + chunk / 8 * kPlane + plane_at(row, chunk % 8);
    if constexpr (DTYPE == CARRY_BF16) {
      *reinterpret_cast<uint4*>(to) = make_uint4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
    } else {
      Raw<DTYPE> r;
      r.w[0] = make_uint4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
      Eight e = unpack<DTYPE>(r);
      store_terms<kTermsX<DTYPE>>(to, D / 64 * kPlane, e.x);
    }
  }
}
// products of sixteen rows with sixteen
template <bool HALF, int N>
__device__ __forceinline__ Part products(const uint32_t (&a0)[N], const uint32_t (&a1)[N], const uint32_t (&b0)[N], const uint32_t (&b1)[N]) {
  Part c = {};
#pragma unroll
  for (int s = 0; s < N; s += 2) {
    mma16<HALF>(c.x[0], a0[s], a1[s], a0[s + 1], a1[s + 1], b0[s], b0[s + 1]);
    mma16<HALF>(c.x[1], a0[s], a1[s], a0[s + 1], a1[s + 1], b1[s], b1[s + 1]);
  }
  return c;
}

template <int DTYPE, int D>
__global__ void __launch_bounds__(kUnitWarps * 32, 2) unit_kernel(const __grid_constant__ ChunkParams p) {
  constexpr bool kHalfType = DTYPE == CARRY_F16;
  constexpr int kWords = D / 8;
  extern __shared__ uint8_t raw[];
  depend_release();
  depend_wait();
  const CarryGdnPrefillArgs& a = p.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int hv = blockIdx.y, group = a.HV / a.H, h = hv / group, c = blockIdx.x * kUnitWarps + warp;
  Unit& sh = reinterpret_cast<Unit*>(raw)[warp];
  const Place place = place_of(p, blockIdx.z, threadIdx.x == 0 && hv == 0 && c == 0 && p.chunk0 == 0 ? a.status : nullptr);
  const int from = (p.chunk0 + c) * kChunk, n = c < p.chunks ? min(place.count - from, kChunk) : 0;
  if (n <= 0) return;
  const long long row0 = place.first + from, slot = place.slot0 + c;
  uint8_t* kq = hv % group == 0 ? p.kq + (slot * a.H + h) * (kTermsX<DTYPE> * (D / 64) * kPlane) : nullptr;

  uint32_t k[2 * kBlocks][kWords];
  load_quarters<D>(p, row0, n, 0, (a.H + h) * D, k);
  GateInputs gate[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) gate[e] = gate_inputs(a, row0 + min(2 * lane + e, n - 1), hv);

  // The norms are on the diagonals of products with themselves: of rows g and g + 8, at the lane with t = g / 2.
  auto square = [&](const Part& d, int half) { return g % 2 ? d.x[half][2 * half + 1] : d.x[half][2 * half]; };
  auto norms = [&](const Part& d, float by, float* to) {
    if (t != g / 2) return;
#pragma unroll
    for (int half = 0; half < 2; ++half) to[g + 8 * half] = a.use_qk_l2norm ? norm_factor(square(d, half), by) : by;
  };
  Part diagonal[kBlocks];
  int live = n;
#pragma unroll
  for (int b = kBlocks - 1; b >= 0; --b) {
    diagonal[b] = products<kHalfType>(k[2 * b], k[2 * b + 1], k[2 * b], k[2 * b + 1]);
#pragma unroll
    for (int half = 1; half >= 0; --half)
      if (t == g / 2 && !(square(diagonal[b], half) < INFINITY)) live = b * kBlock + g + 8 * half;
  }
  live = __reduce_min_sync(~0u, live);
  if (!kHalfType && live < n && !a.use_qk_l2norm) {
    // squares beyond fp32, which fp16's are not, matter to the norm alone: what is not finite is what products with zeros leave
    live = n;
#pragma unroll
    for (int b = kBlocks - 1; b >= 0; --b) {
      float none[4] = {};
#pragma unroll
      for (int s = 0; s < kWords; s += 2) mma16<kHalfType>(none, k[2 * b][s], k[2 * b + 1][s], k[2 * b][s + 1], k[2 * b + 1][s + 1], 0, 0);
#pragma unroll
      for (int half = 1; half >= 0; --half)
        if (none[2 * half] != 0.0f) live = b * kBlock + g + 8 * half;
    }
    live = __reduce_min_sync(~0u, live);
  }
  if (live < n) {                                 // the same for all lanes
#pragma unroll
    for (int r = 0; r < 2 * kBlocks; ++r)
#pragma unroll
      for (int e = 0; e < kWords; ++e) k[r][e] = 8 * r + g < live ? k[r][e] : 0;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) diagonal[b] = products<kHalfType>(k[2 * b], k[2 * b + 1], k[2 * b], k[2 * b + 1]);
  }
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) norms(diagonal[b], 1.0f, sh.key + b * kBlock);
  if (kq) {
#pragma unroll
    for (int r = 0; r < 2 * kBlocks; ++r) store_quarter<DTYPE, D>(kq, 8 * r + g, k[r]);
  }
  const float3 across = unit_gates(sh, gate, live);
  __syncwarp();

  // L and P, a row of blocks at a time.  Within a block decays are powers of differences; between blocks products of a decay to the one's end, over
  // what lies between, and from the other's start, all at most 1.
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int i0 = b * kBlock + g;
    uint32_t q[2][kWords];
    load_quarters<D>(p, row0, n, b * kBlock, h * D, q);
    float decay[2][4];
    {
      const float gi[2] = {sh.G[i0], sh.G[i0 + 8]}, less[2] = {sh.G_less[i0], sh.G_less[i0 + 8]}, by[2] = {sh.beta[i0] * sh.key[i0], sh.beta[i0 + 8] * sh.key[i0 + 8]};
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 8 * x + 2 * t + e % 2, i = g + e / 2 * 8;
          decay[x][e] = j <= i ? exp2_quick(gi[e / 2] - sh.G[b * kBlock + j] + (less[e / 2] - sh.G_less[b * kBlock + j])) * sh.key[b * kBlock + j] : 0.0f;
          sh.D[b][i][j] = j < i ? diagonal[b].x[x][e] * by[e / 2] * decay[x][e] : 0.0f;
        }
#pragma unroll
      for (int m = 0; m < b; ++m) {
        Part l = products<kHalfType>(k[2 * b], k[2 * b + 1], k[2 * m], k[2 * m + 1]);
        const float over = m == b - 1 ? 1.0f : b == 2 ? across.x : m == 1 ? across.y : across.x * across.y;
        const float f[2] = {by[0] * sh.from_block[i0] * over, by[1] * sh.from_block[i0 + 8] * over};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int j = m * kBlock + 8 * x + 2 * t;
          const float2 to = mul2(*reinterpret_cast<const float2*>(&sh.to_block[j]), *reinterpret_cast<const float2*>(&sh.key[j]));
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sh.L[pair_of(b - 1, m)][2 * x + e][lane] = mul2(mul2(make_float2(l.x[x][2 * e], l.x[x][2 * e + 1]), make_float2(f[e], f[e])), to);
        }
      }
    }
    if (kq) {
      store_quarter<DTYPE, D>(kq, kChunk + i0, q[0]);
      store_quarter<DTYPE, D>(kq, kChunk + i0 + 8, q[1]);
    }
    norms(products<kHalfType>(q[0], q[1], q[0], q[1]), a.scale, sh.query + b * kBlock);
    __syncwarp();
    const float by[2] = {sh.query[i0], sh.query[i0 + 8]};
#pragma unroll
    for (int m = 0; m <= b; ++m) {
      Part y = products<kHalfType>(q[0], q[1], k[2 * m], k[2 * m + 1]);
      const float over = m >= b - 1 ? 1.0f : b == 2 ? across.x : m == 1 ? across.y : across.x * across.y;
      const float f[2] = {by[0] * sh.from_block[i0] * over, by[1] * sh.from_block[i0 + 8] * over};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int j = m * kBlock + 8 * x + 2 * t;
        const float2 to = mul2(*reinterpret_cast<const float2*>(&sh.to_block[j]), *reinterpret_cast<const float2*>(&sh.key[j]));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 z = make_float2(y.x[x][2 * e], y.x[x][2 * e + 1]);
          const float2 d = make_float2(decay[x][2 * e], decay[x][2 * e + 1]), s = make_float2(by[e], by[e]);
          sh.P[pair_of(b, m)][2 * x + e][lane] = m == b ? make_float2(d.x == 0.0f ? 0.0f : z.x * s.x * d.x, d.y == 0.0f ? 0.0f : z.y * s.y * d.y)
                                                        : mul2(mul2(z, make_float2(f[e], f[e])), to);
        }
      }
    }
  }
  __syncwarp();
  {
    // the factors of the chunk's rows
    float* vec = p.vec + (slot * a.HV + hv) * kVec;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = lane + 32 * e;
      const bool there = i < live;
      vec[i] = there ? sh.beta[i] * sh.from_start[i] * sh.key[i] : 0.0f;
      vec[kChunk + i] = sh.beta[i];
      vec[2 * kChunk + i] = there ? sh.to_end[i] * sh.key[i] : 0.0f;
      vec[3 * kChunk + i] = there ? sh.from_start[i] * sh.query[i] : i < n ? kNotANumber : 0.0f;
    }
    if (lane < 8) vec[kDecayAt + lane] = lane > 0 ? 0.0f : live < n ? kNotANumber : across.z;
  }

  // The inverses of the blocks on the diagonal, by substitution, a column to a lane, two blocks at a time.
#pragma unroll
  for (int b = 0; b < kBlocks; b += 2) {
    float (&m)[kBlock][20] = sh.D[b + lane / 16];
    const int j = lane % 16;
    float x[kBlock];
#pragma unroll
    for (int i = 0; i < kBlock; ++i) {
      float s[4] = {i == j ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < i; n += 4) {
        const float4 l = *reinterpret_cast<const float4*>(&m[i][n]);
        s[0] = fmaf(-l.x, x[n], s[0]);
        if (n + 1 < i) s[1] = fmaf(-l.y, x[n + 1], s[1]);
        if (n + 2 < i) s[2] = fmaf(-l.z, x[n + 2], s[2]);
        if (n + 3 < i) s[3] = fmaf(-l.w, x[n + 3], s[3]);
      }
      x[i] = (s[0] + s[1]) + (s[2] + s[3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kBlock; ++i) m[i][j] = x[i];
  }
  __syncwarp();

  Split W[10];                                    // W_jb at pair_of(b, j)
  uint8_t* tile = p.t + (slot * a.HV + hv) * (kTermsT<DTYPE> * kPlane);
  const uint32_t staged = smem_addr(sh.rows[0]);
  // sixteen rows, of which blocks 0 .. b are given, into the tile
  auto put_rows = [&](int b, int row, auto block) {
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
      const int r = lane % 8 + lane / 16 * 8, chunk = 2 * j + lane / 8 % 2;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (j <= b) store_transposed(staged + x * (kBlock * 128) + plane_at(r, chunk), block(j).w[x]);
        else *reinterpret_cast<uint4*>(sh.rows[x] + plane_at(r, chunk)) = make_uint4(0, 0, 0, 0);
      }
    }
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<uint4*>(tile + x * kPlane + row * 128 + (e * 32 + lane) * 16) = *reinterpret_cast<const uint4*>(sh.rows[x] + (e * 32 + lane) * 16);
    __syncwarp();
  };
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const float (&m)[kBlock][20] = sh.D[b];
    Part d, turned;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = g + e / 2 * 8, j = 8 * x + 2 * t + e % 2;
        d.x[x][e] = m[i][j];
        turned.x[x][e] = m[j][i];
      }
    W[pair_of(b, b)] = split(turned);
    if (b > 0) {
      const Split inverse = split(d);
      Split l[kBlocks];
#pragma unroll
      for (int k = 0; k < b; ++k) {
        Part y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 z = sh.L[pair_of(b - 1, k)][e][lane];
          y.x[e / 2][e % 2 * 2] = z.x;
          y.x[e / 2][e % 2 * 2 + 1] = z.y;
        }
        l[k] = split(y);
      }
#pragma unroll
      for (int j = 0; j < b; ++j) {
        Part sum = {}, w = {};
#pragma unroll
        for (int k = j; k < b; ++k) multiply<kTerms>(sum, W[pair_of(k, j)], l[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum.x[e / 4][e % 4] = -sum.x[e / 4][e % 4];
        multiply<kTerms>(w, split(sum), inverse);
        W[pair_of(b, j)] = split(w);
      }
    }
    put_rows(b, b * kBlock, [&](int j) -> const Split& { return W[pair_of(b, j)]; });
    Split pt[kBlocks];
    {
      Part sum[kBlocks] = {};
#pragma unroll
      for (int k = 0; k <= b; ++k) {
        Part y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 z = sh.P[pair_of(b, k)][e][lane];
          y.x[e / 2][e % 2 * 2] = z.x;
          y.x[e / 2][e % 2 * 2 + 1] = z.y;
        }
        const Split right = split(y);
#pragma unroll
        for (int j = 0; j <= k; ++j) multiply<2>(sum[j], W[pair_of(k, j)], right);
      }
#pragma unroll
      for (int j = 0; j <= b; ++j) pt[j] = split(sum[j]);
    }
    put_rows(b, kChunk + b * kBlock, [&](int j) -> const Split& { return pt[j]; });
  }
}

// ---- along a sequence ------------------------------------------------------------------------------------------------

// A CTA has 32 or 64 columns of a head's state.  Right sides lie with their three terms side by side, so that one product takes all terms and
// reads its left side once: each in a plane of 64 columns, or two of 32 in one and the third in the first half of another.  Where two CTAs share
// a processor, the second half of the state's other plane has the third term of R and U.
template <int DTYPE, int D, int STAGES, int COLUMNS>
struct SequenceShared {
  static constexpr bool kAlone = STAGES == 2, kWide = COLUMNS == 64;
  uint8_t kq[STAGES][kTermsX<DTYPE>][D / 64][kPlane], t[STAGES][kTermsT<DTYPE>][kPlane];
  uint8_t u[kWide ? 3 : kAlone ? 2 : 1][kChunk * 128], s[kWide ? 3 : 2][D * 128];     // R, and then U with its decays; the state
  alignas(16) uint8_t v[kAlone ? 1 : kChunk][COLUMNS * (DTYPE == CARRY_F32 ? 4 : 2)];
  alignas(16) float vec[2][kVec];
  // what has come, and what is free again: with one stage keys, queries, T and values are each asked for again as soon as they have been used
  uint64_t full[STAGES], free[STAGES], q_full, t_full, v_full, vec_full[2], q_free, t_free, v_free;
  uint64_t s_ready, r_ready, u_ready, scored, solved, added;
  // of a chunk: the first token whose value in a column is not finite, and whether there is one; for three chunks in turn, of which one is being
  // written, one read and one made ready
  int bad[3][COLUMNS], any_bad[3];
  uint32_t tmem;
  int poison, at_end;       // warps of rows that have met a chunk without its T
};

// this thread's columns of each term's product, summed, the smallest first
template <int W, int COLUMNS>
__device__ __forceinline__ void load_sums(uint32_t at, float2 (&x)[W / 2]) {
  uint32_t r[kTerms][W];
#pragma unroll
  for (int t = 0; t < kTerms; ++t) {
    if constexpr (W == 8) tmem_load8(at + t * COLUMNS, r[t]);
    else tmem_load16(at + t * COLUMNS, r[t]);
  }
  wait_loads();
  auto two = [&](int t, int j) { return make_float2(__uint_as_float(r[t][j]), __uint_as_float(r[t][j + 1])); };
#pragma unroll
  for (int j = 0; j < W; j += 2) x[j / 2] = add2(add2(two(2, j), two(1, j)), two(0, j));
}

// GROUPS of 128 threads share a row's columns.  With two stages of operands a CTA has a processor for itself, and what counts is the chain of a
// chunk's products; with one, two CTAs share a processor, and what one waits for the other uses.
template <int DTYPE, int D, int GROUPS, int STAGES, int COLUMNS>
__global__ void __launch_bounds__(GROUPS * 128 + 64, STAGES == 1 && DTYPE == CARRY_BF16 ? 2 : 1) sequence_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kX = kTermsX<DTYPE>, kT = kTermsT<DTYPE>, kPlanes = D / 64, W = COLUMNS / GROUPS;
  constexpr int kRowThreads = GROUPS * 128, kLoadWarp = kRowThreads / 32, kIssueWarp = kLoadWarp + 1, kValueBytes = DTYPE == CARRY_F32 ? 4 : 2;
  using Shared = SequenceShared<DTYPE, D, STAGES, COLUMNS>;
  constexpr bool kAlone = Shared::kAlone, kWide = Shared::kWide;
  extern __shared__ uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
  depend_release();
  depend_wait();
  const CarryGdnPrefillArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hv = blockIdx.y, h = hv / (a.HV / a.H), b = p.b0 + blockIdx.z;
  const Place place = place_of(p, blockIdx.z, nullptr);
  const int from = p.chunk0 * kChunk, left = place.count - from, chunks = min((left + kChunk - 1) / kChunk, p.chunks);
  if (chunks <= 0 && p.chunk0 > 0) return;                  // the launches before have done with the request
  auto lost = [&]() -> int& {                               // read anew where it is used: nothing of it takes a register in between
    uint32_t x, y, z;
    asm volatile("mov.u32 %0, %%ctaid.x;\nmov.u32 %1, %%ctaid.y;\nmov.u32 %2, %%ctaid.z;" : "=r"(x), "=r"(y), "=r"(z));
    return p.lost[((int64_t)z * a.HV + y) * (D / 32) + x];
  };
  if (p.lost && p.chunk0 > 0 && lost()) return;             // final_state is not where they left off
  if (tid == 0) {
    sh.poison = sh.at_end = 0;
    for (int i = 0; i < STAGES; ++i) {
      barrier_init(&sh.full[i], 1);
      barrier_init(&sh.free[i], 1);
    }
    for (uint64_t* bar : {&sh.q_full, &sh.t_full, &sh.q_free, &sh.t_free}) barrier_init(bar, 1);
    barrier_init(&sh.v_full, 32);
    barrier_init(&sh.v_free, kRowThreads / 2);
    barrier_init(&sh.vec_full[0], 1);
    barrier_init(&sh.vec_full[1], 1);
    barrier_init(&sh.s_ready, kRowThreads);
    barrier_init(&sh.r_ready, kRowThreads / 2);
    barrier_init(&sh.u_ready, kRowThreads);
    barrier_init(&sh.scored, 1);
    barrier_init(&sh.solved, 1);
    barrier_init(&sh.added, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < 3 * COLUMNS) {
    sh.bad[tid / COLUMNS][tid % COLUMNS] = kChunk;
    sh.any_bad[tid / COLUMNS] = 0;
  }
  // columns 0 and on: [K; Q] S, and, when that is read, K^T U; behind them [T; P T] R
  constexpr uint32_t kSolvedAt = kTerms * COLUMNS, kTmem = kWide ? 512 : 256;
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "n"(kTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* poison = &sh.poison;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, barrier_wait(bar, parity, poison, a.status)) != 0; };

  if (tid < kRowThreads) {
    // ---- a row to a thread, some of its columns: of the products' rows (keys, queries), and of the state's (K) ----
    const int row = warp % 4 * 32 + lane, first = warp / 4 * W, column0 = blockIdx.x * COLUMNS + first, token = row % kChunk;
    const uint32_t at = tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + first;
    const bool key = row < kChunk, has_state = row < D;
    uint8_t* const third = kAlone ? sh.u[kAlone] : sh.s[1];   // where R's and U's third term lies, and its first column there
    constexpr int kThirdColumn = kAlone ? 0 : COLUMNS;
    // this thread's numbers into an operand's terms; `last`: of the third one
    auto put = [&](uint8_t* tile, int plane, uint8_t* last, int last_column, float2 (&x)[W / 2]) {
#pragma unroll
      for (int j = 0; j < W; j += 8)
#pragma unroll
        for (int t = 0; t < kTerms; ++t) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = take_term(x[j / 2 + e]);
          uint8_t* to = kWide ? tile + t * plane + plane_at(row, (first + j) / 8)
                        : t < 2 ? tile + plane_at(row, (t * COLUMNS + first + j) / 8) : last + plane_at(row, (last_column + first + j) / 8);
          *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
    float2 S[W / 2];
    {
      const float* state = p.chunk0 > 0 ? a.final_state + b * a.stride_final_req : a.initial_state ? a.initial_state + b * a.stride_initial_req : nullptr;
      auto number = [&](int j) { return state && has_state ? state[((long long)hv * D + column0 + j) * D + row] : 0.0f; };
#pragma unroll
      for (int j = 0; j < W; j += 2) S[j / 2] = make_float2(number(j), number(j + 1));
    }
    auto put_state = [&]() {
      if (has_state) {
        float2 x[W / 2];
#pragma unroll
        for (int j = 0; j < W / 2; ++j) x[j] = S[j];
        put(sh.s[0], D * 128, sh.s[1], 0, x);
        fence_proxy();
      }
      fence_before();
      barrier_arrive(&sh.s_ready);
    };
    // A chunk's factors, and a key's beta v.  Values come from memory into registers a chunk ahead, or, where that would be in the other
    // CTA's way, into shared memory.
    float of_state = 0.0f, of_added = 0.0f, next_decay = 0.0f;
    float2 o[W / 2];                              // a key's beta v; a query's part of the output that comes from the state
    Raw<DTYPE> v[W / 8];
    auto fetch = [&](int c) {
      const int i = c * kChunk + token;
#pragma unroll
      for (int j = 0; j < W / 8; ++j)
        if (key && i < left) v[j] = load_row<DTYPE>(a.mixed_qkv, (long long)(place.first + from + i) * a.stride_mixed_tok + (2 * a.H + hv) * D + column0 + j * 8, p.aligned);
    };
    auto begin = [&](int c) {
      if (!wait(kAlone ? &sh.full[c % STAGES] : &sh.vec_full[c & 1], c / 2 & 1)) return false;
      const float* vec = sh.vec[c & 1];
      of_state = key ? -vec[token] : vec[3 * kChunk + token];
      of_added = vec[2 * kChunk + token];
      const float2 end = *reinterpret_cast<const float2*>(&vec[kDecayAt]);
      next_decay = end.x;
      if (end.y != 0.0f) {                        // the chunk's T is not there.  All rows' warps get here, with all done that the chunks ahead give; then the others stop
        __syncwarp();
        if (lane == 0 && atomicAdd(&sh.at_end, 1) == kRowThreads / 32 - 1) *poison = 1;
        return false;
      }
      if (!key) return true;                      // only keys' threads hold the values back
      const float beta = vec[kChunk + token];
      if (!kAlone && !wait(&sh.v_full, c & 1)) return false;
      const bool there = c * kChunk + token < left;         // behind the last token lies what an earlier chunk had
#pragma unroll
      for (int j = 0; j < W; j += 8) {
        if (!kAlone) v[j / 8] = load_raw<DTYPE>(sh.v[kAlone ? 0 : token], first + j);
        const Eight e = unpack<DTYPE>(v[j / 8]);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[j / 2 + k] = there ? mul2(e.x[k], make_float2(beta, beta)) : make_float2(0.0f, 0.0f);
      }
      // What is not finite would reach the rows ahead of it, as zero times that; its column becomes NaN from its token on instead.
      float2 none = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < W / 2; ++j) none = fma2(o[j], make_float2(0.0f, 0.0f), none);
      if (!(none.x + none.y == 0.0f)) {
#pragma unroll
        for (int j = 0; j < W; ++j) {
          float& y = j % 2 ? o[j / 2].y : o[j / 2].x;
          if (isfinite(y)) continue;
          atomicMin(&sh.bad[c % 3][first + j], token);
          sh.any_bad[c % 3] = 1;
          y = 0.0f;
        }
      }
      return true;
    };
    bool healthy = true;
    if (chunks > 0) {
      if (kAlone) fetch(0);
      else healthy = begin(0);
      put_state();
    }
    for (int c = 0; c < chunks && healthy; ++c) {
      const int parity = c & 1;
      float2 x[W / 2];
      test_come_late(warp, c);
      if (kAlone) healthy = begin(c);
      healthy = healthy && wait(&sh.scored, parity);
      if (!healthy) break;
      fence_after();
      load_sums<W, COLUMNS>(at, x);
      if (key) {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) x[j] = fma2(make_float2(of_state, of_state), x[j], o[j]);
        put(sh.u[0], kChunk * 128, third, kThirdColumn, x);
        fence_proxy();
        fence_before();
        barrier_arrive(&sh.r_ready);
        if (kAlone && c + 1 < chunks) fetch(c + 1);
        if (!kAlone) barrier_arrive(&sh.v_free);  // not before the values have been used: a load that is merely under way may be overtaken by the next copy
      } else {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) o[j] = mul2(make_float2(of_state, of_state), x[j]);
        fence_before();
        barrier_arrive(&sh.u_ready);
      }
      test_come_late(warp, c + 1);
      test_hold_up(a.HV, warp);
      if (tid < COLUMNS) sh.bad[(c + 2) % 3][tid] = kChunk;
      if (tid == 0) sh.any_bad[(c + 2) % 3] = 0;
      healthy = wait(&sh.solved, parity);
      if (!healthy) break;
      const int* bad = sh.bad[c % 3] + first;
      const bool spoilt = sh.any_bad[c % 3];
      fence_after();
      load_sums<W, COLUMNS>(at + kSolvedAt, x);
      if (key) {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) x[j] = mul2(make_float2(of_added, of_added), x[j]);
        put(sh.u[0], kChunk * 128, third, kThirdColumn, x);
        fence_proxy();
        fence_before();
        barrier_arrive(&sh.u_ready);
      } else {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) x[j] = add2(x[j], o[j]);
        if (spoilt) {
#pragma unroll
          for (int j = 0; j < W; ++j)
            if (bad[j] <= token) (j % 2 ? x[j / 2].y : x[j / 2].x) = kNotANumber;
        }
        if (!kAlone) healthy = wait(&sh.u_ready, parity);   // stores that are under way hold up the fences of the keys' threads, all the more of two CTAs'
        if (!healthy) break;
        if (c * kChunk + token < left) {
          const long long to = (long long)(place.first + from + c * kChunk + token) * a.stride_out_tok + hv * D + column0;
          if (p.out_aligned) {
#pragma unroll
            for (int j = 0; j < W / 2; j += 4) {
              if (a.out_dtype == CARRY_F32) {
                float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + to + 2 * j);
                q[0] = make_float4(x[j].x, x[j].y, x[j + 1].x, x[j + 1].y);
                q[1] = make_float4(x[j + 2].x, x[j + 2].y, x[j + 3].x, x[j + 3].y);
              } else {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const __half2 y = __float22half2_rn(x[j + e]);
                  w[e] = a.out_dtype == CARRY_BF16 ? pack_bf16(x[j + e].x, x[j + e].y) : *reinterpret_cast<const uint32_t*>(&y);
                }
                *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + to + 2 * j) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < W; ++j) store_from_float(a.out, to + j, a.out_dtype, j % 2 ? x[j / 2].y : x[j / 2].x);
          }
        }
      }
      test_come_late(warp, c + 2);
      const float decay = next_decay;
      if (!kAlone && c + 1 < chunks) healthy = begin(c + 1);
      healthy = healthy && wait(&sh.added, parity);
      if (!healthy) break;
      fence_after();
      load_sums<W, COLUMNS>(at, x);
#pragma unroll
      for (int j = 0; j < W / 2; ++j) S[j] = fma2(make_float2(decay, decay), S[j], x[j]);
      if (spoilt) {
#pragma unroll
        for (int j = 0; j < W; ++j)
          if (bad[j] < kChunk) (j % 2 ? S[j / 2].y : S[j / 2].x) = kNotANumber;
      }
      if (c + 1 < chunks) put_state();
    }
    if (healthy && has_state) {
      float* state = a.final_state + b * a.stride_final_req;
#pragma unroll
      for (int j = 0; j < W; ++j) state[((long long)hv * D + column0 + j) * D + row] = j % 2 ? S[j / 2].y : S[j / 2].x;
    }
  } else if (warp == kLoadWarp) {
    // ---- tiles and factors out of the workspace, values out of the rows ----
    constexpr uint32_t kBytesKq = kX * kPlanes * kPlane, kBytesT = kT * kPlane, kSide = kPlane / 2, kBytesV = COLUMNS * kValueBytes;
    for (int c = 0; c < chunks; ++c) {
      const int stage = c % STAGES;
      const bool reused = c >= STAGES;
      test_come_late(warp, c);
      const uint32_t turn = (c / STAGES - 1) & 1;           // of the use before
      const uint8_t* tile = p.kq + ((place.slot0 + c) * a.H + h) * kBytesKq;
      const long long place_hv = (place.slot0 + c) * a.HV + hv;
      if constexpr (kAlone) {
        if (reused && !wait(&sh.free[stage], turn)) break;
        if (lane == 0) {
          barrier_expect(&sh.full[stage], kBytesKq + kBytesT + kVec * 4 + test_extra_bytes(a.HV, hv, c));
          bulk_copy(sh.vec[stage], p.vec + place_hv * kVec, kVec * 4, &sh.full[stage]);
          bulk_copy(sh.kq[stage], tile, kBytesKq, &sh.full[stage]);
          bulk_copy(sh.t[stage], p.t + place_hv * kBytesT, kBytesT, &sh.full[stage]);
        }
        __syncwarp();
        continue;
      }
      auto side = [&](int which, uint64_t* bar) {           // keys or queries: a half of every plane
        barrier_expect(bar, kBytesKq / 2);
        for (int i = which * kSide; i < (int)kBytesKq; i += kPlane) bulk_copy(sh.kq[0][0][0] + i, tile + i, kSide, bar);
      };
      // in the order in which what was there is done with
      if (reused && !wait(&sh.v_free, turn)) break;
      const int tokens = min(left - c * kChunk, kChunk);
      const long long at = (long long)(place.first + from + c * kChunk) * a.stride_mixed_tok + (2 * a.H + hv) * D + blockIdx.x * COLUMNS;
      if (p.aligned) {                            // sixteen bytes at a time: bulk copies of such short rows would hold up the tiles'
        for (int i = lane; i < tokens * (int)(kBytesV / 16); i += 32) {
          const int token = i / (kBytesV / 16), part = i % (kBytesV / 16) * 16;
          __pipeline_memcpy_async(sh.v[token] + part, reinterpret_cast<const uint8_t*>(a.mixed_qkv) + (at + token * a.stride_mixed_tok) * kValueBytes + part, 16);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&sh.v_full)) : "memory");
      } else {
        for (int i = 0; i < tokens * (COLUMNS / 32); ++i) {
          const int token = i / (COLUMNS / 32), column = i % (COLUMNS / 32) * 32 + lane;
          if constexpr (kValueBytes == 4)
            reinterpret_cast<float*>(sh.v[token])[column] = reinterpret_cast<const float*>(a.mixed_qkv)[at + token * a.stride_mixed_tok + column];
          else
            reinterpret_cast<uint16_t*>(sh.v[token])[column] = reinterpret_cast<const uint16_t*>(a.mixed_qkv)[at + token * a.stride_mixed_tok + column];
        }
        barrier_arrive(&sh.v_full);
      }
      if (reused && !wait(&sh.q_free, turn)) break;
      if (lane == 0) {
        // [K; Q] S of the chunk before is done: the state that it took was ready, and the factors of the chunk before that had been read by then
        barrier_expect(&sh.vec_full[c & 1], kVec * 4);
        bulk_copy(sh.vec[c & 1], p.vec + place_hv * kVec, kVec * 4, &sh.vec_full[c & 1]);
        side(1, &sh.q_full);
      }
      __syncwarp();
      if (reused && !wait(&sh.t_free, turn)) break;
      if (lane == 0) {
        barrier_expect(&sh.t_full, kBytesT + test_extra_bytes(a.HV, hv, c));
        bulk_copy(sh.t[0], p.t + place_hv * kBytesT, kBytesT, &sh.t_full);
      }
      __syncwarp();
      if (reused && !wait(&sh.free[0], turn)) break;
      if (lane == 0) side(0, &sh.full[0]);
      __syncwarp();
    }
  } else {
    // ---- products: a left side's term x with the right side's terms 0 .. kTerms - 1 - x, which are its next columns ----
    const uint32_t elected = elect(), base = __shfl_sync(~0u, tmem, 0);
    // the third term lies that far behind the first two
    const uint32_t state = operand(sh.s[0], D * 128), rows = operand(sh.u[0], kAlone || kWide ? kChunk * 128 : smem_addr(sh.s[1]) + COLUMNS * 2 - smem_addr(sh.u[0]));
    for (int c = 0; c < chunks; ++c) {
      const int parity = c & 1, stage = c % STAGES;
      const uint32_t turn = c / STAGES & 1;
      test_come_late(warp, c);
      const uint32_t kq = operand(sh.kq[stage], 16), t = operand(sh.t[stage], 16), keys = operand(sh.kq[stage], D == 128 ? kPlane : 0);
      if (!wait(&sh.full[stage], turn) || (!kAlone && !wait(&sh.q_full, turn)) || !wait(&sh.s_ready, parity)) break;
      fence_after();
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_shared(elected, base, kq + x * (kPlanes * kPlane / 16) + k / 4 * (kPlane / 16) + k % 4 * 2, state + k * 128,
                     instruction_bf16((kTerms - x) * COLUMNS, false, true), x + k > 0);
      mma_commit(elected, &sh.scored);
      if (!kAlone) mma_commit(elected, &sh.q_free);
      if ((!kAlone && !wait(&sh.t_full, turn)) || !wait(&sh.r_ready, parity)) break;
      fence_after();
#pragma unroll
      for (int x = 0; x < kT; ++x)
#pragma unroll
        for (int k = 0; k < kChunk / 16; ++k)
          mma_shared(elected, base + kSolvedAt, t + x * (kPlane / 16) + k * 2, rows + k * 128, instruction_bf16((kTerms - x) * COLUMNS, false, true), x + k > 0);
      mma_commit(elected, &sh.solved);
      if (!kAlone) mma_commit(elected, &sh.t_free);
      if (!wait(&sh.u_ready, parity)) break;
      fence_after();
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int k = 0; k < kChunk / 16; ++k)
          mma_shared(elected, base, keys + x * (kPlanes * kPlane / 16) + k * 128, rows + k * 128, instruction_bf16((kTerms - x) * COLUMNS, true, true), x + k > 0);
      mma_commit(elected, &sh.added);
      mma_commit(elected, &sh.free[stage]);
    }
  }
  if (*poison) {
    for (int k = 0; k < 1 << 12; ++k) __nanosleep(64);      // products and copies in flight still use shared and tensor memory
  }
  fence_before();
  __syncthreads();
  if (p.lost && threadIdx.x == 0) lost() = *poison;
  if (warp == kIssueWarp) {
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem) : "memory");
  }
}

// ---- the launches ----------------------------------------------------------------------------------------------------

// How a call is cut: so many requests, and so many chunks of each, to a launch, that the workspace stays within a bound.
struct Layout {
  int requests, chunks, total;  // total: chunks of the longest request
  bool packed;
  int64_t places, kq, t, vec, lost;   // bytes
};
#ifdef CARRY_TEST_WAIT_EXPIRY
constexpr int64_t kWorkspaceBound = 1LL << 26;
#else
constexpr int64_t kWorkspaceBound = 1LL << 30;
#endif

Layout lay_out(const CarryGdnPrefillArgs& a) {
  const int64_t terms = a.qkv_dtype == CARRY_BF16 ? 1 : a.qkv_dtype == CARRY_F16 ? 2 : 3, terms_t = a.qkv_dtype == CARRY_F32 ? 3 : 2;
  const int64_t per_kq = a.H * terms * (a.K / 64) * kPlane, per_t = a.HV * terms_t * kPlane, per_vec = (int64_t)a.HV * kVec * 4;
  const int64_t per_lost = (int64_t)a.HV * (a.K / 32) * 4, per = per_kq + per_t + per_vec + per_lost;
  Layout l;
  l.total = (a.max_query + kChunk - 1) / kChunk;
  const int64_t most = kWorkspaceBound / per > 1 ? kWorkspaceBound / per : 1, follows = a.N / kChunk + a.B, grid = (int64_t)a.B * l.total;
  l.packed = follows <= most && follows < grid;
  if (l.packed || grid <= most) {
    l.requests = a.B;
    l.chunks = l.total;
    l.places = l.packed ? follows : grid;
  } else {
    // Turns are deep, of no more requests than are eight rounds of CTAs, two to a processor: those without rows left cost their empty CTAs in every turn.
    // 16384 tokens among 256 requests of one token, 64 heads of 128: 8.5 ms, and 99 with all requests in turns of one chunk; 16 requests of 8192: 9.4 and 9.2.
    // With four rounds 7.7 and 10.0, with sixteen 10.5 and 9.4.
    const int64_t fill = 16LL * sm_count() / ((int64_t)a.HV * (a.K / 32)) + 1, deep = most / l.total;
    const int64_t wanted = deep > fill ? deep : fill, bound = wanted < most ? wanted : most;
    const int64_t groups = (a.B + bound - 1) / bound;
    l.requests = (int)((a.B + groups - 1) / groups);
    l.chunks = (int)(most / l.requests < l.total ? most / l.requests : l.total);
    l.places = (int64_t)l.requests * l.chunks;
  }
  l.kq = l.places * per_kq;
  l.t = l.places * per_t;
  l.vec = l.places * per_vec;
  l.lost = l.chunks < l.total ? l.requests * per_lost : 0;     // a launch has no more requests than places
  return l;
}

template <class K>
int allow_shared(K kernel, size_t smem, bool (&ready)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev < 64 && ready[dev]) return CARRY_GDN_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    cudaGetLastError();
    return CARRY_GDN_ERR_LAUNCH;
  }
  if (dev < 64) ready[dev] = true;
  return CARRY_GDN_OK;
}

template <int DTYPE, int D, int GROUPS, int STAGES, int COLUMNS>
int launch_sequence(const ChunkParams& p, int requests, cudaStream_t stream) {
  constexpr size_t smem = sizeof(SequenceShared<DTYPE, D, STAGES, COLUMNS>) + 1024;
  static_assert(smem <= 227 * 1024, "a CTA's shared memory");
  static_assert(STAGES == 2 || DTYPE != CARRY_BF16 || 2 * (smem + 1024) <= 228 * 1024, "two CTAs to a processor");
  static thread_local bool ready[64];
  const int rc = allow_shared(sequence_kernel<DTYPE, D, GROUPS, STAGES, COLUMNS>, smem, ready);
  if (rc != CARRY_GDN_OK) return rc;
  return launch_dependent(sequence_kernel<DTYPE, D, GROUPS, STAGES, COLUMNS>, dim3(D / COLUMNS, (unsigned)p.a.HV, (unsigned)requests), GROUPS * 128 + 64, smem, stream, p);
}

template <int DTYPE, int D>
int launch_chunks(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  constexpr int kSize = DTYPE == CARRY_F32 ? 4 : 2;
  constexpr size_t smem = DTYPE == CARRY_F32 ? sizeof(PrepareShared<D>) + 1024 : kUnitWarps * sizeof(Unit);
  static thread_local bool ready[64];
  int rc;
  if constexpr (DTYPE == CARRY_F32) rc = allow_shared(prepare_kernel<D>, smem, ready);
  else rc = allow_shared(unit_kernel<DTYPE, D>, smem, ready);
  if (rc != CARRY_GDN_OK) return rc;
  const Layout l = lay_out(a);
  ChunkParams p = {};
  p.a = a;
  p.packed = l.packed;
  p.aligned = reinterpret_cast<uintptr_t>(a.mixed_qkv) % 16 == 0 && a.stride_mixed_tok * kSize % 16 == 0;
  const int out_size = a.out_dtype == CARRY_F32 ? 4 : 2;
  p.out_aligned = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.stride_out_tok * out_size % 16 == 0;
  p.kq = static_cast<uint8_t*>(a.workspace);
  p.t = p.kq + l.kq;
  p.vec = reinterpret_cast<float*>(p.t + l.t);
  if (l.lost) p.lost = reinterpret_cast<int*>(p.t + l.t + l.vec);
  for (int b = 0; b < a.B; b += l.requests)
    for (int c = 0; c < l.total; c += l.chunks) {
      p.b0 = b;
      p.chunk0 = c;
      p.chunks = l.total - c < l.chunks ? l.total - c : l.chunks;
      const int requests = a.B - b < l.requests ? a.B - b : l.requests;
      if constexpr (DTYPE == CARRY_F32)
        rc = launch_dependent(prepare_kernel<D>, dim3((unsigned)p.chunks, (unsigned)a.HV, (unsigned)requests), kPrepareThreads, smem, stream, p);
      else
        rc = launch_dependent(unit_kernel<DTYPE, D>, dim3((unsigned)(p.chunks + kUnitWarps - 1) / kUnitWarps, (unsigned)a.HV, (unsigned)requests), kUnitWarps * 32, smem,
                              stream, p);
      if (rc != CARRY_GDN_OK) return rc;
      // one CTA to a processor while that is all there are (a prompt of 2048 tokens with 32 heads: 117 us, 146 in the other form; two of them 228 and 211)
      // More CTAs than that: in bf16 two to a processor (sixteen prompts of 4096 tokens, side by side, 2.40 ms, 2.59 with 64 columns to one CTA); in fp16, whose keys and
      // queries fill shared memory, 64 columns, for which the left sides are read once and not twice (two prompts of 3001: 323 us and not 410); in
      // fp32 as well where there is room, at 64 wide (eight of 1000: 384 us and not 441).
      const bool alone = (int64_t)requests * a.HV * (D / 32) <= sm_count();
      if constexpr (DTYPE == CARRY_BF16) rc = alone ? launch_sequence<DTYPE, D, 4, 2, 32>(p, requests, stream) : launch_sequence<DTYPE, D, 2, 1, 32>(p, requests, stream);
      else if constexpr (DTYPE == CARRY_F16 || D == 64) rc = alone ? launch_sequence<DTYPE, D, 4, 1, 32>(p, requests, stream) : launch_sequence<DTYPE, D, 4, 1, 64>(p, requests, stream);
      else rc = launch_sequence<DTYPE, D, 4, 1, 32>(p, requests, stream);
      if (rc != CARRY_GDN_OK) return rc;
    }
  return CARRY_GDN_OK;
}

template <int DTYPE>
int launch_width(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  return a.K == 64 ? launch_chunks<DTYPE, 64>(a, stream) : launch_chunks<DTYPE, 128>(a, stream);
}

// Up to so many tokens of a request go token by token.  A token costs 0.35 us where every row of the states has lanes of its own, a chunk 25 us
// and 2.5 to 4 for each further one; with 128 heads a token 0.85 us, a chunk 36; in fp32, whose products take four times as many, 0.3 to 1.1 and 25 to 90.
bool in_chunks(const CarryGdnPrefillArgs& a) { return a.max_query > (a.qkv_dtype == CARRY_F32 ? 96 : delta_rows_alone(a) ? 64 : 40); }

}  // namespace

int64_t delta_workspace(const CarryGdnPrefillArgs& a) {
  if (!in_chunks(a)) return 0;
  const Layout l = lay_out(a);
  return l.kq + l.t + l.vec + l.lost;
}

int launch_delta(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  if (!in_chunks(a)) return launch_delta_recurrent(a, stream);
  return a.qkv_dtype == CARRY_F32 ? launch_width<CARRY_F32>(a, stream)
         : a.qkv_dtype == CARRY_BF16 ? launch_width<CARRY_BF16>(a, stream) : launch_width<CARRY_F16>(a, stream);
}

}  // namespace carry
