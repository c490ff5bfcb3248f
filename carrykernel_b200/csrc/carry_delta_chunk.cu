// The gated delta rule in chunks of 64 tokens, on the fifth-generation tensor cores.
//
// With G_i the running sum of log alpha within a chunk and S the state at its start (as [K, V]), the rows u_i that a chunk adds
// are the solution of a triangular system,
//   (I + L) U = R,   R = diag(beta) (V - diag(exp G) K S),   L_ij = beta_i exp(G_i - G_j) k_i . k_j  for j < i,
// and with T = (I + L)^-1 and P_ij = exp(G_i - G_j) (scale q_i) . k_j for j <= i:
//   U = T R,   O = diag(exp G) (scale Q) S + (P T) R,   S' = exp(G_64) S + K^T diag(exp(G_64 - G)) U.
//
// T and P T do not depend on the state: prepare_kernel forms them for every chunk and head side by side.  sequence_kernel then walks a
// request's chunks, a CTA for some columns of a head's state, with three products to a chunk that wait for one another:
//   [K; Q] S  (128 x columns, over K),   [T; P T] R  (128 x columns, over 64 tokens),   K^T U  (K x columns, over 64 tokens).
// The state itself stays in registers, in fp32; its products take it as a sum of bf16 numbers.
//
// Precision.  Keys and queries in bf16 are operands as they are (norms and decays multiply rows of the products, in fp32); in fp16 they are
// the sum of two bf16 numbers, in fp32 of three.  What is computed is split too: S, R and U into three, T into two (three with fp32
// operands), and products of terms are formed down to 2^-18 of the largest.  The final state is then within 1e-6 of the
// recurrence in 64 bits; two terms throughout would leave it 3.5e-6 off, and one (plain bf16 products) 2.4e-3.
#include "carry_delta.cuh"
#include "carry_tensor.cuh"

namespace carry {
namespace {

constexpr int kChunk = 64, kPlane = 128 * 128, kVec = 4 * kChunk + 8, kTerms = 3;
constexpr float kLn2 = 0.69314718055994531f, kLeastLog = -200.0f;

struct ChunkParams {
  CarryGdnPrefillArgs a;
  int b0, chunk0, chunks;   // the launch's requests begin at b0; its chunks are chunk0 .. chunk0 + chunks - 1 of every request
  int packed;               // places in the workspace follow the rows (a launch that covers everything), or requests times chunks
  int aligned, out_aligned; // rows are on the grid of 16 bytes
  uint8_t *kq, *t;          // workspace: [place][H] tiles of keys and queries, [place][HV] tiles of T and P T,
  float* vec;               // [place][HV] factors of a chunk's rows
};

struct Place {
  int first, count;         // the request's rows
  long long slot0;          // of its chunk chunk0
};
__device__ __forceinline__ Place place_of(const ChunkParams& p, int z, int* status) {
  const int b = p.b0 + z;
  const PrefillRequest r = prefill_request(p.a, b, status);
  return {r.first, r.count, p.packed ? r.first / kChunk + b : (long long)z * p.chunks};
}

// bf16 numbers that a key's or query's numbers come as, and those of T
template <int DTYPE>
constexpr int kTermsX = DTYPE == CARRY_BF16 ? 1 : DTYPE == CARRY_F16 ? 2 : 3;
template <int DTYPE>
constexpr int kTermsT = DTYPE == CARRY_F32 ? 3 : 2;

// two numbers' next bf16 term, which is taken off them
__device__ __forceinline__ uint32_t take_term(float& x, float& y) {
  const uint32_t u = pack_bf16(x, y);
  x -= __uint_as_float(u << 16);
  y -= __uint_as_float(u & 0xffff0000u);
  return u;
}
// eight numbers as TERMS chunks of 16 bytes, `apart` bytes from one another
template <int TERMS>
__device__ __forceinline__ void store_terms(uint8_t* to, int apart, float (&x)[8]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = take_term(x[2 * e], x[2 * e + 1]);
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

constexpr int kPrepareThreads = 256, kPad = 68, kPadX = 36;

template <int TERMS, int TERMS_T, int D>
struct PrepareShared {
  uint8_t kq[TERMS][D / 64][kPlane];      // rows 0 .. 63 keys, 64 .. 127 queries
  uint8_t t[TERMS_T][kPlane];             // rows 0 .. 63 T, 64 .. 127 P and then P T
  alignas(16) float L[kChunk][kPad], T[kChunk][kPad], X[32][kPadX];
  float2 G[kChunk];                       // running sum of log2 alpha, and what its rounding left out
  float beta[kChunk], norm[2 * kChunk];   // norm: what makes a key a unit one, and a query one times `scale`
  uint64_t scored, multiplied;
  uint32_t tmem;
  int poison;
};

// A chunk's gates and the factors of its rows, by one warp; lane l has tokens 2 l and 2 l + 1.
template <class Shared>
__device__ __forceinline__ void chunk_gates(const ChunkParams& p, Shared& sh, long long row, int n, int hv, float* vec) {
  const int lane = threadIdx.x % 32;
  double g[2];
  float beta[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float log_alpha = 0.0f;
    beta[e] = 0.0f;
    if (2 * lane + e < n) prefill_gates(p.a, row + 2 * lane + e, hv, log_alpha, beta[e]);
    g[e] = (double)(log_alpha < kLeastLog ? kLeastLog : log_alpha) * 1.4426950408889634;     // exp(-200) is 0, and sums stay finite
  }
  double sum = g[0] + g[1];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const double below = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += below;
  }
  const double G[2] = {sum - g[1], sum}, last = __shfl_sync(~0u, sum, 31);
  auto power = [](double x) {
    const float hi = (float)x;
    return exp2f(hi) * fmaf((float)(x - hi), kLn2, 1.0f);
  };
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    const bool there = i < n;
    const float hi = (float)G[e], decay = power(G[e]);
    sh.G[i] = make_float2(hi, (float)(G[e] - hi));
    sh.beta[i] = beta[e];
    vec[i] = there ? beta[e] * decay * sh.norm[i] : 0.0f;
    vec[kChunk + i] = beta[e];
    vec[2 * kChunk + i] = there ? power(last - G[e]) * sh.norm[i] : 0.0f;
    vec[3 * kChunk + i] = there ? decay * sh.norm[kChunk + i] : 0.0f;
  }
  if (lane < 8) vec[4 * kChunk + lane] = power(last);
}

// T = (I + L)^-1 in fp32: the 16 x 16 blocks on the diagonal by substitution, a column to a thread, then twice
// T21 = -T22 L21 T11 for neighbouring blocks.  The entries of T are bounded as those of the recurrence are.
template <class Shared>
__device__ __forceinline__ void invert(Shared& sh) {
  const int tid = threadIdx.x;
  if (tid < kChunk) {
    const int b = tid / 16 * 16, j = tid % 16;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == j ? 1.0f : 0.0f;
#pragma unroll
      for (int k = 0; k < i; ++k) s = fmaf(-sh.L[b + i][b + k], x[k], s);
      x[i] = s;
      sh.T[b + i][b + j] = s;
    }
  } else {
    for (int e = tid - kChunk; e < kChunk * kChunk; e += kPrepareThreads - kChunk)
      if (e % kChunk / 16 > e / kChunk / 16) sh.T[e / kChunk][e % kChunk] = 0.0f;
  }
  __syncthreads();
  {
    const int b = tid / 128 * 32, r = tid % 128 / 8, c = tid % 8 * 2, x = tid / 128 * 16;
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float l = sh.L[b + 16 + r][b + k];
      s[0] = fmaf(l, sh.T[b + k][b + c], s[0]);
      s[1] = fmaf(l, sh.T[b + k][b + c + 1], s[1]);
    }
    sh.X[x + r][c] = s[0];
    sh.X[x + r][c + 1] = s[1];
    __syncthreads();
    s[0] = s[1] = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float l = sh.T[b + 16 + r][b + 16 + k];
      s[0] = fmaf(-l, sh.X[x + k][c], s[0]);
      s[1] = fmaf(-l, sh.X[x + k][c + 1], s[1]);
    }
    sh.T[b + 16 + r][b + c] = s[0];
    sh.T[b + 16 + r][b + c + 1] = s[1];
    __syncthreads();
  }
  const int r = tid / 8, c = tid % 8 * 4;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int k = 0; k < 32; ++k) {
    const float l = sh.L[32 + r][k];
    const float4 y = *reinterpret_cast<const float4*>(&sh.T[k][c]);
    s = make_float4(fmaf(l, y.x, s.x), fmaf(l, y.y, s.y), fmaf(l, y.z, s.z), fmaf(l, y.w, s.w));
  }
  *reinterpret_cast<float4*>(&sh.X[r][c]) = s;
  __syncthreads();
  s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int k = 0; k < 32; ++k) {
    const float l = -sh.T[32 + r][32 + k];
    const float4 y = *reinterpret_cast<const float4*>(&sh.X[k][c]);
    s = make_float4(fmaf(l, y.x, s.x), fmaf(l, y.y, s.y), fmaf(l, y.z, s.z), fmaf(l, y.w, s.w));
  }
  *reinterpret_cast<float4*>(&sh.T[32 + r][c]) = s;
  __syncthreads();
}

template <int DTYPE, int D>
__global__ void __launch_bounds__(kPrepareThreads, 2) prepare_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kX = kTermsX<DTYPE>, kT = kTermsT<DTYPE>, kPlanes = D / 64;
  using Shared = PrepareShared<kX, kT, D>;
  extern __shared__ uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
  depend_release();
  depend_wait();
  const CarryGdnPrefillArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, h = blockIdx.y, group = a.HV / a.H, c = blockIdx.x;
  const Place place = place_of(p, blockIdx.z, tid == 0 && h == 0 && c == 0 && p.chunk0 == 0 ? a.status : nullptr);
  const int from = (p.chunk0 + c) * kChunk, n = min(place.count - from, kChunk);
  if (n <= 0) return;
  const long long row0 = place.first + from, slot = place.slot0 + c;
  if (tid == 0) {
    sh.poison = 0;
    barrier_init(&sh.scored, 1);
    barrier_init(&sh.multiplied, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 128;" ::"r"(smem_addr(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // keys and queries as operands, and their norms; rows behind the last token are zeros, whatever memory holds there
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
#pragma unroll 4
  for (int row = warp * kRows + lane / kLanes; row < 2 * kChunk; row += kPrepareThreads / 32 * kRows) {
    const int token = row % kChunk, chunk = lane % kLanes;
    float x[8] = {};
    if (token < n) {
      const Eight e = unpack<DTYPE>(load_row<DTYPE>(a.mixed_qkv, (row0 + token) * a.stride_mixed_tok + (row < kChunk ? a.H + h : h) * D + chunk * 8, p.aligned));
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[2 * i] = e.x[i].x; x[2 * i + 1] = e.x[i].y; }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
    if (chunk == 0) sh.norm[row] = (a.use_qk_l2norm ? __fdiv_rn(1.0f, sqrtf(sum + kL2Eps)) : 1.0f) * (row < kChunk ? 1.0f : a.scale);
    store_terms<kX>(sh.kq[0][chunk / 8] + plane_at(row, chunk % 8), kPlanes * kPlane, x);
  }
  fence_proxy();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* poison = &sh.poison;
  // the whole CTA goes on, or none of it
  auto wait = [&](uint64_t* bar, uint32_t parity) { return !__syncthreads_or(!barrier_wait(bar, parity, poison, a.status)); };

  bool healthy = true;
  if (warp == 0) {
    const uint32_t elected = elect(), base = __shfl_sync(~0u, tmem, 0);
#pragma unroll
    for (int x = 0; x < kX; ++x)
#pragma unroll
      for (int y = 0; y < kX; ++y)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t step = k / 4 * (kPlane / 16) + k % 4 * 2;
          mma_shared(elected, base, operand(sh.kq[x], 16) + step, operand(sh.kq[y], 16) + step, instruction_bf16(kChunk, false, false), x + y + k > 0);
        }
    mma_commit(elected, &sh.scored);
  }
  if (tid == 0) {
    bulk_store(p.kq + (slot * a.H + h) * (kX * kPlanes * kPlane), sh.kq, kX * kPlanes * kPlane);
    bulk_commit();
  }
  // products of keys and queries with keys: a row to a thread, half of its columns
  const int row = warp % 4 * 32 + lane, i = row % kChunk, first = warp / 4 * 32;
  const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
  float dots[32];
  healthy = wait(&sh.scored, 0);
  if (healthy) {
    fence_after();
    tmem_load(tmem + lanes + first, dots);
    wait_loads();
  }
  for (int g = 0; g < group && healthy; ++g) {
    const int hv = h * group + g;
    if (tid == 0 && g > 0) bulk_wait_read();
    if (warp == 0) chunk_gates(p, sh, row0, n, hv, p.vec + (slot * a.HV + hv) * kVec);
    __syncthreads();
    const float2 G = sh.G[i];
    const float by = row < kChunk ? sh.beta[i] * sh.norm[i] : sh.norm[row];
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = first + j + e;
        const float2 to = sh.G[col];
        const float decay = exp2f((G.x - to.x) + (G.y - to.y));
        const bool counts = row < kChunk ? col < i : col <= i;
        x[e] = counts ? dots[j + e] * by * sh.norm[col] * decay : 0.0f;
      }
      if (row < kChunk) {
        *reinterpret_cast<float4*>(&sh.L[i][first + j]) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(&sh.L[i][first + j + 4]) = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        store_terms<kT>(sh.t[0] + plane_at(row, (first + j) / 8), kPlane, x);
      }
    }
    __syncthreads();
    invert(sh);
    {
      const int r = tid / 4, q = tid % 4 * 16;
#pragma unroll
      for (int j = 0; j < 16; j += 8) {
        const float4 u = *reinterpret_cast<const float4*>(&sh.T[r][q + j]), v = *reinterpret_cast<const float4*>(&sh.T[r][q + j + 4]);
        float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        store_terms<kT>(sh.t[0] + plane_at(r, (q + j) / 8), kPlane, x);
      }
    }
    fence_proxy();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) {                              // [T; P] T: of it, P T
      const uint32_t elected = elect(), base = __shfl_sync(~0u, tmem, 0) + kChunk;
#pragma unroll
      for (int x = 0; x < kT; ++x)
#pragma unroll
        for (int y = 0; x + y < kT; ++y)
#pragma unroll
          for (int k = 0; k < kChunk / 16; ++k)
            mma_shared(elected, base, operand(sh.t[x], 16) + k * 2, operand(sh.t[y], 16) + k * 128, instruction_bf16(kChunk, false, true), x + y + k > 0);
      mma_commit(elected, &sh.multiplied);
    }
    healthy = wait(&sh.multiplied, g & 1);
    if (!healthy) break;
    fence_after();
    if (row >= kChunk) {
      float y[32];
      tmem_load(tmem + lanes + kChunk + first, y);
      wait_loads();
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[j + e];
        store_terms<kT>(sh.t[0] + plane_at(row, (first + j) / 8), kPlane, x);
      }
    }
    fence_proxy();
    fence_before();
    __syncthreads();
    fence_after();
    if (tid == 0) {
      bulk_store(p.t + (slot * a.HV + hv) * (kT * kPlane), sh.t, kT * kPlane);
      bulk_commit();
    }
  }
  if (tid == 0) bulk_wait();
  if (*poison) {
    for (int k = 0; k < 1 << 12; ++k) __nanosleep(64);      // products in flight still use shared and tensor memory
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 128;" ::"r"(tmem) : "memory");
  }
}

// ---- along a sequence ------------------------------------------------------------------------------------------------

constexpr int kRowThreads = 256, kLoadWarp = kRowThreads / 32, kIssueWarp = kLoadWarp + 1, kSequenceThreads = (kIssueWarp + 1) * 32;

template <int TERMS, int TERMS_T, int D, int STAGES>
struct SequenceShared {
  uint8_t kq[STAGES][TERMS][D / 64][kPlane], t[STAGES][TERMS_T][kPlane];
  uint8_t s[kTerms][D * 128], u[kTerms][kChunk * 128];    // the state; R, and then U with its decays
  alignas(16) float vec[STAGES][kVec];
  uint64_t full[STAGES], free[STAGES], s_ready, r_ready, u_ready, scored, solved, added;
  uint32_t tmem;
  int poison;
};

template <int W>
__device__ __forceinline__ void load_columns(uint32_t at, float (&x)[W]) {
  if constexpr (W == 32) tmem_load(at, x);
  else tmem_load16(at, reinterpret_cast<uint32_t(&)[16]>(x));
  wait_loads();
}

// COLUMNS of a head's state to a CTA
template <int DTYPE, int D, int COLUMNS, int STAGES>
__global__ void __launch_bounds__(kSequenceThreads, 1) sequence_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kX = kTermsX<DTYPE>, kT = kTermsT<DTYPE>, kPlanes = D / 64, W = COLUMNS / 2;
  using Shared = SequenceShared<kX, kT, D, STAGES>;
  extern __shared__ uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
  depend_release();
  depend_wait();
  const CarryGdnPrefillArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hv = blockIdx.y, h = hv / (a.HV / a.H), b = p.b0 + blockIdx.z;
  const Place place = place_of(p, blockIdx.z, nullptr);
  const int from = p.chunk0 * kChunk, left = place.count - from, chunks = min((left + kChunk - 1) / kChunk, p.chunks);
  if (chunks <= 0 && p.chunk0 > 0) return;                  // the launches before have done with the request
  if (tid == 0) {
    sh.poison = 0;
    for (int i = 0; i < STAGES; ++i) {
      barrier_init(&sh.full[i], 1);
      barrier_init(&sh.free[i], 1);
    }
    barrier_init(&sh.s_ready, kRowThreads);
    barrier_init(&sh.r_ready, kRowThreads / 2);
    barrier_init(&sh.u_ready, kRowThreads);
    barrier_init(&sh.scored, 1);
    barrier_init(&sh.solved, 1);
    barrier_init(&sh.added, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  constexpr uint32_t kTmem = COLUMNS == 64 ? 256 : 128;
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "n"(kTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* poison = &sh.poison;

  if (tid < kRowThreads) {
    // ---- a row to a thread, half of its columns: of the products' rows (keys, queries), and of the state's (K) ----
    const int row = warp % 4 * 32 + lane, first = warp / 4 * W, column0 = blockIdx.x * COLUMNS + first, token = row % kChunk;
    const uint32_t at = tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + first;
    const bool key = row < kChunk, has_state = row < D;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, barrier_wait(bar, parity, poison, a.status)) != 0; };
    // numbers of a row in an operand: TERMS of them, columns first .. first + W - 1
    auto put = [&](uint8_t* tile, int apart, float (&x)[W]) {
#pragma unroll
      for (int j = 0; j < W; j += 8) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[j + e];
        store_terms<kTerms>(tile + plane_at(row, (first + j) / 8), apart, y);
      }
    };
    float S[W];
    {
      const float* state = p.chunk0 > 0 ? a.final_state + b * a.stride_final_req : a.initial_state ? a.initial_state + b * a.stride_initial_req : nullptr;
#pragma unroll
      for (int j = 0; j < W; ++j) S[j] = state && has_state ? state[((long long)hv * D + column0 + j) * D + row] : 0.0f;
    }
    auto put_state = [&]() {
      if (has_state) {
        float x[W];
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = S[j];
        put(sh.s[0], D * 128, x);
        fence_proxy();
      }
      fence_before();
      barrier_arrive(&sh.s_ready);
    };
    Raw<DTYPE> v[W / 8];
    auto fetch = [&](int c) {
      const int i = c * kChunk + token;
#pragma unroll
      for (int j = 0; j < W / 8; ++j) {
        if (key && i < left) v[j] = load_row<DTYPE>(a.mixed_qkv, (long long)(place.first + from + i) * a.stride_mixed_tok + (2 * a.H + hv) * D + column0 + j * 8, p.aligned);
      }
    };
    bool healthy = true;
    if (chunks > 0) {
      fetch(0);
      put_state();
    }
    for (int c = 0; c < chunks; ++c) {
      const int stage = c % STAGES, parity = c & 1;
      const bool there = c * kChunk + token < left;
      healthy = wait(&sh.full[stage], c / STAGES & 1);
      if (!healthy) break;
      const float* vec = sh.vec[stage];
      const float of_state = key ? vec[token] : vec[3 * kChunk + token], beta = vec[kChunk + token], of_added = vec[2 * kChunk + token], decay = vec[4 * kChunk];
      float x[W], o[W];
      healthy = wait(&sh.scored, parity);
      if (!healthy) break;
      fence_after();
      load_columns<W>(at, x);
      if (key) {
#pragma unroll
        for (int j = 0; j < W; j += 8) {
          const Eight e = unpack<DTYPE>(v[j / 8]);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[j + k] = there ? fmaf(-of_state, x[j + k], beta * (k % 2 ? e.x[k / 2].y : e.x[k / 2].x)) : 0.0f;
        }
        put(sh.u[0], kChunk * 128, x);
        fence_proxy();
        fence_before();
        barrier_arrive(&sh.r_ready);
        if (c + 1 < chunks) fetch(c + 1);
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = of_state * x[j];
        fence_before();
        barrier_arrive(&sh.u_ready);
      }
      healthy = wait(&sh.solved, parity);
      if (!healthy) break;
      fence_after();
      load_columns<W>(at + COLUMNS, x);
      if (key) {
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] *= of_added;
        put(sh.u[0], kChunk * 128, x);
        fence_proxy();
        fence_before();
        barrier_arrive(&sh.u_ready);
      } else if (there) {
        const long long to = (long long)(place.first + from + c * kChunk + token) * a.stride_out_tok + hv * D + column0;
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] += o[j];
        if (p.out_aligned) {
#pragma unroll
          for (int j = 0; j < W; j += 8) {
            if (a.out_dtype == CARRY_F32) {
              float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + to + j);
              q[0] = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
              q[1] = make_float4(x[j + 4], x[j + 5], x[j + 6], x[j + 7]);
            } else {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __half2 y = __floats2half2_rn(x[j + 2 * e], x[j + 2 * e + 1]);
                w[e] = a.out_dtype == CARRY_BF16 ? pack_bf16(x[j + 2 * e], x[j + 2 * e + 1]) : *reinterpret_cast<const uint32_t*>(&y);
              }
              *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + to + j) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) store_from_float(a.out, to + j, a.out_dtype, x[j]);
        }
      }
      healthy = wait(&sh.added, parity);
      if (!healthy) break;
      fence_after();
      load_columns<W>(at + 2 * COLUMNS, x);
#pragma unroll
      for (int j = 0; j < W; ++j) S[j] = fmaf(decay, S[j], x[j]);
      if (c + 1 < chunks) put_state();
    }
    if (healthy && has_state) {
      float* state = a.final_state + b * a.stride_final_req;
#pragma unroll
      for (int j = 0; j < W; ++j) state[((long long)hv * D + column0 + j) * D + row] = S[j];
    }
  } else if (warp == kLoadWarp) {
    // ---- tiles and factors out of the workspace ----
    if (lane == 0) {
      constexpr uint32_t kBytesKq = kX * kPlanes * kPlane, kBytesT = kT * kPlane;
      for (int c = 0; c < chunks; ++c) {
        const int stage = c % STAGES;
        if (c >= STAGES && !barrier_wait(&sh.free[stage], c / STAGES - 1 & 1, poison, a.status)) break;
        barrier_expect(&sh.full[stage], kBytesKq + kBytesT + kVec * 4);
        const long long slot = place.slot0 + c;
        bulk_copy(sh.vec[stage], p.vec + (slot * a.HV + hv) * kVec, kVec * 4, &sh.full[stage]);
        bulk_copy(sh.kq[stage], p.kq + (slot * a.H + h) * kBytesKq, kBytesKq, &sh.full[stage]);
        bulk_copy(sh.t[stage], p.t + (slot * a.HV + hv) * kBytesT, kBytesT, &sh.full[stage]);
      }
    }
    __syncwarp();
  } else {
    // ---- products ----
    const uint32_t elected = elect(), base = __shfl_sync(~0u, tmem, 0);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, barrier_wait(bar, parity, poison, a.status)) != 0; };
    const uint32_t state = operand(sh.s, 16), rows = operand(sh.u, 16);
    constexpr uint32_t kStateTerm = D * 128 / 16, kRowsTerm = kChunk * 128 / 16;
    for (int c = 0; c < chunks; ++c) {
      const int stage = c % STAGES, parity = c & 1;
      const uint32_t kq = operand(sh.kq[stage], 16), t = operand(sh.t[stage], 16), keys = operand(sh.kq[stage], D == 128 ? kPlane : 0);
      if (!wait(&sh.full[stage], c / STAGES & 1) || !wait(&sh.s_ready, parity)) break;
      fence_after();
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int y = 0; x + y < kTerms; ++y)
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_shared(elected, base, kq + x * (kPlanes * kPlane / 16) + k / 4 * (kPlane / 16) + k % 4 * 2, state + y * kStateTerm + k * 128,
                       instruction_bf16(COLUMNS, false, true), x + y + k > 0);
      mma_commit(elected, &sh.scored);
      if (!wait(&sh.r_ready, parity)) break;
      fence_after();
#pragma unroll
      for (int x = 0; x < kT; ++x)
#pragma unroll
        for (int y = 0; x + y < kTerms; ++y)
#pragma unroll
          for (int k = 0; k < kChunk / 16; ++k)
            mma_shared(elected, base + COLUMNS, t + x * (kPlane / 16) + k * 2, rows + y * kRowsTerm + k * 128, instruction_bf16(COLUMNS, false, true), x + y + k > 0);
      mma_commit(elected, &sh.solved);
      if (!wait(&sh.u_ready, parity)) break;
      fence_after();
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int y = 0; x + y < kTerms; ++y)
#pragma unroll
          for (int k = 0; k < kChunk / 16; ++k)
            mma_shared(elected, base + 2 * COLUMNS, keys + x * (kPlanes * kPlane / 16) + k * 128, rows + y * kRowsTerm + k * 128,
                       instruction_bf16(COLUMNS, true, true), x + y + k > 0);
      mma_commit(elected, &sh.added);
      mma_commit(elected, &sh.free[stage]);
    }
  }
  if (*poison) {
    for (int k = 0; k < 1 << 12; ++k) __nanosleep(64);      // products and copies in flight still use shared and tensor memory
  }
  fence_before();
  __syncthreads();
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
  int64_t places, kq, t, vec;   // bytes
};
constexpr int64_t kWorkspaceBound = 256LL << 20;

Layout lay_out(const CarryGdnPrefillArgs& a) {
  const int64_t terms = a.qkv_dtype == CARRY_BF16 ? 1 : a.qkv_dtype == CARRY_F16 ? 2 : 3, terms_t = a.qkv_dtype == CARRY_F32 ? 3 : 2;
  const int64_t per_kq = a.H * terms * (a.K / 64) * kPlane, per_t = a.HV * terms_t * kPlane, per_vec = (int64_t)a.HV * kVec * 4;
  const int64_t per = per_kq + per_t + per_vec;
  Layout l;
  l.total = (a.max_query + kChunk - 1) / kChunk;
  const int64_t most = kWorkspaceBound / per > 1 ? kWorkspaceBound / per : 1, follows = a.N / kChunk + a.B, grid = (int64_t)a.B * l.total;
  l.packed = follows <= most && follows < grid;
  if (l.packed || grid <= most) {
    l.requests = a.B;
    l.chunks = l.total;
    l.places = l.packed ? follows : grid;
  } else {
    l.requests = (int)(most < a.B ? most : a.B);
    l.chunks = (int)(most / l.requests < l.total ? most / l.requests : l.total);
    l.places = (int64_t)l.requests * l.chunks;
  }
  l.kq = l.places * per_kq;
  l.t = l.places * per_t;
  l.vec = l.places * per_vec;
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

template <int DTYPE, int D, int COLUMNS, int STAGES>
int launch_sequence(const ChunkParams& p, int requests, cudaStream_t stream) {
  constexpr size_t smem = sizeof(SequenceShared<kTermsX<DTYPE>, kTermsT<DTYPE>, D, STAGES>) + 1024;
  static_assert(smem <= 227 * 1024, "a CTA's shared memory");
  static thread_local bool ready[64];
  const int rc = allow_shared(sequence_kernel<DTYPE, D, COLUMNS, STAGES>, smem, ready);
  if (rc != CARRY_GDN_OK) return rc;
  return launch_dependent(sequence_kernel<DTYPE, D, COLUMNS, STAGES>, dim3(D / COLUMNS, (unsigned)p.a.HV, (unsigned)requests), kSequenceThreads, smem, stream, p);
}

template <int DTYPE, int D>
int launch_chunks(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  constexpr int kSize = DTYPE == CARRY_F32 ? 4 : 2, kX = kTermsX<DTYPE>;
  constexpr size_t smem = sizeof(PrepareShared<kX, kTermsT<DTYPE>, D>) + 1024;
  static thread_local bool ready[64];
  int rc = allow_shared(prepare_kernel<DTYPE, D>, smem, ready);
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
  for (int b = 0; b < a.B; b += l.requests)
    for (int c = 0; c < l.total; c += l.chunks) {
      p.b0 = b;
      p.chunk0 = c;
      p.chunks = l.total - c < l.chunks ? l.total - c : l.chunks;
      const int requests = a.B - b < l.requests ? a.B - b : l.requests;
      rc = launch_dependent(prepare_kernel<DTYPE, D>, dim3((unsigned)p.chunks, (unsigned)a.H, (unsigned)requests), kPrepareThreads, smem, stream, p);
      if (rc != CARRY_GDN_OK) return rc;
      const bool narrow = (int64_t)requests * a.HV * (D / 64) < sm_count();
      rc = narrow ? launch_sequence<DTYPE, D, 32, kX == 1 ? 2 : 1>(p, requests, stream) : launch_sequence<DTYPE, D, 64, kX == 1 ? 2 : 1>(p, requests, stream);
      if (rc != CARRY_GDN_OK) return rc;
    }
  return CARRY_GDN_OK;
}

template <int DTYPE>
int launch_width(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  return a.K == 64 ? launch_chunks<DTYPE, 64>(a, stream) : launch_chunks<DTYPE, 128>(a, stream);
}

constexpr int kFewTokens = 64;
bool in_chunks(const CarryGdnPrefillArgs& a) { return a.max_query > kFewTokens; }

}  // namespace

int64_t delta_workspace(const CarryGdnPrefillArgs& a) {
  if (!in_chunks(a)) return 0;
  const Layout l = lay_out(a);
  return l.kq + l.t + l.vec;
}

int launch_delta(const CarryGdnPrefillArgs& a, cudaStream_t stream) {
  if (!in_chunks(a)) return launch_delta_recurrent(a, stream);
  return a.qkv_dtype == CARRY_F32 ? launch_width<CARRY_F32>(a, stream)
         : a.qkv_dtype == CARRY_BF16 ? launch_width<CARRY_BF16>(a, stream) : launch_width<CARRY_F16>(a, stream);
}

}  // namespace carry
