// Attention over the 8-bit key/value cache for many query rows of a request: chunks of a prompt.
//
// A CTA has 256 rows (query tokens times the query heads of one key/value head) as two tiles of 128, and walks the
// request's tokens 64 at a time.  The work is in five places that run side by side:
//  * one warp brings codes in (bulk copies, three steps ahead) and notes their scales;
//  * four warps turn a step's codes into fp16, keys and values (e4m3 is a subset of fp16);
//  * one warp issues the matrix products on the fifth-generation tensor cores: S = Q K^T, operands in shared memory,
//    and O += P V with the weights P in tensor memory;
//  * four warps for each row tile take its scores out of tensor memory, a row to a thread, and put the weights back in
//    their place.  While one tile's weights are formed, the other's products run.
// What bounds it: a step takes 2200 cycles.  Its 2 x 128 x 64 exponentials are 1024 of the special function units, and its products some
// 1330 of the tensor cores (64 columns of scores come at two thirds of the rate of 128, which tensor memory has no room for beside
// the outputs and a second step's scores); neither is full, at 43 % of the cycles each, and what is left is the chain of a row
// tile's step, out of tensor memory and back.  A chunk of 2048 tokens at 16384, 32 heads over 8 of 128: 580 to 600 us, 870 to 900 TFLOP/s,
// 55 % of the burst rate of a large matrix product, at a clock that the GPU's power brings down to 1.5 to 1.6 GHz.
// A CTA's way in and out is some 7 us: six prompts of up to 2000 tokens and 16 heads take 92 to 95 us, 425 TFLOP/s, half of it that.
//
// A row's weights are relative to a maximum that is replaced, and O rescaled, only when it is outgrown by 2^4.  With the value
// scales of their blocks they count in a unit of the row's own, the largest weight times scale that it has met to within a
// power of two, which is looked at again when the maximum moves or a scale is 2^4 above it: blocks that a row does not see, or hardly
// weighs, cost it no bits.  A weight is formed times 2^7, so it stays below fp16's 2^16, and has all its bits down to 2^-21 of
// the row's largest.  The sum takes the scale off again, block by block; scales below 2^-60 of the unit count as 2^-60 in both places, so
// that neither flushes: their values are lost to fp16 and their weights are not.
#include "carry_kv_attention.cuh"

namespace carry {
namespace {

constexpr int kTokens = 64, kStages = 3, kRawStages = 3, kNotes = 8, kTileRows = 128, kCtaRows = 2 * kTileRows;
constexpr int kRowPlane = kTileRows * 128, kTokenPlane = kTokens * 128;        // bytes of a plane: 64 columns of all rows, all tokens
constexpr int kSoftmaxThreads = kCtaRows, kConvertThreads = 128;
constexpr int kFetchWarp = (kSoftmaxThreads + kConvertThreads) / 32, kIssueWarp = kFetchWarp + 1, kAllThreads = (kIssueWarp + 1) * 32;
constexpr int kBlocks = kTokens / kGranule;
constexpr float kUp = 7.0f, kSlack = 4.0f, kLow = -60.0f, kUnitFloor = -100.0f;

template <int D>
struct Shared {
  uint8_t q[2][D / 64][kRowPlane], k[kStages][D / 64][kTokenPlane], v[kStages][D / 64][kTokenPlane];
  uint8_t raw_k[kRawStages][kTokens * D], raw_v[kRawStages][kTokens * D];        // codes as the cache has them
  // of a step's blocks: key scale, log2 of the value scale (minus infinity below 2^-100) and one over it, and of the step the
  // largest of the logarithms.  A step's notes are written again kNotes steps later, when everybody is long done with it:
  // kRawStages + kStages steps at most are under way.
  alignas(16) float ks[kNotes][kBlocks], vs[kNotes][kBlocks], vs_inv[kNotes][kBlocks];
  float vs_top[kNotes];
  uint64_t raw_full[kRawStages], raw_free[kRawStages], k_full[kStages], v_full[kStages], k_free[kStages], v_free[kStages];
  // The rows' threads wait here for a step's notes, and not at k_full, which runs up to three steps ahead of them: once
  // everybody has left the weights of step - 1, the keys of step + 3 can be there before a late warp asks for those of `step`,
  // and a phase that is two behind is not seen.  The notes of step + 8 wait for the weights of step + 2.
  uint64_t noted[kNotes];
  uint64_t s_full[2][2], p_full[2][2], o_done[2][2];   // by tile, and by step's parity
  uint32_t tmem;
  int poison;
};
static_assert(kRawStages + kStages < kNotes, "notes outlive their step");

// ---- waiting ---------------------------------------------------------------------------------------------------------

// Polls of a barrier, each of which the hardware may hold for a while.  The test-only build has a warp of every row tile
// come late to each of its steps, and the other warps to every third or fifth, by more than the others' work on three: results must
// not depend on it.  And there,
// in a cache of three heads, the first copies of request 0's head 1, of the first part where its context is cut, announce 16 bytes
// more than they bring: a wait runs out, and the rows are left as they were.
#ifdef CARRY_TEST_WAIT_EXPIRY
constexpr int kSpinLimit = 1 << 14;
__device__ __forceinline__ void test_come_late(int warp, int step) {
  if (warp < kSoftmaxThreads / 32 ? warp % 4 == step % 4 : (warp + step) % (warp % 2 ? 3 : 5) == 0) __nanosleep(4000);
}
__device__ __forceinline__ uint32_t test_extra_bytes(int heads, int pair, int part, int step) { return heads == 3 && pair == 1 && part == 0 && step == 0 ? 16 : 0; }
#else
constexpr int kSpinLimit = 1 << 20;
__device__ __forceinline__ void test_come_late(int, int) {}
__device__ __forceinline__ uint32_t test_extra_bytes(int, int, int, int) { return 0; }
#endif

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrier_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// arrives, with so many bytes of copies to come
__device__ __forceinline__ void barrier_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_copy(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(to)), "l"(from),
               "r"(bytes), "r"(smem_addr(bar)) : "memory");
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
// number in its group.  The low word of its descriptor counts addresses in units of 16 bytes, so that places further on are
// sums: the issuing thread has a few cycles for each product.  `lead`: bytes between planes of 64 columns, where columns
// are contiguous along the side that is not summed over.
__device__ __forceinline__ uint32_t operand(const void* p, uint32_t lead) { return smem_addr(p) >> 4 | (lead >> 4) << 16; }
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;   // bytes between groups, version, kind of exchange
// fp16 operands, fp32 sums, 128 rows, N columns; `across`: the second operand is contiguous along N
__host__ __device__ constexpr uint32_t instruction(int N, bool across) {
  return 1u << 4 | (across ? 1u << 16 : 0u) | static_cast<uint32_t>(N / 8) << 17 | static_cast<uint32_t>(128 / 16) << 24;
}
// A whole warp comes here, with the same operands in every lane, and one lane (`elected`) issues: what the operands are
// worked out from then stays in uniform registers, which the instruction takes.
__device__ __forceinline__ void mma_shared(uint32_t elected, uint32_t d, uint32_t a, uint32_t b, uint32_t what, bool add) {
  asm volatile("{\n.reg .pred p, q;\n.reg .b64 a, b;\nsetp.ne.b32 p, %5, 0;\nsetp.ne.b32 q, %6, 0;\nmov.b64 a, {%1, %4};\nmov.b64 b, {%2, %4};\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(what), "r"(kOperandHigh),
               "r"(static_cast<uint32_t>(add)), "r"(elected) : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t elected, uint32_t d, uint32_t a, uint32_t b, uint32_t what, bool add) {
  asm volatile("{\n.reg .pred p, q;\n.reg .b64 b;\nsetp.ne.b32 p, %5, 0;\nsetp.ne.b32 q, %6, 0;\nmov.b64 b, {%2, %4};\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(what), "r"(kOperandHigh),
               "r"(static_cast<uint32_t>(add)), "r"(elected) : "memory");
}
// the barrier's phase ends when every product issued so far has
__device__ __forceinline__ void mma_commit(uint32_t elected, uint64_t* bar) {
  asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_addr(bar)),
               "r"(elected) : "memory");
}
__device__ __forceinline__ uint32_t elect() {
  uint32_t mine;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(mine));
  return mine;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

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
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at) : "memory");
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

// Where a row lies, or null for one that is not there.  Each lane works out its own row's place (that takes some forty
// instructions), and D / 8 or eight lanes that have a row between them get it from there.
template <class T>
__device__ __forceinline__ T* place_of(T* mine, int row) {
  return reinterpret_cast<T*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(mine), row));
}

// A warp's 32 query rows as fp16, scaled by powers of two, into their tile; returns what a product of this lane's row
// counts, in log2's scale.  Rows come in whole lines of memory, and each lane then has a row, in place.
template <int D>
__device__ __forceinline__ float stage_queries(const AttnParams& p, const KvRequest& r, int h, int first_row, uint8_t (*tile)[kRowPlane], int tile_row) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;      // lanes to a row, rows at a time
  const int lane = threadIdx.x % 32, chunk = lane % kLanes, row = first_row + lane, token = token_of(p, row);
  const uint16_t* mine = token < r.todo ? reinterpret_cast<const uint16_t*>(p.a.q) + row_place(p, r, h, row, token, p.a.stride_q_tok, p.a.stride_q_head) : nullptr;
#pragma unroll 4
  for (int n = 0; n < 32; n += kRows) {
    const uint16_t* q = place_of(mine, n + lane / kLanes);
    uint8_t* to = tile[chunk / 8] + plane_at(tile_row + n + lane / kLanes, chunk % 8);
    if (!q) {
      *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
    } else if (reinterpret_cast<uintptr_t>(q) % 16 == 0) {
      __pipeline_memcpy_async(to, q + chunk * 8, 16);
    } else {
#pragma unroll 1
      for (int e = 0; e < 8; ++e) reinterpret_cast<uint16_t*>(to)[e] = q[chunk * 8 + e];
    }
  }
  __pipeline_commit();
  __pipeline_wait_prior(0);
  __syncwarp();
  const bool bf16 = p.a.dtype == CARRY_BF16;
  uint32_t top = 0;
#pragma unroll 4
  for (int c = 0; c < kLanes; ++c) {
    const uint4 u = *reinterpret_cast<const uint4*>(tile[c / 8] + plane_at(tile_row + lane, c % 8));
    top = __vmaxu2(__vmaxu2(top, __vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu)), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
  }
  top = max(top >> 16, top & 0xffffu);
  top = bf16 ? top << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top))));
  const int e = up_exponent(top);
  const float up = copysignf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), p.a.scale);
#pragma unroll 4
  for (int c = 0; c < kLanes; ++c) {
    uint4* at = reinterpret_cast<uint4*>(tile[c / 8] + plane_at(tile_row + lane, c % 8));
    const uint4 u = *at;
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = bf16 ? make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u)) : unpack_half2(w[k]);
      w[k] = pack_half2(x.x * up, x.y * up);
    }
    *at = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return fabsf(p.a.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// 128 bytes of each of a warp's 32 rows, which lane l has of row l, to memory by way of shared memory: eight lanes then
// write a row's.  `mine` is where this lane's go, or null; SIZE: of a number.
template <int SIZE>
__device__ __forceinline__ void store_lines(uint8_t* scratch, const uint4 (&x)[8], uint8_t* mine) {
  const int lane = threadIdx.x % 32;
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(scratch + plane_at(lane, c)) = x[c];
  __syncwarp();
#pragma unroll 2
  for (int n = 0; n < 8; ++n) {
    const int row = n * 4 + lane / 8, chunk = lane % 8;
    uint8_t* to = place_of(mine, row);
    const uint4 u = *reinterpret_cast<const uint4*>(scratch + plane_at(row, chunk));
    if (!to) continue;
    to += chunk * 16;
    if (reinterpret_cast<uintptr_t>(to) % 16 == 0) {
      *reinterpret_cast<uint4*>(to) = u;
    } else if constexpr (SIZE == 2) {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) reinterpret_cast<uint16_t*>(to)[e] = static_cast<uint16_t>(w[e / 2] >> (e % 2 * 16));
    }
  }
}

// A converting thread's codes of a step: chunk tid % (D / 16) of tokens tid / (D / 16) + i * kStride.  Tokens at or beyond
// the length (`left` of the step are below it) and those of padding pages are zeros, whatever memory holds there.
template <int D>
__device__ __forceinline__ void convert(const uint8_t* raw, uint8_t (*tile)[kTokenPlane], const float* ks, int left, int tid) {
  constexpr int kChunks = D / 16, kStride = kConvertThreads / kChunks, kCodes = kTokens / kStride;
  const int chunk = tid % kChunks, turn = chunk / 4;         // the planes' stores take turns, or they would meet in the banks
  // rows differ by a multiple of eight, so they lie alike in their groups
  uint8_t* first = tile[chunk / 4] + plane_at(tid / kChunks, chunk % 4 * 2 + turn);
  uint8_t* second = tile[chunk / 4] + plane_at(tid / kChunks, chunk % 4 * 2 + 1 - turn);
  uint4 x[kCodes];
#pragma unroll
  for (int i = 0; i < kCodes; ++i) x[i] = *reinterpret_cast<const uint4*>(raw + tid * 16 + i * kStride * D);
#pragma unroll
  for (int i = 0; i < kCodes; ++i) {
    const int token = tid / kChunks + i * kStride;
    if (token >= left || ks[token / kGranule] == kNoTokens) x[i] = make_uint4(0, 0, 0, 0);
    uint4 lo, hi;
    halves_of(x[i].x, lo.x, lo.y);
    halves_of(x[i].y, lo.z, lo.w);
    halves_of(x[i].z, hi.x, hi.y);
    halves_of(x[i].w, hi.z, hi.w);
    *reinterpret_cast<uint4*>(first + i * kStride * 128) = turn ? hi : lo;
    *reinterpret_cast<uint4*>(second + i * kStride * 128) = turn ? lo : hi;
  }
}

// What the fetching warp knows of the steps to come: lane l has granule l of each.  What a step waits for has been asked for
// before: its scales a step, the page ids behind them two steps ago.
template <int D>
struct Fetch {
  struct Granule {
    int id, in_page;
    float ks, vs;
  };
  const AttnParams& p;
  const int b, h, step0, length;
  Granule now, next, after;
  __device__ __forceinline__ Fetch(const AttnParams& p, int b, int h, int step0, int length) : p(p), b(b), h(h), step0(step0), length(length) {}
  __device__ __forceinline__ void find(int step, Granule& g) const {
    const int lane = threadIdx.x % 32, granule = (step0 + step) * kBlocks + lane;
    g.id = lane < kBlocks ? page_id(p, b, granule, length) : 0;
    g.in_page = granule - page_index(p, granule) * p.page_granules;
  }
  __device__ __forceinline__ void scales(Granule& g) const {
    const CarryGdnKvCache& c = p.a.cache;
    const int block = h * divide(p.page_granules, p.block_granules, p.block_shift) + divide(g.in_page, p.block_granules, p.block_shift);
    g.ks = g.id > 0 ? c.k_scale[g.id * c.stride_ks_page + block] : kNoTokens;
    g.vs = g.id > 0 ? c.v_scale[g.id * c.stride_vs_page + block] : 0.0f;
  }
  __device__ __forceinline__ void begin() {
    find(0, now);
    find(1, next);
    scales(now);
  }
  __device__ __forceinline__ void ahead(int step) {
    find(step + 2, after);
    scales(next);
  }
  __device__ __forceinline__ void advance() {
    now = next;
    next = after;
  }
};

template <int D>
__global__ void __launch_bounds__(kAllThreads, 1) kv_prefill_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ uint8_t raw[];
  Shared<D>& sh = *reinterpret_cast<Shared<D>*>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
  depend_release();
  depend_wait();
  const CarryGdnKvCache& c = p.a.cache;
  // The longest contexts go first.  Those of the first `cut` row tiles are cut into parts, and come last.
  const int cut = p.padded / kCtaRows, whole = gridDim.y - cut * p.splits, late = (int)blockIdx.y - whole;
  const int splits = late < 0 ? 1 : p.splits, part_number = late < 0 ? 0 : late % splits;
  const int b = blockIdx.x / c.HKV, h = blockIdx.x % c.HKV, first_row = cut * kCtaRows + (late < 0 ? -1 - late : -1 - late / splits) * kCtaRows;
  const int warp = threadIdx.x / 32;
  const KvRequest r = kv_request(c, p.a.rows, b, first_row == 0 && h == 0 && threadIdx.x == 0 ? p.a.status : nullptr);
  if (first_row >= r.todo * p.group) return;
  const int tiles = first_row + kTileRows < r.todo * p.group ? 2 : 1;      // a second tile without rows takes no part
  const int last = min(token_of(p, first_row + kCtaRows - 1), r.todo - 1);
  const int length = max(min(r.length, r.length - r.count + last + 1), 0), all_steps = (length + kTokens - 1) / kTokens;
  const int share = (all_steps + splits - 1) / splits, step0 = min(share * part_number, all_steps), steps = min(share, all_steps - step0);

  if (threadIdx.x == 0) {
    sh.poison = 0;
    for (int i = 0; i < kRawStages; ++i) {
      barrier_init(&sh.raw_full[i], 1);
      barrier_init(&sh.raw_free[i], kConvertThreads);
    }
    for (int i = 0; i < kStages; ++i) {
      barrier_init(&sh.k_full[i], kConvertThreads);
      barrier_init(&sh.v_full[i], kConvertThreads);
      barrier_init(&sh.k_free[i], 1);
      barrier_init(&sh.v_free[i], 1);
    }
    for (int i = 0; i < kNotes; ++i) barrier_init(&sh.noted[i], 1);
    for (int i = 0; i < 4; ++i) {
      barrier_init(&sh.s_full[i / 2][i % 2], 1);
      barrier_init(&sh.p_full[i / 2][i % 2], kTileRows);
      barrier_init(&sh.o_done[i / 2][i % 2], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the fetching warp's first trips to memory run while the queries are staged
  Fetch<D> fetch(p, b, h, step0, length);
  if (warp == kFetchWarp) fetch.begin();
  float unit_q = 0.0f;
  if (threadIdx.x < kSoftmaxThreads) {
    unit_q = stage_queries<D>(p, r, h, first_row + warp * 32, sh.q[warp / 4], warp % 4 * 32);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;                  // columns 0, 128: scores of the tiles, 64 of a step and 64 of the next; 256, 384: outputs
  volatile int* poison = &sh.poison;

  if (threadIdx.x < kSoftmaxThreads) {
    // ---- a row to a thread ----
    const int tile = threadIdx.x / kTileRows, row = first_row + threadIdx.x, i = token_of(p, row);
    const int sees = i < r.todo ? r.length - r.count + i + 1 : 0;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t s_at = tmem + lanes + tile * 128, o_at = tmem + lanes + 256 + tile * 128;
    // outputs count in 2^(unit - kUp), which is `in_unit`, beside 2^top
    float top = -INFINITY, sum = 0.0f, unit = kUnitFloor, in_unit = exp2f(kUnitFloor - kUp);
    bool healthy = true;
    for (int step = 0; step < steps && tile < tiles; ++step) {
      const int note = step % kNotes, turn = step & 1;
      test_come_late(warp, step);
      healthy = __all_sync(~0u, barrier_wait(&sh.noted[note], step / kNotes & 1, poison, p.a.status) &&
                                    barrier_wait(&sh.s_full[tile][turn], step / 2 & 1, poison, p.a.status));
      if (!healthy) break;
      fence_after();
      float x[2][32], now = top, by[kBlocks], peak[kBlocks], ks[kBlocks], vs[kBlocks], vs_inv[kBlocks];
      tmem_load(s_at + turn * 64, x[0]);
      tmem_load(s_at + turn * 64 + 32, x[1]);
      *reinterpret_cast<float4*>(ks) = *reinterpret_cast<const float4*>(sh.ks[note]);
      *reinterpret_cast<float4*>(vs) = *reinterpret_cast<const float4*>(sh.vs[note]);
      *reinterpret_cast<float4*>(vs_inv) = *reinterpret_cast<const float4*>(sh.vs_inv[note]);
      const float vs_top = sh.vs_top[note];
      const int limit = sees - (step0 + step) * kTokens;
      bool all = limit >= kTokens;
#pragma unroll
      for (int block = 0; block < kBlocks; ++block) all = all && ks[block] != kNoTokens;
      all = __all_sync(~0u, all);
      wait_loads();
      if (!all) {
#pragma unroll
        for (int e = 0; e < kTokens; ++e) x[e / 32][e % 32] = e < limit && ks[e / 16] != kNoTokens ? x[e / 32][e % 32] : -INFINITY;
      }
#pragma unroll
      for (int block = 0; block < kBlocks; ++block) {
        const float* y = x[block / 2] + block % 2 * 16;
        float m = fmaxf(y[0], y[1]), n = fmaxf(y[2], y[3]);
#pragma unroll
        for (int e = 4; e < 16; e += 4) {
          m = fmaxf(m, fmaxf(y[e], y[e + 1]));
          n = fmaxf(n, fmaxf(y[e + 2], y[e + 3]));
        }
        by[block] = fmaxf(unit_q * ks[block], 0x1p-126f);
        peak[block] = fmaxf(m, n) * by[block];
        now = fmaxf(now, peak[block]);
      }
      if (__any_sync(~0u, now > top + kSlack || (vs_top > unit + kSlack && now > -INFINITY))) {
        const float moved = now == -INFINITY ? 0.0f : top - now, zero = now == -INFINITY ? 0.0f : now, had = unit + moved;
        float then = fmaxf(had, kUnitFloor);
#pragma unroll
        for (int block = 0; block < kBlocks; ++block) then = fmaxf(then, peak[block] + vs[block] - zero);
        unit = ceilf(then);                       // a whole number, so that powers of two are exact in it
        in_unit = exp2f(unit - kUp);
        top = now;
        sum *= exp2_fast(moved);
        if (step > 0) {
          healthy = __all_sync(~0u, barrier_wait(&sh.o_done[tile][turn ^ 1], (step - 1) / 2 & 1, poison, p.a.status));
          if (!healthy) break;
          fence_after();
          const float less = exp2_fast(had - unit);
#pragma unroll 1
          for (int n = 0; n < D / 16; ++n) {
            uint32_t o[16];
            tmem_load16(o_at + n * 16, o);
            wait_loads();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * less);
            tmem_store16(o_at + n * 16, o);
          }
          wait_stores();
        }
      }
      const float rest = (top == -INFINITY ? 0.0f : top) - kUp;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[16];
#pragma unroll
        for (int block = 2 * half; block < 2 * half + 2; ++block) {
          const float* z = x[half] + block % 2 * 16;
          const float less = fmaxf(vs[block] - unit, kLow) - rest;
          float2 total = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float2 y = fma2(make_float2(z[e], z[e + 1]), make_float2(by[block], by[block]), make_float2(less, less));
            const float2 q = make_float2(exp2_fast(y.x), exp2_fast(y.y));
            total = add2(total, q);
            w[block % 2 * 8 + e / 2] = pack_half2(q.x, q.y);
          }
          sum = fmaf(total.x + total.y, fminf(in_unit * vs_inv[block], exp2f(-kLow - kUp)), sum);
        }
        tmem_store16(s_at + turn * 64 + half * 16, w);           // over scores that this warp has read
      }
      wait_stores();
      fence_before();
      barrier_arrive(&sh.p_full[tile][turn]);
    }
    if (healthy && steps > 0 && tile < tiles) {
      healthy = __all_sync(~0u, barrier_wait(&sh.o_done[tile][(steps - 1) & 1], (steps - 1) / 2 & 1, poison, p.a.status));
      fence_after();
    }
    if (!healthy && splits > 1 && i < r.todo) parts_of(p, part_number, blockIdx.x).sum[row] = kNoPart;
    if (healthy && first_row + warp * 32 < r.todo * p.group) {       // a warp without rows has nothing to leave
      const float by = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
      const Parts part = parts_of(p, part_number, blockIdx.x);
      if (splits > 1 && i < r.todo) {
        part.top[row] = top;
        part.sum[row] = sum;
      }
      // every score has been formed by now, so the queries' memory is free: 4 KB to a warp
      uint8_t* scratch = sh.q[0][0] + warp * 4096;
      uint16_t* mine = i < r.todo ? reinterpret_cast<uint16_t*>(p.a.out) + row_place(p, r, h, row, i, p.a.stride_out_tok, p.a.stride_out_head) : nullptr;
      auto numbers = [&](int n, float (&x)[32]) {  // columns 32 n and on
        if (steps > 0) tmem_load(o_at + n * 32, x);
        wait_loads();
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = sum == 0.0f ? 0.0f : x[e] * by * in_unit;
      };
      float x[32];
      uint4 line[8];
      if (splits > 1) {
#pragma unroll 1
        for (int n = 0; n < D / 32; ++n) {
          numbers(n, x);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            line[e] = make_uint4(__float_as_uint(x[4 * e]), __float_as_uint(x[4 * e + 1]), __float_as_uint(x[4 * e + 2]), __float_as_uint(x[4 * e + 3]));
          store_lines<4>(scratch, line, i < r.todo ? reinterpret_cast<uint8_t*>(part.o + (long long)row * D + n * 32) : nullptr);
        }
      } else {
#pragma unroll 1
        for (int n = 0; n < D / 64; ++n) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            numbers(n * 2 + half, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              auto two = [&](int k) { return p.a.dtype == CARRY_BF16 ? pack_bf16(x[8 * e + k], x[8 * e + k + 1]) : pack_half2(x[8 * e + k], x[8 * e + k + 1]); };
              line[half * 4 + e] = make_uint4(two(0), two(2), two(4), two(6));
            }
          }
          store_lines<2>(scratch, line, mine ? reinterpret_cast<uint8_t*>(mine + n * 64) : nullptr);
        }
      }
    }
  } else if (threadIdx.x < kSoftmaxThreads + kConvertThreads) {
    // ---- codes to operands ----
    const int tid = threadIdx.x - kSoftmaxThreads;
    int raw = 0, stage = 0, raw_parity = 0, parity = 1;
    for (int step = 0; step < steps; ++step) {
      const int left = length - (step0 + step) * kTokens;
      const float* ks = sh.ks[step % kNotes];
      test_come_late(warp, step);
      if (!barrier_wait(&sh.raw_full[raw], raw_parity, poison, p.a.status)) break;
      if (step >= kStages && !barrier_wait(&sh.k_free[stage], parity, poison, p.a.status)) break;
      convert<D>(sh.raw_k[raw], sh.k[stage], ks, left, tid);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      barrier_arrive(&sh.k_full[stage]);
      if (step >= kStages && !barrier_wait(&sh.v_free[stage], parity, poison, p.a.status)) break;
      convert<D>(sh.raw_v[raw], sh.v[stage], ks, left, tid);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      barrier_arrive(&sh.v_full[stage]);
      barrier_arrive(&sh.raw_free[raw]);
      if (++raw == kRawStages) { raw = 0; raw_parity ^= 1; }
      if (++stage == kStages) { stage = 0; parity ^= 1; }
    }
  } else if (warp == kFetchWarp) {
    // ---- codes and scales out of the cache ----
    const int lane = threadIdx.x % 32;
    int raw = 0, parity = 1;
    for (int step = 0; step < steps; ++step) {
      fetch.ahead(step);
      test_come_late(warp, step);
      const typename Fetch<D>::Granule& now = fetch.now;
      if (step >= kRawStages && !__all_sync(~0u, barrier_wait(&sh.raw_free[raw], parity, poison, p.a.status))) break;
      const uint32_t there = __ballot_sync(~0u, now.id > 0);
      const bool counts = now.vs >= exp2f(kUnitFloor);
      const uint32_t bits = __float_as_uint(now.vs);
      const float vs = counts ? static_cast<int>(bits >> 23) - 127 + __log2f(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u)) : -INFINITY;
      float most = vs;
#pragma unroll
      for (int d = kBlocks / 2; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
      const int note = step % kNotes;
      if (lane < kBlocks) {
        sh.ks[note][lane] = now.ks;
        sh.vs[note][lane] = vs;
        sh.vs_inv[note][lane] = counts ? __fdiv_rn(1.0f, now.vs) : INFINITY;
      }
      if (lane == 0) sh.vs_top[note] = most;
      __syncwarp();
      if (lane == 0) {                            // what was written above goes with both
        barrier_arrive(&sh.noted[note]);
        barrier_expect(&sh.raw_full[raw], 2 * kGranule * D * __popc(there) + test_extra_bytes(c.HKV, blockIdx.x, part_number, step));
      }
      __syncwarp();
      if (now.id > 0) {
        const int at = (h * c.page + now.in_page * kGranule) * D, to = lane * kGranule * D;
        bulk_copy(sh.raw_k[raw] + to, c.k_codes + now.id * c.stride_k_page + at, kGranule * D, &sh.raw_full[raw]);
        bulk_copy(sh.raw_v[raw] + to, c.v_codes + now.id * c.stride_v_page + at, kGranule * D, &sh.raw_full[raw]);
      }
      fetch.advance();
      if (++raw == kRawStages) { raw = 0; parity ^= 1; }
    }
  } else {
    // ---- products ----
    const uint32_t elected = elect(), base = __shfl_sync(~0u, tmem, 0);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, barrier_wait(bar, parity, poison, p.a.status)) != 0; };
    constexpr uint32_t kRowStep = kRowPlane >> 4, kTokenStep = kTokenPlane >> 4, kStageStep = kTokenStep * (D / 64);
    const uint32_t q0 = operand(sh.q, 16), k0 = operand(sh.k, 16), v0 = operand(sh.v, kTokenPlane);
    auto scores = [&](int tile, int step) {
      const uint32_t q = q0 + tile * kRowStep * (D / 64), keys = k0 + step % kStages * kStageStep, to = base + tile * 128 + (step & 1) * 64;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        mma_shared(elected, to, q + k / 4 * kRowStep + k % 4 * 2, keys + k / 4 * kTokenStep + k % 4 * 2, instruction(kTokens, false), k > 0);
      mma_commit(elected, &sh.s_full[tile][step & 1]);
      if (tile + 1 == tiles) mma_commit(elected, &sh.k_free[step % kStages]);
    };
    bool healthy = true;
    for (int step = 0; step < 2 && step < steps && healthy; ++step) {
      healthy = wait(&sh.k_full[step], 0);
      if (!healthy) break;
      fence_after();
      scores(0, step);
      if (tiles == 2) scores(1, step);
    }
    for (int step = 0; healthy && step < steps; ++step) {
      const int stage = step % kStages, turn = step & 1, parity = step / kStages & 1;
      const uint32_t values = v0 + stage * kStageStep;
      test_come_late(warp, step);
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        if (tile >= tiles) break;
        healthy = (tile > 0 || wait(&sh.v_full[stage], parity)) &&
                  wait(&sh.p_full[tile][turn], step / 2 & 1);
        if (!healthy) break;
        fence_after();
#pragma unroll
        for (int k = 0; k < kTokens / 16; ++k)
          mma_tensor(elected, base + 256 + tile * 128, base + tile * 128 + turn * 64 + k * 8,
                     values + k * 128, instruction(D, true), step > 0 || k > 0);
        mma_commit(elected, &sh.o_done[tile][turn]);
        if (tile + 1 == tiles) mma_commit(elected, &sh.v_free[stage]);
        if (step + 2 < steps) {
          healthy = tile > 0 || wait(&sh.k_full[(step + 2) % kStages], (step + 2) / kStages & 1);
          if (!healthy) break;
          fence_after();
          scores(tile, step + 2);                 // where this step's weights were: products run in order
        }
      }
    }
  }
  if (*poison) {
    // products and copies in flight still use shared and tensor memory: a bounded time for them to end
    for (int i = 0; i < 1 << 12; ++i) __nanosleep(64);
  }
  fence_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

long long row_tiles(const CarryGdnKvAttentionArgs& a) {
  return ((long long)a.rows.max_query * (a.HQ / a.cache.HKV) + kCtaRows - 1) / kCtaRows;
}

// What does not fill the processors is cut: the CTAs beyond the last full round of one to a processor (all of them, where
// they are few), which are the first row tiles' of every (request, head).  Into as many parts, of two steps or more, as bring
// the end nearest, counted in steps of 64 tokens: a part costs some four of its own, and its outputs, written and read, a
// twentieth; the join four.  A chunk of 2048 tokens, 32 heads over 8, at 16384 tokens has 256 CTAs and takes 600 us either way, for
// the processors that stay idle leave the others their power; one of 1280 has 160 and takes 379 us, 592 uncut.  Four requests of
// 16 tokens over 941 take 19.7 us, 27.4 with parts of eight steps or more.
void lay_out(const CarryGdnKvAttentionArgs& a, int& splits, int& padded) {
  const long long tiles = row_tiles(a), pairs = (long long)a.cache.HKV * a.rows.B, sms = sm_count();
  splits = 1;
  padded = tiles > 65535 ? -1 : 0;
  if (pairs == 0 || sms == 0) return;
  const long long late = tiles * pairs % sms, cut = tiles - (tiles * pairs - late) / pairs;
  if (cut == 0 || cut > 1024 || tiles > 30000) return;
  const long long cached = max((long long)a.cache.max_pages * a.cache.page - a.rows.max_query, 0LL);
  const long long steps = (cached + min(cut * kCtaRows / (a.HQ / a.cache.HKV), (long long)a.rows.max_query) + 63) / 64;
  long long least = (late + sms - 1) / sms * (steps + 4);
  for (int n = 2; n <= 32 && n * 2 <= steps; ++n) {
    const long long cost = (late * n + sms - 1) / sms * ((steps + n - 1) / n + 4) + cut * pairs * n * a.cache.D / (20 * 128) + 4;
    if (cost < least) {
      least = cost;
      splits = n;
      padded = (int)cut * kCtaRows;
    }
  }
}

template <int D>
int launch(const AttnParams& p, cudaStream_t stream) {
  constexpr size_t smem = sizeof(Shared<D>) + 1024;
  static thread_local bool ready[64];
  const int rc = prepare(kv_prefill_kernel<D>, smem, ready);
  if (rc != CARRY_GDN_OK) return rc;
  const long long tiles = row_tiles(p.a), cut = p.padded / kCtaRows;
  const dim3 grid((unsigned)p.a.cache.HKV * p.a.rows.B, (unsigned)(tiles - cut + cut * p.splits));
  return launch_dependent(kv_prefill_kernel<D>, grid, kAllThreads, smem, stream, p);
}

}  // namespace

int64_t kv_prefill_workspace(const CarryGdnKvAttentionArgs& a) {
  int splits, padded;
  lay_out(a, splits, padded);
  return padded < 0 ? CARRY_GDN_ERR_TOO_LARGE : parts_bytes(a, splits, padded);
}

int launch_kv_prefill(AttnParams p, cudaStream_t stream) {
  lay_out(p.a, p.splits, p.padded);
  const int rc = p.a.cache.D == 64 ? launch<64>(p, stream) : launch<128>(p, stream);
  return rc == CARRY_GDN_OK && p.splits > 1 ? launch_join_parts(p, stream) : rc;
}

}  // namespace carry
