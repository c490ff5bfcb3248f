// What the kernels on the fifth-generation tensor cores share: barriers in shared memory with bounded waits, bulk copies,
// operands, products and tensor memory.
#pragma once

#include "carry_gdn_common.cuh"

namespace carry {

// Polls of a barrier, each of which the hardware may hold for a while.
#ifdef CARRY_TEST_WAIT_EXPIRY
constexpr int kSpinLimit = 1 << 14;
#else
constexpr int kSpinLimit = 1 << 20;
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
__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
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

// where the 16-byte chunk `chunk` (eight numbers) of a row of a plane lies
__device__ __forceinline__ int plane_at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// bf16 operands, fp32 sums, 128 rows, N columns; `across`: that operand is contiguous along the side that is not summed over
__host__ __device__ constexpr uint32_t instruction_bf16(int N, bool a_across, bool b_across) {
  return instruction(N, b_across) | 1u << 7 | 1u << 10 | (a_across ? 1u << 15 : 0u);
}
// shared memory to global memory, in the calling thread's open group of copies
__device__ __forceinline__ void bulk_store(void* to, const void* from, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_addr(from)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

}  // namespace carry
