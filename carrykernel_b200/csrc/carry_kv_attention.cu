// Attention over the 8-bit key/value cache.
//
// Scores s = scale * q . k and outputs sum_j softmax_j(s) v_j in one pass over the cache, with the running maximum and
// sum of an online softmax.  Keys and values stay e4m3 until they are on the processor: tiles come into a ring of
// shared-memory stages by asynchronous copies, and the codes become the fp16 operands of the matrix instructions there
// (e4m3 is a subset of fp16).  What each rounding to 16 bits costs:
//  * a query row is scaled by a power of two until its largest number is in [2^14, 2^15): bf16 and fp16 numbers fit fp16
//    exactly down to 2^-29 of the largest, fp32 ones go in two parts (22 bits);
//  * the weights p of the softmax are fp16 (2^-12 of each, against 2^-9 for the rounding of a bf16 output), with fp32
//    queries in two parts.  They carry the value scale of their block relative to the largest scale that the warp
//    has met or, where those lie far apart, to the row's largest weight times scale, and 2^15: weights down to 2^-21 of the
//    largest have all their bits, and to 2^-29 where scales are the same (in the tensor-memory kernel always to the row's, and 2^7).
// Scores, maxima, sums and outputs are fp32.
//
// Up to 16 rows of a (request, head) go to carry_kv_decode.cu, more to carry_kv_prefill.cu or, where they are fp32, to
// carry_kv_chunk.cu (32 rows of 256 (request, head)s over 4096 tokens: 208 us on the tensor-memory kernel, 241 in a warp's
// registers).
#include "carry_kv_attention.cuh"

namespace carry {
namespace {

constexpr int kJoinWarps = 4, kJoinThreads = kJoinWarps * 32;

// Joins the parts of a context, a row to a warp: lane s has part s's weight, then the lanes have the columns.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_parts_kernel(const __grid_constant__ AttnParams p) {
  depend_release();
  depend_wait();
  const int lane = threadIdx.x % 32, row = blockIdx.y * kJoinWarps + threadIdx.x / 32;
  const int b = blockIdx.x / p.a.cache.HKV, h = blockIdx.x % p.a.cache.HKV, i = token_of(p, row);
  const KvRequest q = kv_request(p.a.cache, p.a.rows, b, nullptr);
  if (i >= q.todo || row >= p.padded) return;
  const Parts mine = parts_of(p, min(lane, p.splits - 1), blockIdx.x);
  float top = lane < p.splits ? mine.top[row] : -INFINITY, w = lane < p.splits ? mine.sum[row] : 0.0f;
  if (__any_sync(~0u, w == kNoPart)) return;
  const float all_top = warp_max(top), base = all_top == -INFINITY ? 0.0f : all_top;
  w *= exp2_fast(top - base - kJoinDown);
  float sum = w, o[D / 32] = {};
#pragma unroll
  for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    const float* x = parts_of(p, s, blockIdx.x).o + (long long)row * D + lane;
    const float by = __shfl_sync(~0u, w, s);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] = fmaf(by, x[e * 32], o[e]);
  }
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
    store_from_float(p.a.out, row_place(p, q, h, row, i, p.a.stride_out_tok, p.a.stride_out_head) + e * 32 + lane, p.a.dtype,
                     sum == 0.0f ? 0.0f : __fdiv_rn(o[e], sum));
}

}  // namespace

int launch_join_parts(const AttnParams& p, cudaStream_t stream) {
  const dim3 grid((unsigned)p.a.cache.HKV * p.a.rows.B, (unsigned)((min(p.rows, p.padded) + kJoinWarps - 1) / kJoinWarps));
  return p.a.cache.D == 64 ? launch_dependent(kv_join_parts_kernel<64>, grid, kJoinThreads, 0, stream, p)
                           : launch_dependent(kv_join_parts_kernel<128>, grid, kJoinThreads, 0, stream, p);
}

int64_t kv_attention_workspace(const CarryGdnKvAttentionArgs& a) {
  if (sm_count() == 0) return CARRY_GDN_ERR_NO_DEVICE;
  return few_rows(a) ? kv_decode_workspace(a) : a.dtype == CARRY_F32 ? kv_chunk_workspace(a) : kv_prefill_workspace(a);
}

int launch_kv_attention(const CarryGdnKvAttentionArgs& a, cudaStream_t stream) {
  AttnParams p = {};
  p.a = a;
  p.group = a.HQ / a.cache.HKV;
  p.page_granules = a.cache.page / kGranule;
  p.block_granules = a.cache.block / kGranule;
  p.group_shift = shift_of(p.group);
  p.page_shift = shift_of(p.page_granules);
  p.block_shift = shift_of(p.block_granules);
  p.rows = a.rows.max_query * p.group;
  p.splits = 1;
  return few_rows(a) ? launch_kv_decode(p, stream) : a.dtype == CARRY_F32 ? launch_kv_chunk(p, stream) : launch_kv_prefill(p, stream);
}

}  // namespace carry
