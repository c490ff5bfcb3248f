// Attention over the 8-bit key/value cache: one warp for each (row, query head), a token at a time.
#include "carry_hybrid.cuh"

namespace carry {
namespace {

constexpr int kWarps = 4;

// sum = sum * keep + x, with the rounding error carried on
__device__ __forceinline__ void add(float& sum, float& low, float keep, float x) {
  const float y = x - low * keep, before = sum * keep, after = before + y;
  low = (after - before) - y;
  sum = after;
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) kv_attention_kernel(const __grid_constant__ CarryGdnKvAttentionArgs a) {
  constexpr int E = D / 32;                       // columns per lane
  depend_release();
  depend_wait();
  const CarryGdnKvCache& c = a.cache;
  const int b = blockIdx.y, lane = threadIdx.x % 32;
  const long long task = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  const int i = (int)(task / a.HQ), hq = (int)(task % a.HQ), h = hq / (a.HQ / c.HKV);
  const KvRequest r = kv_request(c, a.rows, b, task == 0 && lane == 0 ? a.status : nullptr);
  if (i >= r.todo) return;
  const int seen = max(min(r.length - r.count + i + 1, r.length), 0);
  const long long row = r.first + i;
  float q[E], o[E] = {}, top = -INFINITY, total = 0.0f;
  float o_low[E] = {}, total_low = 0.0f;          // what the sums have lost to rounding
#pragma unroll
  for (int e = 0; e < E; ++e)
    q[e] = load_as_float(a.q, row * a.stride_q_tok + hq * a.stride_q_head + lane * E + e, a.dtype) * a.scale;
  int page = 0;
  for (int j = 0; j < seen; ++j) {
    if (j % c.page == 0) page = kv_page(c, b, j / c.page, lane == 0 ? a.status : nullptr);
    if (page == 0) continue;
    const long long at = ((long long)h * c.page + j % c.page) * D + lane * E;
    const long long s_at = h * (c.page / c.block) + j % c.page / c.block;
    const uint8_t *kc = c.k_codes + page * c.stride_k_page + at, *vc = c.v_codes + page * c.stride_v_page + at;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], __half2float(__half(__nv_cvt_fp8_to_halfraw(kc[e], __NV_E4M3))), s);
#pragma unroll
    for (int x = 16; x > 0; x /= 2) s += __shfl_xor_sync(~0u, s, x);
    s *= c.k_scale[page * c.stride_ks_page + s_at];
    const float now = fmaxf(top, s), base = now == -INFINITY ? 0.0f : now;
    const float keep = expf(top - base), p = expf(s - base), pv = p * c.v_scale[page * c.stride_vs_page + s_at];
    top = now;
    add(total, total_low, keep, p);
#pragma unroll
    for (int e = 0; e < E; ++e) add(o[e], o_low[e], keep, pv * __half2float(__half(__nv_cvt_fp8_to_halfraw(vc[e], __NV_E4M3))));
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    store_from_float(a.out, row * a.stride_out_tok + hq * a.stride_out_head + lane * E + e, a.dtype,
                     total == 0.0f ? 0.0f : o[e] / total);
}

}  // namespace

int64_t kv_attention_workspace(const CarryGdnKvAttentionArgs&) { return 0; }

int launch_kv_attention(const CarryGdnKvAttentionArgs& a, cudaStream_t stream) {
  const long long tasks = (long long)a.rows.max_query * a.HQ;
  const dim3 grid((unsigned)((tasks + kWarps - 1) / kWarps), a.rows.B);
  if (a.cache.D == 64) return launch_dependent(kv_attention_kernel<64>, grid, kWarps * 32, 0, stream, a);
  return launch_dependent(kv_attention_kernel<128>, grid, kWarps * 32, 0, stream, a);
}

}  // namespace carry
