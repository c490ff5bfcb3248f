/*
 * carry_gdn.h -- C ABI of libcarry_gdn.so: the fused Gated-DeltaNet decode step
 * on an INT8 recurrent state with an error-feedback residual, for NVIDIA B200
 * (sm_100a).
 *
 * Every entry point takes plain device pointers and sizes and a CUDA stream
 * handle (a cudaStream_t passed as void*).  The library never allocates device
 * memory, never synchronises and never changes the current device: the caller
 * makes the right device current, owns every buffer and keeps it alive until
 * the stream has run the kernel.  Return value: 0 on success, a negative
 * CARRY_GDN_ERR_* otherwise; nothing throws across this boundary.  Every entry
 * point reads away the CUDA runtime's per-thread "last error" first, so that a
 * launch failure it reports is its own.
 *
 * What each entry point replaces in tomalmog/carrykernel (paths relative to
 * that project) is cited above it.
 */
#ifndef CARRY_GDN_H_
#define CARRY_GDN_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CARRY_GDN_ABI_VERSION 4

/* element types of activations / outputs */
enum { CARRY_F32 = 0, CARRY_BF16 = 1, CARRY_F16 = 2 };

/* residual storage: ids 0..3 are statequant/kernel.py:59-63; 4 and 5 are new */
enum {
  CARRY_RES_FP32 = 0,
  CARRY_RES_FP16 = 1,
  CARRY_RES_FP8 = 2,  /* e5m2 */
  CARRY_RES_INT8 = 3, /* codes + scale */
  CARRY_RES_INT4 = 4, /* two codes per byte along the contiguous axis, even index low nibble */
  CARRY_RES_NONE = 5  /* no error feedback: plain re-quantisation */
};

/* granularity of a scale: one per V channel, or one per (slot, head) matrix */
enum { CARRY_SCALE_PER_V = 0, CARRY_SCALE_PER_HEAD = 1 };

/* scale floor: max(amax, 1e-12)/qmax (statequant/kernel.py:110,173) or
 * max(amax/qmax, 1e-12) (vllm_integration/quantized_packed_decode.py:206,213) */
enum { CARRY_EPS_ON_AMAX = 0, CARRY_EPS_ON_SCALE = 1 };

enum {
  CARRY_GDN_OK = 0,
  CARRY_GDN_ERR_NULL = -1,        /* a required pointer is NULL */
  CARRY_GDN_ERR_SHAPE = -2,       /* a dimension is non-positive or inconsistent */
  CARRY_GDN_ERR_DTYPE = -3,       /* unknown element type id */
  CARRY_GDN_ERR_FORMAT = -4,      /* unknown residual format / scale mode, or odd length for int4 */
  CARRY_GDN_ERR_UNSUPPORTED = -5, /* tile too large for one SM's shared memory */
  CARRY_GDN_ERR_LAUNCH = -6,      /* the CUDA runtime refused the launch */
  CARRY_GDN_ERR_NO_DEVICE = -7,   /* no usable sm_100 device is current */
  CARRY_GDN_ERR_TOO_LARGE = -8    /* beyond a stated fixed capacity */
};

/* bits of the optional device-side status word (OR-ed in by the kernels) */
enum {
  CARRY_GDN_STATUS_BAD_SLOT = 1,   /* a slot id was >= num_slots; that request was treated as padding */
  CARRY_GDN_STATUS_TIMEOUT = 2,    /* an asynchronous copy did not complete within the wait limit: that CTA
                                      stopped loading and storing and left its remaining tiles untouched */
  CARRY_GDN_STATUS_BAD_RANGE = 4   /* key/value cache: a page id, a length or a query range lay outside of what the
                                      call was given; what lay outside was skipped */
};

/*
 * One fused step in the statequant layout: state [B, HV, K, V], V contiguous.
 * Replaces ext.gdn_quant_step(14 tensors, qmax, res_fmt, block_v)
 * (cuda/gdn_state_kernel.cu:310-348, bound at :373-377) and the Triton launch in
 * statequant/kernel.py:379-408.  Output buffers may alias the matching inputs
 * (in-place update); they must not partially overlap anything else.
 */
typedef struct CarryGdnStepArgs {
  const int8_t* h_in;      /* [B,HV,K,V] state codes */
  const float* scale_in;   /* [B,HV,V] (PER_V) or [B,HV] (PER_HEAD) */
  const void* e_in;        /* residual, [B,HV,K,V] in res_fmt ([.., V/2] bytes for INT4); NULL for RES_NONE */
  const float* e_scale_in; /* [B,HV,V] or [B,HV]; INT8/INT4 only, else may be NULL */
  const void* q;           /* [B,HV,K] qkv_dtype */
  const void* k;           /* [B,HV,K] */
  const void* v;           /* [B,HV,V] */
  const float* alpha;      /* [B,HV] decay */
  const float* beta;       /* [B,HV] write strength */
  void* o;                 /* [B,HV,V] o_dtype */
  int8_t* h_out;
  float* scale_out;
  void* e_out;
  float* e_scale_out;
  int32_t B, HV, K, V;
  int32_t qkv_dtype;        /* CARRY_F32 | CARRY_BF16 | CARRY_F16 */
  int32_t o_dtype;
  float qmax;               /* 2^(bits-1) - 1 */
  int32_t res_fmt;          /* CARRY_RES_* */
  int32_t resid_scale_mode; /* CARRY_SCALE_* (INT8/INT4 residual) */
  int32_t state_scale_mode; /* CARRY_SCALE_* */
  int32_t eps_mode;         /* CARRY_EPS_* */
  int32_t* status;          /* optional device word, may be NULL */
} CarryGdnStepArgs;

int carry_gdn_quant_step(const CarryGdnStepArgs* args, void* stream);

/*
 * T chained steps from a floating-point state, in one call: h0 [B, HV, K, V] fp32 is quantised (scale =
 * max(amax_K |h0|, 1e-12) * (1 / qmax), codes = round_half_even(h0 / scale), zero residual), then every request's
 * token t = 0 .. T-1 is applied as carry_gdn_quant_step would.  Replaces the loop of statequant/kernel.py:435-452.
 * `step` gives the formats, the sizes and the final state's buffers (h_out, scale_out, e_out); its *_in pointers are
 * not read.  q, k, v, alpha, beta and o carry T in front: [T, B, HV, ...].  Only what the one-launch kernel takes is
 * supported (K = V = 128, a floating-point residual, per-V state scales); anything else returns
 * CARRY_GDN_ERR_UNSUPPORTED and the caller loops over tokens.
 */
typedef struct CarryGdnDecodeArgs {
  CarryGdnStepArgs step;
  const float* h0;
  int32_t T;
} CarryGdnDecodeArgs;

int carry_gdn_quant_decode(const CarryGdnDecodeArgs* args, void* stream);

/*
 * Unquantised fp32 step, state [B, HV, K, V] fp32.  Replaces
 * ext.gdn_fp32_step (cuda/gdn_state_kernel.cu:350-371) and
 * statequant/kernel.py:411-433.  h_out may alias h_in.
 */
typedef struct CarryGdnFp32Args {
  const float* h_in;
  const void* q;
  const void* k;
  const void* v;
  const float* alpha;
  const float* beta;
  void* o;
  float* h_out;
  int32_t B, HV, K, V;
  int32_t qkv_dtype;
  int32_t o_dtype;
} CarryGdnFp32Args;

int carry_gdn_fp32_step(const CarryGdnFp32Args* args, void* stream);

/*
 * One slot-indexed step, in place on a paged pool [slots, HV, V, K] (K
 * contiguous).  Replaces the Triton launch of _quant_int8_kernel
 * (vllm_integration/quantized_packed_decode.py:303-326; kernel :101-239).
 * Request n uses slot ssm_state_indices[n]; a slot id <= 0 is padding: zeros go
 * to out[n] and the pool is not touched.  Two requests must not name the same
 * slot.  Strides are in elements.
 */
typedef struct CarryGdnPackedArgs {
  const void* mixed_qkv;  /* [B, 2*H*K + HV*V], last stride 1: q | k | v */
  int64_t stride_mixed_tok;
  int32_t qkv_dtype;
  const void* a;          /* [B, HV] */
  int64_t stride_a_tok;
  const void* b;          /* [B, HV] */
  int64_t stride_b_tok;
  int32_t ab_dtype;
  const void* A_log;      /* [HV] */
  int32_t A_log_dtype;
  const void* dt_bias;    /* [HV] */
  int32_t dt_bias_dtype;
  float scale;            /* multiplies q after the optional L2 norm */
  int8_t* state_codes;    /* [slots, HV, V, K] */
  float* state_scale;     /* [slots, HV, V] */
  int8_t* resid_codes;    /* [slots, HV, V, K] (INT8) or [slots, HV, V, K/2] (INT4) */
  float* resid_scale;     /* [slots, HV, V] (PER_V) or [slots, HV] (PER_HEAD) */
  int64_t stride_state_slot;
  int64_t stride_resid_slot;
  int64_t stride_sscale_slot;
  int64_t stride_rscale_slot;
  void* out;              /* [B, 1, HV, V] contiguous */
  int32_t out_dtype;
  const int32_t* ssm_state_indices; /* [B] */
  int64_t stride_indices;
  int32_t B, H, HV, K, V;
  int32_t num_slots;
  int32_t use_qk_l2norm;
  int32_t res_fmt;          /* CARRY_RES_INT8 | CARRY_RES_INT4 */
  int32_t resid_scale_mode; /* CARRY_SCALE_* */
  int32_t eps_mode;         /* CARRY_EPS_* */
  float qmax;               /* state grid, 127 for 8 bits */
  int32_t* status;          /* optional device word, may be NULL */
} CarryGdnPackedArgs;

int carry_gdn_packed_decode(const CarryGdnPackedArgs* args, void* stream);

/*
 * T consecutive tokens of every request in one call: the same step applied T
 * times to each request's slot, with the slot's tile held on chip in between,
 * so the state crosses HBM once per call instead of once per token.  Results
 * are those of T calls of carry_gdn_packed_decode, bit for bit.  No such entry
 * exists in the reference; it is the multi-token decode that vLLM reaches
 * through its speculative-decoding path (the sibling of the call
 * vllm_integration/quantized_packed_decode.py:242 mirrors).
 *
 * `step` describes token 0 exactly as for carry_gdn_packed_decode, with
 * mixed_qkv [B, T, width], a and b [B, T, HV] and out [B, T, HV, V] contiguous:
 * stride_*_tok are the strides between requests, stride_*_t those between the
 * tokens of one request (in elements).  Only the shapes the streaming kernel
 * takes are supported (K = V = 128, 16-byte aligned rows); anything else
 * returns CARRY_GDN_ERR_UNSUPPORTED and the caller loops over tokens.
 */
typedef struct CarryGdnPackedMultiArgs {
  CarryGdnPackedArgs step;
  int32_t T;
  int64_t stride_mixed_t;
  int64_t stride_a_t;
  int64_t stride_b_t;
} CarryGdnPackedMultiArgs;

int carry_gdn_packed_decode_multi(const CarryGdnPackedMultiArgs* args, void* stream);

/*
 * The slot pool of one layer -- the four tensors carry_gdn_packed_decode
 * updates -- for the calls that move a request's state in and out of it.  The
 * reference keeps the pool as four torch tensors and seeds it with eager ops
 * (init_quantized_state, vllm_integration/quantized_packed_decode.py:330-352);
 * it names what a serving engine additionally needs of it -- the residual has
 * to survive paging, preemption, prefix-cache reuse and speculative-decode
 * rollback -- as work not done (same file :50-54).  Within a slot the tensors
 * are contiguous [HV, V, K]; strides between slots are in elements.
 */
typedef struct CarryGdnPool {
  int8_t* state_codes;    /* [slots, HV, V, K] */
  float* state_scale;     /* [slots, HV, V] */
  int8_t* resid_codes;    /* [slots, HV, V, K] (INT8) or [slots, HV, V, K/2] (INT4) */
  float* resid_scale;     /* [slots, HV, V] (PER_V) or [slots, HV] (PER_HEAD) */
  int64_t stride_state_slot;
  int64_t stride_resid_slot;
  int64_t stride_sscale_slot;
  int64_t stride_rscale_slot;
  int32_t num_slots, HV, V, K;
  int32_t res_fmt;          /* CARRY_RES_INT8 | CARRY_RES_INT4 */
  int32_t resid_scale_mode; /* CARRY_SCALE_* */
} CarryGdnPool;

/*
 * Prefill hand-off: quantise the floating-point state h[n] ([HV, V, K], K
 * contiguous -- the final state a prefill kernel returns) of request n into
 * slot slots[n].  State codes and scales are those of init_quantized_state
 * (quantized_packed_decode.py:346-350): scale = max(amax_K|h|, 1e-12) / qmax,
 * codes = round_half_even(h / scale).  keep_error == 0 zeroes the slot's
 * residual, as the reference does; keep_error != 0 stores the quantisation
 * error h - codes * scale as the residual instead (encoded like a decode step
 * encodes it), so the first decode step already feeds it back.  A slot id <= 0
 * is padding and skipped.  Two requests must not name the same slot.
 */
typedef struct CarryGdnPoolStoreArgs {
  CarryGdnPool pool;
  const void* h;          /* [B, HV, V, K] */
  int64_t stride_h_req;   /* elements between requests */
  int32_t h_dtype;        /* CARRY_F32 | CARRY_BF16 | CARRY_F16 */
  const int32_t* slots;   /* [B] */
  int64_t stride_slots;
  int32_t B;
  int32_t keep_error;
  float qmax;             /* state grid, 127 for 8 bits */
  int32_t* status;        /* optional device word, may be NULL */
} CarryGdnPoolStoreArgs;

int carry_gdn_pool_store(const CarryGdnPoolStoreArgs* args, void* stream);

/*
 * The reverse: h[n] = codes * scale (+ resid_codes * resid_scale when
 * with_residual != 0, which is the state the next decode step re-quantises)
 * for slot slots[n], each product rounded to fp32 before the sum.  Hands a
 * request back to a kernel that wants a floating-point state (a further prefill
 * chunk, a swap-out in an engine's own format).  A slot id <= 0 writes zeros.
 */
typedef struct CarryGdnPoolLoadArgs {
  CarryGdnPool pool;      /* read only */
  void* h;                /* [B, HV, V, K] */
  int64_t stride_h_req;
  int32_t h_dtype;
  const int32_t* slots;   /* [B] */
  int64_t stride_slots;
  int32_t B;
  int32_t with_residual;
  int32_t* status;
} CarryGdnPoolLoadArgs;

int carry_gdn_pool_load(const CarryGdnPoolLoadArgs* args, void* stream);

/*
 * Copy whole slots, residual included, bit for bit: slot src_slots[n] of `src`
 * to slot dst_slots[n] of `dst` (the same pool, or a second pool of the same
 * shape and formats: a spill pool for preempted requests, a checkpoint before
 * speculative tokens, a prefix-cache entry).  Pairs with either id <= 0 are
 * skipped.  No destination slot may be the source or destination of another
 * pair of the same call.
 */
typedef struct CarryGdnPoolCopyArgs {
  CarryGdnPool src;       /* read only */
  CarryGdnPool dst;
  const int32_t* src_slots; /* [B] */
  int64_t stride_src_slots;
  const int32_t* dst_slots; /* [B] */
  int64_t stride_dst_slots;
  int32_t B;
  int32_t* status;
} CarryGdnPoolCopyArgs;

int carry_gdn_pool_copy(const CarryGdnPoolCopyArgs* args, void* stream);

/*
 * The same for one slot of a whole stack of layers in one launch: slot src_slot
 * of src[l] to slot dst_slot of dst[l] for every layer l.  `src` and `dst` are
 * host arrays of `layers` pools of one shape and format; the slot ids are
 * given by value and have to lie in 1 .. num_slots - 1 of every pool
 * (CARRY_GDN_ERR_SHAPE otherwise).  What a cache manager does when it preempts,
 * resumes, forks, checkpoints or rolls back one request.
 */
typedef struct CarryGdnPoolCopyLayersArgs {
  const CarryGdnPool* src;
  const CarryGdnPool* dst;
  int32_t layers;
  int32_t src_slot, dst_slot;
} CarryGdnPoolCopyLayersArgs;

int carry_gdn_pool_copy_layers(const CarryGdnPoolCopyLayersArgs* args, void* stream);

/*
 * The key/value cache of one full-attention layer, in 8 bits: pages of `page`
 * tokens, e4m3 codes [pages, HKV, page, D] and one fp32 scale for every `block`
 * tokens of a head, [pages, HKV, page / block]; a value is code * scale.  The
 * scales that carry_gdn_kv_append writes are powers of two, 2^-100 to 2^119;
 * those of a cache that was filled elsewhere may be any numbers of that range,
 * or 0 for blocks whose codes are all 0.
 * Request b holds lengths[b] tokens, token j of it in page
 * block_table[b][j / page]; a page id <= 0 is padding, its tokens are not
 * there.  A page id >= num_pages and a length beyond max_pages * page are
 * flagged with CARRY_GDN_STATUS_BAD_RANGE and treated as padding and as that
 * bound.  Within a page the tensors are contiguous; strides between pages and
 * between the table's rows are in elements.  D is 64 or 128, page and block are
 * multiples of 16, block divides page and is at most 128; code pages start on
 * 16-byte boundaries.  B and HKV are at most 65535, their product and a page of
 * all heads below 2^31, a request's tokens 2^30.
 */
typedef struct CarryGdnKvCache {
  uint8_t* k_codes;
  float* k_scale;
  uint8_t* v_codes;
  float* v_scale;
  int64_t stride_k_page, stride_ks_page, stride_v_page, stride_vs_page;
  const int32_t* block_table; /* [B, max_pages] */
  int64_t stride_table;
  const int32_t* lengths;     /* [B], with the call's own tokens among them */
  int32_t num_pages, HKV, page, block, D, max_pages;
} CarryGdnKvCache;

/*
 * The new tokens of a call: N rows, those of request b being
 * query_start[b] .. query_start[b + 1] - 1 (at most max_query of them; more,
 * and rows outside 0 .. N - 1, are skipped and flagged), or, with query_start
 * NULL, max_query = N / B rows each.  Row i of n of a request stands at
 * position lengths[b] - n + i of its context.
 */
typedef struct CarryGdnKvRows {
  const int32_t* query_start; /* [B + 1], or NULL */
  int32_t B, N, max_query;
} CarryGdnKvRows;

/*
 * Append: the rows' keys and values become codes at their positions.  The scale
 * of a block is the smallest power of two s with amax / s <= 448, amax over the
 * block's tokens so far; where it grows, the codes of the block's earlier
 * tokens are rounded to it (exactly, down to e4m3's subnormals).  A larger scale
 * that earlier tokens have stays, a power of two or not.  A block whose first
 * token is among the new ones is started afresh.  A token whose key or
 * value has a number that is not finite gets a NaN key and takes no part in the
 * scale: the queries that see it become NaN, no others.  Rows at a negative
 * position or in a padding page are skipped.  No two requests may append to one
 * page.
 */
typedef struct CarryGdnKvAppendArgs {
  CarryGdnKvCache cache;
  CarryGdnKvRows rows;
  const void* k;          /* [N, HKV, D], D contiguous */
  const void* v;
  int64_t stride_k_tok, stride_k_head, stride_v_tok, stride_v_head;
  int32_t dtype;          /* CARRY_F32 | CARRY_BF16 | CARRY_F16 */
  int32_t* status;        /* optional device word, may be NULL */
} CarryGdnKvAppendArgs;

int carry_gdn_kv_append(const CarryGdnKvAppendArgs* args, void* stream);

/*
 * Attention of the rows' queries over the cache: out = sum_j softmax_j(scale *
 * q . k_j) v_j over the tokens j of the request up to the row's own position.
 * HQ is a multiple of HKV; query head h reads key/value head h / (HQ / HKV).  A
 * row that sees no token is zero.  Value codes have to be finite where they are
 * within a request's length.  `workspace` holds partial results and is at least
 * carry_gdn_kv_attention_workspace() bytes, 16-byte aligned; nothing is kept
 * in it between calls.
 */
typedef struct CarryGdnKvAttentionArgs {
  CarryGdnKvCache cache;  /* read only */
  CarryGdnKvRows rows;
  const void* q;          /* [N, HQ, D], D contiguous */
  int64_t stride_q_tok, stride_q_head;
  void* out;              /* [N, HQ, D], D contiguous */
  int64_t stride_out_tok, stride_out_head;
  void* workspace;
  int64_t workspace_bytes;
  float scale;
  int32_t HQ;
  int32_t dtype;          /* of q and out */
  int32_t* status;
} CarryGdnKvAttentionArgs;

int carry_gdn_kv_attention(const CarryGdnKvAttentionArgs* args, void* stream);

/* Bytes of workspace that a call with these arguments needs (0 for none), or a
 * negative CARRY_GDN_ERR_*.  Looks at sizes only: no pointer is read. */
int64_t carry_gdn_kv_attention_workspace(const CarryGdnKvAttentionArgs* args);

/*
 * The entry of a layer: h = x + residual (fp32), residual_out = h rounded to its
 * type, y = h * rsqrt(mean(h^2) + eps) * weight, and y in e4m3 codes with a
 * scale per row (group == 0: scale [N]) or per 128 columns (group == 128: scale
 * [N, ceil(W / 128)], contiguous): scale = max(amax|y|, 1e-12) / 448.  A row
 * of h with a number that is not finite, or whose product with its weight is
 * not in fp32, gets NaN codes and scales throughout.  Squares below fp32's
 * range count as 0: eps stands in for them.  residual may be NULL (h = x); residual_out
 * may be NULL, or alias residual or x.  W is at most 32768.
 */
typedef struct CarryGdnNormArgs {
  const void* x;          /* [N, W], W contiguous */
  const void* residual;   /* [N, W] */
  void* residual_out;     /* [N, W] */
  const void* weight;     /* [W] */
  uint8_t* codes;         /* [N, W] */
  float* scale;
  int64_t stride_x, stride_residual, stride_residual_out, stride_codes;
  float eps;
  int32_t N, W, group;
  int32_t x_dtype, residual_dtype, weight_dtype; /* residual_dtype: of residual and residual_out */
} CarryGdnNormArgs;

int carry_gdn_add_rms_norm_quant(const CarryGdnNormArgs* args, void* stream);

/*
 * The gated delta rule over whole sequences, from a floating-point state (or
 * none) to a floating-point state: what goes ahead of carry_gdn_packed_decode for
 * a prompt, between carry_gdn_pool_load and carry_gdn_pool_store for a further
 * chunk of one.  The recurrence, gates, head map and L2 norm are those of
 * carry_gdn_packed_decode with the state left unquantized:
 *   S <- alpha S;  u = beta (v - S k);  S <- S + u k^T;  o = S (scale q)
 * for every token of a request in turn, with q and k divided by
 * sqrt(sum of squares + 1e-6) where use_qk_l2norm is set.  The rows of request
 * b are query_start[b] .. query_start[b + 1] - 1 (at most max_query; more, and
 * rows outside 0 .. N - 1, are skipped and flagged with
 * CARRY_GDN_STATUS_BAD_RANGE), or, with query_start NULL, max_query = N / B
 * each.  query_start does not fall: no two requests share a row, and other rows are left alone.  Where it does fall,
 * CARRY_GDN_STATUS_BAD_RANGE is set, and what the call's rows and states get is not defined.  A request
 * without rows hands its state on.
 *
 * A key that is not finite, and a decay or a write strength that is NaN, leave the
 * state of the heads that read them not finite from their token on, a value its row of
 * the state, a number of initial_state its row; outputs ahead of it and other rows are what
 * they were.  In chunks such a row is NaN throughout, and states and values count as infinite beyond bf16's largest
 * number (3.39e38).  With use_qk_l2norm the squares
 * of a key's numbers, and of a query's, have to add up to less than fp32's largest number: where a
 * query's do not, its token's outputs are NaN, and where a key's do not, the state and the outputs from its chunk or token on.  Without it
 * the products of a key with the other keys, and with the queries, of its 64 tokens have to be in fp32's range, whatever their write strengths.
 * A token's decay below exp(-200) is 0.
 *
 * K and V are 64 or 128 (one width for both), B and HV at most 65535, N at most 2^30.
 * final_state may be initial_state; outputs share no memory with inputs other than that, nor with
 * one another (a stride of final_state or out below a request's or token's size is refused).
 * `workspace` is at least
 * carry_gdn_prefill_workspace() bytes, 16-byte aligned; nothing is kept in it
 * between calls, and two that may run at a time need one each.  It is at most some 1 GiB: what does not fit is worked off in
 * turns.  Where a wait runs out (CARRY_GDN_STATUS_TIMEOUT), the further outputs and the state of the
 * columns (32 or 64 of a head's V) that waited are left as they were.
 */
typedef struct CarryGdnPrefillArgs {
  const void* mixed_qkv;      /* [N, 2*H*K + HV*V] = q | k | v, as in carry_gdn_packed_decode */
  int64_t stride_mixed_tok;
  const void* a;              /* [N, HV] */
  int64_t stride_a_tok;
  const void* b;              /* [N, HV] */
  int64_t stride_b_tok;
  const void* A_log;          /* [HV] */
  const void* dt_bias;        /* [HV] */
  const float* initial_state; /* [B, HV, V, K], dense within a request, or NULL for zeros */
  int64_t stride_initial_req;
  float* final_state;         /* [B, HV, V, K] */
  int64_t stride_final_req;
  void* out;                  /* [N, HV, V], dense within a token */
  int64_t stride_out_tok;
  const int32_t* query_start; /* [B + 1], or NULL */
  void* workspace;
  int64_t workspace_bytes;
  int32_t* status;            /* optional device word, may be NULL */
  float scale;
  int32_t B, N, max_query, H, HV, K, V;
  int32_t qkv_dtype, ab_dtype, A_log_dtype, dt_bias_dtype, out_dtype;
  int32_t use_qk_l2norm;
} CarryGdnPrefillArgs;

int carry_gdn_prefill(const CarryGdnPrefillArgs* args, void* stream);

/* Bytes of workspace that a call with these arguments needs (0 for none), or a
 * negative CARRY_GDN_ERR_*.  Looks at sizes only: no pointer is read. */
int64_t carry_gdn_prefill_workspace(const CarryGdnPrefillArgs* args);

/*
 * RMS norm of every query and key head and the rotation by the token's
 * position: y = x * rsqrt(mean(x^2) + eps) * (weight + weight_offset), and of
 * y's first `rotary` numbers the pairs (y1, y2) -> (y1 cos - y2 sin, y2 cos +
 * y1 sin).  Pair i < rotary / 2 is (y[i], y[i + rotary / 2]), or (y[2 i],
 * y[2 i + 1]) where `interleaved` is set; its cos and sin are columns i and
 * rotary / 2 + i of row p of cos_sin, p the token's position on the pair's axis:
 * the first sections[0] pairs are axis 0's, the next sections[1] axis 1's, and so
 * on.  A token with a negative position is left alone (nothing of it is
 * written), and so is one with a position beyond the table, which is flagged
 * with CARRY_GDN_STATUS_BAD_RANGE.  A head with a number that is not finite
 * becomes NaN.  Squares below fp32's range count as 0: eps stands in for them.
 * q_out and k_out may be q and k.  D is even and at most 512, rotary even and at
 * most D, axes 1 to 4, HQ and HK at most 65535.  Heads that are written share no memory: along the
 * smaller of an output's two strides they have to lie within the larger one.
 */
typedef struct CarryGdnRotateArgs {
  const void* q;          /* [N, HQ, D], D contiguous */
  const void* k;          /* [N, HK, D] */
  void* q_out;
  void* k_out;
  int64_t stride_q_tok, stride_q_head, stride_k_tok, stride_k_head;
  int64_t stride_q_out_tok, stride_q_out_head, stride_k_out_tok, stride_k_out_head;
  const void* q_weight;   /* [D] */
  const void* k_weight;   /* [D] */
  const void* cos_sin;    /* [table_rows, rotary] = cos | sin */
  int64_t stride_table, table_rows;
  const void* positions;  /* [axes, N], int32 or int64, N contiguous */
  int64_t stride_positions;
  int32_t* status;        /* optional device word, may be NULL */
  float eps, weight_offset;
  int32_t N, HQ, HK, D, rotary, axes, sections[4];
  int32_t positions_64, interleaved;
  int32_t dtype, weight_dtype, table_dtype; /* dtype: of q, k, q_out and k_out */
} CarryGdnRotateArgs;

int carry_gdn_qk_norm_rope(const CarryGdnRotateArgs* args, void* stream);

/* Human-readable text for a CARRY_GDN_ERR_* code (static storage). */
const char* carry_gdn_strerror(int code);

/* CARRY_GDN_ABI_VERSION the library was built with. */
int carry_gdn_abi_version(void);

/*
 * Which kernel the last successful call on this host thread selected:
 * 0 = none yet, 1 = generic tile kernel, 2 = 128x128 streaming kernel (of either layout),
 * 3 = multi-token kernel, 4 = a pool store / load / copy kernel,
 * 5 = 128x128 streaming kernel, step without error feedback,
 * 6 = slot-indexed kernel for 64x64 heads, 7 = kernel of chained steps,
 * 8 = statequant-layout kernel for 64x64 heads, 9 = key/value append, 10 = attention over the
 * key/value cache, 11 = layer norm with 8-bit output, 12 = norm and rotation of queries and keys, 13 = gated
 * delta rule over sequences, token by token, 14 = the same in chunks.
 * Diagnostic only (tests use it to prove which path ran).
 */
int carry_gdn_last_kernel(void);

#ifdef __cplusplus
}
#endif
#endif /* CARRY_GDN_H_ */
