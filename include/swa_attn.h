/*
 * swa_attn.h -- C ABI of the B200 (sm_100a) causal sliding-window + sink-token + GQA
 * attention, forward and backward.
 *
 * This is the drop-in boundary for the reference project's autograd Function
 * (junhown3/FlashAttention-GPT-OSS-finetuning, flash_attention_gpt_oss.py):
 *
 *   swa_fwd            replaces FlashSWDAWithSink.forward's kernel launch
 *                      (flash_attention_gpt_oss.py:356-379: allocate o, M; launch
 *                      _flash_attention_forward_swa_kernel).
 *   swa_bwd            replaces FlashSWDAWithSink.backward's work
 *                      (flash_attention_gpt_oss.py:397-435: Delta in torch, launch
 *                      _flash_attention_backward_swa_kernel, cast dk/dv).
 *   swa_bwd_preprocess the Delta = rowsum(dO * O) line (flash_attention_gpt_oss.py:403).
 *   swa_bwd_dq         the dQ half of _flash_attention_backward_swa_kernel
 *                      (flash_attention_gpt_oss.py:316-321, 334-338).
 *   swa_bwd_dkdv       the dK/dV half of that kernel (flash_attention_gpt_oss.py:295-304,
 *                      323-332), made deterministic: no atomics.
 *
 * Conventions
 *   - Tensors are [B, H, L, D] with the last dimension contiguous; the strides of the first
 *     three dimensions are given in ELEMENTS (like the reference's x.stride(0..2)).
 *   - q, o, dout, dq: [B, Hq, L, D]; k, v, dk, dv: [B, Hkv, L, D]; one dtype for all of
 *     them (fp16 or bf16).  Query head h reads KV head h / (Hq / Hkv).
 *   - Key j is visible to query i iff j <= i and (i - j < window_size or j < sink_size).
 *   - lse: [B, Hq, swa_lse_row_stride(L)] fp32, contiguous (rows padded to a multiple of 64).
 *     It is private to this library: it holds the base-2 log-sum-exp of the scaled scores
 *     (log2(e) * ln-LSE), -inf for a row that sees no key, +inf in the padding rows.  (The
 *     reference saves the row maximum M instead.)
 *   - Every entry point is asynchronous on `stream` (a cudaStream_t, NULL = legacy default
 *     stream), allocates nothing, and returns a SwaStatus.  Work on the device never
 *     waits on another launch.
 */
#ifndef SWA_ATTN_H_
#define SWA_ATTN_H_

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define SWA_API __attribute__((visibility("default")))
#else
#define SWA_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef enum SwaStatus {
  SWA_OK = 0,
  SWA_ERR_INVALID_ARG = 1,   /* null pointer, negative size, inconsistent shapes        */
  SWA_ERR_UNSUPPORTED = 2,   /* head_dim / dtype / alignment this build does not cover  */
  SWA_ERR_LAUNCH = 3,        /* the CUDA launch itself failed (see swa_last_cuda_error) */
  SWA_ERR_DEVICE_TIMEOUT = 4,/* a bounded on-device wait gave up                        */
  SWA_ERR_WORKSPACE = 5,     /* workspace missing or smaller than swa_bwd_workspace_size */
  SWA_ERR_TOO_LARGE = 6,     /* problem needs more scratch than swa_bwd_no_alloc holds   */
  SWA_ERR_BAD_PAGE = 7       /* a page table entry or a length was out of range          */
} SwaStatus;

typedef enum SwaDtype { SWA_F16 = 0, SWA_BF16 = 1 } SwaDtype;

/* Problem description shared by all entry points. */
typedef struct SwaProblem {
  int32_t batch;        /* B   */
  int32_t n_q_heads;    /* Hq  */
  int32_t n_kv_heads;   /* Hkv (Hq % Hkv == 0) */
  int32_t seq_len;      /* L   */
  int32_t head_dim;     /* D: 16, 32, 64 or 128 in this build (reference allows D <= 128) */
  int32_t window_size;  /* W: counts the diagonal; W <= 0 leaves only the sinks visible   */
  int32_t sink_size;    /* S: first S key positions always visible (causally)            */
  int32_t dtype;        /* SwaDtype */
  float softmax_scale;  /* scale applied to QK^T (the reference defaults it to 1/sqrt(D)) */
} SwaProblem;

/* A [B, H, L, D] tensor: device pointer + element strides of dims 0..2 (dim 3 stride 1). */
typedef struct SwaTensor {
  void* ptr;
  int64_t stride_b, stride_h, stride_l;
} SwaTensor;

typedef struct SwaFwdArgs {
  SwaProblem p;
  SwaTensor q, k, v;  /* inputs  */
  SwaTensor o;        /* output, [B, Hq, L, D] */
  float* lse;         /* output, [B, Hq, swa_lse_row_stride(L)] contiguous fp32 */
} SwaFwdArgs;

typedef struct SwaBwdArgs {
  SwaProblem p;
  SwaTensor q, k, v, o, dout;  /* inputs (o and lse from swa_fwd) */
  const float* lse;
  SwaTensor dq, dk, dv;        /* outputs, dtype of the inputs */
  void* workspace;             /* device scratch, >= swa_bwd_workspace_size(&p) bytes, 256-B aligned */
  size_t workspace_bytes;
} SwaBwdArgs;

/* Forward: o = softmax(mask(scale * q k^T)) v and the row log-sum-exp.
 * Replaces flash_attention_gpt_oss.py:356-379. */
SWA_API int swa_fwd(const SwaFwdArgs* args, void* stream);

/* Scratch the backward needs (Delta rows and the sink-key partial sums), in bytes. */
SWA_API size_t swa_bwd_workspace_size(const SwaProblem* p);

/* Kernels swa_bwd_dkdv launches for this problem: the dK/dV kernel, plus the far sink-pair
 * kernel and the sink-row reduction when there are sink keys (0 for an invalid problem). */
SWA_API int swa_bwd_dkdv_launch_count(const SwaProblem* p);

/* Full backward: dQ (which also writes Delta) then dK/dV.  Replaces
 * flash_attention_gpt_oss.py:397-435.  Where the GQA-packed dQ kernel takes the problem and
 * the sink keys' contributions from rows far past their window are few (one sink tile of at
 * most 16 keys, head dim 64), the dQ kernel also accumulates those contributions, so the
 * sequence launches one kernel fewer than swa_bwd_dq followed by swa_bwd_dkdv. */
SWA_API int swa_bwd(const SwaBwdArgs* args, void* stream);

/* Kernels swa_bwd launches for this problem (0 for an invalid or empty problem). */
SWA_API int swa_bwd_launch_count(const SwaProblem* p);

/* Delta[b,h,i] = sum_d dout * o, written to the front of the workspace (stand-alone; swa_bwd
 * and swa_bwd_dq compute it inside the dQ pass).  Replaces flash_attention_gpt_oss.py:403. */
SWA_API int swa_bwd_preprocess(const SwaBwdArgs* args, void* stream);

/* dq; also computes Delta = rowsum(dout * o) and writes it to the workspace, where
 * swa_bwd_dkdv reads it.  Replaces flash_attention_gpt_oss.py:306-321, 334-338, 403. */
SWA_API int swa_bwd_dq(const SwaBwdArgs* args, void* stream);

/* dk, dv, deterministic (each KV tile owned by one CTA, GQA group looped inside); needs
 * Delta in the workspace (from swa_bwd_dq or swa_bwd_preprocess).  Replaces
 * flash_attention_gpt_oss.py:295-304, 323-332. */
SWA_API int swa_bwd_dkdv(const SwaBwdArgs* args, void* stream);

/* Learned per-head sink logits: an additional mode with no counterpart in the reference
 * (whose sinks are the first sink_size key tokens; both can be combined).  This is the form
 * GPT-OSS itself uses: query head h has a learned logit sink_logits[h] (fp32 device array of
 * n_q_heads values, natural-log units, NOT multiplied by softmax_scale) that joins every
 * row's softmax as one more column with no value vector:
 *   P = softmax([scale * q k^T (masked), sink_logits[h]]),  o = P[:, :L] v.
 * -inf means no sink for that head.  lse then includes the sink column, so a row that sees
 * no key has o = 0 and lse = log2(e) * sink_logits[h]. */
SWA_API int swa_fwd_sink_logits(const SwaFwdArgs* args, const float* sink_logits, void* stream);

/* Backward of swa_fwd_sink_logits (its o and lse): dq, dk, dv as swa_bwd, plus
 * dsink_logits[h] = d loss / d sink_logits[h] = -sum_{b,i} P_sink[b,h,i] * Delta[b,h,i]
 * (fp32 device array of n_q_heads values, overwritten; deterministic). */
SWA_API int swa_bwd_sink_logits(const SwaBwdArgs* args, const float* sink_logits,
                                float* dsink_logits, void* stream);

/* ------------------------------------------------------------------------------------
 * Variable-length (packed) batches: an additional mode with no counterpart in the reference
 * (which takes dense [B, H, L, D] only, flash_attention_gpt_oss.py:348).  `batch` sequences
 * of different lengths are packed along one token axis: q, o, dout, dq are [T, Hq, D] and
 * k, v, dk, dv are [T, Hkv, D] (T = cu_seqlens[batch]); sequence b holds tokens
 * [cu_seqlens[b], cu_seqlens[b+1]) and attends only inside itself, with the usual mask in
 * its own positions (key j visible to query i iff j <= i and (i - j < W or j < S), i and j
 * counted from the sequence's first token).  cu_seqlens is a HOST array of batch + 1
 * non-decreasing int32 offsets starting at 0.  SwaProblem.seq_len is ignored.
 * lse: n_q_heads * swa_varlen_lse_floats(...) fp32; sequence b owns a [Hq, round_up(L_b, 64)]
 * block after those of sequences 0..b-1.  Every sequence runs the dense kernels as a
 * one-sequence problem; the sequences are spread over a pool of 4 library-owned streams per
 * device (created on first use, kept until exit) that fork from and join back into `stream`
 * with events, so they overlap on the GPU while the call stays ordered on `stream`.
 * ------------------------------------------------------------------------------------ */

/* A packed [T, H, D] tensor: device pointer + element strides of the token and head dims. */
typedef struct SwaPackedTensor {
  void* ptr;
  int64_t stride_t, stride_h;
} SwaPackedTensor;

typedef struct SwaVarlenFwdArgs {
  SwaProblem p;                /* batch = number of sequences; seq_len ignored            */
  const int32_t* cu_seqlens;   /* host, batch + 1 entries                                 */
  SwaPackedTensor q, k, v;     /* inputs                                                  */
  SwaPackedTensor o;           /* output [T, Hq, D]                                       */
  float* lse;                  /* output, swa_varlen_lse_floats(&p, cu_seqlens) floats    */
  const float* sink_logits;    /* optional [Hq] learned sink logits (see swa_fwd_sink_logits) */
} SwaVarlenFwdArgs;

typedef struct SwaVarlenBwdArgs {
  SwaProblem p;
  const int32_t* cu_seqlens;   /* host, batch + 1 entries                                 */
  SwaPackedTensor q, k, v, o, dout;
  const float* lse;            /* from swa_varlen_fwd                                     */
  SwaPackedTensor dq, dk, dv;  /* outputs                                                 */
  const float* sink_logits;    /* optional, as given to the forward                       */
  float* dsink_logits;         /* [Hq] output when sink_logits is set (else ignored)      */
  void* workspace;             /* >= swa_varlen_bwd_workspace_size bytes, 256-B aligned   */
  size_t workspace_bytes;
} SwaVarlenBwdArgs;

/* Size of the varlen lse buffer in floats (0 for invalid arguments). */
SWA_API size_t swa_varlen_lse_floats(const SwaProblem* p, const int32_t* cu_seqlens);

/* Scratch swa_varlen_bwd needs: one 256-byte aligned swa_bwd_workspace_size region per
 * non-empty sequence (sequences overlap on the GPU, each with its own region). */
SWA_API size_t swa_varlen_bwd_workspace_size(const SwaProblem* p, const int32_t* cu_seqlens);

/* Forward over packed sequences (swa_fwd per sequence). */
SWA_API int swa_varlen_fwd(const SwaVarlenFwdArgs* args, void* stream);

/* Backward over packed sequences (swa_bwd per sequence, deterministic; with sink_logits,
 * dsink_logits sums the sequences' contributions in sequence order). */
SWA_API int swa_varlen_bwd(const SwaVarlenBwdArgs* args, void* stream);

/* ------------------------------------------------------------------------------------
 * Rotary positions (an additional operator with no counterpart in the reference, which takes
 * q and k as they are).  Frequency i of n_freq turns one pair of a head's values by the angle
 * theta_i = position[axis[i]] * inv_freq[i]:
 *   (x, y) -> scale * (x cos theta_i - y sin theta_i, y cos theta_i + x sin theta_i),
 * where the pair is (i, n_freq + i), or (2 i, 2 i + 1) with `interleaved`; values from
 * 2 n_freq on are copied.  A token has one position per axis (time, height, width for images
 * and video; one axis for text).  With `inverse` the angle is negated: the gradient of the
 * inputs from the gradient of the outputs.  Angles are formed in 64 bits, products and sums in
 * 32, one rounding to the tensors' type at the end.
 * ------------------------------------------------------------------------------------ */
#define SWA_ROTARY_MAX_FREQS 64

typedef struct SwaRotary {
  const float* inv_freq;       /* device, n_freq values                                   */
  const void* positions;       /* device, int32 or int64: positions[axis, b, l]           */
  int64_t pos_stride_axis, pos_stride_b, pos_stride_l; /* in elements; 0 broadcasts       */
  int32_t pos_is_64;           /* 1: positions are int64                                  */
  int32_t n_axes;              /* >= 1                                                    */
  int32_t n_freq;              /* 0 .. 64, 2 n_freq <= head_dim                           */
  int32_t interleaved;
  float scale;
  uint8_t axis[SWA_ROTARY_MAX_FREQS]; /* axis of each frequency, < n_axes                 */
} SwaRotary;

typedef struct SwaRotaryArgs {
  int32_t batch, n_q_heads, n_kv_heads, seq_len, head_dim; /* head_dim even, <= 128       */
  int32_t dtype;               /* SwaDtype                                                */
  int32_t inverse;
  SwaRotary r;
  SwaTensor q, k;              /* [B, Hq, L, D], [B, Hkv, L, D]; k.ptr NULL: q alone       */
  SwaTensor q_out, k_out;      /* may be the inputs themselves (same pointer and strides)  */
} SwaRotaryArgs;

/* Rotate q and k.  Any strides >= 0 (rows need not be 16-byte aligned; aligned ones are read
 * and written 16 bytes at a time).  Outputs must not overlap inputs unless they are them. */
SWA_API int swa_rotary(const SwaRotaryArgs* args, void* stream);

/* ------------------------------------------------------------------------------------
 * Paged key-value cache (additional operators with no counterpart in the reference, which
 * trains only).  Keys and values of a sequence lie in pages of page_size rows from one pool;
 * slot j of sequence b is row j % page_size of page page_table[b, j / page_size].  seq_lens[b]
 * slots are in use.  All integer arrays are DEVICE arrays: no call reads them on the host.
 * Table entries behind a sequence's last page are not read.  An entry outside [0, n_pages) or
 * a length above max_pages * page_size that a call meets is never followed: rows of such pages
 * are neither read nor written, the sequence's attention output is NaN, an eviction leaves the
 * sequence as it is, all heads of it alike, and a following swa_check_device returns
 * SWA_ERR_BAD_PAGE.  (An append writes those of its tokens whose own page is in range; an
 * eviction meets the entries of all pages in use of the sequences that it would cut.)  A
 * negative length counts as 0.
 * ------------------------------------------------------------------------------------ */
typedef struct SwaPagedKV {
  void* k;                     /* [n_pages, n_kv_heads, page_size, D], D contiguous        */
  void* v;
  int64_t k_stride_page, k_stride_head, k_stride_row; /* elements, multiples of 8          */
  int64_t v_stride_page, v_stride_head, v_stride_row;
  const int32_t* page_table;   /* [batch, max_pages], row stride table_stride              */
  int64_t table_stride;
  int32_t* seq_lens;           /* [batch]; written by swa_paged_evict alone: caches that it
                                  cuts do not share it                                     */
  const int32_t* seen;         /* [batch] tokens seen so far; NULL: seq_lens, which holds
                                  until the first eviction                                 */
  float* weights;              /* [batch, n_kv_heads, max_pages * page_size], or NULL      */
  int32_t* positions;          /* same shape: the token number of each slot, or NULL       */
  int64_t w_stride_b, w_stride_h, p_stride_b, p_stride_h; /* elements                      */
  int32_t n_pages, page_size, max_pages; /* page_size: a multiple of 16                    */
  int32_t batch, n_kv_heads, head_dim, dtype; /* head_dim 16, 32, 64 or 128               */
} SwaPagedKV;

typedef struct SwaPagedAppendArgs {
  SwaPagedKV cache;            /* seq_lens (and seen) already count the new tokens         */
  const int32_t* cu_new;       /* device, batch + 1 offsets of the packed new tokens, or
                                  NULL: n_tokens / batch tokens for every sequence         */
  int32_t n_tokens;
  int32_t n_q_heads;           /* 0: no q                                                  */
  SwaPackedTensor k, v;        /* new tokens, [n_tokens, n_kv_heads, D]                    */
  SwaPackedTensor q, q_out;    /* [n_tokens, n_q_heads, D]: rotated beside k               */
  int32_t use_rotary;          /* 0: k is written as it is (and q must be absent)          */
  SwaRotary r;                 /* positions[axis, 0, token]                                */
} SwaPagedAppendArgs;

/* Write new tokens into the cache, rotating k (and q) on the way.  Token i of sequence b goes
 * to slot seq_lens[b] - new_b + i; its weight becomes 0 and its position the token number
 * seen[b] - new_b + i (where those arrays are given).  A token before the first of cu_new's offsets
 * or behind the last is no sequence's: it is written to no page and reported like a bad one. */
SWA_API int swa_paged_append(const SwaPagedAppendArgs* args, void* stream);

typedef struct SwaPagedDecodeArgs {
  SwaPagedKV cache;
  int32_t n_q_heads;           /* Hq, a multiple of n_kv_heads                             */
  int32_t window_size, sink_size; /* over slots, the newest token at slot seq_lens[b] - 1  */
  float softmax_scale;
  SwaPackedTensor q, o;        /* [batch, n_q_heads, D]; stride_t is the batch stride      */
  float* lse;                  /* [batch, n_q_heads] contiguous fp32, or NULL              */
  const float* sink_logits;    /* [n_q_heads] fp32 or NULL (see swa_fwd_sink_logits)       */
  float* weights_out;          /* NULL, or like cache.weights (may be it): see below       */
  int64_t wo_stride_b, wo_stride_h;
  float decay;
  void* workspace;             /* >= swa_paged_decode_workspace_size bytes, 256-B aligned  */
  size_t workspace_bytes;
} SwaPagedDecodeArgs;

/* Attention of one new token per sequence over its cache: slot j < n = seq_lens[b] is visible
 * iff n - 1 - j < window_size or j < sink_size.  lse as in swa_fwd.  With weights_out:
 *   weights_out[b, h, j] = decay * cache.weights[b, h, j] + sum over the query heads of KV
 * head h of their softmax weight on slot j (0 where it is not visible), for j < n.  Rows of a
 * sequence with a page or a length out of range are left as they are. */
SWA_API int swa_paged_decode(const SwaPagedDecodeArgs* args, void* stream);

/* Scratch that swa_paged_decode needs, by the sizes, the window and the sinks (of the pointers
 * it matters whether lse and weights_out are NULL); may be 0. */
SWA_API size_t swa_paged_decode_workspace_size(const SwaPagedDecodeArgs* args);

typedef struct SwaPagedEvictArgs {
  SwaPagedKV cache;            /* weights, positions and seen given, seen not seq_lens     */
  int32_t keep;                /* slots left to a sequence that is cut                     */
  int32_t trigger;             /* sequences with more slots than max(trigger, keep) are cut */
  int32_t sink_size;           /* tokens numbered below it are held ...                    */
  int32_t recent;              /* ... and those from seen[b] - recent on                   */
  void* workspace;             /* >= swa_paged_evict_workspace_size bytes, 256-B aligned   */
  size_t workspace_bytes;
} SwaPagedEvictArgs;

/* Cut every sequence longer than max(trigger, keep) down to keep slots, each KV head by its own
 * weights: held tokens stay first, then those of the largest weights (ties: the lowest slot;
 * NaN counts as -inf).  A kept slot below `keep` stays where it is; the i-th slot that comes
 * free below `keep` takes key, value, weight and position of the i-th kept slot from `keep` on,
 * and seq_lens[b] becomes keep.  Pages of a sequence that is cut must not belong to another
 * sequence too. */
SWA_API int swa_paged_evict(const SwaPagedEvictArgs* args, void* stream);
SWA_API size_t swa_paged_evict_workspace_size(const SwaPagedEvictArgs* args);

/* Backward that allocates nothing and takes no workspace.  No counterpart in the reference.
 *
 * For callers that cannot call cudaMalloc: a host that hands this library only its tensors
 * (an FFI/ctypes binding with no device allocator of its own, an engine that owns all device
 * memory through a fixed pool and forbids side allocations).  Same inputs, outputs and
 * results as swa_bwd; args->workspace and args->workspace_bytes are ignored.  Its scratch is
 * a static device array of SWA_NO_ALLOC_SCRATCH_BYTES (16 MiB) that every GPU which loads
 * this library keeps until the process exits; problems whose swa_bwd_workspace_size exceeds
 * it get SWA_ERR_TOO_LARGE.  The first call on each device looks up the array's device
 * address (cudaGetSymbolAddress) with that device current, so make that first call before
 * any stream capture.  All calls share the one array and each call writes every scratch byte
 * it reads, so nothing carries over between calls, but calls that overlap on the GPU (other
 * streams, other host threads, same device) race on it: serialise them. */
#define SWA_NO_ALLOC_SCRATCH_BYTES ((size_t)16 << 20)
SWA_API int swa_bwd_no_alloc(const SwaBwdArgs* args, void* stream);

/* (Every entry point: the library caches per device ordinal the addresses of its device-side
 * flag and scratch arrays for the life of the process, so it must not outlive a reset of the
 * device or of its primary context.)
 *
 * Synchronise `stream`, then report (and clear) the current device's on-device error flag:
 * SWA_ERR_DEVICE_TIMEOUT if a bounded wait inside a kernel gave up since the last check
 * (that launch's outputs are then undefined), SWA_ERR_BAD_PAGE if a paged call, on whichever cache
 * or stream of the device, met a page or a length out of range (a timeout is reported first, the
 * page by the next call), SWA_OK otherwise. */
SWA_API int swa_check_device(void* stream);

/* Enqueue on `stream` a copy of the current device's on-device error flag into
 * `*host_flag` (host memory, preferably pinned so the copy stays asynchronous) and return
 * without waiting.  Once the stream has passed that point, *host_flag != 0 means that a
 * bounded wait of some earlier launch gave up (its outputs are undefined, and later launches
 * skip their work until swa_check_device clears the flag).  Lets a host poll for timeouts
 * without synchronising every call.  No counterpart in the reference. */
SWA_API int swa_device_status_async(int* host_flag, void* stream);

/* Failure-path self-test: launches a kernel whose bounded on-device wait (on a barrier that
 * nothing arrives at) gives up after `limit_us` microseconds (1 .. 1e6) and records the
 * error; a following swa_check_device returns SWA_ERR_DEVICE_TIMEOUT.  No counterpart in the
 * reference (its kernels have no bounded waits). */
SWA_API int swa_selftest_wait_timeout(int limit_us, void* stream);

/* Human-readable name of a SwaStatus. */
SWA_API const char* swa_status_string(int status);

/* Text of the last CUDA error seen by a launch on this host thread ("" if none). */
SWA_API const char* swa_last_cuda_error(void);

/* Row stride (elements) of the lse buffer for sequence length L: L rounded up to 64. */
SWA_API int swa_lse_row_stride(int seq_len);

/* Version of this library (major*10000 + minor*100 + patch). */
SWA_API int swa_version(void);

#ifdef __cplusplus
}
#endif

#endif /* SWA_ATTN_H_ */
