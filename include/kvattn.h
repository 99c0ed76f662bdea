/* kvattn.h -- C ABI of the MI355X (gfx950) decode-phase KV-cache attention library.
 *
 * Drop-in for the attention call inside a GPT-2 decode step: the same q / K-cache /
 * V-cache / out pointer layouts as the reference engine, the same [NH, maxT, hs] cache
 * slot per (batch, head), a device-resident current length (so captured graphs stay
 * valid while the length grows), and the FP32 / BF16 / INT8 / FP8-E4M3 KV switch, here a
 * run-time argument instead of a compile-time macro.
 *
 * Layouts (reference names; element type below):
 *   qkv       [B][3][NH][hs]             Q, K, V of the current token
 *   kv_cache  [2][B][NH][maxT][hs]       K block then V block; K(b,h,j) at
 *                                        ((b*NH+h)*maxT + j)*hs, V adds B*NH*maxT*hs
 *   kv_scale  [2][B][NH][maxT] float     per-row scales, 8-bit and 4-bit caches only
 *   out       [B][NH][hs]
 *   part_out  [B][NH][S][hs] float, part_max / part_lse [B][NH][S] float
 * Element types: kv_dtype F32 -> qkv, kv_cache, out are float.  BF16 -> bfloat16.
 * INT8 / FP8_E4M3 -> kv_cache holds one byte per element, qkv and out are bfloat16.
 * INT4 / FP4_E2M1 -> kv_cache holds half a byte per element, qkv and out are bfloat16.
 *
 * Lengths: the number of attended positions of sequence b is cur_len + 1 where cur_len
 * is read ON THE DEVICE when the kernels run: from d_cur_len[0] for every sequence, or
 * from d_cur_len[b] when lens_per_seq != 0 (ragged batches).  d_cur_len == NULL means
 * the library's own device-resident length, see kvattn_cur_len_symbol().  Device lengths
 * are clamped into [0, maxT-1]; the host never reads them.
 *
 * Every entry point only enqueues work on `stream` (a hipStream_t; NULL = the null
 * stream), returns a kvattn_status and never exits the process.  All except the
 * cooperative strategy are legal inside hipStreamBeginCapture / hipStreamEndCapture.
 * Only hs == 64 is supported (one 64-lane wavefront spans one head row).
 */
#ifndef KVATTN_H
#define KVATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum kvattn_status {
    KVATTN_OK = 0,
    KVATTN_ERR_NULL_POINTER = 1,    /* a required pointer is NULL */
    KVATTN_ERR_MISALIGNED = 2,      /* qkv / kv_cache / out / workspace not 16-byte aligned */
    KVATTN_ERR_HEAD_DIM = 3,        /* hs != 64 */
    KVATTN_ERR_SHAPE = 4,           /* B, NH or maxT < 1, or a size that overflows */
    KVATTN_ERR_DTYPE = 5,           /* unknown kv_dtype, or kv_scale missing for 8-bit */
    KVATTN_ERR_STRATEGY = 6,        /* unknown strategy */
    KVATTN_ERR_WORKSPACE = 7,       /* workspace missing or smaller than required */
    KVATTN_ERR_SPLIT = 8,           /* S or seg_rows out of range */
    KVATTN_ERR_COOP_TOO_LARGE = 9,  /* cooperative grid exceeds co-resident capacity */
    KVATTN_ERR_LDS = 10,            /* fused_single scores for maxT do not fit in LDS */
    KVATTN_ERR_CAPTURE = 11,        /* cooperative launch requested inside stream capture */
    KVATTN_ERR_LENGTH = 12,         /* host length hint outside [0, maxT-1] */
    KVATTN_ERR_HIP = 13,            /* a HIP runtime call failed; see kvattn_last_hip_error */
    KVATTN_ERR_GRID_TOO_LARGE = 14, /* explicit SPLIT_DESIGNATED grid exceeds what the GPU holds
                                       at once (its mergers wait for their producers) */
    KVATTN_ERR_MERGE_TIMEOUT = 15   /* kvattn_workspace_status: a designated merger stopped
                                       waiting for its producers (and computed their segments
                                       itself), or a cooperative merger stopped waiting at the
                                       grid barrier (and wrote NaN) */
} kvattn_status;

typedef enum kvattn_dtype {
    KVATTN_KV_F32 = 0,       /* reference ENABLE_FP32 build (Makefile:78-79) */
    KVATTN_KV_BF16 = 1,      /* reference default BF16 build (Makefile:88-89) */
    KVATTN_KV_INT8 = 2,      /* reference USE_KV_W8 + USE_INT8 (Makefile:80-82,100-106) */
    KVATTN_KV_FP8_E4M3 = 3,  /* reference USE_KV_W8 + USE_FP8 (Makefile:83-85,100-106) */
    /* 4-bit caches: 32 bytes a row, channel 2i in the low half of byte i and 2i+1 in the high
     * half, one float scale a row (1/7 and 1/6 rounded to float); qkv and out are bf16.  No
     * reference counterpart (its cache types end at 8 bits).  Taken by kvattn_cache_write, kvattn_append, kvattn_decode,
     * kvattn_append_decode (two launches), kvattn_plan and the kvattn_paged_* calls; the others
     * return KVATTN_ERR_DTYPE.  Attention over them has one strategy, KVATTN_SPLIT_LASTBLOCK
     * (KVATTN_AUTO takes it), takes S > 0 and S < 0 (a multiple of 64) on paged caches too, needs
     * no workspace where kvattn_plan reports one segment and the batch has one length, and takes
     * at most 65535 sequences. */
    KVATTN_KV_INT4 = 4,      /* scale = amax * (1/7); the half byte holds round(x / scale) + 8 */
    KVATTN_KV_FP4_E2M1 = 5   /* scale = amax * (1/6); sign and one of 0 .5 1 1.5 2 3 4 6,
                                to nearest, ties to the even code */
} kvattn_dtype;

typedef enum kvattn_strategy {
    KVATTN_AUTO = 0,                /* fused_single for short contexts and for many heads of
                                       up to 1024 positions (contiguous F32, BF16 and FP8
                                       caches), else a split plan chosen from len_hint, the
                                       shape and the cache type:
                                       the designated merger while its grid is small, one
                                       segment per (b,h) for many short heads, split +
                                       merge kernels once the call is bandwidth bound */
    KVATTN_FUSED_SINGLE = 1,        /* one workgroup per (b,h), scores staged in LDS */
    KVATTN_SPLIT_MERGE = 2,         /* flash-decoding: split kernel + merge kernel */
    KVATTN_SINGLE_LAUNCH_COOP = 3,  /* split + grid barrier + merge, cooperative launch */
    KVATTN_SINGLE_LAUNCH_GRAPH = 4, /* split + merge pair replayed as one hipGraph launch */
    KVATTN_SPLIT_LASTBLOCK = 5,     /* split kernel whose last finishing segment of each
                                       (b,h) merges: one ordinary launch, capturable */
    KVATTN_SPLIT_DESIGNATED = 6     /* split kernel in which segment 0 of each (b,h) merges:
                                       the other segments publish tagged partials and finish,
                                       segment 0 polls for them; one ordinary launch,
                                       capturable; at most 64 segments per (b,h).  AUTO's
                                       choice for latency-bound calls (with a length hint:
                                       grids of up to 768 workgroups, 1024 for up to 64
                                       heads with long segments, and 64 MiB of cache). */
} kvattn_strategy;

/* Human-readable text of a status code. */
const char* kvattn_strerror(int status);

/* The hipError_t of the most recent failing HIP call on this thread (0 if none). */
int kvattn_last_hip_error(void);

/* Device address of the library's device-resident length for the current device.
 * Replaces cudaGetSymbolAddress(&d_cur_len_ptr, g_cur_len)
 * (inference_gpt2_opt.cu:252-254; g_cur_len at Inference_gpt2/attention_kvcache.cuh:35-40). */
int kvattn_cur_len_symbol(int** d_cur_len);

/* Blocking write of the library's device-resident length.
 * Replaces cudaMemcpyToSymbol(g_cur_len, &cur_len, sizeof(int))
 * (inference_gpt2_opt.cu:409,548). */
int kvattn_set_cur_len(int cur_len);

/* Enqueue the write of cur_len into *d_cur_len (NULL: the library's own device length) on
 * `stream`, without a host synchronisation; capturable.  Replaces the per-token
 * cudaMemcpyToSymbol(g_cur_len, ...) before each graph replay (inference_gpt2_opt.cu:548),
 * which blocks the host until the copy is done. */
int kvattn_set_cur_len_async(int* d_cur_len, int cur_len, void* stream);

/* Append the current token's K and V (from qkv) into column cur_len of every (b,h) slot.
 * F32/BF16 copy the elements; INT8/FP8 quantise each 64-element row with
 * scale = amax/127 (INT8) or amax/448 (FP8), store the codes and the FP32 scale.
 * Replaces kv_cache_write_kernel (Inference_gpt2/attention_kvcache.cuh:46-64) and
 * kv_cache_write_kernel_w8 (Inference_gpt2/attention_kvcache_w8.cuh:115-155), launched at
 * inference_gpt2_opt.cu:302-303 and :329.  kv_scale must be NULL for F32/BF16. */
int kvattn_cache_write(void* kv_cache, float* kv_scale, const void* qkv,
                       int B, int NH, int hs, int maxT,
                       const int* d_cur_len, int lens_per_seq,
                       int kv_dtype, void* stream);

/* kvattn_cache_write with one length for the whole batch (lens_per_seq = 0): the append
 * with exactly the arguments of the reference's launch (kv_cache_write_kernel[_w8] at
 * inference_gpt2_opt.cu:302-303, 329), plus the dtype and the stream. */
int kvattn_append(void* kv_cache, float* kv_scale, const void* qkv,
                  int B, int NH, int hs, int maxT, const int* d_cur_len,
                  int kv_dtype, void* stream);

/* Short-context path: one workgroup per (b,h), scores staged in LDS.
 * Replaces attention_forward_kv_small (Inference_gpt2/attention_kvcache.cuh:453-459) and
 * attention_forward_kv_small_w8 (Inference_gpt2/attention_kvcache_w8.cuh:529-536). */
int kvattn_forward_small(void* out, const void* qkv, const void* kv_cache,
                         const float* kv_scale, int B, int NH, int hs, int maxT,
                         const int* d_cur_len, int lens_per_seq,
                         int kv_dtype, void* stream);

/* Long-context path with caller-owned partials of S segments per (b,h).  As in the
 * reference, B == 1 takes a single launch and B > 1 (or a capture) the split + merge pair
 * over the caller's partials.  The single launch is the designated merger (SPLIT_DESIGNATED
 * over the reference partition), not a cooperative launch: on this stack a cooperative
 * dispatch alone costs ~20 us of GPU time.  Its tagged partials live in the library's static
 * scratch array (the one kvattn_decode_static uses), so the call only enqueues: it allocates
 * nothing and never synchronises, as the reference's launches over caller-owned partials
 * (inference_gpt2_opt.cu:710-716).  S > 64, a grid the GPU cannot hold at once, or more than
 * about 9,200 slots (NH * S) take the split + merge pair instead.  Like kvattn_decode_static, calls
 * that overlap in time on one GPU (unordered streams, concurrent host threads) share the
 * array and may find each other's words: a merger never takes another call's word (each
 * carries its call's identity), but may wait for its bound and compute its producers'
 * segments itself (kvattn_scratch_status counts those).  Ordered calls, on one stream or
 * across streams, do not interfere.
 * Replaces attention_forward_kv_large (Inference_gpt2/attention_kvcache.cuh:464-487) and
 * attention_forward_kv_large_w8 (Inference_gpt2/attention_kvcache_w8.cuh:541-566). */
int kvattn_forward_large(void* out, const void* qkv, const void* kv_cache,
                         const float* kv_scale, int B, int NH, int hs, int maxT,
                         const int* d_cur_len, int lens_per_seq,
                         float* part_out, float* part_lse, float* part_max, int S,
                         int kv_dtype, void* stream);

/* Split phase alone: segment s of (b,h) covers [s*chunk, min((s+1)*chunk, total)) with
 * chunk = ceil(total/S); an empty segment writes (max=-FLT_MAX, lse=0, out=0).
 * Replaces the attention_kv_split_kernel[_w8] launches used under graph capture
 * (inference_gpt2_opt.cu:310-312,338-339; kernels at attention_kvcache.cuh:185-288 and
 * attention_kvcache_w8.cuh:260-363). */
int kvattn_split(float* part_out, float* part_lse, float* part_max,
                 const void* qkv, const void* kv_cache, const float* kv_scale,
                 int B, int NH, int hs, int maxT,
                 const int* d_cur_len, int lens_per_seq, int S,
                 int kv_dtype, void* stream);

/* Merge phase alone: out = sum_s e_s*part_out_s / sum_s e_s*part_lse_s with
 * e_s = exp(part_max_s - max_s part_max_s).  `out` is float when kv_dtype is F32, else
 * bfloat16.  Replaces the attention_kv_merge_kernel[_w8] launches
 * (inference_gpt2_opt.cu:313-314,340-341; kernels at attention_kvcache.cuh:298-318 and
 * attention_kvcache_w8.cuh:374-396). */
int kvattn_merge(void* out, const float* part_out, const float* part_lse,
                 const float* part_max, int B, int NH, int hs, int S,
                 int kv_dtype, void* stream);

/* Bytes of workspace kvattn_decode needs for (B, NH, hs, maxT, S).  S > 0 sizes for
 * exactly S segments per (b,h); S == 0 sizes for every automatic choice. */
size_t kvattn_workspace_bytes(int B, int NH, int hs, int maxT, int S);

/* Zero the workspace (merge counters, status words).  Call once after allocating a
 * workspace and before the first kvattn_decode on it; the kernels leave the counters at
 * zero after every call, and the designated merger's partial words carry the dispatch that
 * wrote them, so they never need clearing.  Enqueues one fill kernel (no hipMemsetAsync),
 * so it may also be captured. */
int kvattn_workspace_init(void* workspace, size_t workspace_bytes, void* stream);

/* The workspace's sticky status: waits for `stream`, then reads the number of merges that
 * stopped waiting since the workspace was initialised or last cleared.  A designated merger
 * (SPLIT_DESIGNATED, AUTO's latency-bound choice) that stops waiting for its producers
 * computes their segments itself, so its output is still the attention (only slower); a
 * cooperative merger that stops waiting at the grid barrier writes NaN for its (b,h).
 * *merge_timeouts (may be NULL) receives that number; clear != 0 resets it.
 * Returns KVATTN_ERR_MERGE_TIMEOUT when it is non-zero, else KVATTN_OK.  Partials left by
 * such a call are never taken for a later call's (each partial word carries the dispatch that
 * wrote it and that dispatch's hardware queue), so the workspace stays usable without
 * re-initialising.
 * No reference counterpart: the reference has no in-kernel wait that can give up, and
 * reports errors by exiting (common.h:123-130). */
int kvattn_workspace_status(void* workspace, size_t workspace_bytes, int clear, void* stream,
                            int* merge_timeouts);

/* kvattn_workspace_status for the library's static scratch array on the current device (the
 * workspace of kvattn_decode_static and of kvattn_forward_large's single launch): waits for
 * `stream`, then *merge_timeouts (may be NULL) receives the number of merges that stopped
 * waiting there since the array was first used or last cleared; clear != 0 resets it.
 * Returns KVATTN_ERR_MERGE_TIMEOUT when it is non-zero, else KVATTN_OK.
 * No reference counterpart (the reference has no in-kernel wait that can give up). */
int kvattn_scratch_status(int clear, void* stream, int* merge_timeouts);

/* Enqueue on `stream` one dispatch that writes the identity the tagged partial words of a
 * dispatch on that stream carry: out[0] its dispatch id (counted per hardware queue),
 * out[1] the address of its hardware queue, out[2] its 32-bit tag (the dispatch id plus a hash
 * of the queue address, top bit set).  out: 3 device words, 8-byte aligned.
 * No reference counterpart: a testing hook showing that calls on different streams, whose
 * dispatch ids coincide, never share a tag. */
int kvattn_call_identity(unsigned long long* out, void* stream);

/* Moves every designated producer of an XCD-local grid (8 or more (b,h) rows) `rot` XCDs
 * (mod 8) away from its merger, for launches (and captures) from this call on, process-wide;
 * 0 (the default) keeps each head's segments on one XCD.  Returns the previous setting.
 * Each designated merger publishes the XCD it runs on and each producer publishes its partial
 * with plain stores (which stay in its XCD's L2) only when that XCD is its own, else
 * write-through, so a producer placed elsewhere, by this setting or by a dispatcher that hands
 * workgroups to XCDs otherwise than the layout expects, costs the merger no wait: the output
 * and the merge-timeout count stay as they are.
 * No reference counterpart: a testing hook for the layout the designated merger relies on. */
int kvattn_set_xcd_layout_offset(int rot);

/* Bound on the polls of a designated merger waiting for its producers' partials (and of a
 * cooperative merger at the grid barrier), for launches (and captures) from this call on,
 * process-wide: polls > 0 sets it, polls == 0 makes every merger of a multi-segment (b,h)
 * stop waiting at once (a fault-injection setting, for testing the fallback and the
 * reporting above), polls < 0 restores the default (2^16 polls, tens of milliseconds).
 * Returns the previous bound.  No reference counterpart (testing and fault-injection hook). */
int kvattn_set_merge_poll_limit(int polls);

/* The launch plan kvattn_decode would use for these arguments, without launching:
 * *strategy_out = the resolved kvattn_strategy (AUTO resolved), *segments_out = the segment
 * slots per (b,h) that the call's workspace must hold, so that
 * kvattn_workspace_bytes(B, NH, hs, maxT, *segments_out) bytes are enough for it,
 * *seg_rows_out = rows per segment (0 when there are no segments or the reference partition
 * ceil(total/S) is used, -1 when the kernels plan the rows from the device length).  The slots
 * are the launch's own (1 for FUSED_SINGLE), except for AUTO's plans for many heads of 257 to
 * 1024 positions (FUSED_SINGLE, or one segment per (b,h) on an INT8 cache): kvattn_decode asks
 * for the workspace of the segments that such a plan stands in for, and these are reported.
 * (FUSED_SINGLE passed by name asks for none.)
 * The plan is that of a call with one length for the batch
 * (lens_per_seq == 0).  A call with per-sequence lengths takes the same plan, except where
 * this one streams a BF16 or INT8 cache through the split + merge kernels (there AUTO keeps
 * its general plan: the last-block merge, or split + merge over segments of up to 512
 * rows), for many heads of 257 to 1024 positions, whose bounds on the heads differ, and for more
 * than 256 heads of a 4-bit cache, which per-sequence lengths of up to 6144 and more positions
 * (maxT, or the hint) split into more and shorter segments.  Its
 * workspace may then differ from the reported one too: S == 0 in kvattn_workspace_bytes is
 * enough for every call.  No reference counterpart: it exposes the AUTO choice, which the reference makes
 * inline in its caller (inference_gpt2_opt.cu:247,304,331: fused_single below a length
 * threshold, split + merge above it). */
int kvattn_plan(int B, int NH, int hs, int maxT, int len_hint, int S, int strategy, int kv_dtype,
                int* strategy_out, int* segments_out, int* seg_rows_out);

/* One decode-attention call with an explicit strategy, the unified entry the per-layer
 * attention block of forward_kv_graph_ready (inference_gpt2_opt.cu:298-347) maps onto.
 *   strategy   kvattn_strategy; AUTO picks from len_hint (the host's view of cur_len,
 *              used for the choice only; -1 = unknown, treated as maxT-1).
 *   len_hint   -1 when the call must serve any length, as a graph captured once and
 *              replayed token after token: with S == 0 the kernels then plan the
 *              segmentation from the device length (one segment up to 256 positions,
 *              about four beyond, segments of at most 512 rows up to 64 of them, longer
 *              rows past 32768 positions), where the reference captures a small and a large
 *              graph and picks one per token (inference_gpt2_opt.cu:420-449,556).  AUTO
 *              with more than 16 heads (B*NH), or a longer maxT, takes fixed rows sized
 *              for maxT instead while its designated grid stays small (kvattn_plan
 *              reports them); segments past a call's length exit at once.
 *   S          segments per (b,h) for the split strategies: S > 0 uses the reference
 *              partition chunk = ceil(total/S); S < 0 uses -S rows per segment; S == 0
 *              lets the library pick the rows per segment (from len_hint, or on the
 *              device) and the per-sequence count from each length.
 *   workspace  device memory of kvattn_workspace_bytes(B, NH, hs, maxT, S) bytes,
 *              initialised once with kvattn_workspace_init; may be NULL for strategy
 *              FUSED_SINGLE and for AUTO up to 256 positions (the hint's, else maxT).
 *              AUTO's plans for many heads beyond that ask for a workspace also where the
 *              launch uses less of it or none (kvattn_plan reports its slots).
 *              Calls sharing a workspace must be ordered: on one stream,
 *              or on several streams ordered by events (the designated merger's words
 *              carry the dispatch and its hardware queue, so a word another stream's call
 *              left is never taken for this call's).  Calls that overlap in time race.
 *   workspace_bytes  the buffer's actual size, the same for every call on the buffer.
 *              One buffer, sized for the largest plan, may serve calls of different
 *              plans (other B, NH or S): the last-block counters sit in a region whose
 *              size follows from workspace_bytes alone, the partials are laid out from
 *              the region's end and the designated merger's tagged words from the
 *              buffer's end, so no call finds its counters or tags where another left
 *              partials.
 */
int kvattn_decode(void* out, const void* qkv, const void* kv_cache, const float* kv_scale,
                  int B, int NH, int hs, int maxT,
                  const int* d_cur_len, int lens_per_seq, int len_hint,
                  void* workspace, size_t workspace_bytes,
                  int S, int strategy, int kv_dtype, void* stream);

/* kvattn_decode without a workspace argument: the partials, merge counters and tagged words
 * live in `scratch`, a static device array of 8 MiB that the library holds on each GPU it
 * runs on until the process ends, so the call allocates nothing (no hipMalloc, no hipFree;
 * a fill kernel clears the array's counters on its first call on a device).
 * No reference counterpart: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * Limits: B*NH <= 16384, and the plan's partials and tagged words (kvattn_workspace_bytes of
 * the slots that kvattn_plan reports, less its status words and counters) within
 * 8 MiB - 64.25 KiB, else KVATTN_ERR_WORKSPACE (AUTO falls back on segments that fit where it
 * can; its plans for many heads are refused with the segments that they stand in for);
 * strategies AUTO, FUSED_SINGLE, SPLIT_MERGE, SPLIT_LASTBLOCK, SPLIT_DESIGNATED (the
 * cooperative launch and the library's graph pair return KVATTN_ERR_STRATEGY: the runtime may
 * allocate for them).  Every call on one GPU shares that GPU's array (with
 * kvattn_forward_large's single launch), which keeps the last call's contents: calls that
 * overlap in time on one GPU (unordered streams, concurrent host threads) race; calls ordered
 * on one stream, or across streams by events, do not.  kvattn_scratch_status reads its merge
 * timeouts. */
int kvattn_decode_static(void* out, const void* qkv, const void* kv_cache, const float* kv_scale,
                         int B, int NH, int hs, int maxT,
                         const int* d_cur_len, int lens_per_seq, int len_hint,
                         int S, int strategy, int kv_dtype, void* stream);

/* kvattn_cache_write followed by kvattn_decode with the same arguments, in one launch
 * (two for SPLIT_MERGE): the current token's K and V rows are taken from qkv in registers
 * (8-bit: quantised exactly as kvattn_cache_write does), written into column cur_len, and
 * used in place of that cache column.  Cache contents and outputs equal those of the two
 * calls.  Replaces the append launch kv_cache_write_kernel[_w8] together with the attention
 * call after it (inference_gpt2_opt.cu:302-316, 329-345); the reference's ranked follow-up
 * removes the same launch by moving the append into the QKV GEMV epilogue instead. */
int kvattn_append_decode(void* out, const void* qkv, void* kv_cache, float* kv_scale,
                         int B, int NH, int hs, int maxT,
                         const int* d_cur_len, int lens_per_seq, int len_hint,
                         void* workspace, size_t workspace_bytes,
                         int S, int strategy, int kv_dtype, void* stream);

/* ---- Paged KV cache ------------------------------------------------------------------
 * No reference counterpart: the reference keeps one contiguous [2][B][NH][maxT][hs] cache
 * per layer and names paged KV management as its gap for multi-request serving
 * (README.md:62-63).  Here a layer's cache may instead be a pool of pages:
 *   pages        [num_pages][2][NH][page_rows][hs] elements (K block, then V block, of
 *                page_rows positions of one sequence for every head)
 *   page_scales  [num_pages][2][NH][page_rows] FP32 row scales (8-bit caches), else NULL
 *   block_table  [B][max_pages] int32: page id holding positions
 *                [i*page_rows, (i+1)*page_rows) of sequence b at block_table[b*max_pages+i]
 * page_rows is a multiple of 64; a sequence holds up to max_pages*page_rows positions
 * (the maxT of these calls).  Table entries outside [0, num_pages) are never dereferenced:
 * their positions are skipped (attention) or not written (append).  Row layout, element
 * types and 8-bit codes are those of the contiguous cache. */

/* kvattn_cache_write into a paged cache. */
int kvattn_paged_cache_write(void* pages, float* page_scales, const int* block_table,
                             int max_pages, int page_rows, int num_pages,
                             const void* qkv, int B, int NH, int hs,
                             const int* d_cur_len, int lens_per_seq, int kv_dtype, void* stream);

/* kvattn_decode (append == 0) or kvattn_append_decode (append != 0) on a paged cache.
 * Strategies: AUTO, SPLIT_MERGE, SPLIT_LASTBLOCK, SPLIT_DESIGNATED, SINGLE_LAUNCH_GRAPH (no
 * FUSED_SINGLE or cooperative launch: short contexts take a single segment of the split
 * kernel).  S == 0 plans the segments on the device, except where AUTO takes the designated
 * merger or one segment per (b,h) with fixed rows (128, 256 or 512: the choice kvattn_decode's
 * AUTO makes for a contiguous cache, hinted lengths of up to 256 positions excepted); S < 0
 * gives -S rows per segment, a multiple of 64 and at most 4096.  Workspace:
 * kvattn_workspace_bytes(B, NH, hs, max_pages*page_rows, S). */
int kvattn_paged_decode(void* out, const void* qkv, void* pages, float* page_scales,
                        const int* block_table, int max_pages, int page_rows, int num_pages,
                        int B, int NH, int hs,
                        const int* d_cur_len, int lens_per_seq, int len_hint,
                        void* workspace, size_t workspace_bytes,
                        int S, int strategy, int kv_dtype, int append, void* stream);

/* Attention of several new tokens of every sequence over a paged 4-bit cache (kv_dtype INT4 or
 * FP4_E2M1; other types: KVATTN_ERR_DTYPE), as verifying drafted tokens needs it: the new rows
 * are in the cache already (kvattn_paged_store), and each token attends the positions up to its
 * own.  The cache is read once for eight tokens of a sequence.
 *   token_start [B+1] device: sequence b's tokens are rows token_start[b] .. token_start[b+1]-1 of
 *               qkv [num_tokens][3][NH][hs] (only Q is read) and out [num_tokens][NH][hs]; their
 *               number may be 0
 *   lens        [B] device: positions of sequence b, its new tokens among them; token i of n
 *               attends the first lens[b] - n + i + 1 of them (none: its output is zero)
 *   max_new     the most tokens of one sequence (1, up to 4, up to 8 and more take different
 *               launches), or any larger number; a sequence with more has the first max_new or more
 *               of them computed
 * Rows of out behind token_start[B] are left as they were.  token_start must not decrease; it and
 * lens are clamped into [0, num_tokens] and [0, max_pages * page_rows].  B <= 65535; B * NH,
 * num_tokens * NH and, where max_new > 8, (B + num_tokens / 8) * NH below 2^24.  Workspace:
 * kvattn_workspace_bytes(num_tokens, NH, hs, max_pages * page_rows, S); S as in kvattn_decode with
 * a 4-bit cache.
 * No reference counterpart (the reference decodes one token at a time). */
int kvattn_paged_decode_tokens(void* out, const void* qkv, const void* pages, const float* page_scales,
                               const int* block_table, int max_pages, int page_rows, int num_pages,
                               const int* token_start, const int* lens, int B, int num_tokens, int max_new,
                               int NH, int hs, void* workspace, size_t workspace_bytes, int S, int kv_dtype,
                               void* stream);

/* ---- Trees of drafted tokens ------------------------------------------------------------
 * A sequence's new tokens may be the nodes of a tree: token 0 its root (the last token that was
 * accepted), every other one a draft behind its parent, an earlier token of the sequence.  Their rows
 * are in the cache already (kvattn_paged_store: token i's at position lens[b] - n + i), but a token
 * attends the positions before the tree and its own branch alone.  A chain of drafts is the tree whose
 * token i has the parent i - 1.  Up to 256 tokens a sequence.  No reference counterpart (the reference
 * decodes one token at a time).
 *   token_start [B+1] device: as in kvattn_paged_decode_tokens; a sequence may have no tokens
 *   parents [num_tokens] device: index of the parent among the sequence's tokens; what is negative or
 *           not below the token's own index counts as none (the token follows the cached prefix)
 *   masks [num_tokens][mask_words] device, 64-bit words, mask_words 1 to 4: bit i % 64 of word i / 64:
 *           the token attends token i of its sequence */

/* The masks of trees (a token's ancestors and itself), made once a step and read by every layer.
 *   positions [num_tokens] (may be NULL): every token's position for its embedding, lens[b] - n + its
 *             depth (0 where that is negative); lens [B] as in kvattn_paged_decode_tokens, needed for
 *             positions alone
 * Tokens from 64 * mask_words on get an empty mask, and the position of a root.  Rows behind
 * token_start[B] are left as they were.  B <= 2^20, num_tokens <= 2^30 (0: nothing is done). */
int kvattn_tree_masks(unsigned long long* masks, int* positions, const int* parents, const int* token_start,
                      const int* lens, int B, int num_tokens, int mask_words, void* stream);

/* Attention of trees' tokens over a paged cache of any kv_dtype (F32: qkv and out float, else bf16).
 * Token i of sequence b's n attends the first lens[b] - n positions and those new tokens j whose
 * position lens[b] - n + j is in [0, lens[b]) and whose bit its mask has, of whatever shape the masks
 * are; one that attends nothing gets zeros.  K and V of positions that a token does not attend never
 * reach its output, also where they are infinite or NaN.  A table entry outside the pool: its positions
 * are skipped.  16 tokens of a sequence share a pass over the cache.
 *   max_new  the most tokens of one sequence, at most 64 * mask_words (or num_tokens is); a sequence with
 *            more has the first max_new or more of them computed
 * B <= 65535; B * NH, num_tokens * NH and B * NH * (max_new or num_tokens, the smaller, / 16 rounded up) below 2^24.
 * Other arguments, limits and the workspace as in kvattn_paged_decode_tokens. */
int kvattn_paged_decode_tree(void* out, const void* qkv, const void* pages, const float* page_scales,
                             const int* block_table, int max_pages, int page_rows, int num_pages,
                             const int* token_start, const int* lens, const unsigned long long* masks, int mask_words,
                             int B, int num_tokens, int max_new, int NH, int hs, void* workspace,
                             size_t workspace_bytes, int S, int kv_dtype, void* stream);

/* After kvattn_verify_tree: K and V rows of every sequence's accepted path to where the next step needs
 * them, behind the prefix.  Row slot_map[token_start[b] + path[d]] goes to slot_map[token_start[b] + d],
 * codes and scales as they are, for every d from 0 until path[d] (entry token_start[b] + d of path) is not above
 * path[d - 1], not below d, or not one of the sequence's tokens.  Steps with a slot outside the pool are
 * skipped; a sequence's slots, and those of different sequences, must differ.  Every kv_dtype.
 * B * NH <= 2^24. */
int kvattn_paged_keep(void* pages, float* page_scales, int page_rows, int num_pages, const long long* slot_map,
                      const int* path, const int* token_start, int B, int num_tokens, int NH, int hs, int kv_dtype,
                      void* stream);

/* ---- Pages from request lengths --------------------------------------------------------
 * The bookkeeping of a paged cache, on the device: no length, table or page count goes through the
 * host, so a captured step allocates too.  No reference counterpart (the reference has one
 * contiguous cache).
 *   pool  int32 [4 + num_pages]: {index of the first free page in the ring, number of free pages, a
 *         word of the library's, unused}, then the ring of free page ids.
 *         kvattn_paged_pool_bytes bytes; kvattn_paged_pool_init makes every page free. */
size_t kvattn_paged_pool_bytes(int num_pages);
int kvattn_paged_pool_init(int* pool, int num_pages, void* stream);

/* Gives every request the pages of its next step.  Request b holds pages for held[b] positions
 * (those of block_table row b), keeps the first kept[b] of them (fewer after refused drafts, 0 when
 * it has ended) and adds fresh[b] tokens:
 *   pages    ceil((kept + fresh) / page_rows) - ceil(held / page_rows) pages are taken from the
 *            ring, in request order, and entered behind the ones held; if negative, the last pages
 *            go back to the ring in the same order (to be taken by later calls).  Entries of
 *            block_table behind a request's pages are left as they were.
 *   held_out [B], lens [B]: kept + fresh.  Either may be its own input (held, kept); apart from that
 *            no output may share memory with an input or another output.
 *   token_start [B+1]: sums of fresh; tokens token_start[b] .. token_start[b+1]-1 are request b's
 *   slot_map [max_tokens]: page * page_rows + row of each token's position, for kvattn_paged_store;
 *            -1 behind the last token, so that a step captured for max_tokens tokens stores no more
 *   positions [max_tokens] (may be NULL): each token's position; left as it was behind the last token
 *   pool_next [2] (may be NULL: the pool itself): the pool's first two words after the call.  With
 *            a buffer of its own the pool's words stay, so the call can be made again.
 * A request is refused, and keeps its pages and kept[b] positions (held_out = held, lens = kept), when
 * it needs pages and those up to its own in request order are more than the free ones, or its tokens
 * end behind max_tokens; its tokens then have slot -1.  So is one whose lengths are not
 * 0 <= kept <= held, 0 <= fresh, kept + fresh <= max_pages * page_rows; it counts as having no
 * tokens.  A granted request is told by lens[b] == kept[b] + fresh[b].  A refused one's token rows
 * stay among token_start's, and what attention and verification of the step write for them means
 * nothing: its kept is the next step's again.  Table entries outside [0, num_pages) give slot -1 and
 * go back to the ring as they are.
 * B <= 4096, max_tokens <= 2^30.  Calls on one pool must be ordered. */
int kvattn_paged_reserve(int* block_table, int max_pages, int page_rows, int num_pages, int* pool,
                         const int* held, const int* kept, const int* fresh, int B, int max_tokens,
                         int* held_out, int* lens, int* token_start, long long* slot_map, int* positions,
                         int* pool_next, void* stream);

/* K and V rows of num_tokens tokens, from qkv [num_tokens][3][NH][hs], into the pool at slots
 * slot_map[t] = page * page_rows + row, for every kv_dtype, as kvattn_paged_cache_write writes a
 * row.  Slots outside [0, num_pages * page_rows) are skipped; the others must differ from one
 * another.  num_tokens * NH <= 2^27, NH <= 2^24. */
int kvattn_paged_store(void* pages, float* page_scales, int page_rows, int num_pages, const long long* slot_map,
                       const void* qkv, int num_tokens, int NH, int hs, int kv_dtype, void* stream);

/* The rows at slot_map[t] out of the pool into kv [num_tokens][2][NH][hs] (K, then V), in the
 * activation type (float for F32, else bf16): code * scale, rounded once.  Rows of skipped slots are
 * left as they were.  As prefill attention over earlier positions reads them. */
int kvattn_paged_load(void* kv, const void* pages, const float* page_scales, int page_rows, int num_pages,
                      const long long* slot_map, int num_tokens, int NH, int hs, int kv_dtype, void* stream);

/* ---- Verification of drafted tokens ----------------------------------------------------
 * Row t = token_start[b] + i holds the target's distribution behind token i of sequence b's n
 * tokens; draft_tokens[t] is the draft that followed it, drawn from draft_probs row t (the last row
 * has none: its draft_tokens entry and its draft_probs row are not read).  With uniform[t] in [0, 1):
 *   drafts are accepted in order while uniform[t] * q(x) < p(x);
 *   at the first that is not, the next token is drawn from max(0, p - q) of its row, or where that
 *   is zero everywhere from its p; if all are accepted, from the last row's p.  A draw is the
 *   lowest token whose running sum passes uniform[last row] times the total, in 64 bits.
 * tokens [num_tokens] (may be draft_tokens): accepted drafts, the drawn token, -1 behind it; counts
 * [B]: accepted plus drawn.  A row without any mass draws nothing (counts: accepted alone).  A sequence without tokens
 * has count 0; rows behind token_start[B] are left as they were.  num_tokens may be 0: then counts and
 * token_start alone are needed.  B <= 65536, V <= 2^24, num_tokens <= 2^30.
 *   target_probs, draft_probs  [num_tokens] rows of V probabilities, row_stride elements apart, float
 *               (dtype KVATTN_KV_F32) or bf16 (KVATTN_KV_BF16); NaN, infinite and negative ones weigh
 *               nothing in a draw.  draft_probs NULL: drafts without probabilities (q = 1 at the draft)
 *   draft_tokens  ids outside [0, V) are refused
 *   workspace   kvattn_verify_workspace_bytes(B, V) bytes or more, 256-byte aligned, zeroed once
 *               (kvattn_workspace_init); every call leaves it zero again, so a buffer of the largest
 *               size serves calls of any B and V.  Calls sharing it must be ordered, and only calls
 *               of this entry point may.
 * No reference counterpart (the reference samples one token at a time on the host). */
size_t kvattn_verify_workspace_bytes(int B, int V);
int kvattn_verify_drafts(int* tokens, int* counts, const void* target_probs, const void* draft_probs,
                         const int* draft_tokens, const float* uniform, const int* token_start, int B,
                         int num_tokens, int V, long long row_stride, int dtype, void* workspace,
                         size_t workspace_bytes, void* stream);

/* Verification of a tree of drafts.  Row t of target_probs is the distribution behind tree token t.  From a
 * sequence's token 0 on, the children of the token reached are tried in the order of their indices: the
 * first one whose running sum of target_probs[t][child's token] passes uniform[t] is accepted and reached
 * next.  (A token that an earlier child is too, an id outside [0, V) and what is not a positive finite
 * number weigh nothing.)  Where none is accepted, the next token is drawn from row t without the tokens
 * of t's children, or where nothing is left without them from all of row t: the lowest token whose
 * running sum passes draw[b] times the total.  Sums are 64 bits wide.  The tokens that come out are the
 * target's, whatever the tree was made from (uniform and draw are independent of it).
 *   tokens [num_tokens] (may be tree_tokens): accepted tokens, the drawn one, -1 behind it
 *   path [num_tokens]: the root's index 0, then the accepted tokens' among the sequence's, -1 behind: the rows that
 *            kvattn_paged_keep keeps
 *   counts [B]: accepted plus drawn (a row without any mass draws nothing)
 *   kept [B] (may be NULL): lens[b] - n + 1 + accepted, the next step's kept of kvattn_paged_reserve; of a
 *            sequence without tokens lens[b].  lens [B], needed for kept alone, as in kvattn_tree_masks.
 *            A request that kvattn_paged_reserve refused keeps what it kept, which the caller sets again
 *   tree_tokens [num_tokens]: every tree token's id (a root's is not read)
 *   uniform [num_tokens], draw [B]: numbers in [0, 1)
 * Tokens of a sequence from the 256th on are not looked at.  Other arguments, limits and the workspace as in
 * kvattn_verify_drafts, which may share the workspace. */
int kvattn_verify_tree(int* tokens, int* path, int* counts, int* kept, const void* target_probs, const int* tree_tokens,
                       const int* parents, const float* uniform, const float* draw, const int* token_start,
                       const int* lens, int B, int num_tokens, int V, long long row_stride, int dtype, void* workspace,
                       size_t workspace_bytes, void* stream);

/* ---- Rules on logits -------------------------------------------------------------------
 * What a sequence's logits go through before a token is chosen.  Device arrays; NULL: no such rule.
 * "Held" are the tokens of the sequence's history and, for a row of a tree, of the row's branch (the
 * tokens whose bits the row's mask has: its ancestors and itself). */
typedef struct kvattn_logit_rules {
    const int* history;          /* [B][max_history] ids; others than 0 .. V - 1 are passed over */
    const int* history_len;      /* [B] of them in use */
    const int* prompt_len;       /* [B] the first of them that are the prompt's: held, but not generated */
    const int* tokens;           /* [rows] id of every row's own token, with masks */
    const unsigned long long* masks;   /* [rows][mask_words] as in kvattn_tree_masks */
    const float* repetition;     /* [B] x of a held token: x / repetition where x > 0, else x * repetition */
    const float* frequency;      /* [B] subtracted for every time a token was generated */
    const float* presence;       /* [B] subtracted once where it was */
    const int* bias_start;       /* [B+1] sequence b's entries of bias_ids and bias */
    const int* bias_ids;         /* [num_bias] */
    const float* bias;           /* [num_bias] added; of an id listed twice the last entry holds */
    const unsigned* allowed;     /* [num_allowed][allowed_stride] bit v % 32 of word v / 32: v is allowed; others: -inf */
    const int* allowed_of;       /* [rows] a row's line of allowed; outside [0, num_allowed): all are.  NULL: line `row` */
    const float* temperature;    /* [B] of the probabilities; not above 0: the likeliest token, the lowest of several */
    int max_history;             /* up to 32768 */
    int mask_words;              /* 1 to 4 */
    int num_bias, max_bias;      /* entries in all, and most of one sequence (further ones are passed over; up to 32768) */
    int num_allowed, allowed_stride;   /* words */
    void* workspace;             /* may be NULL: see kvattn_logits_workspace_bytes */
    size_t workspace_bytes;
} kvattn_logit_rules;

/* Bytes of a workspace with which rows of probabilities are cut into slices, several workgroups a row, where there are few
 * rows (without one, and where out overlaps logits, a row is one workgroup's): 8-byte aligned, zeroed once
 * (kvattn_workspace_init), of no further content between calls.  Calls sharing it must be ordered, and only calls of
 * kvattn_process_logits may.  The slices of a row wait for one another's maxima, within the bound of
 * kvattn_set_merge_poll_limit; one that stops waiting works the others' out itself (the result is the same, bit for
 * bit).  So where another stream's work keeps some of them off the GPU for long, the others wait for the whole bound and
 * then do up to as many slices' work as their row has: without a workspace a call has no such wait. */
size_t kvattn_logits_workspace_bytes(void);

/* The rules on rows of V logits, in the order above, in float: repetition, frequency and presence, bias, allowed.
 *   probs 0: the logits (-inf where not allowed); 1: softmax(x / temperature), as kvattn_verify_drafts and
 *            kvattn_verify_tree take it; a row that allows nothing becomes zeros, one with a NaN or +inf that is
 *            allowed NaN where it is not zero (the likeliest token is looked for among numbers; zeros where there
 *            are none)
 *   rules    host struct, read by the call (the arrays it names are read when the kernel runs); NULL: none
 *   token_start [B+1] device: rows token_start[b] .. token_start[b+1]-1 are sequence b's; rows behind token_start[B]
 *            are left as they were.  NULL: row b is sequence b's (rows == B)
 *   dtype, out_dtype  KVATTN_KV_F32 or KVATTN_KV_BF16; out may be logits where the types and strides are the same.
 *            What lies behind a row's V elements is neither read nor written
 * V <= 2^18, rows <= 2^21, B <= 2^20.  KVATTN_ERR_LDS: the table of named tokens does not fit in LDS (probabilities of
 * rows that are one workgroup's: V / 8 bytes for the map and V / 16 for its sums, V / 8 with allowed, 8 bytes, with
 * biases 12, for each of min(V, max_history + 64 mask_words + max_bias) entries, in 156 KB).  With a workspace, and
 * outputs that are not the logits' own memory, any table fits: rows are then cut into slices, some rows at a time.
 * No reference counterpart (the reference takes the argmax or samples on the host, without rules). */
int kvattn_process_logits(void* out, const void* logits, const kvattn_logit_rules* rules, const int* token_start,
                          int B, int rows, int V, long long row_stride, long long out_stride, int dtype, int out_dtype,
                          int probs, void* stream);

/* The decode step's fully connected layer, used after the attention for the output
 * projection: for b < B, m < M
 *   pre = w_scale[m] * sum_k W[m][k] * x[b][k] + bias[m]      (w_scale: 8-bit weights only)
 *   pre_gelu[b][m] = pre (if pre_gelu != NULL);  out[b][m] = gelu ? GELU_tanh(pre) : pre
 * with FP32 accumulation.  Types by w_dtype (a kvattn_dtype):
 *   F32        W, x, bias, out, pre_gelu float
 *   BF16       W, x, bias, out, pre_gelu bf16
 *   INT8, FP8  W one code per weight ([M][K] bytes) with one FP32 scale per row; x, bias,
 *              out, pre_gelu bf16
 * W is row-major [M][K]; x [B][K]; out [B][M].  Requires K % 16 == 0 (any length: rows
 * beyond 64 * 16 chunks of 16 bytes are walked in blocks, as the reference's tail loops walk
 * any K), 16-byte aligned W and x.  bias may be NULL.  One or two vectors (and few vectors
 * where the matrix cores do not pay) take one wave per row; from 8192 rows on (a vocabulary
 * projection) a wave takes 4 rows of 8-bit weights, 2 of wider ones, so that more weight
 * bytes are in flight.
 * Replaces launch_GEMV6_fused (Inference_gpt2/GEMV.cuh:132-206) and launch_GEMV6_w8x2
 * (Inference_gpt2/GEMV_w8.cuh:64-184), which matmul_forward[_w8] calls for one decode token
 * (inference_gpt2_opt.cu:106-132); the attention output projection is at :349-355.  Batches
 * (from 3 vectors on; up to 1024 rows of more than 1600 columns from 3 to 5, FP32 weights
 * from 4 to 12) go through the matrix cores with FP32 sums, where the reference takes
 * cuBLASLt; other B > 1 read the weights once for all B vectors when a row fits in one
 * block.  A vector's result may differ in its last bits with the size of the batch (another
 * order of the same sums). */
int kvattn_gemv(void* out, void* pre_gelu, const void* W, const float* w_scale, const void* x,
                const void* bias, int B, int M, int K, int w_dtype, int gelu, void* stream);

/* kvattn_gemv with the output type given: out and pre_gelu are float (out_dtype
 * KVATTN_KV_F32) or bf16 (KVATTN_KV_BF16), whatever the weights; x and bias keep the
 * activation type of w_dtype.  Replaces the reference's instantiations with an output type
 * other than the activations', such as the vocabulary projection over the 8-bit embedding
 * table, launch_GEMV6_w8x2<float, floatX>(logits, NULL, w8_wte, lnf, w8_wte_s, NULL, Vp, C,
 * false, stream) (inference_gpt2_opt.cu:389-394). */
int kvattn_gemv_ex(void* out, void* pre_gelu, const void* W, const float* w_scale, const void* x,
                   const void* bias, int B, int M, int K, int w_dtype, int out_dtype, int gelu, void* stream);

/* The QKV projection with the KV append in its epilogue: kvattn_gemv with M = 3 * NH * hs
 * (no GELU) into qkv [B][3][NH][hs], whose K and V rows also go to column cur_len of
 * kv_cache [2][B][NH][maxT][hs], as kvattn_cache_write would write them, bit for bit.
 *   kv_dtype F32 / BF16: the cache holds the activation type (float for F32 weights, bf16
 *     otherwise); kv_scale and the workspace are not used.
 *   kv_dtype INT8 / FP8_E4M3 (bf16 activations): codes and one row scale per (b, K|V, h) in
 *     kv_scale [2][B][NH][maxT], from the bf16 values in qkv with the append's quantiser.
 *     On the vector units the 64 channels of a row come from 16 workgroups, so they meet
 *     in the workspace (a batch on the matrix cores does not use it, but it is checked alike):
 *     kvattn_gemv_qkv_append_workspace_bytes(B, NH) bytes, 256-byte aligned, zeroed once
 *     (kvattn_workspace_init); each word there carries the call that wrote it, so the
 *     workspace needs no clearing between calls.  Calls sharing a workspace must be ordered
 *     (one stream).
 * d_cur_len as in kvattn_decode (NULL: the library's device length).  hs must be 64.
 * Replaces the QKV GEMV followed by the append launch (inference_gpt2_opt.cu:290-303, 329;
 * the append kernels attention_kvcache.cuh:46-64, attention_kvcache_w8.cuh:115-155), one
 * launch fewer per layer. */
size_t kvattn_gemv_qkv_append_workspace_bytes(int B, int NH);
int kvattn_gemv_qkv_append(void* qkv, const void* W, const float* w_scale, const void* x,
                           const void* bias, int B, int NH, int hs, int K, void* kv_cache,
                           float* kv_scale, int maxT, const int* d_cur_len, int lens_per_seq,
                           int w_dtype, int kv_dtype, void* workspace, size_t workspace_bytes,
                           void* stream);

/* ---- 4-bit weights with a scale for every group --------------------------------------------
 * kvattn_gemv_ex on INT4 or FP4_E2M1 codes whose scales are bf16, one for every `group` (32, 64 or 128)
 * neighbours of a row: weight [m][k] = code * scale[m][k / group], codes as in the 4-bit caches (INT4: half byte - 8,
 * here -8 too; FP4: sign and one of 0 .5 1 1.5 2 3 4 6).  K is a multiple of group, K <= 2^20, M < 2^29, M K < 2^40.
 * No reference counterpart (its weights end at 8 bits, with one scale a row).
 * Weights are laid out once for the kernels: w4, 16-byte aligned, of kvattn_w4_bytes(M, K, group) bytes (0: such a
 * matrix is refused); what is in it depends on M, K and group. */
size_t kvattn_w4_bytes(int M, int K, int group);

/* Lays out codes [M][K / 2] bytes (column 2i in the low half of byte i, 16-byte aligned) and scales [M][K / group] bf16. */
int kvattn_w4_pack(void* w4, const void* codes, const void* scales, int M, int K, int group, int w_dtype, void* stream);

/* Codes and lays out W [M][K], float or bf16 (src_dtype): scale = bf16(largest magnitude / 7, FP4: / 6), codes of w / scale
 * to nearest, ties to even, within -7 .. 7 (FP4: -6 .. 6). */
int kvattn_w4_quantize(void* w4, const void* W, int M, int K, int group, int src_dtype, int w_dtype, void* stream);

/* out[b][m] = act(sum_k weight[m][k] x[b][k] + bias[m]) with FP32 sums; x, bias (may be NULL) bf16, out and pre_gelu
 * (may be NULL) float or bf16 by out_dtype; gelu as in kvattn_gemv.  Any B, on the matrix cores; M <= 2^28 - 32, B M and
 * B K < 2^31.  A vector that is not finite spoils its own outputs alone (of INT4 codes an infinity gives NaN). */
int kvattn_gemv_w4(void* out, void* pre_gelu, const void* w4, const void* x, const void* bias, int B, int M, int K,
                   int group, int w_dtype, int out_dtype, int gelu, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* KVATTN_H */
