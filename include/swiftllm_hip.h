/*
 * swiftllm_hip.h — C ABI of libswiftllm_hip.so, the MI355X (gfx950) decode
 * hot path: paged-attention decode (single pass and split-K), the
 * reshape_and_cache KV-cache write, and MoE top-k routing / dispatch.
 *
 * Every entry point:
 *   - takes caller-owned device pointers on the current HIP device;
 *   - allocates nothing (scratch memory is passed in by the caller, except
 *     for swiftllm_hip_launch_paged_attention_v2_noalloc, whose scratch is a
 *     static device array);
 *   - is asynchronous on the given stream (NULL = the default stream);
 *   - validates its arguments synchronously on the host before any launch.
 *
 * Device memory layouts (row-major, fp16 = IEEE binary16):
 *   query, output       [num_seqs, num_heads, head_dim]
 *   key/value cache     [num_blocks, num_kv_heads, head_dim, block_size]
 *   block_tables        int32 [num_seqs, max_num_blocks_per_seq]
 *   context_lens        int32 [num_seqs]
 *   key, value (new)    [num_tokens, num_kv_heads, head_dim]
 *   slot_mapping        int32 [num_tokens]; slot = block * block_size + offset
 *
 * Reference interfaces replaced (paths relative to the swiftllm repository):
 *   crates/swiftllm-cuda/kernels/paged_attention.cu:230-327  (extern "C" launchers)
 *   crates/swiftllm-cuda/src/bindings.rs:8-113              (params structs, wrappers)
 *   crates/swiftllm-cuda/src/lib.rs:16-42                   (CudaError variants)
 */
#ifndef SWIFTLLM_HIP_H
#define SWIFTLLM_HIP_H

#include <stddef.h>
#include <stdint.h>

#if defined(__has_include)
#if __has_include(<hip/hip_runtime_api.h>)
#include <hip/hip_runtime_api.h>
#define SWIFTLLM_HIP_HAVE_RUNTIME_API 1
#endif
#endif
#ifndef SWIFTLLM_HIP_HAVE_RUNTIME_API
typedef struct ihipStream_t* hipStream_t;
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------ */
/* Status codes. Negative values mirror the CudaError variants of            */
/* crates/swiftllm-cuda/src/lib.rs:16-42, in declaration order.              */
/* ------------------------------------------------------------------------ */
typedef enum swiftllm_status {
    SWIFTLLM_OK = 0,
    SWIFTLLM_ERR_INIT = -1,              /* CudaError::InitError        */
    SWIFTLLM_ERR_KERNEL = -2,            /* CudaError::KernelError      */
    SWIFTLLM_ERR_MEMORY = -3,            /* CudaError::MemoryError      */
    SWIFTLLM_ERR_INVALID_PARAMETER = -4, /* CudaError::InvalidParameter */
    SWIFTLLM_ERR_DEVICE_NOT_FOUND = -5,  /* CudaError::DeviceNotFound   */
    SWIFTLLM_ERR_NOT_SUPPORTED = -6      /* CudaError::NotSupported     */
} swiftllm_status;

/* Status of the most recent call made on this host thread (the void
 * launchers report failures only through this), and its message (the
 * String payload of the CudaError variant). The message pointer stays valid
 * until the next call on the same thread. */
int swiftllm_hip_last_error(void);
const char* swiftllm_hip_last_error_message(void);

/* Library version string, e.g. "0.1.0 gfx950". */
const char* swiftllm_hip_version(void);

/* SWIFTLLM_OK when at least one HIP device is visible, else
 * SWIFTLLM_ERR_DEVICE_NOT_FOUND (the no-device behaviour of bindings.rs:72-75). */
int swiftllm_hip_device_check(void);

/* ------------------------------------------------------------------------ */
/* 1. Drop-in launchers: same names and parameter lists as                   */
/*    paged_attention.cu:232-300, with hipStream_t for cudaStream_t.         */
/*    They return void; failures are readable via swiftllm_hip_last_error(). */
/* ------------------------------------------------------------------------ */

/* Replaces launch_paged_attention_v1 (paged_attention.cu:232-269).
 * Single-pass decode: out[s,h] = softmax(scale * q[s,h] . K^T) . V over the
 * first context_lens[s] tokens of sequence s, with kv head h / (H / Hkv).
 * head_dim in {64, 128}; block_size 16; num_heads % num_kv_heads == 0.
 * context_lens[s] <= 0 writes zeros. */
void launch_paged_attention_v1(void* output, void* query, void* key_cache,
                               void* value_cache, int* block_tables,
                               int* context_lens, float scale, int num_seqs,
                               int num_heads, int num_kv_heads, int head_dim,
                               int block_size, int max_num_blocks_per_seq,
                               hipStream_t stream);

/* Replaces launch_reshape_and_cache (paged_attention.cu:271-300).
 * key_cache[slot / bs, h, d, slot % bs] = key[t, h, d] (bit copy), same for
 * value. Tokens with slot_mapping[t] < 0 are skipped (padding). */
void launch_reshape_and_cache(void* key, void* value, void* key_cache,
                              void* value_cache, int* slot_mapping,
                              int num_tokens, int num_kv_heads, int head_dim,
                              int block_size, hipStream_t stream);

/* Split-K decode (the intent of paged_attention_v2_kernel,
 * paged_attention.cu:139-163, whose body is empty and which has no
 * launcher). The context of each sequence is cut into partitions of
 * partition_size tokens (a multiple of 16). A first kernel attends each
 * partition and keeps (max logit, exp sum, partial output) in `workspace`;
 * a second kernel rescales and reduces the partitions of every sequence
 * that has more than one (a sequence with a single partition is written by
 * the first kernel directly). partition_size is the finest cut of a large
 * batch: an item may take several neighbouring partitions, as many as the
 * batch's lengths leave each workgroup of the GPU. Batches of few sequences
 * (at most two per team of workgroups, where the workspace has the room) are
 * cut into equal ranges of blocks instead, one per team, whatever the
 * partitions, and tables too short for a split to pay (at most 96 blocks)
 * are attended in a single pass; the size query's answer depends on the
 * current device's compute units.
 * partition_size 0 selects balanced scheduling: the blocks of all sequences
 * are split into equal ranges, one per team of waves for large batches, so
 * a ragged batch has no long tail; ranges that cut a sequence leave
 * fragments that a second kernel combines. Tables of at most 64 blocks (32
 * for more than four sequences times kv heads per compute unit), whose
 * longest context is no long tail, may run in a single pass. Shapes it cannot take (more
 * than 4096 sequences, or teams so wide that fewer than four fit in the
 * resident grid) fall back to partitions of 512 tokens; the workspace size
 * query covers both.
 * `workspace` holds at least
 * swiftllm_hip_paged_attention_v2_workspace_size() bytes, 256-byte aligned;
 * it is plain scratch (no initialisation, contents unspecified after the
 * call). Calls that share a workspace must be ordered on one stream. */
void launch_paged_attention_v2(void* output, void* workspace,
                               size_t workspace_bytes, void* query,
                               void* key_cache, void* value_cache,
                               int* block_tables, int* context_lens,
                               float scale, int num_seqs, int num_heads,
                               int num_kv_heads, int head_dim, int block_size,
                               int max_num_blocks_per_seq, int partition_size,
                               hipStream_t stream);

/* Bytes of workspace launch_paged_attention_v2 needs for these sizes. */
size_t swiftllm_hip_paged_attention_v2_workspace_size(
    int num_seqs, int num_heads, int num_kv_heads, int head_dim,
    int block_size, int max_num_blocks_per_seq, int partition_size);

/* Zero-fills `bytes` bytes at `workspace` with a kernel (no memset node, so
 * it may be captured in a graph). No workspace of this library needs it; it
 * is there for callers that want deterministic scratch contents. */
int swiftllm_hip_workspace_clear(void* workspace, size_t bytes,
                                 hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 2. Status-returning twins of the launchers (same arguments; return a     */
/*    swiftllm_status). num_blocks bounds every block id read from           */
/*    block_tables / slot_mapping: ids outside [0, num_blocks) are skipped.  */
/*    Pass num_blocks <= 0 when the pool size is unknown (no bound);         */
/*    negative ids are skipped in either case.                               */
/* ------------------------------------------------------------------------ */
int swiftllm_hip_launch_paged_attention_v1(
    void* output, const void* query, const void* key_cache,
    const void* value_cache, const int* block_tables, const int* context_lens,
    float scale, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
    int block_size, int max_num_blocks_per_seq, int num_blocks,
    hipStream_t stream);

int swiftllm_hip_launch_paged_attention_v2(
    void* output, void* workspace, size_t workspace_bytes, const void* query,
    const void* key_cache, const void* value_cache, const int* block_tables,
    const int* context_lens, float scale, int num_seqs, int num_heads,
    int num_kv_heads, int head_dim, int block_size, int max_num_blocks_per_seq,
    int partition_size, int num_blocks, hipStream_t stream);

int swiftllm_hip_launch_reshape_and_cache(
    const void* key, const void* value, void* key_cache, void* value_cache,
    const int* slot_mapping, int num_tokens, int num_kv_heads, int head_dim,
    int block_size, int num_blocks, hipStream_t stream);

/* Bytes of the static device scratch behind
 * swiftllm_hip_launch_paged_attention_v2_noalloc (one copy per device). The
 * array is part of libswiftllm_hip.so's code object, so every process that
 * runs any kernel of the library on a device holds these 64 MiB there from
 * the code object's load until the process ends, whether or not it ever
 * calls the no-alloc entry point. */
#define SWIFTLLM_HIP_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)

/* No counterpart in the reference. For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc): swiftllm_hip_launch_paged_attention_v2 without the
 * workspace arguments. Its split-K scratch is a static device array of
 * SWIFTLLM_HIP_NOALLOC_SCRATCH_BYTES bytes, reserved on each device when
 * the library's code object loads there (first use of any of its kernels)
 * and held until the process ends; the first call on a device looks up the
 * array's address, and nothing is allocated or freed per call.
 * Sizes whose workspace (swiftllm_hip_paged_attention_v2_workspace_size for
 * the mode the call runs) exceeds that return SWIFTLLM_ERR_INVALID_PARAMETER.
 * All calls on one device share the array: calls that overlap on a device
 * (several streams or host threads) race and must be ordered on one stream. */
int swiftllm_hip_launch_paged_attention_v2_noalloc(
    void* output, const void* query, const void* key_cache,
    const void* value_cache, const int* block_tables, const int* context_lens,
    float scale, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
    int block_size, int max_num_blocks_per_seq, int partition_size,
    int num_blocks, hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 3. Params-struct twins of crates/swiftllm-cuda/src/bindings.rs.           */
/*    size_t stands for usize, float for f32.                                */
/* ------------------------------------------------------------------------ */

/* bindings.rs:8-30 (PagedAttentionParams). */
typedef struct swiftllm_paged_attention_params {
    size_t num_seqs;
    size_t num_heads;
    size_t num_kv_heads;
    size_t head_dim;
    size_t block_size;
    float scale;
    size_t max_context_len;
} swiftllm_paged_attention_params;

/* bindings.rs:78-92 (ReshapeCacheParams). */
typedef struct swiftllm_reshape_cache_params {
    size_t num_tokens;
    size_t num_kv_heads;
    size_t head_dim;
    size_t block_size;
} swiftllm_reshape_cache_params;

/* Replaces bindings::paged_attention_decode (bindings.rs:56-76). The row
 * stride of block_tables is ceil(max_context_len / block_size), the only
 * stride the Rust signature can imply. Runs the single-pass kernel. */
int swiftllm_hip_paged_attention_decode(
    void* output, const void* query, const void* key_cache,
    const void* value_cache, const int32_t* block_tables,
    const int32_t* context_lens, const swiftllm_paged_attention_params* params,
    hipStream_t stream);

/* Replaces bindings::reshape_and_cache (bindings.rs:94-113). */
int swiftllm_hip_reshape_and_cache(const void* key, const void* value,
                                   void* key_cache, void* value_cache,
                                   const int32_t* slot_mapping,
                                   const swiftllm_reshape_cache_params* params,
                                   hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 3a. Paged prefill (causal attention over a packed batch of prompts).      */
/* ------------------------------------------------------------------------ */

/* Replaces bindings::paged_attention_prefill (bindings.rs:32-54): the steps
 * of PagedAttention::prefill (paged_attention.rs:154-189) after the K/V
 * write. query / output fp16 [T, H, D] packed: sequence s owns tokens
 * [start_s, start_s + context_lens[s]), start_s the sum of the lengths
 * before it. Token i of s attends to tokens j <= i of s, whose K/V sit in
 * the cache at slot_mapping[start_s + j]; the slots of a sequence must walk
 * its block table from position 0 (table[p / 16] * 16 + p % 16). A value that
 * is not finite also makes NaN of earlier tokens that one wave (32 query
 * rows) serves together with a token of its 16-token block or a later one;
 * a key that is not finite does not.
 * params->max_context_len bounds every context_lens[s]; above 2^24 tokens it
 * can return SWIFTLLM_ERR_NOT_SUPPORTED (grid size). */
int swiftllm_hip_paged_attention_prefill(
    void* output, const void* query, const void* key_cache,
    const void* value_cache, const int32_t* slot_mapping,
    const int32_t* context_lens, const swiftllm_paged_attention_params* params,
    hipStream_t stream);

/* The same with plain arguments and a pool bound: blocks outside
 * [0, num_blocks) are skipped (num_blocks <= 0: no bound; negative block ids
 * are always skipped). */
int swiftllm_hip_launch_paged_prefill(void* output, const void* query,
                                      const void* key_cache,
                                      const void* value_cache,
                                      const int32_t* slot_mapping,
                                      const int32_t* context_lens, float scale,
                                      int num_seqs, int num_heads,
                                      int num_kv_heads, int head_dim,
                                      int block_size, int max_context_len,
                                      int num_blocks, hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 3b. Block copies of the KV cache. block_mapping holds num_pairs (src, dst) */
/*     int64 pairs in memory the device can read (device memory or pinned    */
/*     host memory). A pair with a negative id is skipped; destinations must */
/*     be distinct and must not be sources in the same call.                 */
/* ------------------------------------------------------------------------ */

/* Replaces launch_copy_blocks (paged_attention.cu:302-327; kernel cu:201-227,
 * whose 2048-thread workgroups fail to launch): K[dst] = K[src] and
 * V[dst] = V[src] for whole [Hkv, D, BS] blocks, one launch. */
void launch_copy_blocks(int64_t* block_mapping, void* key_cache,
                        void* value_cache, int num_pairs, int num_kv_heads,
                        int head_dim, int block_size, hipStream_t stream);

/* Status twin of launch_copy_blocks; ids outside [0, num_blocks) are skipped
 * (num_blocks <= 0: no bound). */
int swiftllm_hip_launch_copy_blocks(const int64_t* block_mapping,
                                    void* key_cache, void* value_cache,
                                    int num_pairs, int num_kv_heads,
                                    int head_dim, int block_size,
                                    int num_blocks, hipStream_t stream);

/* Replaces bindings::copy_blocks (bindings.rs:200-223): the same pairs in
 * the K and V caches of every layer. key_caches / value_caches are host
 * arrays of num_layers device pointers. */
int swiftllm_hip_copy_blocks(void* const* key_caches,
                             void* const* value_caches,
                             const int64_t* block_mapping, size_t num_pairs,
                             size_t num_layers, size_t num_kv_heads,
                             size_t head_dim, size_t block_size,
                             hipStream_t stream);

/* Replaces bindings::swap_blocks (bindings.rs:225-242):
 * dst[dst_id * block_size_bytes, + block_size_bytes) =
 * src[src_id * block_size_bytes, + block_size_bytes) for every pair. src
 * and dst are device memory or pinned host memory (hipHostMalloc), in any
 * combination; one kernel moves every block. */
int swiftllm_hip_swap_blocks(const void* src, void* dst,
                             const int64_t* block_mapping, size_t num_pairs,
                             size_t block_size_bytes, hipStream_t stream);

/* swiftllm_hip_swap_blocks with pool bounds: pairs whose src id is outside
 * [0, src_blocks) or whose dst id is outside [0, dst_blocks) are skipped
 * (a bound <= 0: none). */
int swiftllm_hip_launch_swap_blocks(const void* src, void* dst,
                                    const int64_t* block_mapping,
                                    size_t num_pairs, size_t block_size_bytes,
                                    long long src_blocks, long long dst_blocks,
                                    hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 4. MoE top-k routing and dispatch. The reference has no kernel for this:  */
/*    MoeMlp::forward (crates/swiftllm-models/src/layers/mlp.rs:240-252)     */
/*    names the steps (router logits, top-k, route, combine) and returns     */
/*    zeros. Conventions follow sampling/mod.rs:366-385 (max-subtracted     */
/*    softmax; stable descending order, ties to the lower expert index).    */
/* ------------------------------------------------------------------------ */

/* logits fp32 [T, E] -> expert_ids int32 [T, K] (descending logit, ties to
 * the lower index) and weights fp32 [T, K] = softmax probabilities of the
 * selected experts renormalised to sum to 1. 1 <= K <= E <= 256, K <= 8. */
int swiftllm_hip_moe_route(const float* logits, int num_tokens,
                           int num_experts, int top_k, int32_t* expert_ids,
                           float* weights, hipStream_t stream);

/* Bytes of workspace swiftllm_hip_moe_dispatch needs. */
size_t swiftllm_hip_moe_dispatch_workspace_size(int num_tokens,
                                                int num_experts, int top_k);

/* Expert-contiguous permutation of the routed token copies.
 *   expert_counts[e]      = #{(t,k) : expert_ids[t,k] = e}
 *   expert_offsets[E + 1] = exclusive prefix sum, offsets[E] = T*K
 *   row(t,k)              = offsets[e] + rank of (t,k) among the entries of
 *                           expert e in (t ascending, k ascending) order
 *   x_perm[row(t,k), :]   = x[t, :]          (fp16 bit copy, hidden wide)
 *   inverse[t, k]         = row(t,k)
 *   sorted_token_ids[row] = t
 * `workspace` (swiftllm_hip_moe_dispatch_workspace_size bytes, 256-byte
 * aligned) is plain scratch: no initialisation. Ids outside [0, E) are
 * dropped (inverse = -1). x_perm may be NULL to compute the index arrays
 * only. */
int swiftllm_hip_moe_dispatch(const int32_t* expert_ids, const void* x,
                              int num_tokens, int top_k, int num_experts,
                              int hidden, int32_t* expert_counts,
                              int32_t* expert_offsets, void* x_perm,
                              int32_t* inverse, int32_t* sorted_token_ids,
                              void* workspace, size_t workspace_bytes,
                              hipStream_t stream);

/* swiftllm_hip_moe_route followed by swiftllm_hip_moe_dispatch, with the
 * routing done inside the dispatch's ranking kernel (one launch fewer, and
 * the ids are not re-read). Same outputs as the two calls; the same
 * workspace size. */
int swiftllm_hip_moe_route_dispatch(const float* logits, const void* x,
                                    int num_tokens, int top_k, int num_experts,
                                    int hidden, int32_t* expert_ids,
                                    float* weights, int32_t* expert_counts,
                                    int32_t* expert_offsets, void* x_perm,
                                    int32_t* inverse, int32_t* sorted_token_ids,
                                    void* workspace, size_t workspace_bytes,
                                    hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 4b. MoE expert computation: steps 3-4 of MoeMlp::forward                 */
/*     (crates/swiftllm-models/src/layers/mlp.rs:240-246) over GatedMlp      */
/*     experts (mlp.rs:118-160: down(silu(gate(x)) * up(x))), Linear weights  */
/*     [out_features, in_features] (layers/mod.rs:22-24). The reference      */
/*     returns zeros for all of it.                                           */
/* ------------------------------------------------------------------------ */

/* Grouped expert GEMM over expert-contiguous rows: expert e owns rows
 * [expert_offsets[e], expert_offsets[e+1]) of `a` (fp16 [m_total, k], e.g.
 * the dispatch's x_perm) and of `c` (fp16 [m_total, n]).
 *   w2 == NULL: c[rows] = a[rows] . w[e]^T
 *   w2 != NULL: c[rows] = silu(a[rows] . w[e]^T) * (a[rows] . w2[e]^T)
 * w and w2 are fp16 [E, n, k]. fp32 accumulation. Supported (NotSupported
 * otherwise): n % 128 == 0 with w2, n % 256 == 0 without; k % 64 == 0 and
 * k <= 2^21; E <= 256. expert_offsets runs non-decreasing from 0 to m_total
 * (as the dispatch writes it): the grid is sized from m_total. Enqueues up
 * to two kernels on `stream`: whole 256-row tiles, and the experts' tails
 * of at most 128 rows (a decode batch: only the second). */
int swiftllm_hip_moe_expert_gemm(const void* a, const void* w, const void* w2,
                                 const int32_t* expert_offsets,
                                 int num_experts, int m_total, int n, int k,
                                 void* c, hipStream_t stream);

/* out[t, :] = fp16( sum_k weights[t, k] * y[inverse[t, k], :] ), fp32
 * fused multiply-adds in k order; entries with inverse outside
 * [0, y_rows) contribute nothing. y fp16 [y_rows, hidden]; hidden % 8 == 0. */
int swiftllm_hip_moe_combine(const void* y, const float* weights,
                             const int32_t* inverse, int num_tokens, int top_k,
                             int hidden, int y_rows, void* out,
                             hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 5. Block-table gather check: materialise the K and V of (seq, kv_head) as */
/*    contiguous [context_len, head_dim] fp16 arrays through the same tile   */
/*    addressing the decode kernel uses (paged_attention.cu:80-87, 114-116). */
/* ------------------------------------------------------------------------ */
int swiftllm_hip_gather_kv(const void* key_cache, const void* value_cache,
                           const int* block_tables, const int* context_lens,
                           int seq, int kv_head, int num_kv_heads,
                           int head_dim, int block_size,
                           int max_num_blocks_per_seq, int max_context_len,
                           void* k_out, void* v_out, hipStream_t stream);

/* Wave-reduction check: the lane reductions the kernels inline (the
 * reference's 32-lane butterflies, paged_attention.cu:17-31, on 64-lane
 * waves), run on caller data so they can be compared lane by lane with a
 * sequential reference. For each row r < num_rows of x (float [num_rows][64])
 * and xi (int32 [num_rows][64]), lane l writes
 *   out[r][0][l] = max of x[r][l % 16 + 16 k], k = 0..3  (softmax row max)
 *   out[r][1][l] = sum of the same four                  (softmax row sum)
 *   out[r][2][l] = max of x[r][0..63]                    (split-K reduce)
 *   out[r][3][l] = sum of x[r][0..63]
 *   scan[r][l]   = xi[r][0] + ... + xi[r][l]             (dispatch offsets)
 * out is float [num_rows][4][64], scan int32 [num_rows][64]. */
int swiftllm_hip_wave_reduce_check(const float* x, const int32_t* xi,
                                   int num_rows, float* out, int32_t* scan,
                                   hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 6. The attention step around the cache. The reference plans a step on the */
/*    host (BlockManager, KvCache::get_slot_mapping), declares rotary         */
/*    embeddings (crates/swiftllm-models/src/layers/attention.rs:297-353) and */
/*    ALiBi / sliding-window options that no kernel of it implements          */
/*    (memory/paged_attention.rs:39-43, 111-135). These entry points do all   */
/*    of it on the device, without a synchronisation, so that a step can be   */
/*    captured in a graph. Values are fp16 (SWIFTLLM_HIP_F16) or bfloat16     */
/*    (SWIFTLLM_HIP_BF16) throughout a call; the cache layout is the one      */
/*    above, block_size 16, head_dim 64 or 128.                               */
/* ------------------------------------------------------------------------ */
#define SWIFTLLM_HIP_F16 0
#define SWIFTLLM_HIP_BF16 1

/* Block tables and slot maps of one step, from request lengths. Sequence s
 * has cached_lens[s] tokens in the cache, in the first ceil(cached / 16)
 * entries of its row of block_tables, and brings new_lens[s] tokens. Its
 * missing blocks are taken from free_blocks in order (sequence by sequence),
 * of which the first min(num_free[0], free_capacity) are there; num_free is
 * device memory. Writes
 *   block_tables[s, ...]   the taken blocks (other entries stay)
 *   context_lens[s]        = cached + new
 *   query_offsets[S + 1]   exclusive sums of the new tokens
 *   positions[t], slot_mapping[t]  of packed token t: its position in its
 *                          sequence and its cache slot (-1 for a block outside
 *                          [0, num_blocks), num_blocks <= 0: no upper bound);
 *                          -1 and -1 for the rows from the last token up to
 *                          num_tokens (padding)
 *   counts[3]              blocks taken, tokens placed, sequences refused
 * A sequence is refused where a length is negative, cached + new does not fit
 * its table, its blocks are missing from the free list or its tokens from
 * num_tokens (both sums run over all sequences before it): it keeps
 * context_lens = cached_lens and no token of it is placed. Blocks past
 * counts[0] were not taken. No output may overlap another argument. */
int swiftllm_hip_plan_step(int32_t* block_tables, const int32_t* cached_lens,
                           const int32_t* new_lens, const int32_t* free_blocks,
                           const int32_t* num_free, int free_capacity,
                           int num_seqs, int max_num_blocks_per_seq,
                           int block_size, int num_tokens, int num_blocks,
                           int32_t* context_lens, int32_t* query_offsets,
                           int32_t* positions, int32_t* slot_mapping,
                           int32_t* counts, hipStream_t stream);

/* Rotary positions of queries and keys, and the cache write of the rotated
 * keys and the values, in one launch. Pair i < rotary_dim / 2 of a head,
 * elements (i, i + rotary_dim / 2) or, interleaved != 0, (2 i, 2 i + 1), turns
 * by positions[t] * inv_freq[i] and is scaled by attn_factor; elements past
 * rotary_dim (even, 0 to head_dim) stay. inv_freq: double
 * [rotary_dim / 2] in device memory, radians per position. query, key and
 * value [T, heads * head_dim] with a stride in elements between tokens (a
 * fused projection is three such views), at most 2^40, and from the first
 * token to the last at most 2^46; query_out [T, num_heads, head_dim]
 * packed, which may be query itself where query_stride is num_heads *
 * head_dim and may overlap no other argument otherwise. Angles are reduced in
 * 64 bits.
 * A token with a negative position is padding: no row of it is written. One
 * whose slot is negative or outside [0, num_blocks * 16) (num_blocks <= 0: no
 * upper bound) has its queries written and nothing else. The slots of a call
 * are distinct. */
int swiftllm_hip_rotary_and_cache(
    void* query_out, const void* query, const void* key, const void* value,
    void* key_cache, void* value_cache, const int32_t* positions,
    const int32_t* slot_mapping, const void* inv_freq, float attn_factor,
    int interleaved, int dtype, int num_tokens, int num_heads,
    int num_kv_heads, int head_dim, int rotary_dim, int block_size,
    long long query_stride, long long key_stride, long long value_stride,
    int num_blocks, hipStream_t stream);

/* Paged attention with shaped scores. A query at position p of sequence s
 * sees key j < context_lens[s] where j <= p and (window == 0 or p - j <
 * window), or where j < prefix_lens[s] (NULL: no prefix): a sliding window of
 * `window` keys, the query's own included, and a prefix that every query
 * sees, in both directions. Its score is
 *   softcap > 0: softcap * tanh(scale q.k / softcap), else scale q.k,
 *   minus alibi_slopes[h] * |p - j| (float [num_heads]; NULL: none).
 * Outputs are the softmax-weighted sums of the seen values with kv head
 * h / (num_heads / num_kv_heads), 32-bit sums rounded once. Blocks whose id is
 * outside [0, num_blocks) (num_blocks <= 0: no upper bound) hold no key, and
 * there are none past max_num_blocks_per_seq * 16: of a longer context the
 * queries keep their positions. A query that sees no key writes zeros. Cache
 * slots that no query of the call sees may hold anything, NaN included. A key
 * that is not finite makes the outputs of the queries that see it NaN or
 * unspecified, a value that is not finite one element of them, or all, not
 * finite; other queries are not touched. dtype is that of query, caches and
 * output; scale and softcap are finite, softcap 0 to 1024. output may be query
 * itself and overlaps no other argument (of caches that is checked where
 * num_blocks is given). */

/* One new token per sequence: the query of sequence s, at position
 * context_lens[s] - 1 (context_lens[s] <= 0: zeros), is row s of query and
 * output [num_seqs, num_heads, head_dim]; with query_offsets [num_seqs + 1]
 * (not NULL, as swiftllm_hip_plan_step writes them) it is the last of the rows
 * query_offsets[s] .. query_offsets[s + 1] - 1 of num_tokens, and a sequence
 * without rows there has no output. `workspace` holds
 * swiftllm_hip_scored_decode_workspace_size() bytes, 256-byte aligned, plain
 * scratch; calls that share one must be ordered on one stream. */
int swiftllm_hip_scored_decode(
    void* output, void* workspace, size_t workspace_bytes, const void* query,
    const void* key_cache, const void* value_cache,
    const int32_t* block_tables, const int32_t* context_lens,
    const int32_t* query_offsets, const float* alibi_slopes,
    const int32_t* prefix_lens, float scale, float softcap, int window,
    int dtype, int num_tokens, int num_seqs, int num_heads, int num_kv_heads,
    int head_dim, int block_size, int max_num_blocks_per_seq, int num_blocks,
    hipStream_t stream);

/* Bytes of workspace it needs for these sizes; 0 where it would refuse them. */
size_t swiftllm_hip_scored_decode_workspace_size(
    int num_seqs, int num_heads, int num_kv_heads, int head_dim,
    int block_size, int max_num_blocks_per_seq);

/* Packed query tokens: rows query_offsets[s] .. query_offsets[s + 1] - 1 of
 * query and output [num_tokens, num_heads, head_dim] are the last tokens of
 * sequence s, at positions up to context_lens[s] - 1, and their keys are in
 * the cache already: whole prompts, or chunks on top of what is cached (the
 * arrays that swiftllm_hip_plan_step writes). query_offsets has num_seqs + 1
 * entries within [0, num_tokens]; a sequence whose offsets are not ascending
 * within it has no rows. If sequences share rows the output is unspecified.
 * Rows of no sequence are left as they were; a row at a negative position is
 * zero. The caches are 16-byte aligned. */
int swiftllm_hip_scored_prefill(
    void* output, const void* query, const void* key_cache,
    const void* value_cache, const int32_t* block_tables,
    const int32_t* context_lens, const int32_t* query_offsets,
    const float* alibi_slopes, const int32_t* prefix_lens, float scale,
    float softcap, int window, int dtype, int num_tokens, int num_seqs,
    int num_heads, int num_kv_heads, int head_dim, int block_size,
    int max_num_blocks_per_seq, int num_blocks, hipStream_t stream);

/* ------------------------------------------------------------------------ */
/* 7. Sequences that come of one another: beams, parallel samples, chats on   */
/*    one prompt. The reference counts references and forks blocks on the     */
/*    host (crates/swiftllm-core/src/memory/block_manager.rs) and has no beam  */
/*    search. As in section 6 nothing synchronises or allocates, all state is  */
/*    device memory, and every call can be captured.                          */
/* ------------------------------------------------------------------------ */
#define SWIFTLLM_HIP_F32 2

/* A beam search's selection. Row r * beam_width + w of logits (dtype F16, BF16
 * or F32; `vocab` values, logits_stride between rows) belongs to beam w of
 * request r, whose sum of log probabilities is beam_scores[row]. The score of
 * going on with token v is beam_scores[row] + log softmax(logits[row])[v], summed
 * and compared in 64 bits; of the softmax's sum the terms within 8192 logits are of
 * 32 bits, which moves all scores of a row alike, by less than 2^-17. Beams' scores
 * closer than that may come in either order. Writes, for every request,
 *   cand_scores, cand_rows, cand_tokens [R, num_candidates]: the largest scores
 *     in descending order (rounded to 32 bits), their rows and tokens; ties go to
 *     the lower beam, then the larger logit, then the lower token
 *   next_scores, next_rows, next_tokens [R, beam_width]: the first of the
 *     candidates whose token is not eos_id (below 0: all go on)
 * Places without a candidate hold -infinity, -1 and -1. A score of -infinity is
 * no candidate: banned tokens (a logit of -infinity, or NaN) and beams without a
 * score (-infinity or NaN; at a request's first step all but one). Where a logit
 * is +infinity, its like share the row. beam_width <= num_candidates <= 64;
 * twice the width leaves every beam a candidate that goes on. next_scores may be
 * beam_scores. `workspace`: plain scratch, 256-byte aligned, of
 * swiftllm_hip_beam_select_workspace_size() bytes; calls that share one must be
 * ordered on one stream. */
int swiftllm_hip_beam_select(
    const void* logits, const float* beam_scores, float* cand_scores,
    int32_t* cand_rows, int32_t* cand_tokens, float* next_scores,
    int32_t* next_rows, int32_t* next_tokens, void* workspace,
    size_t workspace_bytes, int dtype, int num_requests, int beam_width,
    int vocab, int num_candidates, long long logits_stride, int eos_id,
    hipStream_t stream);

/* The same for the rows of a step: one that brought no token, query_offsets[row + 1]
 * <= query_offsets[row] (num_requests * beam_width + 1 entries, as
 * swiftllm_hip_plan_step writes them; NULL: every row did), has no logits and
 * counts as one of a beam without a score. */
int swiftllm_hip_beam_select_rows(
    const void* logits, const float* beam_scores, const int32_t* query_offsets,
    float* cand_scores, int32_t* cand_rows, int32_t* cand_tokens,
    float* next_scores, int32_t* next_rows, int32_t* next_tokens,
    void* workspace, size_t workspace_bytes, int dtype, int num_requests,
    int beam_width, int vocab, int num_candidates, long long logits_stride,
    int eos_id, hipStream_t stream);

/* Bytes of workspace they need for these sizes; 0 where they would refuse them. */
size_t swiftllm_hip_beam_select_workspace_size(int num_requests,
                                               int beam_width, int vocab,
                                               int num_candidates);

/* Tables and references of rows that go on from others. Row i of
 * block_tables_out and context_lens_out continues row parents[i] of
 * block_tables and context_lens (any number that is no row: it ends, with a
 * context of 0). ref_counts[b] is how many rows hold block b, in all tables of
 * the pool; it loses the old rows' holds and gains the new ones'. A partly
 * filled last block is about to be written: the rows whose last block it is, of
 * whatever parents, get a block of their own each, but for the last of them where
 * ref_counts[b], before any copy, counts nobody else. Copies take the lowest blocks that nothing refers to, rows in order; copy_pairs int64
 * [num_seqs][2] holds their (source, destination) for swiftllm_hip_copy_blocks,
 * which has to run before the next token is written, and -1 behind them. A row
 * that finds none loses its last, partly filled block: its context ends with
 * the whole ones. Writes free_blocks[0 .. num_free) = the blocks that nothing
 * refers to then, in ascending order (room for num_blocks; entries behind stay),
 * and counts[2] = copies, rows cut. taken (NULL: none): the first taken[0] of
 * free_blocks as they come in were taken since (counts of
 * swiftllm_hip_plan_step) and get their first reference here. new_lens [num_seqs]
 * (NULL: not wanted): 1 for rows that go on, 0 for those that ended or were cut,
 * which the next swiftllm_hip_plan_step takes. Entries of a row
 * behind its context stay as they were; ids outside [0, num_blocks) are carried
 * along and not counted. No output may overlap another argument. */
int swiftllm_hip_fork_pages(
    int32_t* block_tables_out, int32_t* context_lens_out,
    const int32_t* block_tables, const int32_t* context_lens,
    const int32_t* parents, int32_t* ref_counts, int32_t* free_blocks,
    int32_t* num_free, const int32_t* taken, int64_t* copy_pairs,
    int32_t* new_lens, int32_t* counts, void* workspace,
    size_t workspace_bytes, int num_seqs, int max_num_blocks_per_seq,
    int block_size, int num_blocks, hipStream_t stream);

/* Brings a pool together: the highest block that something refers to moves to
 * the lowest that nothing does, and so on while it lies above it, at most
 * max_moves of them. copy_pairs int64 [max_moves][2] holds the moves for
 * swiftllm_hip_copy_blocks, -1 behind them; new_ids[num_blocks] every block's
 * new id (its own where it stays), block_tables_out the tables with those, which
 * may be block_tables itself, ref_counts_out the references by the new ids,
 * free_blocks[0 .. num_free) the free blocks in ascending order, counts[2] =
 * moves, blocks in use. ref_counts are up to date: blocks that a plan took since
 * have had their reference (swiftllm_hip_fork_pages). Every other holder of a
 * block takes its new id from new_ids. No other output may overlap an argument. */
int swiftllm_hip_compact_pages(
    int32_t* block_tables_out, int32_t* ref_counts_out,
    const int32_t* block_tables, const int32_t* context_lens,
    const int32_t* ref_counts, int32_t* free_blocks, int32_t* num_free,
    int64_t* copy_pairs, int32_t* new_ids, int32_t* counts, void* workspace,
    size_t workspace_bytes, int num_seqs, int max_num_blocks_per_seq,
    int block_size, int num_blocks, int max_moves, hipStream_t stream);

/* The plan of a step's attention over shared blocks, once for all of its layers.
 * Group g is the sequences group_offsets[g] .. group_offsets[g + 1] - 1 (device
 * memory, num_groups + 1 entries ascending within [0, num_seqs]; otherwise no
 * group shares anything); a sequence of no group shares nothing. Writes
 * shared_blocks[g], the leading blocks that every sequence of the group with a
 * context uses, and all of them the same (0 where none has a context), and the
 * plan. It reads a group's blocks once where that saves min_saved blocks of a kv
 * head or more; below 0 where it is the faster way by the library's own rule. The
 * plan: swiftllm_hip_plan_shared_size() bytes, 256-byte aligned, for
 * swiftllm_hip_shared_decode calls with the same sizes, which take the contexts
 * and what is shared from it. */
int swiftllm_hip_plan_shared(void* plan, size_t plan_bytes,
                             int32_t* shared_blocks,
                             const int32_t* block_tables,
                             const int32_t* context_lens,
                             const int32_t* group_offsets, int num_groups,
                             int num_seqs, int num_heads, int num_kv_heads,
                             int head_dim, int block_size,
                             int max_num_blocks_per_seq, int min_saved,
                             hipStream_t stream);

/* Bytes of a plan; 0 where swiftllm_hip_plan_shared would refuse the sizes. */
size_t swiftllm_hip_plan_shared_size(int num_seqs, int num_heads,
                                     int num_kv_heads, int head_dim,
                                     int block_size,
                                     int max_num_blocks_per_seq);

/* swiftllm_hip_scored_decode without windows, where sequences share blocks: the
 * blocks that a group shares are read once for all of its sequences. Contexts are
 * the plan's; block_tables are those that it was made from. A plan of other sizes
 * writes nothing. Values that are not finite and unknown blocks are as there;
 * weights are rounded to dtype, as in swiftllm_hip_scored_prefill. The caches are
 * 16-byte aligned; output overlaps no other argument. `workspace`: plain scratch,
 * 256-byte aligned, of swiftllm_hip_shared_decode_workspace_size() bytes; calls
 * that share one must be ordered on one stream. */
int swiftllm_hip_shared_decode(
    void* output, void* workspace, size_t workspace_bytes, const void* plan,
    size_t plan_bytes, const void* query, const void* key_cache,
    const void* value_cache, const int32_t* block_tables,
    const int32_t* query_offsets, const float* alibi_slopes, float scale,
    float softcap, int dtype, int num_tokens, int num_seqs, int num_heads,
    int num_kv_heads, int head_dim, int block_size, int max_num_blocks_per_seq,
    int num_blocks, hipStream_t stream);

/* Bytes of workspace it needs for these sizes; 0 where it would refuse them. */
size_t swiftllm_hip_shared_decode_workspace_size(
    int num_seqs, int num_heads, int num_kv_heads, int head_dim,
    int block_size, int max_num_blocks_per_seq);

/* Bytes of workspace (plain scratch, 256-byte aligned) that
 * swiftllm_hip_fork_pages and swiftllm_hip_compact_pages need; 0 where they
 * would refuse the sizes. Calls that share one must be ordered on one stream. */
size_t swiftllm_hip_pages_workspace_size(int num_seqs, int num_blocks);

/* ------------------------------------------------------------------------ */
/* 8. Host-side metadata (no device work).                                   */
/* ------------------------------------------------------------------------ */

/* KvCache::get_slot_mapping (crates/swiftllm-core/src/memory/kv_cache.rs:
 * 186-216): out[i] = table[(start + i) / bs] * bs + (start + i) % bs.
 * Returns SWIFTLLM_ERR_INVALID_PARAMETER when a position falls outside the
 * table ("Block ... not allocated") or a slot does not fit in int32. */
int swiftllm_hip_slot_mapping(const uint64_t* block_table, size_t table_len,
                              size_t block_size, size_t start_pos,
                              size_t num_tokens, int32_t* out);

/* Packs per-sequence block tables (Vec<Vec<usize>> in BatchedCacheMetadata,
 * kv_cache.rs:250-286) given in CSR form (table_offsets[num_seqs + 1] into
 * block_ids) into an int32 [num_seqs, max_blocks_per_seq] array padded with
 * 0, and context lengths into int32 [num_seqs]. max_blocks_per_seq must be
 * >= every table length and every ceil(context_len / block_size). */
int swiftllm_hip_pack_block_tables(const uint64_t* block_ids,
                                   const uint64_t* table_offsets,
                                   const uint64_t* context_lens,
                                   size_t num_seqs, size_t block_size,
                                   size_t max_blocks_per_seq,
                                   int32_t* block_tables_out,
                                   int32_t* context_lens_out);

#ifdef __cplusplus
}
#endif

#endif /* SWIFTLLM_HIP_H */
