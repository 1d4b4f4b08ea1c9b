/* Kernel-level C ABI of the B200 speculative-decode library (libg4dense_b200.so).
 *
 * These entry points expose single hot-path operators on caller-owned DEVICE buffers, so a
 * host that already manages CUDA memory can bind them the way the reference's host binds its
 * compute shaders. All pointers are device pointers unless stated otherwise; `stream` is a
 * cudaStream_t (NULL = legacy default stream). Functions return 0 on success or a CUDA error
 * code, with a message in g4b_last_error() (thread-local), mirroring the reference's
 * g4dense_engine_last_error convention (src/c_api.cpp:28-31).
 */
#ifndef G4DENSE_B200_OPS_H
#define G4DENSE_B200_OPS_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define G4B_API __attribute__((visibility("default")))

G4B_API const char* g4b_last_error(void);

/* A prepared INT4 G64 affine matrix. Replaces the reference's weight binding for
 * GemvInt4 / GemmInt4Batch (shaders/GemvInt4.hlsl:24-25, shaders/GemmInt4Batch.hlsl:296-301):
 * W [N][K/8] u32 (nibble c%8 of word c/8, low nibble first), S and B [N][K/64] bf16, all in
 * the container's row-major layout. The matrix is repacked once into the B200 streaming
 * layout; the source buffers may be freed afterwards. K must be a multiple of 64. */
typedef struct g4b_qmat g4b_qmat;
G4B_API int g4b_qmat_create(const uint32_t* W, const uint16_t* S, const uint16_t* B, int N, int K,
                            void* stream, g4b_qmat** out);
G4B_API void g4b_qmat_destroy(g4b_qmat* q);

/* out[m][n] = sum_k (q[n][k] * s + b) * x[m][k] for m < M <= 128: the batched INT4 GEMM
 * (shaders/GemmInt4Batch.hlsl:64-143; M = 1 is GemvInt4, shaders/GemvInt4.hlsl:31-54).
 * M <= 16 runs the HBM-streaming verify GEMM; 17 <= M <= 128 (prefill chunks) the tcgen05
 * tensor-core GEMM. x is fp32 [M][ldx], out fp32 [M][ldo]. Launches two kernels: activation
 * preparation and the GEMM. Calls on one matrix must be stream-ordered (they share the
 * matrix's workspace). */
G4B_API int g4b_qmat_gemm(g4b_qmat* q, const float* x, int ldx, int M, float* out, int ldo, void* stream);
/* The two halves of g4b_qmat_gemm, for timing the GEMM kernel alone. */
G4B_API int g4b_qmat_prepare_input(g4b_qmat* q, const float* x, int ldx, int M, void* stream);
G4B_API int g4b_qmat_run(g4b_qmat* q, int M, float* out, int ldo, void* stream);
/* The verify GEMM kernel (M <= 16) without its in-kernel split-K sum, leaving the partials in
 * the matrix's workspace (for timing the weight stream alone). */
G4B_API int g4b_qmat_run_partial(g4b_qmat* q, int M, void* stream);
/* g4b_qmat_run for M = 1..16 (the verify GEMM only) without any allocation: the same kernel,
 * grid and slot order (bit-identical output), but the split-K scratch -- partial slots and
 * per-row-group arrival counters -- is a fixed static device buffer inside the library (8 MiB of
 * slots, 4096 row groups) instead of the matrix's own workspace. No counterpart in the reference,
 * whose shaders take their scratch from buffers bound by the host. For callers that must not
 * allocate device memory at call time: code running inside a caching allocator's callbacks or on
 * a device whose memory a pool has fully reserved, and latency-sensitive loops where
 * cudaMalloc/cudaFree would synchronize the device.
 *   - Rejects (non-zero return, message in g4b_last_error) M outside 1..16 (17..128 rows need
 *     g4b_qmat_run's tensor-core path), and a matrix whose launch at this M needs more than
 *     8 MiB of slots or more than 4096 row groups (N > 1048576).
 *   - The static buffer lives in a module that CUDA loads lazily; loading it reserves its
 *     device memory. g4b_qmat_create loads it on the matrix's device (it allocates anyway), so
 *     this call itself allocates nothing. It must run on the device the matrix was created on.
 *   - The counters are cleared on `stream` before the launch.
 *   - The scratch is shared by every caller on a device: overlapping calls (other streams,
 *     other threads) race and must be ordered by the caller.
 *   - Not valid across a device or primary-context reset: the cached scratch address dies
 *     with the context. Create the matrix again after a reset. */
G4B_API int g4b_qmat_run_noalloc(g4b_qmat* q, int M, float* out, int ldo, void* stream);
/* Synchronizes and reports whether any launch on q hit a bounded-wait timeout. */
G4B_API int g4b_qmat_check_error(g4b_qmat* q);
/* INT8 G64 affine GEMV, the reference's GemvInt8 (shaders/GemvInt8.hlsl:13-33, row dot
 * shaders/Common.hlsli:225-269): out[r] = sum_k (W[r][k] * s + b) * x[k] for r < rows, with W
 * [rows][K] u8, S and B [rows][K/64] bf16, x [K] fp32, out [rows] fp32. K a multiple of 64; W and
 * x 16-byte aligned. */
G4B_API int g4b_gemv_int8(const uint8_t* W, const uint16_t* S, const uint16_t* B, const float* x, float* out,
                          int rows, int K, void* stream);
/* Attention output gate, the reference's AttnGate (shaders/AttnGate.hlsl:15-32):
 * out[m][c] = ctx[m][c] * sigmoid(gate[m][c]) for c < n, m < batch; strides in floats. */
G4B_API int g4b_attn_gate(const float* ctx, const float* gate, float* out, int n, int batch, int ctx_stride,
                          int gate_stride, int out_stride, void* stream);
/* Token sampling on a device logits row, the reference's sample_token (src/sampling.cpp:92-169):
 * greedy argmax (ties to the lowest index) when temperature <= 0; otherwise the top_k (or 256)
 * largest logits, a top-p cut measured against the full-vocabulary softmax, and a
 * temperature-scaled draw with the xorshift64* generator seeded with `seed` (the caller derives it
 * as the reference's seed_for does, src/sampling.cpp:63-72). logits: fp32 [vocab] device memory,
 * vocab <= 262144; top_k 0..256 (0 = 256-wide shortlist); top_p in (0, 1]. `workspace` is
 * g4b_sample_workspace() bytes of device memory, used by one stream at a time; the token is
 * written to out_token (device memory). Two kernel launches. */
G4B_API size_t g4b_sample_workspace(void);
G4B_API int g4b_sample_token(const float* logits, int vocab, float temperature, float top_p, int top_k,
                             uint64_t seed, void* workspace, uint32_t* out_token, void* stream);
/* out4 = {N, K, grid CTAs at M=5, split-K slots per row group} */
G4B_API int g4b_qmat_info(const g4b_qmat* q, int* out4);

/* ---------------------------------------------------------------------------------------------
 * Batched tree verification over a paged K/V cache. The reference verifies one sequence's chain of
 * drafts over a contiguous ring (src/speculator.cpp, src/kv_cache.cpp) and has no counterpart of
 * these; they are what a server needs to run the same round for many sequences at once, each with
 * a tree of drafts:
 *
 *   g4b_tree_attention   every layer: the nodes over their sequence's pages and their ancestors
 *   g4b_sample_rows      one token per node from its logits row and a given uniform number
 *   g4b_tree_accept      the path along the drawn tokens
 *   g4b_pages_reserve    pages for the accepted rows
 *   g4b_pages_commit     the accepted nodes' K/V rows into those pages
 *   g4b_pages_fork / _free / _compact / _copy   sharing, releasing and moving pages
 *
 * A round needs no host synchronization: lengths, counts and tables stay on the device. All calls
 * are asynchronous on `stream`, a stream of the current device, on which all arrays have to be; they
 * allocate nothing, and can be captured in a CUDA graph. Array
 * arguments are device memory; indices that a call finds out of range on the device are never
 * followed: what they name is skipped (in the attention, a page id out of range reads as zeros).
 * Calls that write a `status` word leave the state as it was when it is not 0. */

typedef enum { G4B_BF16 = 0, G4B_FP16 = 1, G4B_FP32 = 2 } g4b_dtype;

/* Attention of drafted trees. Sequence s has cu_nodes[s + 1] - cu_nodes[s] nodes (0 to max_nodes),
 * node 0 its pending token, and lens[s] cached tokens, position j of which is row j % page_size of
 * page table[s][j / page_size]. Node i sits at position lens[s] + depth[i] and sees every cached
 * key and those nodes j of its own sequence whose bit (j % 32) is set in word j / 32 of its mask
 * row; a window w > 0 hides keys w or more positions before the node. With one node per sequence
 * this is decoding attention; with a lower-triangular mask, a chunk of a prompt.
 *   out[i][h] = sum_j p_j v_j[h / g],  p = softmax_j(scale * q[i][h] . k_j[h / g]),  g = heads / kv_heads
 * A node that sees no key gets zeros. Values behind a hidden key, past lens[s] in a page, or in
 * another sequence are never used, whatever they are (NaN and infinities included). Softmax and
 * sums are fp32; the probabilities are rounded to the cache's type before the product with V.
 * scale > 0; head_dim 64, 128, 256 or 512; page_size a multiple of 8; max_nodes 1..256; dtype G4B_BF16 or
 * G4B_FP16 for q, K, V and out alike; pointers 16-byte aligned, strides multiples of 8 elements. */
typedef struct g4b_tree_attention_args {
    const void* q;            /* [n_tokens][heads][head_dim] */
    const void* k_pool;       /* [n_pages][page_size][kv_heads][head_dim] */
    const void* v_pool;
    const void* k_new;        /* [n_tokens][kv_heads][head_dim]: the nodes' own keys and values */
    const void* v_new;
    void* out;                /* [n_tokens][heads][head_dim] */
    const int32_t* table;     /* [n_seqs][table_width] */
    const int32_t* lens;      /* [n_seqs] */
    const int32_t* cu_nodes;  /* [n_seqs + 1] */
    const uint32_t* mask;     /* [n_tokens][mask_words], mask_words >= (max_nodes + 31) / 32 */
    const int32_t* depth;     /* [n_tokens], below the tree's node count; may be NULL when window is 0 */
    void* workspace;          /* g4b_tree_attention_workspace() bytes, used by one stream at a time */
    size_t workspace_bytes;
    int64_t q_stride, out_stride, new_stride;  /* elements from one token to the next */
    int64_t page_stride;                       /* elements from one page of a pool to the next */
    int n_seqs, n_tokens, max_nodes, n_pages, page_size, table_width, mask_words;
    int heads, kv_heads, head_dim, window, dtype;
    float scale;
} g4b_tree_attention_args;
/* 0 when the shape is not supported. */
G4B_API size_t g4b_tree_attention_workspace(int max_nodes, int heads, int kv_heads, int head_dim);
G4B_API int g4b_tree_attention(const g4b_tree_attention_args* args, void* stream);
/* Waits for all streams of the current device and reports whether a launch on it hit a bounded-wait
 * timeout since the last call. */
G4B_API int g4b_tree_attention_check_error(void);

/* One token per logits row. With l the row, m its maximum and T = temperature[r], entries are
 * weighted exp((l - m) / T), held as whole multiples of 2^-40 so that sums are exact and the draw
 * does not depend on their order. In descending order of l (ties to the lower index) the kept
 * entries are the top_k[r] first (0: all), of those the smallest prefix that holds top_p[r] of
 * their mass (1: all), of those the ones whose weight is at least min_p[r] of the maximum's. The
 * token is the first kept entry in index order at which the running kept mass exceeds uniform[r]
 * times the whole. temperature <= 0 picks the maximum. NaN and -inf are never kept; a row without
 * any other entry gives token -1, probability 0. prob (may be NULL) receives the token's share of
 * the kept mass, kept (may be NULL) their number. Any of temperature, top_k, top_p and min_p may
 * be NULL (1, 0, 1, 0); a top_p or min_p of NaN is off, a temperature of NaN picks the maximum. Differs
 * from g4b_sample_token, which keeps the reference's order and its 256-entry bound. vocab 1..262144; stride in elements; dtype any g4b_dtype. One kernel launch. */
G4B_API int g4b_sample_rows(const void* logits, int dtype, int rows, int vocab, int64_t stride,
                            const float* uniform, const float* temperature, const int32_t* top_k,
                            const float* top_p, const float* min_p, int32_t* token, float* prob, int32_t* kept,
                            void* stream);

/* Walks each sequence's tree: from node 0 to the lowest child whose token is the one drawn at the
 * current node (sampled[]), as long as there is one. parents[i] is relative to the sequence's
 * first node, and smaller than i. path[s] receives the accepted nodes (relative, -1 behind the
 * last; at most path_width), count[s] their number, next[s] the token drawn at the last of them,
 * which becomes the next round's pending token. A sequence without nodes gets count 0, next -1.
 * At most 256 nodes a sequence. */
G4B_API int g4b_tree_accept(const int32_t* tokens, const int32_t* parents, const int32_t* sampled,
                            const int32_t* cu_nodes, int n_seqs, int n_tokens, int32_t* path, int path_width,
                            int32_t* count, int32_t* next, void* stream);

/* A pool of pages: n_planes planes (one per layer's K and V) of n_pages pages of page_size rows of
 * row_bytes bytes. Base and strides multiples of 16 bytes; the rows of one page are contiguous. */
typedef struct g4b_page_pool {
    void* base;
    int64_t plane_stride, page_stride; /* bytes */
    int n_planes, n_pages, page_size, row_bytes;
} g4b_page_pool;

/* The keeping of n_seqs (up to 4096) sequences' pages: refs [n_pages] (up to 2^24) counts how many
 * sequences hold a page (0: free), table [n_seqs][table_width] (below 2^31 cells) lists each sequence's
 * pages (-1: none), lens [n_seqs] its tokens. Each call reads refs, table and lens and writes refs_out,
 * table_out and lens_out (those it changes), which may be the same arrays. New pages are the free pages
 * of lowest id, in (sequence, position) order: results depend on the state alone. status: 0 done, 1 too
 * few free pages, 2 more pages than the table row holds (or a negative length), 3 a bad sequence index,
 * 4 a page id out of range in the table, the largest where several hold; the outputs then equal the
 * inputs. */
typedef struct g4b_page_tables {
    const int32_t *refs, *table, *lens;
    int32_t *refs_out, *table_out, *lens_out;
    int n_pages, n_seqs, table_width, page_size;
} g4b_page_tables;

/* Fills the empty table entries that sequence s needs to hold lens[s] + grow[s] tokens. */
G4B_API int g4b_pages_reserve(const g4b_page_tables* t, const int32_t* grow, int32_t* status, void* stream);
/* dst[i] (an empty sequence, named once) becomes a continuation of src[i]: full pages are shared, a
 * partial last page is copied to a page of its own in every plane, so each sequence only ever
 * writes rows of pages that it alone holds. */
G4B_API int g4b_pages_fork(const g4b_page_pool* pool, const g4b_page_tables* t, const int32_t* src,
                           const int32_t* dst, int n, int32_t* status, void* stream);
/* Releases the pages of the n sequences seqs[] and empties them. */
G4B_API int g4b_pages_free(const g4b_page_tables* t, const int32_t* seqs, int n, void* stream);
/* Moves live pages so that they fill ids 0 .. live - 1: the k-th live page at or past `live` goes to
 * the k-th free page before it. moves [1 + 2 * n_pages] receives their number and the (from, to)
 * pairs, -1 behind them. lens is not read. */
G4B_API int g4b_pages_compact(const g4b_page_pool* pool, const g4b_page_tables* t, int32_t* moves, void* stream);
/* Page src[i] of one pool to page dst[i] of another (same planes, page_size and row_bytes), or of
 * the same one when no page is both a source and a destination. */
G4B_API int g4b_pages_copy(const g4b_page_pool* from, const g4b_page_pool* to, const int32_t* src,
                           const int32_t* dst, int n, void* stream);
/* Writes rows [n_planes][n_tokens][row_bytes] (plane stride rows_plane_stride bytes) of sequence s's
 * nodes path[s][0 .. count[s]) (NULL path: the first count[s]) at positions lens[s] onwards of its
 * pages, and lens_out[s] = lens[s] + count[s]. A row whose node is not one of the sequence's own, or
 * whose position has no page, ends that sequence's commit: the rows ahead of it are written, and the
 * length grows by those alone. status (may be NULL) is g4b_pages_reserve's: nothing is committed
 * unless it is 0. */
G4B_API int g4b_pages_commit(const g4b_page_pool* pool, const int32_t* table, int table_width, const int32_t* lens,
                             int n_seqs, const void* rows, int64_t rows_plane_stride, int n_tokens,
                             const int32_t* cu_nodes, const int32_t* path, int path_width, const int32_t* count,
                             const int32_t* status, int32_t* lens_out, void* stream);

#ifdef __cplusplus
}
#endif
#endif
