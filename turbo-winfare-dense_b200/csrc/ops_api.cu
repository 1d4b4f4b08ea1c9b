// Kernel-level C ABI (include/g4dense_b200_ops.h): prepared INT4 G64 matrices and the
// verify GEMM on caller-owned device buffers.
#include "g4dense_b200_ops.h"

#include <climits>
#include <cstdio>
#include <mutex>
#include <string>

#include "common.cuh"
#include "kernels.h"
#include "pages.h"
#include "pgemm.h"
#include "sample_rows.h"
#include "tree_attn.h"
#include "vgemm.h"

namespace {
thread_local std::string g_err;
int fail(cudaError_t e, const char* where) {
    g_err = std::string(where) + ": " + cudaGetErrorString(e);
    return (int)e;
}
int fail_msg(const char* msg) {
    g_err = msg;
    return (int)cudaErrorInvalidValue;
}
}  // namespace

namespace {
// Library-owned split-K scratch of g4b_qmat_run_noalloc: 8 MiB of partial slots and one
// arrival counter per 256-row group. Static device memory is part of the module image, so
// using it allocates nothing at call time.
constexpr size_t kNoAllocPartFloats = (size_t)2 << 20;  // 8 MiB
constexpr int kNoAllocCounters = 4096;                 // N <= 4096 * 256 rows
__device__ __align__(256) float g_noalloc_part[kNoAllocPartFloats];
__device__ __align__(256) unsigned g_noalloc_cnt[kNoAllocCounters];

struct NoAllocScratch {
    float* part = nullptr;
    unsigned* cnt = nullptr;
};
constexpr int kMaxDevices = 64;
std::mutex g_noalloc_mu;
NoAllocScratch g_noalloc[kMaxDevices];  // symbol addresses per device ordinal

// Looks up the device addresses of the static scratch on `dev` (the current device) and caches
// them. The first lookup on a device loads the module holding the arrays, which reserves their
// device memory; g4b_qmat_create calls this so that the no-alloc call itself never does. A
// later lookup allocates nothing and refreshes the cache (the addresses are only valid for the
// primary context they were taken in).
cudaError_t noalloc_scratch_setup(int dev) {
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    void* part = nullptr;
    void* cnt = nullptr;
    cudaError_t e;
    if ((e = cudaGetSymbolAddress(&part, g_noalloc_part)) != cudaSuccess) return e;
    if ((e = cudaGetSymbolAddress(&cnt, g_noalloc_cnt)) != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(g_noalloc_mu);
    g_noalloc[dev].part = static_cast<float*>(part);
    g_noalloc[dev].cnt = static_cast<unsigned*>(cnt);
    return cudaSuccess;
}
}  // namespace

struct g4b_qmat {
    int N, K, ktiles, n_wrg, n_crg;
    void* w;          // repacked weights
    void* bfrag;      // B fragments for one input of up to 16 rows
    float* part;      // split-K partials
    unsigned* cnt;    // split-K arrival counters [n_crg], zero between launches
    int max_slots;    // slots per row group sized for every M
    int* err;         // device error word of the bounded waits
    // prefill GEMM (17..128 rows): its weight layout, split-K slots and tile counters
    void* pw;
    float* ppart;
    unsigned* pcnt;
    int n_tiles, pmax_slots;
    int dev;          // device the matrix lives on
};

extern "C" {

const char* g4b_last_error(void) { return g_err.c_str(); }

int g4b_qmat_create(const uint32_t* W, const uint16_t* S, const uint16_t* B, int N, int K, void* stream,
                    g4b_qmat** out) {
    if (!out || !W || !S || !B || N <= 0 || K <= 0 || K % 64) return fail_msg("g4b_qmat_create: bad arguments");
    cudaStream_t st = (cudaStream_t)stream;
    int dev = 0;
    cudaError_t e0 = cudaGetDevice(&dev);
    if (e0 != cudaSuccess) return fail(e0, "g4b_qmat_create: cudaGetDevice");
    // Loads the module that holds g4b_qmat_run_noalloc's static scratch on this device now,
    // while allocating is allowed: under lazy module loading the first symbol lookup reserves
    // that module's device memory.
    if ((e0 = noalloc_scratch_setup(dev)) != cudaSuccess) return fail(e0, "g4b_qmat_create: static scratch set-up");
    auto* q = new g4b_qmat{};
    q->dev = dev;
    q->N = N;
    q->K = K;
    q->ktiles = vgemm_ktiles(K);
    q->n_wrg = (N + 63) / 64;
    q->n_crg = vgemm_n_crg(N);
    cudaError_t e;
    if ((e = cudaMalloc(&q->w, vgemm_weight_bytes(N, K))) != cudaSuccess) { delete q; return fail(e, "cudaMalloc(weights)"); }
    if ((e = g4b_repack(W, S, B, N, K, q->w, st)) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "repack"); }
    const int Kp = q->ktiles * 128;
    if ((e = cudaMalloc(&q->bfrag, g4b::bfrag_capacity(Kp))) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "cudaMalloc(bfrag)"); }
    q->max_slots = vgemm_plan_slots(q->n_crg, q->ktiles);
    const size_t part_bytes = (size_t)q->n_crg * q->max_slots * g4b::kMaxM * 256 * sizeof(float);
    if ((e = cudaMalloc(&q->part, part_bytes)) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "cudaMalloc(part)"); }
    if ((e = cudaMalloc(&q->cnt, q->n_crg * sizeof(unsigned))) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "cudaMalloc(cnt)"); }
    if ((e = cudaMemsetAsync(q->cnt, 0, q->n_crg * sizeof(unsigned), st)) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "memset"); }
    if ((e = cudaMalloc(&q->err, sizeof(int))) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "cudaMalloc(err)"); }
    q->n_tiles = pgemm_n_tiles(N);
    q->pmax_slots = pgemm_max_slots(q->n_tiles, K / 64, pgemm_grid(q->n_tiles, K / 64));
    if ((e = cudaMalloc(&q->pw, pgemm_weight_bytes(N, K))) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "cudaMalloc(prefill weights)"); }
    if ((e = pgemm_repack(W, S, B, N, K, q->pw, st)) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "prefill repack"); }
    if ((e = cudaMalloc(&q->ppart, pgemm_part_floats(q->n_tiles, q->pmax_slots) * sizeof(float))) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "cudaMalloc(prefill part)"); }
    if ((e = cudaMalloc(&q->pcnt, q->n_tiles * sizeof(unsigned))) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "cudaMalloc(prefill cnt)"); }
    if ((e = cudaMemsetAsync(q->pcnt, 0, q->n_tiles * sizeof(unsigned), st)) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "memset"); }
    if ((e = cudaMemsetAsync(q->err, 0, sizeof(int), st)) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "memset"); }
    if ((e = cudaStreamSynchronize(st)) != cudaSuccess) { g4b_qmat_destroy(q); return fail(e, "g4b_qmat_create"); }
    *out = q;
    return 0;
}

void g4b_qmat_destroy(g4b_qmat* q) {
    if (!q) return;
    cudaFree(q->w);
    cudaFree(q->bfrag);
    cudaFree(q->part);
    cudaFree(q->cnt);
    cudaFree(q->err);
    cudaFree(q->pw);
    cudaFree(q->ppart);
    cudaFree(q->pcnt);
    delete q;
}

int g4b_qmat_prepare_input(g4b_qmat* q, const float* x, int ldx, int M, void* stream) {
    if (!q || !x || M < 1 || M > g4b::kPrefillRows || ldx < q->K)
        return fail_msg("g4b_qmat_prepare_input: bad arguments");
    cudaError_t e = g4b_bfrag_from_f32(x, ldx, M, q->K, q->bfrag, (cudaStream_t)stream, false);
    return e == cudaSuccess ? 0 : fail(e, "bfrag_from_f32");
}

static PartView qmat_view(const g4b_qmat* q, int M) {
    PartView v;
    v.part = q->part;
    v.max_slots = q->max_slots;
    v.n_crg = q->n_crg;
    v.ktiles = q->ktiles;
    v.grid = vgemm_grid(M, q->n_crg, q->ktiles);
    return v;
}

static VgemmParams qmat_params(g4b_qmat* q, int M) {
    const g4b::BFragView v = g4b::bfrag_view(q->bfrag, q->ktiles * 128, M);
    VgemmParams p{};
    p.w = q->w;
    p.bfrag = v.frag;
    p.gsum = v.gsum;
    p.out = qmat_view(q, M);
    p.N = q->N;
    p.M = M;
    p.n_wrg = q->n_wrg;
    p.err = q->err;
    return p;
}

// GEMM kernel without its split-K sum: leaves the partials in the matrix's workspace.
int g4b_qmat_run_partial(g4b_qmat* q, int M, void* stream) {
    if (!q || M < 1 || M > g4b::kMaxM) return fail_msg("g4b_qmat_run_partial: bad arguments");
    cudaError_t e = vgemm_launch(qmat_params(q, M), (cudaStream_t)stream, false);
    return e == cudaSuccess ? 0 : fail(e, "vgemm_launch");
}

int g4b_qmat_run(g4b_qmat* q, int M, float* out, int ldo, void* stream) {
    if (!q || !out || M < 1 || M > g4b::kPrefillRows || ldo < q->N) return fail_msg("g4b_qmat_run: bad arguments");
    if (M > g4b::kMaxM) {
        PgemmParams pp{};
        pp.w = q->pw;
        pp.act = q->bfrag;
        pp.g_layout = q->ktiles * 2;
        pp.y = out;
        pp.ldy = ldo;
        pp.part = q->ppart;
        pp.cnt = q->pcnt;
        pp.N = q->N;
        pp.K = q->K;
        pp.M = M;
        pp.n_tiles = q->n_tiles;
        pp.max_slots = q->pmax_slots;
        pp.err = q->err;
        cudaError_t e = pgemm_launch(pp, (cudaStream_t)stream, false);
        return e == cudaSuccess ? 0 : fail(e, "pgemm_launch");
    }
    VgemmParams p = qmat_params(q, M);
    p.y = out;
    p.ldy = ldo;
    p.cnt = q->cnt;
    cudaError_t e = vgemm_launch(p, (cudaStream_t)stream, false);
    return e == cudaSuccess ? 0 : fail(e, "vgemm_launch");
}

// ---------------------------------------------------------------- allocation-free run


int g4b_qmat_run_noalloc(g4b_qmat* q, int M, float* out, int ldo, void* stream) {
    if (!q || !out || ldo < q->N) return fail_msg("g4b_qmat_run_noalloc: bad arguments");
    if (M < 1 || M > g4b::kMaxM)
        return fail_msg("g4b_qmat_run_noalloc: M must be 1..16 (the verify GEMM only; 17..128 rows need "
                        "g4b_qmat_run's tensor-core path and its allocated workspace)");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fail(e, "g4b_qmat_run_noalloc: cudaGetDevice");
    if (dev != q->dev) return fail_msg("g4b_qmat_run_noalloc: the current device is not the matrix's device");
    NoAllocScratch sc;
    {
        std::lock_guard<std::mutex> lock(g_noalloc_mu);
        sc = g_noalloc[dev];
    }
    if (!sc.part) return fail_msg("g4b_qmat_run_noalloc: static scratch not set up on this device");
    VgemmParams p = qmat_params(q, M);
    // Exactly the slots this launch needs (the matrix's own workspace is sized for every M).
    const int slots = vgemm_max_slots(p.out.grid, q->n_crg, q->ktiles);
    const size_t need = (size_t)q->n_crg * slots * g4b::kMaxM * 256;
    if (need > kNoAllocPartFloats || q->n_crg > kNoAllocCounters) {
        char msg[256];
        std::snprintf(msg, sizeof msg,
                      "g4b_qmat_run_noalloc: this matrix needs %.1f MiB of split-K scratch at M = %d (%d row groups x "
                      "%d slots); the static buffer holds 8 MiB and %d row groups -- use g4b_qmat_run",
                      need * 4.0 / (1 << 20), M, q->n_crg, slots, kNoAllocCounters);
        return fail_msg(msg);
    }
    p.out.part = sc.part;
    p.out.max_slots = slots;
    p.y = out;
    p.ldy = ldo;
    p.cnt = sc.cnt;
    const cudaStream_t st = (cudaStream_t)stream;
    // The arrival counters must start at zero; a complete launch leaves them at zero, a failed
    // one may not, so they are cleared on the stream first.
    if ((e = cudaMemsetAsync(sc.cnt, 0, (size_t)q->n_crg * sizeof(unsigned), st)) != cudaSuccess)
        return fail(e, "g4b_qmat_run_noalloc: clearing counters");
    e = vgemm_launch(p, st, false);
    return e == cudaSuccess ? 0 : fail(e, "g4b_qmat_run_noalloc: vgemm_launch");
}

int g4b_qmat_gemm(g4b_qmat* q, const float* x, int ldx, int M, float* out, int ldo, void* stream) {
    int rc = g4b_qmat_prepare_input(q, x, ldx, M, stream);
    return rc ? rc : g4b_qmat_run(q, M, out, ldo, stream);
}

int g4b_qmat_info(const g4b_qmat* q, int* out4) {
    if (!q || !out4) return fail_msg("g4b_qmat_info: bad arguments");
    out4[0] = q->N;
    out4[1] = q->K;
    out4[2] = vgemm_grid(5, q->n_crg, q->ktiles);
    out4[3] = q->max_slots;
    return 0;
}

int g4b_gemv_int8(const uint8_t* W, const uint16_t* S, const uint16_t* B, const float* x, float* out, int rows,
                  int K, void* stream) {
    if (!W || !S || !B || !x || !out || rows <= 0 || K <= 0 || K % 64)
        return fail_msg("g4b_gemv_int8: bad arguments (K must be a positive multiple of 64)");
    if ((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(x)) & 15)
        return fail_msg("g4b_gemv_int8: W and x must be 16-byte aligned");
    const cudaError_t e = g4b::gemv_int8_launch(W, S, B, x, out, rows, K, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_gemv_int8");
}

int g4b_attn_gate(const float* ctx, const float* gate, float* out, int n, int batch, int ctx_stride, int gate_stride,
                  int out_stride, void* stream) {
    if (!ctx || !gate || !out || n <= 0 || batch < 0 || ctx_stride < n || gate_stride < n || out_stride < n)
        return fail_msg("g4b_attn_gate: bad arguments");
    if (batch == 0) return 0;
    const cudaError_t e =
        g4b::attn_gate_launch(ctx, gate, out, n, batch, ctx_stride, gate_stride, out_stride, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_attn_gate");
}

size_t g4b_sample_workspace(void) { return g4b_sample_workspace_bytes(); }

int g4b_sample_token(const float* logits, int vocab, float temperature, float top_p, int top_k, uint64_t seed,
                     void* workspace, uint32_t* out_token, void* stream) {
    if (!logits || !workspace || vocab < 1 || vocab > 262144 || top_k < 0 || top_k > 256 || !(top_p > 0.f) ||
        top_p > 1.f || !(temperature >= 0.f))
        return fail_msg("g4b_sample_token: bad arguments (vocab 1..262144, top_k 0..256, top_p in (0, 1], "
                        "temperature >= 0)");
    const cudaError_t e = g4b_sample_launch(logits, vocab, temperature, top_p, top_k, seed, workspace, out_token,
                                            static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? 0 : fail(e, "g4b_sample_token");
}

// ---------------------------------------------------------------- tree verification, paged cache

size_t g4b_tree_attention_workspace(int max_nodes, int heads, int kv_heads, int head_dim) {
    if (max_nodes < 1 || max_nodes > 256 || kv_heads < 1 || heads < kv_heads || heads % kv_heads ||
        (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512) ||
        (int64_t)heads * (head_dim > max_nodes ? head_dim : max_nodes) > INT32_MAX - 256)  // 32-bit offsets and rows
        return 0;
    return g4b::tree_attn_workspace(max_nodes, heads, kv_heads, head_dim);
}

int g4b_tree_attention(const g4b_tree_attention_args* x, void* stream) {
    if (!x) return fail_msg("g4b_tree_attention: null arguments");
    const size_t need = g4b_tree_attention_workspace(x->max_nodes, x->heads, x->kv_heads, x->head_dim);
    if (!need)
        return fail_msg("g4b_tree_attention: max_nodes must be 1..256, heads a multiple of kv_heads and head_dim 64, "
                        "128, 256 or 512");
    if (x->dtype != G4B_BF16 && x->dtype != G4B_FP16)
        return fail_msg("g4b_tree_attention: dtype must be G4B_BF16 or G4B_FP16");
    if (x->n_seqs < 0 || x->n_tokens < 0 || x->n_pages < 1 || x->table_width < 1 || x->window < 0)
        return fail_msg("g4b_tree_attention: negative or empty sizes");
    if (x->page_size < 8 || x->page_size % 8 || (int64_t)x->page_size * x->table_width > INT32_MAX - 1024)
        return fail_msg("g4b_tree_attention: page_size must be a multiple of 8, and page_size * table_width fit 31 bits");
    if (x->mask_words < (x->max_nodes + 31) / 32)
        return fail_msg("g4b_tree_attention: mask_words must hold max_nodes bits");
    const int64_t row = (int64_t)x->kv_heads * x->head_dim, qrow = (int64_t)x->heads * x->head_dim;
    if (x->q_stride < qrow || x->out_stride < qrow || x->new_stride < row || x->page_stride < row * x->page_size ||
        ((x->q_stride | x->out_stride | x->new_stride | x->page_stride) & 7))
        return fail_msg("g4b_tree_attention: strides must cover a row and be multiples of 8 elements");
    if (!(x->scale > 0.f) || x->scale > 1e30f) return fail_msg("g4b_tree_attention: scale must be positive");
    if (x->n_seqs == 0 || x->n_tokens == 0) return 0;
    if (!x->q || !x->k_pool || !x->v_pool || !x->k_new || !x->v_new || !x->out || !x->table || !x->lens ||
        !x->cu_nodes || !x->mask || !x->workspace || (x->window && !x->depth))
        return fail_msg("g4b_tree_attention: null pointer");
    if ((reinterpret_cast<uintptr_t>(x->q) | reinterpret_cast<uintptr_t>(x->k_pool) |
         reinterpret_cast<uintptr_t>(x->v_pool) | reinterpret_cast<uintptr_t>(x->k_new) |
         reinterpret_cast<uintptr_t>(x->v_new) | reinterpret_cast<uintptr_t>(x->out) |
         reinterpret_cast<uintptr_t>(x->workspace)) & 15)
        return fail_msg("g4b_tree_attention: q, K, V, out and workspace must be 16-byte aligned");
    if (x->workspace_bytes < need) return fail_msg("g4b_tree_attention: workspace too small");
    g4b::TreeAttnArgs a{};
    a.q = x->q;
    a.k_pool = x->k_pool;
    a.v_pool = x->v_pool;
    a.k_new = x->k_new;
    a.v_new = x->v_new;
    a.out = x->out;
    a.table = x->table;
    a.lens = x->lens;
    a.cu = x->cu_nodes;
    a.mask = x->mask;
    a.depth = x->depth;
    a.work = x->workspace;
    a.q_stride = x->q_stride;
    a.page_stride = x->page_stride;
    a.new_stride = x->new_stride;
    a.out_stride = x->out_stride;
    a.seqs = x->n_seqs;
    a.n_tokens = x->n_tokens;
    a.max_nodes = x->max_nodes;
    a.pages = x->n_pages;
    a.page_size = x->page_size;
    a.width = x->table_width;
    a.mask_words = x->mask_words;
    a.heads = x->heads;
    a.kv_heads = x->kv_heads;
    a.dim = x->head_dim;
    a.window = x->window;
    a.bf16 = x->dtype == G4B_BF16;
    a.scale = x->scale;
    if (!g4b::tree_attn_countable(a))
        return fail_msg("g4b_tree_attention: 128-key tiles are counted in 32 bits: n_seqs * kv_heads * page_size * "
                        "table_width is too large");
    const cudaError_t e = g4b::tree_attn_launch(a, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_tree_attention");
}

int g4b_tree_attention_check_error(void) {
    const int e = g4b::tree_attn_error();
    if (e < 0) return fail(cudaGetLastError(), "g4b_tree_attention_check_error");
    if (e) return fail_msg("g4b_tree_attention: a bounded wait gave up (keys or values never arrived)");
    return 0;
}

int g4b_sample_rows(const void* logits, int dtype, int rows, int vocab, int64_t stride, const float* uniform,
                    const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                    int32_t* token, float* prob, int32_t* kept, void* stream) {
    if (dtype < G4B_BF16 || dtype > G4B_FP32 || rows < 0 || rows > (1 << 26) || vocab < 1 ||
        vocab > g4b::kSampleRowsVocab || stride < vocab)
        return fail_msg("g4b_sample_rows: bad arguments (dtype bf16, fp16 or fp32, vocab 1..262144, stride >= vocab)");
    if (rows == 0) return 0;
    if (!logits || !uniform || !token) return fail_msg("g4b_sample_rows: null pointer");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == G4B_FP32 ? 4 : 2))
        return fail_msg("g4b_sample_rows: logits are not aligned to their type");
    g4b::SampleRowsArgs a{logits, uniform, temperature, top_k, top_p, min_p, token, prob, kept, stride, rows, vocab, dtype};
    const cudaError_t e = g4b::sample_rows_launch(a, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_sample_rows");
}

int g4b_tree_accept(const int32_t* tokens, const int32_t* parents, const int32_t* sampled, const int32_t* cu_nodes,
                    int n_seqs, int n_tokens, int32_t* path, int path_width, int32_t* count, int32_t* next,
                    void* stream) {
    if (n_seqs < 0 || n_tokens < 0 || path_width < 1) return fail_msg("g4b_tree_accept: bad sizes");
    if (n_seqs == 0) return 0;
    if (!cu_nodes || !path || !count || !next || (n_tokens && (!tokens || !parents || !sampled)))
        return fail_msg("g4b_tree_accept: null pointer");
    const cudaError_t e = g4b::tree_accept(tokens, parents, sampled, cu_nodes, n_seqs, n_tokens, path, path_width,
                                           count, next, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_tree_accept");
}

namespace {
const char* bad_pool(const g4b_page_pool* p) {
    if (!p || !p->base) return "null pool";
    if (p->n_planes < 1 || p->n_pages < 1 || p->n_pages > (1 << 24) || p->page_size < 1 || p->row_bytes < 16)
        return "pool sizes must be positive (at most 2^24 pages)";
    if ((reinterpret_cast<uintptr_t>(p->base) & 15) || (p->row_bytes & 15) || (p->plane_stride & 15) ||
        (p->page_stride & 15))
        return "pool base, strides and row_bytes must be multiples of 16 bytes";
    if (p->page_stride < (int64_t)p->page_size * p->row_bytes) return "page_stride must cover a page";
    return nullptr;
}
const char* bad_tables(const g4b_page_tables* t, bool lens, bool lens_out) {
    if (!t || !t->refs || !t->table || !t->refs_out || !t->table_out || (lens && !t->lens) ||
        (lens_out && !t->lens_out))
        return "null tables";
    if (t->n_pages < 1 || t->n_pages > (1 << 24) || t->n_seqs < 1 || t->n_seqs > g4b::kMaxPageSeqs ||
        t->table_width < 1 || t->page_size < 1 || (int64_t)t->table_width * t->page_size > INT32_MAX)
        return "sizes out of range (1..4096 sequences, at most 2^24 pages, table_width * page_size in 31 bits)";
    if ((int64_t)t->n_seqs * t->table_width > INT32_MAX) return "a table of 2^31 cells or more";  // counts are 32 bits
    return nullptr;
}
g4b::PagePool pool_of(const g4b_page_pool* p) {
    return {static_cast<char*>(p->base), p->plane_stride, p->page_stride, p->n_planes, p->n_pages, p->page_size,
            p->row_bytes};
}
g4b::PageTables tables_of(const g4b_page_tables* t) {
    return {t->refs, t->table, t->lens, t->refs_out, t->table_out, t->lens_out, t->n_pages, t->n_seqs,
            t->table_width, t->page_size};
}
int bad(const char* call, const char* why) {
    g_err = std::string(call) + ": " + why;
    return (int)cudaErrorInvalidValue;
}
}  // namespace

int g4b_pages_reserve(const g4b_page_tables* t, const int32_t* grow, int32_t* status, void* stream) {
    if (const char* why = bad_tables(t, true, false)) return bad("g4b_pages_reserve", why);
    if (!grow || !status) return bad("g4b_pages_reserve", "null pointer");
    const cudaError_t e = g4b::pages_reserve(tables_of(t), grow, status, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_pages_reserve");
}

int g4b_pages_fork(const g4b_page_pool* pool, const g4b_page_tables* t, const int32_t* src, const int32_t* dst, int n,
                   int32_t* status, void* stream) {
    if (const char* why = bad_pool(pool)) return bad("g4b_pages_fork", why);
    if (const char* why = bad_tables(t, true, true)) return bad("g4b_pages_fork", why);
    if (n < 0 || n > g4b::kMaxPageSeqs || !status || (n && (!src || !dst)))
        return bad("g4b_pages_fork", "null pointer or more than 4096 forks");
    if (pool->n_pages != t->n_pages || pool->page_size != t->page_size)
        return bad("g4b_pages_fork", "pool and tables differ in pages or page_size");
    const cudaError_t e = g4b::pages_fork(pool_of(pool), tables_of(t), src, dst, n, status, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_pages_fork");
}

int g4b_pages_free(const g4b_page_tables* t, const int32_t* seqs, int n, void* stream) {
    if (const char* why = bad_tables(t, true, true)) return bad("g4b_pages_free", why);
    if (n < 0 || (n && !seqs)) return bad("g4b_pages_free", "null pointer");
    const cudaError_t e = g4b::pages_free(tables_of(t), seqs, n, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_pages_free");
}

int g4b_pages_compact(const g4b_page_pool* pool, const g4b_page_tables* t, int32_t* moves, void* stream) {
    if (const char* why = bad_pool(pool)) return bad("g4b_pages_compact", why);
    if (const char* why = bad_tables(t, false, false)) return bad("g4b_pages_compact", why);
    if (!moves) return bad("g4b_pages_compact", "null pointer");
    if (pool->n_pages != t->n_pages) return bad("g4b_pages_compact", "pool and tables differ in pages");
    const cudaError_t e = g4b::pages_compact(pool_of(pool), tables_of(t), moves, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_pages_compact");
}

int g4b_pages_copy(const g4b_page_pool* from, const g4b_page_pool* to, const int32_t* src, const int32_t* dst, int n,
                   void* stream) {
    if (const char* why = bad_pool(from)) return bad("g4b_pages_copy", why);
    if (const char* why = bad_pool(to)) return bad("g4b_pages_copy", why);
    if (from->n_planes != to->n_planes || from->page_size != to->page_size || from->row_bytes != to->row_bytes)
        return bad("g4b_pages_copy", "the pools differ in planes, page_size or row_bytes");
    if (n < 0 || (n && (!src || !dst))) return bad("g4b_pages_copy", "null pointer");
    if (n == 0) return 0;
    const cudaError_t e = g4b::pages_copy(pool_of(from), pool_of(to), src, dst, n, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_pages_copy");
}

int g4b_pages_commit(const g4b_page_pool* pool, const int32_t* table, int table_width, const int32_t* lens, int n_seqs,
                     const void* rows, int64_t rows_plane_stride, int n_tokens, const int32_t* cu_nodes,
                     const int32_t* path, int path_width, const int32_t* count, const int32_t* status,
                     int32_t* lens_out, void* stream) {
    if (const char* why = bad_pool(pool)) return bad("g4b_pages_commit", why);
    if (n_seqs < 0 || n_seqs > g4b::kMaxPageSeqs || table_width < 1 || n_tokens < 0 || (path && path_width < 1))
        return bad("g4b_pages_commit", "sizes out of range");
    if (n_seqs == 0) return 0;
    if (!table || !lens || !cu_nodes || !count || !lens_out || (n_tokens && !rows))
        return bad("g4b_pages_commit", "null pointer");
    if ((reinterpret_cast<uintptr_t>(rows) & 15) || (rows_plane_stride & 15))
        return bad("g4b_pages_commit", "rows and their plane stride must be multiples of 16 bytes");
    const cudaError_t e = g4b::pages_commit(pool_of(pool), table, table_width, lens, n_seqs,
                                            static_cast<const char*>(rows), rows_plane_stride, n_tokens, cu_nodes, path,
                                            path_width, count, status, lens_out, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : fail(e, "g4b_pages_commit");
}

int g4b_qmat_check_error(g4b_qmat* q) {
    if (!q) return fail_msg("g4b_qmat_check_error: null handle");
    int h = 0;
    cudaError_t e = cudaMemcpy(&h, q->err, sizeof(int), cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return fail(e, "g4b_qmat_check_error");
    if (h) return fail_msg("INT4 GEMM: a bounded wait gave up (weights or fragments never arrived)");
    return 0;
}

}  // extern "C"
