// Attention of drafted token trees over a paged K/V cache, on the 5th-generation tensor cores.
//
// Node i of sequence s (its pending token is node 0) sits at position lens[s] + depth(i). It sees
// the cached keys j < lens[s] and, among its own sequence's nodes, those whose bit is set in its
// mask row; a window w > 0 hides keys w or more positions back. out = sum_j p_j v_j with p =
// softmax over the keys it sees of scale * q.k, and zero for a node that sees none.
//
// Bound. A key is read once per K/V head for all rows (nodes x query heads of the group) and costs
// 4 dim bytes and 4 dim rows operations: below about 250 rows the K/V stream through HBM is the
// floor, so the kernel is built around keeping that stream busy.
//
// Work. An item is (sequence, K/V head, group of up to 128 rows); its keys are cut into 128-key
// tiles, first the cached ones, then the nodes' own. All items' tiles, in one line, are dealt in
// equal shares to one block per SM, whatever the lengths: a block's share may start and end inside
// an item, whose parts (running maximum, sum, unnormalised output) a second kernel joins. Items
// that one block covers are written directly.
//
// Per tile, S^T[key][row] = K Q^T and O^T[dim][row] += V^T P^T: with the keys and the dimensions on
// the 128-lane side of the MMA the row count is its N, so a tree of 5 nodes costs N = 16 and not a
// padded 128. Roles:
//   * warp 0 streams K of tile t + 1, then V of tile t, through a ring of 32 KB slots (128 keys x
//     128 dims) by TMA: one box per (page part, 64 dims), swizzled as the MMA reads it;
//   * warp 1 (one thread) issues the MMAs, S^T into two alternating TMEM buffers;
//   * two groups of four warps take half of the rows each, a thread one key of all its rows: they
//     hold the softmax in fp32, write P^T (rounded to the cache's type, 8 rows a store) and, when a
//     row's score exceeds its reference maximum by more than 8 (in powers of two), move the
//     reference and rescale that row of O^T in TMEM. In between only a vote of the group is needed,
//     so most tiles run without any reduction over keys; the sums are reduced once per part.
// What a node must not see never reaches the MMA: scores are replaced, not added to, and in tiles
// that hold hidden keys the rows of V past the end are zeroed; an infinity or NaN in a V row that
// some nodes see and others do not is taken out of the product and added back for those that do.
//
// Every wait is bounded (2 s); a block that gives up records it in a device word and leaves.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"
#include "tree_attn.h"

#include <algorithm>
#include <cstring>

namespace g4b {

namespace {

constexpr int kKeys = 128;           // keys per tile: the M of S^T
constexpr int kThreads = 384;        // producer, MMA, two idle warps, 8 softmax warps
constexpr int kSoftWarps = 8;
constexpr uint32_t kBoxBytes = kKeys * 128;  // 128 keys x 64 dims of 16 bits
constexpr int kMaxSlots = 8;
constexpr int kTreeBox = 16;         // node rows per TMA box
constexpr float kUnset = 1e30f;      // negated reference of a row that has seen no key
constexpr float kLazy = 8.f;         // a reference moves when a score exceeds it by 2^8
constexpr size_t kSmemLimit = 232448;

__device__ int g_tree_err;  // set when a bounded wait gives up

struct Ctl {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t s_full[2], s_free[2];
    uint64_t q_ready, p_full, o_done, v_ready[4], v_fix[4], done;
    uint32_t tmem_base;
    int abort, poison;
    int seq0;            // where this block's share starts
    long long rem0, begin, end;
    long long scan[kThreads / 32 + 1];
    float nref[128];     // negated reference maximum of a row, in powers of two
    float corr[128];     // factor of a row's sum and output when its reference moves
    float inv[128];
    float red[4][128];
    int start[128];      // first cached position a row sees
    int depth[128];
    uint32_t mask[8][128];
};

struct Params {
    const char* q;
    char* out;
    const char* v_pool;
    const char* v_new;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;
    const uint32_t* mask;
    const int32_t* depth;
    float* part;   // [2 x blocks][N][dim]
    float2* ml;    // [2 x blocks][N]
    long long q_stride, out_stride, page_stride, new_stride;  // elements
    int seqs, n_tokens, max_nodes, pages, page_size, width, mask_words, heads, kv_heads, window;
    int N, slots, box, grid, tmem_cols;
    float c;       // scale * log2(e)
};

// One sequence's share of the work.
struct Seq {
    int len, first, n;   // cached tokens, first node, nodes
    int start, base;     // first cached position any node may see, and the first tile's
    int pre, tiles, groups;
};

__device__ __forceinline__ Seq load_seq(const Params& p, int b) {
    Seq s;
    const int gqa = p.heads / p.kv_heads;
    s.first = min(max(p.cu[b], 0), p.n_tokens);
    s.n = min(min(max(p.cu[b + 1] - s.first, 0), p.n_tokens - s.first), p.max_nodes);
    s.len = min(max(p.lens[b], 0), p.width * p.page_size);
    s.start = p.window ? max(0, s.len - p.window + 1) : 0;
    s.base = s.start / p.box * p.box;
    s.pre = s.start < s.len ? (s.len - s.base + kKeys - 1) / kKeys : 0;
    s.tiles = s.n ? s.pre + (s.n + kKeys - 1) / kKeys : 0;
    s.groups = (s.n * gqa + p.N - 1) / p.N;
    return s;
}

// Sum of the block's values, to every thread.
__device__ __forceinline__ long long block_total(long long v, long long* red) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) red[w] = v;
    __syncthreads();
    long long t = 0;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}

__device__ __forceinline__ long long seq_tiles(const Params& p, int b) {
    const Seq s = load_seq(p, b);
    return (long long)s.tiles * s.groups * p.kv_heads;
}

__device__ __forceinline__ long long share_begin(long long total, int grid, int c) { return total * c / grid; }

// Walks the parts of items in this block's share.
struct Walk {
    Seq s;
    int b, h, g, t;
    long long pos, end;
    int t0, t1;  // the part: tiles t0 .. t1 - 1 of item (b, h, g)
    __device__ void open(const Params& p, const Ctl& c) {
        pos = c.begin;
        end = c.end;
        b = c.seq0;
        if (pos >= end) return;
        s = load_seq(p, b);
        const long long per = (long long)s.tiles * s.groups;
        h = (int)(c.rem0 / per);
        const long long r = c.rem0 % per;
        g = (int)(r / s.tiles);
        t = (int)(r % s.tiles);
    }
    __device__ bool next(const Params& p) {
        if (pos >= end) return false;
        if (t == s.tiles) {
            t = 0;
            if (++g == s.groups) {
                g = 0;
                if (++h == p.kv_heads) {
                    h = 0;
                    do s = load_seq(p, ++b);
                    while (s.tiles == 0);
                }
            }
        }
        t0 = t;
        t1 = (int)min((long long)s.tiles, t0 + (end - pos));
        pos += t1 - t0;
        t = t1;
        return true;
    }
    // Keys of tile i up to its last one any row may see, and whether some of them are hidden from
    // some row.
    __device__ __forceinline__ int keys(int i) const {
        return i < s.pre ? min(kKeys, s.len - (s.base + i * kKeys)) : min(kKeys, s.n - (i - s.pre) * kKeys);
    }
    __device__ __forceinline__ bool windowed(const Params& p, int i) const {  // rows start inside the tile
        return p.window && i < s.pre && s.base + i * kKeys < s.start + s.n - 1;
    }
    __device__ __forceinline__ bool edge(const Params& p, int i) const {
        return i >= s.pre || keys(i) < kKeys || windowed(p, i) || s.base + i * kKeys < s.start;
    }
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait_sleep(bar, parity, 1000000u)) {
        if (*abort) return false;
        if (global_ns() - t0 > kWaitLimitNs) {
            *abort = 1;
            atomicExch(&g_tree_err, 1);
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ void group_bar(int grp) { asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory"); }
__device__ __forceinline__ bool group_or(int grp, bool v) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(1 + grp)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    uint32_t r;
    if (kBf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <bool kBf16>
__device__ __forceinline__ uint16_t pack1(float a) {
    return kBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(a)) : __half_as_ushort(__float2half_rn(a));
}
template <bool kBf16>
__device__ __forceinline__ float unpack1(uint16_t v) {
    return kBf16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}
template <bool kBf16>
__device__ __forceinline__ bool not_finite(uint16_t v) {
    return kBf16 ? (v & 0x7f80) == 0x7f80 : (v & 0x7c00) == 0x7c00;
}

// Reduce-scatter of per-lane values v[0 .. P) (P a power of two, 8 .. 64) over the warp: each step
// sends the half the lane gives away. Afterwards the lane holds max(1, P / 32) reduced values in
// v[0 ..], of rows scatter_row<P>(lane) onwards (for P < 32 several lanes hold the same row).
template <int P, bool kMax>
__device__ __forceinline__ void reduce_scatter(float (&v)[P], int lane) {
    auto op = [](float a, float b) { return kMax ? fmaxf(a, b) : a + b; };
    int bit = 16;
#pragma unroll
    for (int n = P / 2; n >= 1 && bit >= 1; n >>= 1, bit >>= 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < P / 2; ++i)
            if (i < n) {
                const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
                v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, bit));
            }
    }
#pragma unroll
    for (int k = 2; k >= 1; k >>= 1)
        if (k <= bit) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], k));
}
template <int P>
__device__ __forceinline__ int scatter_row(int lane) {
    int r = 0, bit = 16;
#pragma unroll
    for (int n = P / 2; n >= 1 && bit >= 1; n >>= 1, bit >>= 1)
        if (lane & bit) r += n;
    return r;
}

__host__ __device__ constexpr int pow2_at_least(int n) { return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 64; }

// Whether row r of the part sees key k (0 .. 127) of tile i.
__device__ __forceinline__ bool sees(const Params& p, const Walk& w, const Ctl& c, int i, int k, int r) {
    if (i < w.s.pre) {
        const int j = w.s.base + i * kKeys + k;
        return j < w.s.len && j >= c.start[r];
    }
    const int j = (i - w.s.pre) * kKeys + k;
    if (j >= w.s.n || !((c.mask[j >> 5][r] >> (j & 31)) & 1)) return false;
    return !p.window || c.depth[r] - min(max(p.depth[w.s.first + j], 0), w.s.n - 1) < p.window;
}

// Address of V's row for key k of tile i (null: no such row).
template <int D>
__device__ __noinline__ const uint16_t* v_row(const Params& p, const Walk& w, int i, int k) {
    if (i < w.s.pre) {
        const int j = w.s.base + i * kKeys + k;
        if (j < w.s.start || j >= w.s.len) return nullptr;
        const int page = p.table[(long long)w.b * p.width + j / p.page_size];
        if (page < 0 || page >= p.pages) return nullptr;
        return reinterpret_cast<const uint16_t*>(p.v_pool) + page * p.page_stride +
               ((long long)(j % p.page_size) * p.kv_heads + w.h) * D;
    }
    const int j = (i - w.s.pre) * kKeys + k;
    if (j >= w.s.n) return nullptr;
    return reinterpret_cast<const uint16_t*>(p.v_new) + (w.s.first + j) * p.new_stride + w.h * D;
}

// The infinities and NaN that were taken out of this part's V tiles, added to the outputs v of rows
// r0 .. r0 + 7 in dimension d.
template <int D, bool kBf16>
__device__ __noinline__ void add_poison(const Params& p, const Walk& w, const Ctl& c, int d, int r0, float (&v)[8]) {
    for (int i = w.t0; i < w.t1; ++i) {
        if (!(i >= w.s.pre || w.windowed(p, i))) continue;
        for (int k = 0; k < w.keys(i); ++k) {
            const uint16_t* row = v_row<D>(p, w, i, k);
            if (!row || !not_finite<kBf16>(row[d])) continue;
            for (int j = 0; j < 8; ++j)
                if (sees(p, w, c, i, k, r0 + j)) v[j] += unpack1<kBf16>(row[d]);
        }
    }
}

// kNH: the most rows a softmax group takes (N / 2 of them are used, a multiple of 8).
template <int D, int kNH, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ CUtensorMap knmap, const __grid_constant__ CUtensorMap vnmap,
                     const __grid_constant__ Params p) {
    constexpr int kHalves = D == 64 ? 1 : 2;                // 64-dim boxes per slot
    constexpr int kChunks = D == 64 ? 1 : D / 128;          // slots per K or V tile
    constexpr uint32_t kSlotBytes = kHalves * kBoxBytes;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int N = p.N, nh = N >> 1, slots = p.slots;
    unsigned char* ring = sm;
    unsigned char* qs = ring + slots * kSlotBytes;             // [D / 64][N rows][64 dims]
    unsigned char* ps = qs + (D / 64) * N * 128;               // [N / 64][128 keys][64 rows]
    Ctl& c = *reinterpret_cast<Ctl*>(ps + ((N + 63) / 64) * kBoxBytes);
    volatile int* abort = &c.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < slots; ++s) {
            mbar_init(&c.full[s], 1);
            mbar_init(&c.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&c.s_full[b], 1);
            mbar_init(&c.s_free[b], kSoftWarps);
        }
        mbar_init(&c.q_ready, kSoftWarps);
        mbar_init(&c.p_full, kSoftWarps);
        mbar_init(&c.o_done, 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&c.v_ready[i], 1);
            mbar_init(&c.v_fix[i], kSoftWarps);
        }
        mbar_init(&c.done, 1);
        c.abort = 0;
        c.poison = 0;
        mbar_init_fence();
    }
    if (warp == 1) tc::alloc(&c.tmem_base, p.tmem_cols);

    // This block's share of all tiles.
    long long mine = 0;
    for (int b = threadIdx.x; b < p.seqs; b += kThreads) mine += seq_tiles(p, b);
    const long long total = block_total(mine, c.scan);
    const long long begin = share_begin(total, gridDim.x, blockIdx.x), end = share_begin(total, gridDim.x, blockIdx.x + 1);
    if (threadIdx.x == 0) {
        c.begin = begin;
        c.end = end;
    }
    long long before = 0;
    for (int b0 = 0; warp == 0 && begin < end && b0 < p.seqs; b0 += 32) {
        const int b = b0 + lane;
        const long long mt = b < p.seqs ? seq_tiles(p, b) : 0;
        long long x = mt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const long long at = before + x - mt;
        if (mt > 0 && begin >= at && begin < at + mt) {
            c.seq0 = b;
            c.rem0 = begin - at;
        }
        before += __shfl_sync(0xffffffffu, x, 31);
        if (before > begin) break;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = c.tmem_base;
    const uint32_t o_col = 2 * (uint32_t)N;  // S^T buffers, then the O^T tiles of 128 dims
    pdl_launch_dependents();

    Walk w;
    w.open(p, c);
    if (warp == 0) {
        // ------------------------------------------------------------------ producer
        int q = 0;
        bool ok = true;
        const int kb = lane & 15, half = lane >> 4;  // up to 16 key boxes, two halves of 64 dims
        auto ids = [&](int i) {  // page of this lane's key box in tile i
            const int j = w.s.base + i * kKeys + kb * p.box;
            return i < w.s.pre && kb * p.box < kKeys && j < w.s.len ? p.table[(long long)w.b * p.width + j / p.page_size] : -1;
        };
        auto load = [&](const CUtensorMap* pool, const CUtensorMap* fresh, int i, int page) {
            const bool old = i < w.s.pre;
            const int rows = old ? p.box : kTreeBox;
            const int boxes = (w.keys(i) + rows - 1) / rows;
            const bool mine = kb < boxes && half < kHalves;
            const int j = w.s.base + i * kKeys + kb * p.box;
            for (int ci = 0; ci < kChunks && ok; ++ci, ++q) {
                const int slot = q % slots;
                if (q >= slots) ok = wait(&c.empty[slot], ((q / slots) + 1) & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                if (lane == 0) mbar_expect_tx(&c.full[slot], (uint32_t)(boxes * rows) * 128 * kHalves);
                __syncwarp();
                if (mine) {
                    unsigned char* dst = ring + slot * kSlotBytes + half * kBoxBytes + kb * rows * 128;
                    const int x = 128 * ci + 64 * half;
                    // A page id out of range is an out-of-range coordinate: the box reads as zeros.
                    if (old) tma_4d(dst, pool, x, w.h, j % p.page_size, page < 0 ? p.pages : page, &c.full[slot]);
                    else tma_3d(dst, fresh, x, w.h, w.s.first + (i - w.s.pre) * kKeys + kb * kTreeBox, &c.full[slot]);
                }
            }
        };
        while (ok && w.next(p)) {
            int id0 = -1, id1 = ids(w.t0);
            for (int i = w.t0; i <= w.t1 && ok; ++i) {
                const int id2 = i + 1 < w.t1 ? ids(i + 1) : -1;
                if (i < w.t1) load(&kmap, &knmap, i, id1);
                if (i > w.t0 && ok) load(&vmap, &vnmap, i - 1, id0);
                id0 = id1;
                id1 = id2;
            }
        }
        // Every issued copy lands before the block can exit.
        if (lane == 0)
            for (int i = max(0, q - slots); i < q; ++i)
                if (!mbar_wait(&c.full[i % slots], (i / slots) & 1)) atomicExch(&g_tree_err, 1);
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        if (lane == 0) {
            const uint32_t id_s = tc::idesc_16(kKeys, N, kBf16, false, false);
            const uint32_t id_o = tc::idesc_16(128, N, kBf16, true, true);
            const uint32_t q_addr = smem_u32(qs), p_addr = smem_u32(ps), r_addr = smem_u32(ring);
            const uint32_t blk = (uint32_t)N * 128;
            int q = 0, tile = 0, otile = 0, part = 0, fix = 0;
            bool ok = true;
            auto issue_s = [&]() {
                const int b = tile & 1;
                if (tile >= 2 && !wait(&c.s_free[b], ((tile >> 1) - 1) & 1, abort)) return false;
                for (int ci = 0; ci < kChunks; ++ci, ++q) {
                    const int slot = q % slots;
                    if (!wait(&c.full[slot], (q / slots) & 1, abort)) return false;
                    tc::fence_after_sync();
                    const uint32_t sa = r_addr + slot * kSlotBytes;
#pragma unroll
                    for (int h = 0; h < kHalves; ++h)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            tc::mma_ss(tmem + b * N, tc::desc_sw128(sa + h * kBoxBytes + kk * 32),
                                       tc::desc_sw128(q_addr + (uint32_t)(2 * ci + h) * blk + kk * 32), id_s,
                                       (ci | h | kk) ? 1u : 0u);
                    tc::commit(&c.empty[slot]);
                }
                tc::commit(&c.s_full[b]);
                ++tile;
                return true;
            };
            auto issue_o = [&](int i) {
                if (!wait(&c.p_full, otile & 1, abort)) return false;
                tc::fence_after_sync();
                const int steps = (w.keys(i) + 15) >> 4;
                const bool edge = w.edge(p, i);
                for (int ci = 0; ci < kChunks; ++ci, ++q) {
                    const int slot = q % slots;
                    if (!wait(&c.full[slot], (q / slots) & 1, abort)) return false;
                    if (edge) {  // the softmax warps clean the chunk first
                        mbar_arrive(&c.v_ready[ci]);
                        if (!wait(&c.v_fix[ci], fix & 1, abort)) return false;
                    }
                    tc::fence_after_sync();
                    const uint32_t sa = r_addr + slot * kSlotBytes;
                    for (int kk = 0; kk < steps; ++kk)
                        // V^T rows are the slot's dims, two 64-dim boxes apart (with D = 64 the lanes
                        // 64 .. 127 multiply whatever follows in shared memory, and are never read).
                        tc::mma_ss(tmem + o_col + ci * N, tc::desc_sw128_mn(sa + kk * 2048, kBoxBytes, 1024),
                                   tc::desc_sw128_mn(p_addr + kk * 2048, kBoxBytes, 1024), id_o,
                                   (i > w.t0 || kk > 0) ? 1u : 0u);
                    tc::commit(&c.empty[slot]);
                }
                tc::commit(&c.o_done);
                fix += edge;
                ++otile;
                return true;
            };
            while (ok && w.next(p)) {
                ok = wait(&c.q_ready, part++ & 1, abort);
                if (ok) {
                    tc::fence_after_sync();
                    ok = issue_s();
                }
                for (int i = w.t0; i < w.t1 && ok; ++i) ok = (i + 1 >= w.t1 || issue_s()) && issue_o(i);
            }
            tc::commit(&c.done);  // every MMA has completed before tensor memory is freed
            if (!mbar_wait(&c.done, 0)) atomicExch(&g_tree_err, 1);
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------------ softmax
        constexpr int kP = pow2_at_least(kNH);
        const int sw = warp - 4, grp = sw >> 2, qd = sw & 3;
        const int tid = sw * 32 + lane, gt = tid & 127;   // 0..255; 0..127 in the group
        const int key = qd * 32 + lane;                   // TMEM lane
        const int r0 = grp * nh;                          // the group's rows r0 .. r0 + nh - 1
        const uint32_t lanes = (uint32_t)(qd * 32) << 16;
        const int gqa = p.heads / p.kv_heads;
        int tile = 0, q = 0, fix = 0;  // tiles, ring slots (as the producer counts them), edge tiles so far
        bool first_part = true;
        float l[kNH];
        // After a wait that gave up, these warps go on (on meaningless values) to the end of the share:
        // none of them may leave while others stand at a barrier of the group.
        while (w.next(p)) {
            // Rows of this part: r -> node (g N + r) / gqa, query head h gqa + (g N + r) % gqa.
            const int R = min(N, w.s.n * gqa - w.g * N);
            if (tid < N) {
                const int node = min((w.g * N + tid) / gqa, w.s.n - 1), tok = w.s.first + node;
                const int dep = p.window ? min(max(p.depth[tok], 0), w.s.n - 1) : 0;
                c.nref[tid] = kUnset;
                c.depth[tid] = dep;
                c.start[tid] = p.window ? max(0, w.s.len + dep - p.window + 1) : 0;
                for (int i = 0; i * 32 < w.s.n; ++i) c.mask[i][tid] = p.mask[(long long)tok * p.mask_words + i];
            }
            if (tid == 0) c.poison = 0;
            // The queries, into the MMA's K-major layout (S of the part before has completed).
            for (int e = tid; e < N * (D / 8); e += 256) {
                const int r = e / (D / 8), ch = e % (D / 8);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < R) {
                    const int row = w.g * N + r;
                    v = __ldg(reinterpret_cast<const uint4*>(
                                  p.q + 2 * ((w.s.first + row / gqa) * p.q_stride + (w.h * gqa + row % gqa) * D)) + ch);
                }
                *reinterpret_cast<uint4*>(qs + (size_t)(ch >> 3) * N * 128 + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
            }
            fence_proxy_async();
            asm volatile("bar.sync 3, 256;" ::: "memory");
            if (lane == 0) mbar_arrive(&c.q_ready);
#pragma unroll
            for (int r = 0; r < kNH; ++r) l[r] = 0.f;

            for (int i = w.t0; i < w.t1; ++i, ++tile) {
                const int b = tile & 1;
                wait(&c.s_full[b], (tile >> 1) & 1, abort);
                tc::fence_after_sync();
                float s[kNH];
#pragma unroll
                for (int e = 0; e < kNH / 8; ++e)
                    if (8 * e < nh) {
                        float v[8];
                        tc::ld8(tmem + lanes + b * N + r0 + 8 * e, v);
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[8 * e + j] = v[j];
                    }
                tc::wait_ld();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.s_free[b]);
                const bool edge = w.edge(p, i);
                if (edge) {
                    if (i < w.s.pre) {
                        const int j = w.s.base + i * kKeys + key;
#pragma unroll
                        for (int r = 0; r < kNH; ++r)
                            if (r < nh && !(j < w.s.len && j >= c.start[r0 + r])) s[r] = -INFINITY;
                    } else {
                        const int j = (i - w.s.pre) * kKeys + key;
                        const int word = (i - w.s.pre) * 4 + qd;
                        const int near = p.window && j < w.s.n
                                             ? min(max(p.depth[w.s.first + j], 0), w.s.n - 1) + p.window
                                             : INT_MAX;
#pragma unroll
                        for (int r = 0; r < kNH; ++r)
                            if (r < nh && !(j < w.s.n && ((c.mask[word][r0 + r] >> lane) & 1) && c.depth[r0 + r] < near))
                                s[r] = -INFINITY;
                    }
                }
                // Does a score exceed its row's reference by more than kLazy?
                float over = -INFINITY;
#pragma unroll
                for (int r = 0; r < kNH; r += 4)
                    if (r < nh) {
                        const float4 f = *reinterpret_cast<const float4*>(&c.nref[r0 + r]);
                        over = fmaxf(fmaxf(over, fmaf(s[r], p.c, f.x)), fmaf(s[r + 1], p.c, f.y));
                        over = fmaxf(fmaxf(over, fmaf(s[r + 2], p.c, f.z)), fmaf(s[r + 3], p.c, f.w));
                    }
                bool waited = false;
                if (group_or(grp, over > kLazy)) {
                    float m[kP];
#pragma unroll
                    for (int r = 0; r < kP; ++r) m[r] = r < kNH && r < nh ? s[r] * p.c : -INFINITY;
                    reduce_scatter<kP, true>(m, lane);
                    const int at = scatter_row<kP>(lane);
#pragma unroll
                    for (int j = 0; j < (kP > 32 ? 2 : 1); ++j)
                        if (at + j < nh) c.red[qd][r0 + at + j] = m[j];
                    group_bar(grp);
                    if (gt < nh) {
                        const int r = r0 + gt;
                        const float top = fmaxf(fmaxf(c.red[0][r], c.red[1][r]), fmaxf(c.red[2][r], c.red[3][r]));
                        const float old = c.nref[r];
                        float f = 1.f;
                        if (top > -INFINITY && (old == kUnset || top + old > kLazy)) {
                            f = old == kUnset ? 0.f : exp2_approx(-old - top);
                            c.nref[r] = -top;
                        }
                        c.corr[r] = f;
                    }
                    group_bar(grp);
#pragma unroll
                    for (int r = 0; r < kNH; ++r)
                        if (r < nh) l[r] *= c.corr[r0 + r];
                    if (i > w.t0) {
                        wait(&c.o_done, (tile - 1) & 1, abort);
                        waited = true;
                        tc::fence_after_sync();
#pragma unroll 1
                        for (int ci = 0; ci < kChunks; ++ci)
#pragma unroll 1
                            for (int e = 0; e < nh; e += 8) {
                                float v[8];
                                const uint32_t ta = tmem + lanes + o_col + ci * N + r0 + e;
                                tc::ld8(ta, v);
                                tc::wait_ld();
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] *= c.corr[r0 + e + j];
                                tc::st8(ta, v);
                            }
                        tc::wait_st();
                    }
                }
#pragma unroll
                for (int r = 0; r < kNH; r += 4)
                    if (r < nh) {
                        const float4 f = *reinterpret_cast<const float4*>(&c.nref[r0 + r]);
                        s[r] = exp2_approx(fmaf(s[r], p.c, f.x));
                        s[r + 1] = exp2_approx(fmaf(s[r + 1], p.c, f.y));
                        s[r + 2] = exp2_approx(fmaf(s[r + 2], p.c, f.z));
                        s[r + 3] = exp2_approx(fmaf(s[r + 3], p.c, f.w));
                        l[r] += s[r];
                        l[r + 1] += s[r + 1];
                        l[r + 2] += s[r + 2];
                        l[r + 3] += s[r + 3];
                    }
                // P V of the tile before has read the buffer.
                if (tile > 0 && !waited) wait(&c.o_done, (tile - 1) & 1, abort);
                const uint32_t prow = key * 128;
#pragma unroll
                for (int e = 0; e < kNH / 8; ++e)
                    if (8 * e < nh) {
                        const int r = r0 + 8 * e;
                        uint4 v;
                        v.x = pack2<kBf16>(s[8 * e], s[8 * e + 1]);
                        v.y = pack2<kBf16>(s[8 * e + 2], s[8 * e + 3]);
                        v.z = pack2<kBf16>(s[8 * e + 4], s[8 * e + 5]);
                        v.w = pack2<kBf16>(s[8 * e + 6], s[8 * e + 7]);
                        *reinterpret_cast<uint4*>(ps + (r >> 6) * kBoxBytes + prow + ((((r & 63) >> 3) ^ (key & 7)) << 4)) = v;
                    }
                fence_proxy_async();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.p_full);
                // Ring slots of this tile's V, in the producer's order: K(t0), then K(i + 1), V(i).
                const int vq = q + (i - w.t0) * 2 * kChunks + (i + 1 < w.t1 ? 2 : 1) * kChunks;
                if (edge) {
                    const int rows = (w.keys(i) + 15) & ~15;
                    const bool scan = i >= w.s.pre || w.windowed(p, i);
                    const int lead = i < w.s.pre ? w.s.start - (w.s.base + i * kKeys) : 0;  // keys before every row's
                    for (int ci = 0; ci < kChunks; ++ci) {
                        const int slot = (vq + ci) % slots;
                        // v_ready first: the slot may still be a use behind, and a parity cannot tell a
                        // phase from the one two before it.
                        wait(&c.v_ready[ci], fix & 1, abort);
                        wait(&c.full[slot], ((vq + ci) / slots) & 1, abort);
                        unsigned char* base = ring + slot * kSlotBytes;
                        for (int e = tid; e < rows * 8 * kHalves; e += 256) {
                            const int k = e / (8 * kHalves), ch = e % (8 * kHalves);
                            uint4* at = reinterpret_cast<uint4*>(base + (ch >> 3) * kBoxBytes + k * 128 + (ch & 7) * 16);
                            if (k >= w.keys(i) || k < lead) {
                                *at = make_uint4(0, 0, 0, 0);
                            } else if (scan) {
                                uint4 v = *at;
                                bool dirty = false;
                                auto clean = [&](uint32_t& x) {
                                    if (not_finite<kBf16>((uint16_t)x)) x &= 0xffff0000u, dirty = true;
                                    if (not_finite<kBf16>((uint16_t)(x >> 16))) x &= 0x0000ffffu, dirty = true;
                                };
                                clean(v.x);
                                clean(v.y);
                                clean(v.z);
                                clean(v.w);
                                if (dirty) {
                                    *at = v;
                                    c.poison = 1;
                                }
                            }
                        }
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&c.v_fix[ci]);
                    }
                    ++fix;
                }
            }
            q += (w.t1 - w.t0) * 2 * kChunks;

            // The part's result: sums over the keys, then O^T.
            float m[kP];
#pragma unroll
            for (int r = 0; r < kP; ++r) m[r] = r < kNH ? l[r < kNH ? r : 0] : 0.f;
            reduce_scatter<kP, false>(m, lane);
            const int at = scatter_row<kP>(lane);
            group_bar(grp);
#pragma unroll
            for (int j = 0; j < (kP > 32 ? 2 : 1); ++j)
                if (at + j < nh) c.red[qd][r0 + at + j] = m[j];
            group_bar(grp);
            const bool whole = w.t0 == 0 && w.t1 == w.s.tiles;
            const int slot = 2 * blockIdx.x + (first_part ? 0 : 1);
            first_part = false;
            if (gt < nh) {
                const int r = r0 + gt;
                const float sum = (c.red[0][r] + c.red[1][r]) + (c.red[2][r] + c.red[3][r]);
                c.inv[r] = sum != 0.f ? 1.f / sum : 0.f;
                if (!whole) p.ml[(long long)slot * N + r] = make_float2(c.nref[r] == kUnset ? -INFINITY : -c.nref[r], sum);
            }
            wait(&c.o_done, (tile - 1) & 1, abort);
            tc::fence_after_sync();
            asm volatile("bar.sync 3, 256;" ::: "memory");  // also: every thread's poison flag
            const bool poison = c.poison != 0;
#pragma unroll 1
            for (int ci = 0; ci < kChunks; ++ci) {
                const int d = 128 * ci + key;
#pragma unroll 1
                for (int e = 0; e < nh && r0 + e < R; e += 8) {
                    float v[8];
                    tc::ld8(tmem + lanes + o_col + ci * N + r0 + e, v);
                    tc::wait_ld();
                    if (D == 64 && key >= 64) continue;
                    if (poison) add_poison<D, kBf16>(p, w, c, d, r0 + e, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int r = r0 + e + j, row = w.g * N + r;
                        if (r >= R) break;
                        if (whole)
                            reinterpret_cast<uint16_t*>(p.out)[(w.s.first + row / gqa) * p.out_stride +
                                                               (w.h * gqa + row % gqa) * D + d] = pack1<kBf16>(v[j] * c.inv[r]);
                        else
                            __stcg(p.part + ((long long)slot * N + r) * D + d, v[j]);
                    }
                }
            }
            tc::fence_before_sync();
            asm volatile("bar.sync 3, 256;" ::: "memory");  // the row state is free for the next part
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::dealloc(tmem, p.tmem_cols);
    }
}

constexpr int kJoinRows = 8;

// Joins the parts of items that several blocks worked on: out = sum_s 2^(m_s - M) O_s over
// sum_s 2^(m_s - M) l_s. A warp per row, kJoinRows rows a block; grid (seqs x kv_heads, row blocks).
template <int D, bool kBf16>
__global__ void __launch_bounds__(32 * kJoinRows) tree_attn_join_kernel(const __grid_constant__ Params p) {
    __shared__ long long red[32];
    pdl_wait();
    const int b = blockIdx.x / p.kv_heads, h = blockIdx.x % p.kv_heads, lane = threadIdx.x & 31;
    const int gqa = p.heads / p.kv_heads;
    const Seq s = load_seq(p, b);
    if (s.n * gqa <= (int)blockIdx.y * kJoinRows) return;
    long long before = 0, all = 0;
    for (int i = threadIdx.x; i < p.seqs; i += 32 * kJoinRows) {
        const long long t = seq_tiles(p, i);
        all += t;
        if (i < b) before += t;
    }
    before = block_total(before, red);
    all = block_total(all, red);
    const int row = blockIdx.y * kJoinRows + (threadIdx.x >> 5);
    if (row >= s.n * gqa) return;
    const int g = row / p.N, r = row % p.N;
    const long long a = before + ((long long)h * s.groups + g) * s.tiles, z = a + s.tiles;
    const auto block_of = [&](long long x) { return (int)(((x + 1) * p.grid - 1) / all); };
    const int c0 = block_of(a), c1 = block_of(z - 1);
    if (c0 == c1 && share_begin(all, p.grid, c0) <= a && share_begin(all, p.grid, c0 + 1) >= z) return;
    const auto slot_of = [&](int c) { return (long long)(2 * c + (share_begin(all, p.grid, c) < a ? 1 : 0)); };
    float top = -INFINITY;
    for (int c = c0 + lane; c <= c1; c += 32) {
        if (share_begin(all, p.grid, c) == share_begin(all, p.grid, c + 1)) continue;
        const float2 x = p.ml[slot_of(c) * p.N + r];
        top = fmaxf(top, x.x);
    }
    top = warp_max(top);
    constexpr int kV = D / 32 > 4 ? 4 : D / 32;  // floats a lane loads at once
    constexpr int kL = D / 32 / kV;
    float o[kL][kV], sum = 0.f;
#pragma unroll
    for (int k = 0; k < kL; ++k)
#pragma unroll
        for (int j = 0; j < kV; ++j) o[k][j] = 0.f;
#pragma unroll 2
    for (int c = c0; c <= c1; ++c) {
        if (share_begin(all, p.grid, c) == share_begin(all, p.grid, c + 1)) continue;
        const float2 x = p.ml[slot_of(c) * p.N + r];
        if (x.x == -INFINITY) continue;  // this part's keys are all hidden from the row
        const float f = exp2_approx(x.x - top);
        sum = fmaf(f, x.y, sum);
        const float* src = p.part + (slot_of(c) * p.N + r) * D;
#pragma unroll
        for (int k = 0; k < kL; ++k) {
            float v[kV];
            if constexpr (kV == 4) *reinterpret_cast<float4*>(v) = __ldcg(reinterpret_cast<const float4*>(src) + k * 32 + lane);
            else *reinterpret_cast<float2*>(v) = __ldcg(reinterpret_cast<const float2*>(src) + k * 32 + lane);
#pragma unroll
            for (int j = 0; j < kV; ++j) o[k][j] = fmaf(f, v[j], o[k][j]);
        }
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    uint32_t* out = reinterpret_cast<uint32_t*>(p.out + 2 * ((s.first + row / gqa) * p.out_stride + (h * gqa + row % gqa) * D));
#pragma unroll
    for (int k = 0; k < kL; ++k)
#pragma unroll
        for (int j = 0; j < kV; j += 2)
            out[(k * 32 + lane) * (kV / 2) + j / 2] = pack2<kBf16>(o[k][j] * inv, o[k][j + 1] * inv);
}

int sm_count() {
    static int n = 0;
    if (!n) {
        int dev = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (n <= 0) n = 148;
    }
    return n;
}

// Rows per item: all of a tree's rows when they fit the tensor memory (two S^T buffers and the O^T
// tiles, N columns each, in 512) and shared memory, else equal groups.
int rows_per_item(int max_nodes, int gqa, int dim) {
    const int cap = dim == 512 ? 80 : 128, rows = max_nodes * gqa;
    const int groups = (rows + cap - 1) / cap;
    return ((rows + groups - 1) / groups + 15) / 16 * 16;
}

struct Shape {
    int N, slots, tmem;
    size_t smem;
};
Shape shape_for(int max_nodes, int gqa, int dim) {
    Shape s;
    s.N = rows_per_item(max_nodes, gqa, dim);
    const size_t slot = (dim == 64 ? 1 : 2) * kBoxBytes;
    const size_t rest = 1024 + (size_t)s.N * dim * 2 + (size_t)((s.N + 63) / 64) * kBoxBytes + sizeof(Ctl);
    s.slots = (int)std::min<size_t>(kMaxSlots, (kSmemLimit - rest) / slot);
    s.smem = rest + s.slots * slot;
    const int cols = s.N * (2 + std::max(1, dim / 128));
    s.tmem = 32;
    while (s.tmem < cols) s.tmem *= 2;
    return s;
}

cudaError_t make_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                     const cuuint32_t* box) {
    using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn) return cudaErrorNotSupported;
        encode = reinterpret_cast<EncodeFn>(fn);
    }
    const cuuint32_t one[4] = {1, 1, 1, 1};
    const CUresult r = encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, const_cast<void*>(base), dims, strides, box, one,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int D, int kNH, bool kBf16>
cudaError_t run(const CUtensorMap* maps, const Params& p, const Shape& sh, cudaStream_t st) {
    auto kern = tree_attn_kernel<D, kNH, kBf16>;
    static bool attr = false;
    if (!attr) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit);
        if (e != cudaSuccess) return e;
        attr = true;
    }
    cudaError_t e = launch(kern, dim3(p.grid), dim3(kThreads), sh.smem, st, false, maps[0], maps[1], maps[2], maps[3], p);
    if (e != cudaSuccess) return e;
    const int rows = p.max_nodes * (p.heads / p.kv_heads);
    return launch(tree_attn_join_kernel<D, kBf16>, dim3(p.seqs * p.kv_heads, (rows + kJoinRows - 1) / kJoinRows),
                  dim3(32 * kJoinRows), 0, st, true, p);
}

template <int D, bool kBf16>
cudaError_t run_rows(const CUtensorMap* maps, const Params& p, const Shape& sh, cudaStream_t st) {
    const int nh = sh.N / 2;
    if (nh <= 8) return run<D, 8, kBf16>(maps, p, sh, st);
    if (nh <= 16) return run<D, 16, kBf16>(maps, p, sh, st);
    if (nh <= 32) return run<D, 32, kBf16>(maps, p, sh, st);
    if constexpr (D == 512) return run<D, 40, kBf16>(maps, p, sh, st);
    else return run<D, 64, kBf16>(maps, p, sh, st);
}

template <int D>
cudaError_t run_type(const CUtensorMap* maps, const Params& p, const Shape& sh, bool bf16, cudaStream_t st) {
    return bf16 ? run_rows<D, true>(maps, p, sh, st) : run_rows<D, false>(maps, p, sh, st);
}

}  // namespace

size_t tree_attn_workspace(int max_nodes, int heads, int kv_heads, int dim) {
    const int N = rows_per_item(max_nodes, heads / kv_heads, dim);
    return (size_t)2 * sm_count() * N * (dim * sizeof(float) + sizeof(float2));
}

cudaError_t tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st) {
    const Shape sh = shape_for(a.max_nodes, a.heads / a.kv_heads, a.dim);
    Params p{};
    p.q = static_cast<const char*>(a.q);
    p.out = static_cast<char*>(a.out);
    p.v_pool = static_cast<const char*>(a.v_pool);
    p.v_new = static_cast<const char*>(a.v_new);
    p.table = a.table;
    p.lens = a.lens;
    p.cu = a.cu;
    p.mask = a.mask;
    p.depth = a.depth;
    p.grid = sm_count();
    p.part = static_cast<float*>(a.work);
    p.ml = reinterpret_cast<float2*>(p.part + (size_t)2 * p.grid * sh.N * a.dim);
    p.q_stride = a.q_stride;
    p.out_stride = a.out_stride;
    p.page_stride = a.page_stride;
    p.new_stride = a.new_stride;
    p.seqs = a.seqs;
    p.n_tokens = a.n_tokens;
    p.max_nodes = a.max_nodes;
    p.pages = a.pages;
    p.page_size = a.page_size;
    p.width = a.width;
    p.mask_words = a.mask_words;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.window = a.window;
    p.N = sh.N;
    p.slots = sh.slots;
    p.tmem_cols = sh.tmem;
    // The largest power of two that divides a page, so that a box never crosses one.
    p.box = std::min(kKeys, a.page_size & -a.page_size);
    p.c = a.scale * 1.4426950408889634f;
    const cuuint64_t row = (cuuint64_t)a.dim * 2, D = a.dim, H = a.kv_heads;
    const cuuint64_t pool_dims[4] = {D, H, (cuuint64_t)a.page_size, (cuuint64_t)a.pages};
    const cuuint64_t pool_strides[3] = {row, row * H, (cuuint64_t)a.page_stride * 2};
    const cuuint32_t pool_box[4] = {64, 1, (cuuint32_t)p.box, 1};
    const cuuint64_t new_dims[3] = {D, H, (cuuint64_t)a.n_tokens};
    const cuuint64_t new_strides[2] = {row, (cuuint64_t)a.new_stride * 2};
    const cuuint32_t new_box[3] = {64, 1, kTreeBox};
    CUtensorMap m[4];
    cudaError_t e;
    if ((e = make_map(&m[0], a.k_pool, 4, pool_dims, pool_strides, pool_box)) != cudaSuccess) return e;
    if ((e = make_map(&m[1], a.v_pool, 4, pool_dims, pool_strides, pool_box)) != cudaSuccess) return e;
    if ((e = make_map(&m[2], a.k_new, 3, new_dims, new_strides, new_box)) != cudaSuccess) return e;
    if ((e = make_map(&m[3], a.v_new, 3, new_dims, new_strides, new_box)) != cudaSuccess) return e;
    switch (a.dim) {
        case 64: return run_type<64>(m, p, sh, a.bf16, st);
        case 128: return run_type<128>(m, p, sh, a.bf16, st);
        case 256: return run_type<256>(m, p, sh, a.bf16, st);
        default: return run_type<512>(m, p, sh, a.bf16, st);
    }
}

int tree_attn_error() {
    int h = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&h, g_tree_err, sizeof(int)) != cudaSuccess) return -1;
    if (h) cudaMemcpyToSymbol(g_tree_err, &zero, sizeof(int));
    return h;
}

}  // namespace g4b
