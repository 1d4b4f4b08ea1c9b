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
//   * one warp deals the block's share out in parts and sets their rows up, one brings their queries in
//     (as its own warp it is done before the part ahead is: with one warp for both, which took 18000
//     cycles over 128 rows of 256, 64-node trees took 160 us instead of 137);
//   * one warp streams K of tile t + 1, then V of tile t, through a ring of 32 KB slots (128 keys x
//     128 dims) by TMA: one box per page part, both 64-dim blocks of it, laid out in eights of keys as the
//     MMA reads them (a copy per block was the limit at 16-row pages: 106 us instead of 87 for 1-node
//     trees over a 1024-key window; slots of 16 KB, which use what is left of shared memory, need more
//     copies and are no faster);
//   * one thread of another issues the MMAs, S^T into two alternating TMEM buffers;
//   * four groups of four warps take a quarter of the rows each, a thread one key of all its rows: they
//     hold the softmax in fp32, write P^T (rounded to the cache's type, 8 rows a store) and, when a
//     row's score exceeds the maximum it last took by more than 8 (in powers of two), move the
//     reference and rescale that row of O^T in TMEM. In between only a vote of the group is needed,
//     so most tiles run without any reduction over keys; the sums are reduced once per part. P is one 16-bit
//     number because both of the MMA's operands have V's type: a second term for the rest would double the
//     P V products and P's shared memory, at 128 rows of 256 at the cost of one of the ring's three slots.
//     The rounding adds at most u sum_j p_j |v_j|, of either sign, to an output that is itself rounded to u;
//     the row sums take the unrounded numbers;
// What a node must not see never reaches the MMA: scores are replaced, not added to, and in tiles
// that hold hidden keys the softmax warps clean V before it is used: rows that no node sees are zeroed; an
// infinity or NaN in a V row that some nodes see and others do not is taken out of the product and added
// back for those that do.
//
// Every wait is bounded (2 s); a block that gives up records it in a device word and leaves.
//
// Measured on one B200 (device time; GB/s of keys, values, queries and outputs read or written once):
// 8 sequences of up to 30000 keys, 9 nodes, 32 heads on 4 of 512: 235 us, 5900 GB/s, 0.90 of the
// measured copy rate; one node each: 213 us. 32 sequences, 64 nodes, 32 heads on 16 of 256, a window of
// 1024 keys: 126 us, 4470 GB/s: 512 short items of ten tiles, whose starts and ends (first maxima, sums,
// outputs) cost three tiles each, and at 128 rows the softmax of a tile, about 4500 cycles, is as
// long as its loads; with 32 nodes 100 us, with one 85. One node of one sequence of 96 keys: 8 us, a chain
// of latencies: launch, lengths, table, keys, two products, output.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"
#include "per_device.h"
#include "tcgen05.cuh"
#include "tma.cuh"
#include "tree_attn.h"

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <cstring>

namespace g4b {

namespace {

constexpr int kKeys = 128;           // keys per tile: the M of S^T
constexpr int kSoftWarps = 16;       // warps 0 .. 15, four groups of four
constexpr int kProducer = 16, kIssuer = 17, kScheduler = 18;  // and 19, the queries
constexpr int kThreads = 640;
// With two groups of twice the rows the row sums alone took 64 registers and spilled: 319 us instead of
// 259 for 9-node trees over 30000 keys. Scores held in registers from the look at their maxima to their
// exponentials spill too (193 us instead of 157 with 64-node trees): they are read from TMEM twice.
// Registers a thread: 96 at launch; 512 x 104 + 128 x 64 is the same total.
constexpr int kSoftRegs = 104, kOtherRegs = 64;
constexpr uint32_t kBoxBytes = kKeys * 128;  // 128 keys x 64 dims of 16 bits
constexpr int kMaxSlots = 8;
constexpr int kParts = 4;            // parts the scheduler is ahead
constexpr int kTreeBox = 8;          // node rows per TMA box: the swizzle's eight
// And at most 8 KB of cached rows: larger boxes leave more places empty between the cached keys and the
// nodes, smaller ones cost more copies. 8 x 30000 keys in 64-row pages, one node each, head dims 512 /
// 128 / 64: 227 / 79 / 81 us with 8 rows a box, 213 / 64 / 62 with 16, 211 / 66 / 53 with 32, 212 / 66 /
// 48 with 64.
constexpr int kBoxCopy = 8192;
constexpr float kUnset = 1e30f;      // negated reference of a row that has seen no key
constexpr float kLazy = 8.f;         // a reference moves when a score exceeds the maximum it was set to by 2^8
// A row's reference lies this far below that maximum, in powers of two: its probabilities, sum and output
// carry the factor until the end. fp16 is subnormal below 2^-14 and stops at 65504; with numbers of up to
// 2^(7 + 8) a probability keeps its 11 bits down to 2^-21 of the maximum and is lost below 2^-32, where
// without the factor a long row's tail was lost below 2^-25 (while the sum still counted it). bf16 has
// the exponents of fp32.
template <bool kBf16>
constexpr float kLift = kBf16 ? 0.f : 7.f;
constexpr size_t kSmemLimit = 232448 - 2048;  // leaves room for blocks of the second kernel
// What starting and finishing an item costs, in tiles, when the shares are cut: it grows with the rows,
// the tiles' time less so. 128 rows an item, dim 256: 131 us over a 1024-key window and 282 over up to
// 4096 keys at 3, 137 and 303 at 2; 64 rows, 13-node trees, dim 128: 22.9 us at 3, 21.4 at 2.
__host__ __device__ constexpr int item_cost(int rows) { return rows > 64 ? 3 : 2; }
// Items of at most this many tiles are not split, which saves the second kernel: one sequence of 300
// keys takes 10.5 us so and 11.1 split, one of 600 (5 tiles) 13.5 and 12.2.
constexpr int kWholeTiles = 4;
constexpr int kFewSeqs = 64;

__device__ int g_tree_err;  // set when a bounded wait gives up

// A part of an item: tiles t0 .. t1 - 1 of (sequence b, K/V head h, row group g).
struct Part {
    int b, h, g, t0, t1;
    // The part's keys stand in a line: `pre` cached ones from position `base` on (whole boxes, the last
    // of them may pass the sequence's end), then the nodes. Tile i is places 128 i .. 128 i + 127.
    int len, first, n, start, base, pre, tiles;
    // Places of tile i up to its last node.
    __device__ __forceinline__ int keys(int i) const { return min(kKeys, pre + n - i * kKeys); }
    // Whether some rows' windows start inside the tile, and whether some places are hidden from some row.
    __device__ __forceinline__ bool windowed(int window, int i) const {
        return window && i * kKeys < pre && base + i * kKeys < start + n - 1;
    }
    __device__ __forceinline__ bool edge(int window, int i) const {
        return (i + 1) * kKeys > len - base || base + i * kKeys < start || windowed(window, i);
    }
};

struct alignas(16) Ctl {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t s_full[2], s_free[2];
    uint64_t part_full[kParts], part_free[kParts];
    Part part[kParts];
    uint64_t q_ready[2], q_free, rows_free[2], p_full, o_done, v_ready[4], v_fix[4], done;
    uint32_t tmem_base;
    int abort, poison[2];
    int v_at[4];                  // slot and phase of an edge tile's V, 128 dims each
    int scan[kThreads / 32];      // units of each warp's run of sequences
    alignas(16) float corr[128];  // factor of a row's sum and output when its reference moves
    alignas(16) float inv[128];
    alignas(16) float red[4][128];
};

static_assert(offsetof(Ctl, corr) % 16 == 0 && offsetof(Ctl, inv) % 16 == 0 && alignof(Ctl) == 16,
              "read in 16-byte pieces");

// What a part's rows carry, twice: the next part's is set up before the current one is written out.
struct Rows {
    long long* out;   // offset of the row's output in elements
    float* nref;      // negated reference of a row, in powers of two
    int* start;       // first cached position a row sees
    int* depth;
    uint32_t* mask;   // [words][N]
};
constexpr int kRowBytes = 8 + 4 * 3;
__host__ __device__ constexpr size_t rows_bytes(int N, int words) { return (size_t)2 * N * (kRowBytes + 4 * words); }
__device__ __forceinline__ Rows rows_of(unsigned char* base, int N, int words, int par) {
    unsigned char* b = base + par * (N * (kRowBytes + 4 * words));
    Rows r;
    r.out = reinterpret_cast<long long*>(b);
    r.nref = reinterpret_cast<float*>(b + N * 8);
    r.start = reinterpret_cast<int*>(b + N * 12);
    r.depth = reinterpret_cast<int*>(b + N * 16);
    r.mask = reinterpret_cast<uint32_t*>(b + N * 20);
    return r;
}

// Division of a whole number below 2^31 by one fixed at launch: with s = ceil(log2 d) and m =
// floor(2^32 (2^s - d) / d) + 1, n / d = (n + mulhi(m, n)) >> s (Granlund and Montgomery).
struct Div {
    uint32_t d, m, s;
    __device__ __forceinline__ int quot(int n) const { return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> s); }
    __device__ __forceinline__ int rem(int n) const { return n - quot(n) * (int)d; }
};
Div make_div(int d) {
    Div x{(uint32_t)d, 0, 0};
    while ((1ll << x.s) < d) ++x.s;
    x.m = (uint32_t)((((1ull << x.s) - (unsigned)d) << 32) / (unsigned)d + 1);
    return x;
}

// An item that starts in a block and goes on in later ones, c0 .. c1 (none: c1 < c0); the first part's
// slot is `slot`, the others' are 2 c.
struct Split {
    int h, g, first, n, c0, c1, slot, total;
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
    Split* split;  // [blocks]
    long long q_stride, out_stride, page_stride, new_stride;  // elements
    int seqs, n_tokens, max_nodes, pages, page_size, width, mask_words, kv_heads, window;
    int N, words, slots, box, box_log, tmem_cols, whole, gqa;
    Div by_rows, by_gqa, by_page, by_grid;  // N, gqa, page_size and the number of blocks
    float c;       // scale * log2(e)
};

// One sequence's share of the work.
struct Seq {
    int len, first, n;   // cached tokens, first node, nodes
    int start, base;     // first cached position any node may see, and the first in the line of keys
    int pre, tiles, groups;  // cached places in that line, tiles, row groups
};

// The sequence's numbers as they stand in memory, within their bounds, and what follows from them.
__device__ __forceinline__ void read_seq(const Params& p, int b, Seq& s) {
    const int from = p.cu[b], to = p.cu[b + 1], len = p.lens[b];
    s.first = min(max(from, 0), p.n_tokens);
    s.n = min(min(max(to - s.first, 0), p.n_tokens - s.first), p.max_nodes);
    s.len = min(max(len, 0), p.width * p.page_size);
}
__device__ __forceinline__ void derive_seq(const Params& p, Seq& s) {
    s.start = p.window ? max(0, s.len - p.window + 1) : 0;
    s.base = s.start >> p.box_log << p.box_log;
    s.pre = (s.len - s.base + p.box - 1) >> p.box_log << p.box_log;
    if (s.start >= s.len) {
        s.base = s.start = s.len;
        s.pre = 0;
    }
    s.tiles = s.n ? (s.pre + s.n + kKeys - 1) / kKeys : 0;
    s.groups = p.by_rows.quot(s.n * p.gqa + p.N - 1);
}

// An item is as long as its tiles and item_cost(p.N) more, ahead of them; 1 where items stay whole.
__device__ __forceinline__ int item_units(const Params& p, const Seq& s) { return p.whole ? 1 : s.tiles + item_cost(p.N); }
__device__ __forceinline__ int seq_units(const Params& p, const Seq& s) {
    return s.tiles ? item_units(p, s) * s.groups * p.kv_heads : 0;
}
__device__ __forceinline__ int seq_units(const Params& p, int b) {
    Seq s;
    read_seq(p, b, s);
    derive_seq(p, s);
    return seq_units(p, s);
}

// First unit of block c when `total` units are dealt to the grid's blocks.
__device__ __forceinline__ int share_begin(const Params& p, int total, int c) {
    const int q = p.by_grid.quot(total);
    return q * c + p.by_grid.quot((total - q * (int)p.by_grid.d) * c);
}

// A place in the ring of slots and the parity of its current use.
struct Place {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void step(int slots) {
        if (++slot == slots) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// Bounded wait that also gives up as soon as another warp of the block has.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    const uint64_t t0 = global_ns();
#pragma unroll 1
    while (!mbar_try_wait_sleep(bar, parity, 1000000u))
        if (*abort || global_ns() - t0 > kWaitLimitNs) {
            *abort = 1;
            return false;
        }
    return true;
}

// Writes down the parts of this block's share, one by one (t0 = t1 ends them), and hands each to
// ready(part). One warp.
template <class Ready>
__device__ __forceinline__ void schedule(const Params& p, Ctl& c, volatile int* abort, Ready ready) {
    Place at;
    const int lane = threadIdx.x & 31;
    // This block's share of all units, and where it starts: skip whole runs, then sequences.
    int total = 0, first = 0, per = p.seqs, runs = 1;
    Seq mine{};
    if (p.seqs > kFewSeqs) {
        runs = kThreads / 32;
        per = (p.seqs + runs - 1) / runs;
        total = warp_sum_int(lane < runs ? c.scan[lane] : 0);
    } else {
#pragma unroll 1
        for (int b = lane; b < p.seqs; b += 32) {
            read_seq(p, b, mine);
            derive_seq(p, mine);
            total += seq_units(p, mine);
        }
        total = warp_sum_int(total);
    }
    int pos = share_begin(p, total, blockIdx.x), before = 0;
    const int end = share_begin(p, total, blockIdx.x + 1);
#pragma unroll 1
    for (; runs > 1 && before + c.scan[first] <= pos && first + 1 < runs; ++first) before += c.scan[first];
    first *= per;
    Seq s{};
    int b = 0, h = 0, g = 0, u = 0, parts = 0;
    if (lane == 0 && !p.whole) p.split[blockIdx.x] = Split{0, 0, 0, 0, 0, -1, 0, 0};
    if (pos < end) {
#pragma unroll 1
        for (int b0 = first; b0 < p.seqs; b0 += 32) {
            if (p.seqs > 32) {
                mine = Seq{};
                if (b0 + lane < p.seqs) read_seq(p, b0 + lane, mine);
                derive_seq(p, mine);
            }
            const int units = seq_units(p, mine);
            int x = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, pos < before + x);
            if (hit) {
                const int who = __ffs(hit) - 1;
                b = b0 + who;
                u = pos - before - __shfl_sync(0xffffffffu, x - units, who);
                s.first = __shfl_sync(0xffffffffu, mine.first, who);
                s.n = __shfl_sync(0xffffffffu, mine.n, who);
                s.len = __shfl_sync(0xffffffffu, mine.len, who);
                break;
            }
            before += __shfl_sync(0xffffffffu, x, 31);
        }
        derive_seq(p, s);
        const int item = item_units(p, s);
        h = u / (item * s.groups);
        u -= h * item * s.groups;
        g = u / item;
        u -= g * item;
    }
#pragma unroll 1
    while (true) {
        int t0 = 0, t1 = 0;
#pragma unroll 1
        while (pos < end && t0 == t1) {
            const int item = item_units(p, s);
            if (u == item) {
                u = 0;
                if (++g == s.groups) {
                    g = 0;
                    if (++h == p.kv_heads) {
                        h = 0;
                        do {
                            read_seq(p, ++b, s);
                            derive_seq(p, s);
                        } while (s.tiles == 0);
                    }
                }
                continue;
            }
            const int v = min(item, u + (end - pos));
            pos += v - u;
            t0 = p.whole ? 0 : max(0, u - item_cost(p.N));
            t1 = p.whole ? s.tiles : max(0, v - item_cost(p.N));
            u = v;
        }
        if (!p.whole && t0 < t1 && t0 == 0 && t1 < s.tiles) {
            // This block's last part, and the first of an item that others finish.
            const int z = pos + item_units(p, s) - u;  // the unit behind the item
            int last = blockIdx.x + 1;
            while (share_begin(p, total, last + 1) < z) ++last;
            if (lane == 0) p.split[blockIdx.x] = Split{h, g, s.first, s.n, (int)blockIdx.x, last, 2 * (int)blockIdx.x + (parts ? 1 : 0), total};
        }
        ++parts;
        if (!__all_sync(0xffffffffu, wait(&c.part_free[at.slot], at.phase ^ 1, abort))) return;
        const Part part{b, h, g, t0, t1, s.len, s.first, s.n, s.start, s.base, s.pre, s.tiles};
        if ((threadIdx.x & 31) == 0) {
            c.part[at.slot] = part;
            mbar_arrive(&c.part_full[at.slot]);
        }
        if (t0 == t1 || !ready(part)) return;
        at.step(kParts);
    }
}

// The next part, for a warp (or its one thread); false at the end.
__device__ __forceinline__ bool next_part(Ctl& c, Place& at, Part& w, bool leader, volatile int* abort) {
    if (!wait(&c.part_full[at.slot], at.phase, abort)) return false;
    w = c.part[at.slot];
    if (leader) mbar_arrive(&c.part_free[at.slot]);
    at.step(kParts);
    return w.t0 < w.t1;
}

__device__ __forceinline__ void group_bar(int grp) { asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory"); }
// The AND over the threads of the softmax warps.
__device__ __forceinline__ bool all_groups(bool v) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.and.pred q, 5, 512, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)v)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ bool group_or(int grp, bool v) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(1 + grp)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ void tma_3d(void* dst, uint64_t map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_5d(void* dst, uint64_t map, int x, int y, int z, int w, int v, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
        "[%7];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void st_shared_zero(uint32_t dst) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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

// Reduce-scatter of eight per-lane values over the warp: each of three exchanges sends the half the
// lane gives away, two more finish the four lanes that share a row. Lane 4 r + (0 .. 3) ends with
// row r's reduction in v[0].
template <bool kMax>
__device__ __forceinline__ void reduce_scatter8(float (&v)[8], int lane) {
    auto op = [](float a, float b) { return kMax ? fmaxf(a, b) : a + b; };
#pragma unroll
    for (int n = 4, bit = 16; n >= 1; n >>= 1, bit >>= 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) {
                const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
                v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, bit));
            }
    }
    v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], 2));
    v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], 1));
}

// Whether row r of the part sees place x of its line of keys.
__device__ __forceinline__ bool sees(const Params& p, const Part& w, const Rows& c, int x, int r) {
    if (x < w.pre) return w.base + x < w.len && w.base + x >= c.start[r];
    const int j = x - w.pre;
    if (j >= w.n || !((c.mask[(j >> 5) * p.N + r] >> (j & 31)) & 1)) return false;
    return !p.window || c.depth[r] - min(max(p.depth[w.first + j], 0), w.n - 1) < p.window;
}

__device__ __forceinline__ unsigned low_bits(int n) { return n >= 32 ? ~0u : (1u << max(n, 0)) - 1; }

// Bit j of lane i's word becomes bit i of lane j's.
__device__ __forceinline__ unsigned transpose_bits(unsigned x, int lane) {
    unsigned m = 0x0000ffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1, m ^= m << o) {
        const unsigned y = __shfl_xor_sync(0xffffffffu, x, o);
        x = lane & o ? (x & ~m) | ((y >> o) & m) : (x & m) | ((y << o) & ~m);
    }
    return x;
}

// Which rows of a group (up to 32) see this lane's key: cached position at + lane, or node j0 + lane from
// there on. A lane puts one row's view of the 32 keys together, from its `start` and its words of `mask`
// (N apart), and the warp turns the words over. Not inlined: the callers' sums stay in registers.
__device__ __forceinline__ unsigned seen_by(const int* start, const uint32_t* mask, int N, int at, int len, int j0, int n, int lane) {
    unsigned word = low_bits(len - at) & ~low_bits(*start - at);
    if (j0 > -32 && j0 < n) {
        unsigned low = mask[(max(j0, 0) >> 5) * N], high = 0;
        if (j0 < 0) low <<= -j0;
        else {
            if ((j0 | 31) + 1 < n) high = mask[((j0 >> 5) + 1) * N];
            low = __funnelshift_r(low, high, j0 & 31);
        }
        word |= low & low_bits(n - j0);
    }
    return transpose_bits(word, lane);
}
// Takes out the rows whose nodes are `window` or more levels below node j.
__device__ __forceinline__ unsigned within(unsigned seen, const int* row_depth, int rows, const int* depth, int j, int n, int window) {
    if (j < 0 || j >= n) return seen;
    const int near = min(max(depth[j], 0), n - 1) + window;
#pragma unroll 1
    for (int k = 0; k < rows; ++k)
        if (row_depth[k] >= near) seen &= ~(1u << k);
    return seen;
}

// V's row at place x (null: no such row).
__device__ const uint16_t* v_row(const Params& p, const Part& w, int x, int dim) {
    if (x < w.pre) {
        const int j = w.base + x;
        if (j < w.start || j >= w.len) return nullptr;
        const int page = p.table[(long long)w.b * p.width + j / p.page_size];
        if (page < 0 || page >= p.pages) return nullptr;
        return reinterpret_cast<const uint16_t*>(p.v_pool) + page * p.page_stride +
               ((long long)(j % p.page_size) * p.kv_heads + w.h) * dim;
    }
    if (x - w.pre >= w.n) return nullptr;
    return reinterpret_cast<const uint16_t*>(p.v_new) + (w.first + x - w.pre) * p.new_stride + w.h * dim;
}

// What the infinities and NaN taken out of this part's V tiles add to row r in dimension d.
template <bool kBf16>
__device__ __noinline__ float poison_of(const Params& p, Part w, Rows c, int dim, int d, int r) {
    float sum = 0.f;
    for (int i = w.t0; i < w.t1; ++i) {
        if (!w.edge(p.window, i)) continue;
        for (int x = i * kKeys; x < i * kKeys + w.keys(i); ++x) {
            if (x < w.pre && !w.windowed(p.window, i)) continue;  // seen by all: still in the product
            const uint16_t* row = v_row(p, w, x, dim);
            if (row && not_finite<kBf16>(row[d]) && sees(p, w, c, x, r)) sum += unpack1<kBf16>(row[d]);
        }
    }
    return sum;
}

// V of an edge tile, 64 x kHalves dims of it: keys 0 .. lead - 1, held .. nodes - 1 and from `keys` to the
// MMA's next step of 16 are nobody's and become zeros; keys lead .. mixed - 1 and nodes .. keys - 1 lose
// their infinities and NaN, which is noted in *found. All softmax warps.
template <int kHalves, bool kBf16>
__device__ __forceinline__ void clean_v(unsigned char* slot, int lead, int mixed, int held, int nodes, int keys, volatile int* found) {
#pragma unroll 1
    for (int x = threadIdx.x; x < ((keys + 15) & ~15) * 8 * kHalves; x += kSoftWarps * 32) {
        const int k = x / (8 * kHalves);  // sixteen bytes of this key
        uint4* at = reinterpret_cast<uint4*>(slot + (k >> 3) * (kHalves * 1024) + (x % (8 * kHalves) >> 3) * 1024 + (k & 7) * 128 + (x & 7) * 16);
        if (k < lead || (k >= held && k < nodes) || k >= keys) {
            *at = make_uint4(0, 0, 0, 0);
        } else if (k < mixed || k >= nodes) {
            const uint4 v = *at;
            const uint32_t bits = kBf16 ? 0x7f807f80u : 0x7c007c00u;  // the exponents
            if (!(__vcmpeq2(v.x & bits, bits) | __vcmpeq2(v.y & bits, bits) | __vcmpeq2(v.z & bits, bits) | __vcmpeq2(v.w & bits, bits))) continue;
            uint16_t* h = reinterpret_cast<uint16_t*>(at);
#pragma unroll 1
            for (int y = 0; y < 8; ++y)
                if (not_finite<kBf16>(h[y])) h[y] = 0;
            *found = 1;
        }
    }
}

// kNH: the most rows a softmax group takes.
template <int D, int kNH, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ CUtensorMap knmap, const __grid_constant__ CUtensorMap vnmap,
                     const __grid_constant__ Params p) {
    constexpr int kHalves = D == 64 ? 1 : 2;                // 64-dim boxes per slot
    constexpr int kChunks = D == 64 ? 1 : D / 128;          // slots per K or V tile
    constexpr uint32_t kSlotBytes = kHalves * kBoxBytes;
    constexpr uint32_t kRows8 = kHalves * 1024;             // eight keys of a slot: [64-dim block][key][64 dims]
    extern __shared__ unsigned char smem_raw[];
    // An offset, not a rounded pointer: the compiler still sees shared memory, and uses its 32-bit
    // addresses and instructions.
    unsigned char* sm = smem_raw + (-smem_u32(smem_raw) & 1023u);
    const int N = p.N, slots = p.slots;
    unsigned char* ring = sm;
    unsigned char* qs = ring + slots * kSlotBytes;             // [D / 64][N rows][64 dims]
    unsigned char* ps = qs + (D / 64) * N * 128;               // [N / 64][128 keys][64 rows]
    unsigned char* rows_at = ps + ((N + 63) / 64) * kBoxBytes;  // row state
    Ctl& c = *reinterpret_cast<Ctl*>(rows_at + rows_bytes(N, p.words));
    volatile int* abort = &c.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0) {  // a lane or two per kind of barrier: one after another they take a microsecond
        const auto init = [&](int from, int n, uint64_t* bars, uint32_t count) {
            if (lane >= from && lane < from + n) mbar_init(bars + lane - from, count);
        };
        init(0, kMaxSlots, c.full, 1);
        init(0, kMaxSlots, c.empty, 1);
        init(8, 2, c.s_full, 1);
        init(8, 2, c.s_free, kSoftWarps);
        init(10, 2, c.q_ready, 2);
        init(10, 2, c.rows_free, kSoftWarps);
        init(12, kParts, c.part_full, 1);
        init(12, kParts, c.part_free, kSoftWarps + 3);
        init(16, 4, c.v_ready, 1);
        init(16, 4, c.v_fix, kSoftWarps);
        init(20, 1, &c.q_free, 1);
        init(21, 1, &c.p_full, kSoftWarps);
        init(22, 1, &c.o_done, 1);
        init(23, 1, &c.done, 1);
        if (lane == 24) c.abort = 0;
        mbar_init_fence();
    }
    if (warp == kIssuer) tc::alloc(&c.tmem_base, p.tmem_cols);

    // With few sequences the scheduling warp adds them up by itself, below; with many each warp adds a run.
    if (p.seqs > kFewSeqs) {
        const int per = (p.seqs + kThreads / 32 - 1) / (kThreads / 32);
        int mine = 0;
#pragma unroll 1
        for (int b = warp * per + lane; b < min(p.seqs, (warp + 1) * per); b += 32) mine += seq_units(p, b);
        mine = warp_sum_int(mine);
        if (lane == 0) c.scan[warp] = mine;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = c.tmem_base;
    const uint32_t o_col = 2 * (uint32_t)N;  // S^T buffers, then the O^T tiles of 128 dims
    pdl_launch_dependents();

    if (warp == kProducer) {
        // ------------------------------------------------------------------ producer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        Part w;
        Place at, list;
        int used = 0;
        bool ok = true;
        const int kb = lane;  // up to 16 key boxes
        const uint64_t kd = reinterpret_cast<uint64_t>(&kmap), vd = reinterpret_cast<uint64_t>(&vmap);
        const uint64_t knd = reinterpret_cast<uint64_t>(&knmap), vnd = reinterpret_cast<uint64_t>(&vnmap);
#pragma unroll 1
        while (ok) {
            ok = next_part(c, list, w, false, abort);
            ok = __all_sync(0xffffffffu, ok);  // every lane has its copy
            if (lane == 0) mbar_arrive(&c.part_free[(list.slot + kParts - 1) % kParts]);
            if (!ok) break;
            const int32_t* row = p.table + (long long)w.b * p.width;
            // Boxes of tile i: cached rows, then nodes; one of up to 16 is this lane's.
            auto cached = [&](int i) { return min(kKeys, max(0, w.pre - i * kKeys)) >> p.box_log; };
            auto ids = [&](int i) {  // its page
                return kb < cached(i) ? row[p.by_page.quot(w.base + i * kKeys + kb * p.box)] : -1;
            };
            int id0 = -1, id1 = ids(w.t0), id2 = -1;
#pragma unroll 1
            for (int st = 2 * w.t0; st <= 2 * w.t1 + 1 && ok; ++st) {  // K of tile i = st / 2, then V of tile i - 1
                const bool is_v = st & 1;
                const int tile = is_v ? (st >> 1) - 1 : st >> 1;
                if (!is_v) id2 = tile + 1 < w.t1 ? ids(tile + 1) : -1;
                const int page = is_v ? id0 : id1;
                if (is_v) {
                    id0 = id1;
                    id1 = id2;
                }
                if (tile < w.t0 || tile >= w.t1) continue;
                const int nc = cached(tile), from = nc * p.box, nn = max(0, w.keys(tile) - from + kTreeBox - 1) / kTreeBox;
                const bool old = kb < nc, mine = kb < nc + nn;
                const int at_row = old ? kb * p.box : from + (kb - nc) * kTreeBox;
                const int x = tile * kKeys + at_row;
                // A page id out of range is an out-of-range coordinate: the box reads as zeros.
                const int z = old ? p.by_page.rem(w.base + x) : w.first + x - w.pre;
                const int pg = page < 0 ? p.pages : page;
                const uint64_t map = old ? (is_v ? vd : kd) : (is_v ? vnd : knd);
                const uint32_t bytes = (uint32_t)(from + nn * kTreeBox) * 128 * kHalves;
#pragma unroll 1
                for (int ci = 0; ci < kChunks; ++ci) {
                    ok = wait(&c.empty[at.slot], at.phase ^ 1, abort);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&c.full[at.slot], bytes);
                    __syncwarp();
                    if (mine) {
                        unsigned char* dst = ring + at.slot * kSlotBytes + (at_row >> 3) * kRows8;
                        const int block = w.h * (D / 64) + ci * kHalves;
                        if (old) tma_5d(dst, map, 0, 0, block, z >> 3, pg, &c.full[at.slot]);
                        else tma_3d(dst, map, 0, z, block, &c.full[at.slot]);
                    }
                    at.step(slots);
                    ++used;
                }
            }
        }
        // Every issued copy lands before the block can exit: the last use of each slot.
        if (lane == 0) {
#pragma unroll 1
            for (int i = max(0, used - slots); i < used; ++i)
                if (!mbar_wait(&c.full[i % slots], (i / slots) & 1)) *abort = 1;
        }
    } else if (warp == kIssuer) {
        // ------------------------------------------------------------------ MMA issuer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        // The whole warp walks the loops, one lane issues: what the instructions need is the same in
        // every lane and can stay in uniform registers.
        const bool leader = tc::elect();
        Part w;
        Place list;
        const uint32_t id_s = tc::idesc_16(kKeys, N, kBf16, false, false);
        const uint32_t id_o = tc::idesc_16(128, N, kBf16, true, true);
        // Descriptors of the ring's first slot, of Q and of P; other places add their distance in
        // 16-byte units.
        const uint64_t k_desc = tc::desc_sw128(smem_u32(ring), kRows8), v_desc = tc::desc_sw128_mn(smem_u32(ring), 1024, kRows8);
        const uint64_t q_desc = tc::desc_sw128(smem_u32(qs)), p_desc = tc::desc_sw128_mn(smem_u32(ps), kBoxBytes, 1024);
        const uint32_t blk = (uint32_t)N * 8;  // one 64-dim block of Q
        // V chunks that fit the ring beside nothing else: the cleaning of an edge tile's first ones
        // can start before its P is there.
        const int ahead = min(kChunks, slots);
        const auto show_v = [&](int ci, const Place& x) {
            *(volatile int*)&c.v_at[ci] = 2 * x.slot + x.phase;
            mbar_arrive(&c.v_ready[ci]);
        };
        Place at;
        int tile = 0, otile = 0, part = 0, fix = 0;
        bool ok = true;
#pragma unroll 1
        while (ok) {
            ok = __all_sync(0xffffffffu, next_part(c, list, w, false, abort));
            if (leader) mbar_arrive(&c.part_free[(list.slot + kParts - 1) % kParts]);
            if (!ok) break;
            const int t0 = __shfl_sync(0xffffffffu, w.t0, 0), t1 = __shfl_sync(0xffffffffu, w.t1, 0);
            ok = __all_sync(0xffffffffu, wait(&c.q_ready[part & 1], (part >> 1) & 1, abort));
            ++part;
            // S of tile i, then O of tile i - 1.
#pragma unroll 1
            for (int i = t0; i <= t1 && ok; ++i) {
                if (i < t1) {
                    const int b = tile & 1;
                    if (tile >= 2) ok = wait(&c.s_free[b], ((tile >> 1) - 1) & 1, abort);
#pragma unroll 1
                    for (int ci = 0; ci < kChunks; ++ci) {
                        ok = ok && wait(&c.full[at.slot], at.phase, abort);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc::fence_after_sync();
                        const uint64_t a = k_desc + at.slot * (kSlotBytes >> 4), q = q_desc + 2 * ci * blk;
                        if (leader) {
#pragma unroll
                            for (int kk = 0; kk < 4 * kHalves; ++kk)
                                tc::mma_ss(tmem + b * N, a + (kk >> 2) * (1024 >> 4) + (kk & 3) * 2,
                                           q + (kk >> 2) * blk + (kk & 3) * 2, id_s, (ci | kk) ? 1u : 0u);
                            tc::commit(&c.empty[at.slot]);
                        }
                        at.step(slots);
                    }
                    if (leader) {
                        tc::commit(&c.s_full[b]);
                        if (i + 1 == t1) tc::commit(&c.q_free);
                    }
                    ++tile;
                }
                if (i > t0 && ok) {
                    const int steps = __shfl_sync(0xffffffffu, (w.keys(i - 1) + 15) >> 4, 0);
                    const bool edge = w.edge(p.window, i - 1);
                    Place look = at;
#pragma unroll 1
                    for (int ci = 0; ci < ahead && edge; ++ci) {
                        ok = ok && wait(&c.full[look.slot], look.phase, abort);
                        if (leader) show_v(ci, look);
                        look.step(slots);
                    }
                    ok = ok && wait(&c.p_full, otile & 1, abort);
#pragma unroll 1
                    for (int ci = 0; ci < kChunks; ++ci) {
                        ok = ok && wait(&c.full[at.slot], at.phase, abort);
                        if (edge) {  // cleaned first
                            if (ci >= ahead && leader) show_v(ci, at);
                            ok = ok && wait(&c.v_fix[ci], fix & 1, abort);
                        }
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc::fence_after_sync();
                        const uint64_t a = v_desc + at.slot * (kSlotBytes >> 4);
                        const uint32_t d = tmem + o_col + ci * N, more = i - 1 > t0 ? 1u : 0u;
                        // V^T rows are the slot's dims (with D = 64 the lanes 64 .. 127 multiply whatever
                        // follows in shared memory, and are never read).
                        if (leader) {
                            if (steps == 8) {
#pragma unroll
                                for (int kk = 0; kk < 8; ++kk)
                                    tc::mma_ss(d, a + kk * (2 * kRows8 >> 4), p_desc + kk * 128, id_o, kk ? 1u : more);
                            } else {
#pragma unroll 1
                                for (int kk = 0; kk < steps; ++kk)
                                    tc::mma_ss(d, a + kk * (2 * kRows8 >> 4), p_desc + kk * 128, id_o, kk ? 1u : more);
                            }
                            tc::commit(&c.empty[at.slot]);
                        }
                        at.step(slots);
                    }
                    if (leader) tc::commit(&c.o_done);
                    fix += edge;
                    ++otile;
                }
            }
        }
        if (leader) {
            tc::commit(&c.done);  // every MMA has completed before tensor memory is freed
            if (!mbar_wait(&c.done, 0)) *abort = 1;
        }
    } else if (warp < kSoftWarps) {
        // ------------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        Part w;
        Place list;
        const int grp = warp >> 2, qd = warp & 3;
        const int gt = threadIdx.x & 127;                 // place in the group
        const int key = qd * 32 + lane;                   // TMEM lane
        // The group's rows r0 .. r0 + nh - 1, in eights; with few rows some groups have none.
        const int r0 = (N >> 3) * grp / 4 * 8, nh = (N >> 3) * (grp + 1) / 4 * 8 - r0;
        const uint32_t lanes = (uint32_t)(qd * 32) << 16;
        int tile = 0, fix = 0;
        float l[kNH];
        // After a wait that gave up, these warps go on (on meaningless values) to the end of the share:
        // none of them may leave while others stand at a barrier of the group.
#pragma unroll 1
        for (int part = 0;; ++part) {
            const bool more = all_groups(next_part(c, list, w, false, abort));
            if (lane == 0) mbar_arrive(&c.part_free[(list.slot + kParts - 1) % kParts]);
            if (!more) break;
            const Rows rs = rows_of(rows_at, N, p.words, part & 1);
            wait(&c.q_ready[part & 1], (part >> 1) & 1, abort);
#pragma unroll
            for (int r = 0; r < kNH; ++r) l[r] = 0.f;

#pragma unroll 1
            for (int i = w.t0; i < w.t1; ++i, ++tile) {
                const int b = tile & 1;
                const uint32_t st = tmem + lanes + b * N + r0;
                wait(&c.s_full[b], (tile >> 1) & 1, abort);
                __syncwarp();
                tc::fence_after_sync();
                const bool edge = w.edge(p.window, i);
                const bool fresh = i == w.t0;
                unsigned seen = ~0u;
                if (edge) {
                    const int x0 = i * kKeys + qd * 32, r = min(r0 + lane, N - 1);
                    seen = seen_by(rs.start + r, rs.mask + r, N, w.base + x0, w.len, x0 - w.pre, w.n, lane);
                    if (p.window && p.window < w.n) seen = within(seen, rs.depth + r0, nh, p.depth + w.first, x0 - w.pre + lane, w.n, p.window);
                }
                // First look. Hidden scores become -inf, in tensor memory too. In a part's first tile each
                // row's maximum is taken; later it matters whether a score exceeds its row's reference by
                // more than kLazy. The scores are read again for the exponentials, which leaves the
                // registers to the row sums.
                float over = -INFINITY;
#pragma unroll 1
                for (int g = 0; g < nh; g += 8) {
                    float v[8];
                    tc::ld8(st + g, v);
                    tc::wait_ld();
                    if (edge) {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (!((seen >> g >> k) & 1)) v[k] = -INFINITY;
                        tc::st8(st + g, v);
                    }
                    if (fresh) {
                        reduce_scatter8<true>(v, lane);
                        c.red[qd][r0 + g + (lane >> 2)] = v[0] * p.c;
                    } else {
                        const float4 n0 = *reinterpret_cast<const float4*>(&rs.nref[r0 + g]), n1 = *reinterpret_cast<const float4*>(&rs.nref[r0 + g + 4]);
                        over = fmaxf(over, fmaxf(fmaf(v[0], p.c, n0.x), fmaf(v[1], p.c, n0.y)));
                        over = fmaxf(over, fmaxf(fmaf(v[2], p.c, n0.z), fmaf(v[3], p.c, n0.w)));
                        over = fmaxf(over, fmaxf(fmaf(v[4], p.c, n1.x), fmaf(v[5], p.c, n1.y)));
                        over = fmaxf(over, fmaxf(fmaf(v[6], p.c, n1.z), fmaf(v[7], p.c, n1.w)));
                    }
                }
                if (edge) tc::wait_st();
                bool waited = tile == 0;
                if (fresh || group_or(grp, over > kLazy + kLift<kBf16>)) {
#pragma unroll 1
                    for (int f = 0; f < nh && !fresh; f += 8) {
                        float m[8];
                        tc::ld8(st + f, m);
                        tc::wait_ld();
                        reduce_scatter8<true>(m, lane);
                        c.red[qd][r0 + f + (lane >> 2)] = m[0] * p.c;
                    }
                    group_bar(grp);
                    if (gt < nh) {
                        const int r = r0 + gt;
                        const float top = fmaxf(fmaxf(c.red[0][r], c.red[1][r]), fmaxf(c.red[2][r], c.red[3][r]));
                        const float old = rs.nref[r];
                        float f = 1.f;
                        if (top > -INFINITY && (old == kUnset || top + old > kLazy + kLift<kBf16>)) {
                            f = old == kUnset ? 0.f : exp2_approx(kLift<kBf16> - old - top);
                            rs.nref[r] = kLift<kBf16> - top;
                        }
                        c.corr[r] = f;
                    }
                    group_bar(grp);
#pragma unroll
                    for (int r = 0; r < kNH; r += 4)
                        if (r < nh && !fresh) {
                            const float4 f = *reinterpret_cast<const float4*>(&c.corr[r0 + r]);
                            l[r] *= f.x;
                            l[r + 1] *= f.y;
                            l[r + 2] *= f.z;
                            l[r + 3] *= f.w;
                        }
                    if (!fresh) {
                        wait(&c.o_done, (tile - 1) & 1, abort);
                        __syncwarp();
                        waited = true;
                        tc::fence_after_sync();
#pragma unroll 1
                        for (int f = 0, ta = tmem + lanes + o_col + r0, ci = 0; ci < kChunks; f += 8, ta += 8) {
                            if (f == nh) {
                                f = 0;
                                ta += N - nh;
                                if (++ci == kChunks) break;
                            }
                            float v[8];
                            tc::ld8(ta, v);
                            tc::wait_ld();
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] *= c.corr[r0 + f + j];
                            tc::st8(ta, v);
                        }
                        tc::wait_st();
                    }
                }
                // P V of the tile before has read the buffer.
                if (!waited) wait(&c.o_done, (tile - 1) & 1, abort);
                unsigned char* const prow = ps + key * 128;
#pragma unroll
                for (int f = 0; f < kNH; f += 8)
                    if (f < nh) {
                        float v[8];
                        tc::ld8(st + f, v);
                        tc::wait_ld();
                        uint32_t pk[4];
#pragma unroll
                        for (int r = 0; r < 8; r += 4) {
                            const float4 n = *reinterpret_cast<const float4*>(&rs.nref[r0 + f + r]);
                            const float e0 = exp2_approx(fmaf(v[r], p.c, n.x)), e1 = exp2_approx(fmaf(v[r + 1], p.c, n.y));
                            const float e2 = exp2_approx(fmaf(v[r + 2], p.c, n.z)), e3 = exp2_approx(fmaf(v[r + 3], p.c, n.w));
                            l[f + r] += e0;
                            l[f + r + 1] += e1;
                            l[f + r + 2] += e2;
                            l[f + r + 3] += e3;
                            pk[r / 2] = pack2<kBf16>(e0, e1);
                            pk[r / 2 + 1] = pack2<kBf16>(e2, e3);
                        }
                        const int r = r0 + f;
                        *reinterpret_cast<uint4*>(prow + (r >> 6) * kBoxBytes + ((((r & 63) >> 3) ^ (key & 7)) << 4)) =
                            make_uint4(pk[0], pk[1], pk[2], pk[3]);
                    }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.s_free[b]);
                fence_proxy_async();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.p_full);

                if (edge) {
                    // V's rows that no row may see become zeros (they may hold anything, and 0 x NaN is NaN);
                    // rows that only some see lose their infinities and NaN, which are noted and added to those
                    // rows' outputs. Nobody's rows: before every window, from the sequence's end to its first
                    // node, past the last node. Rows that some see and others do not: where windows start, and
                    // the nodes.
                    const int keys = w.keys(i), at = w.base + i * kKeys, nodes = min(kKeys, max(0, w.pre - i * kKeys));
                    const int held = min(nodes, max(0, w.len - at));
                    const int lead = max(0, min(held, w.start - at));
                    const int mixed = p.window ? min(held, max(lead, w.start + w.n - 1 - at)) : lead;
#pragma unroll 1
                    for (int ci = 0; ci < kChunks; ++ci) {
                        // The issuing warp shows where V is once it is there: the slot might still be a use
                        // behind, and a parity cannot tell a phase from the one two before it.
                        bool ok = wait(&c.v_ready[ci], fix & 1, abort);
                        const int v_at = *(volatile int*)&c.v_at[ci];
                        ok = ok && wait(&c.full[v_at >> 1], v_at & 1, abort);
                        if (ok) clean_v<kHalves, kBf16>(ring + (v_at >> 1) * kSlotBytes, lead, mixed, held, nodes, keys, &c.poison[part & 1]);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&c.v_fix[ci]);
                    }
                    ++fix;
                }
            }

            // The part's result: sums over the keys, then O^T.
            group_bar(grp);
#pragma unroll
            for (int r = 0; r < kNH; r += 8)
                if (r < nh) {
                    float m[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) m[j] = l[r + j];
                    reduce_scatter8<false>(m, lane);
                    c.red[qd][r0 + r + (lane >> 2)] = m[0];
                }
            group_bar(grp);
            const bool whole = w.t1 - w.t0 == w.tiles;
            const int slot = 2 * blockIdx.x + (part ? 1 : 0);
            if (gt < nh) {
                const int r = r0 + gt;
                const float sum = (c.red[0][r] + c.red[1][r]) + (c.red[2][r] + c.red[3][r]);
                c.inv[r] = sum != 0.f ? 1.f / sum : 0.f;
                if (!whole) p.ml[(long long)slot * N + r] = make_float2(rs.nref[r] == kUnset ? -INFINITY : -rs.nref[r], sum);
            }
            group_bar(grp);
            wait(&c.o_done, (tile - 1) & 1, abort);
            __syncwarp();
            tc::fence_after_sync();
            const int held = min(nh, min(N, w.n * p.gqa - w.g * N) - r0);  // the group's rows that exist
            const uint32_t ot = tmem + lanes + o_col + r0;
            if (*(volatile int*)&c.poison[part & 1]) {
#pragma unroll 1
                for (int ci = 0; ci < kChunks; ++ci)
#pragma unroll 1
                    for (int f = 0; f < held; f += 8) {
                        float v[8];
                        tc::ld8(ot + ci * N + f, v);
                        tc::wait_ld();
                        if (128 * ci + key < D)
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] += poison_of<kBf16>(p, w, rs, D, 128 * ci + key, r0 + f + j);
                        __syncwarp();
                        tc::st8(ot + ci * N + f, v);
                    }
                tc::wait_st();
            }
#pragma unroll 1
            for (int ci = 0; ci < kChunks; ++ci) {
                const int d = 128 * ci + key;
                uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + d;
                float* dst = p.part + ((long long)slot * N + r0) * D + d;
#pragma unroll 1
                for (int g = 0; g < held; g += 8) {
                    float v[8];
                    tc::ld8(ot + ci * N + g, v);
                    tc::wait_ld();
                    if (D == 64 && key >= 64) continue;
                    if (whole) {
                        // Lanes swap so that each holds two dims of four rows: fewer, wider stores.
                        const float4 i0 = *reinterpret_cast<const float4*>(&c.inv[r0 + g]), i1 = *reinterpret_cast<const float4*>(&c.inv[r0 + g + 4]);
                        v[0] *= i0.x, v[1] *= i0.y, v[2] *= i0.z, v[3] *= i0.w;
                        v[4] *= i1.x, v[5] *= i1.y, v[6] *= i1.z, v[7] *= i1.w;
                        const bool odd = lane & 1;
                        const int row = r0 + g + (odd ? 4 : 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float got = __shfl_xor_sync(0xffffffffu, odd ? v[e] : v[e + 4], 1);
                            const uint32_t two = odd ? pack2<kBf16>(got, v[e + 4]) : pack2<kBf16>(v[e], got);
                            if (row + e - r0 < held) *reinterpret_cast<uint32_t*>(out + rs.out[row + e] - odd) = two;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (g + e < held) __stcg(dst + (g + e) * D, v[e]);
                    }
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.rows_free[part & 1]);
        }
    } else if (warp == kScheduler) {
        // ------------------------------------------------------------------ scheduler
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        // Deals the parts out, and sets up each part's rows while the one before is worked on.
        int part = 0;
        schedule(p, c, abort, [&](const Part& w) {
            const int par = part & 1, row0 = w.g * N;
            const Rows rs = rows_of(rows_at, N, p.words, par);
            // Rows of a part: r -> node (g N + r) / gqa, query head h gqa + (g N + r) % gqa.
            const bool ok = part < 2 || wait(&c.rows_free[par], ((part >> 1) - 1) & 1, abort);
            ++part;
            if (!__all_sync(0xffffffffu, ok)) return false;
#pragma unroll 1
            for (int r = lane; r < N; r += 32) {
                const int node = p.by_gqa.quot(row0 + r), hd = row0 + r - node * p.gqa, tok = w.first + min(node, w.n - 1);
                rs.out[r] = tok * p.out_stride + (w.h * p.gqa + hd) * D;
                rs.nref[r] = kUnset;
                const int dep = p.window ? min(max(p.depth[tok], 0), w.n - 1) : 0;
                rs.depth[r] = dep;
                rs.start[r] = p.window ? max(0, w.len + dep - p.window + 1) : 0;
#pragma unroll 1
                for (int i = 0; i * 32 < w.n; ++i) rs.mask[i * N + r] = p.mask[(long long)tok * p.mask_words + i];
            }
            if (lane == 0) c.poison[par] = 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.q_ready[par]);
            return true;
        });
    } else {
        // ------------------------------------------------------------------ queries
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        // Each part's queries into the MMA's K-major layout, once S of the part before has completed.
        // Eight rows at once, four lanes on 64 bytes of each: a lane's rows all have its place in the swizzle.
        const int sub = lane >> 2, q4 = lane & 3;
        const uint32_t q_at = smem_u32(qs), even = (q4 ^ sub) << 4, odd = ((q4 + 4) ^ sub) << 4;
        Part w;
        Place list;
#pragma unroll 1
        for (int part = 0;; ++part) {
            bool ok = __all_sync(0xffffffffu, next_part(c, list, w, false, abort));
            if (lane == 0) mbar_arrive(&c.part_free[(list.slot + kParts - 1) % kParts]);
            ok = ok && (part == 0 || wait(&c.q_free, (part - 1) & 1, abort));
            if (!__all_sync(0xffffffffu, ok)) break;
            const int row0 = w.g * N, R = min(N, w.n * p.gqa - row0);
#pragma unroll 2
            for (int r = sub; r < N; r += 8) {
                const int node = p.by_gqa.quot(row0 + r), hd = row0 + r - node * p.gqa;
                const char* from = p.q + 2 * ((w.first + node) * p.q_stride + (w.h * p.gqa + hd) * D + q4 * 8);
                uint32_t to = q_at + r * 128;
#pragma unroll
                for (int k = 0; k < D / 32; k += 2, to += N * 128) {
                    if (r < R) {
                        cp_async16(to + even, from + k * 64);
                        cp_async16(to + odd, from + k * 64 + 64);
                    } else {
                        st_shared_zero(to + even);
                        st_shared_zero(to + odd);
                    }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.q_ready[part & 1]);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && *abort) atomicExch(&g_tree_err, 1);
    if (warp == kIssuer) {
        tc::fence_after_sync();
        tc::dealloc(tmem, p.tmem_cols);
    }
}

constexpr int kJoinRows = 4;

// Joins the parts of items that several blocks worked on: out = sum_s 2^(m_s - M) O_s over
// sum_s 2^(m_s - M) l_s. A warp per row, kJoinRows rows a block; grid (blocks of the first kernel, row
// blocks): an item belongs to the block it starts in, which wrote down where the others are.
template <int D, bool kBf16>
__global__ void __launch_bounds__(32 * kJoinRows) tree_attn_join_kernel(const __grid_constant__ Params p) {
    const int lane = threadIdx.x & 31, r = blockIdx.y * kJoinRows + (threadIdx.x >> 5);
    pdl_wait();
    const Split s = p.split[blockIdx.x];
    const int row = s.g * p.N + r, c0 = s.c0, c1 = s.c1, h = s.h;
    if (c1 < c0 || r >= p.N || row >= s.n * p.gqa) return;
    const auto slot_of = [&](int c) { return (long long)(c == c0 ? s.slot : 2 * c); };
    float top = -INFINITY;
    for (int c = c0 + lane; c <= c1; c += 32) {
        if (share_begin(p, s.total, c) == share_begin(p, s.total, c + 1)) continue;  // a block without work
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
        if (share_begin(p, s.total, c) == share_begin(p, s.total, c + 1)) continue;  // a block without work
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
    const int node = p.by_gqa.quot(row);
    uint32_t* out = reinterpret_cast<uint32_t*>(p.out + 2 * ((s.first + node) * p.out_stride + (h * p.gqa + row - node * p.gqa) * D));
#pragma unroll
    for (int k = 0; k < kL; ++k)
#pragma unroll
        for (int j = 0; j < kV; j += 2)
            out[(k * 32 + lane) * (kV / 2) + j / 2] = pack2<kBf16>(o[k][j] * inv, o[k][j + 1] * inv);
}

// Multiprocessors of the current device.
int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    const bool kept = dev >= 0 && dev < 64;
    if (kept && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    if (kept) known[dev].store(n, std::memory_order_relaxed);
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
    int N, words, slots, tmem;
    size_t smem;
};
Shape shape_for(int max_nodes, int gqa, int dim) {
    Shape s;
    s.N = rows_per_item(max_nodes, gqa, dim);
    const size_t slot = (dim == 64 ? 1 : 2) * kBoxBytes;
    s.words = (max_nodes + 31) / 32;
    const size_t rest = 1024 + (size_t)s.N * dim * 2 + (size_t)((s.N + 63) / 64) * kBoxBytes + rows_bytes(s.N, s.words) + sizeof(Ctl);
    s.slots = (int)std::min<size_t>(kMaxSlots, (kSmemLimit - rest) / slot);
    s.smem = rest + s.slots * slot;
    const int cols = s.N * (2 + std::max(1, dim / 128));
    s.tmem = 32;
    while (s.tmem < cols) s.tmem *= 2;
    return s;
}

// Rows of a TMA box: the largest power of two that divides a page, so that a box never crosses one.
int box_rows(const TreeAttnArgs& a) {
    return std::min(kBoxCopy / (a.dim == 64 ? 128 : 256), a.page_size & -a.page_size);
}
// The most tiles an item can have, and the most items.
long long most_tiles(const TreeAttnArgs& a) {
    return ((long long)a.width * a.page_size + 2 * box_rows(a) + a.max_nodes + kKeys - 1) / kKeys;
}
long long most_items(const TreeAttnArgs& a, int N) {
    return (long long)a.seqs * a.kv_heads * ((a.max_nodes * (a.heads / a.kv_heads) + N - 1) / N);
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
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, const_cast<void*>(base), dims, strides, box, one,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int D, int kNH, bool kBf16>
cudaError_t run(const CUtensorMap* maps, const Params& p, const Shape& sh, cudaStream_t st) {
    auto kern = tree_attn_kernel<D, kNH, kBf16>;
    static OncePerDevice attributes;
    cudaError_t e = attributes([&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit);
    });
    if (e != cudaSuccess) return e;
    e = launch(kern, dim3(p.by_grid.d), dim3(kThreads), sh.smem, st, false, maps[0], maps[1], maps[2], maps[3], p);
    if (e != cudaSuccess || p.whole) return e;
    return launch(tree_attn_join_kernel<D, kBf16>, dim3(p.by_grid.d, (p.N + kJoinRows - 1) / kJoinRows),
                  dim3(32 * kJoinRows), 0, st, true, p);
}

template <int D, bool kBf16>
cudaError_t run_rows(const CUtensorMap* maps, const Params& p, const Shape& sh, cudaStream_t st) {
    const int units = (sh.N / 8 + 3) / 4;  // rows of the largest softmax group, in eights
    if (units <= 1) return run<D, 8, kBf16>(maps, p, sh, st);
    if (units <= 2) return run<D, 16, kBf16>(maps, p, sh, st);
    if constexpr (D == 512) return run<D, 24, kBf16>(maps, p, sh, st);
    else return run<D, 32, kBf16>(maps, p, sh, st);
}

template <int D>
cudaError_t run_type(const CUtensorMap* maps, const Params& p, const Shape& sh, bool bf16, cudaStream_t st) {
    return bf16 ? run_rows<D, true>(maps, p, sh, st) : run_rows<D, false>(maps, p, sh, st);
}

}  // namespace

size_t tree_attn_workspace(int max_nodes, int heads, int kv_heads, int dim) {
    const int N = rows_per_item(max_nodes, heads / kv_heads, dim);
    return (size_t)2 * sm_count() * N * (dim * sizeof(float) + sizeof(float2)) + sm_count() * sizeof(Split);
}

bool tree_attn_countable(const TreeAttnArgs& a) {
    const int N = rows_per_item(a.max_nodes, a.heads / a.kv_heads, a.dim);
    return most_items(a, N) <= INT32_MAX && most_items(a, N) * (most_tiles(a) + item_cost(N)) <= INT32_MAX;
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
    int grid = sm_count();
    p.part = static_cast<float*>(a.work);
    p.ml = reinterpret_cast<float2*>(p.part + (size_t)2 * grid * sh.N * a.dim);
    p.split = reinterpret_cast<Split*>(p.ml + (size_t)2 * grid * sh.N);
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
    p.gqa = a.heads / a.kv_heads;
    p.kv_heads = a.kv_heads;
    p.window = a.window;
    p.N = sh.N;
    p.words = sh.words;
    p.slots = sh.slots;
    p.tmem_cols = sh.tmem;
    p.box = box_rows(a);
    while (1 << p.box_log < p.box) ++p.box_log;
    const long long tiles = most_tiles(a), items = most_items(a, sh.N);
    p.whole = tiles <= kWholeTiles;
    if (p.whole) grid = (int)std::min<long long>(grid, items);
    p.by_rows = make_div(sh.N);
    p.by_gqa = make_div(p.gqa);
    p.by_page = make_div(a.page_size);
    p.by_grid = make_div(grid);
    p.c = a.scale * 1.4426950408889634f;
    // A row is H D / 64 blocks of 64 dims; a box takes up to two of them, of eight rows each, so that one
    // copy lays a slot's rows out in the MMA's eights whatever the number of rows.
    const cuuint64_t row = (cuuint64_t)a.dim * a.kv_heads * 2, blocks = (cuuint64_t)a.kv_heads * (a.dim / 64);
    const cuuint32_t wide = a.dim == 64 ? 1 : 2;
    const cuuint64_t pool_dims[5] = {64, 8, blocks, (cuuint64_t)a.page_size / 8, (cuuint64_t)a.pages};
    const cuuint64_t pool_strides[4] = {row, 128, row * 8, (cuuint64_t)a.page_stride * 2};
    const cuuint32_t pool_box[5] = {64, 8, wide, (cuuint32_t)p.box / 8, 1};
    const cuuint64_t new_dims[3] = {64, (cuuint64_t)a.n_tokens, blocks};
    const cuuint64_t new_strides[2] = {(cuuint64_t)a.new_stride * 2, 128};
    const cuuint32_t new_box[3] = {64, kTreeBox, wide};
    CUtensorMap m[4];
    cudaError_t e;
    if ((e = make_map(&m[0], a.k_pool, 5, pool_dims, pool_strides, pool_box)) != cudaSuccess) return e;
    if ((e = make_map(&m[1], a.v_pool, 5, pool_dims, pool_strides, pool_box)) != cudaSuccess) return e;
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
    // The copies go to the legacy stream, which does not wait for non-blocking ones.
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    if (cudaMemcpyFromSymbol(&h, g_tree_err, sizeof(int)) != cudaSuccess) return -1;
    if (h) cudaMemcpyToSymbol(g_tree_err, &zero, sizeof(int));
    return h;
}

}  // namespace g4b
