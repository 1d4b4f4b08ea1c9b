// One token per logits row from a given uniform number: temperature, top-k, top-p and min-p per row
// over the whole vocabulary.
//
// With l the row's logits, m their maximum and T the temperature, an entry's weight is the whole
// number w_i = floor(2^40 exp((l_i - m) / T)) (at most 2^40, so a row of 262144 sums below 2^58).
// In descending order of l, ties to the lower index, the kept entries are a prefix: at most top_k
// of them; of those, the ones before which less than top_p of their mass lies; of those, the ones
// with exp((l_i - m) / T) >= min_p. With W the kept mass and r = floor(u W), the token is the first
// kept entry in index order at which the running mass exceeds r. NaN and -inf are never kept, a
// temperature <= 0 (or NaN) keeps the maximum alone, and a row without a finite entry or +inf gives -1.
// T may be anything else, infinite or tiny: differences that overflow fp32 count as infinite.
// Whole-number weights make every sum exact, so the token does not depend on how the row is split
// or in which order the parts are added.
//
// The reference's sampler (src/sampling.cpp:92-169) keeps at most 256 entries and draws in
// descending order; this one has no bound on the kept entries, and measures top_p after the
// temperature and top_k.
//
// A row is one cluster of 1 to 16 blocks. Each reads its slice of up to 64 KB from memory
// once, into shared memory, and passes over it there; blocks exchange through distributed shared
// memory, one cluster barrier an exchange:
//   * the maximum;
//   * where top_k or top_p cut, a histogram of 256 bins of 1/8 in (m - l) / T, which spreads a row's
//     likely entries evenly (counts, and for a cut by mass the exact masses);
//   * usual cuts leave a few hundred entries at and above the bin that is cut: these go to the first
//     block, which ranks up to kRanked of them all against all, searches longer lists for the last
//     key that stays, and finishes alone. Where they are more than kList (nucleus sampling of a flat
//     row), the bin is split into 256 again, the part that is cut is searched, and the threshold goes
//     back to all blocks. Ties by the thousand end in a search over the 50-bit keys (ordered logit
//     bits, inverted index) of all blocks, 8 bits a step;
//   * without a list, the kept masses per block; the block in whose range r falls finds the token.
// A top_k of up to 512 needs no histogram of all entries: the k-th largest of the threads' own maxima
// bounds the k-th largest entry from below.
//
// The floor is one read of the logits. What bounds the kernel behind it: for greedy rows and top-k cuts,
// that a block brings its whole slice in, waits for it and then passes over it, two blocks an SM in
// three and a half rounds that hardly overlap; with an exponential for every entry about 35
// instructions an entry, and three shared atomics on top for a cut by mass. Measured on one B200, 128 rows of
// 262144 bf16 logits (10 us of reading): 46 us greedy, 76 with top_k 40 and top_p 0.9, 101 with the
// temperature alone, 272 with top_p 0.95 alone, 135 for a mix; fp16 a little less (44, 74, 100, 263, 132),
// fp32 (21 us of reading) 90, 139, 157, 425 and 200; one row of 4096: 10 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "per_device.h"
#include "sample_rows.h"

namespace cg = cooperative_groups;

namespace g4b {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kSliceBytes = 65536;          // of a row that a block holds: two blocks fit an SM
constexpr int kRounds = kSliceBytes / 2 / (8 * kThreads);  // a thread takes eight consecutive entries a round
constexpr int kIndexBits = 18;              // vocabularies up to 262144
constexpr int kIndexMask = (1 << kIndexBits) - 1;
constexpr int kBins = 256;
constexpr int kList = 1024;                 // entries the first block takes
constexpr int kCand = 2048;                 // entries of one bin that a block sets aside
typedef unsigned long long u64;

// Masses in three 16-bit parts of their addends, whose sums over a slice fit 32 bits.
struct Bins {
    unsigned count[kBins], lo[kBins], mid[kBins], hi[kBins];
};
struct Pair {
    u64 a, b;
};
struct alignas(16) Shared {
    Bins bins[2];
    Pair ex[2][16];      // every block's, by rank
    u64 red[2][kWarps];
    unsigned red32[2][kWarps];
    u64 part[kRounds][kWarps];
    u64 cum_count[kBins], cum_mass[kBins];
    alignas(16) u64 key[kList + 2];  // the list, in the first block
    u64 weight[kThreads];  // kept masses by index
    u64 named[kList];      // the list sorted, and what a block names for it
    uint16_t cand[kCand];    // places in the slice of what is set aside
    u64 answer;
    int bin, staged, cands;
};

static_assert(sizeof(Shared) % 16 == 0, "the slice behind it is read in 16-byte pieces");

__device__ __forceinline__ unsigned order_bits(float l) {
    const unsigned u = __float_as_uint(l == 0.f ? 0.f : l);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_order(unsigned o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// Key of an entry: larger is earlier in the descending order.
__device__ __forceinline__ u64 key_of(float l, int index) {
    return ((u64)order_bits(l) << kIndexBits) | (u64)(kIndexMask - index);
}
__device__ __forceinline__ int key_index(u64 k) { return kIndexMask - (int)(k & kIndexMask); }
__device__ __forceinline__ float key_logit(u64 k) { return from_order((unsigned)(k >> kIndexBits)); }

// Sum over the warp, in three parts whose sums fit the 32-bit reduction.
__device__ __forceinline__ u64 warp_sum64(u64 v) {
    constexpr u64 kPart = (1u << 26) - 1;
    return (u64)__reduce_add_sync(0xffffffffu, (unsigned)(v & kPart)) +
           ((u64)__reduce_add_sync(0xffffffffu, (unsigned)((v >> 26) & kPart)) << 26) +
           ((u64)__reduce_add_sync(0xffffffffu, (unsigned)(v >> 52)) << 52);
}
__device__ __forceinline__ u64 warp_max64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The row's numbers that turn a logit into a weight.
struct Scale {
    float m, t, r, bins;  // maximum, temperature, 1 / t, 32 / t (at most FLT_MAX)
    bool inf, simple;
    __device__ void set(float max, float temperature) {
        m = max;
        t = temperature;
        r = 1.f / t;
        bins = fminf(32.f / t, FLT_MAX);  // finite: a distance of 0 stays in the first bin
        inf = m == INFINITY;
        // Out of this range the reciprocal or the remainder below could leave the normal numbers.
        simple = t > 1e-18f && t < 1e18f;
    }
    // exp((l - m) / t). The quotient is the correctly rounded one of a division, from the correctly
    // rounded reciprocal and one exact remainder (Markstein's theorem), as t is the same for all.
    __device__ __forceinline__ float share(float l) const {
        if (inf) return l == m ? 1.f : 0.f;
        const float a = l - m;
        float q = fmaxf(a * r, -200.f);  // below -104 the exponential is 0 either way
        if (simple) q = fmaf(fmaf(-q, t, a), r, q);
        else q = a > -INFINITY ? a / t : a;  // and nothing at -inf, also by an infinite t
        return expf(q);
    }
    static __device__ __forceinline__ u64 weight(float share) { return (u64)(share * 1099511627776.f); }
    // Four times the bin of a logit, ordered as the logits are: the scaled distance from the maximum,
    // made whole by adding 2^23 (which leaves it in the low bits) and cut to a multiple of four. -inf
    // is in the last bin, as all that is far below; +inf below +inf gives NaN, which fminf drops.
    __device__ __forceinline__ float place(float l) const { return (m - l) * bins; }  // in quarters of a bin
    __device__ __forceinline__ unsigned bin4(float l) const {
        const float x = inf && l == m ? 0.f : fminf(place(l), 1020.f);
        return __float_as_uint(x + 8388608.f) & 0x3fcu;
    }
    __device__ __forceinline__ int bin(float l) const { return (int)(bin4(l) >> 2); }
    // Cheap first test: a logit for which this is false is in a later bin (the last has none).
    __device__ __forceinline__ bool near(float l, int bin) const {
        return !(place(l) > (bin < kBins - 1 ? (float)(4 * bin + 8) : INFINITY));
    }
    // Which of 256 parts of its bin, from what the bin's rounding kept.
    __device__ __forceinline__ int sub(float l) const {
        const float x = inf && l == m ? 0.f : place(l);
        return (int)fminf(fmaxf((x - (float)bin4(l) + 0.5f) * 64.f, 0.f), 255.f);
    }
};

template <class T>
__device__ __forceinline__ void read8(const T* at, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(at);
        const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(h[i]);
    }
}

// Least and largest of eight values; the least is NaN where one of them is.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <class T>
__device__ __forceinline__ void extremes8(const T* at, float& least, float& most) {
    if constexpr (sizeof(T) == 4) {
        float v[8];
        read8(at, v);
        least = min_nan(min_nan(min_nan(v[0], v[1]), min_nan(v[2], v[3])), min_nan(min_nan(v[4], v[5]), min_nan(v[6], v[7])));
        most = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const uint4 a = *reinterpret_cast<const uint4*>(at);
        const T2* h = reinterpret_cast<const T2*>(&a);
        const T2 lo = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
        const T2 hi = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        least = min_nan(static_cast<float>(lo.x), static_cast<float>(lo.y));
        most = fmaxf(static_cast<float>(hi.x), static_cast<float>(hi.y));
    }
}

// One row of one cluster.
template <class T>
struct Row {
    Shared& sm;
    T* data;  // the slice, padded with -inf to a multiple of eight
    cg::cluster_group cl;
    int base, n, rounds, blocks, rank, phase;
    Scale sc;

    __device__ Row(Shared& s, T* d) : sm(s), data(d), cl(cg::this_cluster()), phase(0) {
        blocks = (int)cl.num_blocks();
        rank = (int)cl.block_rank();
    }
    // A block's shared memory may be reached from others only once that block has started. Every block says so at
    // its entry, started(), and waits for the others' word ahead of the first exchange, meet(): the slice is read
    // in between, so the wait costs nothing where the blocks start together.
    __device__ __forceinline__ void started() const {
        if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    }
    __device__ __forceinline__ void meet() const {
        if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    // All blocks' writes before it are seen by all after it. The block meets first, so that one warp's
    // release stands for all threads' writes, and the other warps need not wait for theirs.
    __device__ __forceinline__ void barrier() {
        __syncthreads();
        if (blocks == 1) return;
        if (threadIdx.x < 32) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        else asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    // each(l, index, round) for this thread's live entries in index order within a round.
    template <class Each>
    __device__ __forceinline__ void pass(Each each) const {
#pragma unroll 1
        for (int j = 0; j < rounds; ++j) {
            const int at = 8 * (j * kThreads + (int)threadIdx.x);
            if (at >= n) continue;
            float v[8];
            read8(data + at, v);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (v[i] > -INFINITY) each(v[i], base + at + i, j);
        }
    }
    // As pass, for all entries, dead ones (and the padding) among them.
    template <class Each>
    __device__ __forceinline__ void pass_all(Each each) const {
#pragma unroll 1
        for (int j = 0; j < rounds; ++j) {
            const int at = 8 * (j * kThreads + (int)threadIdx.x);
            if (at >= n) continue;
            float v[8];
            read8(data + at, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) each(v[i], base + at + i);
        }
    }
    // each(l, index) for the few entries that test(l) holds for: the tests of eight entries make one
    // mask and one branch.
    template <class Test, class Each>
    __device__ __forceinline__ void pass_few(Test test, Each each) const {
#pragma unroll 1
        for (int j = 0; j < rounds; ++j) {
            const int at = 8 * (j * kThreads + (int)threadIdx.x);
            if (at >= n) continue;
            float v[8];
            read8(data + at, v);
            unsigned hits = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) hits |= test(v[i]) ? 1u << i : 0u;
#pragma unroll 1
            for (; hits; hits &= hits - 1) {
                const int i = __ffs(hits) - 1;
                each(static_cast<float>(data[at + i]), base + at + i);
            }
        }
    }
    // The block's largest a and sum of b.
    __device__ uint2 block_max_sum(unsigned a, unsigned b) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        a = __reduce_max_sync(0xffffffffu, a);
        b = __reduce_add_sync(0xffffffffu, b);
        __syncthreads();
        if (lane == 0) sm.red32[0][w] = a, sm.red32[1][w] = b;
        __syncthreads();
        return {__reduce_max_sync(0xffffffffu, lane < kWarps ? sm.red32[0][lane] : 0),
                __reduce_add_sync(0xffffffffu, lane < kWarps ? sm.red32[1][lane] : 0)};
    }
    __device__ Pair block_max(u64 a, u64 b) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        a = warp_max64(a);
        b = warp_max64(b);
        __syncthreads();
        if (lane == 0) sm.red[0][w] = a, sm.red[1][w] = b;
        __syncthreads();
        return {warp_max64(lane < kWarps ? sm.red[0][lane] : 0), warp_max64(lane < kWarps ? sm.red[1][lane] : 0)};
    }
    __device__ u64 block_sum(u64 a) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        a = warp_sum64(a);
        __syncthreads();
        if (lane == 0) sm.red[0][w] = a;
        __syncthreads();
        return warp_sum64(lane < kWarps ? sm.red[0][lane] : 0);
    }
    // Each block's pair, folded over the cluster, after meet(). A block writes its own into every block before
    // the barrier: what is read after it is local. Two buffers in turn: one is written again only after the
    // next barrier, which the readers of the last use have passed.
    template <class Fold>
    __device__ void exchange(Pair mine, Fold fold) {
        if ((int)threadIdx.x < blocks) *cl.map_shared_rank(&sm.ex[phase][rank], threadIdx.x) = mine;
        barrier();
#pragma unroll 1
        for (int b = 0; b < blocks; ++b) fold(b, sm.ex[phase][b]);
        phase ^= 1;
    }

    __device__ Bins& clear() {
        Bins& b = sm.bins[phase];
#pragma unroll
        for (int i = threadIdx.x; i < 4 * kBins; i += kThreads) b.count[i] = 0;
        __syncthreads();
        return b;
    }
    static __device__ __forceinline__ void add(Bins& b, int i, u64 w, bool mass) {
        atomicAdd(&b.count[i], 1u);
        if (!mass) return;
        if (w & 0xffff) atomicAdd(&b.lo[i], (unsigned)(w & 0xffff));
        if ((w >> 16) & 0xffff) atomicAdd(&b.mid[i], (unsigned)((w >> 16) & 0xffff));
        if (w >> 32) atomicAdd(&b.hi[i], (unsigned)(w >> 32));
    }
    // Running counts (and masses) over the cluster's bins, in every block. Each block adds up its share
    // of the bins over all blocks, a lane a (bin, block), and hands the sums to all: reading every
    // bin of every block everywhere would be sixteen times the traffic between SMs.
    __device__ void merge(bool mass) {
        barrier();
        const int t = threadIdx.x, lane = t & 31, w = t >> 5;
        if (t < kBins) {
            const int src = t & (blocks - 1), bin = (t + rank * kBins) / blocks;
            const Bins* b = cl.map_shared_rank(&sm.bins[phase], src);
            unsigned c = b->count[bin];
            u64 m = mass ? b->lo[bin] + ((u64)b->mid[bin] << 16) + ((u64)b->hi[bin] << 32) : 0;
            for (int o = blocks >> 1; o > 0; o >>= 1) {
                c += __shfl_xor_sync(0xffffffffu, c, o);
                if (mass) m += __shfl_xor_sync(0xffffffffu, m, o);
            }
            *cl.map_shared_rank(&sm.cum_count[bin], src) = c;
            if (mass) *cl.map_shared_rank(&sm.cum_mass[bin], src) = m;
        }
        barrier();
        u64 c = t < kBins ? sm.cum_count[t] : 0, m = t < kBins && mass ? sm.cum_mass[t] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, (unsigned)c, o);  // counts fit 32 bits
            if (lane >= o) c += x;
        }
        if (mass)
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, m, o);
                if (lane >= o) m += y;
            }
        __syncthreads();
        if (t < kBins && lane == 31) sm.red[0][w] = c, sm.red[1][w] = m;
        __syncthreads();
        if (t < kBins) {
            for (int i = 0; i < w; ++i) c += sm.red[0][i], m += sm.red[1][i];
            sm.cum_count[t] = c;
            sm.cum_mass[t] = m;
        }
        if (t == 0) sm.bin = kBins - 1;
        __syncthreads();
        phase ^= 1;
    }
    // The bin in which the last kept entry lies: it starts below the goal, and ends at or above it.
    __device__ int cut_bin(bool mass, u64 before, double goal) {
        if (threadIdx.x < kBins) {
            const u64* cum = mass ? sm.cum_mass : sm.cum_count;
            const int t = threadIdx.x;
            const u64 lo = t ? cum[t - 1] : 0;
            if (cum[t] != lo && (double)(before + lo) < goal && !((double)(before + cum[t]) < goal)) sm.bin = t;
        }
        __syncthreads();
        return sm.bin;
    }

    // Entries that each(put) passes to put(l, index) go to the first block's list, block by block. Their
    // number in the cluster is returned; over kList of them are not listed.
    template <class Each>
    __device__ int gather(Each each) {
        if (threadIdx.x == 0) sm.staged = 0;
        __syncthreads();
        each([&](float l, int index) {
            const int at = atomicAdd(&sm.staged, 1);
            if (at < kList) sm.named[at] = key_of(l, index);
        });
        __syncthreads();
        const int mine = sm.staged;
        int first = 0, all = 0;
        exchange({(u64)mine, 0}, [&](int b, Pair x) { first += b < rank ? (int)x.a : 0, all += (int)x.a; });
        if (all <= kList) {
            u64* list = cl.map_shared_rank(sm.key, 0);
            for (int i = threadIdx.x; i < mine; i += kThreads) list[first + i] = sm.named[i];
        }
        barrier();
        return all;
    }
    // Sets a bin's entries aside, in the order they come; at most kCand of them.
    __device__ void set_aside(int bin) {
        if (threadIdx.x == 0) sm.cands = 0;
        __syncthreads();
        pass_few([&](float l) { return sc.bin4(l) == 4u * bin; }, [&](float l, int index) {
            const int at = atomicAdd(&sm.cands, 1);
            if (at < kCand) sm.cand[at] = (uint16_t)(index - base);
        });
        __syncthreads();
    }
    template <class Each>
    __device__ __forceinline__ void pass_aside(Each each) const {
        const int m = min(sm.cands, kCand);
#pragma unroll 1
        for (int i = threadIdx.x; i < m; i += kThreads) {
            const int at = sm.cand[i];
            each(static_cast<float>(data[at]), base + at);
        }
    }

    // Key of the last kept entry, searched for over keys: of those at or above `from`, the k largest
    // stay, or the ones before which less than `goal` of mass lies. The slow way, for ties.
    __device__ __noinline__ u64 search(bool mass, double goal, u64 from) {
        u64 before = 0, lo = from, hi = ~0ull;
        // Every step leaves 1/256 of a 50-bit range of keys, or less: seven steps reach one key.
        for (int step = 0; step < 9; ++step) {
            u64 top = 0, low = 0;  // the largest key and, inverted, the smallest
            pass([&](float l, int index, int) {
                const u64 c = key_of(l, index);
                if (c >= lo && c <= hi) top = max(top, c), low = max(low, ~c);
            });
            const Pair mine = block_max(top, low);
            Pair all{0, 0};
            exchange(mine, [&](int, Pair x) { all = {max(all.a, x.a), max(all.b, x.b)}; });
            hi = all.a;
            lo = ~all.b;
            if (hi <= lo) return lo;
            const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 8);
            Bins& b = clear();
            pass([&](float l, int index, int) {
                const u64 c = key_of(l, index);
                if (c >= lo && c <= hi) add(b, (int)((hi - c) >> shift), mass ? Scale::weight(sc.share(l)) : 0, mass);
            });
            merge(mass);
            const int bin = cut_bin(mass, before, goal);
            if (bin) before += (mass ? sm.cum_mass : sm.cum_count)[bin - 1];
            const u64 first = hi - ((u64)bin << shift), span = ((u64)1 << shift) - 1;
            __syncthreads();
            hi = first;
            lo = max(lo, first >= span ? first - span : 0);
        }
        return lo;
    }
};

__device__ __forceinline__ void write(const SampleRowsArgs& a, int r, int token, float prob, int kept) {
    a.token[r] = token;
    if (a.prob) a.prob[r] = prob;
    if (a.kept) a.kept[r] = kept;
}

__device__ __forceinline__ u64 draw(float u, u64 total) {
    const double x = floor((double)u * (double)total);
    return min(x > 0.0 ? (u64)x : 0ull, total - 1);  // also for numbers outside [0, 1)
}

// Exclusive running sum over the block's threads of one value each, and the whole.
__device__ u64 block_scan(Shared& sm, u64 v, u64* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    u64 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sm.red[0][w] = x;
    __syncthreads();
    u64 ahead = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        const u64 s = sm.red[0][i];
        ahead += i < w ? s : 0;
        all += s;
    }
    *total = all;
    return ahead + x - v;
}

// Lists up to this long are ranked, each key against all; longer ones are searched in 8-bit steps.
// With every list ranked, 128 rows of 262144 took 88 us at top_k 256 (85 so) and 285 at top_p 0.95 (271).
constexpr int kRanked = 256;

// Puts the list's n <= kRanked keys into sm.named in descending order, several neighbouring threads a
// key.
__device__ __noinline__ void rank_list(Shared& sm, int n) {
    const int t = threadIdx.x;
    if (t == 0) sm.key[n] = 0;  // keys are loaded in pairs
    __syncthreads();
    int share = kThreads / kRanked;  // threads a key
    while (share < 32 && 2 * share * n <= kThreads) share *= 2;
    const int part = t % share, i = t / share;
    const u64 mine = i < n ? sm.key[i] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = 2 * part; j < n; j += 2 * share) {
        const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(&sm.key[j]);
        rank += (k.x > mine) + (k.y > mine);
    }
    for (int o = share >> 1; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (i < n && part == 0) sm.named[rank] = mine;
    __syncthreads();
}

// As Row::search, over the list alone (two keys a thread, 0: none): the last of the keys at or above
// `from` that stays. `before` is what lies ahead of the list.
__device__ __noinline__ u64 search_list(Shared& sm, const u64 (&key)[2], const u64 (&w)[2], bool mass, u64 before,
                                        double goal, u64 from) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    u64 lo = max(from, (u64)1), hi = ~0ull;
    Bins& b = sm.bins[0];  // all remote reads of it ended before the last barrier
    for (int step = 0; step < 9; ++step) {
        u64 top = 0, low = 0;
        bool in[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            in[i] = key[i] >= lo && key[i] <= hi;
            if (in[i]) top = max(top, key[i]), low = max(low, ~key[i]);
        }
        top = warp_max64(top);
        low = warp_max64(low);
        __syncthreads();
        if (lane == 0) sm.red[0][warp] = top, sm.red[1][warp] = low;
        for (int i = t; i < 4 * kBins; i += kThreads) b.count[i] = 0;
        if (t == 0) sm.bin = kBins - 1;
        __syncthreads();
        hi = warp_max64(lane < kWarps ? sm.red[0][lane] : 0);
        lo = ~warp_max64(lane < kWarps ? sm.red[1][lane] : 0);
        if (hi <= lo) return lo;
        const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 8);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (in[i]) {
                const int x = (int)((hi - key[i]) >> shift);
                const u64 v = mass ? w[i] : 1;
                atomicAdd(&b.lo[x], (unsigned)v & 0xffff);
                if (mass) atomicAdd(&b.mid[x], (unsigned)v >> 16);
                if (v >> 32) atomicAdd(&b.hi[x], (unsigned)(v >> 32));
            }
        __syncthreads();
        u64 own = t < kBins ? b.lo[t] + ((u64)b.mid[t] << 16) + ((u64)b.hi[t] << 32) : 0, x = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sm.red[0][warp] = x;
        __syncthreads();
        for (int i = 0; i < warp && i < kBins / 32; ++i) x += sm.red[0][i];
        if (own && (double)(before + x - own) < goal && !((double)(before + x) < goal)) {
            sm.bin = t;
            sm.answer = before + x - own;
        }
        __syncthreads();
        before = sm.answer;
        const u64 first = hi - ((u64)sm.bin << shift), span = ((u64)1 << shift) - 1;
        hi = first;
        lo = max(lo, first >= span ? first - span : 0);
    }
    return lo;
}

// The end of a row whose list (in the first block) holds every entry that may be kept: the first k
// of it, then the cuts by mass and by min-p, then the draw.
__device__ __noinline__ void finish_list(const SampleRowsArgs& a, int r, Shared& sm, const Scale& sc, int n, u64 k,
                                         float p, double goal, float low) {
    const int t = threadIdx.x;
    u64 key[2], w[2], mass, total;
    float e[2];
    bool in[2];
    if (n <= kRanked) {
        rank_list(sm, n);
        // Two neighbours of the descending order a thread.
        const int m = (int)min((u64)n, k);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            key[i] = 2 * t + i < m ? sm.named[2 * t + i] : 0;
            e[i] = 2 * t + i < m ? sc.share(key_logit(key[i])) : 0.f;
            w[i] = Scale::weight(e[i]);
        }
        const u64 before = block_scan(sm, w[0] + w[1], &mass);
        if (k != ~0ull) goal = (double)p * (double)mass;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = 2 * t + i;
            const u64 ahead = before + (i ? w[0] : 0);
            in[i] = x < m && (x == 0 || ((p >= 1.f || (double)ahead < goal) && e[i] >= low));
        }
    } else {
        u64 from = 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            key[i] = t + i * kThreads < n ? sm.key[t + i * kThreads] : 0;
            e[i] = key[i] ? sc.share(key_logit(key[i])) : 0.f;
            w[i] = Scale::weight(e[i]);
        }
        if (k < (u64)n) from = search_list(sm, key, w, false, 0, (double)k, 1);
        block_scan(sm, (key[0] >= from ? w[0] : 0) + (key[1] >= from ? w[1] : 0), &mass);
        if (k != ~0ull) goal = (double)p * (double)mass;
        if (p <= 0.f) from = search_list(sm, key, w, false, 0, 1.0, 1);
        else if (p < 1.f) from = search_list(sm, key, w, true, 0, goal, from);
#pragma unroll
        for (int i = 0; i < 2; ++i) in[i] = key[i] >= from && key[i] && e[i] >= low;
        __syncthreads();
    }
    sm.weight[t] = 0;
    if (t == 0) sm.staged = 0;
    __syncthreads();
    // The draw goes in index order: kept masses by the index's upper bits, a thread a bucket. (64-bit
    // atomics in shared memory are loops, 60 to 2500 cycles a warp by how many lanes meet; so as many
    // buckets as there are threads, and no such atomics where every entry takes part.)
    const int shift = max(0, 23 - __clz(max(1, a.vocab - 1)));
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (in[i]) atomicAdd(&sm.weight[key_index(key[i]) >> shift], w[i]);
    const int kept = __syncthreads_count(in[0]) + __syncthreads_count(in[1]);
    const u64 bucket = sm.weight[t], at = block_scan(sm, bucket, &total);
    const u64 target = draw(a.uniform[r], total);
    if (target >= at && target < at + bucket) {
        sm.bin = t;
        sm.answer = target - at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (in[i] && key_index(key[i]) >> shift == sm.bin) {  // that bucket's entries
            const int x = atomicAdd(&sm.staged, 1);
            sm.key[x] = key[i];
            sm.named[x] = w[i];
        }
    __syncthreads();
    const int c = sm.staged;
    for (int i = t; i < c; i += kThreads) {
        const u64 mine = sm.key[i];
        u64 below = 0;
        for (int j = 0; j < c; ++j) below += key_index(sm.key[j]) < key_index(mine) ? sm.named[j] : 0;
        if (sm.answer >= below && sm.answer < below + sm.named[i])
            write(a, r, key_index(mine), sc.share(key_logit(mine)) / ((float)total * 9.094947017729282e-13f), kept);  // 2^-40
    }
}
static_assert((kIndexMask >> 9) + 1 == kThreads, "a thread a bucket");

template <class T>
__device__ __forceinline__ void sample_row(const SampleRowsArgs& a, Shared& sm, Row<T>& row, int r) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* in = static_cast<const T*>(a.logits) + r * a.stride;
    const T* from = in + row.base;
    constexpr int kWide = 16 / sizeof(T);
    if (reinterpret_cast<uintptr_t>(from) % 16 == 0) {
        const int whole = row.n / kWide;
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(row.data);
#pragma unroll 4
        for (int i = tid; i < whole; i += kThreads)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i * 16), "l"(from + i * kWide) : "memory");
        for (int i = whole * kWide + tid; i < row.n; i += kThreads) row.data[i] = from[i];
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
#pragma unroll 4
        for (int i = tid; i < row.n; i += kThreads) row.data[i] = from[i];
    }
    if (tid < ((row.n + 7) & ~7) - row.n) row.data[row.n + tid] = static_cast<T>(-INFINITY);
    __syncthreads();

    // The maximum and the number of live entries. Eights with a NaN or -inf among them (their least
    // says so) are looked at one by one, and NaN becomes -inf.
    float m = -INFINITY;
    unsigned live = 0;
#pragma unroll 1
    for (int j = 0; j < row.rounds; ++j) {
        const int at = 8 * (j * kThreads + tid);
        if (at >= row.n) continue;
        float least, most;
        extremes8(row.data + at, least, most);
        if (least > -INFINITY) {
            m = fmaxf(m, most);
            live += 8;
        } else {
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                const float v = static_cast<float>(row.data[at + i]);
                if (v > -INFINITY) m = fmaxf(m, v), ++live;
                else row.data[at + i] = static_cast<T>(-INFINITY);
            }
        }
    }
    const float own_max = m;
    const uint2 own = row.block_max_sum(m > -INFINITY ? order_bits(m) : 0, live);
    u64 top = 0, alive = 0;
    row.meet();
    row.exchange({own.x, own.y}, [&](int, Pair x) { top = max(top, x.a), alive += x.b; });
    const float t = a.temperature ? a.temperature[r] : 1.f;
    const bool lead = row.rank == 0 && tid == 0;
    if (top == 0) {
        if (lead) write(a, r, -1, 0.f, 0);
        return;
    }
    m = from_order((unsigned)top);
    if (!(t > 0.f)) {
        unsigned first = 0;  // the lowest index that holds the maximum, inverted
        row.pass([&](float l, int index, int) {
            if (l == m) first = max(first, (unsigned)(kIndexMask - index) + 1);
        });
        first = row.block_max_sum(first, 0).x;
        u64 best = 0;
        row.exchange({first, 0}, [&](int, Pair x) { best = max(best, x.a); });
        if (lead) write(a, r, kIndexMask + 1 - (int)best, 1.f, 1);
        return;
    }
    row.sc.set(m, t);
    const Scale sc = row.sc;
    const int want = a.top_k ? a.top_k[r] : 0;
    float p = a.top_p ? a.top_p[r] : 1.f;
    if (!(p < 1.f)) p = 1.f;  // a NaN setting is off
    float low = a.min_p ? a.min_p[r] : 0.f;
    low = low > 0.f ? fminf(low, 1.f) : 0.f;
    u64 k = want > 0 && (u64)want < alive ? (u64)want : ~0ull;
    if (p <= 0.f) k = 1;  // the first entry always stays
    const bool by_mass = k == ~0ull && p < 1.f;

    u64 from_key = 0;  // the last kept key, as far as it is known
    if (k != ~0ull || by_mass) {
        // Few entries: the k-th largest of the threads' own maxima is at most the k-th largest entry, so
        // its bin bounds a list without a count of all entries.
        if (!by_mass && k <= kList / 2 && k <= (u64)row.blocks * kThreads / 2) {
            Bins& b = row.clear();
            if (own_max > -INFINITY) atomicAdd(&b.count[sc.bin(own_max)], 1u);
            row.merge(false);
            const int bin = row.cut_bin(false, 0, (double)k);
            const int n = row.gather([&](auto put) {
                row.pass_few([&](float l) { return sc.near(l, bin); }, [&](float l, int index) {
                    if (sc.bin(l) <= bin && l > -INFINITY) put(l, index);
                });
            });
            if (n <= kList) {
                if (row.rank == 0) finish_list(a, r, sm, sc, n, k, p, 0.0, low);
                return;
            }
        }
        Bins& b = row.clear();
        // The last bin is not counted, and has no mass: it holds what the others do not.
        if (by_mass)
            row.pass_all([&](float l, int) {
                const unsigned at = sc.bin4(l);
                if (at == 4 * (kBins - 1)) return;
                const u64 w = Scale::weight(sc.share(l));
                char* c = reinterpret_cast<char*>(&b) + at;
                atomicAdd(reinterpret_cast<unsigned*>(c), 1u);
                atomicAdd(reinterpret_cast<unsigned*>(c + sizeof(b.count)), (unsigned)w & 0xffff);
                atomicAdd(reinterpret_cast<unsigned*>(c + 2 * sizeof(b.count)), (unsigned)w >> 16);
                if (w >> 32) atomicAdd(reinterpret_cast<unsigned*>(c + 3 * sizeof(b.count)), (unsigned)(w >> 32));
            });
        else
            row.pass_all([&](float l, int) {
                const unsigned at = sc.bin4(l);
                if (at < 4 * (kBins - 1)) atomicAdd(reinterpret_cast<unsigned*>(reinterpret_cast<char*>(&b) + at), 1u);
            });
        row.merge(by_mass);
        double goal = by_mass ? (double)p * (double)sm.cum_mass[kBins - 1] : (double)k;
        const int bin = row.cut_bin(by_mass, 0, goal);
        const u64 held = bin == kBins - 1 ? alive : sm.cum_count[bin];
        if (held <= kList) {
            const int n = row.gather([&](auto put) {
                row.pass_few([&](float l) { return sc.near(l, bin); }, [&](float l, int index) {
                    if (sc.bin(l) <= bin && l > -INFINITY) put(l, index);
                });
            });
            if (row.rank == 0) finish_list(a, r, sm, sc, n, k, p, goal, low);
            return;
        }
        const u64 ahead = bin ? (by_mass ? sm.cum_mass : sm.cum_count)[bin - 1] : 0;
        const u64 in_bin = held - (bin ? sm.cum_count[bin - 1] : 0);
        __syncthreads();
        u64 key = 0;
        bool found = false;
        if (bin < kBins - 1) {  // the bin in 256 parts
            row.set_aside(bin);
            Bins& s = row.clear();
            row.pass_aside([&](float l, int) { Row<T>::add(s, sc.sub(l), by_mass ? Scale::weight(sc.share(l)) : 0, by_mass); });
            row.merge(by_mass);
            const int part = row.cut_bin(by_mass, ahead, goal);
            const u64 lo = part ? sm.cum_count[part - 1] : 0, before = ahead + (part ? (by_mass ? sm.cum_mass : sm.cum_count)[part - 1] : 0);
            const u64 here = sm.cum_count[part] - lo;
            if (sm.cum_count[kBins - 1] == in_bin && here <= kList) {  // no block had too many
                const int n = row.gather([&](auto put) {
                    row.pass_aside([&](float l, int index) {
                        if (sc.sub(l) == part) put(l, index);
                    });
                });
                if (row.rank == 0) {
                    u64 own[2], w[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        own[i] = tid + i * kThreads < n ? sm.key[tid + i * kThreads] : 0;
                        w[i] = own[i] && by_mass ? Scale::weight(sc.share(key_logit(own[i]))) : 0;
                    }
                    const u64 last = search_list(sm, own, w, by_mass, before, goal, 1);
                    __syncthreads();
                    if (tid < row.blocks) *row.cl.map_shared_rank(&sm.answer, tid) = last;
                }
                row.barrier();
                key = sm.answer;
                found = true;
            }
        }
        if (!found) key = row.search(by_mass, goal, 0);
        from_key = key;
        if (!by_mass && p > 0.f && p < 1.f) {  // the k that stay, then the cut by their mass
            u64 mass = 0;
            row.pass([&](float l, int index, int) {
                if (key_of(l, index) >= from_key) mass += Scale::weight(sc.share(l));
            });
            const u64 mine = row.block_sum(mass);
            u64 sum = 0;
            row.exchange({mine, 0}, [&](int, Pair x) { sum += x.a; });
            goal = (double)p * (double)sum;
            from_key = max(from_key, row.search(true, goal, from_key));
        }
    }

    // Kept mass in index order: per (round, warp), then block by block.
    const float edge = from_key ? key_logit(from_key) : -INFINITY;
    const float far = low > 0.f ? (0.01f - logf(low)) * 32.f * 1.001f : INFINITY;  // places past which no share reaches low
    const int edge_index = from_key ? key_index(from_key) : kIndexMask;
    const bool some = from_key || low > 0.f;  // most entries are cut: skip their exponentials
    const auto weigh = [&](float l, int index, float& e) -> u64 {
        if (some && (l < edge || (l == edge && index > edge_index) || sc.place(l) > far)) return ~0ull;
        e = sc.share(l);
        return e >= low ? Scale::weight(e) : ~0ull;
    };
    unsigned count = 0;
#pragma unroll 1
    for (int j = 0; j < row.rounds; ++j) {
        const int at = 8 * (j * kThreads + tid);
        u64 sum = 0;
        if (at < row.n) {
            float v[8];
            read8(row.data + at, v);
            if (!some) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum += Scale::weight(sc.share(v[i]));  // 0 for -inf
                    count += v[i] > -INFINITY;
                }
            } else {
                unsigned hits = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) hits |= v[i] >= edge && v[i] > -INFINITY && !(sc.place(v[i]) > far) ? 1u << i : 0u;
#pragma unroll 1
                for (; hits; hits &= hits - 1) {
                    const int i = __ffs(hits) - 1;
                    float e;
                    const u64 w = weigh(static_cast<float>(row.data[at + i]), row.base + at + i, e);
                    if (w != ~0ull) sum += w, ++count;
                }
            }
        }
        sum = warp_sum64(sum);
        if (lane == 0) sm.part[j][warp] = sum;
    }
    count = row.block_max_sum(0, count).y;  // its barriers also show the parts
    u64 slice = 0;
    if (tid < row.rounds * kWarps) slice = sm.part[0][tid];
    const Pair mine{row.block_sum(slice), count};
    u64 total = 0, ahead = 0, kept = 0;
    row.exchange(mine, [&](int b, Pair x) {
        if (b < row.rank) ahead += x.a;
        total += x.a;
        kept += x.b;
    });
    u64 goal = draw(a.uniform[r], total);
    if (goal < ahead || goal >= ahead + mine.a) return;
    goal -= ahead;
    // The (round, warp) part that holds it: one warp looks, four parts a lane.
    if (warp == 0) {
        u64 w[4], x = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = 4 * lane + i < row.rounds * kWarps ? sm.part[0][4 * lane + i] : 0;
            x += w[i];
        }
        u64 at = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        at = x - at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (goal >= at && goal < at + w[i]) {
                sm.bin = 4 * lane + i;
                sm.answer = goal - at;
            }
            at += w[i];
        }
        __syncwarp();
        const int j = sm.bin / kWarps, at8 = 8 * (j * kThreads + (sm.bin % kWarps) * 32 + lane);
        goal = sm.answer;
        u64 own = 0;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = -INFINITY;
        if (at8 < row.n) read8(row.data + at8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (v[i] > -INFINITY) {
                float e;
                const u64 w = weigh(v[i], row.base + at8 + i, e);
                if (w != ~0ull) own += w;
            }
        u64 upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        u64 run = upto - own;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (v[i] > -INFINITY) {
                float e;
                const u64 w = weigh(v[i], row.base + at8 + i, e);
                if (w == ~0ull) continue;
                if (goal >= run && goal < run + w)
                    write(a, r, row.base + at8 + i, e / ((float)total * 9.094947017729282e-13f), (int)kept);  // 2^-40
                run += w;
            }
    }
}
template <class T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(SampleRowsArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared& sm = *reinterpret_cast<Shared*>(raw);
    Row<T> row(sm, reinterpret_cast<T*>(raw + sizeof(Shared)));
    row.started();
    const int per = ((a.vocab + row.blocks - 1) / row.blocks + 7) & ~7;
    row.base = row.rank * per;
    row.n = max(0, min(per, a.vocab - row.base));
    row.rounds = (row.n + 8 * kThreads - 1) / (8 * kThreads);
    sample_row(a, sm, row, blockIdx.x / row.blocks);
}
static_assert(kRounds * kWarps == 128, "the last search looks at 128 parts");

template <class T>
cudaError_t run(const SampleRowsArgs& a, cudaStream_t st) {
    // As few blocks a row as hold it, so that a row's barriers weigh little; more, down to 4096 entries
    // each, while all rows' blocks are resident at once: then latency counts.
    int blocks = 1;
    const auto span = [&](int n) { return ((a.vocab + n - 1) / n + 7) & ~7; };
    while (span(blocks) * sizeof(T) > kSliceBytes) blocks *= 2;
    while (blocks < 16 && span(blocks) > 4096 && 2ll * a.rows * blocks <= 2 * 148) blocks *= 2;
    const int per = span(blocks);
    const size_t smem = sizeof(Shared) + (size_t)per * sizeof(T);
    auto kern = sample_rows_kernel<T>;
    static OncePerDevice attributes;
    const cudaError_t e = attributes([&] {
        const cudaError_t x = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (x != cudaSuccess) return x;
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)(sizeof(Shared) + kSliceBytes));
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)blocks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

cudaError_t sample_rows_launch(const SampleRowsArgs& a, cudaStream_t st) {
    return a.dtype == 0 ? run<__nv_bfloat16>(a, st) : a.dtype == 1 ? run<__half>(a, st) : run<float>(a, st);
}

}  // namespace g4b
