// One token per logits row from a given uniform number: temperature, top-k, top-p and min-p per row
// over the whole vocabulary.
//
// With l the row's logits, m their maximum and T the temperature, an entry's weight is the whole
// number w_i = floor(2^40 exp((l_i - m) / T)) (at most 2^40, so a row of 262144 sums below 2^58).
// In descending order of l, ties to the lower index, the kept entries are a prefix: at most top_k
// of them; of those, the ones before which less than top_p of their mass lies; of those, the ones
// with exp((l_i - m) / T) >= min_p. With W the kept mass and r = floor(u W), the token is the first
// kept entry in index order at which the running mass exceeds r. NaN and -inf are never kept, a
// temperature <= 0 keeps the maximum alone, and a row without a finite entry (or +inf) gives -1.
// Whole-number weights make every sum exact, so the token does not depend on how the row is split
// or in which order the parts are added.
//
// The reference's sampler (src/sampling.cpp:92-169) keeps at most 256 entries and draws in
// descending order; this one has no bound on the kept entries, and measures top_p after the
// temperature and top_k.
//
// A row is held in the registers of one cluster of 1 to 16 blocks (up to 16384 entries a block),
// read from memory once. The prefix's end, as a 50-bit key (ordered logit bits, inverted index), is
// found by counting: first 256 bins of 1/8 in (m - l) / T, which spread a row's likely entries
// evenly, then 256 bins over the range of keys that is left, until one key is left. Each block
// counts in shared memory; the blocks exchange bins through distributed shared memory, one
// cluster barrier a step.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "launch.cuh"
#include "sample_rows.h"

namespace cg = cooperative_groups;

namespace g4b {

namespace {

constexpr int kThreads = 1024;
constexpr int kPer = 16;                    // entries a thread holds
constexpr int kSpan = kThreads * kPer;      // entries a block holds
constexpr int kIndexBits = 18;              // vocabularies up to 262144
constexpr int kBins = 256;
typedef unsigned long long u64;

struct Bins {  // counts and masses; a mass is the sum of three 16-bit parts, whose sums fit 32 bits
    unsigned count[kBins], lo[kBins], mid[kBins], hi[kBins];
};
struct Exchange {
    u64 a, b;
};
struct Smem {
    Bins bins[2];
    Exchange ex[2];
    u64 red[2][32];
    u64 part[4][32];
    u64 cum_count[kBins], cum_mass[kBins];
    int bin;
};

__device__ __forceinline__ unsigned order_bits(float l) {  // 0: never kept
    if (!(l > -INFINITY)) return 0;
    const unsigned u = __float_as_uint(l == 0.f ? 0.f : l);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_order(unsigned o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_max64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <class T>
__device__ __forceinline__ float as_f32(T x) { return static_cast<float>(x); }

template <class T>
struct Row {
    float l[kPer];  // entry 4 k + j is index base + 4096 k + 4 tid + j
    float m, heat;
    int base, n;    // this block's slice of the row
    Smem* sm;
    cg::cluster_group cl;
    int phase;

    __device__ Row(Smem* s) : sm(s), cl(cg::this_cluster()), phase(0) {}

    __device__ int index(int k, int j) const { return base + 4096 * k + 4 * (int)threadIdx.x + j; }
    __device__ u64 key(int e) const {
        const unsigned o = order_bits(l[e]);
        return o ? ((u64)o << kIndexBits) | (u64)((1 << kIndexBits) - 1 - index(e >> 2, e & 3)) : 0;
    }
    __device__ float share(int e) const { return l[e] == m ? 1.f : expf((l[e] - m) / heat); }
    static __device__ u64 weight(float e) { return (u64)(e * 1099511627776.f); }

    __device__ void barrier() {
        if (cl.num_blocks() > 1) cl.sync();
        else __syncthreads();
    }

    // The cluster's largest a and largest b.
    __device__ Exchange reduce_max(u64 a, u64 b) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        a = warp_max64(a);
        b = warp_max64(b);
        __syncthreads();
        if (lane == 0) {
            sm->red[0][w] = a;
            sm->red[1][w] = b;
        }
        __syncthreads();
        if (w == 0) {
            a = warp_max64(sm->red[0][lane]);
            b = warp_max64(sm->red[1][lane]);
            if (lane == 0) sm->ex[phase] = {a, b};
        }
        barrier();
        Exchange r{0, 0};
        for (unsigned c = 0; c < cl.num_blocks(); ++c) {
            const Exchange x = *cl.map_shared_rank(&sm->ex[phase], c);
            r.a = max(r.a, x.a);
            r.b = max(r.b, x.b);
        }
        phase ^= 1;
        return r;
    }

    __device__ Bins& clear_bins() {
        Bins& b = sm->bins[phase];
        unsigned* z = b.count;
        z[threadIdx.x] = 0;  // 4 x 256 counters, 1024 threads
        __syncthreads();
        return b;
    }
    __device__ static void add(Bins& b, int i, u64 w, bool mass) {
        atomicAdd(&b.count[i], 1u);
        if (mass && w) {
            atomicAdd(&b.lo[i], (unsigned)(w & 0xffff));
            if (w >> 16) atomicAdd(&b.mid[i], (unsigned)((w >> 16) & 0xffff));
            if (w >> 32) atomicAdd(&b.hi[i], (unsigned)(w >> 32));
        }
    }
    // Running counts and masses over the cluster's bins, in every block.
    __device__ void merge() {
        barrier();
        const int t = threadIdx.x, lane = t & 31, w = t >> 5;
        u64 c = 0, m = 0;
        if (t < kBins)
            for (unsigned r = 0; r < cl.num_blocks(); ++r) {
                const Bins* b = cl.map_shared_rank(&sm->bins[phase], r);
                c += b->count[t];
                m += b->lo[t] + ((u64)b->mid[t] << 16) + ((u64)b->hi[t] << 32);
            }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 x = __shfl_up_sync(0xffffffffu, c, o), y = __shfl_up_sync(0xffffffffu, m, o);
            if (lane >= o) c += x, m += y;
        }
        __syncthreads();
        if (t < kBins && lane == 31) sm->red[0][w] = c, sm->red[1][w] = m;
        __syncthreads();
        if (t < kBins) {
            for (int i = 0; i < w; ++i) c += sm->red[0][i], m += sm->red[1][i];
            sm->cum_count[t] = c;
            sm->cum_mass[t] = m;
        }
        if (t == 0) sm->bin = kBins;
        __syncthreads();
        phase ^= 1;
    }

    // Narrows the kept prefix: its last key is returned, 0 when all entries stay. With `mass`, an
    // entry stays while the mass before it is below p times the mass of the entries at or above
    // `from`; otherwise the `k` largest stay.
    __device__ u64 last_kept(bool mass, u64 k, double p, u64 from) {
        Bins& b = clear_bins();
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const u64 c = key(e);
            if (c && c >= from) {
                const float x = l[e] == m ? 0.f : (m - l[e]) / heat;
                add(b, (int)fminf(x * 8.f, 255.f), mass ? weight(share(e)) : 0, mass);
            }
        }
        merge();
        const u64 all = mass ? sm->cum_mass[kBins - 1] : sm->cum_count[kBins - 1];
        const double goal = mass ? p * (double)all : (double)k;
        if (!((double)all > goal)) return 0;  // k at or above the entries there are
        u64 before = 0, lo = from, hi = ~0ull;
        bool first = true;
        int bin = 0;
        // Every step leaves 1/256 of a 50-bit range of keys, or less: seven steps reach one key.
        for (int step = 0; step < 8; ++step) {
            // The bin in which the last kept entry lies.
            const u64* cum = mass ? sm->cum_mass : sm->cum_count;
            if (threadIdx.x < kBins) {
                const int t = threadIdx.x;
                const u64 at = before + (t ? cum[t - 1] : 0);
                if (cum[t] != (t ? cum[t - 1] : 0) && (double)at < goal && !((double)(before + cum[t]) < goal)) sm->bin = t;
            }
            __syncthreads();
            bin = sm->bin;
            before += bin ? cum[bin - 1] : 0;
            u64 top = 0, low = 0;  // largest key and, inverted, smallest key in that bin
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const u64 c = key(e);
                bool in = c && c >= lo && c <= hi;
                if (first && in) {
                    const float x = l[e] == m ? 0.f : (m - l[e]) / heat;
                    in = (int)fminf(x * 8.f, 255.f) == bin;
                }
                if (in) {
                    top = max(top, c);
                    low = max(low, ~c);
                }
            }
            first = false;
            const Exchange r = reduce_max(top, low);
            hi = r.a;
            lo = ~r.b;
            if (hi == lo) return lo;
            const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 8);
            Bins& b2 = clear_bins();
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const u64 c = key(e);
                if (c && c >= lo && c <= hi) add(b2, (int)((hi - c) >> shift), mass ? weight(share(e)) : 0, mass);
            }
            merge();
            // The chosen bin's key range, for the next step.
            if (threadIdx.x < kBins) {
                const u64* cm = mass ? sm->cum_mass : sm->cum_count;
                const int t = threadIdx.x;
                const u64 at = before + (t ? cm[t - 1] : 0);
                if (cm[t] != (t ? cm[t - 1] : 0) && (double)at < goal && !((double)(before + cm[t]) < goal)) sm->bin = t;
            }
            __syncthreads();
            const u64 top_key = hi - ((u64)sm->bin << shift);
            const u64 span = ((u64)1 << shift) - 1;
            hi = top_key;
            lo = max(lo, top_key >= span ? top_key - span : 0);
            __syncthreads();
        }
        return lo;
    }
};

template <class T>
__global__ void __launch_bounds__(kThreads, 1) sample_rows_kernel(SampleRowsArgs a) {
    __shared__ Smem sm;
    Row<T> row(&sm);
    const int rank = (int)row.cl.block_rank(), blocks = (int)row.cl.num_blocks();
    const int r = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* in = static_cast<const T*>(a.logits) + r * a.stride;
    const int per = ((a.vocab + blocks - 1) / blocks + 7) & ~7;
    row.base = rank * per;
    row.n = min(per, a.vocab - row.base);
    const bool vec = reinterpret_cast<uintptr_t>(in) % (4 * sizeof(T)) == 0;
    u64 best = 0;
#pragma unroll
    for (int k = 0; k < kPer / 4; ++k) {
        const int at = 4096 * k + 4 * tid;
        T x[4];
        if (vec && at + 3 < row.n) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(x) = __ldcs(reinterpret_cast<const uint4*>(in + row.base + at));
            else *reinterpret_cast<uint2*>(x) = __ldcs(reinterpret_cast<const uint2*>(in + row.base + at));
#pragma unroll
            for (int j = 0; j < 4; ++j) row.l[4 * k + j] = as_f32(x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) row.l[4 * k + j] = at + j < row.n ? as_f32(in[row.base + at + j]) : -INFINITY;
        }
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) best = max(best, row.key(e));
    best = row.reduce_max(best, 0).a;
    const float t = a.temperature ? a.temperature[r] : 1.f;
    const bool lead = rank == 0 && tid == 0;
    if (best == 0 || !(t > 0.f)) {
        if (lead) {
            a.token[r] = best ? (1 << kIndexBits) - 1 - (int)(best & ((1 << kIndexBits) - 1)) : -1;
            if (a.prob) a.prob[r] = best ? 1.f : 0.f;
            if (a.kept) a.kept[r] = best ? 1 : 0;
        }
        row.barrier();  // no block leaves while its shared memory is read
        return;
    }
    row.m = from_order((unsigned)(best >> kIndexBits));
    row.heat = t;
    const int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.f;
    float low = a.min_p ? a.min_p[r] : 0.f;
    low = low > 0.f ? fminf(low, 1.f) : 0.f;
    u64 from = 1;
    if (k > 0 && k < a.vocab) from = max(from, row.last_kept(false, k, 0.0, 1));
    if (p < 1.f) from = max(from, p > 0.f ? row.last_kept(true, 0, (double)p, from) : best);

    // Kept mass in index order: per (4096-entry tile, warp), then block by block.
    u64 w[4] = {0, 0, 0, 0};
    unsigned cnt = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const u64 c = row.key(e);
        if (c && c >= from) {
            const float x = row.share(e);
            if (x >= low) {
                w[e >> 2] += Row<T>::weight(x);
                ++cnt;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const u64 s = warp_sum64(w[q]);
        if (lane == 0) sm.part[q][warp] = s;
    }
    const u64 c = warp_sum64(cnt);
    if (lane == 0) sm.red[0][warp] = c;
    __syncthreads();
    if (warp == 0) {
        u64 s = sm.part[0][lane] + sm.part[1][lane] + sm.part[2][lane] + sm.part[3][lane];
        s = warp_sum64(s);
        const u64 n = warp_sum64(sm.red[0][lane]);
        if (lane == 0) sm.ex[row.phase] = {s, n};
    }
    row.barrier();
    u64 total = 0, ahead = 0, kept = 0;
    u64 mine = 0;
    for (int b = 0; b < blocks; ++b) {
        const Exchange x = *row.cl.map_shared_rank(&sm.ex[row.phase], b);
        if (b < rank) ahead += x.a;
        if (b == rank) mine = x.a;
        total += x.a;
        kept += x.b;
    }
    row.barrier();  // no block leaves while its shared memory is read
    const float u = a.uniform[r];
    const double scaled = floor((double)u * (double)total);
    u64 goal = scaled > 0.0 ? (u64)scaled : 0;
    goal = min(goal, total - 1);
    if (goal < ahead || goal >= ahead + mine) return;
    goal -= ahead;
    // The (tile, warp) part that holds it, then the thread and the entry.
    u64 run = 0;
    int q = 0, wv = 0;
    for (q = 0; q < 4; ++q) {
        u64 s = 0;
        for (int i = 0; i < 32; ++i) s += sm.part[q][i];
        if (goal < run + s) break;
        run += s;
    }
    for (wv = 0; wv < 32; ++wv) {
        if (goal < run + sm.part[q][wv]) break;
        run += sm.part[q][wv];
    }
    if (wv != warp) return;
    u64 part = q == 0 ? w[0] : q == 1 ? w[1] : q == 2 ? w[2] : w[3];
    u64 incl = part;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (goal < run + incl - part || goal >= run + incl) return;
    run += incl - part;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if ((e >> 2) != q) continue;
        const u64 ky = row.key(e);
        const float x = row.share(e);
        if (!ky || ky < from || !(x >= low)) continue;
        const u64 wt = Row<T>::weight(x);
        if (goal >= run && goal < run + wt) {
            a.token[r] = row.index(e >> 2, e & 3);
            if (a.prob) a.prob[r] = x / ((float)total * 9.094947017729282e-13f);  // 2^-40
            if (a.kept) a.kept[r] = (int)kept;
        }
        run += wt;
    }
}

template <class T>
cudaError_t run(const SampleRowsArgs& a, cudaStream_t st) {
    int blocks = 1;
    while (blocks * kSpan < a.vocab) blocks *= 2;
    auto kern = sample_rows_kernel<T>;
    if (blocks > 8) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * blocks));
    cfg.blockDim = dim3(kThreads);
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
