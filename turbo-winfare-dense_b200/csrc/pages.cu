// Page keeping of a paged K/V cache: reserving, forking, freeing, compacting and copying pages,
// and committing the rows of an accepted path. The reference keeps one contiguous ring per
// sequence (src/kv_cache.cpp) and has no counterpart.
//
// State is three arrays: a reference count per page (0 = free), a block table row per sequence
// (-1 = no page) and a length per sequence. There is no free list: new pages are the free pages
// of lowest id, given out in (sequence, position) order, so the result depends on the state
// alone and never on the order in which pages came back. Reference counts change by integer
// atomics, whose sums do not depend on their order.
//
// Each call runs the metadata in ONE thread block of 1024 threads: a block scan over the counts costs
// less than a second launch or a grid barrier, as long as refs and table are some KB. With 64 sequences of
// 30000 tokens in 16-row pages (126000 pages, 95 % of them taken, a table of half a megabyte) that block's
// walks are the call: a reserve of one page a sequence 166 us, a fork of 32 sequences 139, a free of 32
// 67, a compaction of 6000 pages 298, the data apart.
// The data moves in a second kernel, launched with programmatic overlap, whose blocks split (page,
// plane, 32 KB part) units, or rows, over all SMs; it is bound by HBM: each byte is read and written once.
// Measured on one B200: 24 forks of partial 32-row pages in 100 planes of 8 KB rows, and their release,
// 111 us (0.58 GB, 0.80 of the measured copy rate, metadata kernels among it), page copies 304 to 312 us for
// 1.8 GB (0.88 to 0.91), a compaction 186 to 189 us for 1.06 GB (0.86).
#include "common.cuh"
#include "launch.cuh"
#include "pages.h"

#include <algorithm>

namespace g4b {

namespace {

constexpr int kMetaThreads = 1024;
constexpr int kSeqsPerThread = kMaxPageSeqs / kMetaThreads;
constexpr int kPartBytes = 32768;  // one copy unit
constexpr int kCopyThreads = 256;

enum PageStatus : int { kPagesOk = 0, kPagesFull = 1, kPagesWidth = 2, kPagesBadSeq = 3, kPagesBadPage = 4 };

// Exclusive block scan of one int per thread (1024 threads); *total receives the block's sum.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) red[w] = x;
    __syncthreads();
    if (w == 0) {
        int s = red[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        red[lane] = s;
    }
    __syncthreads();
    *total = red[31];
    return x - v + (w ? red[w - 1] : 0);
}

__device__ __forceinline__ void copy_ints(int32_t* out, const int32_t* in, long long n) {
    if (out == in) return;
    for (long long i = threadIdx.x; i < n; i += kMetaThreads) out[i] = in[i];
}

__device__ __forceinline__ int pages_for(int rows, int page_size) {
    return (int)(((long long)rows + page_size - 1) / page_size);
}

// Whether `need` of the pages are free.
__device__ bool enough_free(const int32_t* refs, int pages, int need) {
    int have = 0;
    for (int b = 0; b < pages && have < need; b += kMetaThreads) {
        const int p = b + threadIdx.x;
        have += __syncthreads_count(p < pages && refs[p] == 0);
    }
    return have >= need;
}

// Walks the free pages in id order, in windows of 1024 pages: use(first, n) is called by every
// thread with ids[0 .. n) holding the free pages of ranks first .. first + n - 1, until `need`
// ranks are out. refs_out of the pages given becomes 1; a window is read before it is written,
// so refs and refs_out may be one array.
template <class Use>
__device__ void give_free(const int32_t* refs, int32_t* refs_out, int pages, int need, int* ids, int* red, Use use) {
    int have = 0, tot;
    for (int b = 0; b < pages && have < need; b += kMetaThreads) {
        const int p = b + threadIdx.x;
        const bool free = p < pages && refs[p] == 0;
        const int r = block_scan(free, red, &tot);
        if (free) {
            ids[r] = p;
            if (have + r < need) refs_out[p] = 1;
        }
        __syncthreads();
        use(have, min(tot, need - have));
        __syncthreads();
        have += tot;
    }
}

__global__ void __launch_bounds__(kMetaThreads)
    reserve_kernel(PageTables t, const int32_t* __restrict__ grow, int32_t* status) {
    __shared__ int red[32], ids[kMetaThreads];
    int first[kSeqsPerThread], fresh[kSeqsPerThread], col[kSeqsPerThread];
    int need = 0, tot;
    bool bad = false;
#pragma unroll
    for (int q = 0; q < kSeqsPerThread; ++q) {
        const int s = q * kMetaThreads + threadIdx.x;
        fresh[q] = col[q] = 0;
        if (s < t.seqs) {
            const long long len = t.lens[s], want = len + grow[s];
            const long long hi = (want + t.page_size - 1) / t.page_size;
            if (len < 0 || grow[s] < 0 || hi > t.width) {
                bad = true;
            } else {
                col[q] = pages_for((int)len, t.page_size);
                // Entries that an earlier reserve has filled are kept.
                for (int c = col[q]; c < hi; ++c) fresh[q] += t.table[(long long)s * t.width + c] < 0;
            }
        }
        first[q] = need + block_scan(fresh[q], red, &tot);
        need += tot;
    }
    bad = __syncthreads_or(bad);
    copy_ints(t.refs_out, t.refs, t.pages);
    copy_ints(t.table_out, t.table, (long long)t.seqs * t.width);
    const bool ok = !bad && enough_free(t.refs, t.pages, need);
    __syncthreads();  // the copies are in place
    if (ok)
        give_free(t.refs, t.refs_out, t.pages, need, ids, red, [&](int from, int n) {
#pragma unroll
            for (int q = 0; q < kSeqsPerThread; ++q) {
                int32_t* row = t.table_out + (long long)(q * kMetaThreads + threadIdx.x) * t.width;
                while (fresh[q] > 0 && first[q] < from + n) {  // this thread owns the sequence's row
                    while (row[col[q]] >= 0) ++col[q];
                    row[col[q]] = ids[first[q] - from];
                    ++first[q];
                    --fresh[q];
                }
            }
        });
    if (threadIdx.x == 0) *status = bad ? kPagesWidth : ok ? kPagesOk : kPagesFull;
}

__global__ void __launch_bounds__(kMetaThreads)
    free_kernel(PageTables t, const int32_t* __restrict__ seqs, int n) {
    copy_ints(t.refs_out, t.refs, t.pages);
    copy_ints(t.table_out, t.table, (long long)t.seqs * t.width);
    copy_ints(t.lens_out, t.lens, t.seqs);
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = warp; i < n; i += kMetaThreads / 32) {
        const int s = seqs[i];
        if (s < 0 || s >= t.seqs) continue;
        int32_t* row = t.table_out + (long long)s * t.width;
        for (int c = lane; c < t.width; c += 32) {
            // The exchange makes a sequence that is named twice lose its references once.
            const int p = atomicExch(&row[c], -1);
            if (p >= 0 && p < t.pages) atomicSub(&t.refs_out[p], 1);
        }
        if (lane == 0) t.lens_out[s] = 0;
    }
}

__global__ void __launch_bounds__(kMetaThreads)
    fork_kernel(PageTables t, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int n,
                int32_t* status) {
    __shared__ int red[32], ids[kMetaThreads];
    __shared__ unsigned seen[kMaxPageSeqs / 32];
    __shared__ int code;
    if (threadIdx.x == 0) code = kPagesOk;
    for (int i = threadIdx.x; i < kMaxPageSeqs / 32; i += kMetaThreads) seen[i] = 0;
    __syncthreads();
    int rank[kSeqsPerThread], need = 0, tot;
#pragma unroll
    for (int q = 0; q < kSeqsPerThread; ++q) {
        const int i = q * kMetaThreads + threadIdx.x;
        bool part = false;
        if (i < n) {
            const int a = src[i], b = dst[i];
            // Every destination is an empty sequence of its own.
            if (a < 0 || a >= t.seqs || b < 0 || b >= t.seqs || t.lens[b] != 0 ||
                (atomicOr(&seen[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1)
                atomicMax(&code, kPagesBadSeq);
            else if (t.lens[a] < 0 || pages_for(t.lens[a], t.page_size) > t.width)
                atomicMax(&code, kPagesWidth);
            else
                part = t.lens[a] % t.page_size != 0;
        }
        rank[q] = need + block_scan(part, red, &tot);
        if (!part) rank[q] = -1;
        need += tot;
    }
    __syncthreads();
    const bool sound = code == kPagesOk;
    __syncthreads();  // all have read it before one raises it again
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (sound)  // every page that a source holds has to exist, and a destination to hold none
        for (int i = warp; i < n; i += kMetaThreads / 32) {
            const int held = pages_for(t.lens[src[i]], t.page_size);
            const int32_t* row = t.table + (long long)src[i] * t.width;
            const int32_t* own = t.table + (long long)dst[i] * t.width;
            // A source that is also a destination would be read and written at once.
            if ((seen[src[i] >> 5] >> (src[i] & 31)) & 1) atomicMax(&code, kPagesBadSeq);
            for (int c = lane; c < t.width; c += 32) {
                if (c < held && (row[c] < 0 || row[c] >= t.pages)) atomicMax(&code, kPagesBadPage);
                if (own[c] >= 0) atomicMax(&code, kPagesBadSeq);
            }
        }
    copy_ints(t.refs_out, t.refs, t.pages);
    copy_ints(t.table_out, t.table, (long long)t.seqs * t.width);
    copy_ints(t.lens_out, t.lens, t.seqs);
    const bool room = enough_free(t.refs, t.pages, need);
    __syncthreads();
    if (code == kPagesOk && room) {
        // The partial last page becomes a page of the destination's own (copied by the second
        // kernel); the free pages are found before the shared ones' counts grow.
        give_free(t.refs, t.refs_out, t.pages, need, ids, red, [&](int from, int m) {
#pragma unroll
            for (int q = 0; q < kSeqsPerThread; ++q) {
                const int i = q * kMetaThreads + threadIdx.x;
                if (rank[q] >= from && rank[q] < from + m)
                    t.table_out[(long long)dst[i] * t.width + t.lens[src[i]] / t.page_size] = ids[rank[q] - from];
            }
        });
        __syncthreads();
        for (int i = warp; i < n; i += kMetaThreads / 32) {
            // No source is a destination, so its row and length are still the input's.
            const int len = t.lens[src[i]], full = len / t.page_size;
            const int32_t* from = t.table + (long long)src[i] * t.width;
            int32_t* to = t.table_out + (long long)dst[i] * t.width;
            for (int c = lane; c < full; c += 32) {
                const int p = from[c];
                to[c] = p;
                atomicAdd(&t.refs_out[p], 1);
            }
            if (lane == 0 && len > 0) t.lens_out[dst[i]] = len;
        }
    }
    if (threadIdx.x == 0) *status = code != kPagesOk ? code : room ? kPagesOk : kPagesFull;
}

__global__ void __launch_bounds__(kMetaThreads) compact_kernel(PageTables t, int32_t* __restrict__ moves) {
    __shared__ int red[32];
    int live = 0, tot;
    for (int b = 0; b < t.pages; b += kMetaThreads) {
        const int p = b + threadIdx.x;
        live += __syncthreads_count(p < t.pages && t.refs[p] != 0);
    }
    for (int i = threadIdx.x; i < 1 + 2 * t.pages; i += kMetaThreads) moves[i] = -1;
    copy_ints(t.refs_out, t.refs, t.pages);
    copy_ints(t.table_out, t.table, (long long)t.seqs * t.width);
    __syncthreads();
    // The k-th live page at or past `live` moves into the k-th free page before it: as many of
    // the one as of the other.
    int n = 0;
    for (int b = 0; b < live; b += kMetaThreads) {
        const int p = b + threadIdx.x;
        const bool hole = p < live && t.refs[p] == 0;
        const int r = n + block_scan(hole, red, &tot);
        if (hole) moves[2 + 2 * r] = p;
        n += tot;
    }
    n = 0;
    for (int b = live; b < t.pages; b += kMetaThreads) {
        const int p = b + threadIdx.x;
        const bool out = p < t.pages && t.refs[p] != 0;
        const int r = n + block_scan(out, red, &tot);
        if (out) moves[1 + 2 * r] = p;
        n += tot;
    }
    if (threadIdx.x == 0) moves[0] = n;
    __syncthreads();
    const long long cells = (long long)t.seqs * t.width;
    for (long long i = threadIdx.x; i < cells; i += kMetaThreads) {
        const int p = t.table_out[i];
        if (p < live || p >= t.pages) continue;
        int lo = 0, hi = n;  // the moves are in ascending order of their sources
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (moves[1 + 2 * mid] < p) lo = mid + 1;
            else hi = mid;
        }
        if (lo < n && moves[1 + 2 * lo] == p) t.table_out[i] = moves[2 + 2 * lo];
    }
    for (int r = threadIdx.x; r < n; r += kMetaThreads) {
        const int from = moves[1 + 2 * r], to = moves[2 + 2 * r];
        t.refs_out[to] = t.refs_out[from];
        t.refs_out[from] = 0;
    }
}

// Copies `bytes` (a multiple of 16, both ends 16-byte aligned) with the calling threads.
template <int kThreads>
__device__ __forceinline__ void copy_bytes(char* to, const char* from, long long bytes, int tid) {
    const long long n = bytes >> 4;
    const uint4* a = reinterpret_cast<const uint4*>(from);
    uint4* b = reinterpret_cast<uint4*>(to);
    long long i = tid;
    for (; i + 3 * kThreads < n; i += 4 * kThreads) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __ldcs(a + i + k * kThreads);
#pragma unroll
        for (int k = 0; k < 4; ++k) __stcs(b + i + k * kThreads, v[k]);
    }
    for (; i < n; i += kThreads) __stcs(b + i, __ldcs(a + i));
}

// The page copies of a fork, a compaction or a plain copy: what(i, &from, &to, &rows) names the
// i-th pair of pages and how many of their rows are copied.
template <class What>
__device__ __forceinline__ void copy_pages(const PagePool& a, const PagePool& b, int n, int tid, What what) {
    const int parts = (int)(((long long)a.page_size * a.row_bytes + kPartBytes - 1) / kPartBytes);
    const long long units = (long long)n * a.planes * parts;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        // Consecutive blocks take consecutive parts of one page, so the moves are spread evenly
        // whatever their number.
        const int part = (int)(u % parts), plane = (int)(u / parts % a.planes), i = (int)(u / parts / a.planes);
        int from, to, rows;
        what(i, from, to, rows);
        if (from < 0 || from >= a.pages || to < 0 || to >= b.pages) continue;
        const long long at = (long long)part * kPartBytes, left = (long long)rows * a.row_bytes - at;
        if (left <= 0) continue;
        copy_bytes<kCopyThreads>(b.base + plane * b.plane_stride + to * b.page_stride + at,
                                 a.base + plane * a.plane_stride + from * a.page_stride + at,
                                 min(left, (long long)kPartBytes), tid);
    }
}

__global__ void __launch_bounds__(kCopyThreads)
    fork_copy_kernel(PagePool pool, PageTables t, const int32_t* src, const int32_t* dst, int n,
                     const int32_t* status) {
    pdl_wait();
    if (*status != kPagesOk) return;
    copy_pages(pool, pool, n, threadIdx.x, [&](int i, int& from, int& to, int& rows) {
        const int len = t.lens_out[src[i]], full = len / t.page_size;
        rows = len % t.page_size;
        from = to = -1;
        if (rows) {
            from = t.table_out[(long long)src[i] * t.width + full];
            to = t.table_out[(long long)dst[i] * t.width + full];
        }
    });
}

__global__ void __launch_bounds__(kCopyThreads) compact_copy_kernel(PagePool pool, const int32_t* moves) {
    pdl_wait();
    copy_pages(pool, pool, moves[0], threadIdx.x, [&](int i, int& from, int& to, int& rows) {
        from = moves[1 + 2 * i];
        to = moves[2 + 2 * i];
        rows = pool.page_size;
    });
}

__global__ void __launch_bounds__(kCopyThreads)
    copy_kernel(PagePool a, PagePool b, const int32_t* src, const int32_t* dst, int n) {
    copy_pages(a, b, n, threadIdx.x, [&](int i, int& from, int& to, int& rows) {
        from = src[i];
        to = dst[i];
        rows = a.page_size;
    });
}

struct Commit {
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu_nodes;
    const int32_t* path;
    const int32_t* count;
    const int32_t* status;
    int width, path_width, n_tokens, pages, page_size;
};

// Calls use(token, page, row) for each of sequence s's accepted rows, up to the first whose node is not one
// of the sequence's own or whose position has no page, and returns their number. A whole warp: a lane
// looks one of 32 rows up, then all take them one by one.
template <class Use>
__device__ __forceinline__ int commit_rows(const Commit& c, int s, int lane, Use use) {
    const int len = c.lens[s];
    const unsigned n = c.status && *c.status != kPagesOk ? 0 : max(0, min(c.count[s], c.path ? c.path_width : INT_MAX));
    const long long first = c.cu_nodes[s], nodes = c.cu_nodes[s + 1] - first;
    for (unsigned b = 0; b < n; b += 32) {
        const unsigned i = b + lane;
        const unsigned pos = (unsigned)len + i, col = pos / (unsigned)c.page_size, row = pos - col * (unsigned)c.page_size;
        int node = -1, page = -1;
        if (i < n && len >= 0) {  // so pos is below 2^32
            node = c.path ? c.path[(long long)s * c.path_width + i] : (int)i;
            if (col < (unsigned)c.width) page = c.table[(long long)s * c.width + col];
        }
        const bool good = node >= 0 && node < nodes && first >= 0 && first + node < c.n_tokens && page >= 0 && page < c.pages;
        const unsigned bad = ~__ballot_sync(0xffffffffu, good);
        const int m = bad ? __ffs(bad) - 1 : 32;
        for (int k = 0; k < m; ++k)
            use(first + __shfl_sync(0xffffffffu, node, k), __shfl_sync(0xffffffffu, page, k),
                __shfl_sync(0xffffffffu, (int)row, k));
        if (bad) return (int)b + m;
    }
    return (int)n;
}

// One warp per (sequence, plane) moves the accepted rows into the sequence's pages.
__global__ void __launch_bounds__(kCopyThreads)
    commit_kernel(PagePool pool, Commit c, const char* __restrict__ rows, long long rows_plane_stride, int32_t* lens_out) {
    const int s = blockIdx.x, lane = threadIdx.x & 31;
    const int plane = blockIdx.y * (kCopyThreads / 32) + (threadIdx.x >> 5);
    if (plane >= pool.planes) return;
    char* to = pool.base + plane * pool.plane_stride;
    const char* from = rows + plane * rows_plane_stride;
    const int n = commit_rows(c, s, lane, [&](long long token, int page, int row) {
        copy_bytes<32>(to + page * pool.page_stride + (long long)row * pool.row_bytes, from + token * pool.row_bytes,
                       pool.row_bytes, lane);
    });
    if (plane == 0 && lane == 0 && lens_out) lens_out[s] = c.lens[s] + n;
}

// One warp per sequence.
__global__ void __launch_bounds__(kCopyThreads) commit_lens_kernel(Commit c, int32_t* lens, int seqs) {
    const int s = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (s >= seqs) return;
    const int n = commit_rows(c, s, lane, [](long long, int, int) {});
    __syncwarp();  // every lane has read the length
    if (lane == 0) lens[s] += n;
}

int copy_blocks(long long units) { return (int)std::min<long long>(std::max<long long>(units, 1), 148 * 8); }
long long copy_units(const PagePool& p, long long n) {
    return n * p.planes * (((long long)p.page_size * p.row_bytes + kPartBytes - 1) / kPartBytes);
}

}  // namespace

cudaError_t pages_reserve(const PageTables& t, const int32_t* grow, int32_t* status, cudaStream_t st) {
    reserve_kernel<<<1, kMetaThreads, 0, st>>>(t, grow, status);
    return cudaGetLastError();
}

cudaError_t pages_free(const PageTables& t, const int32_t* seqs, int n, cudaStream_t st) {
    free_kernel<<<1, kMetaThreads, 0, st>>>(t, seqs, n);
    return cudaGetLastError();
}

cudaError_t pages_fork(const PagePool& pool, const PageTables& t, const int32_t* src, const int32_t* dst, int n,
                       int32_t* status, cudaStream_t st) {
    fork_kernel<<<1, kMetaThreads, 0, st>>>(t, src, dst, n, status);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || n == 0) return e;
    return launch(fork_copy_kernel, dim3(copy_blocks(copy_units(pool, n))), dim3(kCopyThreads), 0, st, true, pool, t,
                  src, dst, n, status);
}

cudaError_t pages_compact(const PagePool& pool, const PageTables& t, int32_t* moves, cudaStream_t st) {
    compact_kernel<<<1, kMetaThreads, 0, st>>>(t, moves);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch(compact_copy_kernel, dim3(copy_blocks(copy_units(pool, pool.pages / 2))), dim3(kCopyThreads), 0, st,
                  true, pool, moves);
}

cudaError_t pages_copy(const PagePool& from, const PagePool& to, const int32_t* src, const int32_t* dst, int n,
                       cudaStream_t st) {
    copy_kernel<<<copy_blocks(copy_units(from, n)), kCopyThreads, 0, st>>>(from, to, src, dst, n);
    return cudaGetLastError();
}

cudaError_t pages_commit(const PagePool& pool, const int32_t* table, int width, const int32_t* lens, int seqs,
                         const char* rows, long long rows_plane_stride, int n_tokens, const int32_t* cu_nodes,
                         const int32_t* path, int path_width, const int32_t* count, const int32_t* status,
                         int32_t* lens_out, cudaStream_t st) {
    const dim3 grid(seqs, (pool.planes + kCopyThreads / 32 - 1) / (kCopyThreads / 32));
    const Commit c{table, lens, cu_nodes, path, count, status, width, path_width, n_tokens, pool.pages, pool.page_size};
    // With one array for both, other blocks still read the old lengths: they change afterwards.
    const bool apart = lens_out != lens;
    commit_kernel<<<grid, kCopyThreads, 0, st>>>(pool, c, rows, rows_plane_stride, apart ? lens_out : nullptr);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || apart) return e;
    commit_lens_kernel<<<(seqs + kCopyThreads / 32 - 1) / (kCopyThreads / 32), kCopyThreads, 0, st>>>(c, lens_out, seqs);
    return cudaGetLastError();
}

}  // namespace g4b
