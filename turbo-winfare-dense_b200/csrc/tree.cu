// Acceptance of drafted token trees: the path from each tree's root along the tokens that were
// drawn at its nodes. A chain's acceptance in the reference (src/speculator.cpp:34-69) is the
// case of one child per node.
//
// One warp per sequence. The tree (up to 256 nodes) comes into shared memory in one round of
// loads; every step looks at all later nodes at once, a lane per node, and takes the lowest
// child of the current node whose token was drawn there. Children come after their parents, so
// the walk ends. It is bound by latency: two rounds of memory and one ballot per accepted level.
#include "common.cuh"
#include "pages.h"

namespace g4b {

namespace {

constexpr int kTreeNodes = 256;

__global__ void __launch_bounds__(32)
    tree_accept_kernel(const int32_t* __restrict__ tokens, const int32_t* __restrict__ parents,
                       const int32_t* __restrict__ sampled, const int32_t* __restrict__ cu_nodes, int n_tokens,
                       int32_t* __restrict__ path, int path_width, int32_t* __restrict__ count,
                       int32_t* __restrict__ next) {
    __shared__ int tok[kTreeNodes], up[kTreeNodes], drawn[kTreeNodes];
    const int s = blockIdx.x, lane = threadIdx.x;
    const int first = min(max(cu_nodes[s], 0), n_tokens);
    const int n = min(min(max(cu_nodes[s + 1] - first, 0), n_tokens - first), kTreeNodes);
    for (int i = lane; i < n; i += 32) {
        tok[i] = tokens[first + i];
        up[i] = parents[first + i];
        drawn[i] = sampled[first + i];
    }
    __syncwarp();
    int32_t* out = path + (long long)s * path_width;
    int cur = 0, taken = 0;
    while (cur < n && taken < path_width) {
        if (lane == 0) out[taken] = cur;
        ++taken;
        const int want = drawn[cur], here = cur;
        cur = n;
        for (int b = (here + 1) & ~31; b < n; b += 32) {
            const int i = b + lane;
            const unsigned hit = __ballot_sync(0xffffffffu, i > here && i < n && up[i] == here && tok[i] == want);
            if (hit) {
                cur = b + __ffs(hit) - 1;
                break;
            }
        }
        if (lane == 0) next[s] = want;
    }
    if (lane == 0) {
        count[s] = taken;
        if (taken == 0) next[s] = -1;
    }
    for (int i = taken + lane; i < path_width; i += 32) out[i] = -1;
}

}  // namespace

cudaError_t tree_accept(const int32_t* tokens, const int32_t* parents, const int32_t* sampled,
                        const int32_t* cu_nodes, int seqs, int n_tokens, int32_t* path, int path_width,
                        int32_t* count, int32_t* next, cudaStream_t st) {
    tree_accept_kernel<<<seqs, 32, 0, st>>>(tokens, parents, sampled, cu_nodes, n_tokens, path, path_width, count,
                                            next);
    return cudaGetLastError();
}

}  // namespace g4b
