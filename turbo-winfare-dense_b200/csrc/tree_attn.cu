// Attention of drafted token trees over a paged K/V cache. Node i of sequence s (its pending token
// is node 0) sits at position lens[s] + depth(i). It sees the cached keys j < lens[s] and, among
// its own sequence's nodes, those whose bit is set in its mask row; a window w > 0 hides keys w or
// more positions back. out = sum_j p_j v_j with p = softmax over the keys it sees of scale * q.k,
// and zero for a node that sees none.
//
// One block per (node, query head): a thread per key of a 128-key tile for the scores, a thread
// per dimension for the products, the online softmax between them in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "tree_attn.h"

namespace g4b {

namespace {

constexpr int kTile = 128;

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

template <class T>
__global__ void __launch_bounds__(kTile) tree_attn_kernel(TreeAttnArgs a) {
    __shared__ float qs[512], p[kTile], red[32];
    __shared__ const T* vrow[kTile];
    const int tok = blockIdx.x, head = blockIdx.y, kvh = head / (a.heads / a.kv_heads), tid = threadIdx.x;
    int s = 0;
    while (s < a.seqs && !(a.cu[s] <= tok && tok < a.cu[s + 1])) ++s;
    if (s == a.seqs) return;
    const int first = a.cu[s], n = min(a.cu[s + 1] - first, a.max_nodes), node = tok - first;
    if (node >= n) return;
    const int len = min(max(a.lens[s], 0), a.width * a.page_size);
    const int dep = a.window ? a.depth[tok] : 0;
    const T* q = static_cast<const T*>(a.q) + tok * a.q_stride + head * a.dim;
    for (int d = tid; d < a.dim; d += kTile) qs[d] = to_f32(q[d]);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const int from = a.window ? max(0, len + dep - a.window + 1) : 0;
    __syncthreads();
    for (int k0 = from / kTile * kTile; k0 < len + n; k0 += kTile) {
        const int j = k0 + tid;
        const T *kr = nullptr, *vr = nullptr;
        if (j >= from && j < len) {
            const int page = a.table[(long long)s * a.width + j / a.page_size];
            if (page >= 0 && page < a.pages) {
                const long long at = page * a.page_stride + ((long long)(j % a.page_size) * a.kv_heads + kvh) * a.dim;
                kr = static_cast<const T*>(a.k_pool) + at;
                vr = static_cast<const T*>(a.v_pool) + at;
            }
        } else if (j >= len && j < len + n) {
            const int i = j - len;
            if (((a.mask[(long long)tok * a.mask_words + i / 32] >> (i % 32)) & 1) &&
                (!a.window || dep - a.depth[first + i] < a.window)) {
                const long long at = (first + i) * a.new_stride + kvh * a.dim;
                kr = static_cast<const T*>(a.k_new) + at;
                vr = static_cast<const T*>(a.v_new) + at;
            }
        }
        float x = -INFINITY;
        if (kr) {
            x = 0.f;
            for (int d = 0; d < a.dim; ++d) x = fmaf(qs[d], to_f32(kr[d]), x);
            x *= a.scale;
        }
        float t = warp_max(x);
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = t;
        vrow[tid] = vr;
        __syncthreads();
        const float mn = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
        p[tid] = kr && mn > -INFINITY ? expf(x - mn) : kr ? 0.f : 0.f;
        __syncthreads();
        const float c = mn == -INFINITY ? 1.f : expf(m - mn);
        m = mn;
        l *= c;
        for (int e = 0; e < 4; ++e) o[e] *= c;
        for (int i = 0; i < kTile; ++i) {
            if (!vrow[i]) continue;
            l += p[i];
            for (int e = 0; e < 4; ++e)
                if (tid + e * kTile < a.dim) o[e] = fmaf(p[i], to_f32(vrow[i][tid + e * kTile]), o[e]);
        }
    }
    T* out = static_cast<T*>(a.out) + tok * a.out_stride + head * a.dim;
    for (int e = 0; e < 4; ++e)
        if (tid + e * kTile < a.dim) out[tid + e * kTile] = from_f32<T>(l != 0.f ? o[e] / l : 0.f);
}

}  // namespace

size_t tree_attn_workspace(int, int, int, int) { return 256; }

cudaError_t tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st) {
    const dim3 grid(a.n_tokens, a.heads);
    if (a.bf16) tree_attn_kernel<__nv_bfloat16><<<grid, kTile, 0, st>>>(a);
    else tree_attn_kernel<__half><<<grid, kTile, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace g4b
