// tree.cuh -- what the kernels of the attention over a cache whose slots are
// not positions share (tree.cu: mma.sync kernel, join, weights; tree_tc.cu:
// tcgen05 kernel).
#pragma once

#include "vbs_b200.h"
#include <cuda.h>
#include "common.cuh"
#include "kernels.h"

namespace vbs {

bool kv_desc_ok(const vbs_cu_kv_t *kv);
bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb);   // bytes from a, from b

struct TreeParams {
    const float *q;
    float *out;
    const uint16_t *kc, *vc;      // layer's first element of sequence 0
    uint64_t seq_stride, pos_step, head_step;
    uint32_t max_ctx, nkh, nqh, G, hd, n_tokens, words, window, ctx_limit;
    uint32_t row_tiles, n_splits, per_split;
    float scale, cap;
    const float *slopes;
    const int32_t *n_ctx, *n_tok;
    const uint32_t *mask;
    const int32_t *q_pos, *k_pos;
    uint32_t k_pos_per_head;
    const float *weights_in;
    float *weights_out;
    // workspace
    float2 *part_ml;              // [slot][split][tile rows]
    float *part_o;                // [slot][split][tile rows][hd], slot = (seq * nkh + kv head) * row_tiles + tile
    float *lse;                   // [seq * nkh + kv head][rows], log2 units, with weights
    uint32_t joined;              // the parts are one cluster and joined in it: no workspace, no second kernel
    uint32_t g_magic;             // ceil(2^32 / G): row / G without a division
    uint32_t *err;
};

constexpr float TREE_LOG2E = 1.4426950408889634f;
// Softmax reference (log2 units): this far below the maximum that set it, moved
// when a weight's exponent would pass TREE_LAZY (2^15.9 rounds to 61152 in
// fp16). The room between is what keeps rescales rare: 3 instead of 5.9 took
// 49.2 us for the 45.9 of 504 rows x 8192 positions.
constexpr float TREE_BELOW = 10.0f, TREE_LAZY = 15.9f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// cap * tanh(x / cap) in log2 units from y = x / cap. Below 0.55 tanh's series
// up to y^15, without a division or an exponential (its next term is 4e-8 of
// the value there): small scores keep their relative accuracy, which 1 - 2 /
// (e^2y + 1) alone, off by 2^-24 of the cap, would not. Below 1 the Pade form
// y (945 + 105 y^2 + y^4) / (945 + 420 y^2 + 15 y^4), off by 6e-8 at most;
// above 1 (e^2y - 1) / (e^2y + 1).
__device__ __forceinline__ float tree_cap_low(float y, float cap2) {
    const float z = y * y;
    float t = fmaf(z, -1.4558344e-3f, 3.5921281e-3f);   // -929569 / 638512875, 21844 / 6081075
    t = fmaf(z, t, -8.8632355e-3f);                     // -1382 / 155925
    t = fmaf(z, t, 2.1869489e-2f);                      // 62 / 2835
    t = fmaf(z, t, -5.3968254e-2f);                     // -17 / 315
    t = fmaf(z, t, 1.3333333e-1f);                      // 2 / 15
    t = fmaf(z, t, -3.3333333e-1f);
    return cap2 * fmaf(y * z, t, y);
}
__device__ __forceinline__ float tree_cap(float y, float cap2) {
    const float a = fminf(fabsf(y), 30.f), z = y * y, e = ex2(a * (2.f * TREE_LOG2E));
    const bool small = a < 1.f;
    const float num = small ? a * fmaf(z, z + 105.f, 945.f) : e - 1.f;
    const float den = small ? fmaf(z, fmaf(z, 15.f, 420.f), 945.f) : e + 1.f;
    const float low = tree_cap_low(y, cap2);
    return y != y ? y : a < 0.55f ? low : copysignf(cap2 * __fdividef(num, den), y);
}

// The same for several scores of a warp, without the upper forms while all are
// below 0.55 (scores well under the cap). A score's result is its own either
// way: the vote also counts scores that nobody sees.
template <int N> __device__ __forceinline__ void tree_cap_all(float (&y)[N], float cap2) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) top = fmaxf(top, fabsf(y[e]));
    if (__all_sync(0xffffffffu, top < 0.55f)) {   // (a NaN stays one either way)
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = tree_cap_low(y[e], cap2);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = tree_cap(y[e], cap2);
    }
}

// Lengths of sequence b; false (flagged once) when they do not fit the cache
// or the call's limit: the sequence is left alone.
__device__ __forceinline__ bool tree_lengths(const TreeParams &p, uint32_t b, uint32_t &nc, uint32_t &nt) {
    const int32_t c = p.n_ctx[b], t = p.n_tok ? p.n_tok[b] : (int32_t)p.n_tokens;
    if (c < 0 || t < 0 || (uint32_t)t > p.n_tokens || (uint64_t)c + t > min(p.max_ctx, p.ctx_limit)) {
        if (threadIdx.x == 0) dev_flag_error(p.err, DERR_BAD_ARG);
        return false;
    }
    nc = (uint32_t)c;
    nt = (uint32_t)t;
    return true;
}

__device__ __forceinline__ int32_t tree_qpos(const TreeParams &p, uint32_t b, uint32_t i, uint32_t nc) {
    return p.q_pos ? p.q_pos[(uint64_t)b * p.n_tokens + i] : (int32_t)(nc + i);
}

// Token of a row (row < 2^20, G <= 256: the product with the rounded-up
// reciprocal is exact).
__device__ __forceinline__ uint32_t tree_token(const TreeParams &p, uint32_t row) {
    return p.G == 1 ? row : __umulhi(row, p.g_magic);
}

// Position of slot t (kpos: the row of k_pos, or NULL).
__device__ __forceinline__ int32_t tree_kpos(const TreeParams &p, const int32_t *kpos, uint32_t b, uint32_t t, uint32_t nc) {
    return kpos ? kpos[t] : (t < nc ? (int32_t)t : tree_qpos(p, b, t - nc, nc));
}

// First slot that any row can see: with a window over plain slots, behind
// the lowest query position's window. All threads of the block call it.
__device__ __forceinline__ uint32_t tree_first(const TreeParams &p, uint32_t b, uint32_t nc, uint32_t nt, int32_t *sh) {
    if (!p.window || p.k_pos) return 0;
    int32_t lo = 0x7FFFFFFF;
    if (p.q_pos) {
        for (uint32_t i = threadIdx.x; i < nt; i += blockDim.x) lo = min(lo, tree_qpos(p, b, i, nc));
        lo = __reduce_min_sync(0xffffffffu, lo);
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = lo;
        __syncthreads();
        for (uint32_t w = 0; w < blockDim.x / 32; ++w) lo = min(lo, sh[w]);
        __syncthreads();
    } else {
        lo = (int32_t)nc;
    }
    const int64_t first = (int64_t)lo - p.window + 1;
    return first <= 0 ? 0u : (uint32_t)min(first, (int64_t)nc) / 64 * 64;   // new tokens are always looked at
}

// This split's positions [t0, t1): equal parts, whole blocks of 64.
__device__ __forceinline__ void tree_part(const TreeParams &p, uint32_t first, uint32_t end, uint32_t split, uint32_t &t0,
                                          uint32_t &t1) {
    const uint32_t span = end - first;
    uint32_t per = (span + p.n_splits - 1) / p.n_splits;
    per = max(p.per_split, (per + 63) / 64 * 64);
    t0 = (uint32_t)min((uint64_t)end, first + (uint64_t)split * per);
    t1 = min(end, t0 + per);
}

// `zero` times the eight halves of v, added up: 0 while all are finite.
__device__ __forceinline__ uint32_t finite4(const uint4 &v, uint32_t zero) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(zero) : "r"(w[k]), "r"(0u));
    return zero & 0x7FFF7FFFu;   // -0 is 0
}

// 64 dims x n positions of one KV head of a cache, from a tensor map of the
// layer's keys or values ([head_dim][position][kv head][seq], rows of 128
// bytes in shared memory, their 16-byte chunks XOR-ed with the position's
// low three bits). Dims from head_dim on and positions from max_ctx on
// arrive as zeros.
__device__ __forceinline__ void tree_tma(uint32_t dst, const CUtensorMap *map, uint32_t dim, uint32_t pos, uint32_t head,
                                         uint32_t seq, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(dim), "r"(pos), "r"(head), "r"(seq), "r"(bar) : "memory");
}

// ---- parts joined in a cluster (CTA rank = part) ---------------------------
__device__ __forceinline__ void cluster_meet() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 cluster_f2(uint32_t a, uint32_t rank) {
    float2 v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [r];\n\t}"
                 : "=f"(v.x), "=f"(v.y) : "r"(a), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_f4(uint32_t a, uint32_t rank) {
    float4 v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a), "r"(rank) : "memory");
    return v;
}

// Every CTA of the cluster has its part's (m, l) per row at `ml` and sums at
// `o` (rows `pitch` bytes apart) of its shared memory, the same places in all;
// the CTAs share the rows' pieces of 16 bytes. Threads tid < n of each call
// it, between the two cluster_meet() that all threads of all CTAs make. Bound
// by the SMs' network: 128 rows of 128 dims from 4 CTAs, 64 KB a CTA, took
// 4700 to 7700 cycles, with deeper loads as with these.
constexpr uint32_t TREE_CLUSTER = 8;
__device__ __forceinline__ void tree_join(const TreeParams &p, uint32_t ml, uint32_t o, uint32_t pitch, uint32_t live, uint32_t R0,
                                          uint32_t kvh, uint32_t b, uint32_t rank, uint32_t tid, uint32_t n) {
    const uint32_t q4 = p.hd / 4, C = p.n_splits;
    for (uint32_t i = rank * n + tid; i < live * q4; i += C * n) {
        const uint32_t r = i / q4, d = i - r * q4;
        float2 x[TREE_CLUSTER];
        float4 v[TREE_CLUSTER];
#pragma unroll
        for (uint32_t c = 0; c < TREE_CLUSTER; ++c) {
            x[c] = make_float2(-INFINITY, 0.f);
            if (c < C) {
                x[c] = cluster_f2(ml + 8 * r, c);
                v[c] = cluster_f4(o + r * pitch + 16 * d, c);
            }
        }
        float M = -INFINITY, L = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t c = 0; c < TREE_CLUSTER; ++c) M = fmaxf(M, x[c].x);
#pragma unroll
        for (uint32_t c = 0; c < TREE_CLUSTER; ++c) {
            if (x[c].y == 0.f) continue;   // an empty part has no sums; a NaN goes through
            const float f = ex2(x[c].x - M);
            L += x[c].y * f;
            a.x = fmaf(v[c].x, f, a.x); a.y = fmaf(v[c].y, f, a.y); a.z = fmaf(v[c].z, f, a.z); a.w = fmaf(v[c].w, f, a.w);
        }
        const float il = L == 0.f ? 0.f : 1.f / L;
        const uint32_t rr = R0 + r, tok = tree_token(p, rr);
        reinterpret_cast<float4 *>(p.out + (((uint64_t)b * p.n_tokens + tok) * p.nqh + kvh * p.G + (rr - tok * p.G)) * p.hd)[d] =
            make_float4(a.x * il, a.y * il, a.z * il, a.w * il);
        if (p.lse && d == 0) p.lse[(uint64_t)(b * p.nkh + kvh) * (p.n_tokens * p.G) + rr] = L == 0.f ? -INFINITY : M + log2f(L);
    }
}

// tree_tc.cu: row tiles of TREE_TC_ROWS, head_dim up to 128.
constexpr uint32_t TREE_TC_ROWS = 128, TREE_TC_SP = 128;
cudaError_t tree_tc_configure(int *clusters);   // clusters[c]: how many of c CTAs run at once
cudaError_t tree_tc_launch(const TreeParams &p, const CUtensorMap &km, const CUtensorMap &vm, uint32_t n_seqs,
                           uint32_t dual, cudaStream_t st);

// Kernel launch whose parts (grid.y) are a cluster, or not.
template <class K, class... A>
inline cudaError_t tree_launch(K kernel, dim3 grid, uint32_t threads, size_t smem, bool joined, cudaStream_t st, const A &...args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
    attr[0].val.clusterDim.y = grid.y;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = joined ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <class K> inline cudaError_t tree_clusters(K kernel, uint32_t threads, size_t smem, int *clusters) {
    for (uint32_t c = 2; c <= TREE_CLUSTER; ++c) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
        attr[0].val.clusterDim.y = c;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(1, c, 1);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters[c], kernel, &cfg);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// tree_wt.cu: the weights per slot, after the attention wrote lse.
cudaError_t tree_weights_configure();
cudaError_t tree_weights_launch(const TreeParams &p, const CUtensorMap &km, uint32_t n_seqs, int n_sm, cudaStream_t st);

}  // namespace vbs
