// tree_wt.cu -- the attention weights per slot of tree.cu's attention:
//   W_t = W_in,t + sum over the rows of a KV head of 2^(x_rt - lse_r),
// x the scores in log2 units, lse from the attention that ran before.
//
// The scores are computed again, transposed, on the tensor cores: S^T = K Q^T
// with the positions as rows, so a thread owns one position, its scores of
// all rows are one line of tensor memory, and the sum over the rows stays in
// a register, in row order: no exchange, no atomics. (Keeping the first
// kernel's scores instead moves 4 bytes per row and position twice: at 128
// rows and 4 x 4096 positions of 8 KV heads 67 MB out and in, 37 us for the
// reading kernel alone, more than K itself.)
//
// CTA = (KV head, up to WT_TILES tiles of 128 positions, sequence); K tiles
// by TMA into a ring; queries in row tiles of 128 (64 above head_dim 128)
// as the second operand, both halves into one accumulator; tiles alternate
// between two streams of 4 warps with two accumulators each, so exponentials
// run beside the next products. Waits are bounded as in tree_tc.cu.
// Bound by the exponentials (2048 cycles of their unit per pair of tiles) and
// the CTA's start: 57 us with the attention for 128 rows x 4 x 4096 positions
// of 8 KV heads of 128, some 25 of them this kernel's (66 with inputs that are
// not in L2).
#include "tree_tc.cuh"

#include <algorithm>

namespace vbs {

namespace {

constexpr int WT_SOFT = 256, WT_THREADS = WT_SOFT + 64;
constexpr int WT_LOADER = WT_SOFT / 32, WT_ISSUER = WT_LOADER + 1;
constexpr uint32_t WT_BLK = TREE_TC_SP * 128u, WT_TILES = 64;

// words of the state behind the queries (bytes)
constexpr uint32_t W_FULL = 0, W_EMPTY = 64, W_S = 128, W_F = 160, W_END = 192, W_TMEM = 200, W_BAD = 204, W_QMAX = 208;
constexpr uint32_t W_ROW = 256;                          // per row: factor and lse (8 bytes), query position and slope (8 bytes)
constexpr uint32_t W_POS = W_ROW + 128 * 16, W_SUM = W_POS, W_BYTES = W_SUM + WT_TILES * TREE_TC_SP * 4;

struct WtParams {
    TreeParams t;
    CUtensorMap km;
    uint32_t ns, hdp, blks, rows, per, q_off, h_off;   // stages, padded head_dim, boxes per tile, rows per tile, tiles per CTA, offsets
};

template <int D>
__global__ void __launch_bounds__(WT_THREADS, 1) tree_weights_kernel(const __grid_constant__ WtParams wp) {
    const TreeParams &p = wp.t;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *const hs = smem + wp.h_off;
    const uint32_t stage0 = smem_u32(smem), base = stage0 + wp.h_off;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t kvh = blockIdx.x, b = blockIdx.z;
    const uint32_t hdp = wp.hdp, chunks = hdp / 8, slot = wp.blks * WT_BLK, q_lo = wp.rows * hdp * 2;
    volatile int *bad = reinterpret_cast<volatile int *>(hs + W_BAD);
    float2 *row_fl = reinterpret_cast<float2 *>(hs + W_ROW);                   // factor, lse
    int2 *row_ps = reinterpret_cast<int2 *>(hs + W_ROW + 128 * 8);             // query position, slope (bits)
    float *sums = reinterpret_cast<float *>(hs + W_SUM);
    uint32_t nc, nt;
    if (!tree_lengths(p, b, nc, nt)) return pdl_wait();   // (nobody ends before the attention has)
    const uint32_t end = nc + nt, R = nt * p.G;
    const uint32_t t0 = blockIdx.y * wp.per * TREE_TC_SP, t1 = min(end, t0 + wp.per * TREE_TC_SP);
    if (t0 >= t1) return pdl_wait();
    const uint64_t out_at = (uint64_t)(b * p.nkh + kvh) * p.max_ctx;
    const uint32_t first = tree_first(p, b, nc, nt, reinterpret_cast<int32_t *>(hs + W_ROW));
    if (t1 <= first || !R) {   // in nobody's window, or nobody there
        for (uint32_t t = t0 + threadIdx.x; t < t1; t += WT_THREADS) p.weights_out[out_at + t] = p.weights_in ? p.weights_in[out_at + t] : 0.f;
        return pdl_wait();
    }
    const uint32_t ntl = (t1 - t0 + TREE_TC_SP - 1) / TREE_TC_SP, rts = (R + wp.rows - 1) / wp.rows;
    const int32_t *kpos = p.k_pos ? p.k_pos + (uint64_t)(p.k_pos_per_head ? b * p.nkh + kvh : b) * p.max_ctx : nullptr;
    auto waits = [&](uint32_t bar, uint32_t parity) -> bool {
        if (mbar_wait_bounded(bar, parity, kWaitNs)) return true;
        *bad = 1;
        return false;
    };
    auto all = [&](bool x) { return __all_sync(0xffffffffu, x); };

    // item: tile i in stage s, once per row tile (stages, phases and tiles are
    // counted along: a division would cost an issuer more than a wait)
    auto load = [&](uint32_t i, uint32_t s) {
        const uint32_t tb = t0 + i * TREE_TC_SP;
        if (lane == 0) {
            mbar_arrive_expect_tx(base + W_FULL + 8 * s, slot);
            for (uint32_t k = 0; k < wp.blks; ++k)
                tree_tma(stage0 + s * slot + k * WT_BLK, &wp.km, 64 * k, tb, kvh, b, base + W_FULL + 8 * s);
        }
        __syncwarp();
    };
    uint32_t it = 0;
    if (warp == WT_LOADER) {
        if (lane == 0) {
            for (uint32_t s = 0; s < wp.ns; ++s) {
                mbar_init(base + W_FULL + 8 * s, 1);
                mbar_init(base + W_EMPTY + 8 * s, 1);
            }
            for (uint32_t a = 0; a < 4; ++a) {
                mbar_init(base + W_S + 8 * a, 1);
                mbar_init(base + W_F + 8 * a, 4);
            }
            mbar_init(base + W_END, 1);
            *bad = 0;
            mbar_fence_init();
        }
        __syncwarp();
        load(0, 0);
        it = 1;
    } else if (warp == WT_ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + W_TMEM), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        int32_t hi = (int32_t)0x80000000;   // highest query position, for the tiles inside everybody's window
        if (p.window)
            for (uint32_t i = lane; i < nt; i += 32) hi = max(hi, tree_qpos(p, b, i, nc));
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) *reinterpret_cast<int32_t *>(hs + W_QMAX) = hi;
    }
    // a row tile's queries; the first one's do not wait for the attention
    float qf[2] = {0.f, 0.f};
    auto queries = [&](uint32_t rt) {
        TcQ<D> q[D > 128 ? 1 : 2];
        const uint32_t row = 8 * warp + (lane & 7);
#pragma unroll
        for (int g = 0; g < (D > 128 ? 1 : 2); ++g) tc_q_load(p, rt * wp.rows + row + 64 * g, R, kvh, b, q[g]);
#pragma unroll 1
        for (int g = 0; g < (D > 128 ? 1 : 2); ++g) {
            const float f = tc_q_store(p, q[0], smem + wp.q_off, wp.rows * 16, q_lo, row + 64 * g, chunks);
            if (g) qf[1] = f;
            else qf[0] = f;
            if constexpr (D <= 128) q[0] = q[1];
        }
        tc_proxy();
    };
    if (warp < WT_LOADER) queries(0);
    for (uint32_t i = threadIdx.x; i < ntl * TREE_TC_SP; i += WT_THREADS) sums[i] = 0.f;
    tc_before();
    __syncthreads();
    tc_after();
    pdl_wait();   // lse of the attention before
    const uint32_t tmem = *reinterpret_cast<uint32_t *>(hs + W_TMEM);
    const int32_t qmax = *reinterpret_cast<const int32_t *>(hs + W_QMAX);

    if (warp == WT_LOADER) {
        for (uint32_t i = 1, s = 1, ph = 1; it < rts * ntl; ++it) {   // ph: parity of the last time round
            if (i == ntl) i = 0;
            if (s == wp.ns) { s = 0; ph ^= 1u; }
            if (!all(!*bad && (it < wp.ns || waits(base + W_EMPTY + 8 * s, ph)))) break;
            load(i++, s++);
        }
        if (*bad && lane == 0)   // copies may still be landing
            for (uint32_t k = it > wp.ns ? it - wp.ns : 0; k < it; ++k)
                mbar_wait_bounded(base + W_FULL + 8 * (k % wp.ns), (k / wp.ns) & 1u, kWaitNs);
        __syncwarp();
    } else {
        const uint32_t w = (warp >> 2) & 1, wq = warp & 3, r = 32 * wq + lane;   // stream, quadrant, position in the tile
        const uint32_t lead = warp == WT_ISSUER ? tc_elect() : 0u;
        const float cap2 = p.cap * TREE_LOG2E;
        bool ok = true;
        uint32_t s = 0, ph = 0;             // issuer: stage and parity
        uint32_t free = 15u, full = 0u;     // parities of the four accumulators' barriers (the first wait for `free` passes)
        for (uint32_t rt = 0; rt < rts; ++rt) {
            const uint32_t rows = min(wp.rows, R - rt * wp.rows), N = (rows + 31) / 32 * 32;
            if (warp < WT_LOADER) {
                // the row tile's queries and numbers: all loads first
                constexpr int NG = D > 128 ? 1 : 2;   // 8s of rows per warp
                if (rt) queries(rt);
                float z[NG], sl[NG];
                int32_t qp[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t row = 8 * (warp + 8 * g) + (lane & 7), rr = row < rows ? rt * wp.rows + row : 0u, tok = tree_token(p, rr);
                    z[g] = row < rows ? __ldcg(p.lse + (uint64_t)(b * p.nkh + kvh) * (p.n_tokens * p.G) + rr) : -INFINITY;
                    qp[g] = tree_qpos(p, b, tok, nc);
                    sl[g] = p.slopes ? p.slopes[kvh * p.G + (rr - tok * p.G)] * TREE_LOG2E : 0.f;
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t row = 8 * (warp + 8 * g) + (lane & 7);
                    if (lane < 8) {
                        // a row that is not there or sees nothing: weight 2^(0 - inf) = 0
                        row_fl[row] = z[g] == -INFINITY ? make_float2(0.f, INFINITY) : make_float2(qf[g], z[g]);
                        row_ps[row] = make_int2(qp[g], __float_as_int(sl[g]));
                    }
                }
            }
            named_bar_sync(1, WT_SOFT + 32);   // queries in place
            if (warp == WT_ISSUER) {
                const uint32_t id = (1u << 4) | ((N >> 3) << 17) | ((TREE_TC_SP >> 4) << 24), qp = wp.rows * 16;
                const uint64_t dk = tc_desc_sw(stage0, 16u, 1024u), dq = tc_desc(stage0 + wp.q_off, qp, 128u);
                for (uint32_t i = 0; ok && i < ntl; ++i) {
                    const uint32_t sw = i & 3;
                    ok = all(!*bad && waits(base + W_FULL + 8 * s, ph) && waits(base + W_F + 8 * sw, (free >> sw) & 1u));
                    free ^= 1u << sw;
                    if (!ok) break;
                    tc_after();
                    const uint64_t d = dk + s * (slot / 16);
#pragma unroll
                    for (uint32_t k = 0; k < D / 16; ++k) {
                        if (k >= hdp / 16) break;
                        const uint64_t da = d + (k >> 2) * (WT_BLK / 16) + (k & 3) * 2, db = dq + 2 * k * (qp / 16);
                        tc_mma_ss(tmem + 128 * sw, da, db + q_lo / 16, id, k ? 1u : 0u, lead);   // the small part first (tree_tc.cu)
                    }
#pragma unroll
                    for (uint32_t k = 0; k < D / 16; ++k) {
                        if (k >= hdp / 16) break;
                        const uint64_t da = d + (k >> 2) * (WT_BLK / 16) + (k & 3) * 2, db = dq + 2 * k * (qp / 16);
                        tc_mma_ss(tmem + 128 * sw, da, db, id, 1u, lead);
                    }
                    if (lead) {
                        tc_commit(base + W_S + 8 * sw);
                        tc_commit(base + W_EMPTY + 8 * s);
                    }
                    __syncwarp();
                    if (++s == wp.ns) { s = 0; ph ^= 1u; }
                }
            } else {
                auto kp_at = [&](uint32_t t) { return t < t1 ? tree_kpos(p, kpos, b, t, nc) : -1; };
                int32_t kn = kp_at(t0 + w * TREE_TC_SP + r);   // the next tile's, ahead
                for (uint32_t i = w; ok && i < ntl; i += 2) {
                    const uint32_t tb = t0 + i * TREE_TC_SP, t = tb + r, sw = i & 3, sa = tmem + ((32u * wq) << 16) + 128 * sw;
                    const bool in = t < t1;
                    const int32_t kp = kn;
                    kn = kp_at(t + 2 * TREE_TC_SP);
                    const bool seen = in && (!kpos || kp >= 0);            // by some row
                    const bool drafts = tb + TREE_TC_SP > nc;              // the mask decides
                    const bool edge = p.window && (kpos || drafts || qmax - (int32_t)tb >= (int32_t)p.window);
                    // rows whose mask shows a drafted position, a bit each (before the wait)
                    uint32_t rows_see[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
                    if (drafts && in && t >= nc) {
                        const uint32_t j = t - nc, g0 = rt * wp.rows;
                        rows_see[0] = rows_see[1] = rows_see[2] = rows_see[3] = 0u;
                        const uint32_t tok0 = tree_token(p, g0), tok1 = tree_token(p, g0 + rows - 1);
#pragma unroll 4
                        for (uint32_t k = tok0; k <= tok1; ++k) {
                            const bool see = p.mask ? (p.mask[((uint64_t)b * p.n_tokens + k) * p.words + (j >> 5)] >> (j & 31)) & 1u : j <= k;
                            // the token's rows of this tile
                            const int lo = max(0, (int)(k * p.G) - (int)g0), hi = min((int)rows, (int)((k + 1) * p.G) - (int)g0);
                            if (see)
#pragma unroll
                                for (int x = 0; x < 4; ++x) rows_see[x] |= ones(hi - 32 * x) & ~ones(lo - 32 * x);
                        }
                    }
                    ok = all(!*bad && waits(base + W_S + 8 * sw, (full >> sw) & 1u));
                    full ^= 1u << sw;
                    if (!ok) break;
                    tc_after();
                    float sum = 0.f;
                    if (!drafts && !edge && !p.slopes && !(p.cap > 0.f)) {
                        uint32_t x[2][32];
                        tc_ld32(sa, x[0]);
                        tc_wait_ld(x[0]);
                        // the next 32 on their way (behind N: columns that nobody reads); short code, it starts cold
#pragma unroll 1
                        for (uint32_t c = 0; c < N; c += 64) {
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                if (c + 32 * u >= N) break;
                                tc_ld32(sa + ((c + 32 * u + 32) & 127), x[u ^ 1]);
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    const float2 fl = row_fl[c + 32 * u + e];
                                    sum += ex2(fmaf(__uint_as_float(x[u][e]), fl.x, -fl.y));
                                }
                                tc_wait_ld(x[u ^ 1]);
                            }
                        }
                    } else {
#pragma unroll 1
                        for (uint32_t c = 0; c < N; c += 16) {
                            uint32_t x[16];
                            tc_ld16(sa + c, x);
                            const uint32_t bits = (c < 64 ? (c < 32 ? rows_see[0] : rows_see[1]) : (c < 96 ? rows_see[2] : rows_see[3])) >> (c & 31);
                            tc_wait_ld(x);
                            float y[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) y[e] = __uint_as_float(x[e]) * row_fl[c + e].x;
                            if (p.cap > 0.f) tree_cap_all(y, cap2);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float2 fl = row_fl[c + e];
                                const int2 ps = row_ps[c + e];
                                float v = y[e];
                                if (p.slopes) v = fmaf(__int_as_float(ps.y), (float)(kp - ps.x), v);
                                const bool see = c + e < rows && ((bits >> e) & 1u) && (!p.window || ps.x - kp < (int32_t)p.window);
                                sum += see ? ex2(v - fl.y) : 0.f;
                            }
                        }
                    }
                    if (seen) sums[i * TREE_TC_SP + r] += sum;
                    tc_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(base + W_F + 8 * sw);
                }
            }
            named_bar_sync(1, WT_SOFT + 32);   // the row tile is through (its products were waited for by those who read them)
        }
        if (warp == WT_ISSUER) {
            if (lead) tc_commit(base + W_END);
            __syncwarp();
        } else {
            for (uint32_t i = w; ok && i < ntl; i += 2) {
                const uint32_t t = t0 + i * TREE_TC_SP + r;
                if (t < t1) p.weights_out[out_at + t] = (p.weights_in ? p.weights_in[out_at + t] : 0.f) + sums[i * TREE_TC_SP + r];
            }
        }
    }
    tc_before();
    __syncthreads();
    if (warp == WT_ISSUER) {
        if (lane == 0) {
            mbar_wait_bounded(base + W_END, 0, kWaitNs);   // the tensor memory goes back after the last product
            if (*bad) dev_flag_error(p.err, DERR_TIMEOUT_FULL);
        }
        __syncwarp();
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace

cudaError_t tree_weights_configure() {
    cudaError_t e = cudaFuncSetAttribute(tree_weights_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tree_weights_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    return e;
}

cudaError_t tree_weights_launch(const TreeParams &t, const CUtensorMap &km, uint32_t n_seqs, int n_sm, cudaStream_t st) {
    WtParams p = {};
    p.t = t;
    p.km = km;
    p.hdp = (t.hd + 15) / 16 * 16;
    p.blks = (t.hd + 63) / 64;
    p.rows = t.hd > 128 ? 64 : 128;
    const uint32_t q_bytes = 2 * p.rows * p.hdp * 2;
    p.ns = std::min(8u, (232448u - q_bytes - W_BYTES) / (p.blks * WT_BLK));   // hd 128: 4, hd 256: 2
    p.q_off = p.ns * p.blks * WT_BLK;
    p.h_off = p.q_off + q_bytes;
    // one CTA per SM: as many tiles each as that takes, at most WT_TILES
    const uint32_t tiles = (t.ctx_limit + TREE_TC_SP - 1) / TREE_TC_SP;
    const uint64_t units = (uint64_t)t.nkh * n_seqs;
    const uint32_t parts = std::max((uint32_t)std::max<uint64_t>(1, n_sm / units), (tiles + WT_TILES - 1) / WT_TILES);
    p.per = (tiles + parts - 1) / parts;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(t.nkh, (tiles + p.per - 1) / p.per, n_seqs);
    cfg.blockDim = dim3(WT_THREADS);
    cfg.dynamicSmemBytes = p.h_off + W_BYTES;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return t.hd > 128 ? cudaLaunchKernelEx(&cfg, tree_weights_kernel<256>, p) : cudaLaunchKernelEx(&cfg, tree_weights_kernel<128>, p);
}

}  // namespace vbs
