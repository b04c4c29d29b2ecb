// tree_tc.cu -- attention of many rows over a cache on the 5th-generation
// tensor cores (tcgen05.mma, scores, weights and accumulators in tensor
// memory). The formula, the split of the positions and the halves of fp32
// queries and weights are those of tree.cu; this kernel serves row tiles of
// 128 with head_dim up to 128.
//
// CTA = (KV head, 128 rows, part of the positions, sequence), positions in
// tiles of 128. Tiles alternate between two streams, each with its own
// scores (128 columns of tensor memory), accumulator (128 columns) and
// softmax state, so one stream's softmax runs beside the other's products;
// the two are joined at the end.
//  * One thread stages K and V tiles (32 KB each at head_dim 128) into a ring
//    with TMA, 64 dims x 128 positions a box, rows of 128 bytes with the
//    128-byte swizzle. The image is a K-major operand for Q K^T (MN =
//    position, K = dim) and an MN-major one for P V (MN = dim, K = position).
//    (Staged with cp.async by 4 warps in the layout without swizzle, a tile
//    took 2100 cycles to issue and was the bottleneck: 82.6 us for 504 rows x
//    8192 positions x 8 KV heads of 128.)
//  * One thread issues tcgen05.mma: S = Qhi K^T + Qlo K^T (both operands in
//    shared memory), O += Phi V + Plo V (P from tensor memory).
//  * 2 x 4 softmax warps, a thread per row: the scores are read 32 columns at
//    a time, once for the maximum and once for the weights, which go back
//    over them as fp16 halves (columns 32 c .. + 15 the high, + 16 .. + 31
//    the low halves of positions 32 c ..). The accumulator is rescaled in
//    place when the maximum moves by more than TREE_LAZY.
//  * A weight is split by cutting its mantissa (hi exact in fp16, lo = p -
//    hi rounded): one AND and one subtraction, no conversion back.
// All waits are bounded; after one ran out the CTA flags the device error
// word, waits for its copies and products, frees its tensor memory and ends.
#include "tree.cuh"

#include <algorithm>

namespace vbs {

namespace {

constexpr int TC_SOFT = 256, TC_THREADS = TC_SOFT + 64;   // softmax warps, the loader, the product issuer
constexpr int TC_LOADER = TC_SOFT / 32, TC_ISSUER = TC_LOADER + 1;
constexpr uint32_t TC_HDR = 1024;   // barriers and flags, then the rows' factors
constexpr uint32_t TC_BLK = TREE_TC_SP * 128u;   // one box: 128 positions x 64 dims

// header words (bytes)
constexpr uint32_t H_FULL = 0, H_EMPTY = 64, H_S = 128, H_P = 144, H_O = 160, H_END = 176, H_TMEM = 192, H_BAD = 196, H_ACC = 200, H_QMAX = 208,
                   H_FAC = 512;

struct TcParams {
    TreeParams t;
    CUtensorMap km, vm;
    uint32_t ns, ring, hdp, blks, q_off, st_off;   // stages, key-position tiles, padded head_dim, boxes per tile, offsets
};

__device__ __forceinline__ uint64_t tc_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
// The same with the 128-byte swizzle (layout type 2): rows of 128 bytes, 8 of
// them in 1024. K-major: sbo = 1024 from 8 rows to the next, a step of 16
// along K advances the address by 32 bytes. MN-major: sbo from 8 K rows to
// the next, lbo from 64 MN elements to the next.
__device__ __forceinline__ uint64_t tc_desc_sw(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return tc_desc(saddr, lbo, sbo) | (2ull << 61);
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u) : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tc_ld32(uint32_t a, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(a));
}
__device__ __forceinline__ void tc_st32(uint32_t a, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tc_ld8(uint32_t a, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(a));
}
__device__ __forceinline__ void tc_st8(uint32_t a, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void tc_ld1(uint32_t a, uint32_t &v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(a));
}
// or of pred over the `n` threads of barrier `id`
__device__ __forceinline__ bool bar_or(uint32_t id, uint32_t n, bool pred) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %3, 0;\n barrier.cta.red.or.pred.aligned q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r) : "r"(id), "r"(n), "r"(pred ? 1u : 0u) : "memory");
    return r != 0;
}
__device__ __forceinline__ uint32_t ones(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }
__device__ __forceinline__ bool not_finite2(uint32_t w) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; }

__global__ void __launch_bounds__(TC_THREADS, 1) tree_tc_kernel(const __grid_constant__ TcParams tp) {
    const TreeParams &p = tp.t;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t kvh = blockIdx.x % p.nkh, tile = blockIdx.x / p.nkh, split = blockIdx.y, b = blockIdx.z;
    const uint32_t G = p.G, R0 = tile * TREE_TC_ROWS, hdp = tp.hdp, chunks = hdp / 8, slot = tp.blks * TC_BLK;
    volatile int *bad = reinterpret_cast<volatile int *>(smem + H_BAD);
    int32_t *sh_min = reinterpret_cast<int32_t *>(smem + 256);   // before the barriers are used
    uint32_t nc, nt;
    if (!tree_lengths(p, b, nc, nt) || R0 >= nt * G) return;
    const uint32_t end = nc + nt, nrows = min(TREE_TC_ROWS, nt * G - R0);
    const uint32_t first = tree_first(p, b, nc, nt, sh_min);
    uint32_t t0, t1;
    tree_part(p, first, end, split, t0, t1);
    const uint64_t slot_id = (uint64_t)(b * p.nkh + kvh) * p.row_tiles + tile;
    float2 *ml = p.part_ml + (slot_id * p.n_splits + split) * TREE_TC_ROWS;
    if (t0 >= t1 && p.n_splits > 1) {
        for (uint32_t r = threadIdx.x; r < TREE_TC_ROWS; r += TC_THREADS) ml[r] = make_float2(-INFINITY, 0.f);
        return;
    }
    const uint32_t nch = (t1 - t0 + TREE_TC_SP - 1) / TREE_TC_SP;
    const uint32_t aw = (nrows + 31) / 32;   // softmax warps of a stream that have rows
    const bool want_pos = p.k_pos || p.window || p.slopes;
    const int32_t *kpos = p.k_pos ? p.k_pos + (uint64_t)(p.k_pos_per_head ? b * p.nkh + kvh : b) * p.max_ctx : nullptr;
    const int32_t *qpos_b = p.q_pos ? p.q_pos + (uint64_t)b * p.n_tokens : nullptr;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < tp.ns; ++s) {
            mbar_init(base + H_FULL + 8 * s, 1);
            mbar_init(base + H_EMPTY + 8 * s, 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(base + H_S + 8 * w, 1);
            mbar_init(base + H_P + 8 * w, aw);
            mbar_init(base + H_O + 8 * w, 1);
        }
        mbar_init(base + H_END, 1);
        *bad = 0;
        reinterpret_cast<int *>(smem + H_ACC)[0] = reinterpret_cast<int *>(smem + H_ACC)[1] = 0;
        *reinterpret_cast<int32_t *>(smem + H_QMAX) = (int32_t)0x80000000;
        mbar_fence_init();
    }
    if (warp == TC_ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + H_TMEM), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *reinterpret_cast<uint32_t *>(smem + H_TMEM);
    auto waits = [&](uint32_t bar, uint32_t parity) -> bool {
        if (mbar_wait_bounded(bar, parity, kWaitNs)) return true;
        *bad = 1;
        return false;
    };

    if (warp == TC_LOADER) {
        // ---------------- loader: items K0 V0 K1 V1 ... --------------------
        const uint32_t items = 2 * nch;
        uint32_t it = 0;
        for (; it < items; ++it) {
            const uint32_t s = it % tp.ns, i = it / 2, tb = t0 + i * TREE_TC_SP;
            if (!__all_sync(0xffffffffu, !*bad && (it < tp.ns || waits(base + H_EMPTY + 8 * s, (it / tp.ns - 1) & 1u)))) break;
            if (!(it & 1) && want_pos) {   // the tile's key positions, before its keys are announced
                for (uint32_t k = lane; k < TREE_TC_SP; k += 32) {
                    const uint32_t t = tb + k;
                    int32_t kp = 0;
                    if (t < t1) kp = kpos ? kpos[t] : (t < nc || !qpos_b ? (int32_t)t : qpos_b[t - nc]);
                    reinterpret_cast<int32_t *>(smem + TC_HDR)[(i % tp.ring) * TREE_TC_SP + k] = kp;
                }
                __syncwarp();
            }
            if (lane == 0) {
                mbar_arrive_expect_tx(base + H_FULL + 8 * s, slot);
                for (uint32_t k = 0; k < tp.blks; ++k)
                    tree_tma(base + tp.st_off + s * slot + k * TC_BLK, (it & 1) ? &tp.vm : &tp.km, 64 * k, tb, kvh, b, base + H_FULL + 8 * s);
            }
            __syncwarp();
        }
        // after a failed wait copies may still be landing: the newest of
        // every slot is waited for before the CTA ends
        if (*bad && lane == 0)
            for (uint32_t k = it > tp.ns ? it - tp.ns : 0; k < it; ++k)
                mbar_wait_bounded(base + H_FULL + 8 * (k % tp.ns), (k / tp.ns) & 1u, kWaitNs);
    }
    if (warp < TC_SOFT / 32) {
        // ---------------- queries: 16 rows per warp -------------------------
        float *fac_sm = reinterpret_cast<float *>(smem + H_FAC);
        const uint32_t r8 = lane & 7, c4 = lane >> 3;
#pragma unroll 1
        for (uint32_t half = 0; half < 2; ++half) {
            const uint32_t r = 16 * warp + 8 * half + r8;
            const bool on = r < nrows;
            const uint32_t rr = R0 + (on ? r : 0u);
            const float *src = p.q + (((uint64_t)b * p.n_tokens + rr / G) * p.nqh + kvh * G + rr % G) * p.hd;
            float4 x[4][2];
            float top = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t c = 4 * j + c4;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    x[j][u] = on && c < p.hd / 8 ? *reinterpret_cast<const float4 *>(src + 8 * c + 4 * u) : make_float4(0.f, 0.f, 0.f, 0.f);
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(x[j][u].x), fabsf(x[j][u].y)), fmaxf(fabsf(x[j][u].z), fabsf(x[j][u].w))));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            int e = (int)((__float_as_uint(top) >> 23) & 255u) - 127;   // as in tree_mma_kernel
            e = (e < -100 || e > 100) ? 0 : 8 - e;
            const float up = __uint_as_float((uint32_t)(127 + e) << 23) * (p.scale < 0.f ? -1.f : 1.f);
            if (c4 == 0)
                fac_sm[r] = fabsf(p.scale) * __uint_as_float((uint32_t)(127 - e) << 23) * (p.cap > 0.f ? 1.f / p.cap : TREE_LOG2E);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t c = 4 * j + c4;
                if (c >= chunks) continue;
                uint32_t hi[4], lo[4];
                const float v[8] = {x[j][0].x, x[j][0].y, x[j][0].z, x[j][0].w, x[j][1].x, x[j][1].y, x[j][1].z, x[j][1].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float v0 = v[2 * k] * up, v1 = v[2 * k + 1] * up;
                    const __half2 h = __floats2half2_rn(v0, v1);
                    const float2 f = __half22float2(h);
                    const __half2 l = __floats2half2_rn(v0 - f.x, v1 - f.y);
                    hi[k] = *reinterpret_cast<const uint32_t *>(&h);
                    lo[k] = *reinterpret_cast<const uint32_t *>(&l);
                }
                uint8_t *d = smem + tp.q_off + c * (TREE_TC_ROWS * 16u) + r * 16u;
                *reinterpret_cast<uint4 *>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(d + chunks * (TREE_TC_ROWS * 16u)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        if (p.window) {   // highest query position of the tile's rows, for the tiles inside everybody's window
            int32_t q = (int32_t)0x80000000;
            if (threadIdx.x < nrows) q = tree_qpos(p, b, (R0 + threadIdx.x) / G, nc);
            q = __reduce_max_sync(0xffffffffu, q);
            if (lane == 0) atomicMax(reinterpret_cast<int32_t *>(smem + H_QMAX), q);
        }
        tc_proxy();
    }
    // queries are in place (the loader has gone ahead: named barrier of the others)
    if (warp != TC_LOADER) named_bar_sync(1, TC_SOFT + 32);

    if (warp == TC_ISSUER) {
        if (lane == 0) {
            // ---------------- tensor core issue (one thread) ----------------
            const uint32_t idq = (1u << 4) | ((TREE_TC_SP >> 3) << 17) | ((TREE_TC_ROWS >> 4) << 24);
            const uint32_t idp = (1u << 4) | (1u << 16) | ((hdp >> 3) << 17) | ((TREE_TC_ROWS >> 4) << 24);
            const uint32_t qa = base + tp.q_off, qlo = chunks * (TREE_TC_ROWS * 16u);   // high halves, low halves
            constexpr uint32_t QCH = TREE_TC_ROWS * 16u;   // bytes per chunk of the queries
            bool ok = true;
            auto pv = [&](uint32_t j) -> bool {
                const uint32_t w = j & 1, s = (2 * j + 1) % tp.ns;
                if (!waits(base + H_FULL + 8 * s, ((2 * j + 1) / tp.ns) & 1u) || !waits(base + H_P + 8 * w, (j / 2) & 1u)) return false;
                tc_after();
                const uint32_t v = base + tp.st_off + s * slot, o = tmem + 256 + 128 * w, pa = tmem + 128 * w;
                const bool acc0 = j >= 2 || reinterpret_cast<volatile int *>(smem + H_ACC)[w];
                const uint32_t steps = (min(TREE_TC_SP, t1 - t0 - j * TREE_TC_SP) + 15) / 16;
                for (uint32_t k = 0; k < steps; ++k) {
                    const uint64_t d = tc_desc_sw(v + k * 2048u, TC_BLK, 1024u);
                    const uint32_t a = pa + 32 * (k >> 1) + 8 * (k & 1);
                    tc_mma_ts(o, a + 16, d, idp, acc0 || k > 0);
                    tc_mma_ts(o, a, d, idp, true);
                }
                tc_commit(base + H_EMPTY + 8 * s);
                tc_commit(base + H_O + 8 * w);
                return true;
            };
            for (uint32_t i = 0; ok && i < nch; ++i) {
                const uint32_t w = i & 1, s = (2 * i) % tp.ns;
                ok = waits(base + H_FULL + 8 * s, ((2 * i) / tp.ns) & 1u);
                if (ok && i >= 2) ok = waits(base + H_O + 8 * w, (i / 2 - 1) & 1u);   // this stream's weights are used up
                if (!ok) break;
                tc_after();
                const uint32_t kk = base + tp.st_off + s * slot, d = tmem + 128 * w;
                for (uint32_t k = 0; k < hdp / 16; ++k) {
                    const uint64_t db = tc_desc_sw(kk + (k >> 2) * TC_BLK + (k & 3) * 32u, 16u, 1024u);
                    tc_mma_ss(d, tc_desc(qa + qlo + 2 * k * QCH, QCH, 128u), db, idq, k > 0);
                    tc_mma_ss(d, tc_desc(qa + 2 * k * QCH, QCH, 128u), db, idq, true);
                }
                tc_commit(base + H_EMPTY + 8 * s);
                tc_commit(base + H_S + 8 * w);
                if (i >= 1) ok = pv(i - 1) && !*bad;
            }
            if (ok) ok = pv(nch - 1);
            if (!ok) *bad = 1;
            tc_commit(base + H_END);   // completes when every product issued here has
        }
        __syncwarp();
    } else if (warp < TC_SOFT / 32) {
        // ---------------- softmax: stream w, row = thread --------------------
        const uint32_t w = warp >> 2, wq = warp & 3, r = 32 * wq + lane;
        const bool active = wq < aw, on = r < nrows;
        const uint32_t rr = R0 + (on ? r : 0u), tok = rr / G, head = kvh * G + rr % G;
        const uint32_t sa = tmem + ((32u * wq) << 16) + 128 * w, oa = sa + 256;
        const float fac = reinterpret_cast<const float *>(smem + H_FAC)[r];
        const int32_t qp = tree_qpos(p, b, tok, nc);
        const float slope = p.slopes ? p.slopes[head] * TREE_LOG2E : 0.f, cap2 = p.cap * TREE_LOG2E;
        const uint32_t *mrow = p.mask ? p.mask + ((uint64_t)b * p.n_tokens + tok) * p.words : nullptr;
        const int32_t qmax = *reinterpret_cast<const int32_t *>(smem + H_QMAX);
        float *sc = p.scores ? p.scores + ((uint64_t)(b * p.nkh + kvh) * (p.n_tokens * G) + rr) * p.score_ld : nullptr;
        float mref = -INFINITY, l = 0.f;
        bool dead = false;
        if (active) {
            for (uint32_t i = w; i < nch; i += 2) {
                const uint32_t tb = t0 + i * TREE_TC_SP;
                const int nval = (int)min(TREE_TC_SP, t1 - tb);
                // every row of the tile sees all of its positions
                const bool whole = tb + TREE_TC_SP <= min(nc, t1) && !kpos && (!p.window || (int64_t)qmax - tb < (int64_t)p.window);
                dead = dead || !__all_sync(0xffffffffu, !*bad && waits(base + H_S + 8 * w, (i / 2) & 1u));
                if (dead) {   // a wait ran out: only the stream's barriers are kept company
                    if (!whole && bar_or(2 + w, 32 * aw, false) && bar_or(2 + w, 32 * aw, false)) bar_or(2 + w, 32 * aw, false);
                    continue;
                }
                tc_after();
                const bool plain = whole && !p.slopes && !(p.cap > 0.f);
                float mx = -INFINITY;
                uint32_t s[32];
                if (plain) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        tc_ld32(sa + 32 * c, s);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(s[e]));
                    }
                    mx *= fac;
                } else {
                    const int32_t *kp = reinterpret_cast<const int32_t *>(smem + TC_HDR) + (i % tp.ring) * TREE_TC_SP;
                    bool hidden = false;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        // visible positions of this row, bit e: tb + 32 c + e
                        const int d0 = (int)(tb + 32 * c) - (int)nc;   // drafted number of bit 0
                        const uint32_t inside = ones(nval - 32 * c);
                        uint32_t see = inside;
                        if (d0 > -32 && on) {
                            if (!mrow) {
                                see &= ones((int)tok - d0 + 1);
                            } else {
                                auto word = [&](int k) -> uint32_t { return k >= 0 && k < (int)p.words ? mrow[k] : 0u; };
                                const int sft = d0 & 31, k0 = (d0 - sft) / 32;   // floor
                                const uint32_t m = sft ? (word(k0) >> sft) | (word(k0 + 1) << (32 - sft)) : word(k0);
                                see &= m | ones(-d0);
                            }
                        }
                        tc_ld32(sa + 32 * c, s);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float x = __uint_as_float(s[e]) * fac;
                            if (p.cap > 0.f) x = tree_cap(x, cap2);
                            if (want_pos) {
                                const int32_t k = kp[32 * c + e];
                                const int64_t dist = (int64_t)qp - k;
                                if (kpos && k < 0) see &= ~(1u << e);
                                if (p.window && dist >= (int64_t)p.window) see &= ~(1u << e);
                                if (p.slopes) x -= slope * (float)dist;
                            }
                            if (!((see >> e) & 1u)) x = -INFINITY;
                            s[e] = __float_as_uint(x);
                            mx = fmaxf(mx, x);
                        }
                        hidden |= (on && (inside & ~see) != 0) || (nval & 15);   // or stale rows behind the end in the last product
                        tc_st32(sa + 32 * c, s);
                    }
                    tc_wait_st();
                    if (!whole && bar_or(2 + w, 32 * aw, hidden)) {
                        // values that some row does not see must be finite, or
                        // 0 * v would reach it
                        const uint32_t vs = (2 * i + 1) % tp.ns, va = base + tp.st_off + vs * slot;
                        const bool here = waits(base + H_FULL + 8 * vs, ((2 * i + 1) / tp.ns) & 1u);
                        bool odd = false;
                        for (uint32_t k = r; here && k < slot / 16; k += 32 * aw) {
                            const uint4 v = lds_u128(va + k * 16);
                            odd |= not_finite2(v.x) || not_finite2(v.y) || not_finite2(v.z) || not_finite2(v.w);
                        }
                        if (bar_or(2 + w, 32 * aw, odd)) {
                            // rare: the rows that see such values add them here,
                            // then they become zeros for the product
                            const float nm = mx > mref + TREE_LAZY ? mx - TREE_BELOW : mref;
                            const float bs = nm == -INFINITY ? 0.f : nm;
                            for (uint32_t c = 0; c < chunks; ++c) {
                                uint32_t o[8];
                                if (i >= 2) { tc_ld8(oa + 8 * c, o); tc_wait_ld(); }
                                else for (int k = 0; k < 8; ++k) o[k] = 0u;
                                for (int j = 0; j < nval; ++j) {
                                    const uint4 v = lds_u128(va + (c >> 3) * TC_BLK + j * 128 + (((c & 7) ^ (j & 7)) << 4));   // the same for all lanes
                                    if (!(not_finite2(v.x) || not_finite2(v.y) || not_finite2(v.z) || not_finite2(v.w))) continue;
                                    uint32_t xs;
                                    tc_ld1(sa + j, xs);
                                    tc_wait_ld();
                                    const float x = __uint_as_float(xs);
                                    const float pr = ex2(x - bs);
                                    const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
                                    for (int k = 0; k < 8; ++k) {
                                        const uint32_t h = (vv[k >> 1] >> (16 * (k & 1))) & 0xFFFFu;
                                        if ((h & 0x7C00u) == 0x7C00u && x != -INFINITY)
                                            o[k] = __float_as_uint(__uint_as_float(o[k]) + pr * f16f(h));
                                    }
                                }
                                tc_st8(oa + 8 * c, o);
                            }
                            tc_wait_st();
                            if (i < 2 && r == 0) reinterpret_cast<volatile int *>(smem + H_ACC)[w] = 1;
                            bar_or(2 + w, 32 * aw, false);
                            for (uint32_t k = r; k < slot / 16; k += 32 * aw) {
                                uint4 v = lds_u128(va + k * 16);
                                uint32_t vv[4] = {v.x, v.y, v.z, v.w};
                                for (int u = 0; u < 4; ++u) {
                                    if ((vv[u] & 0x7C00u) == 0x7C00u) vv[u] &= 0xFFFF0000u;
                                    if ((vv[u] & 0x7C000000u) == 0x7C000000u) vv[u] &= 0x0000FFFFu;
                                }
                                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(va + k * 16), "r"(vv[0]), "r"(vv[1]),
                                             "r"(vv[2]), "r"(vv[3]) : "memory");
                            }
                            tc_proxy();
                        }
                    }
                }
                // running reference; the accumulator follows when it moves
                const bool moves = mx > mref + TREE_LAZY;
                if (__any_sync(0xffffffffu, moves)) {
                    float f = 1.f;
                    if (moves) {
                        f = mref == -INFINITY ? 1.f : ex2(mref - (mx - TREE_BELOW));   // nothing seen before: nothing to scale
                        mref = mx - TREE_BELOW;
                        l *= f;
                    }
                    if (i >= 2) {
                        for (uint32_t c = 0; c < hdp; c += 8) {
                            uint32_t o[8];
                            tc_ld8(oa + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tc_st8(oa + c, o);
                        }
                    }
                }
                const float bs = mref == -INFINITY ? 0.f : mref, f = plain ? fac : 1.f;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    if (32 * c >= nval) break;   // behind the end: the products stop there too
                    tc_ld32(sa + 32 * c, s);
                    tc_wait_ld();
                    if (sc && on) {
                        float *d = sc + tb + 32 * c;
                        if (32 * c + 32 <= nval) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                *reinterpret_cast<float4 *>(d + e) = make_float4(__uint_as_float(s[e]) * f, __uint_as_float(s[e + 1]) * f,
                                                                                 __uint_as_float(s[e + 2]) * f, __uint_as_float(s[e + 3]) * f);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (32 * c + e < nval) d[e] = __uint_as_float(s[e]) * f;
                        }
                    }
                    uint32_t out[32];
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float p0 = ex2(fmaf(__uint_as_float(s[e]), f, -bs)), p1 = ex2(fmaf(__uint_as_float(s[e + 1]), f, -bs));
                        sum[(e >> 1) & 3] += p0 + p1;
                        const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u);
                        const float h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                        const __half2 hi = __floats2half2_rn(h0, h1), lo = __floats2half2_rn(p0 - h0, p1 - h1);
                        out[e >> 1] = *reinterpret_cast<const uint32_t *>(&hi);
                        out[16 + (e >> 1)] = *reinterpret_cast<const uint32_t *>(&lo);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tc_st32(sa + 32 * c, out);
                }
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(base + H_P + 8 * w);
            }
        }
        // ---------------- join of the two streams, and out -------------------
        const uint32_t streams = nch > 1 ? 2u : 1u;
        float2 *ml_sm = reinterpret_cast<float2 *>(smem + tp.q_off);   // over the queries, once all products are done
        const bool ok = __all_sync(0xffffffffu, waits(base + H_END, 0) && !*bad);
        tc_after();
        ml_sm[w * TREE_TC_ROWS + r] = make_float2(active ? mref : -INFINITY, active ? l : 0.f);
        named_bar_sync(4, TC_SOFT);
        if (active && ok) {
            const float2 a = ml_sm[r], c = streams > 1 ? ml_sm[TREE_TC_ROWS + r] : make_float2(-INFINITY, 0.f);
            const float M = fmaxf(a.x, c.x);
            const float f0 = a.x == -INFINITY ? 0.f : ex2(a.x - M), f1 = c.x == -INFINITY ? 0.f : ex2(c.x - M);
            const float L = a.y * f0 + c.y * f1;
            const bool many = p.n_splits > 1;
            const float il = many ? 1.f : (L == 0.f ? 0.f : 1.f / L);
            float *dst = many ? p.part_o + ((slot_id * p.n_splits + split) * TREE_TC_ROWS + r) * p.hd
                              : p.out + (((uint64_t)b * p.n_tokens + tok) * p.nqh + head) * p.hd;
            for (uint32_t c8 = w; c8 < p.hd / 8; c8 += 2) {
                uint32_t x[8], y[8];
                tc_ld8(tmem + ((32u * wq) << 16) + 256 + 8 * c8, x);
                if (streams > 1) tc_ld8(tmem + ((32u * wq) << 16) + 384 + 8 * c8, y);
                tc_wait_ld();
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    v[k] = __uint_as_float(x[k]) * f0;
                    if (streams > 1) v[k] = fmaf(__uint_as_float(y[k]), f1, v[k]);
                    v[k] = !many && L == 0.f ? 0.f : v[k] * il;
                }
                if (on) {
                    *reinterpret_cast<float4 *>(dst + 8 * c8) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4 *>(dst + 8 * c8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
            if (on && w == 0) {
                if (many) ml[r] = make_float2(M, L);
                else if (p.lse) p.lse[(uint64_t)(b * p.nkh + kvh) * (p.n_tokens * G) + rr] = L == 0.f ? -INFINITY : M + log2f(L);
            }
        }
        if (*bad && threadIdx.x == 0) dev_flag_error(p.err, DERR_TIMEOUT_FULL);
    }
    tc_before();
    __syncthreads();
    if (warp == TC_ISSUER) {
        if (lane == 0) mbar_wait_bounded(base + H_END, 0, kWaitNs);   // the tensor memory goes back after the last product
        __syncwarp();
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace

cudaError_t tree_tc_configure() {
    return cudaFuncSetAttribute(tree_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
}

cudaError_t tree_tc_launch(const TreeParams &t, const CUtensorMap &km, const CUtensorMap &vm, uint32_t n_seqs, cudaStream_t st) {
    TcParams p = {};
    p.t = t;
    p.km = km;
    p.vm = vm;
    p.hdp = (t.hd + 15) / 16 * 16;
    p.blks = (t.hd + 63) / 64;
    // as many stages as shared memory holds, 8 at most; a key-position tile
    // is overwritten `ring` tiles later, after the value tile of its own
    // position in the ring of stages was released
    for (p.ns = 8;; --p.ns) {
        p.ring = (p.ns + 1) / 2;
        p.q_off = TC_HDR + p.ring * TREE_TC_SP * 4;
        p.st_off = (p.q_off + 2 * p.hdp * 2 * TREE_TC_ROWS + 1023) / 1024 * 1024;   // the swizzle wants whole 1024 bytes
        if (p.st_off + p.ns * p.blks * TC_BLK <= 232448) break;
    }
    const dim3 grid(t.nkh * t.row_tiles, t.n_splits, n_seqs);
    tree_tc_kernel<<<grid, TC_THREADS, p.st_off + p.ns * p.blks * TC_BLK, st>>>(p);
    return cudaGetLastError();
}

}  // namespace vbs
