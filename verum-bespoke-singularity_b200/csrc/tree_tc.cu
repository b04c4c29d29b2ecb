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
// the two are joined at the end. Or 256 rows, 128 a stream, that share the
// tiles: half the bytes of K and V, twice the time of a tile.
//  * One thread stages K and V tiles (32 KB each at head_dim 128) into a ring
//    with TMA, 64 dims x 128 positions a box, rows of 128 bytes with the
//    128-byte swizzle. The image is a K-major operand for Q K^T (MN =
//    position, K = dim) and an MN-major one for P V (MN = dim, K = position).
//    (Staged with cp.async by 4 warps in the layout without swizzle, a tile
//    took 2100 cycles to issue and was the bottleneck: 82.6 us for 504 rows x
//    8192 positions x 8 KV heads of 128.)
//  * One thread issues tcgen05.mma: S = Qhi K^T + Qlo K^T (both operands in
//    shared memory), O += Phi V + Plo V (P from tensor memory).
//  * 2 x 4 softmax warps, a thread per row: the scores are read once for the
//    maximum, and again for the weights, which go back over them as fp16
//    halves (columns 32 c .. + 15 the high, + 16 .. + 31 the low halves of
//    positions 32 c ..) and are announced 64 positions at a time. The sums are
//    rescaled when the maximum moves by more than TREE_LAZY. A load from tensor
//    memory answers after some 250 cycles while products run, so 32 or 64
//    columns go at a time (16 each: 504 rows x 8192 positions 57.3 us, then 53.3).
//  * The tensor cores cut accumulators instead of rounding them, towards zero:
//    left in tensor memory over 30 tiles a result lost 8.5e-6 (zero-mean
//    values; 1.5e-5 and more with values of one sign). So an accumulator lives
//    for one tile, the rows' threads add it to their fp32 sums in registers
//    (setmaxnreg gives them 232, but the compiler counts with the launch's 168
//    and spills 352 bytes), and a score's low halves go first, while its
//    accumulator is small.
// All waits are bounded; after one ran out the CTA flags the device error
// word, waits for its copies and products, frees its tensor memory and ends.
#include "tree_tc.cuh"

#include <algorithm>

namespace vbs {

namespace {

constexpr int TC_SOFT = 256, TC_THREADS = TC_SOFT + 128;   // softmax warps; the loader, the issuers of Q K^T and of P V, one idle
constexpr int TC_LOADER = TC_SOFT / 32, TC_QK = TC_LOADER + 1, TC_PV = TC_LOADER + 2;
// registers: 384 x 168 at the launch = 256 x 232 + 128 x 40 (64,512 each)
constexpr int TC_REGS_SOFT = 232, TC_REGS_OTHER = 40;
static_assert(TC_SOFT * TC_REGS_SOFT + (TC_THREADS - TC_SOFT) * TC_REGS_OTHER <= TC_THREADS * 168, "more than launched waits forever");
constexpr uint32_t TC_PITCH = 128 * 4 + 16;   // bytes of a row of sums in shared memory: conflict-free for a thread per row
constexpr uint32_t TC_BLK = TREE_TC_SP * 128u;   // one box: 128 positions x 64 dims

// words of the state behind the queries (bytes); barriers first
constexpr uint32_t H_FULL = 0, H_EMPTY = 64, H_S = 128, H_P = 144, H_O = 176, H_END = 192, H_TMEM = 200, H_BAD = 204, H_ACC = 208,
                   H_QMAX = 216;
constexpr uint32_t H_FAC = 256, H_BYTES = H_FAC + 1024;   // then the rows' score factors

struct TcParams {
    TreeParams t;
    CUtensorMap km, vm;
    uint32_t dual;   // row tiles of 256, 128 rows a stream
    uint32_t ns, hdp, blks, q_off, h_off;   // stages, padded head_dim, boxes per tile, offsets of the queries and the state
};

__global__ void __launch_bounds__(TC_THREADS, 1) tree_tc_kernel(const __grid_constant__ TcParams tp) {
    const TreeParams &p = tp.t;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *const hs = smem + tp.h_off;
    const uint32_t stage0 = smem_u32(smem), base = stage0 + tp.h_off;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t kvh = blockIdx.x % p.nkh, tile = blockIdx.x / p.nkh, split = blockIdx.y, b = blockIdx.z;
    const uint32_t TR = TREE_TC_ROWS << tp.dual, R0 = tile * TR;
    const uint32_t hdp = tp.hdp, chunks = hdp / 8, slot = tp.blks * TC_BLK, q_bytes = 2 * hdp * 2 * TREE_TC_ROWS;
    volatile int *bad = reinterpret_cast<volatile int *>(hs + H_BAD);
    float *fac_sm = reinterpret_cast<float *>(hs + H_FAC);

    // the queries start on their way before anything else is known
    TcQ<128> q;
    if (warp < TC_LOADER) tc_q_load(p, R0 + 16 * warp + (lane & 7), p.n_tokens * p.G, kvh, b, q);   // (rows behind n_tok too: their scores are nobody's)
    if (warp == TC_LOADER && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tp.km) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tp.vm) : "memory");
        for (uint32_t s = 0; s < tp.ns; ++s) {
            mbar_init(base + H_FULL + 8 * s, 1);
            mbar_init(base + H_EMPTY + 8 * s, 1);
        }
        for (uint32_t w = 0; w < 2; ++w) {
            mbar_init(base + H_S + 8 * w, 1);
            mbar_init(base + H_O + 8 * w, 1);
        }
        mbar_init(base + H_END, 2);
        *bad = 0;
        reinterpret_cast<int *>(hs + H_ACC)[0] = reinterpret_cast<int *>(hs + H_ACC)[1] = 0;
        mbar_fence_init();
    }
    pdl_launch_dependents();
    uint32_t nc, nt;
    if (!tree_lengths(p, b, nc, nt) || R0 >= nt * p.G) return;
    const uint32_t end = nc + nt, nrows = min(TR, nt * p.G - R0);
    const uint32_t first = tree_first(p, b, nc, nt, reinterpret_cast<int32_t *>(hs + H_FAC));
    uint32_t t0, t1;
    tree_part(p, first, end, split, t0, t1);
    const uint64_t slot_id = (uint64_t)(b * p.nkh + kvh) * p.row_tiles + tile;
    float2 *ml = p.part_ml + (slot_id * p.n_splits + split) * TR;
    const uint32_t two = tp.dual && nrows > TREE_TC_ROWS;
    // parts joined in a cluster: (m, l) and sums of the rows here, behind what
    // the streams' own join uses (all products are done by then)
    const uint32_t jm = two ? 0u : 2 * TREE_TC_ROWS * 8 + TREE_TC_ROWS * TC_PITCH, jo = jm + 2 * TREE_TC_ROWS * 8, jp = p.hd * 4 + 16;
    float2 *const jml = reinterpret_cast<float2 *>(smem + jm);
    if (t0 >= t1 && p.n_splits > 1) {
        for (uint32_t r = threadIdx.x; r < TR; r += TC_THREADS) (p.joined ? jml : ml)[r] = make_float2(-INFINITY, 0.f);
        if (p.joined) {
            cluster_meet();
            if (threadIdx.x < TC_SOFT) tree_join(p, stage0 + jm, stage0 + jo, jp, nrows, R0, kvh, b, split, threadIdx.x, TC_SOFT);
            cluster_meet();
        }
        return;
    }
    // step n: position tile n (dual: n / 2) for stream n % 2, the stream's
    // (n / 2)th; the streams share the rows and alternate tiles, or (dual)
    // have 128 rows each and share the tiles
    const uint32_t nch = (t1 - t0 + TREE_TC_SP - 1) / TREE_TC_SP;
    const uint32_t steps = two ? 2 * nch : nch;
    const uint32_t aw0 = (min(nrows, TREE_TC_ROWS) + 31) / 32, aw1 = two ? (nrows - TREE_TC_ROWS + 31) / 32 : aw0;   // 32s of rows
    auto waits = [&](uint32_t bar, uint32_t parity) -> bool {
        if (mbar_wait_bounded(bar, parity, kWaitNs)) return true;
        *bad = 1;
        return false;
    };
    auto all = [&](bool x) { return __all_sync(0xffffffffu, x); };
    // ---------------- loader: items K0 V0 K1 V1 ... ------------------------
    // (stages and phases are counted along: a division would cost an issuer more than a wait)
    auto load = [&](uint32_t it, uint32_t s) {
        const uint32_t tb = t0 + it / 2 * TREE_TC_SP;
        if (lane == 0) {
            mbar_arrive_expect_tx(base + H_FULL + 8 * s, slot);
            for (uint32_t k = 0; k < tp.blks; ++k)
                tree_tma(stage0 + s * slot + k * TC_BLK, (it & 1) ? &tp.vm : &tp.km, 64 * k, tb, kvh, b, base + H_FULL + 8 * s);
        }
        __syncwarp();
    };
    uint32_t it = 0;
    if (warp == TC_LOADER) {
        load(it++, 0);   // the first keys are needed first; the rest follows behind the barrier
        if (lane == 0) {
            for (uint32_t w = 0; w < 2; ++w) {
                mbar_init(base + H_P + 16 * w, w ? aw1 : aw0);       // weights of the tile's first 64 positions
                mbar_init(base + H_P + 16 * w + 8, w ? aw1 : aw0);   // and of the others
            }
            mbar_fence_init();
        }
        __syncwarp();
    } else if (warp == TC_QK) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + H_TMEM), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp == TC_PV) {
        int32_t hi = (int32_t)0x80000000;   // highest query position of the rows, for the tiles inside everybody's window
        if (p.window)
            for (uint32_t r = lane; r < nrows; r += 32) hi = max(hi, tree_qpos(p, b, tree_token(p, R0 + r), nc));
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) *reinterpret_cast<int32_t *>(hs + H_QMAX) = hi;
    } else if (warp < TC_LOADER) {
        // 8 rows at a time, two times 8 per warp and 128 rows; places of rows
        // that are not there keep what they hold (nobody reads their scores)
#pragma unroll 1
        for (uint32_t g = 0; g < (two ? 4u : 2u); ++g) {
            const uint32_t r0 = 16 * warp + 8 * (g & 1), x = g >> 1, n0 = TREE_TC_ROWS * ((g + 1) >> 1) + 16 * warp + 8 * ((g + 1) & 1);
            if (x * TREE_TC_ROWS + r0 >= nrows) break;
            TcQ<128> next;
            if (n0 < nrows) tc_q_load(p, R0 + n0 + (lane & 7), p.n_tokens * p.G, kvh, b, next);
            const float f = tc_q_store(p, q, smem + tp.q_off + x * q_bytes, TREE_TC_ROWS * 16, q_bytes / 2, r0 + (lane & 7), chunks);
            if (lane < 8) fac_sm[x * TREE_TC_ROWS + r0 + lane] = f;
            q = next;
        }
        tc_proxy();
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *reinterpret_cast<uint32_t *>(hs + H_TMEM);
    // the warpgroup of the loader and the issuers gives its registers away
    if (warp >= TC_LOADER) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_REGS_OTHER));
    if (warp == TC_LOADER) {
        for (uint32_t s = 1, ph = 1; it < 2 * nch; ++it) {   // ph: parity of the last time round
            if (!all(!*bad && (it < tp.ns || waits(base + H_EMPTY + 8 * s, ph)))) break;
            load(it, s);
            if (++s == tp.ns) { s = 0; ph ^= 1u; }
        }
        // after a failed wait copies may still be landing: the newest of
        // every slot is waited for before the CTA ends
        if (*bad && lane == 0)
            for (uint32_t k = it > tp.ns ? it - tp.ns : 0; k < it; ++k)
                mbar_wait_bounded(base + H_FULL + 8 * (k % tp.ns), (k / tp.ns) & 1u, kWaitNs);
        __syncwarp();
    } else if (warp == TC_QK) {
        // ---------------- S = Qhi K^T + Qlo K^T ------------------------------
        // (the two issuers wait apart from one another, so the tensor core
        // has the one's products while the other waits)
        const uint32_t idq = (1u << 4) | ((TREE_TC_SP >> 3) << 17) | ((TREE_TC_ROWS >> 4) << 24);
        constexpr uint32_t QCH = TREE_TC_ROWS * 16u;   // bytes per chunk of the queries
        const uint64_t dq0 = tc_desc(stage0 + tp.q_off, QCH, 128u), dk = tc_desc_sw(stage0, 16u, 1024u);
        const uint32_t qlo = q_bytes / 32, lead = tc_elect();   // the low halves' offset, in descriptor units
        for (uint32_t n = 0, s = 0, ph = 0; n < steps; ++n) {
            const uint32_t w = n & 1;
            // this stream's last weights used up, and then the keys here. In
            // this order: with an odd number of stages an issuer meets every
            // other phase of a stage, and a parity tells neighbours apart. The
            // phase between, values of a tile before, is over once that tile's
            // second product is; asked earlier, three stages can still be
            // waiting for those values, and they pass for these keys.
            if (!all(!*bad && (n < 2 || waits(base + H_O + 8 * w, (n / 2 - 1) & 1u)) && waits(base + H_FULL + 8 * s, ph))) break;
            tc_after();
            const uint64_t d = dk + s * (slot / 16), dq = dq0 + (two && w ? q_bytes / 16 : 0u);
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                if (k >= hdp / 16) break;
                tc_mma_ss(tmem + 128 * w, dq + qlo + 2 * k * (QCH / 16), d + (k >> 2) * (TC_BLK / 16) + (k & 3) * 2, idq, k ? 1u : 0u, lead);
            }
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                if (k >= hdp / 16) break;
                tc_mma_ss(tmem + 128 * w, dq + 2 * k * (QCH / 16), d + (k >> 2) * (TC_BLK / 16) + (k & 3) * 2, idq, 1u, lead);
            }
            if (lead) {
                tc_commit(base + H_S + 8 * w);
                if (!two || w) tc_commit(base + H_EMPTY + 8 * s);
            }
            __syncwarp();
            if (!two || w) {   // on to the next tile's keys, two stages further
                s += 2;
                if (s >= tp.ns) { s -= tp.ns; ph ^= 1u; }
            }
        }
        if (lead) tc_commit(base + H_END);   // with the other issuer's: every product has completed
        __syncwarp();
    } else if (warp == TC_PV) {
        // ---------------- O += Phi V + Plo V ---------------------------------
        const uint32_t idp = (1u << 4) | (1u << 16) | ((hdp >> 3) << 17) | ((TREE_TC_ROWS >> 4) << 24);
        const uint64_t dv = tc_desc_sw(stage0, TC_BLK, 1024u);
        const uint32_t lead = tc_elect();
        bool ok = true;
        for (uint32_t n = 0, s = 1, ph = 0; ok && n < steps; ++n) {
            const uint32_t w = n & 1, i = two ? n >> 1 : n;
            if (!all(!*bad && waits(base + H_FULL + 8 * s, ph) && waits(base + H_P + 16 * w, (n >> 1) & 1u))) break;
            tc_after();
            const uint64_t d = dv + s * (slot / 16);
            const uint32_t o = tmem + 256 + 128 * w, pa = tmem + 128 * w;
            // every tile its own accumulator, unless the softmax put something there itself
            const uint32_t acc0 = reinterpret_cast<volatile uint32_t *>(hs + H_ACC)[w];
            const uint32_t ks = (min(TREE_TC_SP, t1 - t0 - i * TREE_TC_SP) + 15) / 16;
#pragma unroll
            for (uint32_t k = 0; k < TREE_TC_SP / 16; ++k) {
                if (k == 4) {   // the second half's weights (announced in any case)
                    ok = all(waits(base + H_P + 16 * w + 8, (n >> 1) & 1u));
                    tc_after();
                }
                if (k >= ks || !ok) break;
                tc_mma_ts(o, pa + 32 * (k >> 1) + 8 * (k & 1) + 16, d + k * 128, idp, k ? 1u : acc0, lead);
                tc_mma_ts(o, pa + 32 * (k >> 1) + 8 * (k & 1), d + k * 128, idp, 1u, lead);
            }
            if (lead) {
                tc_commit(base + H_O + 8 * w);
                if (!two || w) tc_commit(base + H_EMPTY + 8 * s);
            }
            __syncwarp();
            if (!two || w) {
                s += 2;
                if (s >= tp.ns) { s -= tp.ns; ph ^= 1u; }
            }
        }
        if (lead) tc_commit(base + H_END);
        __syncwarp();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_REGS_SOFT));
        // ---------------- softmax: stream w, row = thread --------------------
        const uint32_t w = warp >> 2, wq = warp & 3, r = 32 * wq + lane;
        const uint32_t ri = two && w ? TREE_TC_ROWS + r : r;   // row of the tile
        const uint32_t aw = w ? aw1 : aw0;
        const bool active = wq < aw, on = ri < nrows;
        const uint32_t rr = R0 + (on ? ri : 0u), tok = tree_token(p, rr), head = kvh * p.G + (rr - tok * p.G);
        const uint32_t sa = tmem + ((32u * wq) << 16) + 128 * w, oa = sa + 256;
        const float fac = on ? fac_sm[ri] : 0.f;
        const int32_t qp = tree_qpos(p, b, tok, nc), qmax = *reinterpret_cast<const int32_t *>(hs + H_QMAX);
        const float slope = p.slopes ? p.slopes[head] * TREE_LOG2E : 0.f;
        const int32_t *kpos = p.k_pos ? p.k_pos + (uint64_t)(p.k_pos_per_head ? b * p.nkh + kvh : b) * p.max_ctx : nullptr;
        float mref = -INFINITY;
        float o[128];   // the row's sums
#pragma unroll
        for (int k = 0; k < 128; ++k) o[k] = 0.f;
        auto gather = [&]() {   // the tile's accumulator into the sums
            // 64 columns a time: a load answers after some 250 cycles while products run
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (64 * c >= (int)hdp) break;
                uint32_t x[2][32];
                tc_ld32(oa + 64 * c, x[0]);
                tc_ld32(oa + 64 * c + 32, x[1]);   // (behind hdp: columns of its own that nobody uses)
                tc_wait_ld(x[0]);
                tc_wait_ld(x[1]);
#pragma unroll
                for (int k = 0; k < 32; ++k) { o[64 * c + k] += __uint_as_float(x[0][k]); o[64 * c + 32 + k] += __uint_as_float(x[1][k]); }
            }
        };
        float2 l = make_float2(0.f, 0.f);
        bool dead = false;
        // the threads that look at one tile's values together: a stream, or
        // both where they share the tiles
        const uint32_t bar = two ? 2 : 2 + w, bar_n = 32 * (two ? aw0 + aw1 : aw), bar_r = r + (two && w ? 32 * aw0 : 0u);
        // the lane's key positions of the next tile
        const uint32_t tstep = two ? TREE_TC_SP : 2 * TREE_TC_SP;
        uint32_t tn = t0 + (two ? 0u : w * TREE_TC_SP);
        int32_t kn[4] = {0, 0, 0, 0};
        if (kpos && active && tn + TREE_TC_SP <= min(nc, t1)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) kn[k] = kpos[tn + 32 * k + lane];
        }
        tn += tstep;
        for (uint32_t n = active ? w : steps; n < steps; n += 2) {
            const uint32_t i = two ? n >> 1 : n, tb = t0 + i * TREE_TC_SP;
            const int nval = (int)min(TREE_TC_SP, t1 - tb);
            // every row of the tile sees all of its positions: by the lowest
            // key position of the tile, negative for a hole
            int32_t low = (int32_t)tb;
            const bool context = tb + TREE_TC_SP <= min(nc, t1);
            if (kpos && context) {
                low = min(min(kn[0], kn[1]), min(kn[2], kn[3]));
                low = __reduce_min_sync(0xffffffffu, low);
            }
            // the tile's key positions where they are not its slots, lane: 32 k + lane
            const bool by_slot = !kpos && tb + TREE_TC_SP <= nc;
            int32_t kc[4] = {kn[0], kn[1], kn[2], kn[3]};
            if (!by_slot && !context && (kpos || p.window || p.slopes)) {
#pragma unroll
                for (int k = 0; k < 4; ++k) kc[k] = 32 * k + lane < nval ? tree_kpos(p, kpos, b, tb + 32 * k + lane, nc) : 0;
            }
            if (kpos && tn + TREE_TC_SP <= nc) {   // the next tile's, ahead
#pragma unroll
                for (int k = 0; k < 4; ++k) kn[k] = kpos[tn + 32 * k + lane];
            }
            tn += tstep;
            const bool whole = context && low >= 0 && (!p.window || qmax - low < (int32_t)p.window);
            // a tile with drafted positions: this row's mask words, before the wait
            const int m0 = (int)((int64_t)tb - nc) >> 5;   // word of the tile's first position (may be negative)
            uint32_t mk[5] = {0u, 0u, 0u, 0u, 0u};
            if (p.mask && on && tb + TREE_TC_SP > nc) {
                const uint32_t *mrow = p.mask + ((uint64_t)b * p.n_tokens + tok) * p.words;
#pragma unroll
                for (int k = 0; k < 5; ++k) mk[k] = m0 + k >= 0 && m0 + k < (int)p.words ? mrow[m0 + k] : 0u;
            }
            // the last tile's accumulator, beside the product of this tile's scores
            if (n >= 2) {
                dead = dead || !all(!*bad && waits(base + H_O + 8 * w, ((n >> 1) - 1) & 1u));
                if (!dead) {
                    tc_after();
                    gather();
                }
            }
            dead = dead || !all(!*bad && waits(base + H_S + 8 * w, (n >> 1) & 1u));
            if (dead) {   // a wait ran out: only the barriers are kept company
                if (!whole && bar_or(bar, bar_n, false) && bar_or(bar, bar_n, false))
                    for (int k = 0; k < 2; ++k) bar_or(bar, bar_n, false);
                continue;
            }
            tc_after();
            if (r == 0) reinterpret_cast<volatile uint32_t *>(hs + H_ACC)[w] = 0;
            // plain: the scores as the product left them; the row's factor goes with the reference
            const bool turned = p.slopes || p.cap > 0.f, plain = whole && !turned;
            const float cap2 = p.cap * TREE_LOG2E;
            float mx = -INFINITY;
            if (plain) {
                uint32_t s[2][32];
                tc_ld32(sa, s[0]);
                tc_wait_ld(s[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c < 3) tc_ld32(sa + 32 * (c + 1), s[(c + 1) & 1]);
                    mx = fmaxf(mx, max32(s[c & 1]));
                    if (c < 3) tc_wait_ld(s[(c + 1) & 1]);
                }
            } else if (turned) {
                // capped, with slope * (key position - query position) added,
                // back into tensor memory
                const bool linear = p.slopes && by_slot;
#pragma unroll 1
                for (int c = 0; c < 8; ++c) {
                    uint32_t s[16];
                    tc_ld16(sa + 16 * c, s);
                    tc_wait_ld(s);
                    float x[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(s[e]) * fac;
                    if (p.cap > 0.f) tree_cap_all(x, cap2);
                    if (linear) {
                        const float d = (float)((int32_t)tb + 16 * c - qp);
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = fmaf(slope, d + (float)e, x[e]);
                    } else if (p.slopes) {
                        const int32_t kp = c < 4 ? (c < 2 ? kc[0] : kc[1]) : (c < 6 ? kc[2] : kc[3]);
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            x[e] = fmaf(slope, (float)(__shfl_sync(0xffffffffu, kp, 16 * (c & 1) + e) - qp), x[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 2) mx = max3(mx, x[e], x[e + 1]);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __float_as_uint(x[e]);
                    tc_st16(sa + 16 * c, s);
                }
                tc_wait_st();
            }
            if (!whole) {
                // what the row does not see becomes -inf, 32 positions at a time
                bool hidden = (nval & 15) != 0;   // stale rows behind the end in the last product
                const float fm = turned ? 1.f : fac;
                mx = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t x[32];
                    tc_ld32(sa + 32 * c, x);
                    const int32_t t = (int32_t)(tb + 32 * c), d0 = t - (int)nc;   // drafted number of bit 0
                    const uint32_t inside = ones(nval - 32 * c);
                    uint32_t see = inside;   // bit e: this row sees position t + e
                    if (d0 > -32 && on) {
                        if (!p.mask) {
                            see &= ones((int)tok - d0 + 1);
                        } else {
                            const uint32_t lo = c == 0 ? mk[0] : c == 1 ? mk[1] : c == 2 ? mk[2] : mk[3];
                            const uint32_t hi = c == 0 ? mk[1] : c == 1 ? mk[2] : c == 2 ? mk[3] : mk[4];
                            see &= __funnelshift_r(lo, hi, d0 & 31) | ones(-d0);
                        }
                    }
                    if (by_slot) {
                        if (p.window && qp >= (int32_t)p.window) see &= ~ones(qp - (int32_t)p.window + 1 - t);   // (slots are 0 or more)
                    } else {
                        const int32_t kp = c == 0 ? kc[0] : c == 1 ? kc[1] : c == 2 ? kc[2] : kc[3];
                        if (kpos) see &= __ballot_sync(0xffffffffu, kp >= 0);
                        if (p.window) {
#pragma unroll 4
                            for (int e = 0; e < 32; ++e)
                                if (qp - __shfl_sync(0xffffffffu, kp, e) >= (int32_t)p.window) see &= ~(1u << e);
                        }
                    }
                    hidden |= on && see != inside;
                    __syncwarp();
                    tc_wait_ld(x);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float v = (see >> e) & 1u ? __uint_as_float(x[e]) * fm : -INFINITY;
                        mx = fmaxf(mx, v);
                        x[e] = __float_as_uint(v);
                    }
                    tc_st32(sa + 32 * c, x);
                }
                tc_wait_st();
                if (bar_or(bar, bar_n, hidden)) {
                    // values that some row does not see must be finite, or
                    // 0 * v would reach it
                    const uint32_t vx = 2 * i + 1, va = stage0 + (vx % tp.ns) * slot;
                    const bool here = waits(base + H_FULL + 8 * (vx % tp.ns), (vx / tp.ns) & 1u);
                    bool odd = false;
                    if (here) {
                        uint32_t zero = 0;
#pragma unroll 8
                        for (uint32_t k = bar_r; k < slot / 16; k += bar_n) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(smem + (vx % tp.ns) * slot + k * 16);
                            zero = finite4(v, zero);
                        }
                        odd = zero != 0u;
                    }
                    if (bar_or(bar, bar_n, odd)) {
                        // rare: the rows that see such values put their part into
                        // the accumulator, then they become zeros for the product
                        const float nm = mx - mref > TREE_LAZY ? mx - TREE_BELOW : mref;
                        const float bs = nm == -INFINITY ? 0.f : nm;
                        for (uint32_t c = 0; c < chunks; ++c) {
                            uint32_t y[8];
                            for (int k = 0; k < 8; ++k) y[k] = 0u;
                            for (int j = 0; j < nval; ++j) {
                                const uint4 v = lds_u128(va + (c >> 3) * TC_BLK + j * 128 + (((c & 7) ^ (j & 7)) << 4));   // the same for all lanes
                                if (!(not_finite2(v.x) || not_finite2(v.y) || not_finite2(v.z) || not_finite2(v.w))) continue;
                                uint32_t xs;
                                tc_ld1(sa + j, xs);
                                tc_wait_ld(xs);
                                const float x = __uint_as_float(xs);
                                const float pr = ex2(x - bs);
                                const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
                                for (int k = 0; k < 8; ++k) {
                                    const uint32_t h = (vv[k >> 1] >> (16 * (k & 1))) & 0xFFFFu;
                                    if ((h & 0x7C00u) == 0x7C00u && x != -INFINITY)
                                        y[k] = __float_as_uint(__uint_as_float(y[k]) + pr * f16f(h));
                                }
                                __syncwarp();
                            }
                            tc_st8(oa + 8 * c, y);
                        }
                        tc_wait_st();
                        if (r == 0) reinterpret_cast<volatile uint32_t *>(hs + H_ACC)[w] = 1;
                        bar_or(bar, bar_n, false);   // all have read them
                        for (uint32_t k = bar_r; k < slot / 16; k += bar_n) {
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
                        bar_or(bar, bar_n, false);   // and all have written
                    }
                }
            }
            // running reference; the sums follow when it moves
            // (the largest weight's exponent, rounded as the weights' are)
            const float f1 = plain ? fac : 1.f;
            const bool moves = fmaf(mx, f1, -mref) > TREE_LAZY;
            if (__any_sync(0xffffffffu, moves)) {
                const float to = fmaf(mx, f1, -TREE_BELOW), f = !moves ? 1.f : ex2(mref - to);   // 0 on the first tile
                if (moves) mref = to;
                l.x *= f;
                l.y *= f;
#pragma unroll
                for (int k = 0; k < 128; ++k) o[k] *= f;
            }
            const float b1 = mref == -INFINITY ? 0.f : mref;
            const float2 f = make_float2(f1, f1), bs = make_float2(-b1, -b1);
            uint32_t s[2][32];
            tc_ld32(sa, s[0]);
            tc_wait_ld(s[0]);
            // 32 positions at a time, the next 32 on their way (they are read
            // before these halves go over them); behind the end: zeros
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (c < 3) tc_ld32(sa + 32 * (c + 1), s[(c + 1) & 1]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t hw[8], lw[8];
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float2 x = fma2(make_float2(__uint_as_float(s[c & 1][16 * u + e]), __uint_as_float(s[c & 1][16 * u + e + 1])), f, bs);
                        const float2 pr = make_float2(ex2(x.x), ex2(x.y));
                        l = add2(l, pr);
                        halves(pr, hw[e >> 1], lw[e >> 1]);
                    }
                    if (c < 3 && u) tc_wait_ld(s[(c + 1) & 1]);
                    tc_st8(sa + 32 * c + 8 * u, hw);
                    tc_st8(sa + 32 * c + 8 * u + 16, lw);
                }
                if (c & 1) {   // 64 positions done
                    tc_wait_st();
                    tc_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(base + H_P + 16 * w + 8 * (c >> 1));
                }
            }
        }
        // ---------------- out --------------------------------------------------
        const bool ok = all(waits(base + H_END, 0) && !*bad);
        tc_after();
        if (active && ok && w < steps) gather();
        float L = l.x + l.y, M = mref;
        const bool join = !two && nch > 1;   // the two streams had the same rows: each ends half of the dims
        const uint32_t half = join ? (p.hd / 8 + 1) / 2 * 8 : 0u;   // stream 0: below
        if (join) {
            float2 *ml_sm = reinterpret_cast<float2 *>(smem);   // over the stages: all products are done
            float *rows_sm = reinterpret_cast<float *>(smem + 2 * TREE_TC_ROWS * 8 + r * TC_PITCH);
            ml_sm[w * TREE_TC_ROWS + r] = make_float2(active ? M : -INFINITY, active ? L : 0.f);
#pragma unroll
            for (int c = 0; c < 128; c += 8) {   // the other stream's half goes over
                if (c >= (int)p.hd || (w == 0) == (c < (int)half)) continue;
                *reinterpret_cast<float4 *>(rows_sm + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                *reinterpret_cast<float4 *>(rows_sm + c + 4) = make_float4(o[c + 4], o[c + 5], o[c + 6], o[c + 7]);
            }
            named_bar_sync(4, TC_SOFT);
            const float2 a = ml_sm[w * TREE_TC_ROWS + r], c = ml_sm[(w ^ 1) * TREE_TC_ROWS + r];
            M = fmaxf(a.x, c.x);
            const float f0 = a.x == -INFINITY ? 0.f : ex2(a.x - M), f1 = c.x == -INFINITY ? 0.f : ex2(c.x - M);
            L = a.y * f0 + c.y * f1;
#pragma unroll
            for (int d = 0; d < 128; d += 4) {
                if (d >= (int)p.hd || (w == 0) != (d < (int)half)) continue;
                const float4 x = *reinterpret_cast<const float4 *>(rows_sm + d);
                o[d] = fmaf(x.x, f1, o[d] * f0);
                o[d + 1] = fmaf(x.y, f1, o[d + 1] * f0);
                o[d + 2] = fmaf(x.z, f1, o[d + 2] * f0);
                o[d + 3] = fmaf(x.w, f1, o[d + 3] * f0);
            }
        }
        if (active && ok && on && (two || join || w == 0)) {
            const bool many = p.n_splits > 1;
            const float il = many ? 1.f : (L == 0.f ? 0.f : 1.f / L);
            float *dst = p.joined ? reinterpret_cast<float *>(smem + jo + ri * jp)
                         : many   ? p.part_o + ((slot_id * p.n_splits + split) * TR + ri) * p.hd
                                  : p.out + (((uint64_t)b * p.n_tokens + tok) * p.nqh + head) * p.hd;
            const bool wide = !p.joined && (reinterpret_cast<uintptr_t>(dst) & 31) == 0;
            // straight from the rows' threads, a whole 32-byte sector each
#pragma unroll
            for (int c = 0; c < 128; c += 8) {
                if (c >= (int)p.hd || (join && (w == 0) != (c < (int)half))) continue;
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = !many && L == 0.f ? 0.f : o[c + k] * il;
                if (wide) {
                    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + c), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                                 "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
                } else {
                    *reinterpret_cast<float4 *>(dst + c) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4 *>(dst + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
            if (two || w == 0) {
                if (many) (p.joined ? jml : ml)[ri] = make_float2(M, L);
                else if (p.lse) p.lse[(uint64_t)(b * p.nkh + kvh) * (p.n_tokens * p.G) + rr] = L == 0.f ? -INFINITY : M + log2f(L);
            }
        }
        if (*bad && threadIdx.x == 0) dev_flag_error(p.err, DERR_TIMEOUT_FULL);
        if (p.joined) {
            cluster_meet();
            tree_join(p, stage0 + jm, stage0 + jo, jp, nrows, R0, kvh, b, split, threadIdx.x, TC_SOFT);
            cluster_meet();
        }
    }
    if (warp >= TC_LOADER && p.joined) {
        cluster_meet();
        cluster_meet();
    }
    tc_before();
    __syncthreads();
    if (warp == TC_QK) {
        if (lane == 0) mbar_wait_bounded(base + H_END, 0, kWaitNs);   // the tensor memory goes back after the last product
        __syncwarp();
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace

cudaError_t tree_tc_configure(int *clusters) {
    const cudaError_t e = cudaFuncSetAttribute(tree_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    return e == cudaSuccess ? tree_clusters(tree_tc_kernel, TC_THREADS, 232448, clusters) : e;
}

cudaError_t tree_tc_launch(const TreeParams &t, const CUtensorMap &km, const CUtensorMap &vm, uint32_t n_seqs, uint32_t dual,
                           cudaStream_t st) {
    TcParams p = {};
    p.t = t;
    p.km = km;
    p.vm = vm;
    p.hdp = (t.hd + 15) / 16 * 16;
    p.blks = (t.hd + 63) / 64;
    p.dual = dual;
    // stages (the swizzle wants whole 1024 bytes), queries, state: as many
    // stages as shared memory holds, 8 at most. hd 128: 5, dual 3.
    const uint32_t q_bytes = 2 * p.hdp * 2 * TREE_TC_ROWS << dual;
    p.ns = std::min(8u, (232448u - q_bytes - H_BYTES) / (p.blks * TC_BLK));
    p.q_off = p.ns * p.blks * TC_BLK;
    p.h_off = p.q_off + q_bytes;
    const dim3 grid(t.nkh * t.row_tiles, t.n_splits, n_seqs);
    return tree_launch(tree_tc_kernel, grid, TC_THREADS, p.h_off + H_BYTES, t.joined, st, p);
}

}  // namespace vbs
