// tree.cu -- attention of new tokens (a tree or chain of drafts, a chunk, one
// token) over a cache whose slots are not positions.
//
//   x_rt = scale q_r . K_t;  capped: c tanh(x / c);  + slope_r (kpos_t - qpos_r)
//   out_r = sum_t p_rt V_t,  p_rt = softmax over the visible t
//   (the weights W_t, sums over the rows of p_rt: tree_wt.cu)
//
// Rows: the n_tok tokens x G query heads of one KV head, row r = token * G +
// head, so a row tile's queries are read in runs. Every key of the context is
// seen by every row, drafted key j by the rows whose mask has bit j.
//
// Work split: CTA = (KV head, row tile, part of the positions, sequence). One
// part writes the result itself. Up to 8 parts are a cluster where all
// clusters fit the SMs at once: each leaves its (m, l, o) in shared memory and
// the CTAs share the rows' join (tree_join): one launch, host time of a call
// 11.4 -> 5 us. Of more parts (m, l, o) go to the caller's workspace and
// tree_merge_kernel joins them.
//
// tree_mma_kernel (few rows, or head_dim above 128): stages of 64 positions of
// K and V come by TMA (128-byte swizzle: ldmatrix without bank conflicts), the
// warps take blocks of 16 positions in turn and wait for stages, never for one
// another; the warp that ends a stage's last block fills it again: mma.sync
// m16n8k16 with fp32 accumulators, online softmax with a lazy rescale, joined
// at the end. fp32 queries and weights are two fp16 halves each (x = hi + lo to
// 2^-22); both halves run on the same B fragments, 16 rows per warp. Bound by
// memory up to some 40 rows. (More rows: tree_tc.cu.)
//  * Queries are scaled per row by a power of two to 2^8..2^9, so neither half
//    leaves fp16's range; the power goes into the score's factor (exact).
//  * The softmax reference stays 10 below the running maximum (log2 units), so
//    the largest weight is 2^10 at first and below 2^16 before a rescale. fp16's
//    smallest step, 2^-24, is then 2^-34 of the largest weight, and what it cuts
//    off 100,000 small weights beside a large one 3e-6 of it (half a step each).
//    (With 6 below, what lay under 2^-31 of the largest added nothing to the
//    result but all of itself to the sum.)
//  * The tensor cores cut their accumulators instead of rounding them: every
//    accumulation loses half a unit of the last place towards zero, 480 of them
//    8.5e-6 of the result. Each block's sum therefore starts at zero and is
//    added to the running one in fp32, and the low halves' part of a score,
//    small as it is, has an accumulator of its own.
//  * A block where some row does not see some key takes the masked path, which
//    also looks for infinities and NaN among its values: 0 * inf would carry
//    them into rows that do not see them, so such a block adds its values
//    one visible key at a time.
#include "backend.h"
#include "tree.cuh"

#include <algorithm>
#include <cmath>

namespace vbs {

template <int HD, int WR, int WP> struct TreeCfg {
    static constexpr int NW = WR * WP, THREADS = NW * 32;
    static constexpr int ROWS = 16 * WR;
    static constexpr int SP = 64;                      // positions per stage, 4 blocks of 16
    static constexpr int BLKS = HD / 64;               // boxes of 64 dims
    static constexpr int BOX = SP * 128, HALF = BLKS * BOX, STAGE = 2 * HALF;   // keys, then values
    static constexpr int NST = 3;
    static constexpr bool QREG = HD <= 128;            // query halves in registers
    static constexpr int QRS = HD * 2 + 16, QSM = QREG ? 0 : ROWS * QRS * 2;
    static constexpr int OLD = HD + 4;                 // floats per row in the join of the warps
    static constexpr int JOIN = WP * ROWS * OLD * 4;
    static constexpr int BODY = NST * STAGE > JOIN ? NST * STAGE : JOIN;
    static constexpr int SMEM = BODY + QSM;
    static constexpr int CTAS = SMEM <= 113 * 1024 ? 2 : 1;   // per SM
    static_assert(WP % 4 == 0, "a stage's 4 blocks go to 4 warps");
};

template <int HD, int WR, int WP>
__global__ void __launch_bounds__(TreeCfg<HD, WR, WP>::THREADS) tree_mma_kernel(const __grid_constant__ TreeParams p,
                                                                                const __grid_constant__ CUtensorMap km,
                                                                                const __grid_constant__ CUtensorMap vm) {
    using C = TreeCfg<HD, WR, WP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ int32_t sh_min[C::NW];
    __shared__ __align__(8) uint64_t bars[2 * C::NST];   // full, empty
    __shared__ uint32_t used[C::NST], issued[C::NST];   // blocks of the stage that are through; 1 + the stage's last tile
    __shared__ int sh_bad;
    __shared__ __align__(8) float2 sh_ml[C::ROWS];       // the part's, where parts are joined in a cluster
    volatile int *bad = &sh_bad;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wr = warp % WR, wp = warp / WR;
    const uint32_t kvh = blockIdx.x % p.nkh, tile = blockIdx.x / p.nkh, split = blockIdx.y, b = blockIdx.z;
    const uint32_t G = p.G, R0 = tile * C::ROWS;
    pdl_launch_dependents();
    uint32_t nc, nt;
    if (!tree_lengths(p, b, nc, nt) || R0 >= nt * G) return;
    const uint32_t end = nc + nt, nrows = nt * G;
    const uint32_t first = tree_first(p, b, nc, nt, sh_min);
    uint32_t t0, t1;
    tree_part(p, first, end, split, t0, t1);
    const uint64_t slot = (uint64_t)(b * p.nkh + kvh) * p.row_tiles + tile;
    float2 *ml = p.part_ml + (slot * p.n_splits + split) * C::ROWS;
    auto joins = [&]() {   // in the cluster: the sums of the warps' join are in the first warp's place
        cluster_meet();
        tree_join(p, smem_u32(sh_ml), smem_u32(smem), C::OLD * 4, min((uint32_t)C::ROWS, nrows - R0), R0, kvh, b, split, threadIdx.x,
                  C::THREADS);
        cluster_meet();
    };
    if (t0 >= t1 && p.n_splits > 1) {   // no positions: an empty part
        for (int r = threadIdx.x; r < C::ROWS; r += C::THREADS) (p.joined ? sh_ml : ml)[r] = make_float2(-INFINITY, 0.f);
        if (p.joined) joins();
        return;
    }
    const uint32_t nch = (t1 - t0 + C::SP - 1) / C::SP, blks = (p.hd + 63) / 64;
    const int32_t *kpos = p.k_pos ? p.k_pos + (uint64_t)(p.k_pos_per_head ? b * p.nkh + kvh : b) * p.max_ctx : nullptr;
    const uint32_t sbase = smem_u32(smem), full0 = smem_u32(bars), empty0 = full0 + 8 * C::NST;
    auto waits = [&](uint32_t bar, uint32_t parity) -> bool {
        if (mbar_wait_bounded(bar, parity, kWaitNs)) return true;
        *bad = 1;
        return false;
    };
    // stage c's keys and values (one thread)
    auto load = [&](uint32_t c) {
        const uint32_t s = c % C::NST, st = sbase + s * C::STAGE;
        asm volatile("st.release.cta.shared.u32 [%0], %1;" ::"r"(smem_u32(&issued[s])), "r"(c + 1) : "memory");
        mbar_arrive_expect_tx(full0 + 8 * s, 2 * blks * C::BOX);
        for (uint32_t k = 0; k < blks; ++k) tree_tma(st + k * C::BOX, &km, 64 * k, t0 + c * C::SP, kvh, b, full0 + 8 * s);
        for (uint32_t k = 0; k < blks; ++k) tree_tma(st + C::HALF + k * C::BOX, &vm, 64 * k, t0 + c * C::SP, kvh, b, full0 + 8 * s);
    };
    // tile c's load has been issued: the tile before it in its stage is done with
    auto under_way = [&](uint32_t c) -> bool {
        const uint32_t at = smem_u32(&issued[c % C::NST]);
        uint32_t n;
        auto there = [&]() {
            asm volatile("ld.acquire.cta.shared.u32 %0, [%1];" : "=r"(n) : "r"(at) : "memory");
            return n > c;
        };
        if (there()) return true;
        const uint64_t since = global_ns();
        while (!there()) {
            if (*bad || global_ns() - since > kWaitNs) {
                *bad = 1;
                return false;
            }
        }
        return true;
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::NST; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 4 * WR);
            used[s] = issued[s] = 0;
        }
        sh_bad = 0;
        mbar_fence_init();
        for (uint32_t c = 0; c < min(nch, (uint32_t)C::NST); ++c) load(c);
    }

    // the two rows of this thread: g and g + 8 of the warp's 16
    const int g = lane >> 2, qd = 2 * (lane & 3);
    uint32_t row[2], tok[2];
    bool on[2];
    float fac[2], slope[2] = {0.f, 0.f};
    int32_t qpos[2];
    const float *qsrc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        row[h] = R0 + 16 * wr + g + 8 * h;
        on[h] = row[h] < nrows;
        const uint32_t rr = on[h] ? row[h] : 0u;
        tok[h] = rr / G;
        const uint32_t head = kvh * G + rr % G;
        qpos[h] = tree_qpos(p, b, tok[h], nc);
        if (p.slopes) slope[h] = p.slopes[head] * TREE_LOG2E;
        qsrc[h] = p.q + (((uint64_t)b * p.n_tokens + tok[h]) * p.nqh + head) * p.hd;
    }
    // query halves as A fragments, scaled by the row's power of two
    uint32_t qh[C::QREG ? HD / 16 : 1][4], ql[C::QREG ? HD / 16 : 1][4];
    {
        float2 x[2][HD / 8];
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
                const bool ok = on[h] && 8 * n + qd < (int)p.hd;
                x[h][n] = ok ? *reinterpret_cast<const float2 *>(qsrc[h] + 8 * n + qd) : make_float2(0.f, 0.f);
                top[h] = fmaxf(top[h], fmaxf(fabsf(x[h][n].x), fabsf(x[h][n].y)));
            }
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            // 2^e with top in [2^8, 2^9) afterwards; zero, tiny or not finite: no scaling
            int e = (int)((__float_as_uint(top[h]) >> 23) & 255u) - 127;
            e = (e < -100 || e > 100) ? 0 : 8 - e;
            const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) { x[h][n].x *= up; x[h][n].y *= up; }
            fac[h] = p.scale * down;
        }
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // a0, a2: row g; a1, a3: row g + 8; k half j / 2
                const float2 v = x[j & 1][2 * kk + (j >> 1)];
                const __half2 hi = __floats2half2_rn(v.x, v.y);
                const float2 f = __half22float2(hi);
                const __half2 lo = __floats2half2_rn(v.x - f.x, v.y - f.y);
                if constexpr (C::QREG) {
                    qh[kk][j] = *reinterpret_cast<const uint32_t *>(&hi);
                    ql[kk][j] = *reinterpret_cast<const uint32_t *>(&lo);
                } else if (wp == 0) {
                    uint8_t *d = smem + C::BODY + (16 * wr + g + 8 * (j & 1)) * C::QRS + (16 * kk + 8 * (j >> 1) + qd) * 2;
                    *reinterpret_cast<__half2 *>(d) = hi;
                    *reinterpret_cast<__half2 *>(d + C::ROWS * C::QRS) = lo;
                }
            }
        }
    }
    const float cap2 = p.cap * TREE_LOG2E;
    const float pre = p.cap > 0.f ? 1.f / p.cap : TREE_LOG2E;
    fac[0] *= pre;
    fac[1] *= pre;
    // highest query position of the warp's rows, for the window's fast path
    int32_t qmax = max(qpos[0], qpos[1]);
    qmax = __reduce_max_sync(0xffffffffu, qmax);

    float o[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float mref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    __syncthreads();   // barriers, and queries in shared memory
    // blocks of 16 positions in turn over the position warps; a block's key
    // positions (lane: position) are read one block ahead
    const uint32_t kks = (p.hd + 31) / 32 * 2, ns = (p.hd + 15) / 16 * 2;   // 16s of dims with keys, 8s with values
    auto kp_at = [&](uint32_t t) { return lane < 16 && t + lane < t1 ? tree_kpos(p, kpos, b, t + lane, nc) : 0x7FFFFFFF; };
    const bool want_pos = kpos || p.window || p.slopes;
    int32_t kn = want_pos ? kp_at(t0 + 16 * wp) : 0;
    // A barrier's parity tells two neighbouring phases apart. 8 warps and 3
    // stages: a warp visits every other tile, so a stage may be a whole tile
    // behind the one that the warp is at; it looks first whether that is under
    // way. (All warps through all stages instead: 131 us for the 110 of 16
    // sequences of up to 8000 positions with a window of 4096.)
    for (uint32_t tb = t0 + 16 * wp, j = wp; tb < t1; tb += 16 * WP, j += WP) {
        const uint32_t c = j / 4, st = sbase + c % C::NST * C::STAGE;
        const int32_t kp = kn;
        if (want_pos) kn = kp_at(tb + 16 * WP);
        if (!__all_sync(0xffffffffu, !*bad && (WP == 4 || under_way(c)) && waits(full0 + 8 * (c % C::NST), (c / C::NST) & 1u))) break;
        {
            const uint32_t kst = st + 16 * (j & 3) * 128, vst = kst + C::HALF, sw = lane & 7;
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, sl[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk += 2) {
                if (kk >= (int)kks) break;
                uint32_t ah[2][4], al[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if constexpr (C::QREG) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) { ah[u][j] = qh[kk + u][j]; al[u][j] = ql[kk + u][j]; }
                    } else {
                        const uint32_t a = sbase + C::BODY + (16 * wr + (lane & 15)) * C::QRS + (16 * (kk + u) + 8 * (lane >> 4)) * 2;
                        ldsm_x4(a, ah[u][0], ah[u][1], ah[u][2], ah[u][3]);
                        ldsm_x4(a + C::ROWS * C::QRS, al[u][0], al[u][1], al[u][2], al[u][3]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4(kst + (kk >> 2) * C::BOX + (8 * j + (lane & 7)) * 128 + ((((2 * kk) & 7) + (lane >> 3)) ^ sw) * 16, b0, b1, b2, b3);
                    mma_f16_acc(sl[j], al[0], b0, b1);
                    mma_f16_acc(s[j], ah[0], b0, b1);
                    mma_f16_acc(sl[j], al[1], b2, b3);
                    mma_f16_acc(s[j], ah[1], b2, b3);
                }
            }
            // x[h][e]: row h, keys tb + {qd, qd+1, 8+qd, 9+qd}
            const float x00 = s[0][0] + sl[0][0], x01 = s[0][1] + sl[0][1], x02 = s[1][0] + sl[1][0], x03 = s[1][1] + sl[1][1];
            const float x10 = s[0][2] + sl[0][2], x11 = s[0][3] + sl[0][3], x12 = s[1][2] + sl[1][2], x13 = s[1][3] + sl[1][3];
            float x[2][4] = {{x00, x01, x02, x03}, {x10, x11, x12, x13}};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[h][e] *= fac[h];
            if (p.cap > 0.f) {
                tree_cap_all(x[0], cap2);
                tree_cap_all(x[1], cap2);
            }
            uint32_t hidden = 0;   // bit 4 h + e: row h does not see key e
            // every row sees every position: by the lowest key position
            const bool context = tb + 16 <= min(nc, t1);
            const int32_t low = want_pos && context ? __reduce_min_sync(0xffffffffu, kp) : 0;
            const bool plain = context && (!kpos || low >= 0) && (!p.window || qmax - low < (int32_t)p.window);
            if (!plain || p.slopes) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t kl = qd + (e & 1) + 8 * (e >> 1), t = tb + kl;
                    const int32_t k = want_pos ? __shfl_sync(0xffffffffu, kp, kl) : 0;
                    const bool in = t < t1, drafted = in && t >= nc;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        bool see = in && (!kpos || k >= 0);
                        if (drafted && on[h])
                            see = see && (p.mask ? (p.mask[((uint64_t)b * p.n_tokens + tok[h]) * p.words + ((t - nc) >> 5)] >>
                                                    ((t - nc) & 31)) & 1u
                                                 : t - nc <= tok[h]);
                        if (p.window) see = see && qpos[h] - k < (int32_t)p.window;
                        if (p.slopes) x[h][e] = fmaf(slope[h], (float)(k - qpos[h]), x[h][e]);
                        if (!see) {
                            x[h][e] = -INFINITY;
                            hidden |= 1u << (4 * h + e);
                        }
                    }
                }
            }
            float pe[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if (mx - mref[h] > TREE_LAZY) {   // (what the weights' exponents are: large scores round)
                    const float r = ex2(mref[h] - (mx - TREE_BELOW));   // 0 on the first block
                    mref[h] = mx - TREE_BELOW;
                    l[h] *= r;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) { o[n][2 * h] *= r; o[n][2 * h + 1] *= r; }
                }
                const float base = mref[h] == -INFINITY ? 0.f : mref[h];   // nothing seen so far: weights 0
#pragma unroll
                for (int e = 0; e < 4; ++e) pe[h][e] = ex2(x[h][e] - base);
                l[h] += (pe[h][0] + pe[h][1]) + (pe[h][2] + pe[h][3]);
            }
            bool apart = false;
            if (__any_sync(0xffffffffu, hidden != 0)) {
                // some row does not see some key: values must be finite for 0 * v to be 0
                uint32_t zero = 0;
#pragma unroll 4
                for (uint32_t i = lane; i < 16 * 8 * blks; i += 32) zero = finite4(lds_u128(vst + (i >> 7) * C::BOX + (i & 127) * 16), zero);
                apart = __any_sync(0xffffffffu, zero != 0u);
            }
            if (!apart) {
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float u = pe[j & 1][2 * (j >> 1)], w = pe[j & 1][2 * (j >> 1) + 1];
                    const __half2 hi = __floats2half2_rn(u, w);
                    const float2 f = __half22float2(hi);
                    const __half2 lo = __floats2half2_rn(u - f.x, w - f.y);
                    ph[j] = *reinterpret_cast<const uint32_t *>(&hi);
                    pl[j] = *reinterpret_cast<const uint32_t *>(&lo);
                }
#pragma unroll
                for (int n = 0; n < HD / 8; n += 2) {
                    if (n >= (int)ns) break;
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4_trans(vst + (n >> 3) * C::BOX + ((lane & 7) + 8 * ((lane >> 3) & 1)) * 128 + (((n & 7) + (lane >> 4)) ^ sw) * 16, b0,
                                  b1, b2, b3);
                    float u0[4] = {0.f, 0.f, 0.f, 0.f}, u1[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_f16_acc(u0, pl, b0, b1);
                    mma_f16_acc(u0, ph, b0, b1);
                    mma_f16_acc(u1, pl, b2, b3);
                    mma_f16_acc(u1, ph, b2, b3);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { o[n][e] += u0[e]; o[n + 1][e] += u1[e]; }
                }
            } else {
#pragma unroll 1
                for (int k = 0; k < 16; ++k) {   // key k's weights of rows g, g + 8 sit in lane (k % 8) / 2 of the quad
                    const int from = (lane & ~3) | ((k & 7) >> 1);
                    float w[2];
                    bool see[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v = 0.f;
                        uint32_t hid = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {   // all lanes shuffle; the key's element is kept
                            const float t = __shfl_sync(0xffffffffu, pe[h][e], from);
                            const uint32_t hb = __shfl_sync(0xffffffffu, (hidden >> (4 * h + e)) & 1u, from);
                            if (e == 2 * (k >> 3) + (k & 1)) { v = t; hid = hb; }
                        }
                        w[h] = v;
                        see[h] = !hid;
                    }
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) {
                        if (n >= (int)ns) break;
                        uint32_t vv;
                        vv = lds_u32(vst + (n >> 3) * C::BOX + k * 128 + (((n & 7) ^ (k & 7)) << 4) + qd * 2);
                        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&vv));
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (see[h]) { o[n][2 * h] = fmaf(w[h], f.x, o[n][2 * h]); o[n][2 * h + 1] = fmaf(w[h], f.y, o[n][2 * h + 1]); }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) {
            // the stage's last block fills it again (it waits for arrivals
            // that are all made by then)
            const uint32_t s = c % C::NST;
            mbar_arrive(empty0 + 8 * s);
            if (atomicAdd(&used[s], 1u) == 4 * WR - 1) {
                used[s] = 0;
                if (c + C::NST < nch && waits(empty0 + 8 * s, (c / C::NST) & 1u)) load(c + C::NST);
            }
        }
        __syncwarp();
    }

    // join the warps that shared these rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    __syncthreads();   // all stages are used up
    float *sh = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float *d = sh + (wp * C::ROWS + 16 * wr + g + 8 * h) * C::OLD;
        if ((lane & 3) == 0) { d[HD] = mref[h]; d[HD + 1] = l[h]; }
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
            *reinterpret_cast<float2 *>(d + 8 * n + qd) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
    __syncthreads();
    if (*bad) {
        if (threadIdx.x == 0) {
            dev_flag_error(p.err, DERR_TIMEOUT_FULL);
            for (int s = 0; s < C::NST; ++s)   // copies may still be landing
                if (issued[s]) mbar_wait_bounded(full0 + 8 * s, ((issued[s] - 1) / C::NST) & 1u, kWaitNs);
        }
        if (p.joined) {   // the others wait for this part
            for (int r = threadIdx.x; r < C::ROWS; r += C::THREADS) sh_ml[r] = make_float2(-INFINITY, 0.f);
            joins();
        }
        return;
    }
    const uint32_t live = min((uint32_t)C::ROWS, nrows - R0), q4 = p.hd / 4;
    float *po = p.part_o + (slot * p.n_splits + split) * C::ROWS * p.hd;
    for (uint32_t i = threadIdx.x; i < live * q4; i += C::THREADS) {
        const uint32_t r = i / q4, d = i % q4 * 4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WP; ++w) M = fmaxf(M, sh[(w * C::ROWS + r) * C::OLD + HD]);
        float L = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WP; ++w) {
            const float *x = sh + (w * C::ROWS + r) * C::OLD;
            const float f = x[HD] == -INFINITY ? 0.f : ex2(x[HD] - M);
            const float4 v = *reinterpret_cast<const float4 *>(x + d);
            L += x[HD + 1] * f;
            a.x = fmaf(v.x, f, a.x); a.y = fmaf(v.y, f, a.y); a.z = fmaf(v.z, f, a.z); a.w = fmaf(v.w, f, a.w);
        }
        if (p.joined) {
            if (d == 0) sh_ml[r] = make_float2(M, L);
            *reinterpret_cast<float4 *>(sh + r * C::OLD + d) = a;   // (read by this thread alone)
        } else if (p.n_splits > 1) {
            if (d == 0) ml[r] = make_float2(M, L);
            *reinterpret_cast<float4 *>(po + (uint64_t)r * p.hd + d) = a;
        } else {
            const uint32_t rr = R0 + r, head = kvh * G + rr % G;
            const float il = L == 0.f ? 0.f : 1.f / L;   // nothing visible: zeros
            if (L == 0.f) a = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4 *>(p.out + (((uint64_t)b * p.n_tokens + rr / G) * p.nqh + head) * p.hd + d) =
                make_float4(a.x * il, a.y * il, a.z * il, a.w * il);
            if (p.lse && d == 0)
                p.lse[(uint64_t)(b * p.nkh + kvh) * (p.n_tokens * G) + rr] = L == 0.f ? -INFINITY : M + log2f(L);
        }
    }
    if (p.joined) joins();
}

// ---------------------------------------------------------------------------
// Join of the parts. Few rows, or more than 32 parts: one CTA per row. The parts' maxima and sums are read at
// once and become their factors in shared memory; then the warps share the
// parts, TREE_MU loads in flight each, and their sums are added in order.
// Both are launched as programmatic dependents of the kernel that writes the
// parts: they are on the SMs when that one ends.
// ---------------------------------------------------------------------------
constexpr int TREE_MW = 8, TREE_MU = 8;
constexpr uint32_t TREE_MAX_PARTS = 1024;

// Many rows of up to 32 parts: a warp per row, a lane per part for the factors, TREE_MU
// parts' loads in flight. (A CTA per row took 22 us for 4032 rows of 8 parts.)
__global__ void __launch_bounds__(TREE_MW * 32) tree_merge_warp_kernel(const __grid_constant__ TreeParams p, uint32_t tile_rows) {
    const uint32_t r = blockIdx.x * TREE_MW + (threadIdx.x >> 5), kvh = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
    uint32_t nc, nt;
    const bool live = tree_lengths(p, b, nc, nt) && r < nt * p.G;
    pdl_wait();
    pdl_launch_dependents();
    if (!live) return;
    const uint32_t tile = r / tile_rows, ri = r - tile * tile_rows, ns = p.n_splits;
    const uint64_t slot = (uint64_t)(b * p.nkh + kvh) * p.row_tiles + tile;
    const float *po = p.part_o + (slot * ns * tile_rows + ri) * p.hd;
    const float2 x = lane < ns ? __ldcg(p.part_ml + (slot * ns + lane) * tile_rows + ri) : make_float2(-INFINITY, 0.f);
    const float M = warp_max(x.x);
    const bool has = !(x.y == 0.f);   // an empty part has no sums (and wrote none); a NaN goes through
    const float f = has ? ex2(x.x - M) : 0.f;
    const float L = warp_sum(has ? x.y * f : 0.f);
    const uint32_t parts = __ballot_sync(0xffffffffu, has);
    const float il = L == 0.f ? 0.f : 1.f / L;
    const uint32_t tok = tree_token(p, r), q4 = p.hd / 4;
    float *out = p.out + (((uint64_t)b * p.n_tokens + tok) * p.nqh + kvh * p.G + (r - tok * p.G)) * p.hd;
    for (uint32_t d0 = 0; d0 < q4; d0 += 32) {   // wider rows take two rounds
        const uint32_t d = d0 + lane;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (uint32_t s0 = 0; s0 < ns; s0 += TREE_MU) {
            float4 v[TREE_MU];
#pragma unroll
            for (int u = 0; u < TREE_MU; ++u)
                v[u] = ((parts >> ((s0 + u) & 31)) & 1u) && s0 + u < ns && d < q4
                           ? __ldcg(reinterpret_cast<const float4 *>(po + (uint64_t)(s0 + u) * tile_rows * p.hd) + d)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < TREE_MU; ++u) {
                const float g = __shfl_sync(0xffffffffu, f, (s0 + u) & 31);
                a.x = fmaf(v[u].x, g, a.x); a.y = fmaf(v[u].y, g, a.y);
                a.z = fmaf(v[u].z, g, a.z); a.w = fmaf(v[u].w, g, a.w);
            }
        }
        if (L == 0.f) a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d < q4) reinterpret_cast<float4 *>(out)[d] = make_float4(a.x * il, a.y * il, a.z * il, a.w * il);
    }
    if (p.lse && lane == 0)
        p.lse[(uint64_t)(b * p.nkh + kvh) * (p.n_tokens * p.G) + r] = L == 0.f ? -INFINITY : M + log2f(L);
}

__global__ void __launch_bounds__(TREE_MW * 32) tree_merge_kernel(const __grid_constant__ TreeParams p, uint32_t tile_rows) {
    __shared__ float fac[TREE_MAX_PARTS];
    __shared__ float sm_m[TREE_MW], sm_l[TREE_MW];
    __shared__ __align__(16) float sm_o[TREE_MW][256];
    const uint32_t r = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t nc, nt;
    const bool live = tree_lengths(p, b, nc, nt) && r < nt * p.G;
    pdl_wait();
    pdl_launch_dependents();
    if (!live) return;
    const uint32_t tile = r / tile_rows, ri = r % tile_rows, ns = p.n_splits;
    const uint64_t slot = (uint64_t)(b * p.nkh + kvh) * p.row_tiles + tile;
    const float2 *ml = p.part_ml + slot * ns * tile_rows + ri;
    const float *po = p.part_o + (slot * ns * tile_rows + ri) * p.hd;
    float2 x[TREE_MAX_PARTS / (TREE_MW * 32)];
    float M = -INFINITY;
#pragma unroll
    for (uint32_t k = 0; k < TREE_MAX_PARTS / (TREE_MW * 32); ++k) {
        const uint32_t s = threadIdx.x + k * TREE_MW * 32;
        x[k] = s < ns ? __ldcg(ml + (uint64_t)s * tile_rows) : make_float2(-INFINITY, 0.f);
        M = fmaxf(M, x[k].x);
    }
    M = warp_max(M);
    if (lane == 0) sm_m[warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TREE_MW; ++w) M = fmaxf(M, sm_m[w]);
    float L = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < TREE_MAX_PARTS / (TREE_MW * 32); ++k) {
        const uint32_t s = threadIdx.x + k * TREE_MW * 32;
        const bool has = !(x[k].y == 0.f);   // an empty part has no sums (and wrote none); a NaN goes through
        const float f = has ? ex2(x[k].x - M) : 0.f;
        if (has) L += x[k].y * f;
        if (s < ns) fac[s] = has ? f : -1.f;
    }
    L = warp_sum(L);
    if (lane == 0) sm_l[warp] = L;
    __syncthreads();
    const uint32_t q4 = p.hd / 4;   // 16-byte pieces of a row; a warp covers 32 pieces, wider rows take two
    for (uint32_t d0 = 0; d0 < q4; d0 += 32) {
        const uint32_t d = d0 + lane;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t s0 = warp; s0 < ns; s0 += TREE_MW * TREE_MU) {
            float4 v[TREE_MU];
#pragma unroll
            for (int u = 0; u < TREE_MU; ++u) {
                const uint32_t s = s0 + u * TREE_MW;
                v[u] = s < ns && !(fac[s] < 0.f) && d < q4 ? __ldcg(reinterpret_cast<const float4 *>(po + (uint64_t)s * tile_rows * p.hd) + d)
                                                         : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < TREE_MU; ++u) {
                const uint32_t s = s0 + u * TREE_MW;
                const float f = s < ns ? fac[s] : 0.f;   // -1 meets zeros
                a.x = fmaf(v[u].x, f, a.x); a.y = fmaf(v[u].y, f, a.y);
                a.z = fmaf(v[u].z, f, a.z); a.w = fmaf(v[u].w, f, a.w);
            }
        }
        *reinterpret_cast<float4 *>(&sm_o[warp][(lane + d0) * 4]) = a;
    }
    __syncthreads();
    L = 0.f;
#pragma unroll
    for (int w = 0; w < TREE_MW; ++w) L += sm_l[w];
    const float il = L == 0.f ? 0.f : 1.f / L;
    const uint32_t tok = tree_token(p, r);
    float *out = p.out + (((uint64_t)b * p.n_tokens + tok) * p.nqh + kvh * p.G + (r - tok * p.G)) * p.hd;
    for (uint32_t d = threadIdx.x; d < p.hd; d += TREE_MW * 32) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < TREE_MW; ++w) v += sm_o[w][d];
        out[d] = L == 0.f ? 0.f : v * il;
    }
    if (p.lse && threadIdx.x == 0)
        p.lse[(uint64_t)(b * p.nkh + kvh) * (p.n_tokens * p.G) + r] = L == 0.f ? -INFINITY : M + log2f(L);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint32_t TREE_JOIN_NS = 800, TREE_MERGE_NS = 3000, TREE_MERGE_RATE = 4000;   // in a cluster; by a second kernel, and bytes per ns of the parts' sums
// Clusters that run at once, by kernel (head_dim up to 64, 128, 256 with 16
// rows, 256 with 32, tcgen05) and size; set by tree_configure.
static int tree_fit[5][TREE_CLUSTER + 1];

struct TreePlan {
    uint32_t rows, tile_rows, row_tiles, n_splits, per_split;
    bool tc, joined;                    // tree_tc_kernel; parts joined in clusters
    size_t ml, o, lse, bytes;   // offsets into the workspace, total
};

// The parts of one kernel's plan: the number that ends first, counting whole
// waves of CTAs on `slots`, a position's and a CTA's time, and the join's.
// Only a plan: the kernels divide what the lengths on the device leave. Up to
// 8 parts can be a cluster that joins them itself, where all clusters run at
// once (`clusters`[parts] of them; waiting ones cost far more than a join).
struct TreeParts { uint64_t ns; uint32_t per, parts; bool joined; };
static TreeParts tree_parts(uint64_t ctas, uint64_t slots, uint32_t span, uint32_t unit, uint32_t pos_ns, uint32_t cta_ns, uint32_t row_bytes,
                            const int *clusters) {
    TreeParts best = {~0ull, 0, 0, false};
    const uint32_t units = (span + unit - 1) / unit;
    for (uint32_t s = 1; s <= std::min(TREE_MAX_PARTS, units);) {
        const uint32_t per = (units + s - 1) / s, parts = (units + per - 1) / per;
        const uint64_t one = (uint64_t)per * unit * pos_ns / 10 + cta_ns;
        const bool joined = parts > 1 && parts <= TREE_CLUSTER && ctas <= (uint64_t)clusters[parts];
        uint64_t ns = (ctas * parts + slots - 1) / slots * one;
        if (joined) ns = one + TREE_JOIN_NS;
        else if (parts > 1) ns += TREE_MERGE_NS + ctas * parts * row_bytes / TREE_MERGE_RATE;
        if (ns < best.ns) best = {ns, per * unit, parts, joined};
        if (per == 1 || ctas * s > 16 * slots) break;
        s = (units + per - 2) / (per - 1);   // the next number that makes a part shorter
    }
    return best;
}

// The kernels that take `rows` rows of a KV head. tree_mma_kernel: 16 rows a
// CTA (32 above head_dim 128, where a CTA has an SM to itself);
// tree_tc_kernel: 128 rows, or 256 of more, which halves what K and V cost
// but doubles a CTA. Measured on full SMs, ns per position and CTA: 30
// (head_dim 128), 22 (64) with two CTAs per SM, 22 and 44 (256; 16 and 32
// rows); 15 and 28.5 (128; 128 and 256 rows), 10 and 19.5 (64).
struct TreeKind {
    bool tc;
    uint32_t rows, per_sm, unit, pos_ns, cta_ns;   // pos_ns in tenths
    const int *clusters;
};
static uint32_t tree_kinds(uint32_t hd, uint32_t rows, TreeKind (&k)[3]) {
    uint32_t n = 0;
    if (hd > 128) {
        k[n++] = rows <= 16 ? TreeKind{false, 16, 1, 64, 220, 6000, tree_fit[2]} : TreeKind{false, 32, 1, 64, 440, 6000, tree_fit[3]};
    } else {
        const bool big = hd > 64;
        k[n++] = {false, 16, 2, 64, big ? 300u : 220u, 4000, tree_fit[big ? 1 : 0]};
        if (rows > 16) k[n++] = {true, TREE_TC_ROWS, 1, TREE_TC_SP, big ? 150u : 100u, 9000, tree_fit[4]};   // (16 rows are one CTA's of the other kernel)
        if (rows > TREE_TC_ROWS) k[n++] = {true, 2 * TREE_TC_ROWS, 1, TREE_TC_SP, big ? 285u : 195u, 12000, tree_fit[4]};
    }
    return n;
}

// Positions that a plan counts with.
static uint32_t tree_span(const vbs_cu_tree_t *t) {
    return t->window && !t->k_pos ? (uint32_t)std::min<uint64_t>(t->ctx_limit, (uint64_t)t->window + t->n_tokens + 63) : t->ctx_limit;
}
static size_t tree_aligned(size_t n) { return (n + 255) / 256 * 256; }

static TreePlan tree_plan(const vbs_cu_kv_t *kv, const vbs_cu_tree_t *t, int n_sm) {
    TreePlan pl = {};
    const uint32_t G = t->n_q_heads / kv->n_kv_heads, hd = kv->head_dim, span = tree_span(t);
    pl.rows = t->n_tokens * G;
    const uint64_t heads = (uint64_t)kv->n_kv_heads * kv->n_seqs;
    TreeParts best = {~0ull, 0, 0, false};
    TreeKind kinds[3];
    const uint32_t n_kinds = tree_kinds(hd, pl.rows, kinds);
    for (uint32_t i = 0; i < n_kinds; ++i) {
        const TreeKind &k = kinds[i];
        const uint32_t tiles = (pl.rows + k.rows - 1) / k.rows;
        const TreeParts one = tree_parts(heads * tiles, (uint64_t)k.per_sm * n_sm, span, k.unit, k.pos_ns, k.cta_ns, k.rows * hd * 4, k.clusters);
        if (one.ns >= best.ns) continue;
        best = one;
        pl.tc = k.tc;
        pl.tile_rows = k.rows;
        pl.row_tiles = tiles;
    }
    pl.per_split = best.per;
    pl.n_splits = best.parts;
    pl.joined = best.joined;
    auto take = [&](size_t n) { const size_t at = pl.bytes; pl.bytes += tree_aligned(n); return at; };
    if (pl.n_splits > 1 && !pl.joined) {
        pl.ml = take(heads * pl.row_tiles * pl.n_splits * pl.tile_rows * sizeof(float2));
        pl.o = take(heads * pl.row_tiles * pl.n_splits * pl.tile_rows * kv->head_dim * sizeof(float));
    }
    if (t->weights_out) pl.lse = take(heads * pl.rows * sizeof(float));
    pl.bytes = std::max<size_t>(pl.bytes, 256);
    return pl;
}

// The largest min over the lines (slope * x + fixed) less own * x, x up to
// span: along the lines' lower envelope while it grows.
struct TreeLine { double slope, fixed; };
static double tree_room(const TreeLine *l, uint32_t n, double own, double span) {
    uint32_t j = 0;
    for (uint32_t i = 1; i < n; ++i)
        if (l[i].fixed < l[j].fixed || (l[i].fixed == l[j].fixed && l[i].slope < l[j].slope)) j = i;
    double x = 0.;
    while (l[j].slope > own) {
        double to = span;
        uint32_t next = j;
        for (uint32_t i = 0; i < n; ++i) {
            if (l[i].slope >= l[j].slope) continue;
            const double at = (l[i].fixed - l[j].fixed) / (l[j].slope - l[i].slope);
            if (at < to) { to = at; next = i; }
        }
        x = std::max(x, to);
        if (next == j) break;
        j = next;
    }
    return l[j].fixed + (l[j].slope - own) * x;
}

// Bytes that every plan up to this description's ctx_limit, n_tokens and
// window fits into. A plan's own need is no guide to another's: it falls to
// nothing where its parts become a cluster and comes back where they do not
// fit one, and a shorter call may take wider row tiles.
// The plan of x positions costs no more than any that tree_parts looked at:
// without parts, or with those that fill the SMs w times, w up to 16, each a
// line in x. It costs at least its positions' share of the SMs, its CTAs'
// fixed time and its join's. The room between bounds CTAs x parts.
static size_t tree_bytes(const vbs_cu_kv_t *kv, const vbs_cu_tree_t *t, int n_sm) {
    const uint32_t hd = kv->head_dim, rows = t->n_tokens * (t->n_q_heads / kv->n_kv_heads);
    const uint64_t heads = (uint64_t)kv->n_kv_heads * kv->n_seqs;
    const uint32_t span = tree_span(t);
    size_t bytes = 0;
    for (uint32_t r = std::min(rows, 16u);;) {   // (row tiles are multiples of 16; up to 16 rows may have a kernel of their own)
        TreeKind kinds[3];
        TreeLine lines[3 * 17];
        const uint32_t n = tree_kinds(hd, r, kinds);
        uint32_t n_lines = 0, step = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const TreeKind &k = kinds[i];
            const uint64_t slots = (uint64_t)k.per_sm * n_sm, ctas = heads * ((r + k.rows - 1) / k.rows), waves = (ctas + slots - 1) / slots;
            const double pos = k.pos_ns / 10., unit = k.unit * pos;
            lines[n_lines++] = {waves * pos, waves * (unit + k.cta_ns)};
            for (uint64_t w = waves; w <= 16; ++w) {
                const double parts = (double)std::min<uint64_t>(w * slots / ctas, TREE_MAX_PARTS);
                lines[n_lines++] = {w * pos / parts, w * (unit / parts + unit + k.cta_ns) + TREE_MERGE_NS + w * slots * (double)(k.rows * hd * 4) / TREE_MERGE_RATE};
            }
        }
        for (uint32_t i = 0; i < n; ++i) {
            const TreeKind &k = kinds[i];
            const uint64_t slots = (uint64_t)k.per_sm * n_sm, ctas = heads * ((r + k.rows - 1) / k.rows);
            if (ctas > 16 * slots) continue;   // (tree_parts ends after one part)
            if (!step) step = k.rows;          // the narrowest that still has parts
            const double room = tree_room(lines, n_lines, ctas * (k.pos_ns / 10.) / slots, span) - TREE_MERGE_NS;
            // (tree_parts cuts off fractions of a nanosecond: one of a CTA's time, one of the join's)
            const double most = std::max(0., room + 1) / ((k.cta_ns - 1.) / slots + (double)(k.rows * hd * 4) / TREE_MERGE_RATE);
            // (tree_parts' last step starts at 16 times the SMs and at most doubles the parts)
            const uint64_t parts = std::min<uint64_t>(32 * slots, ctas * std::min<uint64_t>((span + k.unit - 1) / k.unit, TREE_MAX_PARTS));
            const size_t all = (size_t)std::min(most, (double)parts) * k.rows;
            bytes = std::max(bytes, tree_aligned(all * sizeof(float2)) + tree_aligned(all * hd * sizeof(float)));
        }
        if (r == rows || !step) break;
        r = std::min<uint64_t>(rows, r / step * step + step);
    }
    return std::max<size_t>(bytes + (t->weights_out ? tree_aligned(heads * rows * sizeof(float)) : 0), 256);
}

static bool tree_desc_ok(const vbs_cu_kv_t *kv, const vbs_cu_tree_t *t) {
    if (!kv_desc_ok(kv) || !t || !t->n_q_heads || t->n_q_heads % kv->n_kv_heads || !t->n_tokens || !t->ctx_limit ||
        t->ctx_limit > kv->max_ctx || t->ctx_limit > 1u << 28 || !t->n_ctx)
        return false;
    if (t->n_tokens > 4096u || t->n_q_heads / kv->n_kv_heads > 256u) return false;
    if (!std::isfinite(t->scale) || !(t->softcap >= 0.f) || !std::isfinite(t->softcap) || t->window > 0x7FFFFFFFu) return false;
    if (t->softcap > 0.f && t->softcap < 1e-6f) return false;   // its reciprocal scales the scores
    if ((uint64_t)t->n_tokens * t->n_q_heads > 0x7FFFFFFFu) return false;   // rows of a sequence: CTAs are counted in 32 bits
    if (t->weights_in && !t->weights_out) return false;
    const uint64_t w = (uint64_t)kv->n_seqs * kv->n_kv_heads * kv->max_ctx * 4;   // (below 2^63: kv_desc_ok)
    return t->weights_in == t->weights_out || !overlap(t->weights_in, w, t->weights_out, w);   // all of it or nothing
}

// Tensor map of one layer's keys or values, boxes of 64 dims x `rows`
// positions. Encoded anew by every call (host arithmetic, no driver call).
static cudaError_t tree_map(CUtensorMap *m, const uint16_t *base, const vbs_cu_kv_t *kv, uint32_t rows) {
    using Fn = decltype(&cuTensorMapEncodeTiled);
    static const Fn encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) == cudaSuccess &&
                       r == cudaDriverEntryPointSuccess ? reinterpret_cast<Fn>(f) : nullptr;
    }();
    if (!encode) return cudaErrorNotSupported;
    const uint64_t pos = kv->head_major ? kv->head_dim : (uint64_t)kv->n_kv_heads * kv->head_dim;
    const uint64_t head = kv->head_major ? (uint64_t)kv->max_ctx * kv->head_dim : kv->head_dim;
    const uint64_t seq = kv->n_seqs > 1 ? kv->seq_stride : pos * kv->max_ctx;
    const cuuint64_t dims[4] = {kv->head_dim, kv->max_ctx, kv->n_kv_heads, kv->n_seqs};
    const cuuint64_t strides[3] = {pos * 2, head * 2, seq * 2};
    const cuuint32_t box[4] = {64, rows, 1, 1}, one[4] = {1, 1, 1, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<uint16_t *>(base), dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

static cudaError_t tree_merge_launch(const TreeParams &p, uint32_t rows, uint32_t n_seqs, uint32_t tile_rows, uint32_t n_sm, cudaStream_t st) {
    // a CTA per row while they all fit the SMs at once (8 each): shorter; a warp per row behind that
    const bool few = p.n_splits <= 32 && (uint64_t)rows * p.nkh * n_seqs > 8u * n_sm;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(few ? (rows + TREE_MW - 1) / TREE_MW : rows, p.nkh, n_seqs);
    cfg.blockDim = dim3(TREE_MW * 32);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return few ? cudaLaunchKernelEx(&cfg, tree_merge_warp_kernel, p, tile_rows) : cudaLaunchKernelEx(&cfg, tree_merge_kernel, p, tile_rows);
}

template <int HD, int WR, int WP>
static cudaError_t tree_go(const TreeParams &p, const CUtensorMap &km, const CUtensorMap &vm, dim3 grid, cudaStream_t st) {
    using C = TreeCfg<HD, WR, WP>;
    return tree_launch(tree_mma_kernel<HD, WR, WP>, grid, C::THREADS, C::SMEM, p.joined, st, p, km, vm);
}
template <int HD, int WR, int WP> static cudaError_t tree_cfg(int *clusters) {
    using C = TreeCfg<HD, WR, WP>;
    const cudaError_t e = cudaFuncSetAttribute(tree_mma_kernel<HD, WR, WP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    return e == cudaSuccess ? tree_clusters(tree_mma_kernel<HD, WR, WP>, C::THREADS, C::SMEM, clusters) : e;
}
cudaError_t tree_configure() {
    cudaError_t e = tree_cfg<64, 1, 4>(tree_fit[0]);
    if (e == cudaSuccess) e = tree_cfg<128, 1, 4>(tree_fit[1]);
    if (e == cudaSuccess) e = tree_cfg<256, 1, 8>(tree_fit[2]);
    if (e == cudaSuccess) e = tree_cfg<256, 2, 4>(tree_fit[3]);
    if (e == cudaSuccess) e = tree_tc_configure(tree_fit[4]);
    if (e == cudaSuccess) e = tree_weights_configure();
    // the join takes the attention kernels' split of shared memory and L1:
    // changing it costs an SM several microseconds between kernels
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tree_merge_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tree_merge_warp_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    return e;
}

}  // namespace vbs

using namespace vbs;

extern "C" {

size_t vbs_cu_tree_workspace(const vbs_cu_kv_t *kv, const vbs_cu_tree_t *t) {
    if (!tree_desc_ok(kv, t)) {
        latch_error("vbs_cu_tree_workspace: invalid arguments");
        return 0;
    }
    DevState *d = backend_current();
    if (!d) { latch_error("vbs_cu_tree_workspace: no usable device"); return 0; }
    return tree_bytes(kv, t, d->n_sm);
}

int vbs_cu_attention_tree(const vbs_cu_kv_t *kv, uint32_t layer, const vbs_cu_tree_t *t, const float *q, float *out, void *work,
                          size_t work_bytes, void *stream) {
    const uint64_t bytes = tree_desc_ok(kv, t) ? (uint64_t)kv->n_seqs * t->n_tokens * t->n_q_heads * kv->head_dim * 4 : 0;
    if (!bytes || layer >= kv->n_layers || !q || !out || !work || overlap(q, bytes, out, bytes) ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(work)) & 15)) {
        latch_error("vbs_cu_attention_tree: invalid arguments");
        return -1;
    }
    DevState *d = backend_current();
    if (!d) { latch_error("vbs_cu_attention_tree: no usable device"); return -1; }
    const TreePlan pl = tree_plan(kv, t, d->n_sm);
    if (work_bytes < pl.bytes) {
        latch_error("vbs_cu_attention_tree: workspace of %zu bytes, needs %zu", work_bytes, pl.bytes);
        return -1;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    TreeParams p = {};
    const uint64_t layer_step = (uint64_t)kv->max_ctx * kv->n_kv_heads * kv->head_dim;
    p.q = q; p.out = out;
    p.kc = kv->k + layer * layer_step;
    p.vc = kv->v + layer * layer_step;
    p.seq_stride = kv->seq_stride;
    p.pos_step = kv->head_major ? kv->head_dim : (uint64_t)kv->n_kv_heads * kv->head_dim;
    p.head_step = kv->head_major ? (uint64_t)kv->max_ctx * kv->head_dim : kv->head_dim;
    p.max_ctx = kv->max_ctx; p.nkh = kv->n_kv_heads; p.nqh = t->n_q_heads; p.G = t->n_q_heads / kv->n_kv_heads;
    p.hd = kv->head_dim; p.n_tokens = t->n_tokens; p.words = (t->n_tokens + 31) / 32; p.window = t->window;
    p.joined = pl.joined; p.ctx_limit = t->ctx_limit; p.row_tiles = pl.row_tiles; p.n_splits = pl.n_splits; p.per_split = pl.per_split;
    p.scale = t->scale; p.cap = t->softcap; p.slopes = t->slopes; p.n_ctx = t->n_ctx; p.n_tok = t->n_tok;
    p.mask = t->mask; p.q_pos = t->q_pos; p.k_pos = t->k_pos; p.k_pos_per_head = t->k_pos_per_head;
    p.weights_in = t->weights_in; p.weights_out = t->weights_out;
    uint8_t *w = static_cast<uint8_t *>(work);
    p.part_ml = reinterpret_cast<float2 *>(w + pl.ml);
    p.part_o = reinterpret_cast<float *>(w + pl.o);
    if (t->weights_out) p.lse = reinterpret_cast<float *>(w + pl.lse);
    p.g_magic = (uint32_t)((0x100000000ull + p.G - 1) / p.G);
    p.err = d->err;
    const dim3 grid(kv->n_kv_heads * pl.row_tiles, pl.n_splits, kv->n_seqs);
    const bool merge = pl.n_splits > 1 && !pl.joined;
    note_launches(1u + merge + (t->weights_out != nullptr));
    CUtensorMap km, vm, wm;
    cudaError_t e = tree_map(&km, p.kc, kv, pl.tc ? TREE_TC_SP : 64);
    if (e == cudaSuccess) e = tree_map(&vm, p.vc, kv, pl.tc ? TREE_TC_SP : 64);
    if (e == cudaSuccess && t->weights_out) e = tree_map(&wm, p.kc, kv, TREE_TC_SP);
    if (e == cudaSuccess)
        e = pl.tc                     ? tree_tc_launch(p, km, vm, kv->n_seqs, pl.tile_rows > TREE_TC_ROWS, st)
            : kv->head_dim <= 64      ? tree_go<64, 1, 4>(p, km, vm, grid, st)
            : kv->head_dim <= 128     ? tree_go<128, 1, 4>(p, km, vm, grid, st)
            : pl.tile_rows == 16      ? tree_go<256, 1, 8>(p, km, vm, grid, st)
                                      : tree_go<256, 2, 4>(p, km, vm, grid, st);
    if (e == cudaSuccess && merge)
        e = tree_merge_launch(p, pl.rows, kv->n_seqs, pl.tile_rows, d->n_sm, st);
    if (e == cudaSuccess && t->weights_out) e = tree_weights_launch(p, wm, kv->n_seqs, d->n_sm, st);
    return cuda_ok(e, "attention_tree") ? 0 : -1;
}

}  // extern "C"
