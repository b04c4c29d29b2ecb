// slots.cu -- the cache whose slots are not positions: rotary positions with
// a store into given slots, the choice of the slots that an eviction keeps,
// and the move of listed rows. (The attention over such a cache: tree.cu.)
//
// The engine keeps position t in slot t (src/vbs_host_math.h:150-159, the
// CACHE primitive) and turns every head by that one position
// (src/vbs_host_math.h:38-51, ROTARY); these kernels take both as lists.
#include "vbs_b200.h"
#include "backend.h"
#include "common.cuh"
#include "kernels.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

namespace vbs {

namespace cg = cooperative_groups;

bool kv_desc_ok(const vbs_cu_kv_t *kv) {
    if (!kv || !kv->k || !kv->v || !kv->n_layers || !kv->max_ctx || !kv->n_kv_heads || !kv->n_seqs) return false;
    if (kv->max_ctx > 0x7FFFFFFFu || !kv->head_dim || kv->head_dim % 8 || kv->head_dim > 256) return false;
    if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) & 15) return false;
    if (kv->n_kv_heads > 65535u || kv->n_seqs > 65535u) return false;
    // the sequences lie apart, and their elements' offsets have room to be added up
    const unsigned __int128 one = (unsigned __int128)kv->max_ctx * kv->n_kv_heads * kv->head_dim * kv->n_layers;
    const unsigned __int128 all = (unsigned __int128)kv->seq_stride * (kv->n_seqs - 1) + one;
    return kv->seq_stride % 8 == 0 && (kv->n_seqs == 1 || kv->seq_stride >= one) && all < ((unsigned __int128)1 << 60);
}

// ---------------------------------------------------------------------------
// Rotary positions and store.
//   q' = R q, K[slot] = fp16(R k), V[slot] = fp16(v); pair (a, b) of R:
//   (a cos - b sin, a sin + b cos) at pos[axis] * turn circles.
// The circle is 2^64 units, so position * turn is one wrapping 64-bit
// product and its top 32 bits are the fraction of a circle, to 2^-32 for
// positions up to 2^20 or so (turn itself is exact to 2^-53): the angle of a
// far position costs no 64-bit float arithmetic.
// Bound by memory: 8 bytes per query element, 6 per cached one. A thread owns
// 8 dims (4 pairs) of every head it visits, so the four sines and cosines
// are computed once and stay in registers; heads are spread over the block
// (and, for few tokens, over blockIdx.y), and the loads of ROPE_U heads are
// issued before the first is used, the first ones before the angles.
// ---------------------------------------------------------------------------
constexpr int ROPE_THREADS = 128, ROPE_U = 2;   // 4093 tokens of 64 + 16 heads of 128: 67.3 us; 256 and 4: 79.4, 128 and 4: 70.7

struct RopeParams {
    vbs_cu_rope_t r;
    const float *q, *k, *v;
    float *q_out;
    uint16_t *kc, *vc;          // layer's first element of sequence 0
    uint64_t q_stride, kv_stride, seq_stride, pos_step, head_step;
    uint32_t nqh, nkh, max_ctx, n_seqs;
    const int32_t *pos, *seq, *slot;
    uint32_t *err;
};

__device__ __forceinline__ uint4 pack_kv(const float4 &a, const float4 &b) {
    uint4 w;
    w.x = f32_to_f16_kv(a.x) | ((uint32_t)f32_to_f16_kv(a.y) << 16);
    w.y = f32_to_f16_kv(a.z) | ((uint32_t)f32_to_f16_kv(a.w) << 16);
    w.z = f32_to_f16_kv(b.x) | ((uint32_t)f32_to_f16_kv(b.y) << 16);
    w.w = f32_to_f16_kv(b.z) | ((uint32_t)f32_to_f16_kv(b.w) << 16);
    return w;
}

__global__ void __launch_bounds__(ROPE_THREADS) rope_store_kernel(const __grid_constant__ RopeParams p) {
    const uint32_t hd = p.r.head_dim, units = hd / 8, rows_blk = ROPE_THREADS / units;
    const uint32_t u = threadIdx.x % units, tok = blockIdx.x;
    uint32_t row = threadIdx.x / units + blockIdx.y * rows_blk;
    if (threadIdx.x >= rows_blk * units) return;
    const uint32_t step = rows_blk * gridDim.y, rot = p.r.rot_dim;
    const uint32_t rows = p.nqh + (p.k ? 2 * p.nkh : 0u);
    // dims of this thread: da.. and db.., 4 each; pairs are inside a float4
    // (adjacent) or across the two (halves)
    const bool turned = 8 * u < rot;
    const bool halves = turned && p.r.halves;
    const uint32_t da = halves ? 4 * u : 8 * u, db = halves ? rot / 2 + 4 * u : 8 * u + 4;

    auto src = [&](uint32_t rw) -> const float * {
        if (rw < p.nqh) return p.q + (uint64_t)tok * p.q_stride + (uint64_t)rw * hd;
        const uint32_t h = rw - p.nqh;
        return h < p.nkh ? p.k + (uint64_t)tok * p.kv_stride + (uint64_t)h * hd
                         : p.v + (uint64_t)tok * p.kv_stride + (uint64_t)(h - p.nkh) * hd;
    };
    float4 xa[ROPE_U], xb[ROPE_U];
    auto fetch = [&](uint32_t r0) {
#pragma unroll
        for (int j = 0; j < ROPE_U; ++j) {
            const uint32_t rw = r0 + j * step;
            if (rw >= rows) continue;   // (a token without a slot is read too: its slot is not waited for)
            const float *s = src(rw);
            xa[j] = *reinterpret_cast<const float4 *>(s + da);
            xb[j] = *reinterpret_cast<const float4 *>(s + db);
        }
    };
    fetch(row);
    int32_t slot = -1;
    uint64_t at0 = 0;
    if (p.k) {
        slot = p.slot[tok];
        const int32_t s = p.seq ? p.seq[tok] : 0;
        if (slot != -1 && (slot < 0 || slot >= (int32_t)p.max_ctx || s < 0 || s >= (int32_t)p.n_seqs)) {
            if (threadIdx.x == 0) dev_flag_error(p.err, DERR_BAD_ARG);
            slot = -1;
        }
        if (slot >= 0) at0 = (uint64_t)s * p.seq_stride + (uint64_t)slot * p.pos_step;
    }
    float c[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = 1.f;
        sn[i] = 0.f;
        if (turned) {
            const uint32_t pr = 4 * u + i;
            const int64_t ps = p.pos[(uint64_t)tok * p.r.n_axes + p.r.axis[pr]];
            const int32_t frac = (int32_t)(((uint64_t)ps * p.r.turn[pr]) >> 32);   // of a circle, in 2^-32
            sincospif((float)frac * 0x1p-31f, &sn[i], &c[i]);
        }
    }
    for (; row < rows; row += step * ROPE_U, fetch(row)) {
#pragma unroll
        for (int j = 0; j < ROPE_U; ++j) {
            const uint32_t rw = row + j * step;
            if (rw >= rows || (rw >= p.nqh && slot < 0)) continue;
            const float4 a = xa[j], b = xb[j];
            float4 ya = a, yb = b;
            if (turned && rw < p.nqh + p.nkh) {
                if (halves) {
                    ya = make_float4(a.x * c[0] - b.x * sn[0], a.y * c[1] - b.y * sn[1], a.z * c[2] - b.z * sn[2],
                                     a.w * c[3] - b.w * sn[3]);
                    yb = make_float4(a.x * sn[0] + b.x * c[0], a.y * sn[1] + b.y * c[1], a.z * sn[2] + b.z * c[2],
                                     a.w * sn[3] + b.w * c[3]);
                } else {
                    ya = make_float4(a.x * c[0] - a.y * sn[0], a.x * sn[0] + a.y * c[0], a.z * c[1] - a.w * sn[1],
                                     a.z * sn[1] + a.w * c[1]);
                    yb = make_float4(b.x * c[2] - b.y * sn[2], b.x * sn[2] + b.y * c[2], b.z * c[3] - b.w * sn[3],
                                     b.z * sn[3] + b.w * c[3]);
                }
            }
            if (rw < p.nqh) {
                float *d = p.q_out + ((uint64_t)tok * p.nqh + rw) * hd;
                *reinterpret_cast<float4 *>(d + da) = ya;
                *reinterpret_cast<float4 *>(d + db) = yb;
            } else {
                const uint32_t h = rw - p.nqh;
                uint16_t *d = (h < p.nkh ? p.kc + at0 + h * p.head_step : p.vc + at0 + (h - p.nkh) * p.head_step);
                const uint4 w = pack_kv(ya, yb);
                if (halves) {   // the two quarters of the unit are apart
                    *reinterpret_cast<uint2 *>(d + da) = make_uint2(w.x, w.y);
                    *reinterpret_cast<uint2 *>(d + db) = make_uint2(w.z, w.w);
                } else {
                    *reinterpret_cast<uint4 *>(d + da) = w;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Choice of the slots to keep: exact selection of the r-th highest of m scores
// per list, ties to the lowest index, result ascending.
// Scores become 32-bit keys in the scores' order:
//  1. a histogram of the keys' top 12 bits (sign, exponent and three mantissa
//     bits spread accumulated weights over a hundred bins or more); the bin
//     that holds the r-th highest is known after it.
//  2. the scores again (out of L2 now): what lies above that bin becomes a bit
//     per key, what lies in it a short list, on which two more histograms (10
//     bits each) find the key; the list's keys above it join the bits, those
//     equal to it get bits of their own. A bin with more than SEL_CAND keys
//     (many equal scores) is searched in place instead of from the list.
//  3. the kept slots are written from the bits, 32 keys a word: their places
//     are the counts of kept slots before them.
// Every warp owns a run of consecutive keys and visits only those, so the
// counts per warp are all that has to be scanned. Reading twice instead of
// keeping the keys in shared memory leaves room for three CTAs per SM (40
// registers) instead of two: the steps are short and wait for one another, and
// other CTAs fill the waits (1024 lists of up to 16384: 77.6 us with the keys
// kept). Bound by instruction issue: 71% of the schedulers' cycles there. A cluster
// of 2, 4 or 8 CTAs shares a list only where there are few long ones:
// histograms and counts are then read from the other CTAs' shared memory.
// ---------------------------------------------------------------------------
constexpr uint32_t SEL_THREADS = 512, SEL_WARPS = SEL_THREADS / 32, SEL_CHUNK_MAX = 393216;
constexpr uint32_t SEL_N_MAX = 8 * SEL_CHUNK_MAX;
constexpr uint32_t SEL_BINS = 4096, SEL_BINS2 = 1024, SEL_CAND = 2048;
constexpr int SEL_U = 8;            // keys in flight per thread
// shared memory: state, histograms (12 bits, then 2 x 10), the list, the bits
constexpr uint32_t SEL_STATE = 512, SEL_FIXED = SEL_STATE + (SEL_BINS + 2 * SEL_BINS2) * 4 + SEL_CAND * 8;

// a bit per key, runs of whole 128s
__host__ __device__ constexpr uint32_t sel_words(uint32_t chunk) { return ((chunk + SEL_WARPS - 1) / SEL_WARPS + 127) / 128 * 4 * SEL_WARPS; }
struct SelectParams {
    const float *scores;
    uint64_t stride;
    uint32_t n_seqs, n_kv_heads, n_limit, keep, first, recent, chunk_max;
    const int32_t *n;
    int32_t *idx, *count;
    uint32_t *err;
};

__device__ __forceinline__ uint32_t score_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.f);               // -0 is 0
    return f != f ? 0u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);   // NaN: below everything
}

constexpr uint32_t SEL_LOWEST = 0x007FFFFFu;   // the key of -inf
__device__ __forceinline__ float score_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Adds 1 to a bin per lane (bin ~0: none); all lanes of the warp call it. The
// lanes that agree with the first make one addition (equal scores).
__device__ __forceinline__ void hist_add(uint32_t *h, uint32_t bin) {
    const uint32_t b0 = __shfl_sync(0xffffffffu, bin, 0);
    const uint32_t same = __ballot_sync(0xffffffffu, bin == b0);
    const bool first = (threadIdx.x & 31) == 0;
    if (bin != 0xFFFFFFFFu && (first || bin != b0)) atomicAdd(&h[bin], first ? (uint32_t)__popc(same) : 1u);
}

// Sum over the lanes up to this one.
__device__ __forceinline__ uint32_t warp_upto(uint32_t x) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= (uint32_t)o) x += y;
    }
    return x;
}

// The bin of `bins` (PER per thread) that holds the r-th highest, and how many
// lie above it, summed over the cluster's histograms; in st[0], st[1]. st[2..]:
// scratch. The block is synchronised on return.
template <int PER>
__device__ __forceinline__ void hist_find(cg::cluster_group &cluster, uint32_t *h, uint32_t r, uint32_t *st) {
    const uint32_t C = cluster.num_blocks(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (C > 1) cluster.sync();
    else __syncthreads();
    uint32_t own[PER], sum = 0;   // bins from the highest down
#pragma unroll
    for (int j = 0; j < PER; ++j) own[j] = 0;
    for (uint32_t c = 0; c < C; ++c) {
        const uint32_t *o = C > 1 ? cluster.map_shared_rank(h, c) : h;
#pragma unroll
        for (int j = 0; j < PER; ++j) own[j] += o[PER * SEL_THREADS - 1 - (PER * tid + j)];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += own[j];
    const uint32_t x = warp_upto(sum);
    if (lane == 31) st[2 + warp] = x;
    __syncthreads();
    uint32_t above = x - sum;
    for (uint32_t w = 0; w < warp; ++w) above += st[2 + w];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (above < r && r <= above + own[j]) { st[0] = PER * SEL_THREADS - 1 - (PER * tid + j); st[1] = above; }
        above += own[j];
    }
    __syncthreads();
}

__global__ void __launch_bounds__(SEL_THREADS) cache_select_kernel(const SelectParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t list = blockIdx.x / C, s = list / p.n_kv_heads % p.n_seqs;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t *st = reinterpret_cast<uint32_t *>(smem);   // [0,18) hist_find, 18 list length, 19 kept in all, 20 ties in all
    uint32_t *n_sure = st + 24, *n_tie = n_sure + SEL_WARPS;   // per warp
    uint32_t *h0 = reinterpret_cast<uint32_t *>(smem + SEL_STATE), *h1 = h0 + SEL_BINS, *h2 = h1 + SEL_BINS2;
    uint2 *cand = reinterpret_cast<uint2 *>(h2 + SEL_BINS2);   // key, place
    uint32_t *w_sure = reinterpret_cast<uint32_t *>(cand + SEL_CAND), *w_tie = w_sure + sel_words(p.chunk_max);

    const int32_t n_in = p.n[s];
    int32_t *out = p.idx + (uint64_t)list * p.keep;
    if (n_in < 0 || (uint32_t)n_in > p.n_limit) {              // the whole cluster takes the same way
        if (tid == 0 && rank == 0) dev_flag_error(p.err, DERR_BAD_ARG);
        return;
    }
    const uint32_t n = (uint32_t)n_in;
    if (list % p.n_kv_heads == 0 && list / p.n_kv_heads < p.n_seqs && rank == 0 && tid == 0)
        p.count[s] = (int32_t)min(n, p.keep);
    if (n <= p.keep) {
        for (uint32_t i = rank * SEL_THREADS + tid; i < p.keep; i += C * SEL_THREADS) out[i] = i < n ? (int32_t)i : -1;
        return;
    }
    // n > keep >= first + recent: the scores between compete for r places
    const uint32_t m0 = p.first, m1 = n - p.recent;
    uint32_t r = p.keep - p.first - p.recent;
    const uint32_t chunk = (n + C - 1) / C, c0 = min(n, rank * chunk), len = min(n, c0 + chunk) - c0;
    const uint32_t seg = ((len + SEL_WARPS - 1) / SEL_WARPS + 127) / 128 * 128;   // keys per warp
    const uint32_t s0 = min(len, warp * seg), s1 = min(len, s0 + seg);
    const float *src = p.scores + (uint64_t)list * p.stride + c0;
    const uint32_t f0 = m0 > c0 ? m0 - c0 : 0u, f1 = m1 > c0 ? m1 - c0 : 0u;   // [f0, f1) of this part compete

    for (uint32_t i = tid; i < SEL_BINS + 2 * SEL_BINS2; i += SEL_THREADS) h0[i] = 0u;
    if (tid < 24 + 2 * SEL_WARPS) st[tid] = 0u;
    __syncthreads();
    // 4 groups of 32 keys: whole, all of them competing; or at an edge
    auto whole = [&](uint32_t i0) { return i0 >= f0 && i0 + 128 <= f1 && i0 + 128 <= s1; };
    // 1. the keys' top 12 bits
    for (uint32_t i0 = s0; i0 < s1; i0 += 32 * SEL_U) {
        float v[SEL_U];
#pragma unroll
        for (int u = 0; u < SEL_U; ++u) v[u] = i0 + 32 * u + lane < s1 ? __ldg(src + i0 + 32 * u + lane) : 0.f;
#pragma unroll
        for (int w = 0; w < SEL_U; w += 4) {
            if (whole(i0 + 32 * w)) {
#pragma unroll
                for (int u = w; u < w + 4; ++u) hist_add(h0, score_key(v[u]) >> 20);
            } else {
#pragma unroll 1
                for (int u = 0; u < 4; ++u) {
                    const uint32_t i = i0 + 32 * (w + u) + lane, k = score_key(u == 0 ? v[w] : u == 1 ? v[w + 1] : u == 2 ? v[w + 2] : v[w + 3]);
                    hist_add(h0, i < s1 && i >= f0 && i < f1 ? k >> 20 : 0xFFFFFFFFu);
                }
            }
        }
    }
    uint32_t T = 0xFFFFFFFFu, need = 0;   // kept: above T, and the first `need` equal to T
    uint32_t b0 = SEL_BINS;               // r 0: nothing of them is kept
    if (r) {
        hist_find<SEL_BINS / SEL_THREADS>(cluster, h0, r, st);
        b0 = st[0];
        r -= st[1];
    }
    // 2. above the bin (or not competing): a bit; in it: listed
    // the bin's lowest score and the lowest above it: floats compare as their
    // keys do. Bin 0 holds NaN alone, above it is all that compares; above the
    // bin of +inf, or with no bin, nothing (a comparison with NaN)
    const float f_lo = score_of(max(b0 << 20, SEL_LOWEST)), f_up = b0 < SEL_BINS - 1 ? score_of(max((b0 + 1) << 20, SEL_LOWEST)) : NAN;
    const bool in_nan = b0 == 0, none = b0 >= SEL_BINS;
    for (uint32_t j0 = s0; j0 < s1; j0 += 32 * SEL_U) {
        float v[SEL_U];
#pragma unroll
        for (int u = 0; u < SEL_U; ++u) v[u] = j0 + 32 * u + lane < s1 ? __ldg(src + j0 + 32 * u + lane) : 0.f;
#pragma unroll
        for (int x = 0; x < SEL_U; x += 4) {
            const uint32_t i0 = j0 + 32 * x;
            if (i0 >= s1) break;
            bool in[4], any = false;
            uint32_t g[4];
            const bool all_in = whole(i0);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                bool sure = v[x + u] >= f_up;
                in[u] = !sure && (in_nan || v[x + u] >= f_lo) && !none;
                if (!all_in) {
                    const uint32_t i = i0 + 32 * u + lane;
                    const bool comp = i >= f0 && i < f1;
                    sure = i < s1 && (!comp || sure);
                    in[u] = in[u] && i < s1 && comp;
                }
                g[u] = __ballot_sync(0xffffffffu, sure);
                any |= in[u];
            }
            if (lane == 0) {   // runs are whole 128s
                *reinterpret_cast<uint4 *>(&w_sure[i0 >> 5]) = make_uint4(g[0], g[1], g[2], g[3]);
                *reinterpret_cast<uint4 *>(&w_tie[i0 >> 5]) = make_uint4(0u, 0u, 0u, 0u);
            }
            if (any) {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (in[u]) {
                        const uint32_t at = atomicAdd(&st[18], 1u);
                        if (at < SEL_CAND) cand[at] = make_uint2(score_key(v[x + u]), i0 + 32 * u + lane);
                    }
            }
            __syncwarp();
        }
    }
    __syncthreads();
    const uint32_t nc = st[18];
    const bool listed = nc <= SEL_CAND;
    // the keys of the bin, from the list or in place; whole warps call f
    auto each = [&](auto f) {
        if (listed) {
            for (uint32_t j0 = warp * 32; j0 < nc; j0 += SEL_THREADS) {
                const uint2 e = j0 + lane < nc ? cand[j0 + lane] : make_uint2(0u, 0u);
                f(j0 + lane < nc, e.y, e.x);
            }
        } else {
            for (uint32_t i0 = s0; i0 < s1; i0 += 32) {
                const uint32_t i = i0 + lane, k = i < s1 ? score_key(__ldg(src + i)) : 0u;
                f(i < s1 && i >= f0 && i < f1 && k >> 20 == b0, i, k);
            }
        }
    };
    if (r) {
        each([&](bool c, uint32_t, uint32_t k) { hist_add(h1, c ? (k >> 10) & 1023u : 0xFFFFFFFFu); });
        hist_find<SEL_BINS2 / SEL_THREADS>(cluster, h1, r, st);
        const uint32_t b1 = st[0];
        r -= st[1];
        each([&](bool c, uint32_t, uint32_t k) { hist_add(h2, c && ((k >> 10) & 1023u) == b1 ? k & 1023u : 0xFFFFFFFFu); });
        hist_find<SEL_BINS2 / SEL_THREADS>(cluster, h2, r, st);
        T = (b0 << 20) | (b1 << 10) | st[0];
        need = r - st[1];
        each([&](bool c, uint32_t i, uint32_t k) {
            if (c && k >= T) atomicOr((k > T ? w_sure : w_tie) + (i >> 5), 1u << (i & 31));
        });
    }
    __syncthreads();
    // what each warp's run keeps for certain, and its ties
    uint32_t at = 0, ties = 0;
    for (uint32_t g = s0 / 32 + lane; s0 < s1 && g < (s1 + 127) / 128 * 4; g += 32) {   // (a run may be empty)
        at += __popc(w_sure[g]);
        ties += __popc(w_tie[g]);
    }
    at = __reduce_add_sync(0xffffffffu, at);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) {
        n_sure[warp] = at;
        n_tie[warp] = ties;
    }
    if (C > 1) {
        if (lane == 0) {
            atomicAdd(&st[19], at);
            atomicAdd(&st[20], ties);
        }
        cluster.sync();
    } else {
        __syncthreads();
    }
    at = ties = 0;   // before this warp's run
    for (uint32_t c = 0; c < rank; ++c) {
        const uint32_t *o = cluster.map_shared_rank(st, c);
        at += o[19];
        ties += o[20];
    }
    for (uint32_t w = 0; w < warp; ++w) {
        at += n_sure[w];
        ties += n_tie[w];
    }
    // 3. out: n > keep, so all places get filled. A lane per word of 32 keys
    // (short runs: per byte) writes its kept slots one after the other. (A
    // lane per key, a word at a time, took 13.6 us of 71.7 for 1024 lists of
    // up to 16384.)
    at += min(ties, need);
    const bool tied = n_tie[warp] != 0;
    const uint32_t w1 = s0 < s1 ? (s1 + 31) / 32 : 0u, sh = seg <= 256 ? 2u : 0u, width = 32u >> sh, first = (lane & ((1u << sh) - 1)) * width;
    const uint32_t span = 0xFFFFFFFFu >> (32 - width);
    for (uint32_t g0 = s0 / 32; g0 < w1; g0 += 32u >> sh) {
        const uint32_t g = g0 + (lane >> sh);
        uint32_t bits = g < w1 ? (w_sure[g] >> first) & span : 0u;
        if (tied) {   // the first of them, up to `need`
            uint32_t e = g < w1 ? (w_tie[g] >> first) & span : 0u;
            const uint32_t mine = __popc(e), upto = warp_upto(mine);
            const uint32_t before = ties + upto - mine, take = before < need ? min(mine, need - before) : 0u;
            for (uint32_t k = mine; k > take; --k) e &= ~(0x80000000u >> __clz(e));
            bits |= e;
            ties += __shfl_sync(0xffffffffu, upto, 31);
        }
        const uint32_t mine = __popc(bits), upto = warp_upto(mine);
        int32_t *o = out + at + (upto - mine);
        const int32_t k0 = (int32_t)(c0 + 32 * g + first);
        for (; bits; bits &= bits - 1) *o++ = k0 + __ffs(bits) - 1;
        __syncwarp();
        at += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (C == 1) return;
    cluster.sync();   // nobody leaves while its shared memory is read
}

// ---------------------------------------------------------------------------
// Row moves. Bound by memory: every row is read once and written once.
// Apart: a thread moves 16-byte pieces of K and V of GX_U rows, all loads
// before the first store. In place: rows only move down, so a CTA takes its
// list in ascending batches (all of a batch's loads, a barrier, its stores);
// the pieces of a row are independent of one another, so slices of the row
// go to CTAs of their own. Lists of up to GA_WARP_MAX entries (an accepted
// branch) take a warp each: 2048 lists of 5 rows of 256 bytes 9.7 us with a
// CTA per list.
// ---------------------------------------------------------------------------
constexpr uint32_t GA_THREADS = 256, GA_U = 4, GA_WARP_MAX = 64;
constexpr uint32_t GX_THREADS = 128, GX_U = 2;   // apart: 90.4 us for 32 x 8 lists of 2048 of 8192 rows of 256 bytes (256 and 4: 129, 256 and 2: 96.2)

struct GatherSide {
    uint16_t *k, *v;
    uint64_t seq_stride, layer_step, pos_step, head_step;
    uint32_t max_ctx;
};
struct GatherParams {
    GatherSide src, dst;
    vbs_cu_gather_t g;
    uint32_t n_seqs, n_kv_heads, cpr;   // 16-byte pieces per row
    uint32_t slice;                     // in place: pieces per CTA
    uint32_t *err;
};

struct GatherList {
    const int32_t *idx;
    uint32_t n;
    int64_t src0, dst0;
    uint64_t so, dof;        // element offsets of (sequence, layer, head) in the caches
    uint64_t aux_s, aux_d;   // of the list's row in the weights and positions
};

__device__ __forceinline__ bool gather_list(const GatherParams &p, uint32_t list, GatherList &l) {
    const uint32_t h = list % p.n_kv_heads, s = list / p.n_kv_heads % p.n_seqs, layer = list / p.n_kv_heads / p.n_seqs;
    const int32_t n = p.g.count[s];
    l.src0 = p.g.src_base ? p.g.src_base[s] : 0;
    l.dst0 = p.g.dst_base ? p.g.dst_base[s] : 0;
    l.idx = p.g.idx + layer * p.g.layer_stride + s * p.g.seq_stride + h * p.g.head_stride;
    l.n = n < 0 ? 0u : (uint32_t)n;
    l.so = s * p.src.seq_stride + layer * p.src.layer_step + h * p.src.head_step;
    l.dof = s * p.dst.seq_stride + layer * p.dst.layer_step + h * p.dst.head_step;
    l.aux_s = (uint64_t)list * p.src.max_ctx;
    l.aux_d = (uint64_t)list * p.dst.max_ctx;
    if (n < 0 || (uint32_t)n > p.g.n_max || l.dst0 < 0 || l.dst0 + n > (int64_t)p.dst.max_ctx) {
        if ((threadIdx.x & 31) == 0) dev_flag_error(p.err, DERR_BAD_ARG);
        return false;
    }
    return true;
}

__global__ void __launch_bounds__(GX_THREADS) gather_apart_kernel(const __grid_constant__ GatherParams p, uint32_t nblk) {
    // the heads of the same rows are neighbours in launch order: in the
    // engine's order their rows are neighbours in memory
    const uint32_t h = blockIdx.x % p.n_kv_heads, x = blockIdx.x / p.n_kv_heads;
    const uint32_t list = x / nblk * p.n_kv_heads + h, rp = GX_THREADS / p.cpr;
    GatherList l;
    if (!gather_list(p, list, l)) return;
    const uint32_t ch = threadIdx.x % p.cpr, r0 = x % nblk * (rp * GX_U) + threadIdx.x / p.cpr;
    if (threadIdx.x >= rp * p.cpr) return;
    int64_t from[GX_U];
    uint4 k[GX_U], v[GX_U];
#pragma unroll
    for (uint32_t u = 0; u < GX_U; ++u) {
        const uint32_t i = r0 + u * rp;
        from[u] = i < l.n ? l.src0 + l.idx[i] : -1;
        if (i < l.n && (from[u] < 0 || from[u] >= (int64_t)p.src.max_ctx)) {
            dev_flag_error(p.err, DERR_BAD_ARG);
            from[u] = -1;
        }
    }
#pragma unroll
    for (uint32_t u = 0; u < GX_U; ++u) {
        if (from[u] < 0) continue;
        const uint64_t o = l.so + (uint64_t)from[u] * p.src.pos_step + ch * 8;
        k[u] = *reinterpret_cast<const uint4 *>(p.src.k + o);
        v[u] = *reinterpret_cast<const uint4 *>(p.src.v + o);
    }
#pragma unroll
    for (uint32_t u = 0; u < GX_U; ++u) {
        if (from[u] < 0) continue;
        const uint64_t to = (uint64_t)l.dst0 + r0 + u * rp;
        const uint64_t o = l.dof + to * p.dst.pos_step + ch * 8;
        *reinterpret_cast<uint4 *>(p.dst.k + o) = k[u];
        *reinterpret_cast<uint4 *>(p.dst.v + o) = v[u];
        if (ch == 0) {
            if (p.g.weights_dst) p.g.weights_dst[l.aux_d + to] = p.g.weights_src[l.aux_s + from[u]];
            if (p.g.pos_dst) p.g.pos_dst[l.aux_d + to] = p.g.pos_src[l.aux_s + from[u]];
        }
    }
}

__global__ void __launch_bounds__(GA_THREADS) gather_inplace_kernel(const __grid_constant__ GatherParams p) {
    GatherList l;
    if (!gather_list(p, blockIdx.x, l)) return;
    // the list first: ascending, and nothing moves up
    int bad = 0;
    for (uint32_t i = threadIdx.x; i < l.n; i += GA_THREADS) {
        const int64_t f = l.src0 + l.idx[i];
        bad |= f < l.dst0 + i || f >= (int64_t)p.src.max_ctx || (i && l.idx[i] <= l.idx[i - 1]);
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) dev_flag_error(p.err, DERR_BAD_ARG);
        return;
    }
    const uint32_t s0 = blockIdx.y * p.slice, w = min(p.slice, p.cpr - s0);   // this CTA's pieces of a row
    const uint32_t rp = GA_THREADS / w, ch = s0 + threadIdx.x % w, rr = threadIdx.x / w;
    const bool on = threadIdx.x < rp * w;
    for (uint32_t b = 0; b < l.n; b += rp * GA_U) {
        int64_t from[GA_U];
        uint4 k[GA_U], v[GA_U];
        float wt[GA_U];
        int32_t ps[GA_U];
#pragma unroll
        for (uint32_t u = 0; u < GA_U; ++u) {
            const uint32_t i = b + rr + u * rp;
            from[u] = on && i < l.n ? l.src0 + l.idx[i] : -1;
            if (from[u] == l.dst0 + i) from[u] = -1;   // stays where it is
            if (from[u] < 0) continue;
            const uint64_t o = l.so + (uint64_t)from[u] * p.src.pos_step + ch * 8;
            k[u] = *reinterpret_cast<const uint4 *>(p.src.k + o);
            v[u] = *reinterpret_cast<const uint4 *>(p.src.v + o);
            if (ch == 0) {
                if (p.g.weights_dst) wt[u] = p.g.weights_src[l.aux_s + from[u]];
                if (p.g.pos_dst) ps[u] = p.g.pos_src[l.aux_s + from[u]];
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < GA_U; ++u) {
            if (from[u] < 0) continue;
            const uint64_t to = (uint64_t)l.dst0 + b + rr + u * rp;
            const uint64_t o = l.dof + to * p.dst.pos_step + ch * 8;
            *reinterpret_cast<uint4 *>(p.dst.k + o) = k[u];
            *reinterpret_cast<uint4 *>(p.dst.v + o) = v[u];
            if (ch == 0) {
                if (p.g.weights_dst) p.g.weights_dst[l.aux_d + to] = wt[u];
                if (p.g.pos_dst) p.g.pos_dst[l.aux_d + to] = ps[u];
            }
        }
        // no barrier: the next batch reads rows behind all that this one
        // writes, and writes only behind its own barrier
    }
}

// In place, short lists: a warp per list, pieces of K and V in ascending rows,
// 8 per lane at a time.
__global__ void __launch_bounds__(GA_THREADS) gather_inplace_warp_kernel(const __grid_constant__ GatherParams p, uint32_t lists) {
    const uint32_t list = blockIdx.x * (GA_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    GatherList l;
    if (list >= lists || !gather_list(p, list, l)) return;
    bool bad = false;
    for (uint32_t i = lane; i < l.n; i += 32) {
        const int64_t f = l.src0 + l.idx[i];
        bad |= f < l.dst0 + i || f >= (int64_t)p.src.max_ctx || (i && l.idx[i] <= l.idx[i - 1]);
    }
    if (__any_sync(0xffffffffu, bad)) {
        if (lane == 0) dev_flag_error(p.err, DERR_BAD_ARG);
        return;
    }
    const uint32_t per = 2 * p.cpr, total = l.n * per;   // pieces: row, then K's and V's
    for (uint32_t k0 = 0; k0 < total; k0 += 32 * 8) {
        uint4 v[8];
        float w[8];
        int32_t ps[8];
        int64_t from[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const uint32_t k = k0 + 32 * u + lane, i = k / per, c = k - i * per;
            from[u] = k < total ? l.src0 + l.idx[i] : -1;
            if (from[u] == l.dst0 + i) from[u] = -1;   // stays where it is
            if (from[u] < 0) continue;
            const uint64_t o = l.so + (uint64_t)from[u] * p.src.pos_step;
            v[u] = *reinterpret_cast<const uint4 *>((c < p.cpr ? p.src.k + o + c * 8 : p.src.v + o + (c - p.cpr) * 8));
            if (c == 0) {
                if (p.g.weights_dst) w[u] = p.g.weights_src[l.aux_s + from[u]];
                if (p.g.pos_dst) ps[u] = p.g.pos_src[l.aux_s + from[u]];
            }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (from[u] < 0) continue;
            const uint32_t k = k0 + 32 * u + lane, i = k / per, c = k - i * per;
            const uint64_t to = (uint64_t)l.dst0 + i, o = l.dof + to * p.dst.pos_step;
            *reinterpret_cast<uint4 *>((c < p.cpr ? p.dst.k + o + c * 8 : p.dst.v + o + (c - p.cpr) * 8)) = v[u];
            if (c == 0) {
                if (p.g.weights_dst) p.g.weights_dst[l.aux_d + to] = w[u];
                if (p.g.pos_dst) p.g.pos_dst[l.aux_d + to] = ps[u];
            }
        }
    }
}

cudaError_t slots_configure() {
    return cudaFuncSetAttribute(cache_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)(SEL_FIXED + 8 * sel_words(SEL_CHUNK_MAX)));
}

static GatherSide gather_side(const vbs_cu_kv_t *kv) {
    GatherSide s = {};
    s.k = kv->k;
    s.v = kv->v;
    s.seq_stride = kv->seq_stride;
    s.layer_step = (uint64_t)kv->max_ctx * kv->n_kv_heads * kv->head_dim;
    s.pos_step = kv->head_major ? kv->head_dim : (uint64_t)kv->n_kv_heads * kv->head_dim;
    s.head_step = kv->head_major ? (uint64_t)kv->max_ctx * kv->head_dim : kv->head_dim;
    s.max_ctx = kv->max_ctx;
    return s;
}

// Elements from the first of a cache to behind its last.
static uint64_t kv_extent(const vbs_cu_kv_t *kv) {
    return (uint64_t)(kv->n_seqs - 1) * kv->seq_stride +
           (uint64_t)kv->n_layers * kv->max_ctx * kv->n_kv_heads * kv->head_dim;
}

bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + nb && y < x + na;
}

// Any of n rows of `row` bytes, `stride` bytes apart from a, and nb bytes from b.
static bool rows_overlap(const void *a, uint64_t n, unsigned __int128 stride, uint64_t row, const void *b, uint64_t nb) {
    const unsigned __int128 x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (!a || !b) return false;
    const unsigned __int128 i = y < x + row ? 0 : (y - x - row) / stride + 1;   // the first row that ends behind b
    return i < n && x + i * stride < y + nb;
}

}  // namespace vbs

using namespace vbs;

extern "C" {

int vbs_cu_rope_init(vbs_cu_rope_t *r, uint32_t head_dim, uint32_t rot_dim, uint32_t halves, float theta,
                     const float *freq_factors, uint32_t n_axes, const uint32_t *sections, uint32_t interleaved) {
    if (!r || !head_dim || head_dim % 8 || head_dim > 256 || !rot_dim || rot_dim % 8 || rot_dim > head_dim ||
        !(theta > 0.f) || !std::isfinite(theta) || n_axes < 1 || n_axes > 4 || (n_axes > 1 && !sections)) {
        latch_error("vbs_cu_rope_init: invalid arguments");
        return -1;
    }
    const uint32_t pairs = rot_dim / 2;
    uint64_t sum = 0;
    for (uint32_t a = 0; sections && a < n_axes; ++a) sum += sections[a];
    if (sections && sum != pairs) {
        latch_error("vbs_cu_rope_init: sections of %llu pairs for %u", (unsigned long long)sum, pairs);
        return -1;
    }
    vbs_cu_rope_t o = {};
    o.head_dim = head_dim;
    o.rot_dim = rot_dim;
    o.n_axes = n_axes;
    o.halves = halves ? 1u : 0u;
    uint32_t a = 0, left = sections ? sections[0] : pairs;
    for (uint32_t p = 0; p < pairs; ++p) {
        double f = std::pow((double)theta, -2.0 * (double)p / (double)rot_dim);
        if (freq_factors) f /= (double)freq_factors[p];
        // circles per position in 2^-64: the fraction alone matters, and a
        // double below 1 scales to an exact integer part
        double c = f / (2.0 * M_PI);
        if (!std::isfinite(c)) {
            latch_error("vbs_cu_rope_init: frequency factor %u is not usable", p);
            return -1;
        }
        c -= std::floor(c);
        const double hi = std::floor(c * 4294967296.0);
        const double lo = (c * 4294967296.0 - hi) * 4294967296.0;
        o.turn[p] = ((uint64_t)hi << 32) + (uint64_t)lo;
        if (interleaved && sections) {
            const uint32_t ax = p % n_axes;
            o.axis[p] = (uint8_t)((uint64_t)p < (uint64_t)n_axes * sections[ax] ? ax : 0u);
        } else {
            while (!left) left = sections[++a];   // the sections' sum is the pairs: a stays below n_axes
            o.axis[p] = (uint8_t)a;
            --left;
        }
    }
    *r = o;
    return 0;
}

int vbs_cu_rope_store(const vbs_cu_rope_t *r, const vbs_cu_kv_t *kv, uint32_t layer, const float *q, uint64_t q_stride,
                      float *q_out, uint32_t n_q_heads, const float *k, const float *v, uint64_t kv_stride,
                      uint32_t n_tokens, const int32_t *pos, const int32_t *seq, const int32_t *slot, void *stream) {
    const bool turn = n_q_heads != 0, store = k || v;
    bool ok = r && r->head_dim && r->head_dim % 8 == 0 && r->head_dim <= 256 && r->rot_dim && r->rot_dim % 8 == 0 &&
              r->rot_dim <= r->head_dim && r->n_axes >= 1 && r->n_axes <= 4 && pos && (turn || store);
    for (uint32_t p = 0; ok && p < r->rot_dim / 2; ++p) ok = r->axis[p] < r->n_axes;
    if (ok && turn) {
        const uint64_t row = (uint64_t)n_q_heads * r->head_dim;
        if (!q_stride) q_stride = row;
        ok = q && q_out && n_q_heads <= 65535u && q_stride >= row && q_stride % 4 == 0 && (q != q_out || q_stride == row) &&
             !((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out)) & 15);
    }
    if (ok && store) {
        ok = k && v && slot && kv_desc_ok(kv) && layer < kv->n_layers && kv->head_dim == r->head_dim;
        if (ok) {
            const uint64_t row = (uint64_t)kv->n_kv_heads * kv->head_dim;
            if (!kv_stride) kv_stride = row;
            ok = kv_stride >= row && kv_stride % 4 == 0 &&
                 !((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15);
        }
    }
    if (ok && turn) {   // queries are written while other tokens' inputs are read
        const uint64_t qrow = (uint64_t)n_q_heads * r->head_dim * 4, krow = store ? (uint64_t)kv->n_kv_heads * r->head_dim * 4 : 0;
        const uint64_t all = n_tokens * qrow;
        ok = (q == q_out || !rows_overlap(q, n_tokens, (unsigned __int128)q_stride * 4, qrow, q_out, all)) &&
             (!store || (!rows_overlap(k, n_tokens, (unsigned __int128)kv_stride * 4, krow, q_out, all) &&
                         !rows_overlap(v, n_tokens, (unsigned __int128)kv_stride * 4, krow, q_out, all)));
    }
    if (!ok) {
        latch_error("vbs_cu_rope_store: invalid arguments");
        return -1;
    }
    DevState *d = backend_current();
    if (!d) { latch_error("vbs_cu_rope_store: no usable device"); return -1; }
    if (!n_tokens) return 0;
    RopeParams p = {};
    p.r = *r;
    p.q = q; p.q_out = q_out; p.q_stride = q_stride; p.nqh = n_q_heads;
    p.pos = pos; p.err = d->err;
    if (store) {
        const GatherSide c = gather_side(kv);
        p.k = k; p.v = v; p.kv_stride = kv_stride; p.nkh = kv->n_kv_heads;
        p.kc = c.k + layer * c.layer_step; p.vc = c.v + layer * c.layer_step;
        p.seq_stride = c.seq_stride; p.pos_step = c.pos_step; p.head_step = c.head_step;
        p.max_ctx = kv->max_ctx; p.n_seqs = kv->n_seqs; p.seq = seq; p.slot = slot;
    }
    // few tokens: a token's heads over several CTAs, until the SMs are covered
    const uint32_t rows = p.nqh + 2 * p.nkh, blk = ROPE_THREADS / (r->head_dim / 8);
    const uint32_t most = (rows + blk - 1) / blk, want = ((uint32_t)d->n_sm * 2 + n_tokens - 1) / n_tokens;
    const dim3 grid(n_tokens, std::max(1u, std::min(most, want)));
    note_launches(1);
    rope_store_kernel<<<grid, ROPE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return cuda_ok(cudaGetLastError(), "rope_store") ? 0 : -1;
}

int vbs_cu_cache_select(const float *scores, uint64_t stride, uint32_t n_layers, uint32_t n_seqs, uint32_t n_kv_heads,
                        const int32_t *n, uint32_t n_limit, uint32_t keep, uint32_t first, uint32_t recent, int32_t *idx,
                        int32_t *count, void *stream) {
    const uint64_t lists = (uint64_t)n_layers * n_seqs * n_kv_heads;
    if (!scores || !n || !idx || !count || !n_layers || !n_seqs || !n_kv_heads || n_layers > 65535u || n_seqs > 65535u ||
        n_kv_heads > 65535u || lists > (1u << 27) || !keep || keep > 0x7FFFFFFFu || (uint64_t)first + recent > keep ||
        n_limit > stride || n_limit > SEL_N_MAX) {
        latch_error("vbs_cu_cache_select: invalid arguments");
        return -1;
    }
    DevState *d = backend_current();
    if (!d) { latch_error("vbs_cu_cache_select: no usable device"); return -1; }
    // CTAs per list: as many as the SMs have room for, 4096 scores each at
    // least; more where the bits of a list do not fit one CTA's shared memory
    uint32_t c = 1;
    while (c < 8 && (n_limit > c * SEL_CHUNK_MAX || (lists * c * 2 <= (uint64_t)d->n_sm && n_limit > c * 4096u))) c *= 2;
    SelectParams p = {};
    p.scores = scores; p.stride = stride; p.n_seqs = n_seqs; p.n_kv_heads = n_kv_heads; p.n_limit = n_limit;
    p.keep = keep; p.first = first; p.recent = recent; p.n = n; p.idx = idx; p.count = count; p.err = d->err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(lists * c));
    cfg.blockDim = dim3(SEL_THREADS);
    p.chunk_max = (n_limit + c - 1) / c;
    cfg.dynamicSmemBytes = SEL_FIXED + 8 * sel_words(p.chunk_max);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    note_launches(1);
    return cuda_ok(cudaLaunchKernelEx(&cfg, cache_select_kernel, p), "cache_select") ? 0 : -1;
}

int vbs_cu_cache_gather(const vbs_cu_kv_t *src, const vbs_cu_kv_t *dst, const vbs_cu_gather_t *g, void *stream) {
    bool ok = kv_desc_ok(src) && kv_desc_ok(dst) && g && g->idx && g->count && g->n_max && src->n_layers == dst->n_layers &&
              src->n_seqs == dst->n_seqs && src->n_kv_heads == dst->n_kv_heads && src->head_dim == dst->head_dim &&
              !g->weights_src == !g->weights_dst && !g->pos_src == !g->pos_dst && g->n_max <= 0x7FFFFFFFu;
    const uint64_t lists = ok ? (uint64_t)src->n_layers * src->n_seqs * src->n_kv_heads : 0;
    bool same = false;
    if (ok) {
        const uint64_t es = kv_extent(src) * 2, ed = kv_extent(dst) * 2;
        const uint64_t as = lists * src->max_ctx * 4, ad = lists * dst->max_ctx * 4;
        same = src->k == dst->k;
        if (same)
            ok = src->v == dst->v && src->max_ctx == dst->max_ctx && !src->head_major == !dst->head_major &&
                 src->seq_stride == dst->seq_stride && g->weights_src == g->weights_dst && g->pos_src == g->pos_dst;
        else
            ok = !overlap(src->k, es, dst->k, ed) && !overlap(src->v, es, dst->v, ed) && !overlap(src->k, es, dst->v, ed) &&
                 !overlap(src->v, es, dst->k, ed) && !overlap(g->weights_src, as, g->weights_dst, ad) &&
                 !overlap(g->pos_src, as, g->pos_dst, ad);
        ok = ok && lists <= (1u << 24);
    }
    if (!ok) {
        latch_error("vbs_cu_cache_gather: invalid arguments");
        return -1;
    }
    DevState *d = backend_current();
    if (!d) { latch_error("vbs_cu_cache_gather: no usable device"); return -1; }
    GatherParams p = {};
    p.src = gather_side(src);
    p.dst = gather_side(dst);
    p.g = *g;
    p.n_seqs = src->n_seqs;
    p.n_kv_heads = src->n_kv_heads;
    p.cpr = src->head_dim / 8;
    p.err = d->err;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    note_launches(1);
    if (same && g->n_max <= GA_WARP_MAX) {
        const uint32_t per = GA_THREADS / 32;
        gather_inplace_warp_kernel<<<(unsigned)((lists + per - 1) / per), GA_THREADS, 0, st>>>(p, (uint32_t)lists);
    } else if (same) {
        // slices of at least 64 bytes, as many as cover the SMs four times
        const uint32_t want = (uint32_t)std::min<uint64_t>(8, ((uint64_t)d->n_sm * 4 + lists - 1) / lists);
        p.slice = std::max(std::min(4u, p.cpr), (p.cpr + want - 1) / want);
        gather_inplace_kernel<<<dim3((unsigned)lists, (p.cpr + p.slice - 1) / p.slice), GA_THREADS, 0, st>>>(p);
    } else {
        const uint32_t rows = GX_THREADS / p.cpr * GX_U;
        const uint64_t nblk = (std::min(g->n_max, dst->max_ctx) + rows - 1) / rows;
        if (lists * nblk > 0x7FFFFFFFull) {
            latch_error("vbs_cu_cache_gather: %llu lists of %u rows are too many for one call", (unsigned long long)lists,
                        g->n_max);
            return -1;
        }
        gather_apart_kernel<<<(unsigned)(lists * nblk), GX_THREADS, 0, st>>>(p, (uint32_t)nblk);
    }
    return cuda_ok(cudaGetLastError(), "cache_gather") ? 0 : -1;
}

}  // extern "C"
