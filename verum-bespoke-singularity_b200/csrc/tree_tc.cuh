// tree_tc.cuh -- what the tcgen05 kernels of tree.cu's attention share: the
// instructions, and the queries as an operand.
#pragma once

#include "tree.cuh"

namespace vbs {

// Shared-memory operand descriptor, layout without swizzle: 8 rows of 16
// bytes contiguous; addresses and offsets in 16-byte units, version 1.
// K-major: lbo from 8 K elements to the next, sbo from 8 rows to the next.
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
// The issuing warp runs in uniform control flow and one elected lane issues:
// descriptors stay in uniform registers. `acc`, `lead`: 0 or 1.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead) : "memory");
}
__device__ __forceinline__ uint32_t tc_elect() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
    return e;
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// The loaded registers pass through the wait, so nothing uses them before.
__device__ __forceinline__ void tc_wait_ld(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), 
                 "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), 
                 "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]) :: "memory");
}
__device__ __forceinline__ void tc_wait_ld(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]) :: "memory");
}
__device__ __forceinline__ void tc_wait_ld(uint32_t &v) { asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v) :: "memory"); }
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
__device__ __forceinline__ void tc_ld16(uint32_t a, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(a));
}
__device__ __forceinline__ void tc_st16(uint32_t a, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                 "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
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

// x * f + c, a - b and a + b on pairs (one instruction for two values)
__device__ __forceinline__ float2 fma2(float2 x, float2 f, float2 c) {
    float2 r;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
        " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(f.x), "f"(f.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
    float2 r;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max32(const uint32_t (&s)[32]) {
    float m[2] = {__uint_as_float(s[0]), __uint_as_float(s[1])};
#pragma unroll
    for (int e = 2; e < 32; e += 2) m[(e >> 1) & 1] = max3(m[(e >> 1) & 1], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
    return fmaxf(m[0], m[1]);
}
// Two weights as fp16 halves: hi the weight cut to fp16's bits (exact), lo =
// p - hi rounded.
__device__ __forceinline__ void halves(float2 p, uint32_t &hi, uint32_t &lo) {
    const float2 h = make_float2(__uint_as_float(__float_as_uint(p.x) & 0xFFFFE000u), __uint_as_float(__float_as_uint(p.y) & 0xFFFFE000u));
    const float2 d = fma2(h, make_float2(-1.f, -1.f), p);
    const __half2 a = __floats2half2_rn(h.x, h.y), b = __floats2half2_rn(d.x, d.y);
    hi = *reinterpret_cast<const uint32_t *>(&a);
    lo = *reinterpret_cast<const uint32_t *>(&b);
}

// The queries of 8 rows per call and warp, rows r0 + lane % 8, 32 dims per
// step: whole sectors from memory, conflict-free 16-byte stores.
template <int D> struct TcQ { float4 x[D / 32][2]; };   // up to D dims

template <int D>
__device__ __forceinline__ void tc_q_load(const TreeParams &p, uint32_t row, uint32_t limit, uint32_t kvh, uint32_t b, TcQ<D> &q) {
    const int lane = threadIdx.x & 31;
    const bool on = row < limit;
    const uint32_t rr = on ? row : 0u, tok = tree_token(p, rr);
    // whole 32-byte sectors where they are aligned: half a sector a lane
    // fetches each twice, the L1 left beside the stages is too small for it
    const bool wide = (reinterpret_cast<uintptr_t>(p.q) & 31) == 0;
    const float *src = p.q + (((uint64_t)b * p.n_tokens + tok) * p.nqh + kvh * p.G + (rr - tok * p.G)) * p.hd;
#pragma unroll
    for (uint32_t j = 0; j < D / 32; ++j) {
        const uint32_t c = 4 * j + (lane >> 3);
        q.x[j][0] = q.x[j][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!on || c >= p.hd / 8) continue;
        if (wide) {
            asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=f"(q.x[j][0].x), "=f"(q.x[j][0].y), "=f"(q.x[j][0].z), "=f"(q.x[j][0].w), "=f"(q.x[j][1].x), "=f"(q.x[j][1].y),
                           "=f"(q.x[j][1].z), "=f"(q.x[j][1].w) : "l"(src + 8 * c));
        } else {
            q.x[j][0] = *reinterpret_cast<const float4 *>(src + 8 * c);
            q.x[j][1] = *reinterpret_cast<const float4 *>(src + 8 * c + 4);
        }
    }
}

// Their halves into the K-major image at `hi` ([chunk of 8 dims][row], chunks
// `pitch` bytes apart, the low halves `lo_off` bytes behind), scaled by the
// row's power of two; returns the score's factor of the lane's row.
template <int D>
__device__ __forceinline__ float tc_q_store(const TreeParams &p, const TcQ<D> &q, uint8_t *hi, uint32_t pitch, uint32_t lo_off, uint32_t r,
                                            uint32_t chunks) {
    const int lane = threadIdx.x & 31;
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u)
            top = fmaxf(top, fmaxf(fmaxf(fabsf(q.x[j][u].x), fabsf(q.x[j][u].y)), fmaxf(fabsf(q.x[j][u].z), fabsf(q.x[j][u].w))));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    int e = (int)((__float_as_uint(top) >> 23) & 255u) - 127;   // as in tree_mma_kernel
    e = (e < -100 || e > 100) ? 0 : 8 - e;
    const float up = __uint_as_float((uint32_t)(127 + e) << 23) * (p.scale < 0.f ? -1.f : 1.f);
#pragma unroll
    for (uint32_t j = 0; j < D / 32; ++j) {
        const uint32_t c = 4 * j + (lane >> 3);
        if (c >= chunks) continue;
        uint32_t h[4], l[4];
        const float v[8] = {q.x[j][0].x, q.x[j][0].y, q.x[j][0].z, q.x[j][0].w, q.x[j][1].x, q.x[j][1].y, q.x[j][1].z, q.x[j][1].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float v0 = v[2 * k] * up, v1 = v[2 * k + 1] * up;
            const __half2 hh = __floats2half2_rn(v0, v1);
            const float2 f = __half22float2(hh);
            const __half2 ll = __floats2half2_rn(v0 - f.x, v1 - f.y);
            h[k] = *reinterpret_cast<const uint32_t *>(&hh);
            l[k] = *reinterpret_cast<const uint32_t *>(&ll);
        }
        uint8_t *d = hi + c * pitch + r * 16u;
        *reinterpret_cast<uint4 *>(d) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(d + lo_off) = make_uint4(l[0], l[1], l[2], l[3]);
    }
    return fabsf(p.scale) * __uint_as_float((uint32_t)(127 - e) << 23) * (p.cap > 0.f ? 1.f / p.cap : TREE_LOG2E);
}

}  // namespace vbs
