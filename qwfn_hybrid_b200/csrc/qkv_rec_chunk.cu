// qkv_rec_chunk.cu -- chunked linear attention with a decay per head, with or without the delta rule, for prompts
// (qkv_rec_chunk), on the 5th-generation tensor cores.
//
// 64 tokens at a time.  With G = sums of g inside the chunk (G_C: the whole chunk's) and S the state before it,
//   A_ij = beta_i (k_i . k_j) e^(G_i - G_j) for j < i,   T = (1 + A)^-1   (lower triangular),
//   U = T R,  R_j = beta_j (v_j - e^(G_j) S k_j)          (without the delta rule U = V),
//   o_i = scale (e^(G_i) S q_i + sum_{j <= i} (q_i . k_j) e^(G_i - G_j) u_j),
//   S  <- e^(G_C) S + sum_j e^(G_C - G_j) u_j k_j^T.
// A CTA walks the chunks of one head of one sequence.  Everything without S -- the scores [k; q] k^T, P = their
// decayed lower triangle for q, and T -- is made by RK_GROUPS producer groups of four warps, a chunk each, up to three
// chunks ahead of the chain through S.  The chain is eight warps and the tensor cores: S [value][key] lies in
// registers, thread (row, half) holding 64 keys of a value row, and every product has the value rows as its
// M = 128, so that its A operand is written to tensor memory by the thread that has just read the last product from
// there (lane = value row: no shuffles, no shared memory); B is k, q, T and P in shared memory as they are.  Per
// chunk: X = S k^T, U = R T^T, O = S q^T, S += (w U) k (k as an MN-major operand, the same bytes), O += U P^T.  A warp of
// its own issues the products, so that no other waits for the tensor cores to take one; S q^T goes behind what the
// chain waits for (beside X, as one product of 128 columns, a 16K prompt took 4% longer).  The chain reads a chunk's O while
// the next chunk's X is made, and stores it while that chunk's part of S is made.
//
// Where the sequences are more than two, the CTAs take the longest first (24 prompts of 24001 rows: 5% less).
//
// Precision.  k and q are exact in bf16, so S, w U and U enter as sums of bf16 terms (three: 24 bits; two for what
// only the rounded output sees, as P; truncated terms, which need no conversion: three of them are the value), and T
// and R, which meet each other, as two f16 terms of rows scaled to [2^12, 2^13) (22 bits; of T's row of a token, of R's
// value row over 32 tokens: what is more than 2^16 below the row's largest loses bits, and below 2^-38 of it is lost),
// three products: state and U keep 32-bit accuracy (2 to 5e-7 of the state's norm against 64 bits).  Sums are F32; the state is scaled and added
// outside the tensor cores (their sums are truncated).  G is summed as pairs of floats: e^(G_i - G_j) needs the
// difference, not the rounded sums.  The output is rounded to bf16 once.
//
// A zero of T or P times a NaN is a NaN, so a chunk with a non-finite input would spread it to earlier
// tokens; such chunks (and those with g > 0, a growing state, which could leave the range of what is scaled) are
// flagged by the producers and run token by token from global memory.  Finite inputs can leave F32's range inside a chunk too
// (long keys, repeated): a value row whose u is finite at its first token and not at a later one has the chunk thrown away and
// run so.  (A row that starts with a state that is not finite has no output to save.)
//
// What bounds it: neither bytes nor the tensor cores (84 products of 32 or 64 cycles a chunk, 48 without the delta rule) but the chain's latency -- four
// round trips from registers through tensor memory and a product a chunk -- and, beside it on the same schedulers, the
// producers'.  A chunk takes 5.0 us (delta rule, 16384 tokens: 1278 us) or 3.3 us (decay alone).  From about 100
// CTAs on it takes longer, 5.6 to 8.4 us at 148 CTAs with k and q of their own: the three roles' loops are more instructions than an SM keeps, and the SMs of a group
// fetch them from one cache (at 148 CTAs warps waited 3.5 cycles per instruction for instructions, at 32 CTAs 0.4; with the
// loops as they are, 1.6 and 0.3).  So the
// code is kept short where time allows: one body for the rows of k and of q, loops over tiles of T and over the terms of a
// product (24 prompts of 24001 rows, 32 heads: 656 -> 556 us); with all products in loops 148 equal CTAs took 16% less than so, but few of
// them 3% more.  Not kept: a long sequence in three parts by clusters of three CTAs (the state is linear in the one it starts
// from) took 1160 instead of 1310 us and, through its registers, made all other sizes 3 to 7% slower; a kernel of the same split on
// mma.sync, 64 value rows per CTA, took 5.9 us per chunk and half a head.
#include "qkv_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace qkv {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr int RK_C = 64, RK_GROUPS = 2, RK_GT = 128, RK_CHAIN = 256, RK_STAGES = 3;
// chain, producers, and a warp that issues the products (in a warpgroup of its own: the others of it leave at once)
constexpr int RK_ISSUER = RK_CHAIN + RK_GROUPS * RK_GT, RK_THREADS = RK_ISSUER + 128;
// A stage.  k and q: 128 rows (tokens of k, then of q) of 128 bytes per 64 keys, two such blocks; T, P: 64 rows of 128
// bytes; all swizzled by 128 bytes.  Until T is split, A and T lie where its terms will, as 16 x 16 tiles on and below the
// diagonal.  Then CF_N arrays of RK_C floats, per-token values of the producers, e^(G_C), the flag.
constexpr int RK_KQ = 0, RK_KSUB = 16384, RK_TH = 32768, RK_TL = 40960, RK_PH = 49152, RK_PM = 57344, RK_COEF = 65536;
enum { CF_X, CF_V, CF_T, CF_Q, CF_W, CF_GS, CF_BS, CF_H, CF_G2, CF_N = CF_G2 + 2 };
constexpr int RK_STAGE = 67 * 1024;
static_assert(RK_COEF + CF_N * RK_C * 4 + 8 <= RK_STAGE, "stage");
constexpr int RK_PITCH = 20, RK_TILE = 16 * RK_PITCH;
static_assert(10 * RK_TILE * 4 <= 2 * 8192, "tiles of A in the place of T");
constexpr int RK_VS = RK_STAGES * RK_STAGE;   // v of one chunk as it is, then the control block
constexpr int RK_BARS = 5;
struct RkCtl {
    uint64_t bar[RK_BARS];    // products done: X, U, S, O's second part; O's first
    uint64_t scored[RK_GROUPS], read;   // a group's scores are there; their columns have been read
    uint32_t tmem;
    int32_t  abort;
    int32_t  seq;
    int32_t  redo;            // the chunk's U left F32's range behind a value row's first token
    float    scale[128];      // inverse scale of R's first 32 tokens, per value row (NaN: not finite from the first token on)
};
constexpr int RK_CTL = RK_VS + RK_C * REC_HD * 2;
constexpr int RK_SMEM = RK_CTL + (int)sizeof(RkCtl);
static_assert(RK_SMEM + 1024 <= 232448, "shared memory of a CTA");
// registers, of 96 at launch: 256 x 152 + 256 x 72 + 128 x 32 = 61440 = 640 x 96
constexpr int RK_CHAIN_REGS = 152, RK_PROD_REGS = 72, RK_ISSUER_REGS = 32;
static_assert(RK_CHAIN * RK_CHAIN_REGS + RK_GROUPS * RK_GT * RK_PROD_REGS + 128 * RK_ISSUER_REGS <= RK_THREADS * 96, "register shares");
// Barriers.  A stage's EMPTY has one per group: the groups take its chunks in turn, and one must not meet the other's.
enum { BAR_FULL = 1, BAR_EMPTY = BAR_FULL + RK_STAGES, BAR_PROD = BAR_EMPTY + RK_STAGES * RK_GROUPS, BAR_HAND = BAR_PROD + RK_GROUPS, BAR_HAND_U, BAR_CHAIN, BAR_END };
static_assert(BAR_END < 16, "named barriers");
constexpr int RK_FULL_N = RK_GT + RK_CHAIN + 32, RK_EMPTY_N = RK_GT + RK_CHAIN, RK_HAND_N = RK_CHAIN + 32;
// tensor memory columns.  S: half h (keys 64 h ..) has its leading and middle terms at 64 h, 64 h + 32, its last at
// TM_S2 or (h = 1) TM_U2; the new part of S comes back over the first 128 (each thread reads and writes its own 64).  X:
// tokens 32 h .. at 32 h; R's two terms replace what its thread has read, then two of w U's; the third takes the place
// of S's last (h = 0).  O's second part replaces U.  Then the producers' scores, and U's terms for O.
// What lets a region be written again, chunk c's last reader of it in brackets: TM_S and w U's terms, bar[2] of c (S's
// product, behind bar[4] in the issuer); S's last terms [X's product], bar[0] of c, and at TM_U2 the thread that writes them is
// the one that read U there; R [U's product], bar[1]; U's two terms for O (TM_UL, TM_UM) [O's second part, which c + 1's S
// does not wait for], bar[3] of c, which each thread waits for before it hands over R (delta rule) or starts c + 1; O and U, the hand-over of
// R (delta rule) or of S, behind every thread's read of them.
constexpr uint32_t TM_S = 0, TM_S2 = 128, TM_UL = 160, TM_X = 192, TM_O1 = 256, TM_U = 320, TM_U2 = 384, TM_G = 416, TM_UM = 480, TM_COLS = 512;

__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The power of two that brings a row whose largest magnitude is m to [2^12, 2^13), and its inverse (both normal
// numbers; rows below 2^-114 are left smaller).
__device__ __forceinline__ float pow2_scale(float m, float &inv) {
    const int e = (__float_as_int(m) >> 23) & 255;
    const int f = min(254 + 12 - e, 253);
    inv = __int_as_float((254 - f) << 23);
    return __int_as_float(f << 23);
}
__device__ __forceinline__ void split_f16(float a, float b, float s, uint32_t &hi, uint32_t &lo) {
    a *= s;
    b *= s;
    const __half2 h = __floats2half2_rn(a, b);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    asm("{\n\t.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xBC00;\n\tfma.rn.f32.f16 %0, l, m, %0;\n\tfma.rn.f32.f16 %1, h, m, %1;\n\t}"
        : "+f"(a), "+f"(b) : "r"(hi));
    const __half2 l = __floats2half2_rn(a, b);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// The leading bf16 term (truncated) of two values; they become what is left of them, exactly.
__device__ __forceinline__ uint32_t take_bf16(float &a, float &b) {
    const uint32_t w = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    asm("{\n\t.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xBF80;\n\tfma.rn.f32.bf16 %0, l, m, %0;\n\tfma.rn.f32.bf16 %1, h, m, %1;\n\t}"
        : "+f"(a), "+f"(b) : "r"(w));   // less the term, by a factor of -1
    return w;
}

// ---- tensor memory and tcgen05 (one CTA)
__device__ __forceinline__ void tm_ld32(uint32_t addr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tm_wait16(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                   "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_st8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// Waits for the thread's loads; v passes through, so that nothing uses it before.
__device__ __forceinline__ void tm_wait_ld(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                   "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
                   "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                   "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28])
                 :
                 : "memory");
    asm volatile("" : "+f"(v[29]), "+f"(v[30]), "+f"(v[31]));
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Operand descriptor, 128-byte swizzle.  K-major (T, P, and k or q against S): groups of 8 rows 1024 bytes apart.
// MN-major (k against w U): blocks of 64 keys RK_KSUB apart (leading offset), groups of 8 tokens 1024 bytes apart.
__device__ __forceinline__ uint64_t rk_desc(uint32_t saddr, uint32_t leading) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor, kind::f16, M = 128: D F32 (bit 4), A and B f16 (0) or bf16 (1) at bits 7 and 10, B MN-major at
// bit 16, N >> 3 at bit 17, M >> 4 at bit 24.
constexpr uint32_t rk_idesc(int n, bool bf16, bool mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void rk_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void rk_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void rk_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(bar))
                 : "memory");
}
// Bounded wait for products (2 s): past the limit the status is set and nothing waits any more.
__device__ __forceinline__ void rk_wait_one(uint64_t *bar, uint32_t parity, RkCtl *ctl, int32_t *status) {
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(bar);
    uint64_t t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(a), "r"(parity), "r"(20000u) : "memory");
        if (ok) break;
        if (*(volatile int32_t *)&ctl->abort) break;
        uint64_t t;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t0 == 0) t0 = t;
        if (t - t0 > WAIT_NS_DEFAULT) {
            *(volatile int32_t *)&ctl->abort = 1;
            atomicOr(status, ST_TIMEOUT);
            break;
        }
    }
}
__device__ __forceinline__ void rk_wait(uint64_t *bar, uint32_t parity, RkCtl *ctl, int32_t *status) {   // by whole warps
    rk_wait_one(bar, parity, ctl, status);
    __syncwarp();
    tc_fence_after();
}

// ---- producers
__device__ __forceinline__ void rk_prefetch(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void rk_cp16_zero(uint32_t dst, const void *src, bool ok) {   // zeros unless ok (src is not read then)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16u : 0u) : "memory");
}
// d += a b on 16 x 16 tiles (pitch RK_PITCH), each factor as two TF32 terms, three products; d in accumulator layout.
__device__ __forceinline__ void rk_tile(float (&d)[2][4], const float *a, const float *b, int g, int t) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = a[(g + (i & 1) * 8) * RK_PITCH + 8 * k + t + (i >> 1) * 4];
            ah[i] = __float_as_uint(x) & 0xffffe000u;
            al[i] = __float_as_uint(x - __uint_as_float(ah[i]));
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            uint32_t bh[2], bl[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float x = b[(8 * k + t + 4 * i) * RK_PITCH + 8 * n + g];
                bh[i] = __float_as_uint(x) & 0xffffe000u;
                bl[i] = __float_as_uint(x - __uint_as_float(bh[i]));
            }
            mma_tf32(d[n], al, bh[0], bh[1]);
            mma_tf32(d[n], ah, bl[0], bl[1]);
            mma_tf32(d[n], ah, bh[0], bh[1]);
        }
    }
}
__device__ __forceinline__ void rk_tile_store(float *o, const float (&d)[2][4], int g, int t) {
#pragma unroll
    for (int n = 0; n < 2; n++) {
        *reinterpret_cast<float2 *>(o + g * RK_PITCH + 8 * n + 2 * t) = make_float2(d[n][0], d[n][1]);
        *reinterpret_cast<float2 *>(o + (g + 8) * RK_PITCH + 8 * n + 2 * t) = make_float2(d[n][2], d[n][3]);
    }
}

// A row's scores x[0 .. 31] with tokens j0 .. times e^(G_i - G_j): zero for j > i (or j = i too, strict).  From row to column
// through the middle of the chunk where they lie on both sides of it.
template <bool DIRECT>
__device__ __forceinline__ void rk_decay(float (&x)[32], const float *cf, int i, int j0, float f, bool strict) {
    if (DIRECT) {
        const float2 *G2 = reinterpret_cast<const float2 *>(cf + CF_G2 * RK_C);
        const float2 r = G2[i];
        const int lim = i - j0 + (strict ? 0 : 1);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            const float4 c = *reinterpret_cast<const float4 *>(G2 + j0 + j);
            const float a = f * ex2((r.x - c.x) + (r.y - c.y)), b = f * ex2((r.x - c.z) + (r.y - c.w));
            x[j] = j < lim ? x[j] * a : 0.0f;
            x[j + 1] = j + 1 < lim ? x[j + 1] * b : 0.0f;
        }
    } else {
        const float g = f * cf[CF_H * RK_C + i];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 c = *reinterpret_cast<const float4 *>(cf + CF_H * RK_C + j);
            x[j] *= g * c.x;
            x[j + 1] *= g * c.y;
            x[j + 2] *= g * c.z;
            x[j + 3] *= g * c.w;
        }
    }
}
__device__ __forceinline__ bool rk_not_finite(const float (&x)[32]) {
    float z = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; j++) z = fmaf(x[j], 0.0f, z);
    return !(z == 0.0f);
}
// Row i's scores with tokens 32 half .. as two bf16 terms.
__device__ __forceinline__ void rk_store_p(uint8_t *sg, int i, int half, float (&x)[32]) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int off = i * 128 + (((4 * half + c) ^ (i & 7)) << 4);
        uint32_t h[4], m[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            h[k] = take_bf16(x[8 * c + 2 * k], x[8 * c + 2 * k + 1]);
            m[k] = take_bf16(x[8 * c + 2 * k], x[8 * c + 2 * k + 1]);
        }
        *reinterpret_cast<uint4 *>(sg + RK_PH + off) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(sg + RK_PM + off) = make_uint4(m[0], m[1], m[2], m[3]);
    }
}
__device__ __forceinline__ void rk_store_a(float *As, int i, int jb, const float (&x)[32]) {   // tiles jb, jb + 1 of row i, as far as the diagonal
    const int ib = i >> 4;
#pragma unroll
    for (int k = 0; k < 2; k++)
        if (jb + k <= ib) {
            float4 *o = reinterpret_cast<float4 *>(As + (ib * (ib + 1) / 2 + jb + k) * RK_TILE + (i & 15) * RK_PITCH);
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] = make_float4(x[16 * k + 4 * c], x[16 * k + 4 * c + 1], x[16 * k + 4 * c + 2], x[16 * k + 4 * c + 3]);
        }
}

// A producer group: chunks grp, grp + RK_GROUPS, ... of the sequence.
template <bool DELTA>
__device__ __forceinline__ void rk_produce(const RecParams &p, uint8_t *sm, RkCtl *ctl, int h, int32_t beg, int32_t end) {
    const int grp = (threadIdx.x - RK_CHAIN) / RK_GT, tid = threadIdx.x % RK_GT, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
    const int hk = h / (p.n_head / p.n_head_k);
    const uint32_t tm = ctl->tmem;
    int c = grp;
    for (int32_t t0 = beg + grp * RK_C, st = grp; t0 < end; c += RK_GROUPS, t0 += RK_GROUPS * RK_C, st = st >= RK_STAGES - RK_GROUPS ? st - (RK_STAGES - RK_GROUPS) : st + RK_GROUPS) {
        uint8_t *sg = sm + st * RK_STAGE;
        const uint32_t su = (uint32_t)__cvta_generic_to_shared(sg);
        float *cf = reinterpret_cast<float *>(sg + RK_COEF);
        float *As = reinterpret_cast<float *>(sg + RK_TH), *gs = cf + CF_GS * RK_C, *bs = cf + CF_BS * RK_C;
        float2 *G2 = reinterpret_cast<float2 *>(cf + CF_G2 * RK_C);   // sums of g up to a token, as two floats
        float gu = 0.0f, bu = 0.0f;
        if (tid < RK_C && t0 + tid < end) {
            gu = p.g[(int64_t)(t0 + tid) * p.n_head + h];
            if (DELTA) bu = p.beta[(int64_t)(t0 + tid) * p.n_head + h];
        }
        bar_sync(BAR_EMPTY + st * RK_GROUPS + grp, RK_EMPTY_N);
        bool bad = false;
        const int ch = tid & 15;
        {   // k, q as they are, zeros behind the sequence: 16 threads a row of 128 values
            const __nv_bfloat16 *kp = static_cast<const __nv_bfloat16 *>(p.k) + (int64_t)hk * REC_HD + ch * 8;
            const __nv_bfloat16 *qp = static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)hk * REC_HD + ch * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int row = 8 * i + (tid >> 4);
                const bool ok = t0 + row < end;
                const int64_t at = ok ? t0 + row : beg;
                const uint32_t off = su + (ch >> 3) * RK_KSUB + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
                rk_cp16_zero(off + RK_KQ, kp + at * p.k_stride, ok);
                rk_cp16_zero(off + RK_KQ + 8192, qp + at * p.q_stride, ok);
            }
        }
        {   // the group's next chunk on its way into L2
            const int32_t r = t0 + RK_GROUPS * RK_C + (tid >> 1);
            if (r < end) {
                const int o = (tid & 1) * 64;
                rk_prefetch(static_cast<const __nv_bfloat16 *>(p.k) + (int64_t)r * p.k_stride + (int64_t)hk * REC_HD + o);
                rk_prefetch(static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)r * p.q_stride + (int64_t)hk * REC_HD + o);
                rk_prefetch(static_cast<const __nv_bfloat16 *>(p.v) + (int64_t)r * p.v_stride + (int64_t)h * REC_HD + o);
            }
        }
        if (tid == 0) cf[CF_N * RK_C + 1] = 0.0f;
        if (tid < RK_C) {
            // in base 2; below 2^-184 = 0: the clamp keeps sums and differences finite.  A growing state
            // (g > 0) could leave the range of what is scaled here: flagged, as what is not finite
            gs[tid] = fmaxf(gu, -128.0f) * 1.4426950408889634f;
            bs[tid] = bu;
            bad |= !(gu <= 0.0f) || !(fabsf(bu) <= 3.0e38f);
        }
        bar_sync(BAR_PROD + grp, RK_GT);
        {   // v (which the chain loads): anything that is not finite?
            const __nv_bfloat16 *vp = static_cast<const __nv_bfloat16 *>(p.v) + (int64_t)h * REC_HD + ch * 8;
            uint32_t vm = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int row = t0 + 8 * i + (tid >> 4);
                if (row < end) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(vp + (int64_t)row * p.v_stride);
                    vm = __vmaxu2(__vmaxu2(vm, __vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu)), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
                }
            }
            bad |= (vm & 0xffffu) >= 0x7f80u || vm >= 0x7f800000u;
        }
        if (wid == 3) {
            // sums of g as pairs of floats (two-sum at each step), two tokens per lane
            const float g0 = gs[2 * lane], g1 = gs[2 * lane + 1];
            float hi = g0 + g1, lo = (g0 - (hi - (hi - g0))) + (g1 - (hi - g0));
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float uh = __shfl_up_sync(0xffffffffu, hi, o), ul = __shfl_up_sync(0xffffffffu, lo, o);
                const float s = hi + uh, b = s - hi;
                const float e = (hi - (s - b)) + (uh - b) + (lo + ul);
                if (lane >= o) {
                    hi = s + e;
                    lo = e - (hi - s);
                }
            }
            const float s = hi - g1, b = s - hi;
            const float e = (hi - (s - b)) + (-g1 - b) + lo, f = s + e;
            *reinterpret_cast<float4 *>(G2 + 2 * lane) = make_float4(f, e - (f - s), hi, lo);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor cores read k and q
        bar_sync(BAR_PROD + grp, RK_GT);
        if (tid == RK_GT - 1) {   // scores: [k; q] k^T, once the other group has read its own
            if (c > 0) rk_wait_one(&ctl->read, (c - 1) & 1, ctl, p.status);
            tc_fence_after();   // its loads of tensor memory come before the products that replace what they read
            const uint64_t kq = rk_desc(su + RK_KQ, 16);
#pragma unroll
            for (int kk = 0; kk < 8; kk++) {
                const uint64_t d = kq + (((kk >> 2) * RK_KSUB + (kk & 3) * 32) >> 4);
                rk_mma_ss(tm + TM_G, d, d, rk_idesc(64, true, false), kk > 0);
            }
            rk_commit(&ctl->scored[grp]);
        }
        if (tid < RK_C) {
            const float2 mine = G2[tid], last = G2[RK_C - 1], mid = G2[RK_C / 2 - 1];
            const float gam = ex2(mine.x) * fmaf(mine.y, 0.6931471805599453f, 1.0f), b = bs[tid], sg_ = tid < RK_C / 2 ? -1.0f : 1.0f;
            cf[CF_X * RK_C + tid] = -b * gam;
            cf[CF_V * RK_C + tid] = b;
            cf[CF_Q * RK_C + tid] = p.scale * gam;
            cf[CF_W * RK_C + tid] = ex2((last.x - mine.x) + (last.y - mine.y));
            cf[CF_H * RK_C + tid] = ex2(sg_ * ((mine.x - mid.x) + (mine.y - mid.y)));   // to, and from, the middle
            if (tid == RK_C - 1) cf[CF_N * RK_C] = gam;
        }
        __syncwarp();
        bar_sync(BAR_PROD + grp, RK_GT);
        rk_wait(&ctl->scored[grp], (c / RK_GROUPS) & 1, ctl, p.status);
        {   // a row per thread: warps 0, 1 rows of k k^T (-A; delta rule), warps 2, 3 of q k^T (P)
            const uint32_t tg = tm + TM_G + ((uint32_t)(32 * wid) << 16);
            const int i = tid & 63;
            const bool of_k = wid < 2;
            if (DELTA || !of_k) {
                const float f = of_k ? -bs[i] : 1.0f;
#pragma unroll 1
                for (int j = 0; j <= (wid & 1); j++) {   // 32 tokens of the row: below the diagonal block, then that
                    float x[32];
                    tm_ld32(tg + 32 * j, x);
                    tm_wait_ld(x);
                    if (j == (wid & 1)) {
                        bad |= rk_not_finite(x);
                        rk_decay<true>(x, cf, i, 32 * j, f, of_k);
                    } else {
                        rk_decay<false>(x, cf, i, 0, f, of_k);
                    }
                    if (of_k) rk_store_a(As, i, 2 * j, x);
                    else rk_store_p(sg, i, j, x);
                }
            }
            if (wid == 2) {   // nothing right of the diagonal blocks
#pragma unroll
                for (int c = 4; c < 8; c++) {
                    const int off = i * 128 + ((c ^ (i & 7)) << 4);
                    *reinterpret_cast<uint4 *>(sg + RK_PH + off) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(sg + RK_PM + off) = make_uint4(0, 0, 0, 0);
                }
            }
            tc_fence_before();
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"((uint32_t)__cvta_generic_to_shared(&ctl->read)) : "memory");
        }
        if (bad) cf[CF_N * RK_C + 1] = 1.0f;
        if (DELTA) {
            bar_sync(BAR_PROD + grp, RK_GT);
            // T in place of A.  The 16 x 16 tiles on the diagonal, one per warp: their 8 x 8 blocks on the diagonal by
            // forward substitution, x_i = [i = column] - sum_{j < i} A_ij x_j, a column per lane, then the block below,
            // -T_11 A_10 T_00, two of its values per lane (A is held negated);
            {
                float *a = As + (wid * (wid + 1) / 2 + wid) * RK_TILE;
                if (lane < 16) {
                    float *d = a + (lane >> 3) * (8 * RK_PITCH + 8), y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        float s0 = i == (lane & 7) ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
                        for (int j = 0; j < i; j += 4) {
                            const float4 u = *reinterpret_cast<const float4 *>(d + i * RK_PITCH + j);
                            s0 = fmaf(u.x, y[j], s0);
                            if (j + 1 < i) s1 = fmaf(u.y, y[j + 1], s1);
                            if (j + 2 < i) s0 = fmaf(u.z, y[j + 2], s0);
                            if (j + 3 < i) s1 = fmaf(u.w, y[j + 3], s1);
                        }
                        y[i] = s0 + s1;
                    }
                    __syncwarp(0xffffu);
#pragma unroll
                    for (int i = 0; i < 8; i++) d[i * RK_PITCH + (lane & 7)] = y[i];
                }
                __syncwarp();
                float *lo = a + (8 + g) * RK_PITCH, *x = a + 2 * t;   // a row of the block below, two columns
#pragma unroll
                for (int s = 0; s < 2; s++) {   // A_10 T_00 in A_10's place, then T_11 times that
                    const float *l = lo + 8 * s, *r = x + (s ? 8 * RK_PITCH : 0);
                    float v0 = 0.0f, v1 = 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; k += 4) {
                        const float4 u = *reinterpret_cast<const float4 *>(l + k);
                        const float2 r0 = *reinterpret_cast<const float2 *>(r + k * RK_PITCH), r1 = *reinterpret_cast<const float2 *>(r + (k + 1) * RK_PITCH);
                        const float2 r2 = *reinterpret_cast<const float2 *>(r + (k + 2) * RK_PITCH), r3 = *reinterpret_cast<const float2 *>(r + (k + 3) * RK_PITCH);
                        v0 = fmaf(u.w, r3.x, fmaf(u.z, r2.x, fmaf(u.y, r1.x, fmaf(u.x, r0.x, v0))));
                        v1 = fmaf(u.w, r3.y, fmaf(u.z, r2.y, fmaf(u.y, r1.y, fmaf(u.x, r0.y, v1))));
                    }
                    __syncwarp();
                    *reinterpret_cast<float2 *>(lo + 2 * t) = make_float2(v0, v1);
                    __syncwarp();
                }
            }
            bar_sync(BAR_PROD + grp, RK_GT);
            // the tiles beside them, T_10 = -T_11 A_10 T_00 (tiles 1, 0; 3, 2), A_10 T_00 first in A_10's place;
            if (wid < 2) {
                float *lo = As + (wid ? 8 : 1) * RK_TILE;                    // tile (1, 0) or (3, 2)
#pragma unroll 1
                for (int k = 0; k < 2; k++) {
                    float u[2][4] = {};
                    rk_tile(u, k ? lo + RK_TILE : lo, k ? lo : As + (wid ? 5 : 0) * RK_TILE, g, t);
                    __syncwarp();
                    rk_tile_store(lo, u, g, t);
                    __syncwarp();
                }
            }
            bar_sync(BAR_PROD + grp, RK_GT);
            {   // then the lower left 32 x 32: -T_1 A_10 T_0, a tile (a, b) of it per warp
                const int a = wid >> 1, b = wid & 1;
                float *lo = As + (a ? 6 : 3) * RK_TILE;                      // tiles (2 + a, 0) and (2 + a, 1)
                float u[2][4] = {}, w[2][4] = {};
#pragma unroll 1
                for (int k = b; k < 2; k++) rk_tile(u, lo + k * RK_TILE, As + k * (1 + b) * RK_TILE, g, t);   // M_ab = -sum_k A_(2+a)k T_kb, in A's place
                bar_sync(BAR_PROD + grp, RK_GT);
                rk_tile_store(lo + b * RK_TILE, u, g, t);
                bar_sync(BAR_PROD + grp, RK_GT);
#pragma unroll 1
                for (int k = 0; k <= a; k++) rk_tile(w, As + (5 + 3 * a + k) * RK_TILE, As + (3 + b + 3 * k) * RK_TILE, g, t);
                bar_sync(BAR_PROD + grp, RK_GT);
                rk_tile_store(lo + b * RK_TILE, w, g, t);
            }
            bar_sync(BAR_PROD + grp, RK_GT);
            {   // T as two f16 terms of scaled rows: row tid / 2, columns 32 (tid % 2) .., zeros right of the diagonal tile
                const int i = tid >> 1, half = tid & 1, ib = i >> 4;
                const float *a = As + (ib * (ib + 1) / 2 + 2 * half) * RK_TILE + (i & 15) * RK_PITCH;
                const int nt = min(2, ib + 1 - 2 * half);
                float y[2][16], mx = 0.0f;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float4 u = j < nt ? *reinterpret_cast<const float4 *>(a + j * RK_TILE + 4 * k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        y[j][4 * k] = u.x; y[j][4 * k + 1] = u.y; y[j][4 * k + 2] = u.z; y[j][4 * k + 3] = u.w;
                        mx = fmaxf(fmaxf(mx, fmaxf(fabsf(u.x), fabsf(u.y))), fmaxf(fabsf(u.z), fabsf(u.w)));
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                float inv;
                const float s = pow2_scale(mx, inv);
                bar_sync(BAR_PROD + grp, RK_GT);   // all have read the tiles that the terms replace
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int c8 = 0; c8 < 2; c8++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) split_f16(y[j][8 * c8 + 2 * k], y[j][8 * c8 + 2 * k + 1], s, hi[k], lo[k]);
                        const int off = i * 128 + (((half * 4 + j * 2 + c8) ^ (i & 7)) << 4);
                        *reinterpret_cast<uint4 *>(sg + RK_TH + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(sg + RK_TL + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                if (!half) cf[CF_T * RK_C + i] = inv;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor cores read this stage
        bar_arrive(BAR_FULL + st, RK_FULL_N);
    }
}

// ---- the chain
// A chunk token by token from global memory, by the chain's warps: 16 value rows each, 8 at a time in registers, 8 lanes a row as
// in k_rec_step.
template <bool DELTA>
__device__ __noinline__ void rk_serial(const RecParams &p, float *state, int h, int32_t t0, int32_t t1) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, sub = lane & 7, hk = h / (p.n_head / p.n_head_k);
#pragma unroll 1
    for (int half = 0; half < 2; half++) {
        const int row = wid * 16 + half * 8 + (lane >> 3);   // and row + 4
        float *S0 = state + row * REC_HD + sub * 4;
        float S[2][16];
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 x = *reinterpret_cast<const float4 *>(S0 + a * 4 * REC_HD + 32 * j);
                S[a][4 * j] = x.x; S[a][4 * j + 1] = x.y; S[a][4 * j + 2] = x.z; S[a][4 * j + 3] = x.w;
            }
#pragma unroll 1
        for (int32_t r = t0; r < t1; r++) {
            float k[16], q[16];
            auto load = [&](const void *x, int64_t stride, float (&o)[16]) {
                const __nv_bfloat16 *at = static_cast<const __nv_bfloat16 *>(x) + r * stride + hk * REC_HD + sub * 4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(at + 32 * j);
                    o[4 * j] = __uint_as_float(w.x << 16); o[4 * j + 1] = __uint_as_float(w.x & 0xffff0000u);
                    o[4 * j + 2] = __uint_as_float(w.y << 16); o[4 * j + 3] = __uint_as_float(w.y & 0xffff0000u);
                }
            };
            load(p.k, p.k_stride, k);
            load(p.q, p.q_stride, q);
            const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(p.v) + r * p.v_stride + h * REC_HD + row;
            float u[2] = {__bfloat162float(v[0]), __bfloat162float(v[4])}, o[2] = {};
            const float eg = expf(p.g[(int64_t)r * p.n_head + h]), b = DELTA ? p.beta[(int64_t)r * p.n_head + h] : 1.0f;
#pragma unroll
            for (int a = 0; a < 2; a++) {
#pragma unroll
                for (int i = 0; i < 16; i++) S[a][i] *= eg;
                if (DELTA) {
                    float d = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; i++) d = fmaf(S[a][i], k[i], d);
#pragma unroll
                    for (int m = 4; m; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
                    u[a] = b * (u[a] - d);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    S[a][i] = fmaf(u[a], k[i], S[a][i]);
                    o[a] = fmaf(S[a][i], q[i], o[a]);
                }
#pragma unroll
                for (int m = 4; m; m >>= 1) o[a] += __shfl_xor_sync(0xffffffffu, o[a], m);
                if (sub == 0) static_cast<__nv_bfloat16 *>(p.out)[((int64_t)r * p.n_head + h) * REC_HD + row + 4 * a] = __float2bfloat16_rn(o[a] * p.scale);
            }
        }
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                *reinterpret_cast<float4 *>(S0 + a * 4 * REC_HD + 32 * j) = make_float4(S[a][4 * j], S[a][4 * j + 1], S[a][4 * j + 2], S[a][4 * j + 3]);
    }
}

// The warp that issues the products: of a chunk in the order in which the chain hands their operands over.
template <bool DELTA>
__device__ __forceinline__ void rk_issue(uint8_t *sm, RkCtl *ctl, int32_t beg, int32_t end, int32_t *status) {
    const uint32_t smu = (uint32_t)__cvta_generic_to_shared(sm), tm = ctl->tmem;
    const bool one = (threadIdx.x & 31) == 0;
    const int n_chunks = (end - beg + RK_C - 1) / RK_C;
    uint32_t parity = 0;
    for (int c = 0, st = 0; c < n_chunks; c++, st = st == RK_STAGES - 1 ? 0 : st + 1) {
        const uint32_t su = smu + st * RK_STAGE;
        bar_sync(BAR_FULL + st, RK_FULL_N);
        if (reinterpret_cast<const float *>(sm + st * RK_STAGE + RK_COEF)[CF_N * RK_C + 1] != 0.0f) {
            bar_arrive(BAR_CHAIN, RK_HAND_N);   // the flag has been read: the chain may release the stage
            continue;
        }
        const uint64_t kq = rk_desc(su + RK_KQ, 16), kt = rk_desc(su + RK_KQ, RK_KSUB);
        const uint64_t th = rk_desc(su + RK_TH, 16), tl = rk_desc(su + RK_TL, 16), ph = rk_desc(su + RK_PH, 16), pm = rk_desc(su + RK_PM, 16);
        bar_sync(BAR_HAND, RK_HAND_N);
        tc_fence_after();
        auto times_s = [&](uint32_t d, uint64_t b, int terms) {   // S times 64 rows of k or q
#pragma unroll (DELTA ? 1 : 3)
            for (int term = 0; term < terms; term++)
#pragma unroll
                for (int kk = 0; kk < 8; kk++)
                    rk_mma(tm + d, tm + (term < 2 ? TM_S + 64 * (kk >> 2) + 32 * term : kk >> 2 ? TM_U2 : TM_S2) + 8 * (kk & 3),
                           b + (((kk >> 2) * RK_KSUB + (kk & 3) * 32) >> 4), rk_idesc(64, true, false), term + kk > 0);
        };
        if (one) {
            if (DELTA) {
                times_s(TM_X, kq, 3);
                rk_commit(&ctl->bar[0]);
            } else {
                times_s(TM_O1, kq + (8192 >> 4), 2);
                rk_commit(&ctl->bar[4]);
            }
        }
        __syncwarp();
        if (DELTA) {
            bar_sync(BAR_HAND, RK_HAND_N);
            tc_fence_after();
            if (one) {   // U: tokens 0 .. 31 of R against all of T, tokens 32 .. 63 against its lower right quarter (the scales differ)
#pragma unroll
                for (int part = 0; part < 2; part++)
#pragma unroll
                    for (int term = 0; term < 3; term++)
#pragma unroll
                        for (int ks = 0; ks < 2; ks++)
                            rk_mma(tm + (part ? TM_U2 : TM_U), tm + TM_X + 32 * part + (term == 1 ? 16 : 0) + 8 * ks,
                                   (term == 2 ? tl : th) + (((part ? 32 * 128 + 64 : 0) + 32 * ks) >> 4),
                                   rk_idesc(part ? 32 : 64, false, false), term + ks > 0);
                rk_commit(&ctl->bar[1]);
                // (not before: the last chunk's output has been read by those who handed R over)
                times_s(TM_O1, kq + (8192 >> 4), 2);
                rk_commit(&ctl->bar[4]);
            }
            __syncwarp();
        }
        bar_sync(DELTA ? BAR_HAND : BAR_CHAIN, RK_HAND_N);
        tc_fence_after();
        rk_wait(&ctl->bar[4], parity, ctl, status);   // the last reader of S's terms, which the new part replaces
        if (one) {   // the new part of S
#pragma unroll (DELTA ? 1 : 3)
            for (int term = 0; term < 3; term++)
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
                    rk_mma(tm + TM_S, tm + (term < 2 ? TM_X + 32 * (ks >> 1) + 16 * term + 8 * (ks & 1) : TM_S2 + 8 * ks), kt + (2048 * ks >> 4), rk_idesc(128, true, true), term + ks > 0);
            rk_commit(&ctl->bar[2]);
        }
        __syncwarp();
        bar_sync(BAR_HAND_U, RK_HAND_N);
        tc_fence_after();
        if (one) {   // O's part from this chunk's tokens
#pragma unroll (DELTA ? 1 : 3)
            for (int term = 0; term < 3; term++)
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
                    rk_mma(tm + TM_U, tm + (term == 1 ? TM_UM : TM_UL) + 8 * ks, (term == 2 ? pm : ph) + (32 * ks >> 4), rk_idesc(64, true, false), term + ks > 0);
            rk_commit(&ctl->bar[3]);
        }
        __syncwarp();
        parity ^= 1;
    }
}

template <bool DELTA>
__device__ __forceinline__ void rk_chain(const RecParams &p, uint8_t *sm, RkCtl *ctl, int seq, int h, int32_t beg, int32_t end) {
    const int tid = threadIdx.x, row = tid & 127, half = tid >> 7;
    const uint32_t tl = ctl->tmem + ((uint32_t)(row & 96) << 16);   // the warp's lanes
    float *S0 = reinterpret_cast<float *>(p.state + (int64_t)p.slot[seq] * p.slot_bytes) + ((int64_t)h * REC_HD + row) * REC_HD;
    const int n_chunks = (end - beg + RK_C - 1) / RK_C;
    for (int c = 0; c < min(n_chunks, RK_STAGES); c++) bar_arrive(BAR_EMPTY + c * RK_GROUPS + c % RK_GROUPS, RK_EMPTY_N);
    float S[64];   // value row `row`, keys 64 half ..
    auto load_state = [&]() {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float4 u = *reinterpret_cast<const float4 *>(S0 + 64 * half + 4 * i);
            S[4 * i] = u.x; S[4 * i + 1] = u.y; S[4 * i + 2] = u.z; S[4 * i + 3] = u.w;
        }
    };
    auto store_state = [&]() {
#pragma unroll
        for (int i = 0; i < 16; i++) *reinterpret_cast<float4 *>(S0 + 64 * half + 4 * i) = make_float4(S[4 * i], S[4 * i + 1], S[4 * i + 2], S[4 * i + 3]);
    };
    // v of the chunk at t0, zeros behind the sequence: copied while the chunk before it is worked on
    const uint32_t vdst = (uint32_t)__cvta_generic_to_shared(sm + RK_VS) + tid * 16;
    auto load_v = [&](int32_t t0) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int32_t r = t0 + 16 * i + (tid >> 4);
            rk_cp16_zero(vdst + i * (16 * 256), static_cast<const __nv_bfloat16 *>(p.v) + (int64_t)(r < end ? r : beg) * p.v_stride + (int64_t)h * REC_HD + (tid & 15) * 8, r < end);
        }
    };
    // What this thread wrote to tensor memory is there: the products that read it may go ahead once all have said so.
    auto hand_over = [&](int bar) {
        tm_wait_st();
        tc_fence_before();
        bar_arrive(bar, RK_HAND_N);
    };
    load_v(beg);
    load_state();
    uint32_t ow[16];         // the last chunk's output of tokens 32 half .., pairs of tokens, on its way to memory
    int32_t out_t0 = -1;     // that chunk's first token (-1: nothing pending)
    uint32_t ph = 0;         // parity of the products' barriers
    auto release = [&](int c) {   // chunk c's stage
        const int next = c + RK_STAGES;
        if (next < n_chunks) bar_arrive(BAR_EMPTY + next % RK_STAGES * RK_GROUPS + next % RK_GROUPS, RK_EMPTY_N);
    };
    auto read_out = [&](int c, uint32_t parity) {   // O of chunk c: scale (e^G S q + P U)
        const float *cf = reinterpret_cast<const float *>(sm + c % RK_STAGES * RK_STAGE + RK_COEF);
        rk_wait(&ctl->bar[3], parity, ctl, p.status);
#pragma unroll
        for (int b = 0; b < 2; b++) {
            float u[16], o[16];
            tm_ld16(tl + TM_O1 + 32 * half + 16 * b, u);
            tm_ld16(tl + TM_U + 32 * half + 16 * b, o);
            tm_wait16(u);
            tm_wait16(o);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 cq = *reinterpret_cast<const float4 *>(cf + CF_Q * RK_C + 32 * half + 16 * b + i);
                const __nv_bfloat162 v0 = __floats2bfloat162_rn(fmaf(cq.x, u[i], p.scale * o[i]), fmaf(cq.y, u[i + 1], p.scale * o[i + 1]));
                const __nv_bfloat162 v1 = __floats2bfloat162_rn(fmaf(cq.z, u[i + 2], p.scale * o[i + 2]), fmaf(cq.w, u[i + 3], p.scale * o[i + 3]));
                ow[8 * b + i / 2] = *reinterpret_cast<const uint32_t *>(&v0);
                ow[8 * b + i / 2 + 1] = *reinterpret_cast<const uint32_t *>(&v1);
            }
        }
        release(c);
    };
    const int64_t out_row = (int64_t)p.n_head * REC_HD;
    auto read_last = [&]() {   // with the delta rule a chunk's O is read while the next chunk's X is made
        if (DELTA && out_t0 >= 0) read_out((out_t0 - beg) / RK_C, ph ^ 1);
    };
    auto finish_out = [&]() {
        if (out_t0 < 0) return;
        __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + (int64_t)(out_t0 + 32 * half) * out_row + (int64_t)h * REC_HD + row;
        const int n = end - out_t0 - 32 * half;
        if (!DELTA && n >= 32) {   // (4% there; with the delta rule the longer code costs as much)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                *reinterpret_cast<uint16_t *>(out) = (uint16_t)ow[i];
                *reinterpret_cast<uint16_t *>(out + out_row) = (uint16_t)(ow[i] >> 16);
                out += 2 * out_row;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (2 * i < n) *reinterpret_cast<uint16_t *>(out) = (uint16_t)ow[i];
                if (2 * i + 1 < n) *reinterpret_cast<uint16_t *>(out + out_row) = (uint16_t)(ow[i] >> 16);
                out += 2 * out_row;
            }
        }
        out_t0 = -1;
    };
    for (int c = 0, st = 0; c < n_chunks; c++, st = st == RK_STAGES - 1 ? 0 : st + 1) {
        const int32_t t0 = beg + c * RK_C;
        const float *cf = reinterpret_cast<const float *>(sm + st * RK_STAGE + RK_COEF);
        asm volatile("cp.async.wait_all;" ::: "memory");   // (this thread's part of v: all see it behind the barrier)
        bar_sync(BAR_FULL + st, RK_FULL_N);
        if (cf[CF_N * RK_C + 1] != 0.0f) {
            read_last();
            finish_out();
            store_state();
            bar_sync(BAR_CHAIN, RK_HAND_N);   // and the issuer has read the flag, which the stage's next chunk clears
            load_v(t0 + RK_C);
            rk_serial<DELTA>(p, S0 - row * REC_HD, h, t0, min(end, t0 + RK_C));
            bar_sync(BAR_CHAIN, RK_CHAIN);
            load_state();
            release(c);
            continue;
        }
        // S as bf16 terms
#pragma unroll
        for (int b = 0; b < 4; b++) {
            uint32_t w0[8], w1[8], w2[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float x = S[16 * b + 2 * i], y = S[16 * b + 2 * i + 1];
                w0[i] = take_bf16(x, y);
                w1[i] = take_bf16(x, y);
                if (DELTA) w2[i] = take_bf16(x, y);
            }
            tm_st8(tl + TM_S + 64 * half + 8 * b, w0);
            tm_st8(tl + TM_S + 64 * half + 32 + 8 * b, w1);
            if (DELTA) tm_st8(tl + (half ? TM_U2 : TM_S2) + 8 * b, w2);
        }
        hand_over(BAR_HAND);
        if (DELTA) read_last();
        else finish_out();
        // R = beta (v - e^G X), or u = v: tokens 32 half ..
        float X[32];
        bool row_ok = true;
        __nv_bfloat162 gone = __float2bfloat162_rn(0.0f);   // NaN once a value of w U is not finite
        const uint16_t *vs = reinterpret_cast<const uint16_t *>(sm + RK_VS) + 32 * half * 128 + row;
        if (DELTA) {
            rk_wait(&ctl->bar[0], ph, ctl, p.status);
            float mx = 0.0f, inv;
            tm_ld32(tl + TM_X + 32 * half, X);
            tm_wait_ld(X);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 cx = *reinterpret_cast<const float4 *>(cf + CF_X * RK_C + 32 * half + i);
                const float4 cv = *reinterpret_cast<const float4 *>(cf + CF_V * RK_C + 32 * half + i);
                X[i] = fmaf(cx.x, X[i], cv.x * __uint_as_float((uint32_t)vs[i * 128] << 16));
                X[i + 1] = fmaf(cx.y, X[i + 1], cv.y * __uint_as_float((uint32_t)vs[(i + 1) * 128] << 16));
                X[i + 2] = fmaf(cx.z, X[i + 2], cv.z * __uint_as_float((uint32_t)vs[(i + 2) * 128] << 16));
                X[i + 3] = fmaf(cx.w, X[i + 3], cv.w * __uint_as_float((uint32_t)vs[(i + 3) * 128] << 16));
                mx = fmaxf(fmaxf(mx, fmaxf(fabsf(X[i]), fabsf(X[i + 1]))), fmaxf(fabsf(X[i + 2]), fabsf(X[i + 3])));
            }
            const float s = pow2_scale(mx, inv);
            if (half == 0 && !(fabsf(X[0]) < __int_as_float(0x7f800000))) inv = __int_as_float(0x7fffffff);
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; i++) split_f16(X[16 * b + 2 * i], X[16 * b + 2 * i + 1], s, hi[i], lo[i]);
                tm_st8(tl + TM_X + 32 * half + 8 * b, hi);
                tm_st8(tl + TM_X + 32 * half + 16 + 8 * b, lo);
            }
            if (half == 0) ctl->scale[row] = inv;
            hand_over(BAR_HAND);
            rk_wait(&ctl->bar[1], ph, ctl, p.status);
            load_v(t0 + RK_C);   // (every thread has read its part)
            tm_ld32(tl + TM_U + 32 * half, X);
            tm_wait_ld(X);
            if (half) {
                const float first = ctl->scale[row];
                row_ok = first == first;
                float Y[32];
                tm_ld32(tl + TM_U2, Y);
                tm_wait_ld(Y);
#pragma unroll
                for (int i = 0; i < 32; i++) X[i] = fmaf(first, X[i], inv * Y[i]);
            } else {
                row_ok = inv == inv;
#pragma unroll
                for (int i = 0; i < 32; i++) X[i] *= inv;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 ct = *reinterpret_cast<const float4 *>(cf + CF_T * RK_C + 32 * half + i);
                X[i] *= ct.x;
                X[i + 1] *= ct.y;
                X[i + 2] *= ct.z;
                X[i + 3] *= ct.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; i++) X[i] = __uint_as_float((uint32_t)vs[i * 128] << 16);
        }
        // w U in three terms for the state
#pragma unroll
        for (int b = 0; b < 2; b++) {
            uint32_t w0[8], w1[8], w2[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float4 cw = *reinterpret_cast<const float4 *>(cf + CF_W * RK_C + 32 * half + 16 * b + 2 * i);
                float x = X[16 * b + 2 * i] * cw.x, y = X[16 * b + 2 * i + 1] * cw.y;
                w0[i] = take_bf16(x, y);
                w1[i] = take_bf16(x, y);
                w2[i] = take_bf16(x, y);
                x = X[16 * b + 2 * i + 2] * cw.z;
                y = X[16 * b + 2 * i + 3] * cw.w;
                w0[i + 1] = take_bf16(x, y);
                w1[i + 1] = take_bf16(x, y);
                w2[i + 1] = take_bf16(x, y);
            }
            if (DELTA)
#pragma unroll
                for (int i = 0; i < 8; i++) gone = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&w0[i]), __float2bfloat162_rn(0.0f), gone);
            tm_st8(tl + TM_X + 32 * half + 8 * b, w0);
            tm_st8(tl + TM_X + 32 * half + 16 + 8 * b, w1);
            tm_st8(tl + TM_S2 + 16 * half + 8 * b, w2);
        }
        // (With the delta rule two waits for products lie between a chunk's hand-overs on one barrier.  Without it nothing does: a
        // fast warp's second arrival must not stand for a slow one's first.)
        if (DELTA && row_ok && (*reinterpret_cast<const uint32_t *>(&gone) & 0x7fff7fffu)) *(volatile int32_t *)&ctl->redo = 1;
        hand_over(DELTA ? BAR_HAND : BAR_CHAIN);
        // U in two terms for the output
#pragma unroll
        for (int b = 0; b < 2; b++) {
            uint32_t w0[8], w1[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float x = X[16 * b + 2 * i], y = X[16 * b + 2 * i + 1];
                w0[i] = take_bf16(x, y);
                w1[i] = take_bf16(x, y);
            }
            tm_st8(tl + TM_UL + 16 * half + 8 * b, w0);
            tm_st8(tl + TM_UM + 16 * half + 8 * b, w1);
        }
        hand_over(BAR_HAND_U);
        if (DELTA) finish_out();
        const float eg = cf[CF_N * RK_C];
        rk_wait(&ctl->bar[2], ph, ctl, p.status);
        if (DELTA && *(volatile int32_t *)&ctl->redo) {   // (written before the hand-over that bar[2] stands behind: all see the same)
            rk_wait(&ctl->bar[3], ph, ctl, p.status);   // nothing reads the stage or U's terms any more
            store_state();
            bar_sync(BAR_CHAIN, RK_CHAIN);
            if (tid == 0) ctl->redo = 0;
            rk_serial<DELTA>(p, S0 - row * REC_HD, h, t0, min(end, t0 + RK_C));
            bar_sync(BAR_CHAIN, RK_CHAIN);
            load_state();
            release(c);
            ph ^= 1;
            continue;
        }
        if (!DELTA) load_v(t0 + RK_C);   // (every thread has read its part)
#pragma unroll
        for (int b = 0; b < 2; b++) {
            tm_ld32(tl + TM_S + 64 * half + 32 * b, X);
            tm_wait_ld(X);
#pragma unroll
            for (int i = 0; i < 32; i++) S[32 * b + i] = fmaf(eg, S[32 * b + i], X[i]);
        }
        if (!DELTA) read_out(c, ph);
        out_t0 = t0;
        ph ^= 1;
    }
    read_last();
    finish_out();
    asm volatile("cp.async.wait_all;" ::: "memory");
    store_state();
}

template <bool DELTA>
__global__ void __launch_bounds__(RK_THREADS, 1) k_rec_chunk(const __grid_constant__ RecParams p) {
    extern __shared__ uint8_t rk_raw[];
    uint8_t *sm = rk_raw + ((1024 - ((uint32_t)__cvta_generic_to_shared(rk_raw) & 1023)) & 1023);   // swizzled tiles: 1024-byte atoms
    RkCtl *ctl = reinterpret_cast<RkCtl *>(sm + RK_CTL);
    const int h = blockIdx.x;
    int seq = blockIdx.y;
    if (gridDim.y > 2) {   // the longest sequences first: the blockIdx.y-th by length
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x, n = gridDim.y;
            auto length = [&](int i) {   // + 1; 0 behind the last sequence (whatever cu holds, each sequence gets one place)
                if (i >= n) return 0u;
                const int32_t a = p.cu[i], b = p.cu[i + 1];
                return b > a ? min((uint32_t)b - (uint32_t)a, 0x7fffffffu) + 1 : 1u;
            };
            const uint32_t l0 = length(lane), l1 = length(lane + 32);
            int r0 = 0, r1 = 0;
#pragma unroll
            for (int j = 0; j < 32; j++) {
                const uint32_t a = __shfl_sync(0xffffffffu, l0, j), b = __shfl_sync(0xffffffffu, l1, j);
                r0 += (a > l0 || (a == l0 && j < lane)) + (b > l0);
                r1 += (a >= l1) + (b > l1 || (b == l1 && j < lane));
            }
            if (l0 && r0 == seq) ctl->seq = lane;
            if (l1 && r1 == seq) ctl->seq = lane + 32;
        }
        __syncthreads();
        seq = ctl->seq;
    }
    const int32_t beg = p.cu[seq], end = p.cu[seq + 1];
    if (beg < 0 || end > p.n_rows || beg > end) {
        if (threadIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
        return;
    }
    if (beg == end) return;
    if (threadIdx.x >= RK_ISSUER && threadIdx.x < RK_ISSUER + 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&ctl->tmem)),
                     "r"(TM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (threadIdx.x == 0) {
        ctl->abort = 0;
        ctl->redo = 0;
        for (int i = 0; i < RK_BARS + RK_GROUPS; i++)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(i < RK_BARS ? &ctl->bar[i] : &ctl->scored[i - RK_BARS])) : "memory");
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&ctl->read)), "r"(RK_GT) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x < RK_CHAIN) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(RK_CHAIN_REGS));
        rk_chain<DELTA>(p, sm, ctl, seq, h, beg, end);
        tc_fence_before();
        bar_arrive(BAR_END, RK_HAND_N + RK_GROUPS * RK_GT);
    } else if (threadIdx.x < RK_ISSUER) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(RK_PROD_REGS));
        rk_produce<DELTA>(p, sm, ctl, h, beg, end);
        tc_fence_before();
        bar_arrive(BAR_END, RK_HAND_N + RK_GROUPS * RK_GT);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(RK_ISSUER_REGS));
        if (threadIdx.x >= RK_ISSUER + 32) return;
        rk_issue<DELTA>(sm, ctl, beg, end, p.status);
        bar_sync(BAR_END, RK_HAND_N + RK_GROUPS * RK_GT);
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(ctl->tmem), "r"(TM_COLS) : "memory");
    }
}

cudaError_t launch_rec_chunk(const RecParams &p, cudaStream_t st) {
    auto *k = p.beta ? k_rec_chunk<true> : k_rec_chunk<false>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, RK_SMEM + 1024);
    if (e != cudaSuccess) return e;
    k<<<dim3(p.n_head, p.n_seq), RK_THREADS, RK_SMEM + 1024, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace qkv
