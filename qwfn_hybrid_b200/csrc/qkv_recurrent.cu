// qkv_recurrent.cu -- the recurrent layers' kernels over the engine's state slabs: the short causal
// convolution (k_rec_conv) and linear attention with a decay per head, with or without the delta rule
// (k_rec_step for a few tokens, k_rec_chunk for prompts).
#include "qkv_internal.h"

#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace qkv {

// The sequence of this launch that row r belongs to (cu: device, exclusive sums), or -1.  The bounds
// that are returned are checked against the batch, whatever cu holds.
__device__ __forceinline__ int rec_find(const int32_t *__restrict__ cu, int n_seq, int32_t n_rows, int32_t r, int32_t &beg,
                                        int32_t &end) {
    int lo = 0, hi = n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] > r) hi = mid;
        else lo = mid + 1;
    }
    beg = cu[lo];
    end = cu[lo + 1];
    return beg >= 0 && beg <= r && r < end && end <= n_rows ? lo : -1;
}

// --------------------------------------------------------------------------------- convolution
// y[t][c] = silu(sum_{j=0..3} w[c][j] x[t - 3 + j][c]) along each sequence, the rows before its first
// being the state's history [c][3] (oldest first); of the leading n_norm channels every 128 (a head of
// q or k) are then divided by max(|y|_2, eps).  Bound by bytes: each row in and out once.
// A thread owns VEC channels (16 bytes of a row) and walks R rows with the last three rows in
// registers; 128 channels are 128 / VEC adjacent lanes, so the norm is a few shuffles.  The thread
// that meets a sequence's first row has read the history, so it also writes the new one (from the
// sequence's last three rows) and, for rollbacks, the ones after fewer rows: no second launch and no
// thread waits for another.
template <typename T> struct RecVec;
template <> struct RecVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[4]) {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ void load(const float *p, float (&v)[4]) { unpack(*reinterpret_cast<const uint4 *>(p), v); }
    static __device__ __forceinline__ void store(float *p, const float (&v)[4]) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
template <> struct RecVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16 *p, float (&v)[8]) { unpack(*reinterpret_cast<const uint4 *>(p), v); }
    static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i]     = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

constexpr int RC_THREADS = 256, RC_HIST = 3;

// The history after the sequence's rows [beg, end) for VEC channels: hist_out[c][j] = row end - 3 + j,
// of the old history where that lies before beg.
template <typename T, int VEC>
__device__ __forceinline__ void rec_conv_hist(const RecConvParams &p, const T *x, int32_t beg, int32_t end,
                                              const float (&old)[RC_HIST][VEC], float *out) {
    float v[RC_HIST][VEC];
#pragma unroll
    for (int j = 0; j < RC_HIST; j++) {
        const int32_t r = end - RC_HIST + j;
        if (r >= beg) {
            RecVec<T>::load(x + (int64_t)r * p.x_stride, v[j]);
        } else {
            const int32_t k = r - beg + RC_HIST;   // 0 .. 2: old history
#pragma unroll
            for (int e = 0; e < VEC; e++) v[j][e] = k == 0 ? old[0][e] : k == 1 ? old[1][e] : old[2][e];
        }
    }
    float flat[RC_HIST * VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++)
#pragma unroll
        for (int j = 0; j < RC_HIST; j++) flat[e * RC_HIST + j] = v[j][e];
#pragma unroll
    for (int i = 0; i < RC_HIST * VEC / 4; i++)
        reinterpret_cast<float4 *>(out)[i] = make_float4(flat[4 * i], flat[4 * i + 1], flat[4 * i + 2], flat[4 * i + 3]);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void rk_cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr int RC_AHEAD = 8;   // rows in flight ahead of the one computed, in shared memory: they cost no registers

template <typename T>
__global__ void __launch_bounds__(RC_THREADS, 2) k_rec_conv(const __grid_constant__ RecConvParams p) {
    __shared__ uint4 ring[RC_AHEAD][RC_THREADS];   // a thread reads what it copied: no barrier
    __shared__ int32_t cu[MAX_SEQ + 1];
    constexpr int VEC = RecVec<T>::N, LANES = 128 / VEC;
    const int per_row = p.channels / VEC;   // a multiple of LANES
    const int64_t id = (int64_t)blockIdx.x * RC_THREADS + threadIdx.x;
    const int64_t blk = id / per_row;
    const int c0 = (int)(id % per_row) * VEC;
    const int32_t r_lo = (int32_t)min((int64_t)p.n_rows, blk * p.rows_per), r_hi = min(p.n_rows, r_lo + p.rows_per);
    const T *x = static_cast<const T *>(p.x) + c0;
    T *y = static_cast<T *>(p.y) + c0;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&ring[0][threadIdx.x]);
    auto fetch = [&](int32_t r) {   // row r (or nothing) into its slot: one group per row
        if (r < r_hi) rk_cp16(mine + ((r - r_lo) & (RC_AHEAD - 1)) * (RC_THREADS * 16), x + (int64_t)r * p.x_stride);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < RC_AHEAD; k++) fetch(r_lo + k);
    for (int i = threadIdx.x; i <= p.n_seq; i += RC_THREADS) cu[i] = p.cu[i];
    float w[VEC][4];
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float4 u = __ldg(reinterpret_cast<const float4 *>(p.w) + c0 + e);
        w[e][0] = u.x; w[e][1] = u.y; w[e][2] = u.z; w[e][3] = u.w;
    }
    __syncthreads();
    const bool norm = c0 < p.n_norm;
    const float max_inv = 1.0f / p.eps;
    const unsigned lanes = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    for (int32_t r = r_lo; r < r_hi;) {
        int32_t beg, end;   // rows of the sequence
        const int i = rec_find(cu, p.n_seq, p.n_rows, r, beg, end);
        if (i < 0) {        // a row of no sequence (of this launch)
            fetch(r + RC_AHEAD);
            r++;
            continue;
        }
        float h[RC_HIST + 1][VEC];   // rows r - 3 .. r
        {
            float *state = reinterpret_cast<float *>(p.state + (int64_t)p.slot[i] * p.slot_bytes) + (int64_t)c0 * RC_HIST;
            float old[RC_HIST][VEC];
            if (r - beg < RC_HIST) {
                float flat[RC_HIST * VEC];
#pragma unroll
                for (int k = 0; k < RC_HIST * VEC / 4; k++) {
                    const float4 u = reinterpret_cast<const float4 *>(state)[k];
                    flat[4 * k] = u.x; flat[4 * k + 1] = u.y; flat[4 * k + 2] = u.z; flat[4 * k + 3] = u.w;
                }
#pragma unroll
                for (int e = 0; e < VEC; e++)
#pragma unroll
                    for (int j = 0; j < RC_HIST; j++) old[j][e] = flat[e * RC_HIST + j];
            }
#pragma unroll
            for (int j = 0; j < RC_HIST; j++) {
                const int32_t q = r - RC_HIST + j;
                if (q >= beg) {
                    RecVec<T>::load(x + (int64_t)q * p.x_stride, h[j]);
                } else {
                    const int32_t k = q - beg + RC_HIST;
#pragma unroll
                    for (int e = 0; e < VEC; e++) h[j][e] = k == 0 ? old[0][e] : k == 1 ? old[1][e] : old[2][e];
                }
            }
            if (r == beg) {
                for (int s = 1; s <= min(p.n_save, end - beg); s++)
                    rec_conv_hist<T, VEC>(p, x, beg, end - s, old,
                                          reinterpret_cast<float *>(p.back + ((int64_t)p.slot[i] * p.n_rollback + s - 1) * p.slot_bytes) +
                                              (int64_t)c0 * RC_HIST);
                rec_conv_hist<T, VEC>(p, x, beg, end, old, state);
            }
        }
        const int32_t lim = min(end, r_hi);
        T *yr = y + (int64_t)r * p.channels;
        for (; r < lim; r += 4) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (r + k >= lim) break;
                float (&h0)[VEC] = h[k & 3], (&h1)[VEC] = h[(k + 1) & 3], (&h2)[VEC] = h[(k + 2) & 3], (&v)[VEC] = h[(k + 3) & 3];
                asm volatile("cp.async.wait_group %0;" ::"n"(RC_AHEAD - 1) : "memory");
                RecVec<T>::unpack(ring[(r + k - r_lo) & (RC_AHEAD - 1)][threadIdx.x], v);
                fetch(r + k + RC_AHEAD);
                float o[VEC], ss = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    float a = v[e] * w[e][3];
                    a = fmaf(h0[e], w[e][0], a);
                    a = fmaf(h1[e], w[e][1], a);
                    a = fmaf(h2[e], w[e][2], a);
                    o[e] = a * rcp(1.0f + ex2(a * -1.4426950408889634f));
                    ss = fmaf(o[e], o[e], ss);
                }
                if (norm) {   // the lanes of a head walk the same rows: all of them are here
#pragma unroll
                    for (int m = LANES / 2; m; m >>= 1) ss += __shfl_xor_sync(lanes, ss, m);
                    float inv = rsqrtf(ss);
                    if (inv > max_inv) inv = max_inv;   // (a NaN stays)
#pragma unroll
                    for (int e = 0; e < VEC; e++) o[e] *= inv;
                }
                RecVec<T>::store(yr, o);
                yr += p.channels;
            }
        }
        r = lim;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

cudaError_t launch_rec_conv(RecConvParams &p, bool bf16, int num_sms, cudaStream_t st) {
    const int64_t per_row = p.channels / (bf16 ? 8 : 4), slots = 2 * num_sms;   // CTAs resident at once
    auto grid_of = [&](int64_t r) { return ((p.n_rows + r - 1) / r * per_row + RC_THREADS - 1) / RC_THREADS; };
    // Rows per thread: one while a wave of CTAs holds them all, else what makes waves times rows least, with the
    // start of a walk (its sequence, the three rows before it) counted as eight rows.
    int64_t best = 1;
    if (grid_of(1) > slots)
        for (int64_t r = 4, least = INT64_MAX; r <= 64; r += 4) {
            const int64_t cost = (grid_of(r) + slots - 1) / slots * (r + 8);
            if (cost < least) {
                least = cost;
                best = r;
            }
        }
    p.rows_per = (int32_t)best;
    const unsigned grid = (unsigned)grid_of(best);
    if (bf16) k_rec_conv<__nv_bfloat16><<<grid, RC_THREADS, 0, st>>>(p);
    else k_rec_conv<float><<<grid, RC_THREADS, 0, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------- linear attention
// Per value head with state S [value][key] (key fastest), token by token:
//   S <- e^g S;  u = v, or with the delta rule u = beta (v - S k);  S <- S + u k^T;  o = scale S q.
// Bound by the state, read and written once whatever T is.  A value row of S needs no other row: 8 lanes hold
// a row, each 16 of its 128 keys as four float4 eight apart (a warp's load covers 4 rows in whole 128-byte
// lines), the row's two dot products are three shuffles, and nothing is shared between warps: every load
// of a thread -- its part of S and of the T rows of k, q, v -- is issued before the first use.
constexpr int RT_THREADS = 128, RT_PASS = 2, RT_ROWS = RT_THREADS / 8 * RT_PASS;   // value rows per CTA

template <int T>
__global__ void __launch_bounds__(RT_THREADS) k_rec_step(const __grid_constant__ RecParams p) {
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, sub = lane & 7;
    const int seq = blockIdx.z, h = blockIdx.y, row0 = blockIdx.x * RT_ROWS + wid * 4 * RT_PASS + (lane >> 3);   // and 4 a rows on
    const int hk = h / (p.n_head / p.n_head_k);
    const int64_t off = ((int64_t)h * REC_HD + row0) * REC_HD + sub * 4, r0 = (int64_t)seq * T;
    float *S0 = reinterpret_cast<float *>(p.state + (int64_t)p.slot[seq] * p.slot_bytes) + off;
    float4 S[RT_PASS][4];
#pragma unroll
    for (int a = 0; a < RT_PASS; a++)
#pragma unroll
        for (int j = 0; j < 4; j++) S[a][j] = *reinterpret_cast<const float4 *>(S0 + a * 4 * REC_HD + j * 32);
    const float *k = static_cast<const float *>(p.k) + r0 * p.k_stride + hk * REC_HD + sub * 4;
    const float *q = static_cast<const float *>(p.q) + r0 * p.q_stride + hk * REC_HD + sub * 4;
    const float *v = static_cast<const float *>(p.v) + r0 * p.v_stride + h * REC_HD + row0;
    float4 kf[T][4], qf[T][4];
    float vf[T][RT_PASS], g[T], b[T];
#pragma unroll
    for (int t = 0; t < T; t++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            kf[t][j] = *reinterpret_cast<const float4 *>(k + t * p.k_stride + j * 32);
            qf[t][j] = *reinterpret_cast<const float4 *>(q + t * p.q_stride + j * 32);
        }
#pragma unroll
        for (int a = 0; a < RT_PASS; a++) vf[t][a] = v[t * p.v_stride + a * 4];
        g[t] = p.g[(r0 + t) * p.n_head + h];
        b[t] = p.beta ? p.beta[(r0 + t) * p.n_head + h] : 0.0f;
    }
    auto store_state = [&](float *dst) {
#pragma unroll
        for (int a = 0; a < RT_PASS; a++)
#pragma unroll
            for (int j = 0; j < 4; j++) *reinterpret_cast<float4 *>(dst + a * 4 * REC_HD + j * 32) = S[a][j];
    };
    auto back = [&](int s) {   // rollback snapshot s - 1: the state s tokens back
        return reinterpret_cast<float *>(p.back + ((int64_t)p.slot[seq] * p.n_rollback + s - 1) * p.slot_bytes) + off;
    };
    if (T <= p.n_save) store_state(back(T));
    float *out = static_cast<float *>(p.out) + (r0 * p.n_head + h) * REC_HD + row0;
#pragma unroll
    for (int t = 0; t < T; t++) {
        const float eg = expf(g[t]);
#pragma unroll
        for (int a = 0; a < RT_PASS; a++) {
            float u = vf[t][a], d = 0.0f, o = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                S[a][j].x *= eg;
                S[a][j].y *= eg;
                S[a][j].z *= eg;
                S[a][j].w *= eg;
            }
            if (p.beta) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    d = fmaf(S[a][j].x, kf[t][j].x, d);
                    d = fmaf(S[a][j].y, kf[t][j].y, d);
                    d = fmaf(S[a][j].z, kf[t][j].z, d);
                    d = fmaf(S[a][j].w, kf[t][j].w, d);
                }
#pragma unroll
                for (int m = 4; m; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
                u = b[t] * (u - d);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                S[a][j].x = fmaf(u, kf[t][j].x, S[a][j].x);
                S[a][j].y = fmaf(u, kf[t][j].y, S[a][j].y);
                S[a][j].z = fmaf(u, kf[t][j].z, S[a][j].z);
                S[a][j].w = fmaf(u, kf[t][j].w, S[a][j].w);
                o = fmaf(S[a][j].x, qf[t][j].x, o);
                o = fmaf(S[a][j].y, qf[t][j].y, o);
                o = fmaf(S[a][j].z, qf[t][j].z, o);
                o = fmaf(S[a][j].w, qf[t][j].w, o);
            }
#pragma unroll
            for (int m = 4; m; m >>= 1) o += __shfl_xor_sync(0xffffffffu, o, m);
            if (sub == 0) out[(int64_t)t * p.n_head * REC_HD + a * 4] = o * p.scale;
        }
        if (t == T - 1) store_state(S0);
        else if (T - 1 - t <= p.n_save) store_state(back(T - 1 - t));
    }
}

cudaError_t launch_rec_step(const RecParams &p, cudaStream_t st) {
    const dim3 grid(REC_HD / RT_ROWS, p.n_head, p.n_seq);
    switch (p.T) {
        case 1: k_rec_step<1><<<grid, RT_THREADS, 0, st>>>(p); break;
        case 2: k_rec_step<2><<<grid, RT_THREADS, 0, st>>>(p); break;
        case 3: k_rec_step<3><<<grid, RT_THREADS, 0, st>>>(p); break;
        default: k_rec_step<4><<<grid, RT_THREADS, 0, st>>>(p); break;
    }
    count_launches(1);
    return cudaGetLastError();
}

// ------------------------------------------------------------------------ chunked linear attention
// 64 tokens at a time.  With G = sums of g inside the chunk (G_C: the whole chunk's) and S the state before it,
//   A_ij = beta_i (k_i . k_j) e^(G_i - G_j) for j < i,   T = (1 + A)^-1   (lower triangular),
//   U = T R,  R_j = beta_j (v_j - e^(G_j) S k_j)          (without the delta rule U = V),
//   o_i = scale (e^(G_i) S q_i + sum_{j <= i} (q_i . k_j) e^(G_i - G_j) u_j),
//   S  <- e^(G_C) S + sum_j e^(G_C - G_j) u_j k_j^T.
// A CTA owns RK_NW * 16 value rows of one head of one sequence and walks its chunks; value rows need nothing
// from one another, so heads and sequences fill the GPU.  Everything without S -- k and q as f16,
// the scores P, T -- is made by RK_PROD producer threads one chunk ahead (two stages in shared memory); the chain
// through S is carried by RK_NW warps of 16 value rows each, wholly in registers: with value rows as the M
// of every product the accumulator of one product (rows: values, columns: tokens or keys) is, register for
// register, the A operand of the next (S -> S k -> R -> U -> S), so the chain has no shared memory,
// shuffle or barrier between its products.  The warps meet at named barriers (no spinning).
// Why mma.sync and not tcgen05: the chain is serial, five dependent products of 16 x 64 x 128 or less per warp
// and chunk; through tensor memory every one of them would add a commit, a wait and a round trip of
// tcgen05.ld and a store, which cost more than these products.
//
// Precision.  bf16 inputs are exact in f16 once a power of two has brought the row's largest value to
// [1, 2); S, R, T and U enter as two f16 terms of a row scaled to [2^12, 2^13) (hi + lo: 22 bits), three
// products where both operands are split, so state and U keep 32-bit accuracy with 16-bit instructions.  The output
// is rounded to bf16, so its two products take the leading term alone (11 bits against 8).  Sums are F32;
// the state is scaled and added outside the tensor cores (their sums are truncated).  G is summed in
// 64 bits and kept as two floats: e^(G_i - G_j) needs the difference, not the rounded sums.
//
// A zero of T or P times a NaN is a NaN, so a chunk with a non-finite input would spread it to earlier
// tokens; such chunks are flagged by the producers and run token by token from global memory.
constexpr int RK_C = 64, RK_NW = 4, RK_GROUPS = 3, RK_GT = 128;    // RK_GROUPS producer groups of RK_GT threads
constexpr int RK_PROD = RK_GROUPS * RK_GT, RK_THREADS = RK_PROD + RK_NW * 32;
constexpr int RK_ROWS = RK_NW * 16;
// a stage (one per group): k, q, P, T (two terms) and v of a chunk, CF_N arrays of RK_C floats, e^(G_C), the flag
constexpr int RK_K = 0, RK_Q = 16384, RK_P = 32768, RK_TH = 40960, RK_TL = 49152, RK_V = 57344;
constexpr int RK_COEF = RK_V + RK_C * RK_ROWS * 2;
enum { CF_G, CF_V, CF_T, CF_Q, CF_W, CF_K, CF_B, CF_N };
constexpr int RK_STAGE = RK_COEF + CF_N * RK_C * 4 + 128;
// a group's scratch: A, then T, as 16 x 16 tiles (per 32 x 32 block: diagonal, below, diagonal), and per-token values
constexpr int RK_PITCH = 20, RK_TILE = 16 * RK_PITCH;
constexpr int RK_SCRATCH = 6 * RK_TILE * 4 + 6 * RK_C * 4;
constexpr int RK_SMEM = RK_GROUPS * (RK_STAGE + RK_SCRATCH);
static_assert(RK_SMEM <= 232448, "shared memory of a CTA");
constexpr int RK_PROD_REGS = 96, RK_CHAIN_REGS = 224;   // of 128 at launch: 384 x 96 + 128 x 224 = 512 x 128
enum { BAR_FULL = 1, BAR_EMPTY = BAR_FULL + RK_GROUPS, BAR_PROD = BAR_EMPTY + RK_GROUPS };
constexpr int RK_PAIR = RK_GT + RK_NW * 32;             // threads that meet at a stage's barriers

__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void stsm4t(uint32_t addr, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The power of two that brings a row whose largest magnitude is m to [2^TE, 2^(TE+1)), and its inverse
// (both normal numbers; rows below 2^(TE-126) are left smaller).
template <int TE>
__device__ __forceinline__ float pow2_scale(float m, float &inv) {
    const int e = (__float_as_int(m) >> 23) & 255;
    const int f = min(254 + TE - e, 253);
    inv = __int_as_float((254 - f) << 23);
    return __int_as_float(f << 23);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void split_f16(float a, float b, float s, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a * s, b * s);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = pack_f16(fmaf(a, s, -f.x), fmaf(b, s, -f.y));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// Row scales of an accumulator tile set (rows g and g + 8 of the lane's quad).
template <int N>
__device__ __forceinline__ void row_scales(const float (&x)[N][4], float &s0, float &s1, float &i0, float &i1) {
    float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
    for (int n = 0; n < N; n++) {
        m0 = fmaxf(m0, fmaxf(fabsf(x[n][0]), fabsf(x[n][1])));
        m1 = fmaxf(m1, fmaxf(fabsf(x[n][2]), fabsf(x[n][3])));
    }
    s0 = pow2_scale<12>(quad_max(m0), i0);
    s1 = pow2_scale<12>(quad_max(m1), i1);
}

// Sixteen words of bf16 pairs, four lanes holding a row of 128 (lane l its 16-byte chunks l, l + 4, l + 8, l + 12).
// Bits of the row's largest magnitude (a NaN is above infinity).
__device__ __forceinline__ uint32_t rk_row_max(const uint4 (&u)[4]) {
    uint32_t m[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        m[i] = __vmaxu2(__vmaxu2(u[i].x & 0x7fff7fffu, u[i].y & 0x7fff7fffu), __vmaxu2(u[i].z & 0x7fff7fffu, u[i].w & 0x7fff7fffu));
    return __vmaxu2(__vmaxu2(m[0], m[1]), __vmaxu2(m[2], m[3]));
}
// The row to f16, times a power of two.
__device__ __forceinline__ void rk_row_f16(const uint4 (&u)[4], float s, uint8_t *dst, int l, int sw) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = pack_f16(__uint_as_float(w[j] << 16) * s, __uint_as_float(w[j] & 0xffff0000u) * s);
        *reinterpret_cast<uint4 *>(dst + (((l + 4 * i) ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}
// The lane's four columns of a 16 x 16 by 16 x 8 product: row a, columns b (pitch RK_PITCH).
__device__ __forceinline__ float4 rk_block(const float *a, const float *b) {
    float4 d = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k4 = 0; k4 < 4; k4++) {
        const float4 u = *reinterpret_cast<const float4 *>(a + 4 * k4);
        const float x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float4 y = *reinterpret_cast<const float4 *>(b + (4 * k4 + k) * RK_PITCH);
            d.x = fmaf(x[k], y.x, d.x);
            d.y = fmaf(x[k], y.y, d.y);
            d.z = fmaf(x[k], y.z, d.z);
            d.w = fmaf(x[k], y.w, d.w);
        }
    }
    return d;
}

// A producer group: chunks grp, grp + RK_GROUPS, ... of the sequence, each into the group's own stage.
template <bool DELTA>
__device__ __forceinline__ void rk_produce(const RecParams &p, uint8_t *sm, int h, int row0, int32_t beg, int32_t end) {
    const int grp = threadIdx.x / RK_GT, tid = threadIdx.x % RK_GT, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
    const int hk = h / (p.n_head / p.n_head_k);
    uint8_t *sg = sm + grp * RK_STAGE;
    const uint32_t su = (uint32_t)__cvta_generic_to_shared(sg);
    float *cf = reinterpret_cast<float *>(sg + RK_COEF);
    float *As = reinterpret_cast<float *>(sm + RK_GROUPS * RK_STAGE + grp * RK_SCRATCH);
    float *gs = As + 6 * RK_TILE, *bs = gs + RK_C, *iK = bs + RK_C, *iQ = iK + RK_C;
    float2 *G2 = reinterpret_cast<float2 *>(iQ + RK_C);   // sums of g up to a token, as two floats
    // This thread's rows of k and q: this one and 32 below (a permutation within eight: the two rows of eight lanes
    // differ in bit 2, so their swizzled 16-byte stores meet different banks), and of v.
    const int x = tid >> 2, row = (x & ~7) | ((x & 1) << 2) | ((x >> 1) & 3);
    const int32_t first = beg + grp * RK_C;
    const __nv_bfloat16 *kp = static_cast<const __nv_bfloat16 *>(p.k) + (int64_t)(first + row) * p.k_stride + (int64_t)hk * REC_HD + t * 8;
    const __nv_bfloat16 *qp = static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)(first + row) * p.q_stride + (int64_t)hk * REC_HD + t * 8;
    const __nv_bfloat16 *vp = static_cast<const __nv_bfloat16 *>(p.v) + (int64_t)(first + (tid >> 3)) * p.v_stride + (int64_t)h * REC_HD + row0 + (tid & 7) * 8;
    // This warp's 16 x 16 tiles of scores, on and below the diagonal: ten of q k^T, then (delta rule) ten of k k^T,
    // of which six lie in the two 32 x 32 blocks of T (tib / 2 == tjb / 2).
    constexpr int NT = DELTA ? 20 : 10;
    const int m = lane >> 3, r = lane & 7;
    for (int32_t t0 = first; t0 < end; t0 += RK_GROUPS * RK_C) {
        uint4 ku[2][4], qu[2][4];
        float gu = 0.0f, bu = 0.0f;
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const bool ok = t0 + 32 * a + row < end;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ku[a][i] = ok ? *reinterpret_cast<const uint4 *>(kp + 32 * a * p.k_stride + 32 * i) : make_uint4(0, 0, 0, 0);
                qu[a][i] = ok ? *reinterpret_cast<const uint4 *>(qp + 32 * a * p.q_stride + 32 * i) : make_uint4(0, 0, 0, 0);
            }
        }
        if (tid < RK_C && t0 + tid < end) {
            gu = p.g[(int64_t)(t0 + tid) * p.n_head + h];
            if (DELTA) bu = p.beta[(int64_t)(t0 + tid) * p.n_head + h];
        }
        bar_sync(BAR_EMPTY + grp, RK_PAIR);
#pragma unroll
        for (int i = 0; i < 4; i++) {   // v as it is, zeros behind the sequence
            const int vr = 16 * i + (tid >> 3), ch = tid & 7;
            const uint32_t off = RK_V + vr * (RK_ROWS * 2) + ((ch ^ (vr & 7)) << 4);
            if (t0 + vr < end) rk_cp16(su + off, vp + 16 * i * p.v_stride);
            else *reinterpret_cast<uint4 *>(sg + off) = make_uint4(0, 0, 0, 0);
        }
        kp += RK_GROUPS * RK_C * p.k_stride;
        qp += RK_GROUPS * RK_C * p.q_stride;
        vp += RK_GROUPS * RK_C * p.v_stride;
        bool bad = false;
        if (tid == 0) cf[CF_N * RK_C + 1] = 0.0f;
#pragma unroll
        for (int a = 0; a < 2; a++) {
            uint32_t mk = rk_row_max(ku[a]), mq = rk_row_max(qu[a]);
            mk = __vmaxu2(mk, __shfl_xor_sync(0xffffffffu, mk, 1));
            mq = __vmaxu2(mq, __shfl_xor_sync(0xffffffffu, mq, 1));
            mk = __vmaxu2(mk, __shfl_xor_sync(0xffffffffu, mk, 2));
            mq = __vmaxu2(mq, __shfl_xor_sync(0xffffffffu, mq, 2));
            mk = max(mk & 0xffffu, mk >> 16);
            mq = max(mq & 0xffffu, mq >> 16);
            bad |= max(mk, mq) >= 0x7f80u;
            float ik, iq;
            const float sk = pow2_scale<0>(__uint_as_float(mk << 16), ik), sq = pow2_scale<0>(__uint_as_float(mq << 16), iq);
            rk_row_f16(ku[a], sk, sg + RK_K + (32 * a + row) * 256, t, row & 7);
            rk_row_f16(qu[a], sq, sg + RK_Q + (32 * a + row) * 256, t, row & 7);
            if (t == 0) {
                iK[32 * a + row] = ik;
                iQ[32 * a + row] = iq;
            }
        }
        if (tid < RK_C) {
            // in base 2; below 2^-184 = 0: the clamp keeps sums and differences finite.  A growing state
            // (g > 0) would leave the range of the f16 scores: flagged, as what is not finite
            gs[tid] = fmaxf(gu, -128.0f) * 1.4426950408889634f;
            bs[tid] = bu;
            bad |= !(gu <= 0.0f) || !(fabsf(bu) <= 3.0e38f);
        }
        bar_sync(BAR_PROD + grp, RK_GT);
        if (bad) cf[CF_N * RK_C + 1] = 1.0f;
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
        // Two passes over the warp's tiles (ids wid + 4 k), as registers allow.
#pragma unroll
        for (int pass = 0; pass < (DELTA ? 2 : 1); pass++) {
            constexpr int PER = 3;
            const int k0 = 3 * pass, id0 = wid + 4 * k0;
            float acc[PER][2][4];
            uint32_t arow[PER], brow[PER];
            int tib[PER], tjb[PER];
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int id = min(id0 + 4 * k, NT - 1), tt = id < 10 ? id : id - 10;
                tib[k] = tt < 1 ? 0 : tt < 3 ? 1 : tt < 6 ? 2 : 3;
                tjb[k] = tt - tib[k] * (tib[k] + 1) / 2;
                arow[k] = su + (id < 10 ? RK_Q : RK_K) + (16 * tib[k] + (m & 1) * 8 + r) * 256;
                brow[k] = su + RK_K + (16 * tjb[k] + (m >> 1) * 8 + r) * 256;
#pragma unroll
                for (int n = 0; n < 2; n++) acc[k][n][0] = acc[k][n][1] = acc[k][n][2] = acc[k][n][3] = 0.0f;
            }
#pragma unroll
            for (int kk = 0; kk < 8; kk++) {
                uint32_t fa[PER][4], fb[PER][4];
#pragma unroll
                for (int k = 0; k < PER; k++)
                    if (4 * (k0 + k) + 4 <= NT || id0 + 4 * k < NT) {
                        ldsm4(fa[k], arow[k] + (((2 * kk + (m >> 1)) ^ r) << 4));
                        ldsm4(fb[k], brow[k] + (((2 * kk + (m & 1)) ^ r) << 4));
                    }
#pragma unroll
                for (int k = 0; k < PER; k++)
                    if (4 * (k0 + k) + 4 <= NT || id0 + 4 * k < NT) {
                        mma_f16(acc[k][0], fa[k], fb[k][0], fb[k][1]);
                        mma_f16(acc[k][1], fa[k], fb[k][2], fb[k][3]);
                    }
            }
            if (pass == 0) {
                bar_sync(BAR_PROD + grp, RK_GT);
                if (tid < RK_C) {
                    const float2 mine = G2[tid], last = G2[RK_C - 1];
                    const float mik = iK[tid], miq = iQ[tid], mb = bs[tid];
                    const float gam = ex2(mine.x) * fmaf(mine.y, 0.6931471805599453f, 1.0f);
                    cf[CF_G * RK_C + tid] = gam;
                    cf[CF_V * RK_C + tid] = mb;
                    cf[CF_Q * RK_C + tid] = p.scale * miq;
                    cf[CF_W * RK_C + tid] = ex2((last.x - mine.x) + (last.y - mine.y));
                    cf[CF_K * RK_C + tid] = mik;
                    cf[CF_B * RK_C + tid] = -mb * mik;
                    if (tid == RK_C - 1) cf[CF_N * RK_C] = gam;
                }
            }
            // times e^(G_i - G_j); everything is read before anything is written
            float4 cg[PER][2];
            float2 rg[PER][2];
#pragma unroll
            for (int k = 0; k < PER; k++) {
                rg[k][0] = G2[16 * tib[k] + g];
                rg[k][1] = G2[16 * tib[k] + g + 8];
#pragma unroll
                for (int n = 0; n < 2; n++) cg[k][n] = *reinterpret_cast<const float4 *>(G2 + 16 * tjb[k] + 8 * n + 2 * t);
            }
            float kb[PER][2];
            float2 kj[PER][2];
#pragma unroll
            for (int k = 0; k < PER; k++)
                if (k0 + k >= 2) {   // tiles of k k^T begin with the third
                    kb[k][0] = -bs[16 * tib[k] + g] * iK[16 * tib[k] + g];
                    kb[k][1] = -bs[16 * tib[k] + g + 8] * iK[16 * tib[k] + g + 8];
#pragma unroll
                    for (int n = 0; n < 2; n++) kj[k][n] = *reinterpret_cast<const float2 *>(iK + 16 * tjb[k] + 8 * n + 2 * t);
                }
#pragma unroll
            for (int k = 0; k < PER; k++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    float *a = acc[k][n];
                    a[0] *= ex2((rg[k][0].x - cg[k][n].x) + (rg[k][0].y - cg[k][n].y));
                    a[1] *= ex2((rg[k][0].x - cg[k][n].z) + (rg[k][0].y - cg[k][n].w));
                    a[2] *= ex2((rg[k][1].x - cg[k][n].x) + (rg[k][1].y - cg[k][n].y));
                    a[3] *= ex2((rg[k][1].x - cg[k][n].z) + (rg[k][1].y - cg[k][n].w));
                    if (tib[k] == tjb[k]) {
                        const int j = 8 * n + 2 * t;
                        a[0] = j <= g ? a[0] : 0.0f;
                        a[1] = j < g ? a[1] : 0.0f;
                        a[2] = j <= g + 8 ? a[2] : 0.0f;
                        a[3] = j < g + 8 ? a[3] : 0.0f;
                    }
                }
#pragma unroll
            for (int k = 0; k < PER; k++)
                if (4 * (k0 + k) + 4 <= NT || id0 + 4 * k < NT) {
                    const int i0 = 16 * tib[k] + g;
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const float *a = acc[k][n];
                        const int off = i0 * 128 + (((2 * tjb[k] + n) ^ (g & 7)) << 4) + t * 4;   // row i0 + 8: the same swizzle
                        if (4 * (k0 + k) + 4 <= 10 || id0 + 4 * k < 10) {
                            *reinterpret_cast<uint32_t *>(sg + RK_P + off) = pack_f16(a[0], a[1]);
                            *reinterpret_cast<uint32_t *>(sg + RK_P + off + 1024) = pack_f16(a[2], a[3]);
                        } else if (tib[k] >= 2 && tjb[k] < 2) {   // A's lower left quarter, |.| <= 512 without k's scales and beta
                            uint32_t hi, lo;
                            split_f16(a[0], a[1], 1.0f, hi, lo);
                            *reinterpret_cast<uint32_t *>(sg + RK_TH + off) = hi;
                            *reinterpret_cast<uint32_t *>(sg + RK_TL + off) = lo;
                            split_f16(a[2], a[3], 1.0f, hi, lo);
                            *reinterpret_cast<uint32_t *>(sg + RK_TH + off + 1024) = hi;
                            *reinterpret_cast<uint32_t *>(sg + RK_TL + off + 1024) = lo;
                        } else {   // -A, tile 3 block + 0, 1, 2
                            float *o = As + ((tib[k] >> 1) * 3 + (tib[k] & 1) + (tjb[k] & 1)) * RK_TILE + g * RK_PITCH + 8 * n + 2 * t;
                            *reinterpret_cast<float2 *>(o) = make_float2(a[0] * kb[k][0] * kj[k][n].x, a[1] * kb[k][0] * kj[k][n].y);
                            *reinterpret_cast<float2 *>(o + 8 * RK_PITCH) = make_float2(a[2] * kb[k][1] * kj[k][n].x, a[3] * kb[k][1] * kj[k][n].y);
                        }
                    }
                }
        }
        if (DELTA) {
            bar_sync(BAR_PROD + grp, RK_GT);
            // T's two diagonal 32 x 32 blocks, in place of A.  The four 16 x 16 blocks on the diagonal by forward
            // substitution, x_i = [i = column] - sum_{j < i} A_ij x_j, one per warp, a column per lane;
            if (lane < 16) {
                float *a = As + ((wid >> 1) * 3 + (wid & 1) * 2) * RK_TILE;
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float s0 = i == lane ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
                    for (int j = 0; j < i; j += 4) {
                        const float4 u = *reinterpret_cast<const float4 *>(a + i * RK_PITCH + j);
                        s0 = fmaf(u.x, y[j], s0);
                        if (j + 1 < i) s1 = fmaf(u.y, y[j + 1], s1);
                        if (j + 2 < i) s0 = fmaf(u.z, y[j + 2], s0);
                        if (j + 3 < i) s1 = fmaf(u.w, y[j + 3], s1);
                    }
                    y[i] = s0 + s1;
                }
                __syncwarp(0xffffu);
#pragma unroll
                for (int i = 0; i < 16; i++) a[i * RK_PITCH + lane] = y[i];
            }
            bar_sync(BAR_PROD + grp, RK_GT);
            {   // then T_10 = -T_11 A_10 T_00, eight columns per warp
                float *tb = As + (wid >> 1) * 3 * RK_TILE, *o = tb + RK_TILE;
                const int i = lane >> 1, col = (wid & 1) * 8 + (lane & 1) * 4;
                const float4 u = rk_block(o + i * RK_PITCH, tb + col);
                bar_sync(BAR_PROD + grp, RK_GT);
                *reinterpret_cast<float4 *>(o + i * RK_PITCH + col) = u;
                __syncwarp();
                const float4 w = rk_block(tb + 2 * RK_TILE + i * RK_PITCH, o + col);
                __syncwarp();
                *reinterpret_cast<float4 *>(o + i * RK_PITCH + col) = w;
            }
            bar_sync(BAR_PROD + grp, RK_GT);
            {   // as two f16 terms of scaled rows: row tid / 2, sixteen columns (none right of the diagonal blocks)
                const int i = tid >> 1, half = tid & 1;
                const bool low = i & 16, in_ = low || !half;
                const float *a = As + ((i >> 5) * 3 + (low ? 1 + half : 0)) * RK_TILE + (i & 15) * RK_PITCH;
                float y[16], mx = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float4 u = *reinterpret_cast<const float4 *>(a + 4 * k);
                    y[4 * k] = u.x; y[4 * k + 1] = u.y; y[4 * k + 2] = u.z; y[4 * k + 3] = u.w;
                }
#pragma unroll
                for (int k = 0; k < 16; k++) mx = fmaxf(mx, fabsf(y[k]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                float inv;
                const float s = pow2_scale<12>(mx, inv);
                if (in_) {
#pragma unroll
                    for (int c8 = 0; c8 < 2; c8++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) split_f16(y[8 * c8 + 2 * k], y[8 * c8 + 2 * k + 1], s, hi[k], lo[k]);
                        const int off = i * 128 + ((((i >> 5) * 4 + half * 2 + c8) ^ (i & 7)) << 4);
                        *reinterpret_cast<uint4 *>(sg + RK_TH + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(sg + RK_TL + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                if (!half) cf[CF_T * RK_C + i] = inv;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        bar_arrive(BAR_FULL + grp, RK_PAIR);
    }
}

// A flagged chunk, token by token, everything from global memory (S too: held in an array that a call
// takes, it would live in local memory on the ordinary path as well).
template <bool DELTA>
__device__ __noinline__ void rk_serial(const RecParams &p, float *S0, int h, int dv, int32_t t0, int32_t t1) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int hk = h / (p.n_head / p.n_head_k);
    float2 *S = reinterpret_cast<float2 *>(S0 + g * REC_HD + 2 * t), *Sb = reinterpret_cast<float2 *>(S0 + (g + 8) * REC_HD + 2 * t);
    for (int32_t r = t0; r < t1; r++) {
        const __nv_bfloat162 *k = reinterpret_cast<const __nv_bfloat162 *>(static_cast<const __nv_bfloat16 *>(p.k) + (int64_t)r * p.k_stride + hk * REC_HD);
        const __nv_bfloat162 *q = reinterpret_cast<const __nv_bfloat162 *>(static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)r * p.q_stride + hk * REC_HD);
        const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(p.v) + (int64_t)r * p.v_stride + h * REC_HD + dv;
        const float eg = expf(p.g[(int64_t)r * p.n_head + h]);
        float u0 = __bfloat162float(v[g]), u1 = __bfloat162float(v[g + 8]), d0 = 0.0f, d1 = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int n = 0; n < 16; n++) {
            const float2 kf = __bfloat1622float2(k[4 * n + t]);
            d0 += S[4 * n].x * eg * kf.x + S[4 * n].y * eg * kf.y;
            d1 += Sb[4 * n].x * eg * kf.x + Sb[4 * n].y * eg * kf.y;
        }
        if (DELTA) {
            const float b = p.beta[(int64_t)r * p.n_head + h];
            u0 = b * (u0 - quad_sum(d0));
            u1 = b * (u1 - quad_sum(d1));
        }
        for (int n = 0; n < 16; n++) {
            const float2 kf = __bfloat1622float2(k[4 * n + t]), qf = __bfloat1622float2(q[4 * n + t]);
            const float2 a = S[4 * n], b = Sb[4 * n];
            const float2 x = make_float2(fmaf(u0, kf.x, a.x * eg), fmaf(u0, kf.y, a.y * eg));
            const float2 y = make_float2(fmaf(u1, kf.x, b.x * eg), fmaf(u1, kf.y, b.y * eg));
            S[4 * n] = x;
            Sb[4 * n] = y;
            o0 += x.x * qf.x + x.y * qf.y;
            o1 += y.x * qf.x + y.y * qf.y;
        }
        o0 = quad_sum(o0);
        o1 = quad_sum(o1);
        if (t == 0) {
            __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(p.out) + ((int64_t)r * p.n_head + h) * REC_HD + dv;
            o[g] = __float2bfloat16_rn(o0 * p.scale);
            o[g + 8] = __float2bfloat16_rn(o1 * p.scale);
        }
    }
}

template <bool DELTA>
__device__ __forceinline__ void rk_chain(const RecParams &p, uint8_t *sm, int seq, int h, int row0, int32_t beg, int32_t end) {
    const int lane = threadIdx.x & 31, wid = (threadIdx.x - RK_PROD) >> 5, g = lane >> 2, t = lane & 3;
    const int m = lane >> 3, r = lane & 7;
    const uint32_t smu = (uint32_t)__cvta_generic_to_shared(sm);
    const int dv = row0 + 16 * wid;
    float *S0 = reinterpret_cast<float *>(p.state + (int64_t)p.slot[seq] * p.slot_bytes) + ((int64_t)h * REC_HD + dv) * REC_HD;
    const int n_chunks = (end - beg + RK_C - 1) / RK_C;
    for (int c = 0; c < min(n_chunks, RK_GROUPS); c++) bar_arrive(BAR_EMPTY + c, RK_PAIR);
    float S[16][4];   // rows dv + g and dv + g + 8, keys 8 n + 2 t, + 1
    auto load_state = [&]() {
#pragma unroll
        for (int n = 0; n < 16; n++) {
            const float2 a = *reinterpret_cast<const float2 *>(S0 + g * REC_HD + 8 * n + 2 * t);
            const float2 b = *reinterpret_cast<const float2 *>(S0 + (g + 8) * REC_HD + 8 * n + 2 * t);
            S[n][0] = a.x; S[n][1] = a.y; S[n][2] = b.x; S[n][3] = b.y;
        }
    };
    auto store_state = [&]() {
#pragma unroll
        for (int n = 0; n < 16; n++) {
            *reinterpret_cast<float2 *>(S0 + g * REC_HD + 8 * n + 2 * t) = make_float2(S[n][0], S[n][1]);
            *reinterpret_cast<float2 *>(S0 + (g + 8) * REC_HD + 8 * n + 2 * t) = make_float2(S[n][2], S[n][3]);
        }
    };
    load_state();
    for (int c = 0, st = 0; c < n_chunks; c++, st = st == RK_GROUPS - 1 ? 0 : st + 1) {
        const int32_t t0 = beg + c * RK_C;
        uint8_t *sg = sm + st * RK_STAGE;
        const uint32_t su = smu + st * RK_STAGE;
        const float *cf = reinterpret_cast<const float *>(sg + RK_COEF);
        bar_sync(BAR_FULL + st, RK_PAIR);
        const uint32_t vrow = su + RK_V + ((m >> 1) * 8 + r) * (RK_ROWS * 2) + (((2 * wid + (m & 1)) ^ r) << 4);
        uint32_t v[4][4];   // v of 16 tokens each: rows g, g + 8 of tokens 0 .. 7, then of 8 .. 15
        uint32_t vm = 0;
#pragma unroll
        for (int np = 0; np < 4; np++) {
            ldsm4t(v[np], vrow + np * 16 * (RK_ROWS * 2));
#pragma unroll
            for (int k = 0; k < 4; k++) vm = __vmaxu2(vm, v[np][k] & 0x7fff7fffu);
        }
        if (__any_sync(0xffffffffu, (vm & 0xffffu) >= 0x7f80u || vm >= 0x7f800000u || cf[CF_N * RK_C + 1] != 0.0f)) {
            store_state();
            rk_serial<DELTA>(p, S0, h, dv, t0, min(end, t0 + RK_C));
            load_state();
            if (c + RK_GROUPS < n_chunks) bar_arrive(BAR_EMPTY + st, RK_PAIR);
            continue;
        }
        float s0, s1, is0, is1;
        row_scales(S, s0, s1, is0, is1);
        float X[8][4], O[8][4];
#pragma unroll
        for (int n = 0; n < 8; n++) X[n][0] = X[n][1] = X[n][2] = X[n][3] = O[n][0] = O[n][1] = O[n][2] = O[n][3] = 0.0f;
        // X = S K^T (delta rule), O = S Q^T (the leading f16 term alone)
        const uint32_t krow = su + ((m >> 1) * 8 + r) * 256;
#pragma unroll
        for (int kk = 0; kk < 8; kk++) {
            uint32_t hi[4], lo[4], b[4];
            if (DELTA) {
                split_f16(S[2 * kk][0], S[2 * kk][1], s0, hi[0], lo[0]);
                split_f16(S[2 * kk][2], S[2 * kk][3], s1, hi[1], lo[1]);
                split_f16(S[2 * kk + 1][0], S[2 * kk + 1][1], s0, hi[2], lo[2]);
                split_f16(S[2 * kk + 1][2], S[2 * kk + 1][3], s1, hi[3], lo[3]);
#pragma unroll
                for (int np = 0; np < 4; np++) {
                    ldsm4(b, krow + RK_K + np * 4096 + (((2 * kk + (m & 1)) ^ r) << 4));
                    mma_f16(X[2 * np], hi, b[0], b[1]);
                    mma_f16(X[2 * np + 1], hi, b[2], b[3]);
                    mma_f16(X[2 * np], lo, b[0], b[1]);
                    mma_f16(X[2 * np + 1], lo, b[2], b[3]);
                }
            } else {
                hi[0] = pack_f16(S[2 * kk][0] * s0, S[2 * kk][1] * s0);
                hi[1] = pack_f16(S[2 * kk][2] * s1, S[2 * kk][3] * s1);
                hi[2] = pack_f16(S[2 * kk + 1][0] * s0, S[2 * kk + 1][1] * s0);
                hi[3] = pack_f16(S[2 * kk + 1][2] * s1, S[2 * kk + 1][3] * s1);
            }
#pragma unroll
            for (int np = 0; np < 4; np++) {
                ldsm4(b, krow + RK_Q + np * 4096 + (((2 * kk + (m & 1)) ^ r) << 4));
                mma_f16(O[2 * np], hi, b[0], b[1]);
                mma_f16(O[2 * np + 1], hi, b[2], b[3]);
            }
        }
        // R = beta (v - e^G X), or v
#pragma unroll
        for (int n = 0; n < 8; n++) {
            float2 cx, cv;
            if (DELTA) {
                const float2 cg = *reinterpret_cast<const float2 *>(cf + CF_G * RK_C + 8 * n + 2 * t);
                const float2 cb = *reinterpret_cast<const float2 *>(cf + CF_B * RK_C + 8 * n + 2 * t);
                cx = make_float2(cg.x * cb.x, cg.y * cb.y);
                cv = *reinterpret_cast<const float2 *>(cf + CF_V * RK_C + 8 * n + 2 * t);
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t w = v[n >> 1][(n & 1) * 2 + k];
                const float v0 = __uint_as_float(w << 16), v1 = __uint_as_float(w & 0xffff0000u), is = k ? is1 : is0;
                X[n][2 * k] = DELTA ? fmaf(cx.x * is, X[n][2 * k], cv.x * v0) : v0;
                X[n][2 * k + 1] = DELTA ? fmaf(cx.y * is, X[n][2 * k + 1], cv.y * v1) : v1;
            }
        }
        const uint32_t trow = su + ((m >> 1) * 8 + r) * 128;   // T and P: rows 16 ip + .., chunks 2 jj + ..
        // U = T R by halves of 32 tokens: U_0 = T_0 R_0, R_1 -= A_10 U_0, U_1 = T_1 R_1.  Two f16 terms of both
        // factors, three products.  X[n] (n = 4 half ..) becomes u times k's scale.
        if (DELTA) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float (&R)[4][4] = *reinterpret_cast<float (*)[4][4]>(&X[4 * half]);
                float r0, r1, ir0, ir1;
                uint32_t hi[2][4], lo[2][4];
                auto split = [&]() {
                    row_scales(R, r0, r1, ir0, ir1);
#pragma unroll
                    for (int jj = 0; jj < 2; jj++) {
                        split_f16(R[2 * jj][0], R[2 * jj][1], r0, hi[jj][0], lo[jj][0]);
                        split_f16(R[2 * jj][2], R[2 * jj][3], r1, hi[jj][1], lo[jj][1]);
                        split_f16(R[2 * jj + 1][0], R[2 * jj + 1][1], r0, hi[jj][2], lo[jj][2]);
                        split_f16(R[2 * jj + 1][2], R[2 * jj + 1][3], r1, hi[jj][3], lo[jj][3]);
                    }
                };
                auto product = [&](float (&d)[2][4], int ip, int jj, int col) {   // tokens 16 ip .., columns 16 col ..
                    uint32_t bh[4], bl[4];
                    ldsm4(bh, trow + RK_TH + ip * 2048 + (((2 * col + (m & 1)) ^ r) << 4));
                    ldsm4(bl, trow + RK_TL + ip * 2048 + (((2 * col + (m & 1)) ^ r) << 4));
                    mma_f16(d[0], hi[jj], bh[0], bh[1]);
                    mma_f16(d[1], hi[jj], bh[2], bh[3]);
                    mma_f16(d[0], lo[jj], bh[0], bh[1]);
                    mma_f16(d[1], lo[jj], bh[2], bh[3]);
                    mma_f16(d[0], hi[jj], bl[0], bl[1]);
                    mma_f16(d[1], hi[jj], bl[2], bl[3]);
                };
                split();
                float d[2][2][4] = {};
                product(d[0], 2 * half, 0, 2 * half);
                product(d[1], 2 * half + 1, 0, 2 * half);
                product(d[1], 2 * half + 1, 1, 2 * half + 1);
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const float2 ct = *reinterpret_cast<const float2 *>(cf + CF_T * RK_C + 8 * (4 * half + n) + 2 * t);
                    const float2 ck = *reinterpret_cast<const float2 *>(cf + CF_K * RK_C + 8 * (4 * half + n) + 2 * t);
                    const float (&e)[4] = d[n >> 1][n & 1];
                    R[n][0] = e[0] * ir0 * ct.x * ck.x;
                    R[n][1] = e[1] * ir0 * ct.y * ck.y;
                    R[n][2] = e[2] * ir1 * ct.x * ck.x;
                    R[n][3] = e[3] * ir1 * ct.y * ck.y;
                }
                if (half == 0) {
                    split();
                    float f[2][2][4] = {};
#pragma unroll
                    for (int ip = 0; ip < 2; ip++)
#pragma unroll
                        for (int jj = 0; jj < 2; jj++) product(f[ip], 2 + ip, jj, jj);
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const float2 cb = *reinterpret_cast<const float2 *>(cf + CF_B * RK_C + 32 + 8 * n + 2 * t);
                        const float (&e)[4] = f[n >> 1][n & 1];
                        X[4 + n][0] = fmaf(cb.x * ir0, e[0], X[4 + n][0]);
                        X[4 + n][1] = fmaf(cb.y * ir0, e[1], X[4 + n][1]);
                        X[4 + n][2] = fmaf(cb.x * ir1, e[2], X[4 + n][2]);
                        X[4 + n][3] = fmaf(cb.y * ir1, e[3], X[4 + n][3]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const float2 ck = *reinterpret_cast<const float2 *>(cf + CF_K * RK_C + 8 * n + 2 * t);
                X[n][0] *= ck.x;
                X[n][1] *= ck.y;
                X[n][2] *= ck.x;
                X[n][3] *= ck.y;
            }
        }
        // O = scale (e^G O + P U), leading f16 terms
        {
            float u0, u1, iu0, iu1;
            row_scales(X, u0, u1, iu0, iu1);
            uint32_t ua[4][4];
#pragma unroll
            for (int jj = 0; jj < 4; jj++) {
                ua[jj][0] = pack_f16(X[2 * jj][0] * u0, X[2 * jj][1] * u0);
                ua[jj][1] = pack_f16(X[2 * jj][2] * u1, X[2 * jj][3] * u1);
                ua[jj][2] = pack_f16(X[2 * jj + 1][0] * u0, X[2 * jj + 1][1] * u0);
                ua[jj][3] = pack_f16(X[2 * jj + 1][2] * u1, X[2 * jj + 1][3] * u1);
            }
#pragma unroll
            for (int ip = 0; ip < 4; ip++) {
                float d[2][4] = {};
#pragma unroll
                for (int jj = 0; jj <= ip; jj++) {
                    uint32_t b[4];
                    ldsm4(b, trow + RK_P + ip * 2048 + (((2 * jj + (m & 1)) ^ r) << 4));
                    mma_f16(d[0], ua[jj], b[0], b[1]);
                    mma_f16(d[1], ua[jj], b[2], b[3]);
                }
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int n = 2 * ip + k;
                    const float2 cg = *reinterpret_cast<const float2 *>(cf + CF_G * RK_C + 8 * n + 2 * t);
                    const float2 q2 = *reinterpret_cast<const float2 *>(cf + CF_Q * RK_C + 8 * n + 2 * t);
                    const float2 q1 = make_float2(cg.x * q2.x, cg.y * q2.y);
                    const __nv_bfloat162 a = __floats2bfloat162_rn(fmaf(q1.x * is0, O[n][0], q2.x * iu0 * d[k][0]),
                                                                   fmaf(q1.y * is0, O[n][1], q2.y * iu0 * d[k][1]));
                    const __nv_bfloat162 b = __floats2bfloat162_rn(fmaf(q1.x * is1, O[n][2], q2.x * iu1 * d[k][2]),
                                                                   fmaf(q1.y * is1, O[n][3], q2.y * iu1 * d[k][3]));
                    o[2 * k] = *reinterpret_cast<const uint32_t *>(&a);
                    o[2 * k + 1] = *reinterpret_cast<const uint32_t *>(&b);
                }
                stsm4t(vrow + ip * 16 * (RK_ROWS * 2), o);   // over the warp's own columns of v
            }
        }
        __syncwarp();
        {
            __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + ((int64_t)t0 * p.n_head + h) * REC_HD + dv + (lane & 1) * 8;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int tok = 16 * i + (lane >> 1);
                const uint4 u = *reinterpret_cast<const uint4 *>(sg + RK_V + tok * (RK_ROWS * 2) + (((2 * wid + (lane & 1)) ^ (tok & 7)) << 4));
                if (t0 + tok < end) *reinterpret_cast<uint4 *>(out + (int64_t)tok * p.n_head * REC_HD) = u;
            }
        }
        // S = e^(G_C) S + (w U) K
        {
            float u0, u1, iu0, iu1;
            uint32_t hi[4][4], lo[4][4];
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const float2 cw = *reinterpret_cast<const float2 *>(cf + CF_W * RK_C + 8 * n + 2 * t);
                X[n][0] *= cw.x;
                X[n][1] *= cw.y;
                X[n][2] *= cw.x;
                X[n][3] *= cw.y;
            }
            row_scales(X, u0, u1, iu0, iu1);
#pragma unroll
            for (int jj = 0; jj < 4; jj++) {
                split_f16(X[2 * jj][0], X[2 * jj][1], u0, hi[jj][0], lo[jj][0]);
                split_f16(X[2 * jj][2], X[2 * jj][3], u1, hi[jj][1], lo[jj][1]);
                split_f16(X[2 * jj + 1][0], X[2 * jj + 1][1], u0, hi[jj][2], lo[jj][2]);
                split_f16(X[2 * jj + 1][2], X[2 * jj + 1][3], u1, hi[jj][3], lo[jj][3]);
            }
            const float eg = cf[CF_N * RK_C];
            const uint32_t ktrow = su + RK_K + ((m & 1) * 8 + r) * 256;
#pragma unroll
            for (int dg = 0; dg < 4; dg++) {
                float d[4][4] = {};
#pragma unroll
                for (int jj = 0; jj < 4; jj++) {
                    uint32_t b0[4], b1[4];
                    ldsm4t(b0, ktrow + jj * 4096 + (((4 * dg + (m >> 1)) ^ r) << 4));
                    ldsm4t(b1, ktrow + jj * 4096 + (((4 * dg + 2 + (m >> 1)) ^ r) << 4));
                    mma_f16(d[0], hi[jj], b0[0], b0[1]);
                    mma_f16(d[1], hi[jj], b0[2], b0[3]);
                    mma_f16(d[2], hi[jj], b1[0], b1[1]);
                    mma_f16(d[3], hi[jj], b1[2], b1[3]);
                    mma_f16(d[0], lo[jj], b0[0], b0[1]);
                    mma_f16(d[1], lo[jj], b0[2], b0[3]);
                    mma_f16(d[2], lo[jj], b1[0], b1[1]);
                    mma_f16(d[3], lo[jj], b1[2], b1[3]);
                }
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    S[4 * dg + n][0] = fmaf(eg, S[4 * dg + n][0], iu0 * d[n][0]);
                    S[4 * dg + n][1] = fmaf(eg, S[4 * dg + n][1], iu0 * d[n][1]);
                    S[4 * dg + n][2] = fmaf(eg, S[4 * dg + n][2], iu1 * d[n][2]);
                    S[4 * dg + n][3] = fmaf(eg, S[4 * dg + n][3], iu1 * d[n][3]);
                }
            }
        }
        if (c + RK_GROUPS < n_chunks) bar_arrive(BAR_EMPTY + st, RK_PAIR);
    }
    store_state();
}

template <bool DELTA>
__global__ void __launch_bounds__(RK_THREADS, 1) k_rec_chunk(const __grid_constant__ RecParams p) {
    extern __shared__ __align__(1024) uint8_t rk_sm[];
    const int seq = blockIdx.z, h = blockIdx.y, row0 = blockIdx.x * RK_ROWS;
    const int32_t beg = p.cu[seq], end = p.cu[seq + 1];
    if (beg < 0 || end > p.n_rows || beg > end) {
        if (threadIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
        return;
    }
    if (beg == end) return;
    if (threadIdx.x < RK_PROD) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(RK_PROD_REGS));
        rk_produce<DELTA>(p, rk_sm, h, row0, beg, end);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(RK_CHAIN_REGS));
        rk_chain<DELTA>(p, rk_sm, seq, h, row0, beg, end);
    }
}

cudaError_t launch_rec_chunk(const RecParams &p, cudaStream_t st) {
    auto *k = p.beta ? k_rec_chunk<true> : k_rec_chunk<false>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, RK_SMEM);
    if (e != cudaSuccess) return e;
    k<<<dim3(REC_HD / RK_ROWS, p.n_head, p.n_seq), RK_THREADS, RK_SMEM, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace qkv
