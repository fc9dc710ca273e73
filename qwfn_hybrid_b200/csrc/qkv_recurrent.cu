// qkv_recurrent.cu -- the recurrent layers' kernels over the engine's state slabs: the short causal
// convolution (k_rec_conv) and linear attention with a decay per head, with or without the delta rule, for a
// few tokens (k_rec_step; prompts: qkv_rec_chunk.cu).
#include "qkv_internal.h"

#include <algorithm>
#include <cuda_bf16.h>

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
// that meets a sequence's first row computes its first three rows, however many of them its walk
// holds, and a walk that starts in the second or third leaves those out: so one thread alone reads a
// channel's history, and it also writes the new one (from the sequence's last three rows) and, for
// rollbacks, the ones after fewer rows.  No second launch, and no thread waits for another.
// Rows go through a ring of asynchronous copies, eight ahead of the one computed, and are normalised two at a time (a
// head's sum is four or five shuffles after one another).  16001 rows of 10240 bf16 channels, 4096 of them normalised: 144 us,
// 4.6 TB/s, 70% of the copy rate (row by row 147; that without the exponential and the reciprocal 130, without the norm as
// well 114).
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

// The lanes of a warp that hold the thread's head of 128 channels.
template <typename T>
__device__ __forceinline__ unsigned rec_head_lanes() { return RecVec<T>::N == 4 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16); }
// One row of a thread's channels (the three rows before it, the row itself, the taps); returns its sum of squares.
template <int VEC>
__device__ __forceinline__ float rec_conv_row(const float (&h0)[VEC], const float (&h1)[VEC], const float (&h2)[VEC], const float (&v)[VEC],
                                              const float (&w)[VEC][4], float (&o)[VEC]) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        float a = v[e] * w[e][3];
        a = fmaf(h0[e], w[e][0], a);
        a = fmaf(h1[e], w[e][1], a);
        a = fmaf(h2[e], w[e][2], a);
        o[e] = a * rcp(1.0f + ex2(a * -1.4426950408889634f));
        ss = fmaf(o[e], o[e], ss);
    }
    return ss;
}
// N rows divided by the norms of the thread's head (the lanes of a head walk the same rows: all of them are here), N shuffles
// on their way at a time.
template <int N, int VEC>
__device__ __forceinline__ void rec_conv_norm(float (&o)[N][VEC], float (&ss)[N], unsigned lanes, float max_inv) {
#pragma unroll
    for (int m = 64 / VEC; m; m >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) ss[i] += __shfl_xor_sync(lanes, ss[i], m);
#pragma unroll
    for (int i = 0; i < N; i++) {
        float inv = rsqrtf(ss[i]);
        if (inv > max_inv) inv = max_inv;   // (a NaN stays)
#pragma unroll
        for (int e = 0; e < VEC; e++) o[i][e] *= inv;
    }
}
// The rows before row r of the sequence [beg, end) into h: of the sequence itself, or at r = beg the history; then
// also the history (and, for rollbacks, the ones some rows back) as it will be after the sequence's rows.
template <typename T>
__device__ __forceinline__ void rec_conv_enter(const RecConvParams &p, const T *x, int c0, int slot, int32_t r, int32_t beg, int32_t end,
                                               float (&h)[RC_HIST + 1][RecVec<T>::N]) {
    constexpr int VEC = RecVec<T>::N;
    if (r != beg) {
#pragma unroll
        for (int j = 0; j < RC_HIST; j++) RecVec<T>::load(x + (int64_t)(r - RC_HIST + j) * p.x_stride, h[j]);
        return;
    }
    float *state = reinterpret_cast<float *>(p.state + (int64_t)slot * p.slot_bytes) + (int64_t)c0 * RC_HIST;
    float flat[RC_HIST * VEC], old[RC_HIST][VEC];
#pragma unroll
    for (int k = 0; k < RC_HIST * VEC / 4; k++) {
        const float4 u = reinterpret_cast<const float4 *>(state)[k];
        flat[4 * k] = u.x; flat[4 * k + 1] = u.y; flat[4 * k + 2] = u.z; flat[4 * k + 3] = u.w;
    }
#pragma unroll
    for (int e = 0; e < VEC; e++)
#pragma unroll
        for (int j = 0; j < RC_HIST; j++) h[j][e] = old[j][e] = flat[e * RC_HIST + j];
    for (int s = 1; s <= min(p.n_save, end - beg); s++)
        rec_conv_hist<T, VEC>(p, x, beg, end - s, old,
                              reinterpret_cast<float *>(p.back + ((int64_t)slot * p.n_rollback + s - 1) * p.slot_bytes) + (int64_t)c0 * RC_HIST);
    rec_conv_hist<T, VEC>(p, x, beg, end, old, state);
}

// The few rows of decode steps: a thread per 16 bytes of a row.
template <typename T>
constexpr int RC_STEP_CTAS = sizeof(T) == 4 ? 4 : 2;   // resident per SM
template <typename T>
__global__ void __launch_bounds__(RC_THREADS, RC_STEP_CTAS<T>) k_rec_conv_rows(const __grid_constant__ RecConvParams p) {
    __shared__ int32_t cu[MAX_SEQ + 1];
    constexpr int VEC = RecVec<T>::N;
    const int per_row = p.channels / VEC;
    const int64_t id = (int64_t)blockIdx.x * RC_THREADS + threadIdx.x;
    const int32_t r = (int32_t)min((int64_t)p.n_rows, id / per_row);
    const int c0 = (int)(id % per_row) * VEC;
    const T *x = static_cast<const T *>(p.x) + c0;
    const bool in = r < p.n_rows;
    float w[VEC][4], h[RC_HIST + 1][VEC];   // rows r - 3 .. r
    if (in) RecVec<T>::load(x + (int64_t)r * p.x_stride, h[3]);
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float4 u = __ldg(reinterpret_cast<const float4 *>(p.w) + c0 + e);
        w[e][0] = u.x; w[e][1] = u.y; w[e][2] = u.z; w[e][3] = u.w;
    }
    for (int i = threadIdx.x; i <= p.n_seq; i += RC_THREADS) cu[i] = p.cu[i];
    __syncthreads();
    if (!in) return;
    int32_t beg, end;
    const int i = rec_find(cu, p.n_seq, p.n_rows, r, beg, end);
    // A row of no sequence (of this launch), or the second or third of one: all lanes of the head leave.
    if (i < 0 || (r > beg && r < beg + RC_HIST)) return;
    rec_conv_enter<T>(p, x, c0, p.slot[i], r, beg, end, h);
    T *y = static_cast<T *>(p.y) + (int64_t)r * p.channels + c0;
    const int n = r == beg ? min(RC_HIST, end - beg) : 1;
#pragma unroll
    for (int k = 0; k < RC_HIST; k++) {
        if (k >= n) break;
        if (k) RecVec<T>::load(x + (int64_t)(r + k) * p.x_stride, h[(k + 3) & 3]);
        float o[1][VEC], ss[1] = {rec_conv_row(h[k & 3], h[(k + 1) & 3], h[(k + 2) & 3], h[(k + 3) & 3], w, o[0])};
        if (c0 < p.n_norm) rec_conv_norm(o, ss, rec_head_lanes<T>(), 1.0f / p.eps);
        RecVec<T>::store(y + (int64_t)k * p.channels, o[0]);
    }
}

constexpr int RC_AHEAD = 8;   // rows in flight ahead of the one computed, in shared memory: they cost no registers

template <typename T>
__global__ void __launch_bounds__(RC_THREADS, 2) k_rec_conv(const __grid_constant__ RecConvParams p) {
    __shared__ uint4 ring[RC_AHEAD][RC_THREADS];   // a thread reads what it copied: no barrier
    __shared__ int32_t cu[MAX_SEQ + 1];
    constexpr int VEC = RecVec<T>::N;
    const int per_row = p.channels / VEC;   // a multiple of the 128 / VEC lanes of a head
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
    if (r_hi <= cu[0] || r_lo >= cu[p.n_seq]) {   // rows of other launches' sequences alone
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }
    const bool norm = c0 < p.n_norm;
    const float max_inv = 1.0f / p.eps;
    const unsigned lanes = rec_head_lanes<T>();
    for (int32_t r = r_lo; r < r_hi;) {
        int32_t beg, end;   // rows of the sequence
        const int i = rec_find(cu, p.n_seq, p.n_rows, r, beg, end);
        if (i < 0 || (r > beg && r < beg + RC_HIST)) {   // of no sequence (of this launch), or of the walk that holds its first row
            // Row r's copy must have arrived: the next one goes to the same slot, and of two on their way either may be last.
            asm volatile("cp.async.wait_group %0;" ::"n"(RC_AHEAD - 1) : "memory");
            fetch(r + RC_AHEAD);
            r++;
            continue;
        }
        float h[RC_HIST + 1][VEC];   // rows r - 3 .. r
        rec_conv_enter<T>(p, x, c0, p.slot[i], r, beg, end, h);
        const int32_t lim = min(end, r == beg ? max(r_hi, beg + RC_HIST) : r_hi);
        T *yr = y + (int64_t)r * p.channels;
        auto row = [&](int k, float (&o)[VEC]) {   // row r + k of the four whose window starts at h[k]
            float (&v)[VEC] = h[(k + 3) & 3];
            asm volatile("cp.async.wait_group %0;" ::"n"(RC_AHEAD - 1) : "memory");
            if (r + k < r_hi) RecVec<T>::unpack(ring[(r + k - r_lo) & (RC_AHEAD - 1)][threadIdx.x], v);
            else RecVec<T>::load(x + (int64_t)(r + k) * p.x_stride, v);   // past the walk: a sequence's second or third row
            fetch(r + k + RC_AHEAD);
            return rec_conv_row(h[k & 3], h[(k + 1) & 3], h[(k + 2) & 3], v, w, o);
        };
        for (; r < lim; r += 4) {
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                if (r + k >= lim) break;
                const bool two = r + k + 1 < lim;
                float o[2][VEC], ss[2];
                ss[0] = row(k, o[0]);
                if (two) {
                    ss[1] = row(k + 1, o[1]);
                } else {
                    ss[1] = 0.0f;
#pragma unroll
                    for (int e = 0; e < VEC; e++) o[1][e] = 0.0f;
                }
                if (norm) rec_conv_norm(o, ss, lanes, max_inv);
                RecVec<T>::store(yr, o[0]);
                if (two) RecVec<T>::store(yr + p.channels, o[1]);
                yr += 2 * p.channels;
            }
        }
        r = lim;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

cudaError_t launch_rec_conv(RecConvParams &p, bool bf16, int num_sms, cudaStream_t st) {
    const int64_t per_row = p.channels / (bf16 ? 8 : 4);
    auto grid_of = [&](int64_t r) { return ((p.n_rows + r - 1) / r * per_row + RC_THREADS - 1) / RC_THREADS; };
    if (grid_of(1) <= (int64_t)num_sms * (bf16 ? RC_STEP_CTAS<__nv_bfloat16> : RC_STEP_CTAS<float>)) {
        // One wave of CTAs holds a thread per 16 bytes: the kernel without the ring of copies, which needs fewer
        // registers and no start of a walk (64 rows of 8192 F32 channels: 6.1 us against 9.9 for walks of four).
        p.rows_per = 1;
        if (bf16) k_rec_conv_rows<__nv_bfloat16><<<(unsigned)grid_of(1), RC_THREADS, 0, st>>>(p);
        else k_rec_conv_rows<float><<<(unsigned)grid_of(1), RC_THREADS, 0, st>>>(p);
    } else {
        // Rows per thread: what makes waves times rows least, with the start of a walk (its sequence, the three
        // rows before it) counted as eight rows.
        int64_t best = 4;
        const int64_t slots = 2 * num_sms;   // CTAs resident at once
        for (int64_t r = 4, least = INT64_MAX; r <= 64; r += 4) {
            const int64_t cost = (grid_of(r) + slots - 1) / slots * (r + 8);
            if (cost < least) {
                least = cost;
                best = r;
            }
        }
        p.rows_per = (int32_t)best;
        if (bf16) k_rec_conv<__nv_bfloat16><<<(unsigned)grid_of(best), RC_THREADS, 0, st>>>(p);
        else k_rec_conv<float><<<(unsigned)grid_of(best), RC_THREADS, 0, st>>>(p);
    }
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

}  // namespace qkv
