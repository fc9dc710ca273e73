// qkv_recurrent.cu -- the recurrent layers' kernels over the engine's state slabs: the short causal
// convolution (k_rec_conv) and linear attention with a decay per head, with or without the delta rule
// (k_rec_step for a few tokens, k_rec_serial for prompts).
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
// that meets a sequence's first row has read the history, so it also writes the new one (from the
// sequence's last three rows) and, for rollbacks, the ones after fewer rows: no second launch and no
// thread waits for another.
template <typename T> struct RecVec;
template <> struct RecVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const float *p, float (&v)[4]) {
        const float4 u = *reinterpret_cast<const float4 *>(p);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
    static __device__ __forceinline__ void store(float *p, const float (&v)[4]) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
template <> struct RecVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16 *p, float (&v)[8]) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
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
__device__ __forceinline__ void rec_conv_hist(const RecConvParams &p, const T *x, int c0, int32_t beg, int32_t end,
                                              const float (&old)[RC_HIST][VEC], float *out) {
    float v[RC_HIST][VEC];
#pragma unroll
    for (int j = 0; j < RC_HIST; j++) {
        const int32_t r = end - RC_HIST + j;
        if (r >= beg) {
            RecVec<T>::load(x + (int64_t)r * p.x_stride + c0, v[j]);
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

template <typename T>
__global__ void __launch_bounds__(RC_THREADS) k_rec_conv(const __grid_constant__ RecConvParams p) {
    constexpr int VEC = RecVec<T>::N, LANES = 128 / VEC;
    const int per_row = p.channels / VEC;   // a multiple of LANES
    const int64_t id = (int64_t)blockIdx.x * RC_THREADS + threadIdx.x;
    const int64_t blk = id / per_row;
    const int c0 = (int)(id % per_row) * VEC;
    const int32_t r_lo = (int32_t)min((int64_t)p.n_rows, blk * p.rows_per), r_hi = min(p.n_rows, r_lo + p.rows_per);
    const T *x = static_cast<const T *>(p.x);
    T *y = static_cast<T *>(p.y);
    float w[VEC][4];
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float4 u = __ldg(reinterpret_cast<const float4 *>(p.w) + c0 + e);
        w[e][0] = u.x; w[e][1] = u.y; w[e][2] = u.z; w[e][3] = u.w;
    }
    const bool norm = c0 < p.n_norm;
    const unsigned lanes = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    float h[RC_HIST][VEC];
    int32_t beg = 0, end = 0;   // rows of the current sequence
    for (int32_t r = r_lo; r < r_hi; r++) {
        if (r >= end || r == r_lo) {
            const int i = rec_find(p.cu, p.n_seq, p.n_rows, r, beg, end);
            if (i < 0) {          // a row of no sequence (of this launch)
                end = 0;
                continue;
            }
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
                    RecVec<T>::load(x + (int64_t)q * p.x_stride + c0, h[j]);
                } else {
                    const int32_t k = q - beg + RC_HIST;
#pragma unroll
                    for (int e = 0; e < VEC; e++) h[j][e] = k == 0 ? old[0][e] : k == 1 ? old[1][e] : old[2][e];
                }
            }
            if (r == beg) {
                for (int s = 1; s <= min(p.n_save, end - beg); s++)
                    rec_conv_hist<T, VEC>(p, x, c0, beg, end - s, old,
                                          reinterpret_cast<float *>(p.back + ((int64_t)p.slot[i] * p.n_rollback + s - 1) * p.slot_bytes) +
                                              (int64_t)c0 * RC_HIST);
                rec_conv_hist<T, VEC>(p, x, c0, beg, end, old, state);
            }
        }
        float v[VEC], o[VEC];
        RecVec<T>::load(x + (int64_t)r * p.x_stride + c0, v);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            float a = v[e] * w[e][3];
            a = fmaf(h[0][e], w[e][0], a);
            a = fmaf(h[1][e], w[e][1], a);
            a = fmaf(h[2][e], w[e][2], a);
            o[e] = a / (1.0f + expf(-a));
            ss = fmaf(o[e], o[e], ss);
            h[0][e] = h[1][e];
            h[1][e] = h[2][e];
            h[2][e] = v[e];
        }
        if (norm) {   // the lanes of a head walk the same rows: all of them are here
#pragma unroll
            for (int m = LANES / 2; m; m >>= 1) ss += __shfl_xor_sync(lanes, ss, m);
            const float inv = 1.0f / fmaxf(sqrtf(ss), p.eps);
#pragma unroll
            for (int e = 0; e < VEC; e++) o[e] *= inv;
        }
        RecVec<T>::store(y + (int64_t)r * p.channels + c0, o);
    }
}

cudaError_t launch_rec_conv(RecConvParams &p, bool bf16, int num_sms, cudaStream_t st) {
    const int per_row = p.channels / (bf16 ? 8 : 4);
    // rows per thread: as many as leave about 1024 threads per SM, at most 32 (three more rows are
    // read at the head of each walk)
    const int64_t want = (int64_t)num_sms * 1024;
    p.rows_per = (int32_t)std::min<int64_t>(32, std::max<int64_t>(1, (int64_t)p.n_rows * per_row / want));
    const int64_t threads = (int64_t)((p.n_rows + p.rows_per - 1) / p.rows_per) * per_row;
    const unsigned grid = (unsigned)((threads + RC_THREADS - 1) / RC_THREADS);
    if (bf16) k_rec_conv<__nv_bfloat16><<<grid, RC_THREADS, 0, st>>>(p);
    else k_rec_conv<float><<<grid, RC_THREADS, 0, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------- linear attention
// Per value head with state S [value][key] (key fastest), token by token:
//   S <- e^g S;  u = v, or with the delta rule u = beta (v - S k);  S <- S + u k^T;  o = scale S q.
// A value row of S needs no other row, so rows are split over CTAs, warps and lanes freely: 8 lanes
// per row, each 16 of its 128 keys as four float4 eight apart (a warp's load covers 4 rows in whole
// 128-byte lines), the row's two dot products by three shuffles.
constexpr int RT_THREADS = 128, RT_ROWS = 32, RT_TOK = 16;
constexpr int RT_PASS = RT_ROWS / 16;   // row quads per warp: 4 warps x 4 rows x RT_PASS

template <typename T>
__global__ void __launch_bounds__(RT_THREADS) k_rec_serial(const __grid_constant__ RecParams p) {
    __shared__ __align__(16) float ks[RT_TOK][REC_HD], qs[RT_TOK][REC_HD];
    __shared__ float vs[RT_TOK][RT_ROWS], os[RT_TOK][RT_ROWS], gs[RT_TOK], bs[RT_TOK];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, sub = lane & 7, rq = lane >> 3;
    const int seq = blockIdx.z, h = blockIdx.y, row0 = blockIdx.x * RT_ROWS;
    const int32_t beg = p.cu ? p.cu[seq] : seq * p.T, end = p.cu ? p.cu[seq + 1] : beg + p.T;
    if (beg < 0 || end > p.n_rows || beg > end) {
        if (tid == 0) atomicOr(p.status, ST_BAD_INDEX);
        return;
    }
    if (beg == end) return;
    const int hk = h / (p.n_head / p.n_head_k);
    const int64_t head_off = ((int64_t)h * REC_HD + row0) * REC_HD;
    float *S0 = reinterpret_cast<float *>(p.state + (int64_t)p.slot[seq] * p.slot_bytes) + head_off;
    float S[RT_PASS][16];
#pragma unroll
    for (int a = 0; a < RT_PASS; a++) {
        const int row = (a * 4 + wid) * 4 + rq;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 u = *reinterpret_cast<const float4 *>(S0 + row * REC_HD + (sub + 8 * j) * 4);
            S[a][4 * j] = u.x; S[a][4 * j + 1] = u.y; S[a][4 * j + 2] = u.z; S[a][4 * j + 3] = u.w;
        }
    }
    auto store_state = [&](float *dst) {
#pragma unroll
        for (int a = 0; a < RT_PASS; a++) {
            const int row = (a * 4 + wid) * 4 + rq;
#pragma unroll
            for (int j = 0; j < 4; j++)
                *reinterpret_cast<float4 *>(dst + row * REC_HD + (sub + 8 * j) * 4) =
                    make_float4(S[a][4 * j], S[a][4 * j + 1], S[a][4 * j + 2], S[a][4 * j + 3]);
        }
    };
    auto back_slab = [&](int s) {   // rollback snapshot s - 1: the state s tokens back
        return reinterpret_cast<float *>(p.back + ((int64_t)p.slot[seq] * p.n_rollback + s - 1) * p.slot_bytes) + head_off;
    };
    if (end - beg <= p.n_save) store_state(back_slab(end - beg));
    const T *q = static_cast<const T *>(p.q) + (int64_t)hk * REC_HD, *k = static_cast<const T *>(p.k) + (int64_t)hk * REC_HD;
    const T *v = static_cast<const T *>(p.v) + (int64_t)h * REC_HD + row0;
    constexpr int VEC = RecVec<T>::N;
    for (int32_t t0 = beg; t0 < end; t0 += RT_TOK) {
        const int nt = min(RT_TOK, end - t0);
        __syncthreads();
        for (int e = tid; e < nt * (REC_HD / VEC); e += RT_THREADS) {
            const int t = e / (REC_HD / VEC), c = e % (REC_HD / VEC) * VEC;
            float f[VEC];
            RecVec<T>::load(k + (int64_t)(t0 + t) * p.k_stride + c, f);
#pragma unroll
            for (int i = 0; i < VEC; i++) ks[t][c + i] = f[i];
            RecVec<T>::load(q + (int64_t)(t0 + t) * p.q_stride + c, f);
#pragma unroll
            for (int i = 0; i < VEC; i++) qs[t][c + i] = f[i];
        }
        for (int e = tid; e < nt * (RT_ROWS / VEC); e += RT_THREADS) {
            const int t = e / (RT_ROWS / VEC), c = e % (RT_ROWS / VEC) * VEC;
            float f[VEC];
            RecVec<T>::load(v + (int64_t)(t0 + t) * p.v_stride + c, f);
#pragma unroll
            for (int i = 0; i < VEC; i++) vs[t][c + i] = f[i];
        }
        if (tid < nt) {
            gs[tid] = expf(p.g[(int64_t)(t0 + tid) * p.n_head + h]);
            bs[tid] = p.beta ? p.beta[(int64_t)(t0 + tid) * p.n_head + h] : 0.0f;
        }
        __syncthreads();
        for (int t = 0; t < nt; t++) {
            float kf[16], qf[16];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 a = *reinterpret_cast<const float4 *>(&ks[t][(sub + 8 * j) * 4]);
                const float4 b = *reinterpret_cast<const float4 *>(&qs[t][(sub + 8 * j) * 4]);
                kf[4 * j] = a.x; kf[4 * j + 1] = a.y; kf[4 * j + 2] = a.z; kf[4 * j + 3] = a.w;
                qf[4 * j] = b.x; qf[4 * j + 1] = b.y; qf[4 * j + 2] = b.z; qf[4 * j + 3] = b.w;
            }
            const float eg = gs[t], be = bs[t];
#pragma unroll
            for (int a = 0; a < RT_PASS; a++) {
                const int row = (a * 4 + wid) * 4 + rq;
                float u = vs[t][row];
#pragma unroll
                for (int i = 0; i < 16; i++) S[a][i] *= eg;
                if (p.beta) {
                    float d = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; i++) d = fmaf(S[a][i], kf[i], d);
#pragma unroll
                    for (int m = 4; m; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
                    u = be * (u - d);
                }
                float o = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    S[a][i] = fmaf(u, kf[i], S[a][i]);
                    o = fmaf(S[a][i], qf[i], o);
                }
#pragma unroll
                for (int m = 4; m; m >>= 1) o += __shfl_xor_sync(0xffffffffu, o, m);
                if (sub == 0) os[t][row] = o * p.scale;
            }
            const int back = end - (t0 + t) - 1;   // tokens after this one
            if (back == 0) store_state(S0);
            else if (back <= p.n_save) store_state(back_slab(back));
        }
        __syncthreads();
        T *out = static_cast<T *>(p.out) + (int64_t)t0 * p.n_head * REC_HD + (int64_t)h * REC_HD + row0;
        for (int e = tid; e < nt * (RT_ROWS / VEC); e += RT_THREADS) {
            const int t = e / (RT_ROWS / VEC), c = e % (RT_ROWS / VEC) * VEC;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) f[i] = os[t][c + i];
            RecVec<T>::store(out + (int64_t)t * p.n_head * REC_HD + c, f);
        }
    }
}

cudaError_t launch_rec_step(const RecParams &p, cudaStream_t st) {
    k_rec_serial<float><<<dim3(REC_HD / RT_ROWS, p.n_head, p.n_seq), RT_THREADS, 0, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

cudaError_t launch_rec_chunk(const RecParams &p, cudaStream_t st) {
    k_rec_serial<__nv_bfloat16><<<dim3(REC_HD / RT_ROWS, p.n_head, p.n_seq), RT_THREADS, 0, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace qkv
