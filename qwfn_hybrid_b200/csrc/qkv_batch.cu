// qkv_batch.cu -- ragged batches: the maps of a batch's rows (k_batch_map) and the q8_0 append of its
// K and V rows through the slot map (k_append_mapped).
#include "qkv_internal.h"

#include <algorithm>
#include <cuda_fp16.h>

namespace qkv {

// ---------------------------------------------------------------------------------------- maps
// Row r of a ragged batch belongs to the sequence i with cu[i] <= r < cu[i+1] (cu: exclusive sums
// of the new rows) and sits at position pos0[i] + r - cu[i]; its cell is page(position / 256) * 256 +
// position % 256 in the slot's block table.  The lengths travel as kernel parameters, so a call
// uploads nothing; 24 bytes a row at most are written, which bounds large batches, and small ones
// are one launch.  A thread takes rows a CTA's width apart, so every store instruction of a warp
// writes adjacent values whatever the outputs' alignment (a row of a two-row tensor may start at any
// 4-byte boundary); the sequence is found by bisection in shared memory.  Blocks behind the rows'
// blocks write the per-sequence block tables.
constexpr int BM_THREADS = 256, BM_PER = 4;   // items per CTA: BM_THREADS * BM_PER

__global__ void __launch_bounds__(BM_THREADS) k_batch_map(const __grid_constant__ BatchMapParams p) {
    __shared__ int32_t cu[BM_SEQ + 1], pos0[BM_SEQ], slot[BM_SEQ];
    const int tid = threadIdx.x;
    for (int i = tid; i <= p.n_seq; i += BM_THREADS) {
        cu[i] = p.cu[i];
        if (i < p.n_seq) {
            pos0[i] = p.pos0[i];
            slot[i] = p.slot[i];
        }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = tid; i <= p.n_seq; i += BM_THREADS) p.cu_out[p.seq0 + i] = cu[i];
    if ((int)blockIdx.x < p.row_blocks) {
#pragma unroll
        for (int k = 0; k < BM_PER; k++) {
            const int64_t r64 = (int64_t)p.row_lo + ((int64_t)blockIdx.x * BM_PER + k) * BM_THREADS + tid;
            if (r64 >= p.row_hi) return;
            const int32_t r = (int32_t)r64;
            int32_t seq = -1, pos = -1;
            int64_t cell = -1;
            if (r < cu[p.n_seq]) {
                int lo = 0, hi = p.n_seq - 1;   // the first i with cu[i + 1] > r
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (cu[mid + 1] > r) hi = mid;
                    else lo = mid + 1;
                }
                seq = p.seq0 + lo;
                pos = pos0[lo] + r - cu[lo];
                const int32_t page = p.bt[(int64_t)slot[lo] * p.max_pages + (pos >> 8)];
                if (page >= 0 && page < p.n_pages) cell = (int64_t)page * PAGE_TOK + (pos & (PAGE_TOK - 1));
                else atomicOr(p.status, ST_BAD_PAGE);
            }
            if (p.seq_out) p.seq_out[r] = seq;
            if (p.pos_out) p.pos_out[r] = pos;
            if (p.cell_out) p.cell_out[r] = cell;
        }
    } else {
#pragma unroll
        for (int k = 0; k < BM_PER; k++) {
            const int64_t e = ((int64_t)(blockIdx.x - p.row_blocks) * BM_PER + k) * BM_THREADS + tid;
            if (e >= (int64_t)p.n_seq * p.max_pages) return;
            const int i = (int)(e / p.max_pages), pg = (int)(e % p.max_pages);
            const int32_t need = (pos0[i] + cu[i + 1] - cu[i] + PAGE_TOK - 1) / PAGE_TOK;
            p.table_out[(int64_t)p.seq0 * p.max_pages + e] = pg < need ? p.bt[(int64_t)slot[i] * p.max_pages + pg] : -1;
        }
    }
}

cudaError_t launch_batch_map(BatchMapParams &p, cudaStream_t st) {
    const int64_t per = BM_THREADS * BM_PER;
    const bool rows = p.seq_out || p.pos_out || p.cell_out;
    p.row_blocks = rows ? (int32_t)((p.row_hi - p.row_lo + per - 1) / per) : 0;
    const int64_t tables = p.table_out ? ((int64_t)p.n_seq * p.max_pages + per - 1) / per : 0;
    const unsigned grid = (unsigned)std::max<int64_t>(1, p.row_blocks + tables);
    if (tables == 0 && p.row_blocks == 0) {   // cu alone
        p.row_blocks = 1;
        p.row_hi = p.row_lo;
    }
    k_batch_map<<<grid, BM_THREADS, 0, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

// ------------------------------------------------------------------------------- mapped append
// Kernel A for rows that lie anywhere in the pool.  CTA = (16 rows of the batch, KV head), 256
// threads, kernel A's rounding and shared-memory staging.  Rows of one sequence are neighbours in
// the batch and in the cache, but a sequence's first row may sit at any position of a 16-token
// group, so the 16 rows of a CTA are up to 16 runs of neighbouring cells.  K rows and scales are
// 16-byte stores per row anyway.  The transposed V (64 tokens of a dim are 64 adjacent bytes) is written
// per dim as runs allow: 4 bytes where four rows fill an aligned word, else bytes; the sectors that two
// CTAs share meet in L2.  Which stores a run takes depends on the cells alone, so all threads agree.
constexpr int AM_TOK = 16;

__global__ void __launch_bounds__(256) k_append_mapped(PoolRef pr, const int64_t *__restrict__ cell,
                                                       const float *__restrict__ K, const float *__restrict__ V,
                                                       int32_t n_rows) {
    __shared__ __align__(16) uint8_t ks[AM_TOK][HD];
    __shared__ __align__(16) uint8_t vs[AM_TOK][HD];
    __shared__ __align__(16) __half kd[AM_TOK][NBLK];
    __shared__ __align__(16) __half vd[AM_TOK][NBLK];
    __shared__ int64_t cs[AM_TOK];
    const int h = blockIdx.y, tid = threadIdx.x, sub = tid & 3;
    const int64_t r0 = (int64_t)blockIdx.x * AM_TOK;
    if (tid < AM_TOK) {
        int64_t c = r0 + tid < n_rows ? cell[r0 + tid] : -1;
        if (c < -1 || c >= (int64_t)pr.n_pages * PAGE_TOK) {
            atomicOr(pr.status, ST_BAD_INDEX);
            c = -1;
        }
        cs[tid] = c;
    }
    __syncthreads();
    float x[2][2][8];   // 2 teams x (K, V) x 8 elements: all loads issued before any use
#pragma unroll
    for (int it = 0; it < 2; it++) {
        const int p = (tid >> 2) + 64 * it, t = p >> 3, b = p & 7;
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            if (cs[t] >= 0) {
                const float4 *src = reinterpret_cast<const float4 *>((kv ? V : K) + (r0 + t) * pr.n_head_kv * HD + h * HD +
                                                                     b * QK + sub * 8);
                const float4 u0 = __ldcs(src), u1 = __ldcs(src + 1);
                x[it][kv][0] = u0.x; x[it][kv][1] = u0.y; x[it][kv][2] = u0.z; x[it][kv][3] = u0.w;
                x[it][kv][4] = u1.x; x[it][kv][5] = u1.y; x[it][kv][6] = u1.z; x[it][kv][7] = u1.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[it][kv][e] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int it = 0; it < 2; it++) {
        const int p = (tid >> 2) + 64 * it, t = p >> 3, b = p & 7;
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[it][kv][e]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const float d  = div127_rn(amax);
            const float id = d != 0.0f ? rcp_rn(d) : 0.0f;
            uint8_t q[8];
#pragma unroll
            for (int e = 0; e < 8; e++) q[e] = (uint8_t)(int8_t)round_half_away(__fmul_rn(x[it][kv][e], id));
            const int dim0 = b * QK + sub * 8;
            *reinterpret_cast<uint2 *>(kv ? &vs[t][dim0] : &ks[t][dim0]) =
                make_uint2(q[0] | q[1] << 8 | q[2] << 16 | (uint32_t)q[3] << 24,
                           q[4] | q[5] << 8 | q[6] << 16 | (uint32_t)q[7] << 24);
            if (sub == 0) (kv ? vd : kd)[t][b] = __float2half_rn(d);
        }
    }
    __syncthreads();
    auto tile_of = [&](int64_t c) {
        return pr.pool + (c >> 8) * pr.page_bytes + (int64_t)(h * TILES_PER_PAGE + ((c >> 6) & 3)) * TILE_BYTES;
    };
    {   // K: row tid >> 4, chunk tid & 15
        const int t = tid >> 4, c = tid & 15;
        if (cs[t] >= 0) {
            const int tt = (int)(cs[t] & 63);
            *reinterpret_cast<uint4 *>(tile_of(cs[t]) + TILE_KQ + tt * HD + ((c ^ kswz(tt)) << 4)) =
                *reinterpret_cast<const uint4 *>(&ks[t][c * 16]);
        }
    }
    for (int t = 0; t < AM_TOK;) {   // V: dim tid
        const int64_t c = cs[t];
        if (c < 0) {
            t++;
            continue;
        }
        uint8_t *dst = tile_of(c) + v_off(tid, (int)(c & 63));
        if ((c & 3) == 0 && t + 3 < AM_TOK && cs[t + 1] == c + 1 && cs[t + 2] == c + 2 && cs[t + 3] == c + 3) {
            *reinterpret_cast<uint32_t *>(dst) =
                vs[t][tid] | vs[t + 1][tid] << 8 | vs[t + 2][tid] << 16 | (uint32_t)vs[t + 3][tid] << 24;
            t += 4;
        } else {
            *dst = vs[t][tid];
            t++;
        }
    }
    if (tid < AM_TOK) {
        if (cs[tid] >= 0)
            *reinterpret_cast<uint4 *>(tile_of(cs[tid]) + kd_off((int)(cs[tid] & 63), 0)) =
                *reinterpret_cast<const uint4 *>(&kd[tid][0]);
    } else if (tid < AM_TOK + AM_TOK * NBLK) {
        const int e = tid - AM_TOK, b = e / AM_TOK, t = e % AM_TOK;
        if (cs[t] >= 0) *reinterpret_cast<__half *>(tile_of(cs[t]) + vd_off(b, (int)(cs[t] & 63))) = vd[t][b];
    }
}

cudaError_t launch_append_mapped(const PoolRef &pr, const int64_t *cell, const float *K, const float *V, int32_t n_rows,
                                 cudaStream_t st) {
    k_append_mapped<<<dim3((unsigned)((n_rows + AM_TOK - 1) / AM_TOK), (unsigned)pr.n_head_kv), 256, 0, st>>>(pr, cell, K, V,
                                                                                                             n_rows);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace qkv
