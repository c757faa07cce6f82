// paged_join.cuh -- device code shared by the two chunk-attention kernels: which rows and keys a CTA has, and
// joining the results of its key splits.
#pragma once
#include <cuda_bf16.h>

#include "kernels.h"
#include "paged.h"

namespace gsvcu {
namespace {

constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A row tile of a sequence: its rows [r0, r0 + rows) among the chunk's packed rows, the keys that some of its
// rows see ([0, np) and [lo, hi), as key tiles: the first n1 tiles, then those from t_lo on).
struct ChunkRange {
    int row0, n, total, len;   // first packed row and rows of the chunk; kv_len as given, and cut to the table
    int r0, rows, p0, p1;      // the tile's packed rows, positions of the first and the last
    int np, lo, hi, n1, t_lo, n_tiles;
    __device__ __forceinline__ int tile_of(int v) const { return v < n1 ? v : v - n1 + t_lo; }
    // Whether some row of the tile sees a key of the page that starts at `key` (others are not looked up: with a window
    // their place in the table may be stale).
    __device__ __forceinline__ bool sees(int key) const { return key < np || (key < hi && key + PAGE > lo); }
};

// False: the tile has no rows. What is out of bounds is cut off, and reported when `report`.
__device__ __forceinline__ bool chunk_range(const ChunkAttnParams& p, int s, int tile, int group, int tile_rows, int key_tile,
                                            bool report, ChunkRange& c) {
    c.row0 = p.batch.row_start[s];
    const int64_t n = (int64_t)p.batch.row_start[s + 1] - c.row0;
    c.total = p.batch.kv_len[s];   // positions count from the true length
    const int np = p.prefix ? p.prefix[s] : 0;
    if (report && (c.row0 < 0 || n < 0 || c.row0 + n > p.batch.n_rows || c.total < 0 || c.total > p.batch.max_kv ||
                   n > p.batch.max_chunk || (s == 0 && c.row0 != 0) ||
                   (s == p.batch.n_seq - 1 && c.row0 + n != p.batch.n_rows)))   // (rows that no sequence owns)
        atomicOr(p.err, PAGED_BAD_LENGTH);
    c.total = max(c.total, 0);
    c.len = min(c.total, p.batch.max_kv);
    if (c.row0 < 0 || c.row0 >= p.batch.n_rows || n <= 0) return false;
    c.n = (int)min(n, (int64_t)(p.batch.n_rows - c.row0));   // (the sizes are at most 2^30 rows times query heads)
    c.r0 = tile * tile_rows;
    c.rows = min(tile_rows, c.n * group - c.r0);
    if (c.rows <= 0) return false;
    c.p0 = c.total - c.n + c.r0 / group;
    c.p1 = c.total - c.n + (c.r0 + c.rows - 1) / group;
    c.np = max(0, min(np, c.len));
    c.hi = max(0, min(c.len, c.p1 + 1));
    c.lo = p.window ? max(0, c.p0 - p.window + 1) : 0;
    if (c.hi <= c.lo) c.lo = c.hi = 0;
    int t_hi;
    if (c.np >= c.lo) {
        c.t_lo = c.n1 = 0;
        t_hi = (max(c.np, c.hi) + key_tile - 1) / key_tile;
    } else {
        c.t_lo = c.lo / key_tile;
        t_hi = (c.hi + key_tile - 1) / key_tile;
        c.n1 = min((c.np + key_tile - 1) / key_tile, c.t_lo);
    }
    c.n_tiles = c.n1 + t_hi - c.t_lo;
    return true;
}

// Four consecutive outputs of one row and head.
template <typename T, int D>
__device__ __forceinline__ void store_out(const ChunkAttnParams& p, bool vec, int64_t row, int head, int d, const float (&o)[4]) {
    T* dst = (T*)p.out + row * p.out_stride + (int64_t)head * D + d;
    if (vec) {
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = narrow<T>(o[i]);
        if constexpr (sizeof(T) == 4) *(float4*)dst = make_float4(v[0], v[1], v[2], v[3]);
        else *(uint2*)dst = *(const uint2*)v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) dst[i] = narrow<T>(o[i]);
    }
}

// Four outputs (and the log-sum-exp) of row r of the tile from their unnormalised sums.
template <typename T, int D>
__device__ __forceinline__ void finish(const ChunkAttnParams& p, const ChunkRange& c, bool vec, int group, int h, int r, int d,
                                       float top, float sum, float (&x)[4]) {
    const int tok = (c.r0 + r) / group, head = h * group + (c.r0 + r) % group;
    if (sum != 0.0f) {   // (a row that sees nothing stays 0; one whose scores are all NaN has no maximum either, but a NaN sum)
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = x[k] / sum;
    }
    store_out<T, D>(p, vec, c.row0 + tok, head, d, x);
    if (p.lse && d == 0)
        p.lse[(int64_t)(c.row0 + tok) * p.n_q_head + head] = (top + log2f(sum)) * LN2;   // (nothing seen: both -infinity)
}

// Splits g, g + per, ... of n_act added up for four outputs of row r; 8 loads in flight whatever the count.
template <int D, int ROWS>
__device__ __forceinline__ void sum_splits(const float* part_o, const float* part_ml, int n_act, int g, int per, int r, int d,
                                           float& top, float& sum, float (&x)[4]) {
    const int mine = (n_act - g + per - 1) / per;
    const int64_t step_ml = 2 * (int64_t)per * ROWS, step_o = (int64_t)per * ROWS * D;
    const float* ml = part_ml + 2 * (g * ROWS + r);
    const float* po = part_o + ((int64_t)g * ROWS + r) * D + d;
    top = NEG_INF;
    sum = x[0] = x[1] = x[2] = x[3] = 0.0f;
    for (int w0 = 0; w0 < mine; w0 += 8) {
        float m[8];
#pragma unroll
        for (int k = 0; k < 8; k++) m[k] = w0 + k < mine ? __ldcg(ml + (w0 + k) * step_ml) : NEG_INF;
#pragma unroll
        for (int k = 0; k < 8; k++) top = fmaxf(top, m[k]);
    }
    const float ref = top == NEG_INF ? 0.0f : top;
    for (int w0 = 0; w0 < mine; w0 += 8) {
        float2 e[8];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const bool in = w0 + k < mine;
            e[k] = in ? __ldcg((const float2*)(ml + (w0 + k) * step_ml)) : make_float2(NEG_INF, 0.0f);
            v[k] = in ? __ldcg((const float4*)(po + (w0 + k) * step_o)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float f = ex2(e[k].x - ref);
            sum = fmaf(f, e[k].y, sum);
            x[0] = fmaf(f, v[k].x, x[0]); x[1] = fmaf(f, v[k].y, x[1]);
            x[2] = fmaf(f, v[k].z, x[2]); x[3] = fmaf(f, v[k].w, x[3]);
        }
    }
}

// Joining as a kernel of its own: a CTA per (unit, 1024 outputs).
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) k_chunk_join(ChunkAttnParams p, int group, int tiles, int n_split, int split_tiles,
                                                    int key_tile, bool vec) {
    constexpr int R = 1024 / D;   // rows of a CTA
    griddep_wait();
    griddep_launch();
    const int64_t unit = blockIdx.x / ((ROWS + R - 1) / R);
    const int r = blockIdx.x % ((ROWS + R - 1) / R) * R + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const int h = (int)(unit % p.kv.n_head), tile = (int)(unit / p.kv.n_head % tiles), s = (int)(unit / p.kv.n_head / tiles);
    ChunkRange c;
    if (!chunk_range(p, s, tile, group, ROWS, key_tile, false, c) || r >= c.rows) return;
    const int n_act = (c.n_tiles + split_tiles - 1) / split_tiles;
    if (n_act <= 1) return;   // (written by the only split)
    const float* part_o = p.part + unit * n_split * (ROWS * (D + 2));
    float top, sum, x[4];
    sum_splits<D, ROWS>(part_o, part_o + (int64_t)n_split * ROWS * D, n_act, 0, 1, r, d, top, sum, x);
    finish<T, D>(p, c, vec, group, h, r, d, top, sum, x);
}

// THREADS threads of the CTA (tid among them; barrier 1), after their split's results are in p.part ([split][ROWS][D]
// unnormalised outputs, then [split][ROWS] {maximum (log2 units), sum}): the CTA that arrives last joins the
// n_act splits and clears the counter. Every sum runs in an order that the sizes alone decide, so the result does
// not depend on the arrival order. buf: shared memory, 8 * THREADS floats.
template <typename T, int D, int ROWS, int THREADS>
__device__ __forceinline__ void join_splits(const ChunkAttnParams& p, const ChunkRange& c, int s, int tile, int h, int group,
                                            int tiles, int n_split, int n_act, bool vec, int tid, int* last, float* buf) {
    auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); };
    const int64_t unit = ((int64_t)s * tiles + tile) * p.kv.n_head + h;
    const float* part_o = p.part + unit * n_split * (ROWS * (D + 2));
    const float* part_ml = part_o + (int64_t)n_split * ROWS * D;
    __threadfence();
    sync();
    if (tid == 0) *last = atomicAdd(p.arrived + unit, 1) == n_act - 1;
    sync();
    if (!*last) return;
    __threadfence();
    if (tid == 0) p.arrived[unit] = 0;
    // thread = four outputs of a row over every per-th split; where rows and outputs are fewer than the threads,
    // per of them share a row's splits
    const int items = c.rows * (D / 4);
    int per = 1;
    while (per * 2 * items <= THREADS && per * 2 <= n_act) per *= 2;
    for (int i = tid; i < items * per; i += THREADS) {
        const int item = per > 1 ? i % items : i, g = per > 1 ? i / items : 0, r = item / (D / 4), d = item % (D / 4) * 4;
        float top, sum, x[4];
        sum_splits<D, ROWS>(part_o, part_ml, n_act, g, per, r, d, top, sum, x);
        if (per > 1) {
            *(float4*)(buf + 8 * i) = make_float4(x[0], x[1], x[2], x[3]);
            *(float2*)(buf + 8 * i + 4) = make_float2(top, sum);
        } else {
            finish<T, D>(p, c, vec, group, h, r, d, top, sum, x);
        }
    }
    if (per > 1) {   // (items * per <= THREADS)
        sync();
        if (tid < items) {
            float top = NEG_INF, sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int g = 0; g < per; g++) top = fmaxf(top, buf[8 * (g * items + tid) + 4]);
            const float ref = top == NEG_INF ? 0.0f : top;
            for (int g = 0; g < per; g++) {
                const float* y = buf + 8 * (g * items + tid);
                const float f = ex2(y[4] - ref);
                sum = fmaf(f, y[5], sum);
#pragma unroll
                for (int k = 0; k < 4; k++) x[k] = fmaf(f, y[k], x[k]);
            }
            finish<T, D>(p, c, vec, group, h, tid / (D / 4), tid % (D / 4) * 4, top, sum, x);
        }
    }
}

}  // namespace
}  // namespace gsvcu
