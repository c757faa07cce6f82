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
    int np, n1, t_lo, n_tiles;
    __device__ __forceinline__ int tile_of(int v) const { return v < n1 ? v : v - n1 + t_lo; }
};

// False: the tile has no rows. What is out of bounds is cut off, and reported when `report`.
__device__ __forceinline__ bool chunk_range(const ChunkAttnParams& p, int s, int tile, int group, int tile_rows, int key_tile,
                                            bool report, ChunkRange& c) {
    c.row0 = p.batch.row_start[s];
    c.n = p.batch.row_start[s + 1] - c.row0;
    c.total = p.batch.kv_len[s];   // positions count from the true length
    const int np = p.prefix ? p.prefix[s] : 0;
    if (report && (c.row0 < 0 || c.n < 0 || c.row0 > p.batch.n_rows - c.n || c.total < 0 || c.total > p.batch.max_kv ||
                   c.n > p.batch.max_chunk))
        atomicOr(p.err, PAGED_BAD_LENGTH);
    c.len = max(0, min(c.total, p.batch.max_kv));
    if (c.row0 < 0 || c.row0 > p.batch.n_rows) return false;
    c.n = min(c.n, p.batch.n_rows - c.row0);
    c.r0 = tile * tile_rows;
    c.rows = min(tile_rows, c.n * group - c.r0);
    if (c.rows <= 0) return false;
    c.p0 = c.total - c.n + c.r0 / group;
    c.p1 = c.total - c.n + (c.r0 + c.rows - 1) / group;
    c.np = max(0, min(np, c.len));
    int hi = max(0, min(c.len, c.p1 + 1)), lo = p.window ? max(0, c.p0 - p.window + 1) : 0;
    if (hi <= lo) lo = hi = 0;
    int t_hi;
    if (c.np >= lo) {
        c.t_lo = c.n1 = 0;
        t_hi = (max(c.np, hi) + key_tile - 1) / key_tile;
    } else {
        c.t_lo = lo / key_tile;
        t_hi = (hi + key_tile - 1) / key_tile;
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

// THREADS threads of the CTA (tid among them; barrier 1), after their split's results are in p.part ([split][ROWS][D] unnormalised outputs, then
// [split][ROWS] {maximum (log2 units), sum}): the CTA that arrives last joins the n_act splits in their order,
// so the result does not depend on the arrival order, and clears the counter.
template <typename T, int D, int ROWS, int THREADS>
__device__ __forceinline__ void join_splits(const ChunkAttnParams& p, const ChunkRange& c, int s, int tile, int h, int group,
                                            int tiles, int n_split, int n_act, bool vec, int tid, int* last) {
    const int64_t unit = ((int64_t)s * tiles + tile) * p.kv.n_head + h;
    const float* part_o = p.part + unit * n_split * (ROWS * (D + 2));
    const float* part_ml = part_o + (int64_t)n_split * ROWS * D;
    __threadfence();
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    if (tid == 0) *last = atomicAdd(p.arrived + unit, 1) == n_act - 1;
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    if (!*last) return;
    __threadfence();
    if (tid == 0) p.arrived[unit] = 0;
    for (int i = tid; i < c.rows * (D / 4); i += THREADS) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float top = NEG_INF;
        for (int w = 0; w < n_act; w++) top = fmaxf(top, __ldcg(part_ml + 2 * ((int64_t)w * ROWS + r)));
        const float ref = top == NEG_INF ? 0.0f : top;
        float sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int w = 0; w < n_act; w++) {
            const float2 e = __ldcg((const float2*)(part_ml + 2 * ((int64_t)w * ROWS + r)));
            const float f = ex2(e.x - ref);
            sum = fmaf(f, e.y, sum);
            const float4 v = __ldcg((const float4*)(part_o + ((int64_t)w * ROWS + r) * D + d));
            x[0] = fmaf(f, v.x, x[0]); x[1] = fmaf(f, v.y, x[1]);
            x[2] = fmaf(f, v.z, x[2]); x[3] = fmaf(f, v.w, x[3]);
        }
        const int tok = (c.r0 + r) / group, head = h * group + (c.r0 + r) % group;
        if (top != NEG_INF) {
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = x[k] / sum;
        }
        store_out<T, D>(p, vec, c.row0 + tok, head, d, x);
        if (p.lse && d == 0)
            p.lse[(int64_t)(c.row0 + tok) * p.n_q_head + head] = top == NEG_INF ? NEG_INF : (top + log2f(sum)) * LN2;
    }
}

}  // namespace
}  // namespace gsvcu
