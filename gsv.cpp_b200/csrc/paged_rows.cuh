// paged_rows.cuh -- device code shared by the kernels that write rows into the paged cache and read them back: where a
// row is, and 8 elements at a time.
#pragma once
#include <cuda_bf16.h>

#include "kernels.h"
#include "paged.h"

namespace gsvcu {
namespace {

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// 8 elements by 16-byte accesses.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *(const float4*)p, b = *((const float4*)p + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        uint4 u = *(const uint4*)p;
        const T* t = (const T*)&u;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(t[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
        *((float4*)p + 1) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 u;
        T* t = (T*)&u;
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = from_f32<T>(x[i]);
        *(uint4*)p = u;
    }
}

// Where a row is in the cache: sequence found by the whole warp, page looked up.
struct Place {
    int64_t block;   // number of its (page, layer, K, head 0) block of 64 tokens within the pool, -1: none
    int token;       // its token in the block
    int64_t pos;     // cache position
};
template <typename P>   // KvAppendParams or KvReadParams
__device__ __forceinline__ Place place_of(const P& p, int row, int lane, bool report) {
    // sequences that end at or before the row: 32 blocks at a time, then the 32 of one block (1200 sequences: 2 loads)
    int s = 0, n = p.batch.n_seq;
    while (n > 32) {
        const int step = (n + 31) / 32, last = (lane + 1) * step - 1;
        const int m = __popc(__ballot_sync(0xffffffffu, last < n && p.batch.row_start[s + last + 1] <= row));
        s += m * step;
        n = min(step, n - m * step);
    }
    s += __popc(__ballot_sync(0xffffffffu, lane < n && p.batch.row_start[s + lane + 1] <= row));
    Place w{-1, 0, 0};
    if (s >= p.batch.n_seq) {   // rows beyond the last sequence
        if (report) atomicOr(p.err, PAGED_BAD_LENGTH);
        return w;
    }
    const int first = p.batch.row_start[s], end = p.batch.row_start[s + 1];
    const int len = p.batch.kv_len[s];
    const int64_t c = (int64_t)len - end + row;   // cache position (negative: before the cache's start)
    if (report && (len < 0 || len > p.batch.max_kv || (int64_t)end - first > p.batch.max_chunk))
        atomicOr(p.err, PAGED_BAD_LENGTH);
    if (row >= first && c >= 0 && c < p.batch.max_pages * PAGE) {
        const int page = p.batch.table[(int64_t)s * p.batch.max_pages + (int)c / PAGE];
        if (page >= 0 && page < p.kv.n_page)
            w.block = ((int64_t)page * p.kv.n_layer + p.kv.layer) * 2 * p.kv.n_head;
        else if (report)
            atomicOr(p.err, PAGED_BAD_PAGE);
    } else if (report && (row < first || c >= 0)) {
        atomicOr(p.err, PAGED_BAD_LENGTH);
    }
    w.token = (int)c & (PAGE - 1);
    w.pos = c;
    return w;
}

// Rotation position of a row at cache position c, clamped to the table.
__device__ __forceinline__ int rotation_position(const KvAppendParams& p, int row, int64_t c, bool report) {
    const int64_t pos = p.pos ? p.pos[row] : c;
    if (report && (pos < 0 || pos >= p.n_pos) && (p.pos || c >= 0)) atomicOr(p.err, PAGED_BAD_POSITION);
    return pos < 0 ? 0 : pos < p.n_pos ? (int)pos : p.n_pos - 1;
}

inline bool fits16(const void* p, int64_t stride, size_t size) {
    return !p || (((uintptr_t)p & 15) == 0 && (stride * (int64_t)size) % 16 == 0);
}
// Threads of a CTA of 256 per row: a warp when rows alone fill the GPU (31k rows of 48 heads x 128: 130 us, 170 with 256
// threads a row, whose angles then serve one head instead of twelve), up to 256 when there are few and latency counts.
inline int threads_per_row(int n_rows) {
    int per_row = 256;
    while (per_row > 32 && (int64_t)per_row * n_rows > 148 * 2048) per_row /= 2;
    return per_row;
}

}  // namespace
}  // namespace gsvcu
