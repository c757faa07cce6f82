// paged_append.cu -- new rows into the paged KV cache, the position rotation applied on the way.
//
// Row i of a sequence's chunk of n rows goes to cache position c = kv_len - n + i: page table[c / 64],
// token slot c % 64. Keys and queries are rotated first: with a = x[i], b = x[i + rot / 2] (or the adjacent
// pair x[2 i], x[2 i + 1]) and the table's cos, sin at the row's position,
//   a' = a cos - b sin,  b' = a sin + b cos,
// in f32, rounded once to the cache's type; elements from rot on and values are only converted. The kernel
// reads every q / k / v element once and writes it once, so HBM bounds it on prompts (31k rows of 48 heads x 128 in
// BF16: 131 us, 6.0 TB/s) and the chain row_start -> kv_len -> table -> store bounds it on single tokens (64 rows of
// 48 heads x 32: 2.7 us).
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

// Where a row goes: sequence found by the whole warp, page looked up.
struct Place {
    int64_t slot;   // element offset of the row's (layer, K, head 0) within the pool, -1: not stored
    int pos;        // rotation position, clamped to the table
};
template <int D>
__device__ __forceinline__ Place place_of(const KvAppendParams& p, int row, int lane, bool report) {
    // sequences that end at or before the row: 32 blocks at a time, then the 32 of one block (1200 sequences: 2 loads)
    int s = 0, n = p.batch.n_seq;
    while (n > 32) {
        const int step = (n + 31) / 32, last = (lane + 1) * step - 1;
        const int m = __popc(__ballot_sync(0xffffffffu, last < n && p.batch.row_start[s + last + 1] <= row));
        s += m * step;
        n = min(step, n - m * step);
    }
    s += __popc(__ballot_sync(0xffffffffu, lane < n && p.batch.row_start[s + lane + 1] <= row));
    Place w{-1, 0};
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
            w.slot = (((int64_t)page * p.kv.n_layer + p.kv.layer) * 2 * p.kv.n_head * PAGE + (int)c % PAGE) * D;
        else if (report)
            atomicOr(p.err, PAGED_BAD_PAGE);
    } else if (report && (row < first || c >= 0)) {
        atomicOr(p.err, PAGED_BAD_LENGTH);
    }
    if (p.rot) {
        const int64_t pos = p.pos ? p.pos[row] : c;
        if (report && (pos < 0 || pos >= p.n_pos) && (p.pos || c >= 0)) atomicOr(p.err, PAGED_BAD_POSITION);
        w.pos = pos < 0 ? 0 : pos < p.n_pos ? (int)pos : p.n_pos - 1;
    }
    return w;
}

// Vector form: thread = (row, unit u of D / 16, head lane). A unit is two runs of 8 elements that rotate with
// the same 8 angles (i and i + rot / 2, or 16 adjacent elements), so its angles stay in registers over the
// heads. A warp works on one row.
template <typename TI, typename T, int D>
__global__ void __launch_bounds__(256) k_kv_append(KvAppendParams p, int head_lanes) {
    constexpr int U = D / 16;
    griddep_wait();
    griddep_launch();
    const int per_row = U * head_lanes, rows_per_cta = 256 / per_row;
    const int row = blockIdx.x * rows_per_cta + threadIdx.x / per_row;
    if (row >= p.batch.n_rows) return;   // (warp-uniform: per_row is a multiple of 32)
    const int t = threadIdx.x % per_row, u = t % U, hl = t / U, lane = threadIdx.x & 31;
    const Place w = place_of<D>(p, row, lane, t == 0);
    const int n_rot = p.rot / 16;
    const bool turn = u < n_rot;
    const int ea = !turn ? u * 16 : p.pairs ? u * 16 : u * 8;
    const int eb = !turn ? ea + 8 : p.pairs ? ea + 8 : p.rot / 2 + u * 8;
    float cs[8], sn[8];
    if (turn) {
        load8(p.cos + (int64_t)w.pos * (p.rot / 2) + u * 8, cs);
        load8(p.sin + (int64_t)w.pos * (p.rot / 2) + u * 8, sn);
    }
    const int nk = p.kv.n_head, heads = p.n_q_head + 2 * nk;
    for (int h = hl; h < heads; h += head_lanes) {
        const bool is_q = h < p.n_q_head, is_v = h >= p.n_q_head + nk;
        const int hh = is_q ? h : is_v ? h - p.n_q_head - nk : h - p.n_q_head;
        const TI* src = is_q ? (const TI*)p.q + row * p.q_stride
                             : is_v ? (const TI*)p.v + row * p.v_stride : (const TI*)p.k + row * p.k_stride;
        src += hh * D;
        float a[8], b[8];
        load8(src + ea, a);
        load8(src + eb, b);
        if (turn && !is_v) {
            if (p.pairs) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float* x = i < 4 ? a + 2 * i : b + 2 * (i - 4);
                    const float x0 = x[0], x1 = x[1];
                    x[0] = x0 * cs[i] - x1 * sn[i];
                    x[1] = x0 * sn[i] + x1 * cs[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x0 = a[i], x1 = b[i];
                    a[i] = x0 * cs[i] - x1 * sn[i];
                    b[i] = x0 * sn[i] + x1 * cs[i];
                }
            }
        }
        T* dst;
        if (is_q)
            dst = (T*)p.q_out + row * p.q_out_stride + hh * D;
        else if (w.slot >= 0)
            dst = (T*)p.kv.pool + w.slot + (int64_t)((is_v ? nk : 0) + hh) * (PAGE * D);
        else
            continue;
        store8(dst + ea, a);
        store8(dst + eb, b);
    }
}

// Element form for rows, tables or rotation widths that 16-byte accesses do not fit: thread = one pair of
// elements, a warp on one row. Any alignment and width in one simple loop for what is rare: bound by its 2-byte accesses
// (31k rows of 48 heads x 128, 120 rotated: 292 us, 131 in the vector form).
template <typename TI, typename T, int D>
__global__ void __launch_bounds__(128) k_kv_append_any(KvAppendParams p) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, row = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= p.batch.n_rows) return;
    const Place w = place_of<D>(p, row, lane, lane == 0);
    const int nk = p.kv.n_head, heads = p.n_q_head + 2 * nk, half = p.rot / 2;
    for (int i = lane; i < heads * (D / 2); i += 32) {
        const int h = i / (D / 2), e = i % (D / 2);
        const bool is_q = h < p.n_q_head, is_v = h >= p.n_q_head + nk;
        const int hh = is_q ? h : is_v ? h - p.n_q_head - nk : h - p.n_q_head;
        const TI* src = is_q ? (const TI*)p.q + row * p.q_stride
                             : is_v ? (const TI*)p.v + row * p.v_stride : (const TI*)p.k + row * p.k_stride;
        src += hh * D;
        const int ea = e < half && !p.pairs ? e : 2 * e, eb = e < half && !p.pairs ? e + half : 2 * e + 1;
        float a = to_f32(src[ea]), b = to_f32(src[eb]);
        if (e < half && !is_v) {
            const float cs = p.cos[(int64_t)w.pos * half + e], sn = p.sin[(int64_t)w.pos * half + e];
            const float x0 = a, x1 = b;
            a = x0 * cs - x1 * sn;
            b = x0 * sn + x1 * cs;
        }
        T* dst;
        if (is_q)
            dst = (T*)p.q_out + row * p.q_out_stride + hh * D;
        else if (w.slot >= 0)
            dst = (T*)p.kv.pool + w.slot + (int64_t)((is_v ? nk : 0) + hh) * (PAGE * D);
        else
            continue;
        dst[ea] = from_f32<T>(a);
        dst[eb] = from_f32<T>(b);
    }
}

bool fits16(const void* p, int64_t stride, size_t size) {
    return !p || (((uintptr_t)p & 15) == 0 && (stride * (int64_t)size) % 16 == 0);
}

template <typename TI, typename T, int D>
void launch(const KvAppendParams& p, cudaStream_t s) {
    const size_t si = sizeof(TI), so = sizeof(T);
    const bool vec = p.rot % 16 == 0 && fits16(p.q, p.q_stride, si) && fits16(p.k, p.k_stride, si) &&
                     fits16(p.v, p.v_stride, si) && fits16(p.q_out, p.q_out_stride, so) &&
                     fits16(p.cos, 0, 4) && fits16(p.sin, 0, 4);
    if (!vec) {
        launch_pdl(k_kv_append_any<TI, T, D>, dim3((p.batch.n_rows + 3) / 4), dim3(128), 0, s, p);
        return;
    }
    // Threads per row: a warp when rows alone fill the GPU (31k rows of 48 heads x 128: 130 us, 170 with 256 threads a
    // row, whose angles then serve one head instead of twelve), up to 256 when there are few and latency counts.
    int per_row = 256;
    while (per_row > 32 && (int64_t)per_row * p.batch.n_rows > 148 * 2048) per_row /= 2;
    const int rows = 256 / per_row;
    launch_pdl(k_kv_append<TI, T, D>, dim3((p.batch.n_rows + rows - 1) / rows), dim3(256), 0, s, p, per_row / (D / 16));
}
template <typename TI, typename T>
void launch_d(const KvAppendParams& p, cudaStream_t s) {
    if (p.kv.head_dim == 32) launch<TI, T, 32>(p, s);
    else if (p.kv.head_dim == 64) launch<TI, T, 64>(p, s);
    else launch<TI, T, 128>(p, s);
}

}  // namespace

void launch_kv_append(const KvAppendParams& p, cudaStream_t s) {
    if (p.batch.n_rows <= 0) return;
    const bool f32 = p.row_dtype == GSVCU_KV_F32;
    if (p.kv.kv_dtype == GSVCU_KV_F32) launch_d<float, float>(p, s);
    else if (p.kv.kv_dtype == GSVCU_KV_F16) f32 ? launch_d<float, __half>(p, s) : launch_d<__half, __half>(p, s);
    else f32 ? launch_d<float, __nv_bfloat16>(p, s) : launch_d<__nv_bfloat16, __nv_bfloat16>(p, s);
}

}  // namespace gsvcu
