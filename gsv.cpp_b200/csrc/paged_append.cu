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
#include "paged_rows.cuh"

namespace gsvcu {
namespace {

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
    const Place w = place_of(p, row, lane, t == 0);
    const int pos = p.rot ? rotation_position(p, row, w.pos, t == 0) : 0;
    const int n_rot = p.rot / 16;
    const bool turn = u < n_rot;
    const int ea = !turn ? u * 16 : p.pairs ? u * 16 : u * 8;
    const int eb = !turn ? ea + 8 : p.pairs ? ea + 8 : p.rot / 2 + u * 8;
    float cs[8], sn[8];
    if (turn) {
        load8(p.cos + (int64_t)pos * (p.rot / 2) + u * 8, cs);
        load8(p.sin + (int64_t)pos * (p.rot / 2) + u * 8, sn);
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
        else if (w.block >= 0)
            dst = (T*)p.kv.pool + ((w.block + (is_v ? nk : 0) + hh) * PAGE + w.token) * D;
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
    const Place w = place_of(p, row, lane, lane == 0);
    const int pos = p.rot ? rotation_position(p, row, w.pos, lane == 0) : 0;
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
            const float cs = p.cos[(int64_t)pos * half + e], sn = p.sin[(int64_t)pos * half + e];
            const float x0 = a, x1 = b;
            a = x0 * cs - x1 * sn;
            b = x0 * sn + x1 * cs;
        }
        T* dst;
        if (is_q)
            dst = (T*)p.q_out + row * p.q_out_stride + hh * D;
        else if (w.block >= 0)
            dst = (T*)p.kv.pool + ((w.block + (is_v ? nk : 0) + hh) * PAGE + w.token) * D;
        else
            continue;
        dst[ea] = from_f32<T>(a);
        dst[eb] = from_f32<T>(b);
    }
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
    const int per_row = threads_per_row(p.batch.n_rows);
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
