// paged_append_norm.cu -- new rows into the paged KV cache with a norm for each head before the rotation, and into 4-bit
// caches (paged_append.cu has the float caches without norms).
//
// Per head of a query or key row, D elements x: y = x * r * w with r = 1 / sqrt(mean(x^2) + eps) in f32; the squares are
// summed in 64 bits and rounded once, so that r, and with it every code next to a border, does not depend on the order of
// the sum. Then the rotation (a' = a cos - b sin, b' = a sin + b cos, each operation rounded) and the rounding to the
// cache's type, or the quantiser of paged_q4.cuh: amax over the 4 lanes of a group, one word of codes per lane.
// Every element is read once and written once: HBM bounds it on prompts, the chain row_start -> kv_len -> table -> store on
// single tokens.
#include "paged_q4.cuh"
#include "paged_rows.cuh"

namespace gsvcu {
namespace {

// Thread = (row, lane u of D / 8, head lane): 8 consecutive elements of a head, whose angles and weights stay in registers
// over the heads. VEC: 16-byte accesses; else element by element, for any alignment and rotation width.
template <typename TI, typename T, int D, bool Q4, bool VEC>
__global__ void __launch_bounds__(256) k_kv_append_norm(KvAppendParams p, int head_lanes) {
    constexpr int U = D / 8;
    __shared__ float turned[VEC ? 1 : 256 * 8];
    griddep_wait();
    griddep_launch();
    const int per_row = U * head_lanes, rows_per_cta = 256 / per_row;
    const int row = blockIdx.x * rows_per_cta + threadIdx.x / per_row;
    if (row >= p.batch.n_rows) return;   // (warp-uniform: per_row is a multiple of 32)
    const int t = threadIdx.x % per_row, u = t % U, hl = t / U, lane = threadIdx.x & 31;
    const Place w = place_of(p, row, lane, t == 0);
    const int e0 = u * 8, half = p.rot / 2;
    // x' = x c + partner s, s negative for the first of a pair
    float cs[8], sn[8], wq[8], wk[8];
    if (p.rot) {
        const int pos = rotation_position(p, row, w.pos, t == 0);
        const float* ct = p.cos + (int64_t)pos * half;
        const float* st = p.sin + (int64_t)pos * half;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int e = e0 + i, a = p.pairs ? e / 2 : e < half ? e : e - half;
            const bool turn = e < p.rot, first = p.pairs ? e % 2 == 0 : e < half;
            cs[i] = turn ? ct[a] : 1.0f;
            sn[i] = turn ? (first ? -st[a] : st[a]) : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        wq[i] = p.q_norm ? p.q_norm[e0 + i] : 1.0f;
        wk[i] = p.k_norm ? p.k_norm[e0 + i] : 1.0f;
    }
    const int nk = p.kv.n_head, heads = p.n_q_head + 2 * nk;
    for (int h0 = 0; h0 < heads; h0 += head_lanes) {   // (all lanes take part in the exchanges)
        const int h = h0 + hl;
        const bool in = h < heads, is_q = h < p.n_q_head, is_v = h >= p.n_q_head + nk;
        const int hh = is_q ? h : is_v ? h - p.n_q_head - nk : h - p.n_q_head;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = 0.0f;
        if (in) {
            const TI* src = is_q ? (const TI*)p.q + row * p.q_stride
                                 : is_v ? (const TI*)p.v + row * p.v_stride : (const TI*)p.k + row * p.k_stride;
            src += hh * D + e0;
            if constexpr (VEC) {
                load8(src, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = to_f32(src[i]);
            }
        }
        if (p.q_norm || p.k_norm) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fma((double)x[i], (double)x[i], ss);
#pragma unroll
            for (int o = 1; o < U; o *= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (!is_v && (is_q ? p.q_norm : p.k_norm)) {
                const float r = __fdiv_rn(1.0f, __fsqrt_rn((float)ss * (1.0f / D) + p.eps));
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = x[i] * r * (is_q ? wq[i] : wk[i]);
            }
        }
        if (p.rot) {
            float y[8];   // partners
            if constexpr (!VEC) {
                float* mine = turned + threadIdx.x * 8;
#pragma unroll
                for (int i = 0; i < 8; i++) mine[i] = x[i];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int e = e0 + i;
                    const int other = e >= p.rot ? e : p.pairs ? e ^ 1 : e < half ? e + half : e - half;
                    y[i] = turned[(threadIdx.x - u) * 8 + other];
                }
                __syncwarp();
            } else if (p.pairs) {
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = x[i ^ 1];
            } else {   // (half is a multiple of 8)
                const int from = e0 < half ? lane + half / 8 : e0 < p.rot ? lane - half / 8 : lane;
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = __shfl_sync(0xffffffffu, x[i], from);
            }
            if (!is_v) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (e0 + i < p.rot) x[i] = x[i] * cs[i] + y[i] * sn[i];
            }
        }
        uint32_t key = 0;
        if constexpr (Q4) {
#pragma unroll
            for (int i = 0; i < 8; i++) key = max(key, q4_key(x[i]));
            key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
            key = max(key, __shfl_xor_sync(0xffffffffu, key, 2));
        }
        if (!in) continue;
        if (is_q || !Q4) {
            if (!is_q && w.block < 0) continue;
            T* dst = is_q ? (T*)p.q_out + row * p.q_out_stride + hh * D
                          : (T*)p.kv.pool + ((w.block + (is_v ? nk : 0) + hh) * PAGE + w.token) * D;
            dst += e0;
            if constexpr (VEC) {
                store8(dst, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) dst[i] = from_f32<T>(x[i]);
            }
        } else if (w.block >= 0) {
            using B = Q4Block<D>;
            float inv;
            const __half d = q4_scale(key, inv);
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) word |= q4_code(x[i], inv) << (4 * i);
            uint8_t* block = (uint8_t*)p.kv.pool + (w.block + (is_v ? nk : 0) + hh) * (int64_t)B::BYTES;
            *(uint32_t*)(block + w.token * B::ROW + q4_place<D>(u)) = word;
            if (u % 4 == 0) ((__half*)(block + B::OFF_SCALES + w.token * B::SCALES))[u / 4] = d;
        }
    }
}

template <typename TI, typename T, int D, bool Q4>
void launch(const KvAppendParams& p, cudaStream_t s) {
    const size_t si = sizeof(TI), so = sizeof(T);
    const bool vec = p.rot % 16 == 0 && fits16(p.q, p.q_stride, si) && fits16(p.k, p.k_stride, si) &&
                     fits16(p.v, p.v_stride, si) && fits16(p.q_out, p.q_out_stride, so);
    const int per_row = threads_per_row(p.batch.n_rows), rows = 256 / per_row;
    launch_pdl(vec ? k_kv_append_norm<TI, T, D, Q4, true> : k_kv_append_norm<TI, T, D, Q4, false>,
               dim3((p.batch.n_rows + rows - 1) / rows), dim3(256), 0, s, p, per_row / (D / 8));
}
template <typename TI, typename T, bool Q4>
void launch_d(const KvAppendParams& p, cudaStream_t s) {
    if (p.kv.head_dim == 32) launch<TI, T, 32, Q4>(p, s);
    else if (p.kv.head_dim == 64) launch<TI, T, 64, Q4>(p, s);
    else launch<TI, T, 128, Q4>(p, s);
}
template <typename TI, typename T>
void launch_q4(const KvAppendParams& p, cudaStream_t s) {
    if (is_q4(p.kv.kv_dtype)) launch_d<TI, T, true>(p, s);
    else launch_d<TI, T, false>(p, s);
}

}  // namespace

void launch_kv_append_norm(const KvAppendParams& p, cudaStream_t s) {
    if (p.batch.n_rows <= 0) return;
    const bool f32 = p.row_dtype == GSVCU_KV_F32;
    const int ty = row_type(p.kv.kv_dtype);
    if (ty == GSVCU_KV_F32) launch_d<float, float, false>(p, s);
    else if (ty == GSVCU_KV_F16) f32 ? launch_q4<float, __half>(p, s) : launch_q4<__half, __half>(p, s);
    else f32 ? launch_q4<float, __nv_bfloat16>(p, s) : launch_q4<__nv_bfloat16, __nv_bfloat16>(p, s);
}

}  // namespace gsvcu
