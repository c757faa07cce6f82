// paged_read.cu -- rows of the paged KV cache read back: the keys and values of the batch's tokens, as packed rows.
//
// Row i of a sequence's chunk of n rows is the token at cache position kv_len - n + i (a chunk of kv_len rows: the whole
// sequence). 4-bit caches: scale * (code - 8), exact in F16 and F32. Every element is read once and written once: bound by
// HBM (102k tokens of 8 heads x 128 from 4 bits to F32: 129.5 us, 6.2 TB/s; 184 with 8 elements a thread, whose F32 stores
// fill half of a sector each, and one head at a time), and by the chain row_start -> kv_len -> table -> load for few rows.
#include "paged_q4.cuh"
#include "paged_rows.cuh"

namespace gsvcu {
namespace {

// Thread = (row, lane u, head lane of the 2 n_head heads of K and V): 16 bytes of a row at a time, and NB heads in flight.
// TC: the cache's element, uint8_t for 4 bits. VEC: rows that 16-byte accesses fit.
template <typename TC, typename T, int D, bool VEC>
__global__ void __launch_bounds__(256) k_kv_read(KvReadParams p, int head_lanes) {
    constexpr bool Q4 = sizeof(TC) == 1;
    constexpr int E = 16 / sizeof(T), U = D / E, NB = 4;   // elements of a thread, threads of a head
    griddep_wait();
    griddep_launch();
    const int per_row = U * head_lanes, rows_per_cta = 256 / per_row;
    const int row = blockIdx.x * rows_per_cta + threadIdx.x / per_row;
    if (row >= p.batch.n_rows) return;   // (warp-uniform: per_row is a multiple of 32)
    const int t = threadIdx.x % per_row, e0 = t % U * E, hl = t / U, lane = threadIdx.x & 31;
    const Place w = place_of(p, row, lane, t == 0);
    if (w.block < 0) return;
    const int nk = p.kv.n_head;
    for (int h0 = hl; h0 < 2 * nk; h0 += NB * head_lanes) {
        float x[NB][E];
        if constexpr (Q4) {
            using B = Q4Block<D>;
            uint32_t code[NB];
            __half d[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int h = min(h0 + b * head_lanes, 2 * nk - 1);
                const uint8_t* block = (const uint8_t*)p.kv.pool + (w.block + h) * (int64_t)B::BYTES;
                const uint8_t* at = block + w.token * B::ROW + q4_place<D>(e0 / 8) + e0 % 8 / 2;
                code[b] = E == 8 ? *(const uint32_t*)at : *(const uint16_t*)at;
                d[b] = ((const __half*)(block + B::OFF_SCALES + w.token * B::SCALES))[e0 / 32];
            }
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < E; i++) x[b][i] = (float)((int)(code[b] >> (4 * i) & 15u) - 8) * __half2float(d[b]);
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const TC* src = (const TC*)p.kv.pool + ((w.block + min(h0 + b * head_lanes, 2 * nk - 1)) * PAGE + w.token) * D + e0;
                struct alignas(E * sizeof(TC)) Run { TC v[E]; };
                const Run y = *(const Run*)src;
#pragma unroll
                for (int i = 0; i < E; i++) x[b][i] = to_f32(y.v[i]);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int h = h0 + b * head_lanes;
            if (h >= 2 * nk) break;
            T* dst = (h < nk ? (T*)p.k + row * p.k_stride + h * D : (T*)p.v + row * p.v_stride + (h - nk) * D) + e0;
            if constexpr (VEC) {
                uint4 u;
                T* y = (T*)&u;
#pragma unroll
                for (int i = 0; i < E; i++) y[i] = from_f32<T>(x[b][i]);
                *(uint4*)dst = u;
            } else {
#pragma unroll
                for (int i = 0; i < E; i++) dst[i] = from_f32<T>(x[b][i]);
            }
        }
    }
}

template <typename TC, typename T, int D>
void launch(const KvReadParams& p, cudaStream_t s) {
    const bool vec = fits16(p.k, p.k_stride, sizeof(T)) && fits16(p.v, p.v_stride, sizeof(T));
    const int per_row = threads_per_row(p.batch.n_rows), rows = 256 / per_row;
    launch_pdl(vec ? k_kv_read<TC, T, D, true> : k_kv_read<TC, T, D, false>, dim3((p.batch.n_rows + rows - 1) / rows),
               dim3(256), 0, s, p, per_row / (D * (int)sizeof(T) / 16));
}
template <typename TC, typename T>
void launch_d(const KvReadParams& p, cudaStream_t s) {
    if (p.kv.head_dim == 32) launch<TC, T, 32>(p, s);
    else if (p.kv.head_dim == 64) launch<TC, T, 64>(p, s);
    else launch<TC, T, 128>(p, s);
}

}  // namespace

void launch_kv_read(const KvReadParams& p, cudaStream_t s) {
    if (p.batch.n_rows <= 0) return;
    const bool f32 = p.row_dtype == GSVCU_KV_F32;
    switch (p.kv.kv_dtype) {
        case GSVCU_KV_F32: launch_d<float, float>(p, s); break;
        case GSVCU_KV_F16: f32 ? launch_d<__half, float>(p, s) : launch_d<__half, __half>(p, s); break;
        case GSVCU_KV_BF16: f32 ? launch_d<__nv_bfloat16, float>(p, s) : launch_d<__nv_bfloat16, __nv_bfloat16>(p, s); break;
        case GSVCU_KV_Q4_F16: f32 ? launch_d<uint8_t, float>(p, s) : launch_d<uint8_t, __half>(p, s); break;
        default: f32 ? launch_d<uint8_t, float>(p, s) : launch_d<uint8_t, __nv_bfloat16>(p, s); break;
    }
}

}  // namespace gsvcu
