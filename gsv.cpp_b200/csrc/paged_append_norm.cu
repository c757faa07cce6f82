// paged_append_norm.cu -- new rows into the paged KV cache with a norm for each head before the rotation, and into 4-bit
// caches (paged_append.cu has the float caches without norms).
//
// Per head of a query or key row, D elements x: y = x * r * w with r = 1 / sqrt(mean(x^2) + eps) in f32; the squares are
// summed in 64 bits and rounded once, so that r, and with it every code next to a border, is the same in both kernels below
// whatever the order of the sum. Then the rotation (a' = a cos - b sin, b' = a sin + b cos, each operation rounded) and the
// rounding to the cache's type, or the quantiser of paged_q4.cuh: the largest magnitude over the lanes of a group, one word of
// codes per 8 elements.
// Every element is read once and written once: HBM bounds it on prompts, the chain row_start -> kv_len -> table -> store on
// single tokens (64 rows of 48 heads x 32: 2.9 us). 31k rows of 48 heads x 128: normalised, rotated, BF16 to BF16 149 to 157 us
// (5.0 to 5.3 TB/s; without norms 131: the sums of squares take a third of the instructions), F32 to F32 268 us (5.7 TB/s);
// into 4 bits 134 to 139 us without norms, 173 with (5.1 and 3.9 TB/s). With 8 elements a lane instead of 16 the first
// was 290 us, with the instruction that converts to F64 200.
#include "paged_q4.cuh"
#include "paged_rows.cuh"

namespace gsvcu {
namespace {

// 16 elements of a row as they were loaded, and as pairs.
template <typename TI> struct Raw { uint4 v[2 * sizeof(TI) / 2]; };
template <typename TI>
__device__ __forceinline__ void fetch(const TI* a, const TI* b, Raw<TI>& r) {
    constexpr int N = sizeof(TI) / 2;   // 16-byte pieces of 8 elements
#pragma unroll
    for (int i = 0; i < N; i++) {
        r.v[i] = ((const uint4*)a)[i];
        r.v[N + i] = ((const uint4*)b)[i];
    }
}
template <typename TI>
__device__ __forceinline__ void unpack(const Raw<TI>& r, float (&x)[16]) {
    const TI* t = (const TI*)r.v;
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = to_f32(t[i]);
}
// |x| * 2^128 as f64 in integer steps (the conversion instruction has a quarter of the rate): exact for normal numbers; a zero
// or subnormal one becomes 2 to 4, whose square is nothing beside any square that F32 can hold, an infinity or NaN one from
// 2^256 on, whose square makes the rounded sum infinite.
__device__ __forceinline__ double magnitude(float x) {
    const uint32_t u = __float_as_uint(x);
    return __hiloint2double((int)(((u >> 3) & 0x0fffffffu) | 0x40000000u), (int)(u << 29));
}
// a' = a c - b s, b' = a s + b c of two pairs: products packed, sums apart (ptxas fuses packed products into packed sums).
__device__ __forceinline__ void turn2(uint64_t& a, uint64_t& b, uint64_t c, uint64_t s) {
    const uint64_t ac = fmul2(a, c), bs = fmul2(b, s), as = fmul2(a, s), bc = fmul2(b, c);
    a = f2pack(f2lo(ac) - f2lo(bs), f2hi(ac) - f2hi(bs));
    b = f2pack(f2lo(as) + f2lo(bc), f2hi(as) + f2hi(bc));
}

// Vector form: thread = (row, unit u of D / 16, head lane). A unit is two runs of 8 elements that rotate with the same 8 angles
// (i and i + rot / 2, or 16 adjacent elements), so angles stay in registers over the heads; the next head's
// elements are on their way while one is worked on. A warp works on one row.
template <typename TI, typename T, int D, bool Q4, bool NORM>
__global__ void __launch_bounds__(256, sizeof(TI) == 4 ? 2 : 3) k_kv_append_norm(KvAppendParams p, int head_lanes) {
    constexpr int U = D / 16;
    __shared__ __align__(16) float weights[2][NORM ? D : 4];   // of q and k heads
    griddep_wait();
    griddep_launch();
    if constexpr (NORM) {
        for (int i = threadIdx.x; i < 2 * D; i += 256) {
            const float* src = i < D ? p.q_norm : p.k_norm;
            weights[i / D][i % D] = src ? src[i % D] : 1.0f;
        }
        __syncthreads();
    }
    const int per_row = U * head_lanes, rows_per_cta = 256 / per_row;
    const int row = blockIdx.x * rows_per_cta + threadIdx.x / per_row;
    if (row >= p.batch.n_rows) return;   // (warp-uniform: per_row is a multiple of 32)
    const int t = threadIdx.x % per_row, u = t % U, hl = t / U, lane = threadIdx.x & 31;
    const int nk = p.kv.n_head, nq = p.n_q_head, heads = nq + 2 * nk, n_rot = p.rot / 16;
    const bool turn = u < n_rot, apart = turn && !p.pairs;
    const int ea = apart ? u * 8 : u * 16, eb = apart ? p.rot / 2 + u * 8 : ea + 8;
    const TI* const q = (const TI*)p.q + row * p.q_stride;   // (heads are counted through q, k and v)
    const TI* const k = (const TI*)p.k + row * p.k_stride - nq * D;
    const TI* const v = (const TI*)p.v + row * p.v_stride - (nq + nk) * D;
    // Heads on their way: two where registers allow it (31k rows of 32/8 x 128 in BF16 into 4 bits: 134 us, 139 with one; with
    // norms, which need more registers: 185 and 174).
    constexpr int AHEAD = sizeof(TI) == 4 || NORM ? 1 : 2;
    Raw<TI> next[AHEAD];
    auto request = [&](int h, Raw<TI>& r) {
        const TI* src = (h < nq ? q : h < nq + nk ? k : v) + h * D;
        if (h < heads) fetch(src + ea, src + eb, r);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) request(hl + i * head_lanes, next[i]);
    const Place w = place_of(p, row, lane, t == 0);
    uint64_t cs[4], sn[4];
    if (p.rot) {
        const int pos = rotation_position(p, row, w.pos, t == 0);
        if (turn) {
            const float* ct = p.cos + (int64_t)pos * (p.rot / 2) + u * 8;
            const float* st = p.sin + (int64_t)pos * (p.rot / 2) + u * 8;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                cs[i] = f2pack(ct[2 * i], ct[2 * i + 1]);
                sn[i] = f2pack(st[2 * i], st[2 * i + 1]);
            }
        }
    }
    T* const q_out = (T*)p.q_out + row * p.q_out_stride;
    using Block = Q4Block<D>;
    const int64_t block = w.block - nq;
    auto work = [&](int h, Raw<TI>& raw) {   // (all lanes take part in the exchanges)
        const bool in = h < heads, is_q = h < nq, is_v = h >= nq + nk;
        float f[16];
        unpack(raw, f);
        request(h + AHEAD * head_lanes, raw);
        uint64_t x[8];       // run a, run b
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = f2pack(f[2 * i], f[2 * i + 1]);
        if (NORM && !__all_sync(0xffffffffu, is_v)) {
            double s0 = 0.0, s1 = 0.0;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const double y0 = magnitude(f[i]), y1 = magnitude(f[i + 1]);
                s0 = fma(y0, y0, s0);
                s1 = fma(y1, y1, s1);
            }
            s0 += s1;
#pragma unroll
            for (int o = 1; o < U; o *= 2) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
            float ss = (float)(s0 * 0x1p-256);
            if (__any_sync(0xffffffffu, isinf(ss))) {   // the sum overflows, or the head has an infinity or a NaN
                int nan = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) nan |= isnan(f[i]);
#pragma unroll
                for (int o = 1; o < U; o *= 2) nan |= __shfl_xor_sync(0xffffffffu, nan, o);
                if (nan) ss = __uint_as_float(0x7fffffffu);
            }
            if (!is_v && (is_q ? p.q_norm : p.k_norm)) {
                const float r = __frcp_rn(__fsqrt_rn(ss * (1.0f / D) + p.eps));
                const uint64_t r2 = f2pack(r, r);
                const float* wt = weights[is_q ? 0 : 1];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float4 y = *(const float4*)(wt + (i < 4 ? ea + 2 * i : eb + 2 * i - 8));
                    x[i] = fmul2(fmul2(x[i], r2), f2pack(y.x, y.y));
                    x[i + 1] = fmul2(fmul2(x[i + 1], r2), f2pack(y.z, y.w));
                }
            }
        }
        if (turn && !is_v) {
            if (p.pairs) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    uint64_t a = f2pack(f2lo(x[i]), f2lo(x[i + 1])), b = f2pack(f2hi(x[i]), f2hi(x[i + 1]));
                    turn2(a, b, cs[i / 2], sn[i / 2]);
                    x[i] = f2pack(f2lo(a), f2lo(b));
                    x[i + 1] = f2pack(f2hi(a), f2hi(b));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) turn2(x[i], x[4 + i], cs[i], sn[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f[2 * i] = f2lo(x[i]);
            f[2 * i + 1] = f2hi(x[i]);
        }
        if (!Q4 || __all_sync(0xffffffffu, is_q || !in)) {
            if (!in || (!is_q && w.block < 0)) return;
            T* dst = is_q ? q_out + h * D : (T*)p.kv.pool + ((block + h) * PAGE + w.token) * D;
            store8(dst + ea, *(const float(*)[8])f);
            store8(dst + eb, *(const float(*)[8])(f + 8));
            return;
        }
        uint32_t key[2] = {0, 0};   // (which lanes share a group: see fits_groups)
#pragma unroll
        for (int i = 0; i < 16; i++) key[i / 8] = max(key[i / 8], q4_key(f[i]));
#pragma unroll
        for (int i = 0; i < 2; i++) key[i] = max(key[i], __shfl_xor_sync(0xffffffffu, key[i], 1));
        const uint32_t both = max(key[0], key[1]);
        if (D == 128 || n_rot == 4) {
#pragma unroll
            for (int i = 0; i < 2; i++) key[i] = max(key[i], __shfl_xor_sync(0xffffffffu, key[i], 2));
        }
        if (!(apart && n_rot % 4 == 0)) key[0] = key[1] = both;
        if (is_q) {
            store8(q_out + h * D + ea, *(const float(*)[8])f);
            store8(q_out + h * D + eb, *(const float(*)[8])(f + 8));
        } else if (in && w.block >= 0) {
            uint8_t* to = (uint8_t*)p.kv.pool + (block + h) * Block::BYTES;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int run = (r ? eb : ea) / 8;
                float inv;
                const __half d = q4_scale(key[r], inv);
                *(uint32_t*)(to + w.token * Block::ROW + q4_place<D>(run)) = q4_word(f + 8 * r, inv);
                if (run % 4 == 0) ((__half*)(to + Block::OFF_SCALES + w.token * Block::SCALES))[run / 4] = d;
            }
        }
    };
    for (int h0 = hl; h0 - hl < heads; h0 += AHEAD * head_lanes) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (i == 0 || h0 - hl + i * head_lanes < heads) work(h0 + i * head_lanes, next[i]);
    }
}
// The vector form's groups of 32 elements: with i and i + rot / 2 in one unit, 4 neighbouring units have one group's four runs
// in their first halves and another's in their second when rot is a multiple of 64; two have all four when rot is 16 or 32;
// other widths mix them. Adjacent elements: two units.
bool fits_groups(const KvAppendParams& p) { return p.pairs || p.rot <= 32 || p.rot % 64 == 0; }

// Any alignment and rotation width: thread = (row, lane u of D / 8, head lane), 8 consecutive elements of a head, whose angles
// and weights stay in registers over the heads; partners through shared memory, rows that 16-byte accesses do not fit element
// by element. For what is rare: 31k rows of 48 heads x 128 in BF16, 96 rotated, into 4 bits 352 us; 120 rotated, rows at odd
// addresses, 449 us.
template <typename TI, typename T, int D, bool Q4>
__global__ void __launch_bounds__(256) k_kv_append_norm_any(KvAppendParams p, int head_lanes, bool aligned) {
    constexpr int U = D / 8;
    __shared__ float turned[256 * 8];
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
            if (aligned) {
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
            if (aligned) {
                store8(dst, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) dst[i] = from_f32<T>(x[i]);
            }
        } else if (w.block >= 0) {
            using B = Q4Block<D>;
            float inv;
            const __half d = q4_scale(key, inv);
            uint8_t* block = (uint8_t*)p.kv.pool + (w.block + (is_v ? nk : 0) + hh) * (int64_t)B::BYTES;
            *(uint32_t*)(block + w.token * B::ROW + q4_place<D>(u)) = q4_word(x, inv);
            if (u % 4 == 0) ((__half*)(block + B::OFF_SCALES + w.token * B::SCALES))[u / 4] = d;
        }
    }
}

template <typename TI, typename T, int D, bool Q4>
void launch(const KvAppendParams& p, cudaStream_t s) {
    const size_t si = sizeof(TI), so = sizeof(T);
    const bool aligned = fits16(p.q, p.q_stride, si) && fits16(p.k, p.k_stride, si) && fits16(p.v, p.v_stride, si) &&
                         fits16(p.q_out, p.q_out_stride, so);
    const bool vec = aligned && p.rot % 16 == 0 && (!Q4 || fits_groups(p));
    const int per_row = threads_per_row(p.batch.n_rows), rows = 256 / per_row;
    const dim3 grid((p.batch.n_rows + rows - 1) / rows);
    auto go = [&](auto kernel) { launch_pdl(kernel, grid, dim3(256), 0, s, p, per_row / (D / 16)); };
    if (!vec) launch_pdl(k_kv_append_norm_any<TI, T, D, Q4>, grid, dim3(256), 0, s, p, per_row / (D / 8), aligned);
    else if (p.q_norm || p.k_norm) go(k_kv_append_norm<TI, T, D, Q4, true>);
    else if constexpr (Q4) go(k_kv_append_norm<TI, T, D, Q4, false>);   // (float caches without norms: paged_append.cu)
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
