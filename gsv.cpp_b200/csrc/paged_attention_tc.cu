// paged_attention_tc.cu -- attention of many new rows over the paged KV cache on the 5th-generation tensor
// cores (F16 / BF16); the operator's formula and the variant for few rows are in paged_attention.cu.
//
// k_chunk_attn_tc: one CTA per (sequence, 256 packed rows, kv head, key split), as two row tiles of 128 rows
// (packed row r = token * g + query head of the group). Key tiles are 128 keys = two pages, each page's
// [64][head dim] block fetched by TMA into a ring that K and V tiles take in turn (K0 V0 K1 V1 ...).
//   warp 0     page numbers (32 per load) and TMA
//   warp 1     MMA: S = Q K^T (both operands in shared memory), O += P V (P in tensor memory, V in shared
//              memory as it lies in the page: the MN-major operand, so nothing is transposed)
//   warps 4-7  softmax of row tile 0, one thread per row (TMEM lane); warps 8-11 of row tile 1
// The MMAs of one row tile run under the other's softmax: S0 S1 | PV0 S0' PV1 S1' | ... Each thread takes its
// 128 scores into registers, writes the weights P over them in tensor memory as 16-bit pairs, and keeps the
// row's sum. A row's reference maximum is raised only when a tile exceeds it by more than 2^TAU, then O in
// tensor memory is scaled once its last PV is done; so P <= 2^TAU, far inside F16. Weights are rounded to the
// cache's type for the product: with the output's own rounding that is sqrt(2) of it, and the sums stay f32.
// Tensor memory: S0 | S1 (128 columns each; P over their first 64) | O0 | O1.
// V rows past kv_len in the last tile are zeroed in shared memory before its product, absent pages are
// zero-filled by TMA (a block index past the pool), masked keys get weight 0.
#include <cuda_bf16.h>

#include "paged.h"
#include "paged_join.cuh"
#include "tc_common.cuh"

namespace gsvcu {
namespace {

using namespace tc;

constexpr int KT = 128;                 // keys per tile
constexpr int ROWS = 256;               // packed rows per CTA
constexpr int THREADS = 384;
constexpr float TAU = 8.0f;             // log2 headroom of P above the row's reference maximum
constexpr uint32_t TM_O = 256;          // tensor-memory column of O0

template <int D>
struct Smem {
    static constexpr int RB = D >= 64 ? 128 : 2 * D;              // bytes of a swizzled row
    static constexpr int ATOMS = D >= 64 ? D / 64 : 1;            // 64-dim column blocks of a tile
    static constexpr int ENTRY = KT * D * 2;                      // bytes of a K or V tile
    static constexpr int NE = D == 128 ? 4 : 8;                   // ring entries
    static constexpr size_t OFF_RING = (size_t)ROWS * D * 2;      // after Q
    static constexpr size_t OFF_BAR = OFF_RING + (size_t)NE * ENTRY;
    static constexpr int NBAR = 2 * NE + 7;                       // full, empty, S full [2], P full [2], O done [2], drain
    static constexpr size_t SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
};

struct TcArgs {
    ChunkAttnParams p;
    CUtensorMap map;   // pool as [block][64][D], box [1][64][min(D, 64)]
    int group, tiles, n_split, split_tiles, n_blocks;
    float c;           // |scale| * log2(e)
    bool negate;       // scale < 0: Q enters negated
    bool vec_q, vec_out;
};

// Shared-memory operand descriptor: address and strides in 16-byte units, version 1, swizzle of RB-byte rows.
template <int RB>
__device__ __forceinline__ uint64_t op_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    constexpr uint64_t mode = RB == 128 ? 2 : 4;   // 128- or 64-byte swizzle
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) |
           ((uint64_t)1 << 46) | (mode << 61);
}
// Instruction descriptor: f32 accumulator, 16-bit operands (0 F16, 1 BF16), B MN-major when `tb`.
__host__ __device__ constexpr uint32_t instr(int type, int tb, int n) {
    return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)tb << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
// D (tensor memory) (+)= A (tensor memory, 16-bit pairs) x B (shared memory).
__device__ __forceinline__ void mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
#define R8(x, i) "+r"(x[i]), "+r"(x[i + 1]), "+r"(x[i + 2]), "+r"(x[i + 3]), "+r"(x[i + 4]), "+r"(x[i + 5]), "+r"(x[i + 6]), "+r"(x[i + 7])
#define R32(x) R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24)
#define W8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define V8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// 32 tensor-memory columns of the warp's lanes; the values count after tmem_wait_ld + bind32.
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : W8(r, 0), W8(r, 8), W8(r, 16), W8(r, 24)
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void bind32(uint32_t (&r)[32]) { asm volatile("" : R32(r) : : "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
        V8(r, 0), V8(r, 8), V8(r, 16), V8(r, 24)
        : "memory");
}
__device__ __forceinline__ void tmem_st16u(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
        V8(r, 0), V8(r, 8)
        : "memory");
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const uint32_t*)&h;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const uint32_t*)&h;
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1) k_chunk_attn_tc(const __grid_constant__ TcArgs a) {
    using L = Smem<D>;
    constexpr int TY = __is_same(T, __half) ? 0 : 1;
    constexpr uint32_t ID_S = instr(TY, 0, KT), ID_O = instr(TY, 1, D);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u);
    const ChunkAttnParams& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t bar0 = su32(sm + L::OFF_BAR);
    auto full = [&](int e) { return bar0 + 8u * e; };
    auto empty = [&](int e) { return bar0 + 8u * (L::NE + e); };
    auto sfull = [&](int t) { return bar0 + 8u * (2 * L::NE + t); };
    auto pfull = [&](int t) { return bar0 + 8u * (2 * L::NE + 2 + t); };
    auto odone = [&](int t) { return bar0 + 8u * (2 * L::NE + 4 + t); };
    const uint32_t drain = bar0 + 8u * (2 * L::NE + 6);
    uint32_t* tmem_slot = (uint32_t*)(sm + L::OFF_BAR + L::NBAR * 8);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    int* last_slot = (int*)(tmem_slot + 2);

    int id = blockIdx.x;
    const int sp = id % a.n_split;
    id /= a.n_split;
    const int h = id % p.kv.n_head;
    id /= p.kv.n_head;
    const int s = id % p.batch.n_seq, tile = a.tiles - 1 - id / p.batch.n_seq;   // the last rows see most keys: first
    griddep_wait();
    griddep_launch();

    ChunkRange c;
    if (!chunk_range(p, s, tile, a.group, ROWS, KT, tid == 0 && sp == 0 && h == 0 && tile == 0, c)) return;
    const int n_act = max(1, (c.n_tiles + a.split_tiles - 1) / a.split_tiles);
    if (sp >= n_act) return;
    const int v0 = sp * a.split_tiles, nt = min(c.n_tiles, v0 + a.split_tiles) - v0;   // this CTA's key tiles
    const int halves = c.rows > 128 ? 2 : 1;
    auto key0 = [&](int j) { return c.tile_of(v0 + j) * KT; };

    if (tid == 0) {
        for (int e = 0; e < L::NE; e++) { bar_init(full(e), 1); bar_init(empty(e), 1); }
        for (int t = 0; t < 2; t++) { bar_init(sfull(t), 1); bar_init(pfull(t), 128); bar_init(odone(t), 1); }
        bar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Q, swizzled as the MMA reads it ([tile][64-dim block][128 rows][RB bytes]), zero past the CTA's rows
    for (int i = tid; i < ROWS * (D / 8); i += THREADS) {
        const int r = i / (D / 8), pc = i % (D / 8);
        if (r >= 128 * halves) break;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < c.rows) {
            const int tok = (c.r0 + r) / a.group, j = (c.r0 + r) % a.group;
            const T* src = (const T*)p.q + (int64_t)(c.row0 + tok) * p.q_stride + (int64_t)(h * a.group + j) * D + pc * 8;
            if (a.vec_q) {
                u = *(const uint4*)src;
            } else {
                T* x = (T*)&u;
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = src[k];
            }
            if (a.negate) { u.x ^= 0x80008000u; u.y ^= 0x80008000u; u.z ^= 0x80008000u; u.w ^= 0x80008000u; }
        }
        const int rt = r & 127, atom = D >= 64 ? pc / 8 : 0, ch = D >= 64 ? pc % 8 : pc;
        const int swz = L::RB == 128 ? rt & 7 : (rt >> 1) & 3;
        *(uint4*)(sm + (size_t)(r >> 7) * 128 * D * 2 + (size_t)atom * 128 * L::RB + rt * L::RB + ((ch ^ swz) << 4)) = u;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ring entry g: K (even) or V (odd) of tile g / 2
        const int32_t* tab = p.batch.table + (int64_t)s * p.batch.max_pages;
        int blk = 0;
        bool ok = true, bad = false;
        int g = 0;
        for (; g < 2 * nt && ok; g++) {
            const int j = g >> 1, e = g % L::NE;
            if ((g & 1) == 0 && (j & 15) == 0) {   // the blocks of 16 tiles: lane = (tile, page)
                const int jj = j + (lane >> 1);
                blk = a.n_blocks;                   // past the pool: zero fill
                if (jj < nt) {
                    const int key = key0(jj) + PAGE * (lane & 1);
                    if (key < c.len) {
                        const int page = tab[key / PAGE];
                        if (page >= 0 && page < p.kv.n_page) blk = ((page * p.kv.n_layer + p.kv.layer) * 2) * p.kv.n_head + h;
                        else bad = true;
                    }
                }
            }
            const int b0 = __shfl_sync(0xffffffffu, blk, (j & 15) * 2), b1 = __shfl_sync(0xffffffffu, blk, (j & 15) * 2 + 1);
            if (lane == 0) {
                ok = bar_wait_short(empty(e), ((uint32_t)(g / L::NE) & 1u) ^ 1u, abort_flag);
                if (ok) {
                    bar_expect_tx(full(e), L::ENTRY);
                    const uint32_t dst = su32(sm + L::OFF_RING + (size_t)e * L::ENTRY);
                    const int dv = (g & 1) ? p.kv.n_head : 0;
#pragma unroll
                    for (int at = 0; at < L::ATOMS; at++) {
                        tma_load_3d(dst + at * KT * L::RB, &a.map, at * 64, 0, b0 < a.n_blocks ? b0 + dv : b0, full(e));
                        tma_load_3d(dst + at * KT * L::RB + PAGE * L::RB, &a.map, at * 64, 0, b1 < a.n_blocks ? b1 + dv : b1, full(e));
                    }
                }
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        }
        if (bad) atomicOr(p.err, PAGED_BAD_PAGE);
        if (lane == 0) {
            if (!ok) {
                atomicOr(p.err, PAGED_WAIT);
                *abort_flag = 1;
                g--;   // its copies were not issued
            }
            // every copy has landed before the CTA may end
            for (int k = g - 1; k >= 0 && k >= g - L::NE; k--)
                for (uint32_t it = 0; it < TC_POLL_LIMIT; it++)
                    if (bar_try(full(k % L::NE), (uint32_t)(k / L::NE) & 1u)) break;
        }
    } else if (warp == 1) {
        const uint32_t sq = su32(sm), ring = su32(sm + L::OFF_RING);
        bool ok = true;
        auto wait_entry = [&](int g) { return bar_wait_short_warp(full(g % L::NE), (uint32_t)(g / L::NE) & 1u, abort_flag); };
        auto scores = [&](int t, int j) {   // S_t = Q_t K_j^T
            if (lane != 0) return;
            const uint32_t k = ring + (uint32_t)((2 * j) % L::NE) * L::ENTRY, q = sq + (uint32_t)t * 128 * D * 2;
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) {
                const uint32_t off = (uint32_t)(kk / 4) * 128 * L::RB + 32u * (kk % 4);   // 64-dim block, 16 dims in it
                umma_f16(tmem + (uint32_t)t * KT, op_desc<L::RB>(q + off, 16, 8 * L::RB), op_desc<L::RB>(k + off, 16, 8 * L::RB),
                         ID_S, (uint32_t)kk);
            }
            umma_commit(sfull(t));
            if (t == halves - 1) umma_commit(empty((2 * j) % L::NE));
        };
        auto values = [&](int t, int j) {   // O_t += P_t V_j
            if (lane != 0) return;
            const uint32_t v = ring + (uint32_t)((2 * j + 1) % L::NE) * L::ENTRY;
#pragma unroll
            for (int kk = 0; kk < KT / 16; kk++)
                mma_ta(tmem + TM_O + (uint32_t)t * 128, tmem + (uint32_t)t * KT + 8u * kk,
                       op_desc<L::RB>(v + (uint32_t)kk * 16 * L::RB, KT * L::RB, 8 * L::RB), ID_O, (uint32_t)(j | kk));
            if (j == nt - 1) umma_commit(odone(t));
            if (t == halves - 1) umma_commit(empty((2 * j + 1) % L::NE));
        };
        if (nt > 0) {
            ok = wait_entry(0);
            if (ok)
                for (int t = 0; t < halves; t++) scores(t, 0);
        }
        for (int j = 0; j < nt && ok; j++) {
            ok = wait_entry(2 * j + 1);
            if (!ok) break;
            const int k0 = key0(j);
            if (k0 + KT > c.len) {   // V rows past the last key: whatever the page holds there, 0 here
                uint8_t* v = sm + L::OFF_RING + (size_t)((2 * j + 1) % L::NE) * L::ENTRY;
                const int r0 = c.len - k0, n16 = L::RB / 16;
                for (int at = 0; at < L::ATOMS; at++)
                    for (int i = r0 * n16 + lane; i < KT * n16; i += 32)
                        *(uint4*)(v + (size_t)at * KT * L::RB + i * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            for (int t = 0; t < halves && ok; t++) {
                ok = bar_wait_short_warp(pfull(t), (uint32_t)j & 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
                values(t, j);
                if (j + 1 < nt) {
                    if (t == 0) ok = wait_entry(2 * j + 2);
                    if (ok) scores(t, j + 1);
                }
            }
        }
        if (lane == 0 && !ok) {
            atomicOr(p.err, PAGED_WAIT);
            *abort_flag = 1;
            umma_commit(drain);   // what was issued ends before the tensor memory is freed
            for (uint32_t it = 0; it < TC_POLL_LIMIT; it++)
                if (bar_try(drain, 0)) break;
        }
    } else if (warp >= 4 && (warp - 4) / 4 < halves) {
        const int t = (warp - 4) / 4, q = warp & 3, r = 128 * t + 32 * q + lane;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16), ts = tl + (uint32_t)t * KT, to = tl + TM_O + (uint32_t)t * 128;
        const int pos = c.total - c.n + (c.r0 + min(r, c.rows - 1)) / a.group;
        const int see_hi = min(c.len, pos + 1), see_lo = p.window ? pos - p.window + 1 : 0;
        float mref = NEG_INF, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < nt && ok; j++) {
            if (!bar_wait_short_warp(sfull(t), (uint32_t)j & 1u, abort_flag)) { ok = false; break; }
            tc_fence_after();
            uint32_t x[4][32];
#pragma unroll
            for (int k = 0; k < 4; k++) tmem_ld32(ts + 32u * k, x[k]);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 4; k++) bind32(x[k]);
            const int k0 = key0(j);
            if (!(k0 + KT <= c.np || (k0 + KT <= min(c.len, c.p0 + 1) && (!p.window || k0 > c.p1 - p.window)))) {
#pragma unroll
                for (int i = 0; i < KT; i++) {
                    const int key = k0 + i;
                    if (!(key < c.np || (key < see_hi && key >= see_lo))) x[i / 32][i % 32] = __float_as_uint(NEG_INF);
                }
            }
            float mx[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                mx[k] = __uint_as_float(x[k][0]);
#pragma unroll
                for (int i = 1; i < 32; i++) mx[k] = fmaxf(mx[k], __uint_as_float(x[k][i]));
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.c;
            // raise the reference maximum of the warp's rows when one of them needs it
            if (__any_sync(0xffffffffu, top > mref + TAU)) {
                const float up = fmaxf(mref, top);
                if (j > 0) {   // (O is at rest: S of this tile was committed after the PV before it)
                    const float f = up == NEG_INF ? 1.0f : ex2(mref - up);
                    l *= f;
#pragma unroll 1
                    for (int d = 0; d < D; d += 32) {
                        uint32_t o[32];
                        tmem_ld32(to + (uint32_t)d, o);
                        tmem_wait_ld();
                        bind32(o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st32(to + (uint32_t)d, o);
                    }
                    tmem_wait_st();
                }
                mref = up;
            }
            const float ref = mref == NEG_INF ? 0.0f : -mref;
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float w0 = ex2(fmaf(__uint_as_float(x[k][2 * i]), a.c, ref));
                    const float w1 = ex2(fmaf(__uint_as_float(x[k][2 * i + 1]), a.c, ref));
                    sum[0] += w0;
                    sum[1] += w1;
                    w[i] = pack2<T>(w0, w1);
                }
                tmem_st16u(ts + 16u * k, w);
            }
            l += sum[0] + sum[1];
            tmem_wait_st();
            tc_fence_before();
            bar_arrive(pfull(t));
        }
        if (ok && nt > 0) ok = bar_wait_short_warp(odone(t), 0, abort_flag);
        tc_fence_after();
        const bool mine = r < c.rows;
        const int tok = (c.r0 + r) / a.group, head = h * a.group + (c.r0 + r) % a.group;
        const int64_t row = c.row0 + tok;
        const int64_t unit = ((int64_t)s * a.tiles + tile) * p.kv.n_head + h;
        float* part = p.part + unit * a.n_split * (ROWS * (D + 2));
        const float il = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        if (ok) {
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
                uint32_t o[32];
                if (nt > 0) {
                    tmem_ld32(to + (uint32_t)d, o);
                    tmem_wait_ld();
                    bind32(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = 0;
                }
                if (!mine) continue;
                if (n_act == 1) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float y[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) y[k] = __uint_as_float(o[i + k]) * il;
                        T* dst = (T*)p.out + row * p.out_stride + (int64_t)head * D + d + i;
                        const uint4 u = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
                        if (a.vec_out) {
                            *(uint4*)dst = u;
                        } else {
                            const T* e = (const T*)&u;
#pragma unroll
                            for (int k = 0; k < 8; k++) dst[k] = e[k];
                        }
                    }
                } else {
                    float* dst = part + ((int64_t)sp * ROWS + r) * D + d;
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *(uint4*)(dst + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
            }
            if (mine) {
                if (n_act > 1)
                    *(float2*)(part + (int64_t)a.n_split * ROWS * D + 2 * ((int64_t)sp * ROWS + r)) = make_float2(mref, l);
                else if (p.lse)
                    p.lse[row * p.n_q_head + head] = mref == NEG_INF ? NEG_INF : (mref + log2f(l)) * LN2;
            }
        } else if (lane == 0) {
            atomicOr(p.err, PAGED_WAIT);
            *abort_flag = 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (n_act > 1) join_splits<T, D, ROWS, THREADS>(p, c, s, tile, h, a.group, a.tiles, a.n_split, n_act, a.vec_out, last_slot);
}

template <typename F>
void pick_tc(int dtype, int dim, F f) {
    if (dtype == GSVCU_KV_F16) {
        if (dim == 32) f(k_chunk_attn_tc<__half, 32>, Smem<32>::SMEM);
        else if (dim == 64) f(k_chunk_attn_tc<__half, 64>, Smem<64>::SMEM);
        else f(k_chunk_attn_tc<__half, 128>, Smem<128>::SMEM);
    } else {
        if (dim == 32) f(k_chunk_attn_tc<__nv_bfloat16, 32>, Smem<32>::SMEM);
        else if (dim == 64) f(k_chunk_attn_tc<__nv_bfloat16, 64>, Smem<64>::SMEM);
        else f(k_chunk_attn_tc<__nv_bfloat16, 128>, Smem<128>::SMEM);
    }
}

}  // namespace

cudaError_t chunk_attention_tc_init_device() {
    cudaError_t e = cudaSuccess;
    for (int ty : {GSVCU_KV_F16, GSVCU_KV_BF16})
        for (int dim : {32, 64, 128})
            pick_tc(ty, dim, [&](auto k, size_t smem) {
                const cudaError_t r = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
                if (e == cudaSuccess) e = r;
            });
    return e;
}

bool launch_chunk_attention_tc(const ChunkAttnParams& p, const ChunkAttnPlan& plan, cudaStream_t s) {
    TcArgs a;
    a.p = p;
    a.group = p.n_q_head / p.kv.n_head;
    a.tiles = plan.tiles;
    a.n_split = plan.n_split;
    a.split_tiles = plan.split_tiles;
    a.n_blocks = p.kv.n_page * p.kv.n_layer * 2 * p.kv.n_head;
    a.c = fabsf(p.scale) * LOG2E;
    a.negate = p.scale < 0.0f;
    a.vec_q = ((uintptr_t)p.q & 15) == 0 && p.q_stride % 8 == 0;
    a.vec_out = ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0;
    const int D = p.kv.head_dim;
    const EncodeTiledFn encode = encode_fn();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)PAGE, (cuuint64_t)a.n_blocks};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)PAGE * D * 2};
    const cuuint32_t box[3] = {(cuuint32_t)(D < 64 ? D : 64), (cuuint32_t)PAGE, 1}, step[3] = {1, 1, 1};
    if (encode(&a.map, p.kv.kv_dtype == GSVCU_KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
               p.kv.pool, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               D >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    const int64_t ctas = (int64_t)p.batch.n_seq * plan.tiles * p.kv.n_head * plan.n_split;
    pick_tc(p.kv.kv_dtype, D, [&](auto k, size_t smem) {
        launch_pdl(k, dim3((unsigned)ctas), dim3(THREADS), smem, s, a);
    });
    return true;
}

}  // namespace gsvcu
