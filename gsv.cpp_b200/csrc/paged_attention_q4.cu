// paged_attention_q4.cu -- attention of few new rows over a 4-bit paged cache (layout and scales: paged_q4.cuh; the
// operator's formula and the float caches: paged_attention.cu).
//
// k_chunk_attn_q4 has the shape of k_chunk_attn: one CTA per (sequence, row tile, kv head, key split), four warps that
// take the split's key tiles in turn, each with its own cp.async ring, running maximum, sum and output; transposed
// products (16 keys x 8 query rows), warps joined in order, splits by the last CTA or by k_chunk_join. All products are F16
// mma.m16n8k16, whatever the rows' type (BF16 queries fit F16 up to 65,504; beyond they count as overflowing):
//   scores   the codes less 8 are exact in F16, and a group of 32 elements is two products, so a group's sum is multiplied
//            by its key's scale in f32 afterwards;
//   values   scale * (code - 8) is exact in F16 too (scales have 8 significant bits) and takes one fused multiply-add per
//            pair: a code moved to bits 6 .. 9 under the exponent of 16 is the number 16 + code, times the scale less 24
//            scales.
// The weights are split into two F16 parts, kept 2^14 up, as in k_chunk_attn.
#include "paged_q4.cuh"

#include <algorithm>

#include "paged.h"
#include "paged_join.cuh"

namespace gsvcu {
namespace {

constexpr int NW = 4;            // warps per CTA
constexpr int UNPACK_ROWS = 1536;
constexpr float BIAS = 14.0f;    // weights are 2^BIAS exp(s - maximum)
__host__ __device__ constexpr int key_tile(int dim) { return dim == 32 ? 64 : 32; }

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes, of which the first n (0 .. 16) are read and the others zero.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int N>   // words
__device__ __forceinline__ void lds(uint32_t a, uint32_t (&x)[N]) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a) : "memory");
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(a) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x[0]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    uint16_t x;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(a) : "memory");
    return x;
}
// d += a b.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Codes 0 .. 7 of a word, less 8, as the pairs (0, 4), (1, 5), (2, 6), (3, 7): under the exponent of 1024 a code in bits 0
// .. 3 is 1024 + code, one in bits 4 .. 7 is 1024 + 16 code.
__device__ __forceinline__ void codes(uint32_t w, uint32_t (&x)[4]) {
    const __half2 low = __float2half2_rn(-1032.0f), up = __float2half2_rn(0.0625f), high = __float2half2_rn(-72.0f);
    const uint32_t v = w >> 8;
    x[0] = bits(__hadd2(half2_of(field<0x000f000fu, 0x64006400u>(w)), low));
    x[1] = bits(__hfma2(half2_of(field<0x00f000f0u, 0x64006400u>(w)), up, high));
    x[2] = bits(__hadd2(half2_of(field<0x000f000fu, 0x64006400u>(v)), low));
    x[3] = bits(__hfma2(half2_of(field<0x00f000f0u, 0x64006400u>(v)), up, high));
}
// Two F16 values, x in the low half, and what their rounding left over.
__device__ __forceinline__ uint32_t pack_split(float x, float y, uint32_t& rest) {
    const __half2 h = __floats2half2_rn(x, y);
    rest = bits(__floats2half2_rn(x - __low2float(h), y - __high2float(h)));
    return bits(h);
}
// [keys][rows] 8 x 8 block of 16-bit values, as a product leaves it, to [rows][keys], as the next one reads it.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// A stage holds KT keys: codes and scales of K, then of V, as they lie in the block.
template <int D, int NT>
struct Cfg {
    using B = Q4Block<D>;
    static constexpr int KT = key_tile(D);
    static constexpr int STAGES = 3;
    static constexpr int ROWS = 8 * NT;
    static constexpr int TILE = KT * (B::ROW + B::SCALES);   // bytes of K (or V)
    static constexpr int QB = 2 * D;                         // bytes of a query row
    static constexpr int OSTR = D + 4;     // row stride of the outputs to be joined: lanes on different banks
    static constexpr size_t RING = (size_t)NW * STAGES * 2 * TILE;
    static constexpr size_t JOIN = (size_t)NW * ROWS * OSTR * 4;   // reuses the ring
    static constexpr size_t OFF_Q = RING > JOIN ? RING : JOIN;
    static constexpr size_t OFF_ML = OFF_Q + (size_t)ROWS * QB;
    static constexpr size_t SMEM = OFF_ML + (size_t)NW * ROWS * 8 + 16;
};
// Queries lie as the products read them: piece 4 G + t of a row, 16 bytes, has the elements 32 G + 8 t + {0, 4, 1, 5, 2, 6,
// 3, 7} (the pairs of codes()); the pieces of odd rows change places, so that two rows fall into different banks.
template <int D>
__device__ __forceinline__ uint32_t query_at(int row, int piece) {
    return (uint32_t)(row * 2 * D + ((piece ^ (D >= 64 ? (row & 1) << 2 : 0)) << 4));
}
// Element j (0 .. D / 8 - 1) of those that lane group g has of every value row.
template <int D>
__device__ __forceinline__ int dim_of(int g, int j) {
    if (D == 128) return 32 * ((2 * g + j / 8) & 3) + 8 * (g >> 1) + j % 8;   // words at places 2 g, 2 g + 1
    if (D == 64) return 32 * (g & 1) + 8 * (g >> 1) + j;                      // the word at place g
    return 4 * g + j;                                                        // half of the word at place g / 2
}

struct SplitArgs {
    ChunkAttnParams p;
    int group, tiles, n_split, split_tiles;
    float c;          // scale * log2(e)
    bool vec_q, vec_out;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(NW * 32) k_chunk_attn_q4(SplitArgs a) {
    using C = Cfg<D, NT>;
    using B = Q4Block<D>;
    constexpr int KT = C::KT, ROWS = C::ROWS, ST = C::STAGES, G = D / 32;
    extern __shared__ __align__(128) uint8_t sm[];
    const ChunkAttnParams& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int id = blockIdx.x;
    const int sp = id % a.n_split;
    id /= a.n_split;
    const int h = id % p.kv.n_head;
    id /= p.kv.n_head;
    const int tile = id % a.tiles, s = id / a.tiles;
    griddep_wait();
    griddep_launch();

    // Without a window this warp's tiles are known before the sequence's length: the first page numbers are fetched
    // beside it (entries past the sequence are not used).
    const int32_t* tab = p.batch.table + (int64_t)s * p.batch.max_pages;
    const int v0 = sp * a.split_tiles;
    int pages = 0;
    if (!p.window) pages = tab[min((v0 + warp + lane * NW) / (PAGE / KT), p.batch.max_pages - 1)];
    ChunkRange c;
    if (!chunk_range(p, s, tile, a.group, ROWS, KT, tid == 0 && sp == 0 && h == 0 && tile == 0, c)) return;
    const int row0 = c.row0, n = c.n, total = c.total, len = c.len, r0 = c.r0, rows = c.rows, p0 = c.p0, p1 = c.p1, np = c.np;
    const int n_tiles = c.n_tiles;
    const int n_act = max(1, (n_tiles + a.split_tiles - 1) / a.split_tiles);
    if (sp >= n_act) return;
    const int v1 = min(n_tiles, v0 + a.split_tiles);
    const int mine = v0 + warp < v1 ? (v1 - v0 - warp + NW - 1) / NW : 0;
    auto key0 = [&](int i) { return c.tile_of(v0 + warp + i * NW) * KT; };

    // ring: the page numbers of 32 tiles ahead sit in the warp's lanes
    const uint32_t ring = smem_addr(sm) + (uint32_t)(warp * ST * 2 * C::TILE);
    bool bad = false;
    auto fetch = [&](int i) {
        if (i < mine) {
            if ((i & 31) == 0 && (i || p.window)) pages = i + lane < mine ? tab[key0(i + lane) / PAGE] : 0;
            const int k0 = key0(i);
            const int page = __shfl_sync(0xffffffffu, pages, i & 31);
            const bool held = page >= 0 && page < p.kv.n_page;
            bad |= !held;
            const uint8_t* kp = (const uint8_t*)p.kv.pool;
            if (held)
                kp += (((int64_t)page * p.kv.n_layer + p.kv.layer) * 2 * p.kv.n_head + h) * B::BYTES + (k0 % PAGE) * B::ROW;
            const int64_t to_v = held ? (int64_t)p.kv.n_head * B::BYTES : 0;
            const uint32_t dst = ring + (uint32_t)((i % ST) * 2 * C::TILE);
            const int keys = held ? len - k0 : 0;
#pragma unroll
            for (int j = 0; j < KT * B::ROW / 512; j++) {
                const int x = (j * 32 + lane) * 16, in = x / B::ROW < keys ? 16 : 0;
                cp16(dst + x, kp + x, in);
                cp16(dst + C::TILE + x, kp + to_v + x, in);
            }
            // scales: K by the lower lanes, V by the upper ones; zero past the last key, so that values there are 0
            static_assert(KT * B::SCALES <= 256, "a piece per lane");
            const int x = (lane & 15) * 16;
            if (x < KT * B::SCALES)
                cp16(dst + (lane >> 4) * C::TILE + KT * B::ROW + x,
                     kp + (held ? (lane >> 4) * to_v + B::OFF_SCALES - (k0 % PAGE) * (B::ROW - B::SCALES) + x : 0),
                     max(0, min(16, keys * B::SCALES - x)));
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) fetch(i);
    // queries into shared memory, zero past the tile's rows (after the first copies are under way)
    uint8_t* sq = sm + C::OFF_Q;
    for (int i = tid; i < ROWS * (D / 8); i += NW * 32) {
        const int r = i / (D / 8), pc = i % (D / 8);
        __half x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = __float2half_rn(0.0f);
        if (r < rows) {
            const int tok = (r0 + r) / a.group, j = (r0 + r) % a.group;
            const T* src = (const T*)p.q + (int64_t)(row0 + tok) * p.q_stride + (int64_t)(h * a.group + j) * D + pc * 8;
            uint4 u;
            if (a.vec_q) {
                u = *(const uint4*)src;
            } else {
                T* y = (T*)&u;
#pragma unroll
                for (int k = 0; k < 8; k++) y[k] = src[k];
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if constexpr (__is_same(T, __half)) x[k] = ((const T*)&u)[k];
                else x[k] = __float2half_rn(__bfloat162float(((const T*)&u)[k]));
            }
        }
        auto two = [&](int k) { return bits(__halves2half2(x[k], x[k + 4])); };
        *(uint4*)(sq + query_at<D>(r, pc)) = make_uint4(two(0), two(1), two(2), two(3));
    }
    __syncthreads();   // queries

    // this lane's rows: 2 of every 8 (fragment columns 2 (lane % 4) and the next)
    const int t4 = lane & 3, col = t4 * 2, kr = lane >> 2;   // kr: the lane's key (or dims) in a fragment
    int see_lo[NT][2], see_hi[NT][2];
#pragma unroll
    for (int b = 0; b < NT; b++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int pos = total - n + (r0 + min(rows - 1, b * 8 + col + e)) / a.group;
            see_hi[b][e] = min(len, pos + 1);
            see_lo[b][e] = p.window ? pos - p.window + 1 : 0;
        }
    float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
    for (int b = 0; b < NT; b++) {
        m[b][0] = m[b][1] = NEG_INF;
        l[b][0] = l[b][1] = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) o[b][d][0] = o[b][d][1] = o[b][d][2] = o[b][d][3] = 0.0f;
    }
    const uint32_t sqa = smem_addr(sq);
    // query fragments: in registers where they are few, else read again for every tile
    constexpr bool QREG = NT * D <= 256;
    uint32_t qr[QREG ? NT : 1][QREG ? G : 1][4];
    if constexpr (QREG) {
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int g = 0; g < G; g++) lds<4>(sqa + query_at<D>(b * 8 + kr, g * 4 + t4), qr[b][g]);
    }

    for (int i = 0; i < mine; i++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
        __syncwarp();
        const uint32_t kt = ring + (uint32_t)((i % ST) * 2 * C::TILE), vt = kt + C::TILE;
        const uint32_t ks = kt + KT * B::ROW, vs = vt + KT * B::ROW;
        float sc[NT][KT / 16][4];   // [key kr, + 8][row col, + 1]
#pragma unroll
        for (int j = 0; j < KT / 16; j++) {
            uint32_t w[2][G];
            float d[2][G];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int key = j * 16 + kr + 8 * e;
                lds<G>(kt + key * B::ROW + t4 * (4 * G), w[e]);
                if constexpr (G == 1) {
                    d[e][0] = __half2float(__ushort_as_half((unsigned short)lds16(ks + key * 2)));
                } else {
                    uint32_t x[G / 2];
                    lds<G / 2>(ks + key * B::SCALES, x);
#pragma unroll
                    for (int g = 0; g < G; g += 2) {
                        d[e][g] = __low2float(half2_of(x[g / 2]));
                        d[e][g + 1] = __high2float(half2_of(x[g / 2]));
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NT; b++) sc[b][j][0] = sc[b][j][1] = sc[b][j][2] = sc[b][j][3] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t x[4], y[4];
                codes(w[0][g], x);
                codes(w[1][g], y);
                const uint32_t f0[4] = {x[0], y[0], x[1], y[1]}, f1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
                for (int b = 0; b < NT; b++) {
                    uint32_t q[4];
                    if constexpr (QREG) {
#pragma unroll
                        for (int k = 0; k < 4; k++) q[k] = qr[b][g][k];
                    } else {
                        lds<4>(sqa + query_at<D>(b * 8 + kr, g * 4 + t4), q);
                    }
                    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma(z, f0, q[0], q[1]);
                    mma(z, f1, q[2], q[3]);
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[b][j][e] = fmaf(z[e], d[e >> 1][g], sc[b][j][e]);
                }
            }
        }
        // scores in log2 units; keys that a row must not see to -infinity
        const int k0 = key0(i);
        const bool whole = k0 + KT <= np || (k0 + KT <= min(len, p0 + 1) && (!p.window || k0 > p1 - p.window));
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int j = 0; j < KT / 16; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[b][j][e] *= a.c;
        if (!whole) {
#pragma unroll
            for (int b = 0; b < NT; b++)
#pragma unroll
                for (int j = 0; j < KT / 16; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = k0 + j * 16 + kr + 8 * (e >> 1);
                        if (!(key < np || (key < see_hi[b][e & 1] && key >= see_lo[b][e & 1]))) sc[b][j][e] = NEG_INF;
                    }
            asm volatile("" ::: "memory");   // keeps the tests out of the tiles that need none
        }
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float top = fmaxf(sc[b][0][e], sc[b][0][e + 2]);
#pragma unroll
                for (int j = 1; j < KT / 16; j++) top = fmaxf(top, fmaxf(sc[b][j][e], sc[b][j][e + 2]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                if (top > m[b][e]) {
                    const float f = ex2(m[b][e] - top);
                    l[b][e] *= f;
#pragma unroll
                    for (int d = 0; d < D / 16; d++) {
                        o[b][d][e] *= f;
                        o[b][d][e + 2] *= f;
                    }
                    m[b][e] = top;
                }
                const float ref = m[b][e] == NEG_INF ? 0.0f : m[b][e] - BIAS;
#pragma unroll
                for (int j = 0; j < KT / 16; j++)
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const float w = ex2(sc[b][j][e + 2 * g] - ref);
                        sc[b][j][e + 2 * g] = w;
                        l[b][e] += w;
                    }
            }
#pragma unroll
        for (int j = 0; j < KT / 16; j++) {
            uint32_t wh[NT][2], wl[NT][2];
#pragma unroll
            for (int b = 0; b < NT; b++)
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    uint32_t rest;
                    wh[b][g] = transpose8(pack_split(sc[b][j][2 * g], sc[b][j][2 * g + 1], rest));
                    wl[b][g] = transpose8(rest);
                }
            // values of the lane's D / 8 dims: [key pair: col, col + 8][dim] halves (key, key + 1)
            uint32_t v[2][D / 8];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int key = j * 16 + col + 8 * e;
                if constexpr (D == 128) {
                    uint32_t x[2], y[2], dx[1], dy[1];
                    lds<2>(vt + key * B::ROW + kr * 8, x);
                    lds<2>(vt + (key + 1) * B::ROW + kr * 8, y);
                    lds<1>(vs + key * B::SCALES + (kr & 1) * 4, dx);
                    lds<1>(vs + (key + 1) * B::SCALES + (kr & 1) * 4, dy);
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const __half2 dd = half2_of(__byte_perm(dx[0], dy[0], g ? 0x7632 : 0x5410));
                        const __half2 off = __hmul2(dd, __float2half2_rn(-24.0f));
                        uint32_t lo[4], hi[4];
                        q4_values(__byte_perm(x[g], y[g], 0x5410), dd, off, lo);
                        q4_values(__byte_perm(x[g], y[g], 0x7632), dd, off, hi);
#pragma unroll
                        for (int k = 0; k < 4; k++) { v[e][g * 8 + k] = lo[k]; v[e][g * 8 + 4 + k] = hi[k]; }
                    }
                } else if constexpr (D == 64) {
                    uint32_t x[1], y[1];
                    lds<1>(vt + key * B::ROW + kr * 4, x);
                    lds<1>(vt + (key + 1) * B::ROW + kr * 4, y);
                    const uint32_t dx = lds16(vs + key * B::SCALES + (kr & 1) * 2);
                    const uint32_t dy = lds16(vs + (key + 1) * B::SCALES + (kr & 1) * 2);
                    const __half2 dd = half2_of(dx | dy << 16), off = __hmul2(dd, __float2half2_rn(-24.0f));
                    uint32_t lo[4], hi[4];
                    q4_values(__byte_perm(x[0], y[0], 0x5410), dd, off, lo);
                    q4_values(__byte_perm(x[0], y[0], 0x7632), dd, off, hi);
#pragma unroll
                    for (int k = 0; k < 4; k++) { v[e][k] = lo[k]; v[e][4 + k] = hi[k]; }
                } else {
                    const uint32_t x = lds16(vt + key * B::ROW + kr * 2), y = lds16(vt + (key + 1) * B::ROW + kr * 2);
                    uint32_t dx[1], lo[4];
                    lds<1>(vs + key * B::SCALES, dx);   // (key is even)
                    const __half2 dd = half2_of(dx[0]), off = __hmul2(dd, __float2half2_rn(-24.0f));
                    q4_values(x | y << 16, dd, off, lo);
#pragma unroll
                    for (int k = 0; k < 4; k++) v[e][k] = lo[k];
                }
            }
#pragma unroll
            for (int d = 0; d < D / 16; d++) {
                const uint32_t va[4] = {v[0][2 * d], v[0][2 * d + 1], v[1][2 * d], v[1][2 * d + 1]};
#pragma unroll
                for (int b = 0; b < NT; b++) {
                    mma(o[b][d], va, wl[b][0], wl[b][1]);
                    mma(o[b][d], va, wh[b][0], wh[b][1]);
                }
            }
        }
        __syncwarp();   // every lane is done with the stage that the next fetch overwrites
        fetch(i + ST - 1);
    }
    if (bad && lane == 0) atomicOr(p.err, PAGED_BAD_PAGE);
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // join the warps
    float* ml = (float*)(sm + C::OFF_ML);   // [NW][ROWS] {m, l}
    float* so = (float*)sm;                 // [NW][ROWS][OSTR]
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NT; b++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float x = l[b][e];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const int r = warp * ROWS + b * 8 + col + e;
            if (lane < 4) {
                ml[2 * r] = m[b][e] - BIAS;   // (what the weights refer to)
                ml[2 * r + 1] = x;
            }
#pragma unroll
            for (int d = 0; d < D / 16; d++) {
                so[r * C::OSTR + dim_of<D>(kr, 2 * d)] = o[b][d][e];
                so[r * C::OSTR + dim_of<D>(kr, 2 * d + 1)] = o[b][d][e + 2];
            }
        }
    __syncthreads();
    const int64_t unit = ((int64_t)s * a.tiles + tile) * p.kv.n_head + h;
    float* part_o = p.part + unit * a.n_split * (ROWS * (D + 2));   // [split][ROWS][D], then [split][ROWS] {m, l}
    float* part_ml = part_o + (int64_t)a.n_split * ROWS * D;
    for (int i = tid; i < rows * (D / 4); i += NW * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float top = NEG_INF;
#pragma unroll
        for (int w = 0; w < NW; w++) top = fmaxf(top, ml[2 * (w * ROWS + r)]);
        const float ref = top == NEG_INF ? 0.0f : top;
        float sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = ex2(ml[2 * (w * ROWS + r)] - ref);
            sum = fmaf(f, ml[2 * (w * ROWS + r) + 1], sum);
            const float4 v = *(const float4*)(so + (w * ROWS + r) * C::OSTR + d);
            x[0] = fmaf(f, v.x, x[0]); x[1] = fmaf(f, v.y, x[1]);
            x[2] = fmaf(f, v.z, x[2]); x[3] = fmaf(f, v.w, x[3]);
        }
        if (n_act == 1) {
            finish<T, D>(p, c, a.vec_out, a.group, h, r, d, top, sum, x);
        } else {
            *(float4*)(part_o + ((int64_t)sp * ROWS + r) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) *(float2*)(part_ml + 2 * ((int64_t)sp * ROWS + r)) = make_float2(top, sum);
        }
    }
    if (n_act == 1) return;

    if constexpr (ROWS == 8)   // (more rows are joined by k_chunk_join)
        join_splits<T, D, ROWS, NW * 32>(p, c, s, tile, h, a.group, a.tiles, a.n_split, n_act, a.vec_out, tid,
                                         (int*)(sm + C::OFF_ML + (size_t)NW * ROWS * 8), (float*)sm);
}

template <typename T, int D, typename F>
void pick_rows(int row_tile, F f) {
    if (row_tile == 8) f(k_chunk_attn_q4<T, D, 1>, Cfg<D, 1>::SMEM);
    else if (row_tile == 16) f(k_chunk_attn_q4<T, D, 2>, Cfg<D, 2>::SMEM);
    else if (row_tile == 24) f(k_chunk_attn_q4<T, D, 3>, Cfg<D, 3>::SMEM);
    else f(k_chunk_attn_q4<T, D, 4>, Cfg<D, 4>::SMEM);
}
template <typename T, typename F>
void pick_dim(int dim, int row_tile, F f) {
    if (dim == 32) pick_rows<T, 32>(row_tile, f);
    else if (dim == 64) pick_rows<T, 64>(row_tile, f);
    else pick_rows<T, 128>(row_tile, f);
}
template <typename F>
void pick(int dtype, int dim, int row_tile, F f) {
    if (dtype == GSVCU_KV_Q4_F16) pick_dim<__half>(dim, row_tile, f);
    else pick_dim<__nv_bfloat16>(dim, row_tile, f);
}

}  // namespace

ChunkAttnPlan chunk_attention_q4_plan(const ChunkAttnParams& p) {
    const int D = p.kv.head_dim, kt = key_tile(D);
    const int64_t packed = (int64_t)p.batch.max_chunk * (p.n_q_head / p.kv.n_head);
    ChunkAttnPlan c;
    if (packed > 32 && p.scale != 0.0f) {
        c = chunk_attention_tc_plan(p);
        // Many row tiles over the same keys: the keys are unpacked once, by a kernel before it.
        const int group = p.n_q_head / p.kv.n_head;
        const int64_t rows = p.window ? std::min(packed, (int64_t)p.window * group) : packed, pages = (p.batch.max_kv + PAGE - 1) / PAGE;
        const int64_t bytes = p.batch.n_seq * pages * (2 * p.kv.n_head * PAGE * D * 2 + 4);
        if (rows >= UNPACK_ROWS && bytes <= UNPACK_LIMIT) {
            c.unpack_pages = (int)pages;
            c.unpacked_floats = (size_t)(bytes / 4);
        }
        return c;
    }
    c.row_tile = packed >= 32 ? 32 : (int)(packed + 7) / 8 * 8;
    c.tiles = (int)((packed + c.row_tile - 1) / c.row_tile);
    const int64_t units = (int64_t)p.batch.n_seq * c.tiles * p.kv.n_head;
    const int max_tiles = (p.batch.max_kv + kt - 1) / kt;
    size_t smem = 0;
    pick(p.kv.kv_dtype, D, c.row_tile, [&](auto, size_t bytes) { smem = bytes; });
    const int64_t slots = 148 * (int64_t)(232448 / (smem + 1024));
    int64_t n = (slots + units / 2) / units;
    if (p.batch.n_seq > 1) {
        const int64_t even = (4 * slots + units - 1) / units, whole = ((int64_t)p.batch.max_kv * 9 * D / 8) >> 17;
        if (n < (even < whole ? even : whole)) n = even < whole ? even : whole;
    }
    const int least = 4 * NW;
    if (n > (max_tiles + least - 1) / least) n = (max_tiles + least - 1) / least;
    if (n < 1) n = 1;
    c.split_tiles = (int)((max_tiles + n - 1) / n);
    c.split_tiles = (c.split_tiles + NW - 1) / NW * NW;
    if (c.split_tiles < NW) c.split_tiles = NW;
    c.n_split = (max_tiles + c.split_tiles - 1) / c.split_tiles;
    if (c.n_split < 1) c.n_split = 1;
    c.key_tile = kt;
    if (c.n_split > 1) {
        c.join_apart = c.row_tile > 8;   // (as chunk_attention_plan)
        c.part_floats = (size_t)units * c.n_split * c.row_tile * (D + 2);
        c.arrivals = c.join_apart ? 0 : (size_t)units;
    }
    return c;
}

bool launch_chunk_attention_q4(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s) {
    SplitArgs a;
    a.p = p;
    a.group = p.n_q_head / p.kv.n_head;
    a.tiles = plan.tiles;
    a.n_split = plan.n_split;
    a.split_tiles = plan.split_tiles;
    a.c = p.scale * LOG2E;
    a.vec_q = ((uintptr_t)p.q & 15) == 0 && p.q_stride % 8 == 0;
    a.vec_out = ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0;
    const int64_t ctas = (int64_t)p.batch.n_seq * plan.tiles * p.kv.n_head * plan.n_split;
    const int bit = ((p.kv.kv_dtype == GSVCU_KV_Q4_F16 ? 0 : 3) + p.kv.head_dim / 64) * 4 + plan.row_tile / 8 - 1;   // 0 .. 23
    bool ok = false;
    pick(p.kv.kv_dtype, p.kv.head_dim, plan.row_tile, [&](auto k, size_t smem) {
        ok = raise_smem(k, smem, ready, bit);
        if (ok) launch_pdl(k, dim3((unsigned)ctas), dim3(NW * 32), smem, s, a);
    });
    return ok;
}

}  // namespace gsvcu
