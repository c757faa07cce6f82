// paged_attention.cu -- attention of a chunk of new tokens over the paged KV cache, split over the keys.
//
// A query row at position p (its chunk's rows are the last of the sequence's kv_len keys) sees key j when
//   j < prefix,  or  j <= p and (no window or j > p - window).
// out = sum_j w_j v_j / sum_j w_j with w_j = exp(scale q.k_j - m), lse = m + log(sum_j w_j); a row that sees
// nothing gives 0 and -infinity. The g query heads that share a kv head are rows of one tile (packed row
// r = token * g + head in the group), so K and V are read once for all of them.
//
// k_chunk_attn: one CTA per (sequence, row tile, kv head, key split). Its four warps take the split's key
// tiles in turn, each with its own cp.async ring, running maximum, sum and output (in registers), so no
// barrier stands inside the loop; they are joined at the end in warp order. With several splits the CTA that
// arrives last joins the splits' results of 8 rows, k_chunk_join those of more, in an order that the sizes alone decide
// (results do not depend on timing).
// Everything is transposed: S^T = K Q^T with 16 keys and 8 query rows per product, O^T = V^T P^T, because few
// rows are the rule here (one decoding token of one head is one row) and 8 is the smaller side of mma.sync.
// F16 / BF16 products run on mma.m16n8k16 with the weights split into two 16-bit parts (w = hi + lo), so
// rounding them costs nothing against the output's own rounding (F16 weights are kept 2^14 up, where hi and lo have 22 bits
// down to 2^-17 of the running maximum's and the last one at 2^-38); F32 ones on mma.m16n8k8.tf32 with both
// operands in two parts (three products), which leaves an error near 2^-22. Sums, maxima and outputs are f32.
// Keys past kv_len are never read (zero-filled), keys that a row must not see get weight 0.
// Decode is bound by HBM: every key is read once, 8 KB (16-bit heads of 32) or 16 KB in flight per warp (64 sequences of
// 600 to 2100 keys, 16 heads of 32: 34.5 us, 5.2 TB/s; one of 131072 keys, 32/8 heads of 128: 88 us, 6.1 TB/s). F32 chunks
// are bound by the tensor pipe and the splitting of operands (4 chunks of up to 333 rows, 16 heads of 32: 67 us). F32 single
// tokens: the 64 sequences 80 us, 4.5 TB/s; one of 131072 keys, 32/8 heads of 128, 465 us, 2.3 TB/s, because its 152 CTAs
// are four more than the one per SM that 130 KB of shared memory allow.
#include <cuda_bf16.h>

#include "kernels.h"
#include "paged.h"
#include "paged_join.cuh"

namespace gsvcu {
namespace {

constexpr int NW = 4;   // warps per CTA
template <typename T> constexpr float BIAS = __is_same(T, __half) ? 14.0f : 0.0f;   // weights are 2^BIAS exp(s - maximum)
// Keys of one warp's tile: 8 KB of K and V, 16 KB for wide F32 rows (a product takes 16 keys at least), 4 KB for
// F16 / BF16 heads of 32, where the CTAs are short and four of them fit an SM (64 slots: 36.9 us against 38.4).
__host__ __device__ constexpr int key_tile(int dim, int size) {
    return dim == 32 ? 32 : size == 2 ? 2048 / dim : 16;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ float lds(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// d += a b, the type's tensor-core product.
__device__ __forceinline__ void mma16(__half, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(__nv_bfloat16, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two 16-bit values of the type, x in the low half, and what their rounding left over.
__device__ __forceinline__ uint32_t pack_split(__half, float x, float y, uint32_t& rest) {
    const __half2 h = __floats2half2_rn(x, y);
    const __half2 r = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    rest = *(const uint32_t*)&r;
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack_split(__nv_bfloat16, float x, float y, uint32_t& rest) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - __low2float(h), y - __high2float(h));
    rest = *(const uint32_t*)&r;
    return *(const uint32_t*)&h;
}
// x = hi + lo to about 22 bits, both with the 10 fraction bits that the tensor core reads: hi rounded (half away
// from zero), lo the exact rest, cut. In integer steps because splitting bounds the F32 kernel: 67 us for a batch of
// ragged chunks, 91 with two rounding conversions. With hi cut too it is 65, but every lo then has x's sign and the
// dropped lo lo products add up (8.6e-7 of the result instead of 3.5e-7).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
// [keys][rows] 8 x 8 block of 16-bit values, as a product leaves it, to [rows][keys], as the next one reads it.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// The same for a pair of f32 values per lane: high and low halves apart.
__device__ __forceinline__ void transpose8(float& x, float& y) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    const uint32_t hi = transpose8(__byte_perm(a, b, 0x7632)), lo = transpose8(__byte_perm(a, b, 0x5410));
    x = __uint_as_float(__byte_perm(lo, hi, 0x5410));
    y = __uint_as_float(__byte_perm(lo, hi, 0x7632));
}

// Key tile of one warp's ring stage: KT keys of K, then of V, rows of RB bytes in 16-byte pieces; piece c of
// row r lies at c ^ swz(r), so the 8 rows of a matrix fragment fall into different banks.
template <typename T, int D, int NT>
struct Cfg {
    static constexpr int RB = D * (int)sizeof(T);
    static constexpr int PIECES = RB / 16;
    static constexpr int KT = key_tile(D, (int)sizeof(T));
    static constexpr int STAGES = RB > 256 ? 2 : 3;
    static constexpr int ROWS = 8 * NT;
    static constexpr int TILE = KT * RB;   // bytes of K (or V)
    static constexpr int QPLANES = sizeof(T) == 4 ? 2 : 1;   // F32: high and low parts
    static constexpr int OSTR = D + 4;     // row stride of the outputs to be joined: lanes on different banks
    static constexpr size_t RING = (size_t)NW * STAGES * 2 * TILE;
    static constexpr size_t JOIN = (size_t)NW * ROWS * OSTR * 4;   // reuses the ring
    static constexpr size_t OFF_Q = RING > JOIN ? RING : JOIN;
    static constexpr size_t OFF_ML = OFF_Q + (size_t)QPLANES * ROWS * RB;
    static constexpr size_t SMEM = OFF_ML + (size_t)NW * ROWS * 8 + 16;
};
template <int RB>
__device__ __forceinline__ uint32_t at(int row, int piece) {
    const int swz = RB == 64 ? (row >> 1) & 3 : row & 7;
    return (uint32_t)(row * RB + ((piece ^ swz) << 4));
}

struct SplitArgs {
    ChunkAttnParams p;
    int group, tiles, n_split, split_tiles;
    float c;          // scale * log2(e)
    bool vec_q, vec_out;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(NW * 32) k_chunk_attn(SplitArgs a) {
    using C = Cfg<T, D, NT>;
    constexpr int KT = C::KT, RB = C::RB, ROWS = C::ROWS, ST = C::STAGES;
    constexpr bool F32 = sizeof(T) == 4;
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
    const int64_t block = (int64_t)PAGE * D;   // elements of one (page, layer, K or V, head)
    bool bad = false;
    auto fetch = [&](int i) {
        if (i < mine) {
            if ((i & 31) == 0 && (i || p.window)) pages = i + lane < mine ? tab[key0(i + lane) / PAGE] : 0;
            const int k0 = key0(i);
            const int page = __shfl_sync(0xffffffffu, pages, i & 31);
            const bool held = page >= 0 && page < p.kv.n_page;
            bad |= !held;
            const T* kp = (const T*)p.kv.pool;
            if (held) kp += (((int64_t)page * p.kv.n_layer + p.kv.layer) * 2 * p.kv.n_head + h) * block + (k0 % PAGE) * D;
            const T* vp = held ? kp + p.kv.n_head * block : kp;
            const uint32_t dst = ring + (uint32_t)((i % ST) * 2 * C::TILE);
            const int keys = held ? len - k0 : 0;
#pragma unroll
            for (int j = 0; j < KT * C::PIECES / 32; j++) {
                const int x = j * 32 + lane, r = x / C::PIECES, pc = x % C::PIECES;
                const bool in = r < keys;
                cp16(dst + at<RB>(r, pc), in ? (const uint8_t*)kp + x * 16 : (const uint8_t*)p.kv.pool, in);
                cp16(dst + C::TILE + at<RB>(r, pc), in ? (const uint8_t*)vp + x * 16 : (const uint8_t*)p.kv.pool, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) fetch(i);
    // queries into shared memory, zero past the tile's rows (after the first copies are under way)
    uint8_t* sq = sm + C::OFF_Q;
    for (int i = tid; i < ROWS * C::PIECES; i += NW * 32) {
        const int r = i / C::PIECES, pc = i % C::PIECES;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const int tok = (r0 + r) / a.group, j = (r0 + r) % a.group;
            const T* src = (const T*)p.q + (int64_t)(row0 + tok) * p.q_stride + (int64_t)(h * a.group + j) * D +
                           pc * (16 / (int)sizeof(T));
            if (a.vec_q) {
                u = *(const uint4*)src;
            } else {
                T* x = (T*)&u;
#pragma unroll
                for (int k = 0; k < 16 / (int)sizeof(T); k++) x[k] = src[k];
            }
        }
        if constexpr (F32) {
            uint4 w;
            uint32_t* x = (uint32_t*)&u;
            uint32_t* y = (uint32_t*)&w;
#pragma unroll
            for (int k = 0; k < 4; k++) split_tf32(__uint_as_float(x[k]), x[k], y[k]);
            *(uint4*)(sq + ROWS * RB + at<RB>(r, pc)) = w;
        }
        *(uint4*)(sq + at<RB>(r, pc)) = u;
    }

    __syncthreads();   // queries

    // this lane's rows: 2 of every 8 (fragment columns 2 (lane % 4) and the next)
    const int col = (lane & 3) * 2, kr = lane >> 2;   // kr: the lane's key (or dim) in a fragment, and + 8
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
    // F16 / BF16 query fragments: in registers where they are few, else read again for every tile
    constexpr bool QREG = !F32 && NT * D <= 256;
    uint32_t qr[QREG ? NT : 1][QREG ? D / 16 : 1][2];
    auto query = [&](int b, int kk, uint32_t (&q)[4]) {   // dims 16 kk .. 16 kk + 31 of rows 8 b .. 8 b + 7
        ldsm4(sqa + at<RB>(b * 8 + (lane & 7), kk * 2 + (lane >> 3)), q);
    };
    if constexpr (QREG) {
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int kk = 0; kk < D / 16; kk += 2) {
                uint32_t q[4];
                query(b, kk, q);
                qr[b][kk][0] = q[0]; qr[b][kk][1] = q[1];
                qr[b][kk + 1][0] = q[2]; qr[b][kk + 1][1] = q[3];
            }
    }

    for (int i = 0; i < mine; i++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
        __syncwarp();
        const uint32_t kt = ring + (uint32_t)((i % ST) * 2 * C::TILE), vt = kt + C::TILE;
        float sc[NT][KT / 16][4];   // [key kr, + 8][row col, + 1]
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int j = 0; j < KT / 16; j++) sc[b][j][0] = sc[b][j][1] = sc[b][j][2] = sc[b][j][3] = 0.0f;
        if constexpr (!F32) {
#pragma unroll
            for (int kk = 0; kk < D / 16; kk += 2) {
                uint32_t qa[NT][4];
#pragma unroll
                for (int b = 0; b < NT; b++) {
                    if constexpr (QREG) {
                        qa[b][0] = qr[b][kk][0]; qa[b][1] = qr[b][kk][1];
                        qa[b][2] = qr[b][kk + 1][0]; qa[b][3] = qr[b][kk + 1][1];
                    } else {
                        query(b, kk, qa[b]);
                    }
                }
#pragma unroll
                for (int j = 0; j < KT / 16; j++)
#pragma unroll
                    for (int k2 = 0; k2 < 2; k2++) {
                        uint32_t ka[4];
                        ldsm4(kt + at<RB>(j * 16 + (lane & 15), (kk + k2) * 2 + (lane >> 4)), ka);
#pragma unroll
                        for (int b = 0; b < NT; b++) mma16(T(), sc[b][j], ka, qa[b][2 * k2], qa[b][2 * k2 + 1]);
                    }
            }
        } else {
            const uint32_t w4 = (lane & 3) * 4;
            float low[NT][KT / 16][4];   // the two products with a low part, added at the end
#pragma unroll
            for (int b = 0; b < NT; b++)
#pragma unroll
                for (int j = 0; j < KT / 16; j++) low[b][j][0] = low[b][j][1] = low[b][j][2] = low[b][j][3] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < D / 8; kk++) {
                uint32_t qh[NT][2], ql[NT][2];
#pragma unroll
                for (int b = 0; b < NT; b++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t x = at<RB>(b * 8 + kr, kk * 2 + e) + w4;
                        qh[b][e] = __float_as_uint(lds(sqa + x));
                        ql[b][e] = __float_as_uint(lds(sqa + ROWS * RB + x));
                    }
#pragma unroll
                for (int j = 0; j < KT / 16; j++) {
                    uint32_t kh[4], kl[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        split_tf32(lds(kt + at<RB>(j * 16 + kr + 8 * (e & 1), kk * 2 + (e >> 1)) + w4), kh[e], kl[e]);
#pragma unroll
                    for (int b = 0; b < NT; b++) {
                        mma8(low[b][j], kl, qh[b][0], qh[b][1]);
                        mma8(low[b][j], kh, ql[b][0], ql[b][1]);
                        mma8(sc[b][j], kh, qh[b][0], qh[b][1]);
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NT; b++)
#pragma unroll
                for (int j = 0; j < KT / 16; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[b][j][e] += low[b][j][e];
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
                const float ref = m[b][e] == NEG_INF ? 0.0f : m[b][e] - BIAS<T>;
#pragma unroll
                for (int j = 0; j < KT / 16; j++)
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const float w = ex2(sc[b][j][e + 2 * g] - ref);
                        sc[b][j][e + 2 * g] = w;
                        l[b][e] += w;
                    }
            }
        if constexpr (!F32) {
#pragma unroll
            for (int j = 0; j < KT / 16; j++) {
                uint32_t wh[NT][2], wl[NT][2];
#pragma unroll
                for (int b = 0; b < NT; b++)
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        uint32_t rest;
                        wh[b][g] = transpose8(pack_split(T(), sc[b][j][2 * g], sc[b][j][2 * g + 1], rest));
                        wl[b][g] = transpose8(rest);
                    }
#pragma unroll
                for (int d = 0; d < D / 16; d++) {
                    uint32_t va[4];
                    ldsm4t(vt + at<RB>(j * 16 + (lane & 7) + ((lane >> 4) << 3), d * 2 + ((lane >> 3) & 1)), va);
#pragma unroll
                    for (int b = 0; b < NT; b++) {
                        mma16(T(), o[b][d], va, wl[b][0], wl[b][1]);
                        mma16(T(), o[b][d], va, wh[b][0], wh[b][1]);
                    }
                }
            }
        } else {
            // the fragment's k index is a key: index lane % 4 takes key 2 (lane % 4), lane % 4 + 4 the next one, as the
            // transposed weights lie. A tile's products are summed by themselves and then added to o (the tensor
            // core's additions truncate: over a long cache that would drift, rounded ones do not).
            uint32_t wh[NT][KT / 8][2], wl[NT][KT / 8][2];
#pragma unroll
            for (int b = 0; b < NT; b++)
#pragma unroll
                for (int j = 0; j < KT / 8; j++) {
                    float x = sc[b][j / 2][2 * (j & 1)], y = sc[b][j / 2][2 * (j & 1) + 1];
                    transpose8(x, y);
                    split_tf32(x, wh[b][j][0], wl[b][j][0]);
                    split_tf32(y, wh[b][j][1], wl[b][j][1]);
                }
#pragma unroll
            for (int d = 0; d < D / 16; d++) {
                float x[NT][4];
#pragma unroll
                for (int b = 0; b < NT; b++) x[b][0] = x[b][1] = x[b][2] = x[b][3] = 0.0f;
#pragma unroll
                for (int j = 0; j < KT / 8; j++) {
                    uint32_t vh[4], vl[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int dim = d * 16 + kr + 8 * (e & 1);
                        split_tf32(lds(vt + at<RB>(j * 8 + col + (e >> 1), dim / 4) + (dim & 3) * 4), vh[e], vl[e]);
                    }
#pragma unroll
                    for (int b = 0; b < NT; b++) {
                        mma8(x[b], vl, wh[b][j][0], wh[b][j][1]);
                        mma8(x[b], vh, wl[b][j][0], wl[b][j][1]);
                        mma8(x[b], vh, wh[b][j][0], wh[b][j][1]);
                    }
                }
#pragma unroll
                for (int b = 0; b < NT; b++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[b][d][e] += x[b][e];
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
                ml[2 * r] = m[b][e] - BIAS<T>;   // (what the weights refer to)
                ml[2 * r + 1] = x;
            }
#pragma unroll
            for (int d = 0; d < D / 16; d++) {
                so[r * C::OSTR + d * 16 + kr] = o[b][d][e];
                so[r * C::OSTR + d * 16 + kr + 8] = o[b][d][e + 2];
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

// Calls f with the kernel's compile-time variant for (type, head dim, row tile).
template <typename T, int D, typename F>
void pick_rows(int row_tile, F f) {
    if (row_tile == 8) f(k_chunk_attn<T, D, 1>, Cfg<T, D, 1>::SMEM);
    else if (row_tile == 16) f(k_chunk_attn<T, D, 2>, Cfg<T, D, 2>::SMEM);
    else if (row_tile == 24) f(k_chunk_attn<T, D, 3>, Cfg<T, D, 3>::SMEM);
    else f(k_chunk_attn<T, D, 4>, Cfg<T, D, 4>::SMEM);
}
template <typename T, typename F>
void pick_dim(int dim, int row_tile, F f) {
    if (dim == 32) pick_rows<T, 32>(row_tile, f);
    else if (dim == 64) pick_rows<T, 64>(row_tile, f);
    else pick_rows<T, 128>(row_tile, f);
}
template <typename F>
void pick(int dtype, int dim, int row_tile, F f) {
    if (dtype == GSVCU_KV_F32) pick_dim<float>(dim, row_tile, f);
    else if (dtype == GSVCU_KV_F16) pick_dim<__half>(dim, row_tile, f);
    else pick_dim<__nv_bfloat16>(dim, row_tile, f);
}

}  // namespace

ChunkAttnPlan chunk_attention_plan(const ChunkAttnParams& p) {
    const int D = p.kv.head_dim, size = p.kv.kv_dtype == GSVCU_KV_F32 ? 4 : 2;
    const int kt = key_tile(D, size);
    const int64_t packed = (int64_t)p.batch.max_chunk * (p.n_q_head / p.kv.n_head);
    ChunkAttnPlan c;
    if (size == 2 && packed > 32 && p.scale != 0.0f) {
        // Many rows of 16-bit types: the tcgen05 kernel (a zero scale would multiply masked -infinities by 0 there).
        // Row tiles per CTA and key splits by the shortest estimate, in units of 100 cycles: a key tile of 128 takes 29 for
        // two row tiles and 20 for one, splitting and joining 150, CTAs run in waves of one per SM. Measured: 4 chunks
        // of up to 570 rows over 1200 keys, 4 heads of 64: 16.4 us with one row tile, 23.9 with two in two splits; 512
        // tokens over 8192 keys (16/4 x 128): 54 us with one row tile in two splits, 48 with two in four.
        c.tensor = true;
        const int max_tiles = (p.batch.max_kv + 127) / 128;
        int64_t best = INT64_MAX;
        int n = 1;
        for (int rows = 256; rows >= 128; rows /= 2) {
            if (rows == 128 && packed <= 128) break;   // (one row tile already)
            const int64_t tiles = (packed + rows - 1) / rows, units = p.batch.n_seq * tiles * p.kv.n_head;
            const int64_t fit = 148 / units < max_tiles ? 148 / units : max_tiles;
            for (int64_t m : {(int64_t)1, fit}) {
                if (m < 1) continue;
                const int64_t waves = (units * m + 147) / 148, per = (max_tiles + m - 1) / m;
                const int64_t cost = waves * per * (rows == 256 && packed > 128 ? 29 : 20) + (m > 1 ? 150 : 0);
                if (cost < best) {
                    best = cost;
                    n = (int)m;
                    c.row_tile = rows;
                    c.tiles = (int)tiles;
                }
            }
        }
        const int64_t units = (int64_t)p.batch.n_seq * c.tiles * p.kv.n_head;
        c.split_tiles = (max_tiles + n - 1) / n;
        c.n_split = (max_tiles + c.split_tiles - 1) / c.split_tiles;
        c.key_tile = 128;
        c.join_apart = c.n_split > 1;
        if (c.n_split > 1) c.part_floats = (size_t)units * c.n_split * c.row_tile * (D + 2);
        return c;
    }
    c.row_tile = packed >= 32 ? 32 : (int)(packed + 7) / 8 * 8;
    if (size == 4 && D > 32 && packed > 32) {
        // F32 heads of 64 and 128: 32 rows leave no registers to overlap anything (2 chunks of 1500 rows over 3000 keys,
        // 16/4 heads of 64: 896 us, 656 with 24 rows, 706 with 16); 16 rows, a quarter less time per CTA, where that
        // saves a wave (512 rows over 2048 keys: 140 us with 24, 114 with 16). Two CTAs per SM.
        auto waves = [&](int rows) { return (p.batch.n_seq * ((packed + rows - 1) / rows) * p.kv.n_head + 295) / 296; };
        c.row_tile = 4 * waves(24) > 3 * waves(16) ? 16 : 24;
    }
    c.tiles = (int)((packed + c.row_tile - 1) / c.row_tile);
    const int64_t units = (int64_t)p.batch.n_seq * c.tiles * p.kv.n_head;
    const int max_tiles = (p.batch.max_kv + kt - 1) / kt;
    // Splits, measured on 148 SMs. Few units: about one wave of CTAs (one sequence of 131072 keys: 88 us, 100 with two
    // waves; the nearest count of splits, which can be a few CTAs more than fit at once). Several sequences: up to four waves, so that lengths even out (32 sequences of 1000 to 9000 keys: 134 us
    // with two splits, 117 with four), while a split still streams 512 KB (64 sequences of 2100 keys at head dim 32: 36 us
    // whole, 40 in two). A split keeps 4 tiles for each warp.
    size_t smem = 0;
    pick(p.kv.kv_dtype, D, c.row_tile, [&](auto, size_t bytes) { smem = bytes; });
    const int64_t slots = 148 * (int64_t)(232448 / (smem + 1024));
    int64_t n = (slots + units / 2) / units;
    if (p.batch.n_seq > 1) {
        const int64_t even = (4 * slots + units - 1) / units, whole = ((int64_t)p.batch.max_kv * 2 * D * size) >> 19;
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
        // Joined by the last CTA while a unit has 8 rows (one sequence of 131072 keys: 89 us, 101 with a second kernel),
        // by a kernel over the whole GPU when it has more (drafts of 5: 18.3 us, 19.5).
        c.join_apart = c.row_tile > 8;
        c.part_floats = (size_t)units * c.n_split * c.row_tile * (D + 2);
        c.arrivals = c.join_apart ? 0 : (size_t)units;
    }
    return c;
}

template <typename T, int D>
static void launch_join_rows(const ChunkAttnParams& p, const ChunkAttnPlan& c, bool vec, cudaStream_t s) {
    const int group = p.n_q_head / p.kv.n_head, rows = 1024 / D;
    const int64_t ctas = (int64_t)p.batch.n_seq * c.tiles * p.kv.n_head * ((c.row_tile + rows - 1) / rows);
    auto go = [&](auto k) {
        launch_pdl(k, dim3((unsigned)ctas), dim3(256), 0, s, p, group, c.tiles, c.n_split, c.split_tiles, c.key_tile, vec);
    };
    if (c.row_tile == 16) go(k_chunk_join<T, D, 16>);
    else if (c.row_tile == 24) go(k_chunk_join<T, D, 24>);
    else if (c.row_tile == 32) go(k_chunk_join<T, D, 32>);
    else if constexpr (sizeof(T) == 2) {
        if (c.row_tile == 128) go(k_chunk_join<T, D, 128>);
        else go(k_chunk_join<T, D, 256>);
    }
}
template <typename T>
static void launch_join(const ChunkAttnParams& p, const ChunkAttnPlan& c, bool vec, cudaStream_t s) {
    if (p.kv.head_dim == 32) launch_join_rows<T, 32>(p, c, vec, s);
    else if (p.kv.head_dim == 64) launch_join_rows<T, 64>(p, c, vec, s);
    else launch_join_rows<T, 128>(p, c, vec, s);
}

int launch_chunk_attention(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s) {
    const size_t size = p.kv.kv_dtype == GSVCU_KV_F32 ? 4 : 2;
    const bool vec_out = ((uintptr_t)p.out & 15) == 0 && (p.out_stride * (int64_t)size) % 16 == 0;
    if (plan.tensor) {
        if (!launch_chunk_attention_tc(p, plan, ready, s)) return 0;
    } else {
        SplitArgs a;
        a.p = p;
        a.group = p.n_q_head / p.kv.n_head;
        a.tiles = plan.tiles;
        a.n_split = plan.n_split;
        a.split_tiles = plan.split_tiles;
        a.c = p.scale * LOG2E;
        a.vec_q = ((uintptr_t)p.q & 15) == 0 && (p.q_stride * (int64_t)size) % 16 == 0;
        a.vec_out = vec_out;
        const int64_t ctas = (int64_t)p.batch.n_seq * plan.tiles * p.kv.n_head * plan.n_split;
        const int bit = (p.kv.kv_dtype * 3 + p.kv.head_dim / 64) * 4 + plan.row_tile / 8 - 1;   // 0 .. 35
        bool ok = false;
        pick(p.kv.kv_dtype, p.kv.head_dim, plan.row_tile, [&](auto k, size_t smem) {
            ok = raise_smem(k, smem, ready, bit);
            if (ok) launch_pdl(k, dim3((unsigned)ctas), dim3(NW * 32), smem, s, a);
        });
        if (!ok) return 0;
    }
    if (!plan.join_apart) return 1;
    if (p.kv.kv_dtype == GSVCU_KV_F32) launch_join<float>(p, plan, vec_out, s);
    else if (p.kv.kv_dtype == GSVCU_KV_F16) launch_join<__half>(p, plan, vec_out, s);
    else launch_join<__nv_bfloat16>(p, plan, vec_out, s);
    return 2;
}

}  // namespace gsvcu
