// paged_attention_q4.cu -- attention of few new rows over a 4-bit paged cache (layout and scales: paged_q4.cuh; the
// operator's formula and the float caches: paged_attention.cu).
//
// k_chunk_attn_q4: the four warps of a CTA take pages of 64 keys in turn, each with its own copies, running maximum, sum and
// output; transposed products (16 keys x 8 query rows), warps joined in order, what several CTAs share by the last of them or
// by k_join_q4, in an order that the sizes alone decide. All products are F16 mma.m16n8k16, whatever the rows' type (BF16
// queries fit F16 up to 65,504; beyond they count as overflowing; small rows enter scaled by a power of two):
//   scores   the codes less 8 are exact in F16, and a group of 32 elements is two products, so a group's sum is multiplied
//            by its key's scale in f32 afterwards;
//   values   scale * (code - 8) is exact in F16 too (scales have 8 significant bits) and takes one fused multiply-add per
//            pair: a code moved to bits 6 .. 9 under the exponent of 16 is the number 16 + code, times the scale less 24
//            scales.
// The weights are kept 2^14 up as in k_chunk_attn, for F16 rows in two parts, for BF16 ones in one.
//
// What bounds it: unpacking, about 1.5 instructions a value, most of them on the half-rate ALU (shifts, masks, byte permutes)
// and FP16 pipes; the copies keep up with one block of K and of V per warp. 131072 keys, 32/8 heads x 128: 46.6 us, 0.50 of the
// measured HBM rate (floor 23.4, F16 cache 88); 262144: 77.0, so 0.23 us per 1000 keys (0.77 of the rate) and 16 us that do not
// grow: a start, a page per warp, the joins. 64 keys at a time need 168 registers at head dim 128 but overlap better than 32 in
// 128 (46.4 against 52.6 us).
#include "paged_q4.cuh"

#include <algorithm>
#include <cfloat>

#include "paged.h"
#include "paged_join.cuh"
#include "tc_common.cuh"

namespace gsvcu {
namespace {

using namespace tc;

constexpr int NW = 4;            // warps per CTA
// Packed rows over the same keys from which these are unpacked first (k_unpack_q4) rather than in every CTA. 1024 rows over
// 16384 keys, 32/8 x 128: 95 us unpacked first, 92 not; 2048: 151 and 170; 4096: 239 and 300; heads of 64: 52 and 50, 79 and 85,
// 132 and 154.
constexpr int UNPACK_ROWS = 1536;
// And the mean over the sequences of a call. 32/8 x 128, 8192 keys each, unpacked first and not: a chunk of 512 tokens and 32
// single ones 555 and 422 us; 512 and 4: 170 and 160; 512 and 2: 152 and 158; 512, 100, 100, 100: 168 and 168; 1024 and 8: 283
// and 297.
constexpr int UNPACK_MEAN = 512;
// Weights are 2^BIAS exp(s - maximum). The maximum is taken off first, then the difference scaled: in one step a score past
// 2^24 would be off from its own maximum by whole steps of F32, its weight infinite in F16, or 0.
constexpr float BIAS = 14.0f;
constexpr int KT = PAGE;         // keys of one warp's tile: a block of the cache
// Keys whose scores are held at a time.
__host__ __device__ constexpr int part_keys(int nt) { return nt == 1 ? 64 : 32; }
// CTAs that the registers of an SM hold (pages dealt out take a few more). One sequence of 131072 keys of 8 heads x 128: 49.4 us
// with four, 46.4 with three.
__host__ __device__ constexpr int resident(int dim, int nt, bool dealt) {
    return nt > 1 ? 2 : dim == 128 ? 3 : dim == 64 || dealt ? 4 : 5;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N>   // words
__device__ __forceinline__ void lds(uint32_t a, uint32_t (&x)[N]) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                     : "r"(a)
                     : "memory");
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
// d = a b.
__device__ __forceinline__ void mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// d += a b.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Codes 0 .. 7 of a word, less 8, as the pairs (0, 4), (1, 5), (2, 6), (3, 7), by the usual way of widening nibbles: under the
// exponent of 1024 a code in bits 0 .. 3 is 1024 + code, one in bits 4 .. 7 is 1024 + 16 code.
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

// A warp has STAGES blocks of K and of V in shared memory (two are no faster than one): the next K comes while the weights and
// their product with V are worked on, the next V during the scores.
template <int D, int NT>
struct Cfg {
    using B = Q4Block<D>;
    static constexpr int STAGES = 1;
    static constexpr int ROWS = 8 * NT;
    static constexpr int QB = 2 * D;                         // bytes of a query row
    static constexpr int OSTR = D + 4;     // row stride of the outputs to be joined: lanes on different banks
    static constexpr size_t RING = (size_t)NW * STAGES * 2 * B::BYTES;
    static constexpr size_t JOIN = (size_t)NW * ROWS * OSTR * 4;   // reuses the blocks
    static constexpr size_t OFF_Q = RING > JOIN ? RING : JOIN;
    static constexpr size_t OFF_ML = OFF_Q + (size_t)ROWS * QB;
    static constexpr size_t OFF_BAR = OFF_ML + (size_t)NW * ROWS * 8 + 16;
    static constexpr size_t SMEM = OFF_BAR + NW * STAGES * 2 * 8;
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
    int group, tiles;
    int2* meta;       // [unit] first CTA of a unit and their number, for k_join_q4
    float c;          // |scale| * log2(e), at least the smallest normal number (a zero would make masked scores NaN)
    uint32_t flip;    // sign bits of a query pair when the scale is negative
    bool vec_q, vec_out;
};

// A unit is a (sequence, row tile, kv head). Short units have a CTA each. Else (DEALT) CTA i takes the pages [i per, (i + 1) per)
// of all units one after the other, so that ragged lengths, windows and units of any number fill the GPU evenly. A unit that
// several CTAs share is joined from their results; CTA i has at most two such, of its first unit (place 2 i) and of its last
// when that goes on (place 2 i + 1).
constexpr int LEAST = 2 * NW;   // pages of a CTA (fewer and the joins cost more than the pages)

// Pages of a sequence over its row tiles and kv heads; one for a unit that sees none (its rows are written all the same).
template <int ROWS>
__device__ __forceinline__ int64_t sequence_pages(const SplitArgs& a, int s, bool report) {
    int64_t n = 0;
    ChunkRange c;
    for (int tile = 0; tile < a.tiles; tile++) {
        if (!chunk_range(a.p, s, tile, a.group, ROWS, KT, report && tile == 0, c)) break;
        n += max(1, c.n_tiles);
    }
    return n * a.p.kv.n_head;
}
// Results g, g + per, ... of n_act CTAs from `first` on added up for four outputs of row r, FLIGHT loads in flight, in an order
// that the sizes alone decide.
template <int D, int ROWS>
__device__ __forceinline__ void sum_parts(const float* part, int first, int n_act, int g, int per, int r, int d, float& top,
                                          float& sum, float (&x)[4]) {
    constexpr int FLIGHT = 16;
    top = NEG_INF;
    sum = x[0] = x[1] = x[2] = x[3] = 0.0f;
    for (int w0 = g; w0 < n_act; w0 += FLIGHT * per) {
        float2 e[FLIGHT];
        float4 v[FLIGHT];
#pragma unroll
        for (int k = 0; k < FLIGHT; k++) {
            const int w = w0 + k * per;
            const float* at = part + (w == 0 ? 2 * (int64_t)first + 1 : 2 * (int64_t)(first + w)) * (ROWS * (D + 2));
            e[k] = w < n_act ? __ldcg((const float2*)(at + ROWS * D + 2 * r)) : make_float2(NEG_INF, 0.0f);
            v[k] = w < n_act ? __ldcg((const float4*)(at + r * D + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float up = top;
#pragma unroll
        for (int k = 0; k < FLIGHT; k++) up = fmaxf(up, e[k].x);
        const float ref = up == NEG_INF ? 0.0f : up, old = ex2(top - ref);
        top = up;
        sum *= old;
        x[0] *= old; x[1] *= old; x[2] *= old; x[3] *= old;
#pragma unroll
        for (int k = 0; k < FLIGHT; k++) {
            const float f = ex2(e[k].x - ref);
            sum = fmaf(f, e[k].y, sum);
            x[0] = fmaf(f, v[k].x, x[0]); x[1] = fmaf(f, v[k].y, x[1]);
            x[2] = fmaf(f, v[k].z, x[2]); x[3] = fmaf(f, v[k].w, x[3]);
        }
    }
}

template <typename T, int D, int NT, bool DEALT>
__global__ void __launch_bounds__(NW * 32, resident(D, NT, DEALT)) k_chunk_attn_q4(SplitArgs a) {
    using C = Cfg<D, NT>;
    using B = Q4Block<D>;
    constexpr int ROWS = C::ROWS, G = D / 32, PK = part_keys(NT), ST = C::STAGES;
    constexpr bool SCALED = !__is_same(T, __half);   // rows may have a factor of their own
    constexpr bool SPLIT = __is_same(T, __half);   // weights in two F16 parts; BF16 outputs have 8 bits, one part has 11
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ int64_t sums[NW], found[2];
    __shared__ int last;
    const ChunkAttnParams& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, heads = p.kv.n_head;
    griddep_wait();
    griddep_launch();

    const uint32_t ring = smem_addr(sm) + (uint32_t)(warp * ST * 2 * B::BYTES);          // [stage] K, V
    const uint32_t bars = smem_addr(sm + C::OFF_BAR) + (uint32_t)warp * ST * 16;
    if (lane == 0) {
        for (int st = 0; st < 2 * ST; st++) bar_init(bars + 8 * st, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    uint32_t phase = 0;   // blocks of K (and of V) that this warp has had
    bool ok = true, bad = false;

    // this CTA's pages [pos, end), and where the first of them is
    int s, tile = 0, h = 0;
    int64_t pos = 0, end = 0, per = 1, off = 0;
    int pages = 0;
    const bool early = !DEALT && !p.window;   // the first page numbers are fetched beside the sequence's length
    if constexpr (!DEALT) {
        int id = blockIdx.x;
        h = id % heads;
        id /= heads;
        tile = id % a.tiles;
        s = id / a.tiles;
        if (early) pages = p.batch.table[(int64_t)s * p.batch.max_pages + min(warp + lane * NW, p.batch.max_pages - 1)];
    } else {
        const int share = (p.batch.n_seq + NW * 32 - 1) / (NW * 32), s0 = min(tid * share, p.batch.n_seq);
        const int s1 = min(s0 + share, p.batch.n_seq);
        int64_t mine = 0;
        for (s = s0; s < s1; s++) mine += sequence_pages<ROWS>(a, s, blockIdx.x == 0);
        int64_t before = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int64_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        if (lane == 31) sums[warp] = before;
        __syncthreads();
        before -= mine;
        int64_t all = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            if (w < warp) before += sums[w];
            all += sums[w];
        }
        per = max((all + gridDim.x - 1) / gridDim.x, (int64_t)LEAST);
        pos = blockIdx.x * per;
        end = min(all, pos + per);
        if (pos >= all) return;
        if (before <= pos && pos < before + mine) {
            for (s = s0; s < s1 - 1; s++) {
                const int64_t n = sequence_pages<ROWS>(a, s, false);
                if (pos < before + n) break;
                before += n;
            }
            found[0] = s;
            found[1] = pos - before;
        }
        __syncthreads();
        s = (int)found[0];
        off = found[1];
    }

    for (;;) {   // units
        ChunkRange c;
        int v0 = 0, v1, first = 0, n_act = 1;   // this unit's pages here, the CTAs that share it
        int64_t taken = 0;
        if constexpr (!DEALT) {
            if (!chunk_range(p, s, tile, a.group, ROWS, KT, tid == 0 && h == 0 && tile == 0, c)) return;
            v1 = c.n_tiles;
        } else {
            int64_t here = 0;   // pages of a head
            while (s < p.batch.n_seq) {
                if (tile < a.tiles && chunk_range(p, s, tile, a.group, ROWS, KT, false, c)) {
                    here = max(1, c.n_tiles);
                    if (off < here * heads) break;
                    off -= here * heads;
                    tile++;
                } else {
                    s++;
                    tile = 0;
                }
            }
            if (s >= p.batch.n_seq) return;   // (not while the lengths stay as they are)
            h = (int)(off / here);
            v0 = (int)(off % here);
            taken = min(here - v0, end - pos);
            v1 = min(v0 + (int)taken, c.n_tiles);
            const int64_t start = pos - v0;
            first = (int)(start / per);
            n_act = (int)((start + here - 1) / per) - first + 1;
        }
        const int32_t* tab = p.batch.table + (int64_t)s * p.batch.max_pages;
        const int row0 = c.row0, n = c.n, total = c.total, len = c.len, r0 = c.r0, rows = c.rows, p0 = c.p0, p1 = c.p1, np = c.np;
        const int mine = ok && v0 + warp < v1 ? (v1 - v0 - warp + NW - 1) / NW : 0;
        auto key0 = [&](int i) { return c.tile_of(v0 + warp + i * NW) * KT; };

        // the page numbers of 32 tiles ahead sit in the warp's lanes
        int fetched_k = -1, fetched_v = -1;
        // K (V) of this warp's tile i; called for i, then the same i for V.
        auto fetch = [&](int i, bool v) {
            if (i >= mine) return;
            (v ? fetched_v : fetched_k) = i;
            if (!v && (i & 31) == 0 && (i || !early)) pages = i + lane < mine ? tab[key0(i + lane) / PAGE] : 0;
            const int page = __shfl_sync(0xffffffffu, pages, i & 31);
            const bool held = page >= 0 && page < p.kv.n_page;
            bad |= !held;
            if (lane == 0) {
                const uint32_t st = 2 * ((phase + i) % ST) + v, bar = bars + 8 * st;
                bar_expect_tx(bar, (held ? B::BYTES : 0) + (phase + i > 0 ? p.fault_extra_tx : 0u));
                const int64_t block = ((int64_t)page * p.kv.n_layer + p.kv.layer) * 2 * p.kv.n_head + h + (v ? p.kv.n_head : 0);
                if (held) bulk_load(ring + st * B::BYTES, (const uint8_t*)p.kv.pool + block * B::BYTES, B::BYTES, bar);
            }
        };
        auto arrived = [&](int i, bool v) {   // bounded
            const uint32_t bar = bars + 8 * (2 * ((phase + i) % ST) + v), parity = (phase + i) / ST & 1u;
            for (uint32_t it = 0; it < p.poll_limit; it++)
                if (__any_sync(0xffffffffu, bar_try_short(bar, parity))) return true;
            return false;
        };
#pragma unroll
        for (int i = 0; i < ST; i++) {
            fetch(i, false);
            fetch(i, true);
        }
        // queries into shared memory, zero past the tile's rows (after the first copies are under way)
        uint8_t* sq = sm + C::OFF_Q;
        float* row_c = (float*)(sm + C::OFF_ML);   // factors of the rows' scores, until the warps are joined
        for (int i = tid; i < ROWS * (D / 8); i += NW * 32) {
            const int r = i / (D / 8), pc = i % (D / 8);
            uint4 u = make_uint4(0, 0, 0, 0);
            if (r < rows) {
                const int tok = (r0 + r) / a.group, j = (r0 + r) % a.group;
                const T* src = (const T*)p.q + (int64_t)(row0 + tok) * p.q_stride + (int64_t)(h * a.group + j) * D + pc * 8;
                if (a.vec_q) {
                    u = *(const uint4*)src;
                } else {
                    T* y = (T*)&u;
#pragma unroll
                    for (int k = 0; k < 8; k++) y[k] = src[k];
                }
            }
            __half x[8];
            if constexpr (SCALED) {   // (every lane of the warp is here: a tile's pieces are a multiple of 32)
                int up = 0;
                float f = 1.0f, own = a.c;
                if (small_queries<D / 8>(u, up)) {
                    f = power_of_two(up);
                    own = fmaxf(own * power_of_two(-up), FLT_MIN);
                }
                if (pc == 0) row_c[r] = own;
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = __float2half_rn(__bfloat162float(((const T*)&u)[k]) * f);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = ((const T*)&u)[k];
            }
            auto two = [&](int k) { return bits(__halves2half2(x[k], x[k + 4])) ^ a.flip; };
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
        float m[NT][2], o[NT][D / 16][4];
        uint64_t l[NT];   // sums of the weights of two rows
#pragma unroll
        for (int b = 0; b < NT; b++) {
            m[b][0] = m[b][1] = NEG_INF;
            l[b] = 0;
#pragma unroll
            for (int d = 0; d < D / 16; d++) o[b][d][0] = o[b][d][1] = o[b][d][2] = o[b][d][3] = 0.0f;
        }
        float cr[NT][2];
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int e = 0; e < 2; e++) cr[b][e] = SCALED ? row_c[b * 8 + col + e] : a.c;
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
            const int first = key0(i);
            ok = arrived(i, false);
            if (!ok) break;
            const uint32_t kt = ring + 2 * ((phase + i) % ST) * B::BYTES, vt = kt + B::BYTES;
            const uint32_t ks = kt + B::OFF_SCALES, vs = vt + B::OFF_SCALES;
#pragma unroll 1
            for (int part = 0; part < KT; part += PK) {
                float sc[NT][PK / 16][4];   // [key kr, + 8][row col, + 1]
#pragma unroll
                for (int j = 0; j < PK / 16; j++) {
                    uint32_t w[2][G];
                    float d[2][G];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int key = part + j * 16 + kr + 8 * e;
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
                            float z[4];
                            mma0(z, f0, q[0], q[1]);
                            mma(z, f1, q[2], q[3]);
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                sc[b][j][e] = g == 0 ? z[e] * d[e >> 1][g] : fmaf(z[e], d[e >> 1][g], sc[b][j][e]);
                        }
                    }
                }
                if (part + PK == KT) {
                    __syncwarp();   // every lane is done with K
                    fetch(i + ST, false);
                }
                // keys that a row must not see to -infinity
                const int k0 = first + part;
                const bool whole = k0 + PK <= np || (k0 + PK <= min(len, p0 + 1) && (!p.window || k0 > p1 - p.window));
                if (!whole) {
#pragma unroll
                    for (int b = 0; b < NT; b++)
#pragma unroll
                        for (int j = 0; j < PK / 16; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int key = k0 + j * 16 + kr + 8 * (e >> 1);
                                if (!(key < np || (key < see_hi[b][e & 1] && key >= see_lo[b][e & 1]))) sc[b][j][e] = NEG_INF;
                            }
                    asm volatile("" ::: "memory");   // keeps the tests out of the tiles that need none
                }
#pragma unroll
                for (int b = 0; b < NT; b++) {
                    float ref[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float top = fmaxf(sc[b][0][e], sc[b][0][e + 2]);
#pragma unroll
                        for (int j = 1; j < PK / 16; j++) top = fmaxf(top, fmaxf(sc[b][j][e], sc[b][j][e + 2]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        if (top > m[b][e]) {
                            const float f = ex2((m[b][e] - top) * cr[b][e]);
                            l[b] = fmul2(l[b], e == 0 ? f2pack(f, 1.0f) : f2pack(1.0f, f));
#pragma unroll
                            for (int d = 0; d < D / 16; d++) {
                                o[b][d][e] *= f;
                                o[b][d][e + 2] *= f;
                            }
                            m[b][e] = top;
                        }
                        ref[e] = m[b][e] == NEG_INF ? 0.0f : -m[b][e];
                    }
                    const uint64_t c2 = f2pack(cr[b][0], cr[b][1]), r2 = f2pack(ref[0], ref[1]), up = f2pack(BIAS, BIAS);
#pragma unroll
                    for (int j = 0; j < PK / 16; j++)
#pragma unroll
                        for (int g = 0; g < 4; g += 2) {
                            const uint64_t x = ffma2(fadd2(f2pack(sc[b][j][g], sc[b][j][g + 1]), r2), c2, up);
                            const uint64_t w = f2pack(ex2(f2lo(x)), ex2(f2hi(x)));
                            sc[b][j][g] = f2lo(w);
                            sc[b][j][g + 1] = f2hi(w);
                            l[b] = fadd2(l[b], w);
                        }
                }
                if (part == 0) {
                    ok = arrived(i, true);
                    if (!ok) break;
                    if (first + KT > len) {   // values past the last key become 0 by their scales
                        for (int x = max(0, len - first) * G + lane; x < KT * G; x += 32)
                            asm volatile("st.shared.u16 [%0], %1;" ::"r"(vs + x * 2), "h"((uint16_t)0) : "memory");
                        __syncwarp();
                    }
                }
#pragma unroll
                for (int j = 0; j < PK / 16; j++) {
                    uint32_t wh[NT][2], wl[NT][2];
#pragma unroll
                    for (int b = 0; b < NT; b++)
#pragma unroll
                        for (int g = 0; g < 2; g++) {
                            if constexpr (SPLIT) {
                                uint32_t rest;
                                wh[b][g] = transpose8(pack_split(sc[b][j][2 * g], sc[b][j][2 * g + 1], rest));
                                wl[b][g] = transpose8(rest);
                            } else {
                                wh[b][g] = transpose8(bits(__floats2half2_rn(sc[b][j][2 * g], sc[b][j][2 * g + 1])));
                            }
                        }
                    // values of the lane's D / 8 dims: [key pair: col, col + 8][dim] halves (key, key + 1)
                    uint32_t v[2][D / 8];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int key = part + j * 16 + col + 8 * e;
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
                            if constexpr (SPLIT) mma(o[b][d], va, wl[b][0], wl[b][1]);
                            mma(o[b][d], va, wh[b][0], wh[b][1]);
                        }
                    }
                }
            }
            if (!ok) break;
            __syncwarp();   // every lane is done with V
            fetch(i + ST, true);
        }
        if (!ok) {   // whatever is on its way lands before the CTA goes on
            if (lane == 0) atomicOr(p.err, PAGED_WAIT);
            for (int k = max(0, fetched_k - ST + 1); k <= fetched_k; k++) arrived(k, false);
            for (int k = max(0, fetched_v - ST + 1); k <= fetched_v; k++) arrived(k, true);
        }
        phase += (uint32_t)mine;
        if (bad && lane == 0) atomicOr(p.err, PAGED_BAD_PAGE);
        bad = false;

        // join the warps
        float* ml = (float*)(sm + C::OFF_ML);   // [NW][ROWS] {m, l}
        float* so = (float*)sm;                 // [NW][ROWS][OSTR]
        __syncthreads();
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float x = e ? f2hi(l[b]) : f2lo(l[b]);
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int r = warp * ROWS + b * 8 + col + e;
                if (lane < 4) {
                    ml[2 * r] = m[b][e] * cr[b][e] - BIAS;   // (what the weights refer to)
                    ml[2 * r + 1] = x;
                }
#pragma unroll
                for (int d = 0; d < D / 16; d++) {
                    so[r * C::OSTR + dim_of<D>(kr, 2 * d)] = o[b][d][e];
                    so[r * C::OSTR + dim_of<D>(kr, 2 * d + 1)] = o[b][d][e + 2];
                }
            }
        __syncthreads();
        const int64_t unit = ((int64_t)s * a.tiles + tile) * heads + h;
        float* part = p.part + (2 * (int64_t)blockIdx.x + ((int)blockIdx.x == first)) * (ROWS * (D + 2));   // [ROWS][D], {m, l}
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
            if (!DEALT || n_act == 1) {
                finish<T, D>(p, c, a.vec_out, a.group, h, r, d, top, sum, x);
            } else {
                *(float4*)(part + r * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                if (d == 0) *(float2*)(part + ROWS * D + 2 * r) = make_float2(top, sum);
            }
        }
        if (DEALT && ROWS > 8 && v0 == 0 && tid == 0) a.meta[unit] = make_int2(first, n_act);   // (joined by k_join_q4)
        if (DEALT && ROWS == 8 && n_act > 1) {
            // The CTA that arrives last joins the unit and clears its counter.
            __threadfence();
            __syncthreads();
            if (tid == 0) last = atomicAdd(p.arrived + unit, 1) == n_act - 1;
            __syncthreads();
            if (last) {
                __threadfence();
                if (tid == 0) p.arrived[unit] = 0;
                // thread = four outputs of a row over every ways-th result; where rows and outputs are fewer than the threads, ways
                // of them share a row's results
                float* buf = (float*)sm;
                const int items = rows * (D / 4);
                int ways = 1;
                while (ways * 2 * items <= NW * 32 && ways * 2 <= n_act) ways *= 2;
                for (int i = tid; i < items * ways; i += NW * 32) {
                    const int item = i % items, g = i / items, r = item / (D / 4), d = item % (D / 4) * 4;
                    float top, sum, x[4];
                    sum_parts<D, ROWS>(p.part, first, n_act, g, ways, r, d, top, sum, x);
                    if (ways > 1) {
                        *(float4*)(buf + 8 * i) = make_float4(x[0], x[1], x[2], x[3]);
                        *(float2*)(buf + 8 * i + 4) = make_float2(top, sum);
                    } else {
                        finish<T, D>(p, c, a.vec_out, a.group, h, r, d, top, sum, x);
                    }
                }
                if (ways > 1) {   // (items * ways <= the threads)
                    __syncthreads();
                    if (tid < items) {
                        float top = NEG_INF, sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        for (int g = 0; g < ways; g++) top = fmaxf(top, buf[8 * (g * items + tid) + 4]);
                        const float ref = top == NEG_INF ? 0.0f : top;
                        for (int g = 0; g < ways; g++) {
                            const float* y = buf + 8 * (g * items + tid);
                            const float f = ex2(y[4] - ref);
                            sum = fmaf(f, y[5], sum);
#pragma unroll
                            for (int k = 0; k < 4; k++) x[k] = fmaf(f, y[k], x[k]);
                        }
                        finish<T, D>(p, c, a.vec_out, a.group, h, tid / (D / 4), tid % (D / 4) * 4, top, sum, x);
                    }
                }
            }
        }
        if (!DEALT) return;
        pos += taken;
        off += taken;
        if (pos >= end) return;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // what follows is copied over what was written here
        __syncthreads();
    }
}

// Units of more than 8 rows: a CTA per (unit, 1024 outputs).
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) k_join_q4(SplitArgs a) {
    constexpr int R = 1024 / D;   // rows of a CTA
    const ChunkAttnParams& p = a.p;
    griddep_wait();
    griddep_launch();
    const int64_t unit = blockIdx.x / ((ROWS + R - 1) / R);
    const int r = blockIdx.x % ((ROWS + R - 1) / R) * R + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const int h = (int)(unit % p.kv.n_head), tile = (int)(unit / p.kv.n_head % a.tiles), s = (int)(unit / p.kv.n_head / a.tiles);
    ChunkRange c;
    if (!chunk_range(p, s, tile, a.group, ROWS, KT, false, c) || r >= c.rows) return;
    const int2 m = a.meta[unit];
    if (m.y <= 1) return;   // (written by the only CTA)
    float top, sum, x[4];
    sum_parts<D, ROWS>(p.part, m.x, m.y, 0, 1, r, d, top, sum, x);
    finish<T, D>(p, c, a.vec_out, a.group, h, r, d, top, sum, x);
}

template <typename T, int D, int NT, typename F>
void pick_dealt(bool dealt, F f) {
    if (dealt) f(k_chunk_attn_q4<T, D, NT, true>, Cfg<D, NT>::SMEM);
    else f(k_chunk_attn_q4<T, D, NT, false>, Cfg<D, NT>::SMEM);
}
template <typename T, int D, typename F>
void pick_rows(int row_tile, bool dealt, F f) {
    if (row_tile == 8) pick_dealt<T, D, 1>(dealt, f);
    else if (row_tile == 16) pick_dealt<T, D, 2>(dealt, f);
    else if (row_tile == 24) pick_dealt<T, D, 3>(dealt, f);
    else pick_dealt<T, D, 4>(dealt, f);
}
template <typename T, typename F>
void pick_dim(int dim, int row_tile, bool dealt, F f) {
    if (dim == 32) pick_rows<T, 32>(row_tile, dealt, f);
    else if (dim == 64) pick_rows<T, 64>(row_tile, dealt, f);
    else pick_rows<T, 128>(row_tile, dealt, f);
}
template <typename F>
void pick(int dtype, int dim, int row_tile, bool dealt, F f) {
    if (dtype == GSVCU_KV_Q4_F16) pick_dim<__half>(dim, row_tile, dealt, f);
    else pick_dim<__nv_bfloat16>(dim, row_tile, dealt, f);
}

}  // namespace

ChunkAttnPlan chunk_attention_q4_plan(const ChunkAttnParams& p) {
    const int D = p.kv.head_dim;
    const int64_t packed = (int64_t)p.batch.max_chunk * (p.n_q_head / p.kv.n_head);
    ChunkAttnPlan c;
    if (packed > 32 && p.scale != 0.0f) {
        c = chunk_attention_tc_plan(p);
        // Many row tiles over the same keys: the keys are unpacked once, by a kernel before it. All sequences' keys are, so it
        // takes some rows of each that has any (at most 1 + n_rows - max_chunk beside idle ones).
        const int group = p.n_q_head / p.kv.n_head;
        const int64_t active = std::min<int64_t>(p.batch.n_seq, 1 + p.batch.n_rows - p.batch.max_chunk);
        auto rows = [&](int64_t tokens) { return group * (p.window ? std::min<int64_t>(tokens, p.window) : tokens); };
        const int64_t pages = (p.batch.max_kv + PAGE - 1) / PAGE;
        const int64_t bytes = p.batch.n_seq * pages * ((int64_t)p.kv.n_head * (4 * PAGE * D) + 4);
        if (rows(p.batch.max_chunk) >= UNPACK_ROWS && rows(p.batch.n_rows / active) >= UNPACK_MEAN && bytes <= UNPACK_LIMIT) {
            c.unpack_pages = (int)pages;
            c.unpacked_floats = (size_t)(bytes / 4);
        }
        return c;
    }
    c.row_tile = packed >= 32 ? 32 : (int)(packed + 7) / 8 * 8;
    c.tiles = (int)((packed + c.row_tile - 1) / c.row_tile);
    const int64_t units = (int64_t)p.batch.n_seq * c.tiles * p.kv.n_head;
    const int max_tiles = (p.batch.max_kv + KT - 1) / KT;
    size_t smem = 0;
    pick(p.kv.kv_dtype, D, c.row_tile, true, [&](auto, size_t bytes) { smem = bytes; });
    const int64_t slots = 148 * std::min((int64_t)(232448 / (smem + 1024)), (int64_t)resident(D, c.row_tile / 8, true));
    c.key_tile = KT;
    // Short units: a CTA for each, nothing to join and no lengths to add up first. 64 slots of 600 to 2100 keys, 16 heads x 32:
    // 31.8 us, 42 dealt out; 4 of 2000 to 4000 keys: 25 and 18; at head dim 128 a page takes longer, and 32 units of 600 to 2100
    // keys are faster dealt out (17.3, 21.4). Many units even out by themselves: 3200 of 2000 to 4000 keys, heads of 32, 141 us,
    // dealt out 164; of 64 187 and 211, of 128 311 and 338; with 32 rows of 32 545 and 591, of 128 1005 and 1100.
    if (max_tiles <= (units >= 4 * slots ? 64 : D < 128 || units >= slots ? 40 : 16)) {
        c.ctas = units;
        return c;
    }
    c.ctas = std::min(slots, (units * std::max(max_tiles, 1) + LEAST - 1) / LEAST);
    c.dealt = true;
    c.join_apart = c.row_tile > 8;   // (as chunk_attention_plan)
    c.part_floats = (size_t)2 * c.ctas * c.row_tile * (D + 2) + (c.join_apart ? 2 * units : 0);
    c.arrivals = c.join_apart ? 0 : (size_t)units;
    return c;
}

template <typename T, int D>
static void launch_join_rows(const SplitArgs& a, int row_tile, unsigned units, cudaStream_t s) {
    const int rows = 1024 / D;
    const unsigned ctas = units * ((row_tile + rows - 1) / rows);
    auto go = [&](auto k) { launch_pdl(k, dim3(ctas), dim3(256), 0, s, a); };
    if (row_tile == 16) go(k_join_q4<T, D, 16>);
    else if (row_tile == 24) go(k_join_q4<T, D, 24>);
    else go(k_join_q4<T, D, 32>);
}
template <typename T>
static void launch_join(const SplitArgs& a, int row_tile, unsigned units, cudaStream_t s) {
    if (a.p.kv.head_dim == 32) launch_join_rows<T, 32>(a, row_tile, units, s);
    else if (a.p.kv.head_dim == 64) launch_join_rows<T, 64>(a, row_tile, units, s);
    else launch_join_rows<T, 128>(a, row_tile, units, s);
}

int launch_chunk_attention_q4(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s) {
    SplitArgs a;
    a.p = p;
    if (!a.p.poll_limit) a.p.poll_limit = TC_SPIN_LIMIT;
    a.group = p.n_q_head / p.kv.n_head;
    a.tiles = plan.tiles;
    a.meta = (int2*)(p.part + (size_t)2 * plan.ctas * plan.row_tile * (p.kv.head_dim + 2));
    a.c = std::max(fabsf(p.scale) * LOG2E, FLT_MIN);
    a.flip = p.scale < 0.0f ? 0x80008000u : 0u;
    a.vec_q = ((uintptr_t)p.q & 15) == 0 && p.q_stride % 8 == 0;
    a.vec_out = ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0;
    const bool f16 = p.kv.kv_dtype == GSVCU_KV_Q4_F16;
    const int bit = ((f16 ? 0 : 3) + p.kv.head_dim / 64) * 4 + plan.row_tile / 8 - 1 + (plan.dealt ? 33 : 0);   // 0 .. 23, 33 .. 56
    bool ok = false;
    pick(p.kv.kv_dtype, p.kv.head_dim, plan.row_tile, plan.dealt, [&](auto k, size_t smem) {
        ok = raise_smem(k, smem, ready, bit);
        if (ok) launch_pdl(k, dim3((unsigned)plan.ctas), dim3(NW * 32), smem, s, a);
    });
    if (!ok || !plan.join_apart) return ok ? 1 : 0;
    const unsigned units = (unsigned)(p.batch.n_seq * plan.tiles * p.kv.n_head);
    if (f16) launch_join<__half>(a, plan.row_tile, units, s);
    else launch_join<__nv_bfloat16>(a, plan.row_tile, units, s);
    return 2;
}

}  // namespace gsvcu
