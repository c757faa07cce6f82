// paged_attention_tc.cu -- attention of many new rows over the paged KV cache on the 5th-generation tensor
// cores (F16 / BF16); the operator's formula and the variant for few rows are in paged_attention.cu.
//
// k_chunk_attn_tc: one CTA per (sequence, 256 packed rows, kv head, key split), as two row tiles of 128 rows
// (packed row r = token * g + query head of the group). Key tiles are 128 keys = two pages, each page's
// [64][head dim] block fetched by TMA into a ring of pairs (V of one tile, K of the next).
//   warp 0     page numbers (32 per load) and TMA
//   warp 1     MMA: S = Q K^T (both operands in shared memory), O += P V (P in tensor memory, V in shared
//              memory as it lies in the page: the MN-major operand, so nothing is transposed)
//   warp 2     clears what the last page holds past the last key
//   warps 4-7  softmax of row tile 0, one thread per row (TMEM lane); warps 8-11 of row tile 1
// The MMAs of one row tile run under the other's softmax: S0 S1 | PV0 S0' PV1 S1' | ... Each thread takes its
// 128 scores into registers, writes the weights P over them in tensor memory as 16-bit pairs, and keeps the
// row's sum. A row's reference maximum is raised only when a tile exceeds it by more than 2^TAU, then O in
// tensor memory is scaled once its last PV is done. Weights are rounded to the cache's type for the product: with
// the output's own rounding that is sqrt(2) of it, and the sums stay f32. F16 weights are kept 2^BIAS up (P <= 2^(TAU +
// BIAS) = 2^15), so that their 11 bits reach down to 2^-25 of the maximum and the last one to 2^-35 (a long light tail
// beside one heavy key); the factor is in the reference, so sums, splits and the log-sum-exp need nothing for it.
// Tensor memory: S0 | S1 (128 columns each; P over their first 64) | O0 | O1. With one row tile its key tiles take
// the two score buffers in turn, and the next scores are computed beside the softmax.
// Products of two row tiles and 128 keys take 2048 cycles at head dim 128, a softmax warp ~1850 per tile; what bounds the
// kernel is the chain weights -> last product -> next scores -> wake, ~2950 cycles (4096 rows over 16384 keys, 32/8 heads of
// 128: 810 to 945 us with the power cap, 1.0 to 1.2 PFLOP/s), at head dims 32 and 64 the softmax warps' instructions.
// V rows past kv_len in the last tile are zeroed in shared memory before its product, absent pages are
// zero-filled by TMA (a block index past the pool), masked keys get weight 0.
#include <cuda_bf16.h>

#include <type_traits>

#include "paged.h"
#include "paged_join.cuh"
#include "tc_common.cuh"

namespace gsvcu {
namespace {

using namespace tc;

constexpr int KT = 128;                 // keys per tile
constexpr int ROWS = 256;               // packed rows per CTA, two row tiles (one of 128 when the call has few CTAs)
constexpr int THREADS = 384;
// Log2 headroom of P above the row's reference maximum, and how far up the weights are kept. F16: TAU 5, 4 or 3 cost
// about 1 % over TAU 8 on scores of deviation 1, TAU 1 2 to 7 %.
template <typename T> constexpr float TAU = __is_same(T, __half) ? 4.0f : 8.0f;
template <typename T> constexpr float BIAS = __is_same(T, __half) ? 11.0f : 0.0f;

template <int D>
struct Smem {
    static constexpr int RB = D >= 64 ? 128 : 2 * D;              // bytes of a swizzled row
    static constexpr int ATOMS = D >= 64 ? D / 64 : 1;            // 64-dim column blocks of a tile
    static constexpr int ENTRY = KT * D * 2;                      // bytes of a K or V tile
    static constexpr int NP = 2;                                  // ring pairs: V of tile i - 1, K of tile i
    // Tensor memory: two score buffers (one per row tile; for tiles in turn when there is one row tile), P over the
    // first half of its scores, then O.
    static constexpr uint32_t TM_O = 2 * KT;
    static constexpr size_t OFF_RING = (size_t)ROWS * D * 2;      // after Q
    static constexpr size_t OFF_BAR = OFF_RING + (size_t)NP * 2 * ENTRY;
    // full, empty [NP], S full [2], P full [2][2 halves], PV done [2] (one per row tile; with one row tile, for its key
    // tiles in turn), V landed, V cleared, drain
    static constexpr int NBAR = 2 * NP + 11;
    static constexpr size_t SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
};

struct TcArgs {
    ChunkAttnParams p;
    CUtensorMap map;   // pool as [block][64][D], box [1][64][min(D, 64)]
    int group, row_tile, tiles, n_split, split_tiles, n_blocks;
    float c;           // |scale| * log2(e)
    bool negate;       // scale < 0: Q enters negated
    bool vec_q, vec_out;
};

// Shared-memory operand descriptors, low word: address and column-block stride lbo in 16-byte units (addresses
// stay below 2^18, so a descriptor moves by adding 16-byte units); high word: 8-row groups at 8 * RB bytes,
// version 1, 128- or 64-byte swizzle of RB-byte rows.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
template <int RB>
constexpr uint32_t DESC_HI = (8 * RB >> 4) | (1u << 14) | ((RB == 128 ? 2u : 4u) << 29);
// Instruction descriptor: f32 accumulator, 16-bit operands (0 F16, 1 BF16), B MN-major when `tb`.
__host__ __device__ constexpr uint32_t instr(int type, int tb, int n) {
    return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)tb << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
// The MMA warp runs its loop as a whole and one elected lane issues: operands then stay in uniform registers.
// (Under a branch on the lane every operand was moved there for each MMA, 60 cycles apiece.)
// D (tensor memory) (+)= A (shared memory) x B (shared memory); descriptors as low words and one high word.
template <uint32_t HI, uint32_t ID, bool ADD>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 a, b;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %5, 0;\n"
        " mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "n"(HI), "n"(ID), "n"((int)ADD)
        : "memory");
}
// D (tensor memory) (+)= A (tensor memory, 16-bit pairs) x B (shared memory).
template <uint32_t HI, uint32_t ID>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t add) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 b;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %5, 0;\n"
        " mov.b64 b, {%2, %3};\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "n"(HI), "n"(ID), "r"(add)
        : "memory");
}
// The barrier completes a phase when every MMA that the elected lane issued before is done.
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar)
        : "memory");
}
// Bounded wait of a converged warp, with a warp-uniform result.
__device__ __forceinline__ bool wait_warp(uint32_t b, uint32_t parity, volatile int* abort_flag, uint32_t limit = TC_SPIN_LIMIT) {
    for (uint32_t it = 0; it < limit; it++) {
        if (__any_sync(0xffffffffu, bar_try_short(b, parity))) return true;
        if (__any_sync(0xffffffffu, *abort_flag)) return false;
    }
    return false;
}
#define REG4(c, x, i) c(x[i]), c(x[i + 1]), c(x[i + 2]), c(x[i + 3])
#define REG8(c, x, i) REG4(c, x, i), REG4(c, x, i + 4)
#define R8(x, i) REG8("+r", x, i)
#define R32(x) R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24)
#define W8(x, i) REG8("=r", x, i)
#define V8(x, i) REG8("r", x, i)
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

// The lowest n bits (n cut to 0 .. 32).
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : 0xffffffffu >> (32 - min(n, 32)); }
// Maxima that keep a NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float max2(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
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

// One pair of weights in EVERY takes its exponentials on the FMA pipe: the special-function unit (16 per cycle
// and SM) would need 2048 cycles for two row tiles of 128 keys, as many as their products at head dim 128.
constexpr int EVERY = 4;
// 2^x of two values on the FMA pipe: x = n + f with n the nearest integer (by the 1.5 * 2^23 addend) and
// |f| <= 1/2, 2^f by its relative minimax polynomial of degree 4 (least squares with Lawson's weights; relative error
// 2.7e-6, which the sums and the log-sum-exp take too: degree 5, 2.1e-7, made F16 chunks 1 to 3 % slower), n added to
// the exponent. Below 2^-126: 2^-126.
// x must not be NaN (rows that hold one have a NaN reference, and the sums and products of their other pairs are NaN).
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
    x = f2pack(fmaxf(f2lo(x), -126.0f), fmaxf(f2hi(x), -126.0f));
    const uint64_t big = f2pack(12582912.0f, 12582912.0f), nbig = f2pack(-12582912.0f, -12582912.0f);
    const uint64_t n = fadd2(x, big);
    const uint64_t f = ffma2(fadd2(n, nbig), f2pack(-1.0f, -1.0f), x);
    auto k = [](float v) { return f2pack(v, v); };
    uint64_t y = ffma2(f, k(0x1.3997d6p-7f), k(0x1.ca1440p-5f));
    y = ffma2(f, y, k(0x1.ec06dap-3f));
    y = ffma2(f, y, k(0x1.62e0dcp-1f));
    y = ffma2(f, y, k(0x1.ffffe8p-1f));
    return f2pack(__int_as_float(__float_as_int(f2lo(y)) + (__float_as_int(f2lo(n)) << 23)),
                  __int_as_float(__float_as_int(f2hi(y)) + (__float_as_int(f2hi(n)) << 23)));
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
    auto empty = [&](int e) { return bar0 + 8u * (L::NP + e); };
    auto sfull = [&](int b) { return bar0 + 8u * (2 * L::NP + b); };
    auto pfull = [&](int b, int half) { return bar0 + 8u * (2 * L::NP + 2 + 2 * b + half); };
    auto pvdone = [&](int t) { return bar0 + 8u * (2 * L::NP + 6 + t); };
    const uint32_t vhere = pvdone(2), vclear = vhere + 8, drain = vhere + 16;
    uint32_t* tmem_slot = (uint32_t*)(sm + L::OFF_BAR + L::NBAR * 8);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

    int id = blockIdx.x;
    const int sp = id % a.n_split;
    id /= a.n_split;
    const int h = id % p.kv.n_head;
    id /= p.kv.n_head;
    const int s = id % p.batch.n_seq, tile = a.tiles - 1 - id / p.batch.n_seq;   // the last rows see most keys: first
    if (tid == 0) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&a.map) : "memory");
    griddep_wait();
    griddep_launch();

    // Without a window the key tiles are known before the sequence's length: warp 0 fetches the first page numbers
    // beside it (lane = tile, page; entries past the sequence are not used).
    const int v0 = sp * a.split_tiles;
    const int32_t* tab = p.batch.table + (int64_t)s * p.batch.max_pages;
    int first_page = 0;
    if (warp == 0 && !p.window) first_page = tab[min(v0 * 2 + lane, p.batch.max_pages - 1)];
    ChunkRange c;
    if (!chunk_range(p, s, tile, a.group, a.row_tile, KT, tid == 0 && sp == 0 && h == 0 && tile == 0, c)) return;
    const int n_act = max(1, (c.n_tiles + a.split_tiles - 1) / a.split_tiles);
    if (sp >= n_act) return;
    const int nt = min(c.n_tiles, v0 + a.split_tiles) - v0;   // this CTA's key tiles
    const int halves = c.rows > 128 ? 2 : 1;
    auto key0 = [&](int j) { return c.tile_of(v0 + j) * KT; };

    if (tid == 0) {
        for (int e = 0; e < L::NP; e++) { bar_init(full(e), 1); bar_init(empty(e), 1); }
        for (int b = 0; b < 2; b++) {
            bar_init(sfull(b), 1);
            bar_init(pfull(b, 0), 4);
            bar_init(pfull(b, 1), 4);
            bar_init(pvdone(b), 1);
        }
        bar_init(vhere, 1);
        bar_init(vclear, 32);
        bar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (this warp's first copies come before the CTA meets)
    }
    // Warp 0's work: pair i is V of tile i - 1, then K of tile i (what the MMA warp needs together).
    int blk = 0;
    bool bad = false;
    uint32_t v0b = 0, v1b = 0;   // K blocks of the tile before (its V follows one pair later)
    auto load_pair = [&](int i) -> bool {
        const int e = i % L::NP;
        if ((i & 15) == 0) {   // the blocks of 16 tiles: lane = (tile, page)
            const int jj = i + (lane >> 1);
            blk = a.n_blocks;   // past the pool: zero fill
            if (jj < nt) {
                const int key = key0(jj) + PAGE * (lane & 1);
                if (c.sees(key)) {
                    const int page = i == 0 && !p.window ? first_page : tab[key / PAGE];
                    if (page >= 0 && page < p.kv.n_page) blk = ((page * p.kv.n_layer + p.kv.layer) * 2) * p.kv.n_head + h;
                    else bad = true;
                }
            }
        }
        const uint32_t k0b = __shfl_sync(0xffffffffu, blk, (i & 15) * 2);
        const uint32_t k1b = __shfl_sync(0xffffffffu, blk, (i & 15) * 2 + 1);
        bool ok = true;
        if (lane == 0) {
            ok = bar_wait_short(empty(e), ((uint32_t)(i / L::NP) & 1u) ^ 1u, abort_flag);
            if (ok) {
                const bool has_v = i > 0, has_k = i < nt;
                bar_expect_tx(full(e), ((int)has_v + (int)has_k) * L::ENTRY + (has_v ? p.fault_extra_tx : 0u));
                const uint32_t dst = su32(sm + L::OFF_RING + (size_t)e * 2 * L::ENTRY);
                auto load = [&](uint32_t to, uint32_t b0, uint32_t b1) {
#pragma unroll
                    for (int at = 0; at < L::ATOMS; at++) {
                        tma_load_3d(to + at * KT * L::RB, &a.map, at * 64, 0, (int)b0, full(e));
                        tma_load_3d(to + at * KT * L::RB + PAGE * L::RB, &a.map, at * 64, 0, (int)b1, full(e));
                    }
                };
                const uint32_t none = a.n_blocks;
                if (has_v) load(dst, v0b == none ? none : v0b + p.kv.n_head, v1b == none ? none : v1b + p.kv.n_head);
                if (has_k) load(dst + L::ENTRY, k0b, k1b);
            }
        }
        v0b = k0b;
        v1b = k1b;
        return __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    };
    const int pairs = nt > 0 ? nt + 1 : 0, early = min(pairs, L::NP);   // the first ones find the ring empty
    if (warp == 0) {
        __syncwarp();
        for (int i = 0; i < early; i++) load_pair(i);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Q, swizzled as the MMA reads it ([tile][64-dim block][128 rows][RB bytes]), zero past the CTA's rows; four loads
    // in flight per thread (one at a time this was a third of a short call)
    constexpr int STEP = THREADS - 32;
    const int tok0 = c.r0 / a.group, rem0 = c.r0 % a.group;
    const float inv = 1.0f / (float)a.group;   // (x + 1/2) / group is far enough from whole numbers for x < 2^20
    for (int i0 = tid - 32; warp > 0 && i0 < 128 * halves * (D / 8); i0 += 4 * STEP) {
        uint4 u[4];
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const int i = i0 + m * STEP, r = i / (D / 8), pc = i % (D / 8);
            u[m] = make_uint4(0, 0, 0, 0);
            if (r < c.rows) {
                const int up = (int)(((float)(rem0 + r) + 0.5f) * inv), j = rem0 + r - up * a.group;
                const T* src = (const T*)p.q + (int64_t)(c.row0 + tok0 + up) * p.q_stride +
                               (int64_t)(h * a.group + j) * D + pc * 8;
                if (a.vec_q) {
                    u[m] = *(const uint4*)src;
                } else {
                    T* x = (T*)&u[m];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = src[k];
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const int i = i0 + m * STEP, r = i / (D / 8), pc = i % (D / 8);
            if (r >= 128 * halves) break;
            if (a.negate) { u[m].x ^= 0x80008000u; u[m].y ^= 0x80008000u; u[m].z ^= 0x80008000u; u[m].w ^= 0x80008000u; }
            const int rt = r & 127, atom = D >= 64 ? pc / 8 : 0, ch = D >= 64 ? pc % 8 : pc;
            const int swz = L::RB == 128 ? rt & 7 : (rt >> 1) & 3;
            *(uint4*)(sm + (size_t)(r >> 7) * 128 * D * 2 + (size_t)atom * 128 * L::RB + rt * L::RB + ((ch ^ swz) << 4)) = u[m];
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Registers move from the TMA / MMA warps to the softmax: 128 x 104 + 256 x 200 = 384 x 168, the launch's own.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 0) {
            int i = early;
            bool ok = true;
            for (; i < pairs && ok; i++) ok = load_pair(i);
            if (bad) atomicOr(p.err, PAGED_BAD_PAGE);
            if (lane == 0) {
                if (!ok) {
                    atomicOr(p.err, PAGED_WAIT);
                    *abort_flag = 1;
                    i--;   // its copies were not issued
                }
                // every copy has landed before the CTA may end
                for (int k = i - 1; k >= 0 && k >= i - L::NP; k--)
                    for (uint32_t it = 0; it < min(TC_POLL_LIMIT, p.poll_limit); it++)
                        if (bar_try(full(k % L::NP), (uint32_t)(k / L::NP) & 1u)) break;
            }
        } else if (warp == 1) {
            constexpr uint32_t HI = DESC_HI<L::RB>;
            const uint32_t tm = __reduce_or_sync(0xffffffffu, tmem);   // (into a uniform register)
            const uint32_t sq = su32(sm), ring = su32(sm + L::OFF_RING);
            const bool cut = nt > 0 && key0(nt - 1) + KT > c.len;
            // The loop is unrolled over the ring, so addresses and most phases are constants: this warp shares its
            // scheduler with two softmax warps, and every instruction between two products is idle tensor time.
            auto scores = [&](int t, int b, int e) {   // S buffer b = Q_t K^T with the K of pair e
                const uint32_t qd = desc_lo(sq + (uint32_t)t * 128 * D * 2, 16);
                const uint32_t kd = desc_lo(ring + (uint32_t)(2 * e + 1) * L::ENTRY, 16);
                const uint32_t st = tm + (uint32_t)b * KT;
                mma_ss<HI, ID_S, false>(st, qd, kd);
#pragma unroll
                for (int kk = 1; kk < D / 16; kk++) {
                    const uint32_t off = (kk / 4 * 128 * L::RB + 32 * (kk % 4)) >> 4;   // 64-dim block, 16 dims in it
                    mma_ss<HI, ID_S, true>(st, qd + off, kd + off);
                }
                commit(sfull(b));
            };
            // O_t += P V with the V of pair e, 64 keys at a time
            auto values = [&](int t, int b, int e, uint32_t add, uint32_t parity) -> bool {
                const uint32_t vd = desc_lo(ring + (uint32_t)(2 * e) * L::ENTRY, KT * L::RB);
                const uint32_t ot = tm + L::TM_O + (uint32_t)t * 128, pt = tm + (uint32_t)b * KT;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    if (!wait_warp(pfull(b, half), parity, abort_flag)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int kk = half * KT / 32; kk < (half + 1) * KT / 32; kk++)
                        mma_ts<HI, ID_O>(ot, pt + 8u * kk, vd + ((kk * 16 * L::RB) >> 4), kk == 0 ? add : 1u);
                }
                return true;
            };
            bool ok = nt == 0 || wait_warp(full(0), 0, abort_flag);
            if (ok && nt > 0) {
                scores(0, 0, 0);
                if (halves == 2) scores(1, 1, 0);
                commit(empty(0));
            }
            // V of tile j and K of tile j + 1 are pair j + 1; at the last tile V has to be cleared first
            auto wait_pair = [&](int j, int e, uint32_t parity) -> bool {
                if (!wait_warp(full(e), parity, abort_flag, p.poll_limit)) return false;
                if (j + 1 < nt || !cut) return true;
                if (lane == 0) bar_arrive(vhere);
                return wait_warp(vclear, 0, abort_flag);
            };
            uint32_t turn = 0;   // parity of how often the ring went round
            if (halves == 2) {
                for (int j0 = 0; j0 < nt && ok; j0 += L::NP, turn ^= 1u) {
#pragma unroll
                    for (int u = 0; u < L::NP; u++) {
                        const int j = j0 + u, e = u ^ 1;
                        if (j >= nt) break;
                        const bool more = j + 1 < nt;
                        ok = wait_pair(j, e, turn ^ (uint32_t)u) && values(0, 0, e, (uint32_t)j, u);
                        if (!ok) break;
                        if (more) scores(0, 0, e);
                        ok = values(1, 1, e, (uint32_t)j, u);
                        if (!ok) break;
                        if (more) scores(1, 1, e);
                        commit(empty(e));
                    }
                }
                commit(pvdone(0));
                commit(pvdone(1));
            } else {   // one row tile: the next scores go to the other buffer, before this tile's product
                for (int j0 = 0; j0 < nt && ok; j0 += L::NP, turn ^= 1u) {
#pragma unroll
                    for (int u = 0; u < L::NP; u++) {
                        const int j = j0 + u, e = u ^ 1;
                        if (j >= nt) break;
                        ok = wait_pair(j, e, turn ^ (uint32_t)u);
                        if (!ok) break;
                        if (j + 1 < nt) scores(0, e, e);
                        ok = values(0, u, e, (uint32_t)j, turn);
                        if (!ok) break;
                        commit(pvdone(u));
                        commit(empty(e));
                    }
                }
            }
            if (!ok) {
                if (lane == 0) {
                    atomicOr(p.err, PAGED_WAIT);
                    *abort_flag = 1;
                }
                commit(drain);   // what was issued ends before the tensor memory is freed
                for (uint32_t it = 0; it < TC_POLL_LIMIT; it++)
                    if (__any_sync(0xffffffffu, bar_try(drain, 0))) break;
            }
            __syncwarp();
        } else if (warp == 2 && nt > 0 && key0(nt - 1) + KT > c.len) {
            // V rows past the last key: whatever the page holds there becomes 0
            const int e = nt % L::NP, n16 = L::RB / 16;
            if (wait_warp(vhere, 0, abort_flag) && wait_warp(full(e), (uint32_t)(nt / L::NP) & 1u, abort_flag)) {
                uint8_t* v = sm + L::OFF_RING + (size_t)e * 2 * L::ENTRY;
                for (int at = 0; at < L::ATOMS; at++)
                    for (int k = (c.len - key0(nt - 1)) * n16 + lane; k < KT * n16; k += 32)
                        *(uint4*)(v + (size_t)at * KT * L::RB + k * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(vclear);
            }
        }
        tc_fence_before();
        __syncthreads();
        if (warp == 1) {
            tc_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        if ((warp - 4) / 4 < halves) {
            const int t = (warp - 4) / 4, q = warp & 3, r = 128 * t + 32 * q + lane;
            const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16), to = tl + L::TM_O + (uint32_t)t * 128;
            const int pos = c.total - c.n + (c.r0 + min(r, c.rows - 1)) / a.group;
            const int see_hi = min(c.len, pos + 1), see_lo = p.window ? pos - p.window + 1 : 0;
            float mref = NEG_INF, l = 0.0f;   // reference (a maximum less BIAS), sum of the weights
            bool ok = true;
            for (int j = 0; j < nt && ok; j++) {
                const int n = halves * j + t, b = n & 1;   // the scores' number, their buffer
                const uint32_t ts = tl + (uint32_t)b * KT;
                if (!bar_wait_short_warp(sfull(b), (uint32_t)n >> 1 & 1u, abort_flag)) { ok = false; break; }
                // With one row tile a warp may be a whole tile ahead of the others, whose weights the product before still
                // needs. Key tile j's product completes phase j / 2 of barrier j & 1; every warp takes each phase in turn (this
                // one long done, so that the wait for the next is never satisfied by the phase before it).
                if (halves == 1 && j > 1 && !bar_wait_short_warp(pvdone(j & 1), (uint32_t)(j - 2) >> 1 & 1u, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t x[4][32];
#pragma unroll
                for (int k = 0; k < 4; k++) tmem_ld32(ts + 32u * k, x[k]);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 4; k++) bind32(x[k]);
                const int k0 = key0(j);
                const bool whole = k0 + KT <= c.np || (k0 + KT <= min(c.len, c.p0 + 1) && (!p.window || k0 > c.p1 - p.window));
                if (!whole) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int at = k0 + 32 * k;   // bit i: the row sees key at + i
                        const uint32_t seen = (below(see_hi - at) & ~below(see_lo - at)) | below(c.np - at);
                        if (seen != 0xffffffffu) {
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (!(seen >> i & 1u)) x[k][i] = __float_as_uint(NEG_INF);
                        }
                    }
                    asm volatile("" ::: "memory");   // keeps the tests out of the tiles that need none
                }
                float mx[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    mx[k] = __uint_as_float(x[k][0]);
#pragma unroll
                    for (int i = 1; i < 31; i += 2) mx[k] = max3(mx[k], __uint_as_float(x[k][i]), __uint_as_float(x[k][i + 1]));
                    mx[k] = max2(mx[k], __uint_as_float(x[k][31]));
                }
                const float top = max2(max2(mx[0], mx[1]), max2(mx[2], mx[3])) * a.c;
                // Raise the reference maximum of the warp's rows when one of them needs it. A score that is NaN or has
                // overflowed makes the row's reference NaN, and with it all that the row gives: the polynomial would take the
                // exponent of such a score for a small one.
                if (__any_sync(0xffffffffu, !(top <= mref + (TAU<T> + BIAS<T>)))) {
                    float up = max2(mref, top - BIAS<T>);
                    if (up == -NEG_INF) up = __int_as_float(0x7fffffff);
                    if (j > 0) {
                        // O must be at rest. With two row tiles it is: these scores were issued after the product before
                        if (halves == 1) {
                            ok = bar_wait_short_warp(pvdone((j - 1) & 1), (uint32_t)(j - 1) >> 1 & 1u, abort_flag);
                            if (!ok) break;
                            tc_fence_after();
                        }
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
                const uint64_t c2 = f2pack(a.c, a.c), ref2 = f2pack(ref, ref);
                uint64_t sum = 0;   // two partial sums
                auto weights = [&](auto tested) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            uint64_t e = ffma2(f2pack(__uint_as_float(x[k][2 * i]), __uint_as_float(x[k][2 * i + 1])), c2, ref2);
                            if (!decltype(tested)::value && i % EVERY == EVERY - 1) e = ex2_pair(e);
                            else e = f2pack(ex2(f2lo(e)), ex2(f2hi(e)));
                            sum = fadd2(sum, e);
                            w[i] = pack2<T>(f2lo(e), f2hi(e));
                        }
                        tmem_st16u(ts + 16u * k, w);
                        if (k & 1) {   // half of the tile's weights: their product may start
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(pfull(b, k >> 1));
                        }
                    }
                };
                if (whole) weights(std::false_type{});
                else weights(std::true_type{});
                l += f2lo(sum) + f2hi(sum);
            }
            if (ok && nt > 0) {   // (two row tiles: one phase, after the last product)
                const int last = halves == 2 ? t : (nt - 1) & 1;
                ok = bar_wait_short_warp(pvdone(last), halves == 2 ? 0u : (uint32_t)(nt - 1) >> 1 & 1u, abort_flag);
            }
            tc_fence_after();
            const bool mine = r < c.rows;
            const int tok = (c.r0 + r) / a.group, head = h * a.group + (c.r0 + r) % a.group;
            const int64_t row = c.row0 + tok;
            const int64_t unit = ((int64_t)s * a.tiles + tile) * p.kv.n_head + h;
            float* part = p.part + unit * a.n_split * (a.row_tile * (D + 2));
            const float il = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            if (ok && n_act == 1) {
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
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float y[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) y[k] = __uint_as_float(o[i + k]) * il;
                        T* dst = (T*)p.out + row * p.out_stride + (int64_t)head * D + d + i;
                        const uint4 u = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]),
                                                   pack2<T>(y[6], y[7]));
                        if (a.vec_out) {
                            *(uint4*)dst = u;
                        } else {
                            const T* e = (const T*)&u;
#pragma unroll
                            for (int k = 0; k < 8; k++) dst[k] = e[k];
                        }
                    }
                }
                if (mine && p.lse)
                    p.lse[row * p.n_q_head + head] = (mref + log2f(l)) * LN2;   // (nothing seen: both -infinity)
            } else if (ok) {
                // Split results (f32, nt > 0) go through shared memory, where this row tile's queries are no longer needed, in
                // two halves of the columns, so that a warp's stores cover whole rows (512 tokens over 8192 keys: 47.9 -> 45.0
                // us; 16-bit outputs, half as wide, are faster straight from the registers): 16-byte pieces, swizzled by row.
                uint8_t* stage = sm + (size_t)(128 * t + 32 * q) * D * 2;
                auto place = [&](int fr, int piece) {
                    return (uint4*)(stage + fr * D * 2 + ((piece ^ (D >= 64 ? fr & 7 : (fr >> 1) & 3)) << 4));
                };
#pragma unroll 1
                for (int d0 = 0; d0 < D; d0 += D / 2) {
#pragma unroll 1
                    for (int d = 0; d < D / 2; d += 16) {
                        float o[16];
                        tmem_ld16(to + (uint32_t)(d0 + d), o);
                        tmem_wait_ld();
                        tmem_bind(o);
#pragma unroll
                        for (int k = 0; k < 16; k += 4)
                            *(float4*)place(lane, (d + k) / 4) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int m = 0; m < D / 8; m++) {
                        const int fr = (32 * m + lane) / (D / 8), pc = (32 * m + lane) % (D / 8), rr = 128 * t + 32 * q + fr;
                        if (rr < c.rows) *(uint4*)(part + ((int64_t)sp * a.row_tile + rr) * D + d0 + pc * 4) = *place(fr, pc);
                    }
                    __syncwarp();
                }
                if (mine)
                    *(float2*)(part + (int64_t)a.n_split * a.row_tile * D + 2 * ((int64_t)sp * a.row_tile + r)) =
                        make_float2(mref, l);
            } else if (lane == 0) {
                atomicOr(p.err, PAGED_WAIT);
                *abort_flag = 1;
            }
        }
        tc_fence_before();
        __syncthreads();
    }
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

bool launch_chunk_attention_tc(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s) {
    TcArgs a;
    a.p = p;
    if (!a.p.poll_limit) a.p.poll_limit = TC_SPIN_LIMIT;
    a.group = p.n_q_head / p.kv.n_head;
    a.row_tile = plan.row_tile;
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
    const int bit = 36 + (p.kv.kv_dtype == GSVCU_KV_F16 ? 0 : 3) + D / 64;   // 36 .. 41
    bool ok = false;
    pick_tc(p.kv.kv_dtype, D, [&](auto k, size_t smem) {
        ok = raise_smem(k, smem, ready, bit);
        if (ok) launch_pdl(k, dim3((unsigned)ctas), dim3(THREADS), smem, s, a);
    });
    return ok;
}

}  // namespace gsvcu
