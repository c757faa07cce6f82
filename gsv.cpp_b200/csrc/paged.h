// paged.h -- host-side launchers of the paged-cache operators (internal to the library): appending keys
// and values with the position rotation (paged_append.cu; with head norms or into 4 bits paged_append_norm.cu), reading
// them back (paged_read.cu) and attention of a chunk of new tokens over the paged cache (paged_attention.cu; over 4 bits
// paged_attention_q4.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/gsvcu.h"

namespace gsvcu {

// Bits of the operators' device status word (reported by gsvcu_sync).
enum { PAGED_BAD_PAGE = 1, PAGED_BAD_LENGTH = 2, PAGED_BAD_POSITION = 4, PAGED_WAIT = 8 };

// 4-bit caches: a kv_dtype names the type of the rows beside it too.
inline bool is_q4(int kv_dtype) { return kv_dtype == GSVCU_KV_Q4_F16 || kv_dtype == GSVCU_KV_Q4_BF16; }
inline int row_type(int kv_dtype) {
    return kv_dtype == GSVCU_KV_Q4_F16 ? GSVCU_KV_F16 : kv_dtype == GSVCU_KV_Q4_BF16 ? GSVCU_KV_BF16 : kv_dtype;
}
inline size_t type_size(int kv_dtype) { return kv_dtype == GSVCU_KV_F32 ? 4 : 2; }   // (of a row's element)

// The cache: pages [page][n_layer][K, V][n_head][PAGE][head_dim] of kv_dtype, seen at one layer.
struct PagedView {
    void* pool = nullptr;
    int kv_dtype = GSVCU_KV_F16;
    int n_page = 0, n_layer = 0, layer = 0, n_head = 0, head_dim = 0;
};
// The batch: sequence s has the packed rows [row_start[s], row_start[s + 1]) and kv_len[s] keys.
struct ChunkView {
    const int32_t* row_start = nullptr;
    const int32_t* kv_len = nullptr;
    const int32_t* table = nullptr;
    int n_seq = 0, max_pages = 0, n_rows = 0, max_chunk = 0, max_kv = 0;
};

struct KvAppendParams {
    PagedView kv;
    ChunkView batch;
    int row_dtype = GSVCU_KV_F32;   // type of the q / k / v rows
    int n_q_head = 0;
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    int64_t q_stride = 0, k_stride = 0, v_stride = 0;   // elements between rows
    const float *cos = nullptr, *sin = nullptr;          // [n_pos][rot / 2]
    int n_pos = 0, rot = 0, pairs = 0;
    const int32_t* pos = nullptr;   // rotation position of every row; null: the cache position
    void* q_out = nullptr;          // rotated q in kv_dtype
    int64_t q_out_stride = 0;
    int32_t* err = nullptr;
    const float *q_norm = nullptr, *k_norm = nullptr;   // [head_dim] weights of the head norms, null: none
    float eps = 0.0f;
};
void launch_kv_append(const KvAppendParams& p, cudaStream_t s);
void launch_kv_append_norm(const KvAppendParams& p, cudaStream_t s);   // head norms and 4-bit caches

struct KvReadParams {
    PagedView kv;
    ChunkView batch;
    int row_dtype = GSVCU_KV_F32;
    void *k = nullptr, *v = nullptr;
    int64_t k_stride = 0, v_stride = 0;   // elements between rows
    int32_t* err = nullptr;
};
void launch_kv_read(const KvReadParams& p, cudaStream_t s);

struct ChunkAttnParams {
    PagedView kv;
    ChunkView batch;
    int n_q_head = 0;
    const void* q = nullptr;
    int64_t q_stride = 0;
    float scale = 1.0f;
    int window = 0;                    // 0: none
    const int32_t* prefix = nullptr;   // [n_seq], null: none
    void* out = nullptr;
    int64_t out_stride = 0;
    float* lse = nullptr;   // [n_rows][n_q_head] or null
    int32_t* err = nullptr;
    float* part = nullptr;       // scratch of chunk_attention_plan
    int32_t* arrived = nullptr;  // zero between launches
    void* unpacked = nullptr;    // pages of a 4-bit cache as F16 [n_seq][unpack_pages][K, V][n_head][PAGE][head_dim], their table
    int32_t* unpacked_table = nullptr;
    // failure-path tests (gsvcu_set_wait_fault): bytes that a pair's barrier expects beyond its copies, polls of its wait (0: the
    // usual limit)
    uint32_t fault_extra_tx = 0, poll_limit = 0;
};
// How one call is cut up, from the sizes alone; scratch it needs.
struct ChunkAttnPlan {
    bool tensor = false;   // the tcgen05 kernel (paged_attention_tc.cu)
    int row_tile = 0;      // packed rows (token x query head of one kv head) of a CTA
    int tiles = 0;         // row tiles per sequence (bound)
    int n_split = 1;       // key splits (bound)
    int key_tile = 0;      // keys of a tile
    int split_tiles = 0;   // key tiles of a split
    bool join_apart = false;   // the splits are joined by a kernel of its own, not by the last CTA
    int64_t ctas = 0;          // 4-bit caches, few rows: CTAs, and whether the pages are dealt out to them
    bool dealt = false;
    int unpack_pages = 0;      // pages per sequence of a 4-bit cache that are unpacked to F16 first (0: the kernel reads the 4 bits)
    size_t unpacked_floats = 0;
    size_t part_floats = 0, arrivals = 0;
};
ChunkAttnPlan chunk_attention_plan(const ChunkAttnParams& p);
// CTAs of the plan's largest launch (pages dealt out: at most 4 join a unit). A grid takes INT32_MAX.
inline int64_t chunk_attention_ctas(const ChunkAttnParams& p, const ChunkAttnPlan& c) {
    return (int64_t)p.batch.n_seq * c.tiles * p.kv.n_head * (c.dealt ? 4 : c.n_split);
}
ChunkAttnPlan chunk_attention_tc_plan(const ChunkAttnParams& p);   // (more than 32 packed rows of a 16-bit type, scale not 0)
// Bytes that unpacked pages may take.
constexpr int64_t UNPACK_LIMIT = (int64_t)2 << 30;
// Kernels launched; 0: none (no tensor map, or no room for the shared memory). `ready`: the caller's record (two words) of
// the kernels whose shared-memory limit is raised on its device (zero at first; raising the 42 of the first word with the
// context would add 16 ms to it).
int launch_chunk_attention(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s);
// 4-bit caches: their plan, and their kernels for few rows (kernels launched as above). `ready`: as above, a word of its own.
ChunkAttnPlan chunk_attention_q4_plan(const ChunkAttnParams& p);
int launch_chunk_attention_q4(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s);
bool launch_chunk_attention_tc(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s);
template <typename K>
inline bool raise_smem(K kernel, size_t bytes, uint64_t* ready, int bit) {
    if (*ready >> bit & 1u) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return false;
    *ready |= (uint64_t)1 << bit;
    return true;
}

}  // namespace gsvcu
