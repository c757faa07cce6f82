// paged.h -- host-side launchers of the paged-cache operators (internal to the library): appending keys
// and values with the position rotation (paged_append.cu) and attention of a chunk of new tokens over the
// paged cache (paged_attention.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/gsvcu.h"

namespace gsvcu {

// Bits of the operators' device status word (reported by gsvcu_sync).
enum { PAGED_BAD_PAGE = 1, PAGED_BAD_LENGTH = 2, PAGED_BAD_POSITION = 4, PAGED_WAIT = 8 };

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
};
void launch_kv_append(const KvAppendParams& p, cudaStream_t s);

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
    // failure-path tests (gsvcu_set_wait_fault): bytes that a pair's barrier expects beyond its copies, polls of its wait (0: the
    // usual limit)
    uint32_t fault_extra_tx = 0, poll_limit = 0;
};
// How one call is cut up, from the sizes alone; scratch it needs.
struct ChunkAttnPlan {
    bool tensor = false;   // the tcgen05 kernel (paged_attention_tc.cu)
    int row_tile = 0;      // packed rows (token x query head of one kv head) of a CTA
    int tiles = 0;         // row tiles per sequence (bound)
    int n_split = 0;       // key splits (bound)
    int key_tile = 0;      // keys of a tile
    int split_tiles = 0;   // key tiles of a split
    bool join_apart = false;   // the splits are joined by a kernel of its own, not by the last CTA
    size_t part_floats = 0, arrivals = 0;
};
ChunkAttnPlan chunk_attention_plan(const ChunkAttnParams& p);
// Kernels launched; 0: none (no tensor map, or no room for the shared memory). `ready`: the caller's record of the
// kernels whose shared-memory limit is raised on its device (zero at first; raising all 42 with the context would add
// 16 ms to it).
int launch_chunk_attention(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s);
bool launch_chunk_attention_tc(const ChunkAttnParams& p, const ChunkAttnPlan& plan, uint64_t* ready, cudaStream_t s);
template <typename K>
inline bool raise_smem(K kernel, size_t bytes, uint64_t* ready, int bit) {
    if (*ready >> bit & 1u) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return false;
    *ready |= (uint64_t)1 << bit;
    return true;
}

}  // namespace gsvcu
