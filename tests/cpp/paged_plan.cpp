// Prints how one call of chunk attention over the paged cache is cut up (csrc/paged.h), for the host-side tests: no GPU.
//   paged_plan kv_dtype head_dim n_kv_head n_q_head n_seq max_pages n_rows max_chunk max_kv window scale
#include <stdio.h>
#include <stdlib.h>

#include "../../gsv.cpp_b200/csrc/paged.h"

int main(int argc, char** argv) {
    if (argc != 12) return 2;
    gsvcu::ChunkAttnParams p;
    p.kv.kv_dtype = atoi(argv[1]);
    p.kv.head_dim = atoi(argv[2]);
    p.kv.n_head = atoi(argv[3]);
    p.n_q_head = atoi(argv[4]);
    p.batch.n_seq = atoi(argv[5]);
    p.batch.max_pages = atoi(argv[6]);
    p.batch.n_rows = atoi(argv[7]);
    p.batch.max_chunk = atoi(argv[8]);
    p.batch.max_kv = atoi(argv[9]);
    p.window = atoi(argv[10]);
    p.scale = (float)atof(argv[11]);
    const gsvcu::ChunkAttnPlan c = gsvcu::chunk_attention_plan(p);
    printf("{\"tensor\": %d, \"row_tile\": %d, \"tiles\": %d, \"n_split\": %d, \"dealt\": %d, \"unpack_pages\": %d, \"ctas\": %lld}\n",
           c.tensor, c.row_tile, c.tiles, c.n_split, c.dealt, c.unpack_pages, (long long)gsvcu::chunk_attention_ctas(p, c));
    return 0;
}
