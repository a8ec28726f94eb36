// Attention of T drafted tokens per sequence over a paged cache that already
// holds their K/V rows behind the context (positions ctx_len .. ctx_len+T-1).
#pragma once

#include <cuda.h>  // CUtensorMap (types only; the encoder is resolved at run time)

#include "kv_cache.cuh"
#include "wait_errors.cuh"

namespace sb {

struct TreeAttnArgs {
    KvCacheArgs c;
    const void *q = nullptr;  // [B][T][n_heads][hd], scaled; token row b*T+t at (b*T+t)*ldq
    long long ldq = 0;
    int bf16 = 0;             // element type of q and out: bf16 or f32
    int B = 0, T = 0, n_heads = 0, rep = 0;  // rep = n_heads / n_kv
    const int *ctx_len = nullptr;  // [B]
    const int *n_new = nullptr;    // [B] or null (T): tokens t >= n_new[b] do not exist
    // Bit j of row i: token i sees token j.  [T][mask_words] (mask_ld 0) or one
    // such block per sequence (mask_ld words apart); null: j <= i.
    const unsigned long long *mask = nullptr;
    long long mask_ld = 0;
    int mask_words = 0;
    void *out = nullptr;      // [B][T][n_heads][hd]
    int n_splits = 1;
    float *part = nullptr;          // n_splits > 1: [tiles][n_splits][rows][hd], unnormalised outputs
    float2 *ml = nullptr;           // n_splits > 1: [tiles][n_splits][rows], their maxima and sums
    // Pages of a multiple of eight positions: K and V as [rows][hd] tensors whose
    // boxes are box_rows rows of 128 bytes (64 of a 64-byte row), swizzled.
    // box_rows 0: rows are copied one by one.
    int box_rows = 0;
    CUtensorMap tmk, tmv;
    unsigned *errors = nullptr;  // wait_errors.cuh
};

// How a call divides its work: rows of one kv head per CTA, tiles of them, and
// the context splits.
struct TreeAttnPlan {
    int rows = 16, row_tiles = 1, n_splits = 1;
    size_t part_floats(const TreeAttnArgs &a) const {
        return (size_t)a.B * a.c.pg.n_kv * row_tiles * n_splits * rows * a.c.hd;
    }
};
TreeAttnPlan tree_attn_plan(const TreeAttnArgs &a, int max_len);
int tree_splits(long long base, int tiles, int resident = 1);
// Fills box_rows (at most max_rows) and the tensor maps where the pages allow.
int tree_tensor_maps(TreeAttnArgs &a, int max_rows);
// Few rows per kv head over a bf16 or int8 cache (attention_tree_rows.cu).
bool tree_attn_rows_wanted(const TreeAttnArgs &a);
TreeAttnPlan tree_attn_rows_plan(const TreeAttnArgs &a, int max_len);
int tree_attn_rows_launch(const TreeAttnArgs &a, cudaStream_t st);
// Many rows per kv head over a bf16 or int8 cache (attention_tree_tc.cu).
bool tree_attn_tc_wanted(const TreeAttnArgs &a);
TreeAttnPlan tree_attn_tc_plan(const TreeAttnArgs &a, int max_len);
int tree_attn_tc_launch(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st);
int tree_attn_launch(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st);

}  // namespace sb
