// dit_train_internal.hpp — shared definitions of the operators of dit_train.h.
#pragma once

#include "dit_internal.hpp"
#include "dit_train.h"

namespace awa {

struct NormFwd {
    const void* x;
    int64_t ldx;
    const float *w, *b;  // [K] or null
    float eps;
    void* y;
    int64_t ldy;
    float2* stats;  // [M] or null
    int M, K;
};
hipError_t launch_layer_norm(int dtype_x, int dtype_y, const NormFwd& a, hipStream_t s);

struct NormGrad {
    const void* dy;
    int64_t lddy;
    const void* x;
    int64_t ldx;
    const uint32_t* xs;  // scale words of 8-bit rows
    int64_t ld_xs;
    const float2* stats;
    const float* w;  // [K] or null
    void* dx;        // or null
    int64_t lddx;
    int dx_f32;      // dx fp32, else bf16
    float *dw, *db;  // [K] or null
    float* part;     // [groups][2][K], or null where neither is wanted
    int groups;      // workgroups
    int M, K;
};
// workgroups of the gradient's kernel, each of which leaves a row of partial sums
int norm_grad_groups(int M, int K);
hipError_t launch_layer_norm_grad(int dtype_dy, int dtype_x, const NormGrad& a, hipStream_t s);

struct GradWeight {
    const void* dy;  // [M][N]
    int64_t lddy;
    const uint8_t* q;  // [M][kp] e4m3
    const uint32_t* s;
    int64_t ld_s;
    void* dw;  // [N][K]
    int64_t ldw;
    float* db;  // [N] or null
    int add, w_f32;
    float* part;  // of the divided tiles: [tile][split] of a tile's sums and db's
    // filled by launch_grad_weight: tiles, how many of them are whole, the others' parts and the rows of one
    int n_tiles, k_tiles, whole, splits, rows_per;
    int M, N, K, kp;
};
// how the work is divided, for the workspace and the launch alike
struct GradWeightPlan {
    int tile, whole, splits, rows_per;
    int64_t work;  // bytes
};
GradWeightPlan grad_weight_plan(int dtype_dy, int M, int N, int K);
hipError_t launch_grad_weight(int dtype_dy, GradWeight& a, hipStream_t s);

// ---- attention to states of another length

// A block of queries and the keys that a workgroup takes it over: columns c = 0 .. of a block are
// query rows q0 + c / pack of the heads head0 + c % pack (head0 the work item's; pack 1: a head's rows).
struct CrossItem {
    int q0, cols;  // first query row, columns
    int k0, kn;    // first key row, keys
    int part;      // slot of the partial results, -1: the only part, written in place
    int first;     // 1: the block's first run of keys
    int group;     // head group, in a table by workgroup (below)
    int pad;
};
// A block whose keys are split: its parts are slots part0 .. part0 + parts - 1.
struct CrossJoin {
    int q0, cols, part0, parts;
};
// Queries of the gradient of keys: up to CROSS_QT rows of a sequence.
constexpr int CROSS_QT = 64;
struct CrossUnit {
    int q0, rows;
};
// Keys of a block: with 64, and their four waves' tiles, two workgroups share a CU, so that one's products fill the
// other's waits (gradients of 16384 queries x 384 keys x 20 heads 304 us with 128 keys in eight waves, 292 so; of four clips
// of up to 5440 x 512 363 and 308).
constexpr int CROSS_KEYS = 64;
// A block of keys and the run of its units (of every head that shares the key head: units ahead of
// heads) that a workgroup takes.
struct CrossKeys {
    int k0, kn;              // first key row, keys
    int unit0, units;        // of its sequences, in the units' table
    int first, count;        // the run, among units x shared heads
    int part;                // slot of partial sums, -1: the only one
    int group;               // key head, in a table by workgroup
};
struct CrossKeyJoin {
    int k0, kn, part0, parts;
};

// The items are a table by workgroup, with entries for every head group and in the order that they should start, where that
// is not too long (CROSS_LISTED), or else one for all head groups.  By workgroup: the XCDs, which take workgroups in turn, get
// lists of equal work, each of neighbouring heads and sequences (whose keys one L2 then holds), the longest first; entries
// without columns (keys) fill the shorter lists.  Gradients of four clips of up to 5440 x 512 297 us by equal counts, 281 so.
constexpr int CROSS_LISTED = 1 << 16;
struct CrossQueries {
    int pack = 1, block = 0;  // heads in a block, columns of a block
    int most_keys = 0;        // of an item
    int n_items = 0, n_joins = 0, n_parts = 0;
    int n_listed = 0;         // entries of a table by workgroup, 0: items is one for all head groups
    const CrossItem* items = nullptr;
    const CrossJoin* joins = nullptr;
};
struct CrossKeySide {
    int n_items = 0, n_joins = 0, n_parts = 0;
    int n_listed = 0;
    const CrossKeys* items = nullptr;
    const CrossKeyJoin* joins = nullptr;
    const CrossUnit* units = nullptr;
};

struct CrossArgs {
    const char *q, *k, *v, *out, *dout;
    char *o, *dq, *dk, *dv;
    // strides in bytes
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head, dout_row, dout_head;
    int64_t o_row, o_head, dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
    const uint8_t* mask;
    float scale, c;  // c = scale log2(e)
    float* lse;
    int64_t ld_lse;
    int heads, kv_heads, head_d;
    int whole;  // DIT_CROSS_WHOLE
    CrossQueries qs;
    CrossKeySide ks;
    float *qpart, *kpart;  // partial results
    // left by the gradient of the queries for that of the keys, [heads][ld_dsum]: rowsum(dout out), and lse in
    // powers of two (infinite for a row without keys, so that its probabilities are 0)
    float *dsum, *lse2;
    int64_t ld_dsum;
};
hipError_t launch_cross_forward(int dtype, const CrossArgs& a, hipStream_t s);
hipError_t launch_cross_grad_queries(int dtype, const CrossArgs& a, hipStream_t s);  // first: it leaves dsum
hipError_t launch_cross_grad_keys(int dtype, const CrossArgs& a, hipStream_t s);
// floats of a partial block of queries (of a head group) and of keys (of a key head)
__host__ __device__ inline int64_t cross_query_part(int block, int head_d) { return (int64_t)block * (head_d + 2); }
__host__ __device__ inline int64_t cross_key_part(int block, int head_d) { return (int64_t)block * 2 * head_d; }

}  // namespace awa
