// arfq_step.h -- what a serving step needs around the K/V cache: the kernels' arguments and their launchers
// (arfq_plan.hip, arfq_rope.hip, arfq_lora.hip, arfq_blocks.hip).
#pragma once
#include "arfq_kv.h"

namespace arfq {

// ---- arfq_plan.hip ----
constexpr int PLAN_PAGE_MAX = 65536;
hipError_t launch_kv_plan(const arfq_kv_step &s, hipStream_t stream);

// ---- arfq_rope.hip ----
constexpr int ROPE_DIM_MAX = 256, ROPE_HEAD_MAX = 1024, ROPE_AXES_MAX = 4;
template <int PAIRS>
struct RopePairsOf {
    double turns[PAIRS];  // of a pair, a position: freq / (2 pi), negative for the way back
    uint8_t axis[PAIRS];
};
using RopePairs = RopePairsOf<ROPE_DIM_MAX / 2>;
struct RopeArgs {
    int rot, dim, heads, tokens;
    const int32_t *positions;
    int64_t position_stride;
    const void *x;
    void *out;
    int64_t x_stride, out_stride;
    float gain;
    bool neighbours, x_f16, out_f16;
};
hipError_t launch_rope(const RopeArgs &a, const RopePairs &pairs, int cus, hipStream_t stream);

// ---- arfq_lora.hip ----
constexpr int64_t LORA_RANK_MAX = 256, LORA_ROWS_MAX = (int64_t)1 << 24;
struct LoraPlan {
    bool tiles = false;  // rows in tiles on the matrix cores; one by one on the vector unit otherwise
    bool one = false;    // rows one by one, both products in one launch
    int splits = 1;      // parts of k
    int k_part = 0;      // values of a part
    size_t ws_bytes = 0; // [splits][rows][rank] f32
};
LoraPlan lora_plan(int cus, const arfq_lora &l, int64_t rows, bool x_f16);
struct LoraArgs {
    arfq_lora l;
    const int32_t *ids;
    int rows;
    const void *x;
    bool x_f16;
    const float *base;
    float *out;
    int64_t base_stride, out_stride;
    float *h;  // the workspace
};
hipError_t launch_lora(const LoraArgs &a, const LoraPlan &p, int cus, hipStream_t stream);

// ---- arfq_blocks.hip ----
hipError_t launch_kv_bounds(const KvArgs &a, int dim, _Float16 *bounds, int cus, hipStream_t stream);

constexpr int64_t BLOCKS_MAX = 1 << 20;
// A call's rows go through in chunks of `rows`.  For each row of a chunk and K/V head the workspace holds the
// scores' keys of all blocks and the chosen blocks' pages, and then the parts of rows in pieces.
struct BlocksPlan {
    int rows = 0;     // of a chunk
    int tiles = 1;    // 16-row tiles of a row's group of q heads
    int pieces = 1;   // of a row's keys, at most
    int width = 0;    // chosen blocks of a row: min(count, max_pages)
    bool in_lds = false;  // the attention's workgroups choose, each for itself
    size_t off_table = 0, off_part = 0, ws_bytes = 0;
};
BlocksPlan blocks_plan(int cus, int heads, int dim, int page, int64_t tokens, int q_heads, int64_t max_pages, int64_t count);
struct BlocksArgs {
    AttnArgs a;  // of the whole call: cache, batch, q, out
    const _Float16 *bounds;
    int count, first, last;
    int32_t *chosen;  // or null
    char *ws;
};
hipError_t launch_blocks(const BlocksArgs &b, int dim, const BlocksPlan &p, int cus, hipStream_t stream);

}  // namespace arfq
