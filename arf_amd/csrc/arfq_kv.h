// arfq_kv.h -- the 4-bit K/V cache: its layout in device memory, the batch description
// its kernels share and their launchers.
//
// A row (one token's K or V of one head, D = 32 NG values) is held as NG groups of a scale
// and 32 codes: d (f16, at most 8 significant bits) and q in [-8, 7], worth d * q.  8 bits
// times q's 3 (or a power of two) are at most 11: d * q is an f16 exactly, so MFMA operands
// made from the cache carry no rounding.
//
// Memory: pages of P tokens (P a multiple of 16), in each page one contiguous region per
// head, [K codes | V codes | K scales | V scales], shaped as the attention kernels' matrix
// operands, so that those load them into registers with no shuffle:
//   K codes   [P][4][NG] dwords.  Dword (key, h, g) holds values 32g+8h .. +7 of the row, code
//             + 8 of value e in nibble (e >> 1) + 4 * (e & 1): nibbles p and p + 4 are
//             neighbours, which one mask turns into a pair of f16.
//   V codes   [P / 4][16][4][NG] bytes.  Byte (b, c, key % 4, g) holds values 32g+c (low
//             nibble) and 32g+16+c: NG dwords have four keys of a matrix row.
//   K scales  [P][NG] f16;  V scales [P / 4][NG][4] f16 (a dword is a pair of keys).
#pragma once
#include "arfq_common.h"
#include "arfq_internal.h"

struct arfq_kv {
    int device = 0;
    int heads = 0, dim = 0, page = 0;
    int64_t pages = 0;
    uint8_t *data = nullptr;  // pages * heads regions
    size_t bytes = 0;
};

namespace arfq {

constexpr int KV_GROUP = 32;
constexpr int KV_PAGE_MAX = 256;
constexpr int KV_TILE = 16;  // keys that share a page: P is a multiple
constexpr int64_t KV_KEYS_MAX = (int64_t)1 << 29;    // of a sequence (max_pages * P)
// sequences of a call: each row of a write, and each item of the attention, looks through them, 64 at a time
constexpr int64_t KV_BATCH_MAX = 16384;
constexpr int64_t KV_ROWS_MAX = (int64_t)1 << 30;    // tokens * heads of a call
constexpr int KV_HEADS_MAX = 1024;

// byte offsets within a (page, head) region
struct KvLayout {
    int64_t region;       // bytes of a (page, head) region
    int off_v, off_ks, off_vs;
};
inline KvLayout kv_layout(int page, int dim) {
    const int codes = page * dim / 2, scales = page * (dim / KV_GROUP) * 2;
    return {2 * ((int64_t)codes + scales), codes, 2 * codes, 2 * codes + scales};
}

// Workgroups of a launch, 256 threads each: a dimension of a grid has fewer than 2^32 threads, so from 2^23
// workgroups on they lie in rows of that many (some of the last row have nothing to do).
constexpr int GRID_ROW = 1 << 23;
inline dim3 grid_of(int64_t blocks) {
    return blocks <= GRID_ROW ? dim3((unsigned)blocks) : dim3(GRID_ROW, (unsigned)((blocks + GRID_ROW - 1) / GRID_ROW));
}
__device__ __forceinline__ int block_of() { return (int)(blockIdx.y * GRID_ROW + blockIdx.x); }

// What every kernel of the cache takes: the cache and the batch.
struct KvArgs {
    uint8_t *data;
    int64_t region;
    int off_v, off_ks, off_vs;
    int heads, page, tiles;  // tiles = page / KV_TILE
    uint32_t page_bytes;     // of all heads: at most 1024 * 72 KB
    uint32_t tile_magic;     // ceil(2^32 / tiles); 0 for one tile a page
    uint32_t tile_mask;      // all bits for one tile a page; 0
    int n_pages;
    // the batch
    int batch, tokens;
    const int32_t *start, *len, *table;
    int max_pages;
};

// Page of 16-key tile `t` of a sequence.  t < 2^27 (32-bit positions), tiles <= 16: the product
// with the rounded-up reciprocal is off by less than t * tiles / 2^32 < 1/2 of a step.
__device__ __forceinline__ int kv_page_of(const KvArgs &a, int t) {
    return (int)(__umulhi((uint32_t)t, a.tile_magic) + ((uint32_t)t & a.tile_mask));
}

// Rows of sequences: start[b] .. start[b + 1] - 1.  `start` does not decrease; where it does, no sequence from
// there on has rows, nor has one whose rows leave the batch's: no two sequences share a row, and all rows lie in
// [0, tokens), whatever the array holds (the bounds on the attention's work list rest on that).

// First token and token count of sequence b, the first with start[b + 1] above some token (none before it
// decreases).
__device__ __forceinline__ void kv_seq(const KvArgs &a, int b, int &t0, int &n) {
    if (!a.start) {
        t0 = b;
        n = b < a.tokens ? 1 : 0;
        return;
    }
    t0 = a.start[b];
    const int t1 = a.start[b + 1];
    n = t0 >= 0 && t1 > t0 && t1 <= a.tokens ? t1 - t0 : 0;
}

// The same for 64 sequences, b in each lane of a wave (0 tokens from a.batch on; without a start a.tokens is no
// more than it).  ended: start has decreased before them; on return, among them too.
__device__ __forceinline__ void kv_seq64(const KvArgs &a, int b, bool &ended, int &t0, int &n) {
    t0 = b;
    n = b < a.tokens ? 1 : 0;
    if (!a.start) return;
    int t1 = t0 = 0;
    if (b < a.batch) {
        t0 = a.start[b];
        t1 = a.start[b + 1];
    }
    n = t0 >= 0 && t1 > t0 && t1 <= a.tokens ? t1 - t0 : 0;
    const uint64_t falls = __ballot(t1 < t0);
    if (!falls && !ended) return;
    if (ended || (falls & (((uint64_t)2 << (threadIdx.x & 63)) - 1))) n = 0;  // (at this lane or one before)
    ended = true;
}

hipError_t launch_kv_write(const KvArgs &a, int dim, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                           int dtype, hipStream_t s);
hipError_t launch_kv_read(const KvArgs &a, int dim, void *k, int64_t k_stride, void *v, int64_t v_stride, int dtype,
                          hipStream_t s);

// ---- attention (arfq_attn.hip, arfq_attn_mixed.hip) ----
// A work list (arfq_attn_list.h): the pieces it aims at, its items at most, those of tiles in more than one piece
// (`cut`), their rows' parts, [cut][heads][rows of a tile][dim + 4] (maximum, sum, -, -, values), and
// for each what the join takes: pieces (0: no item) and which of them, first row, rows, first token.
struct AttnListPlan {
    int target = 1, slots = 0, cut = 0, round = 1;
    size_t part_bytes = 0, join_bytes = 0;
};
struct AttnList {
    int target, slots, cut, round;  // round: items that give every compute unit a workgroup
    float *part;
    int4 *join;                     // null: no row has two pieces
};
struct AttnArgs {
    KvArgs c;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;  // elements between tokens
    int q_dtype, out_dtype;
    int group;  // q heads of a K/V head
    float scale, softcap;
    int window;  // 0: none
    int causal;
    int few_rows;         // sequences with at most so many rows are in `few` (16-row tiles), others in `many` (128)
    AttnList few, many;
};
struct AttnPlan {
    int few_rows = 0;
    AttnListPlan few, many;
    size_t ws_bytes = 0;  // few's parts, many's, few's join, many's
};
bool attn_dim_ok(int dim);
hipError_t launch_attn(const AttnArgs &a, int dim, hipStream_t s);
// both lists
hipError_t launch_attn_mixed(const AttnArgs &a, int dim, hipStream_t s);

}  // namespace arfq
