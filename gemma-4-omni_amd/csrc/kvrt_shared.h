// kvrt_shared.h — attention after a prefix that all sessions of a call share, with scores
// optionally capped by a tanh and biased by distance: arguments of its kernels.
#pragma once

#include "kvrt_internal.h"

namespace kvrt {

struct SharedArgs {
    KVView kv;
    Lengths len;
    const uint16_t *q;        // [n, Hq, Q, D] contiguous
    uint16_t *out;            // [n, Hq, Q, D] contiguous
    int32_t *err;
    const PrefixMask *pmask;  // prefix-attention masks by slot, or null
    const float *slopes;      // [Hq] bias by distance, or null
    float *part_o;            // partials [kv head][row][part][D], rows in (item, query, head) order
    float2 *part_ml;          // their (max, sum)
    float scale;              // scale * log2(e)
    float cap;                // cap * log2(e), 0: none
    float inv_cap;            // scale / cap
    int n_items, group, qn;
    int window;               // 0: none; otherwise below 2^30
    int capacity;             // lengths are taken as at most this
    int prefix_slot;          // -1: none
    // Units (workgroups): first those of the prefix alone, rows of all items in tiles of
    // kSharedTile<D> rows, keys in pre_splits ranges (pre_tiles 0: none); then those of
    // each item, its rows in own_tiles tiles, keys in own_splits ranges: its own keys, with
    // `joined` those of the prefix before them.
    // own_per > 0 (items of one tile): an item's keys go to ranges of that many key tiles,
    // own_splits at most, all items' to own_wgs units for each KV head.
    int pre_tiles, pre_splits, own_tiles, own_splits, joined;
    int own_per, own_wgs;
    int parts;                // partials of a row; 1: units write the answer
    int large;                // the rows of K and V seen are more than half the last cache
    int slots[kMaxItems];
};

// Rows of a tile: four waves of two 16-row blocks, one from head_dim 256 on, where two
// blocks' accumulators and queries would fill a wave's registers.
constexpr int shared_tile(int head_dim) { return head_dim <= 128 ? 128 : 64; }
constexpr int kSharedKeys = 32;  // keys of a staged tile

hipError_t launch_shared(const SharedArgs &a, int head_dim, hipStream_t s);       // and the join of its partials
hipError_t launch_shared_wide(const SharedArgs &a, int head_dim, hipStream_t s);  // head_dim 256, 512

}  // namespace kvrt
