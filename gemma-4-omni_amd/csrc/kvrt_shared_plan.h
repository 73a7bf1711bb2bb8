// kvrt_shared_plan.h — how a call of shared-prefix attention is divided: which of its kernels runs
// it, on which tiles and key ranges. Host arithmetic alone, from the call's sizes, so that it can
// be checked without a GPU. It takes 0.3 us for one session, 2 for four and for a chunk, 7 for 64
// and 12 for 64 of 32768 rows, in every call that is not a graph's.
#pragma once

#include <algorithm>
#include <cmath>

#include "kvrt_shared.h"

namespace kvrt {

constexpr int kMaxSharedParts = 128;  // key ranges of an item, and of the prefix
constexpr double kMaxSharedUnits = 1 << 23;  // workgroups

// Bytes of the partials of `rows` rows: outputs, then (max, sum).
inline size_t shared_part_bytes(int64_t rows, int64_t parts, int D) {
    return parts == 1 ? 0 : (size_t)rows * parts * (D * 4 + 8) + 256;
}

// How a call's rows and keys are divided (SharedArgs), its partials within `room` bytes: pre_keys
// of the prefix are seen, and own[i] of item i's rows. joined: each item's workgroups read the
// prefix too, as the head of its own keys. The shortest time of a simple model is taken, and
// returned, us: a launch lasts as long as its longest unit, and at least as its units' work
// shared by 256 CUs (two and more on one overlap in part: kShare); a unit takes some us a key
// tile and kUnit of its own; partials are joined by a second launch. The constants were fitted to
// 1152 measured calls (1 to 16 items of 1 to 512 rows, 512 to 33768 keys), which they met with
// 4 to 9 % (rms); the kernels have since become up to 15 % faster (head_dim 512, calls past the
// caches), without a new fit.
inline double shared_plan(SharedArgs &a, int D, int64_t pre_keys, const int64_t *own, bool joined, size_t room) {
    const int hkv = a.kv.kv_heads, tile = shared_tile(D), dim = D == 64 ? 0 : D == 128 ? 1 : D == 256 ? 2 : 3;
    const int64_t per_item = (int64_t)a.group * a.qn, rows = per_item * a.n_items;
    const auto tiles_of = [](int64_t keys) { return (keys + kSharedKeys - 1) / kSharedKeys + (keys % kSharedKeys > 1 ? 1 : 0); };
    const auto cost = [&](int64_t r) {
        // up to 16 rows, up to 64, up to 128 (head_dim 64 and 128)
        static const double us[3][4] = {{0.75, 0.8, 1.0, 1.9}, {0.8, 1.0, 1.2, 2.4}, {1.2, 1.5}};
        return us[r <= 16 ? 0 : r <= 64 ? 1 : 2][dim];
    };
    // (by head_dim 64, 128, 256, 512; a launch alone is 1.5 us)
    static const double kUnits[4] = {1.1, 4.3, 4.2, 7.1}, kJoins[4] = {3.8, 1.1, 1.4, 0.1}, kShares[4] = {0.6, 0.6, 0.87, 0.89};
    static const double kParts[4] = {0.02, 0.01, 0.03, 0.06};  // us a part of a row
    constexpr double kLaunch = 1.5, kJoinBytes = 3.2e6;  // us, bytes a us
    const double kUnit = kUnits[dim], kBytes = D == 512 ? 4.6e6 : 5.2e6;
    a.own_tiles = (int)((per_item + tile - 1) / tile);
    a.joined = joined;
    a.pre_tiles = a.prefix_slot < 0 || a.joined ? 0 : (int)((rows + tile - 1) / tile);
    const int64_t pre = tiles_of(pre_keys);
    int64_t items[kMaxItems], most = 1;
    for (int i = 0; i < a.n_items; ++i) {
        items[i] = std::max<int64_t>(1, tiles_of(own[i]) + (a.joined ? pre : 0));
        most = std::max(most, items[i]);
    }
    const double cp = cost(std::min<int64_t>(rows, tile)), co = cost(std::min<int64_t>(per_item, tile));
    const double share = kShares[dim] / 256;
    int64_t all_own = 0;
    for (int i = 0; i < a.n_items; ++i) all_own += own[i];
    // (the 64-row tiles of one item that head_dim 256 and 512 have do not meet in the L2)
    const double floor = (double)(all_own * (D >= 256 ? a.own_tiles : 1) + pre_keys) * hkv * D * 4 / kBytes;
    const bool ragged = !a.joined && a.own_tiles == 1;
    // ranges of an item of t tiles: even ones, or of `per` tiles where items differ
    const auto ranges = [](int64_t t, int64_t per) { return std::max<int64_t>(1, (t + per - 1) / per); };
    double best = 1e30;
    int64_t best_pre = 1, best_per = most;
    for (int64_t per = 1;; per = std::min(most, per + 1 + per / 4)) {
        const int64_t splits = ranges(most, per);
        if (splits <= kMaxSharedParts) {
            double work = 0, units = 0;
            for (int i = 0; i < a.n_items; ++i) {
                const double u = (double)(ragged ? ranges(items[i], per) : splits);
                units += u * a.own_tiles;
                work += (items[i] * co + u * kUnit) * a.own_tiles;
            }
            for (int64_t pp = 1;; pp = std::min(pre, pp + 1 + pp / 4)) {
                const int64_t ps = a.pre_tiles ? ranges(pre, pp) : 0;
                const double c = (units + a.pre_tiles * ps) * hkv / 256;  // units on a CU, whole ones
                if (ps <= kMaxSharedParts && (c <= kMaxSharedUnits / 256 || splits + ps <= 2) &&
                    shared_part_bytes(rows * hkv, splits + ps, D) <= room) {
                    double all = hkv * (work + a.pre_tiles * (pre * cp + ps * kUnit)) * share;
                    if (c > 1) all *= std::ceil(c) / c;
                    const double longest = std::max((double)std::min(per, most) * co, a.pre_tiles ? pp * cp : 0.0) + kUnit;
                    const int64_t parts = splits + ps;
                    double t = std::max(all, longest);
                    t = std::max(t, floor) + kLaunch;
                    if (parts > 1) t += kJoins[dim] + kParts[dim] * parts + (double)rows * hkv * parts * D * 8 / kJoinBytes;
                    if (t < best) best = t, best_pre = ps, best_per = per;
                }
                if (!a.pre_tiles || pp >= pre) break;
            }
        }
        if (per >= most) break;
    }
    a.pre_splits = (int)best_pre;
    a.own_splits = (int)ranges(most, best_per);
    a.own_per = a.own_wgs = 0;
    if (ragged && a.own_splits > 1) {
        a.own_per = (int)best_per;
        for (int i = 0; i < a.n_items; ++i) a.own_wgs += (int)ranges(items[i], best_per);
    }
    a.parts = a.pre_splits + a.own_splits;
    return best;
}

// The shape of a call on the prefill's tiles (PrefillArgs: row blocks and key parts of a
// workgroup, key ranges), for items whose rows see `keys` keys at most, `all` together, and its
// time, us: the chain of 32-key blocks that a wave walks, in rounds of 256 workgroups that
// overlap where LDS holds more than one to a CU, and the merge of ranges. Fitted to 5000 calls
// (1 to 8 items of 16 to 2200 rows, 300 to 20000 keys, every shape, 1 to 32 ranges), which the
// times meet with 4 to 8 % (rms); the shape taken is 1.5 % slower than the best on average, the
// prefill's rule for shorter chunks 10 %.
inline double chunk_shape(SharedChunkArgs &a, int D, int64_t keys, int64_t all, size_t room) {
    struct Shape {
        int rw, parts;
        double block, paged, more;  // us a block, the same for PAGED, ... times workgroups on a CU
        double base, merge, bytes;  // us, us, bytes a us of the partials
    };
    static const Shape kShapes[4][4] = {
        {{4, 1, 0.67, 0.85, 0.62, 5.7, 2.3, 3.1e6}, {2, 2, 0.67, 0.9, 0.65, 6.3, 2.2, 2.7e6},
         {2, 4, 0.96, 1.2, 1.0, 6.9, 1.9, 1.6e6}, {1, 4, 0.74, 0, 0.76, 6.0, 2.1, 1.9e6}},
        {{4, 1, 0.78, 1.0, 0.73, 7.2, 2.0, 3.6e6}, {2, 2, 0.82, 1.08, 0.75, 7.5, 1.9, 3.0e6},
         {2, 4, 1.25, 1.55, 1.0, 8.5, 1.6, 2.0e6}, {1, 4, 1.05, 0, 1.0, 7.2, 1.3, 1.6e6}},
        {{4, 1, 1.19, 1.42, 1.0, 9.0, 2.2, 3.9e6}, {2, 2, 1.25, 1.55, 1.0, 11.1, 1.1, 2.9e6}},
        {{4, 1, 2.0, 2.25, 1.0, 15.0, 1.0, 4.4e6}},
    };
    const int hkv = a.kv.kv_heads, dim = D == 64 ? 0 : D == 128 ? 1 : D == 256 ? 2 : 3;
    const bool paged = a.kv.layout == KVRT_LAYOUT_PAGED;
    const int64_t rows = (int64_t)a.group * a.qn, blocks = (keys + kPfKeys - 1) / kPfKeys;
    const double read = (double)all * hkv * D * 4 / 5.2e6;
    double best = 1e30;
    for (const Shape &s : kShapes[dim]) {
        const int64_t tiles = s.rw ? (rows + 32 * s.rw - 1) / (32 * s.rw) : 0;
        if (s.rw == 0 || (paged && s.paged == 0) || tiles > 65535) continue;  // (a grid's third dimension)
        for (int64_t nks = 1; nks == 1 || (nks <= 32 && nks * 2 <= blocks); nks += 1 + nks / 4) {
            if (shared_part_bytes(rows * a.n_items * hkv, nks, D) > room) break;
            const int64_t chain = ((blocks + nks - 1) / nks + s.parts - 1) / s.parts;
            const int64_t round = (tiles * hkv * a.n_items * nks + 255) / 256;
            const double walk = chain * (paged ? s.paged : s.block) * std::max(1.0, round * s.more);
            // (up to head_dim 128 they overlap in part)
            double t = std::max(walk, read) + (D <= 128 ? 0.2 : 0.0) * std::min(walk, read) + s.base;
            if (nks > 1) t += s.merge + (double)rows * a.n_items * hkv * nks * D * 8 / s.bytes;
            if (t < best) best = t, a.row_waves = s.rw, a.key_parts = s.parts, a.n_ksplit = (int)nks;
        }
    }
    return best;
}

// Divides a call for the kernels that take it: `a` and, with tiles_ok, `p` hold everything but the
// division. True: p runs it, on the prefill's tiles; else a. own[i]: rows of item i that its
// queries see, pre_keys: of the prefix. Partials take `room` bytes at most (a division that
// leaves none is always among them).
inline bool plan_shared_call(SharedArgs &a, SharedChunkArgs &p, int D, bool tiles_ok, int64_t pre_keys, const int64_t *own,
                             size_t room) {
    // the prefix's keys once for the rows of all items, or for each item with its own keys
    // (also where no row sees the prefix now: a replay may find it otherwise)
    const bool shared = a.prefix_slot >= 0;
    double time = shared_plan(a, D, pre_keys, own, shared, room);
    if (shared && pre_keys > 0) {
        SharedArgs apart = a;
        const double t = shared_plan(apart, D, pre_keys, own, false, room);
        if (t < time) a = apart, time = t;
    }
    // Or, without masks, on the prefill's tiles: 32 rows a wave, as chunks have them. us a call,
    // joined / apart / on the prefill's tiles, prefix 4096 and 100 rows each, by rows of an
    // item and KV head: 16 items, 8 KV heads of 128: 1 row 48 / 12 / 28, 16 49 / 27 / 29, 64
    // 61 / 54 / 43, 256 142 / 192 / 112; 4 items, one KV head of 512: 1 row 16 / 18 / 27, 128
    // 38 / 35 / 41, 512 65 / 74 / 57.
    if (!tiles_ok) return false;
    int64_t keys = 0, all = pre_keys;  // most keys that the rows of a tile see; all of them
    for (int i = 0; i < a.n_items; ++i) keys = std::max(keys, own[i]), all += own[i];
    keys += pre_keys;
    if (a.window > 0) keys = std::min<int64_t>(keys, a.window + 15);
    return chunk_shape(p, D, keys, all, room) < time;
}

}  // namespace kvrt
