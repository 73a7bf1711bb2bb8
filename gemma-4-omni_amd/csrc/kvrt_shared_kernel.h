// kvrt_shared_kernel.h — attention of many sessions behind one shared prefix (gfx950).
//
// A session sees the prefix slot's P rows and then its own L: query row i of Q sits at
// position P + L - Q + i, and the softmax runs over both. Scores are
//   s = f(q . k * scale) + slope_h * (key - position),   f(x) = x or cap * tanh(x / cap)
// in fp32, weights 2^(s log2 e - m) with a running max m, and the sum and the products
// with V accumulate in fp32; weights enter P V as two bf16 terms (2^-17 relative: one
// term's 2^-9 would show in the bf16 outputs of few-key rows).
//
// Why units: the prefix's keys are the same for every session, so a workgroup takes up to
// shared_tile(D) rows of all sessions (query heads of one KV head) over a range of them and
// reads each key once per tile of rows, where a decode per session reads it once per session.
// A session's own keys go to workgroups of their own. Each unit leaves (max, sum, output) of
// its rows, which a second launch joins by their maxima. Where a session's rows nearly fill a
// tile, or one launch is all that a short call is worth, its units take the prefix's keys and
// its own in one walk (`joined`); the host weighs the two (shared_plan). Chunks without masks
// have the prefill's 32-row tiles instead (kvrt_shared_chunk.hip).
//
// A workgroup is four waves that stage 32-key tiles of K and V together by LDS DMA, STAGES of
// them in flight (three, four at head_dim 256 and six at 128 took as long; two at 512, which
// fill the LDS), one barrier per tile.
// With more than 16 rows (WIDE) a wave has up to two blocks of 16 rows and all dims of their
// outputs; with up to 16 rows every wave computes the scores of all of them, and a quarter of
// the dims: the scores' 2 D/32 matrix instructions are cheap beside the tile's bytes, and
// waves need neither exchange nor join anything.
//   S^T (16 keys x 16 rows) = K Q^T    D/32   v_mfma_f32_16x16x32_bf16, for two key halves
//   O^T (16 dims x 16 rows) += V^T P^T  2      v_mfma_f32_16x16x32_bf16 per 16 dims
// Lane layouts: A[row l%16][k 8(l/16)+j], B[k 8(l/16)+j][col l%16], D[row 4(l/16)+i][col
// l%16]. The second product's inner index is free: k = 8(l/16)+j is key 16(j/4) + 4(l/16)
// + j%4, the keys whose weights the lane holds, so weights go from one product's result
// to the other's operand in their registers; V is read transposed (ds_read_b64_tr_b16).
//
// A DMA instruction leaves 1 KiB: rows ins, ins + D/16, ... of the tile one after another.
// Instructions lie 1 KiB and a padding apart, 16 bytes for K and 32 for V, so that 16 lanes
// that read one 16-byte chunk of 16 rows (K), and 32 that read 32 bytes of 8 rows (V), find
// each of the 64 banks once, and every operand's address is one register (at head_dim 64
// and 128 two, by kx) and a constant.
//
// What bounds it (kernel times under the profiler): with many sessions or keys the bytes (64
// sessions, one row each, 8 KV heads of 128, behind 4096 rows: 245 MB in 48.3 us, 5.1 TB/s, and
// 4.6 us of joins; 16 paged ones behind 1024: 119 MB in 28.6 us, 4.2 TB/s; a copy of 1 GiB 5.1).
// With few, the chain of a unit: launch, lengths, first bytes, 0.8 us a tile of 16 rows at
// head_dim 128, and the join's launch (four sessions behind 2048 rows: 7.4 + 3.5 us). At 512 a
// tile of 64 rows takes 2.4 us, with one wave on a SIMD: of a wave's life 13 % are matrix
// instructions and 12 % vector ones, the LDS is busy for 14 to 19 %, 35 % pass in waits for
// loads and LDS reads and 37 % between instructions.
//
// A unit whose V holds a seen infinity adds its rows up again one by one: 64 sessions behind
// 4096 rows with one in the prefix 4.6 ms.
#pragma once

#include "kvrt_shared.h"
#include "kvrt_wave.h"

namespace kvrt {

// LDS DMA of 16 bytes per lane from base + off (bytes), base uniform; ONCE: of rows that are
// not read again.
template <bool ONCE>
__device__ __forceinline__ void shared_dma(const void *base, uint32_t off, uint32_t lds) {
    if constexpr (ONCE) asm volatile("global_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
    else asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}
template <bool ONCE>
__device__ __forceinline__ void shared_dma(const void *at, uint32_t lds) {
    if constexpr (ONCE) dma_load16(at, lds);
    else dma_load16_cached(at, lds);
}

__device__ __forceinline__ f32x4_t mfma_bf16(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                   0, 0);
}

// The largest of three in one instruction (fmaxf of values that cross a branch takes another
// for each of them, on account of signalling NaN). Assembly that reads a matrix
// instruction's result needs its wait: settle() comes between.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ void settle(f32x4_t &a, f32x4_t &b) {
    asm volatile("s_nop 15" : "+v"(a), "+v"(b));  // 16 states: more than an 8-pass instruction asks for
}

// x of the lanes before and this one, combined: lane 63 has all of them. Steps within 16
// lanes and then over them are register moves (DPP); shuffles through LDS take ten times
// their latency ahead of a workgroup's first load.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or(int none, int x) {
    return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xF, false);
}
template <class Op>
__device__ __forceinline__ int wave_scan(int x, int none, Op op) {
    x = op(x, dpp_or<0x111, 0xF>(none, x));  // from 1, 2, 4, 8 lanes below in the row of 16
    x = op(x, dpp_or<0x112, 0xF>(none, x));
    x = op(x, dpp_or<0x114, 0xF>(none, x));
    x = op(x, dpp_or<0x118, 0xF>(none, x));
    x = op(x, dpp_or<0x142, 0xA>(none, x));  // lane 15 to row 1, 47 to row 3
    x = op(x, dpp_or<0x143, 0xC>(none, x));  // lane 31 to rows 2 and 3
    return x;
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(x, 63); }

template <int D>
struct SharedShape {
    static constexpr int STAGES = D == 512 ? 2 : 3;
    static constexpr int CHUNKS = D / 8;     // 16-byte chunks of a row
    static constexpr int IPB = D / 16;       // DMA instructions of a K (or V) tile
    static constexpr int IPW = IPB / 4;      // ... per wave
    static constexpr int KP = 1024 + 16, VP = 1024 + 32;  // bytes between instructions
    static constexpr int KBLK = IPB * KP, VBLK = IPB * VP, STAGE = KBLK + VBLK;
    // chunk c of an instruction's row number `sub` of K lies in place c ^ kx(sub)
    static __device__ __forceinline__ int kx(int sub) {
        return D == 128 ? (sub & 1) << 3 : D == 64 ? ((sub >> 1) & 1) << 2 : 0;
    }
};

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// One of the two runs of keys a unit walks: the prefix's or an item's own.
struct Segment {
    int slot;        // whose rows
    int lo, last;    // keys [lo, last] that some row of the unit sees
    int tile0, tiles;
    int off;         // a row's position in this run of keys: its own position + off
    int len;         // rows stored
    int all_lo, all_hi;  // keys [all_lo, all_hi) that every row sees
};

__device__ __forceinline__ Segment segment_of(int slot, int len, int off, int minpos, int maxpos, int window) {
    Segment s;
    s.slot = slot;
    s.off = off;
    s.len = len;
    const int end = max(min(len, off + maxpos + 1), 0);
    s.lo = window > 0 ? min(max(off + minpos - window + 1, 0), end) : 0;
    s.last = end - 1;
    s.tile0 = s.lo / kSharedKeys;
    s.tiles = end > s.lo ? (end + kSharedKeys - 1) / kSharedKeys - s.tile0 : 0;
    s.all_lo = window > 0 ? off + maxpos - window + 1 : 0;
    s.all_hi = min(off + minpos + 1, len);
    return s;
}

// A unit's work: tiles [x0, x1) of its list (the prefix's tiles, then its own), rows row0
// .. row0 + nrows - 1 of the call's (item, query, head) order, KV head kvh.
struct SharedUnit {
    Segment pre, own;
    int kvh, row0, nrows, x0, x1, part;
    bool once;  // no other unit reads its rows
    int lens;  // lane i: length of item i
};

// Outputs dim0 .. dim0 + DIMS - 1 of row f of a unit by one wave, each key's weight one fp32
// number, 2^(score - m); those that are not numbers are stored. Keys over lanes and halves of the
// dims over halves of the wave for the scores; dims over lanes for the values. The arguments are
// read again here, so that the loop over the tiles holds no registers for a row that may never
// come. kept: the unit's queries, where answers have taken their place in memory.
template <int D, int LAYOUT, int DIMS>
__device__ __forceinline__ void row_again(const SharedUnit &u, const uint16_t *kept, int f, int dim0, float m, float sum,
                                          int lane) {
    constexpr int E = (DIMS + 63) / 64;  // dims per lane
    uint64_t args = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(args));
    const auto &a = *reinterpret_cast<const SharedArgs __attribute__((address_space(4))) *>(args);
    const int per_item = a.group * a.qn;
    int item, rem, qr, hr;
    udivmod_uniform(f, per_item, item, rem);
    udivmod_uniform(rem, a.group, qr, hr);
    const int head = u.kvh * a.group + hr;
    const int len = min(max(a.len.lens[(int64_t)a.slots[item] * a.len.stride + a.len.offset], 0), a.capacity);
    const int pos = len - a.qn + qr;
    KVView kv;
    kv.k = a.kv.k, kv.v = a.kv.v, kv.page_table = a.kv.page_table;
    kv.slot_stride = a.kv.slot_stride, kv.head_stride = a.kv.head_stride, kv.row_stride = a.kv.row_stride;
    kv.kv_heads = a.kv.kv_heads, kv.rows = a.kv.rows, kv.pt_stride = a.kv.pt_stride;
    kv.block_shift = a.kv.block_shift, kv.pool_pages = a.kv.pool_pages;
    const int64_t row = ((int64_t)item * (a.kv.kv_heads * a.group) + head) * a.qn + qr;
    const auto *kg = static_cast<const uint16_t *>(a.kv.k), *vg = static_cast<const uint16_t *>(a.kv.v);
    const int half = D / 2 * (lane >> 5);
    const uint16_t *q = a.parts == 1 && a.out == a.q ? kept + (f - u.row0) * D : a.q + row * D;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma clang loop unroll(disable)
    for (int x = u.x0; x < u.x1; ++x) {
        const bool own = x >= u.pre.tiles;
        const int tile = own ? u.own.tile0 + x - u.pre.tiles : u.pre.tile0 + x;
        const int slot = own ? u.own.slot : u.pre.slot, at = pos + (own ? u.own.off : u.pre.off);
        const int lo = own ? u.own.lo : u.pre.lo, last = own ? u.own.last : u.pre.last;
        const int key = tile * kSharedKeys + (lane & 31);
        bool seen = key >= lo && key <= min(at, last) && (a.window == 0 || key > at - a.window);
        if (a.pmask && key < a.pmask[slot].len) seen &= (a.pmask[slot].bits[(key >> 5) & (kPrefixWords - 1)] >> (key & 31) & 1u) != 0;
        const int64_t off = seen ? row_offset<LAYOUT>(kv, slot, u.kvh, key, D) : -1;  // (-1: its page is not mapped)
        float t = pair<OpSum, 32>(dot_rows(q + half, kg + (off < 0 ? 0 : off) + half, D / 2));
        if (a.cap != 0.f) {
            float one[1] = {t};
            cap_scores<1>(one, a.inv_cap, a.cap);
            t = one[0];
        } else {
            t *= a.scale;
        }
        if (a.slopes) t = fmaf(log2_slope(a.slopes[head]), (float)(key - at), t);
        const float p = off < 0 ? 0.f : __builtin_amdgcn_exp2f(t - m);
        const uint32_t some = (uint32_t)__ballot(off >= 0);
#pragma clang loop unroll(disable)
        for (int j = 0; j < kSharedKeys; ++j) {
            const float w = __shfl(p, j);
            const uint16_t *v = vg + __shfl(off, j) + dim0;
            if (!(some >> j & 1u)) continue;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (64 * e + lane < DIMS) acc[e] = fmaf(w, bf16_to_f32(v[64 * e + lane]), acc[e]);
        }
    }
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = 64 * e + lane;
        if (d >= DIMS || acc[e] - acc[e] == 0.f) continue;
        if (a.parts == 1) a.out[row * D + dim0 + d] = f32_to_bf16(acc[e] * inv);
        else a.part_o[(((int64_t)u.kvh * a.n_items * per_item + f) * a.parts + u.part) * D + dim0 + d] = acc[e];
    }
}

// BLOCKS: 16-row blocks per wave, of the unit's blocks wave, wave + 4 (past its last one
// they are computed and not stored: a branch would part the matrix instructions); 0: the
// unit has one, which all waves share.
template <int D, int LAYOUT, int BLOCKS>
__device__ __forceinline__ void shared_unit(const SharedArgs &a, const SharedUnit &u, uint8_t *lds, int *again) {
    using S = SharedShape<D>;
    constexpr bool WIDE = BLOCKS > 0;
    constexpr int RS = WIDE ? BLOCKS : 1;
    constexpr int NB = WIDE ? D / 16 : D / 64;              // 16-dim blocks per wave
    constexpr int NS = S::STAGES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int b0 = WIDE ? 0 : wave * NB;
    const int nblocks = (u.nrows + 15) / 16;                // of the unit's rows
    const bool some = !WIDE || wave < nblocks;              // this wave has rows

    // A negative scale is moved into q's sign bits (exact), so that the largest score has the
    // largest product; a zero scale stays above 0, so that a masked score (-INFINITY) keeps
    // its weight of 0. Scores that are capped or biased are made one by one, in log2 units.
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    const bool made = a.cap != 0.f || a.slopes;
    const float unit = made ? 1.f : fmaxf(fabsf(a.scale), 1e-37f);
    // this lane's rows
    const int per_item = a.group * a.qn;
    int pos[RS];          // own position; -1 - P and below: a lane without a row sees nothing
    float slope[RS];
    uint4 qop[RS][D / 32];
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        const int r = 16 * (WIDE ? wave + 4 * s : 0) + col;
        const bool valid = r < u.nrows;
        const int f = u.row0 + (valid ? r : 0);
        int item, rem, qr, hr;
        udivmod_uniform(f, per_item, item, rem);
        udivmod_uniform(rem, a.group, qr, hr);
        const int len = __shfl(u.lens, item);
        pos[s] = valid ? len - a.qn + qr : INT32_MIN / 2;
        const int head = u.kvh * a.group + hr;
        const uint16_t *qp = a.q + (((int64_t)item * (a.kv.kv_heads * a.group) + head) * a.qn + qr) * D + 8 * grp;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) qop[s][c] = *reinterpret_cast<const uint4 *>(qp + 32 * c);
        slope[s] = a.slopes ? log2_slope(a.slopes[head]) : 0.f;
    }
    // masks of the two slots: length, and word `lane & 15`
    int plen_p = 0, plen_o = 0;
    uint32_t pw_p = ~0u, pw_o = ~0u;
    if (a.pmask) {
        if (u.pre.tiles > 0) load_prefix(a.pmask, u.pre.slot, lane, plen_p, pw_p);
        if (u.own.tiles > 0) load_prefix(a.pmask, u.own.slot, lane, plen_o, pw_o);
    }

    float m[RS], l[RS];
    f32x4_t o[RS][NB];
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        m[s] = kNegBig, l[s] = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) o[s][b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }

    // ---- staging: wave w fetches instructions w, w + 4, ... of a tile's K and V rows
    bool bad = false;
    const uint32_t lds_at = lds_addr(lds);
    const auto *kg = static_cast<const uint16_t *>(a.kv.k), *vg = static_cast<const uint16_t *>(a.kv.v);
    // PAGED: entry `lane` past win_page of the table of slot win_slot, loaded again where a tile
    // leaves it (64 pages: every 32 tiles at 16 keys a page)
    int window = -1, win_slot = -1, win_page = 0;
    auto where = [&](int x, int &key0) __attribute__((always_inline)) {
        const bool own = x >= u.pre.tiles;
        const auto pick = [&](int pre, int its) __attribute__((always_inline)) { return own ? its : pre; };
        Segment g;
        g.slot = pick(u.pre.slot, u.own.slot), g.lo = pick(u.pre.lo, u.own.lo), g.last = pick(u.pre.last, u.own.last);
        g.off = pick(u.pre.off, u.own.off), g.all_lo = pick(u.pre.all_lo, u.own.all_lo);
        g.all_hi = pick(u.pre.all_hi, u.own.all_hi);
        key0 = ((own ? u.own.tile0 - u.pre.tiles : u.pre.tile0) + x) * kSharedKeys;
        return g;
    };
    auto stage_as = [&](auto once_c, auto of_k, auto of_v, int x, int buf) __attribute__((always_inline)) {
        constexpr bool ONCE = decltype(once_c)::value, OF_K = decltype(of_k)::value, OF_V = decltype(of_v)::value;
        int key0;
        const Segment g = where(x, key0);
        const int64_t head = LAYOUT == KVRT_LAYOUT_PAGED
                                 ? 0
                                 : (int64_t)g.slot * a.kv.slot_stride + (int64_t)u.kvh * a.kv.head_stride;
        const int ring0 = LAYOUT == KVRT_LAYOUT_RING ? key0 % a.kv.rows : 0;
        const int sub = lane / S::CHUNKS, c = lane % S::CHUNKS;
        int page0 = 0, page1 = 0;  // of the tile's two halves, where pages hold 16 keys and more
        if constexpr (LAYOUT == KVRT_LAYOUT_PAGED) {
            const int p0 = min(max(key0, g.lo), g.last) >> a.kv.block_shift;
            const int p1 = min(max(key0 + 16, g.lo), g.last) >> a.kv.block_shift;
            const int end = min(key0 + kSharedKeys - 1, g.last) >> a.kv.block_shift;
            if (g.slot != win_slot || end - win_page >= 64) {
                win_slot = g.slot, win_page = p0;
                window = load_page_window(a.kv, win_slot, win_page, lane);
            }
            if constexpr (D < 512) {  // (at 512 a shuffle a row is as fast)
                page0 = __builtin_amdgcn_readlane(window, p0 - win_page);
                page1 = __builtin_amdgcn_readlane(window, p1 - win_page);
            }
        }
#pragma unroll
        for (int i = 0; i < S::IPW; ++i) {
            const int ins = 4 * i + wave, r = ins + S::IPB * sub;
            const int key = min(max(key0 + r, g.lo), g.last);  // rows nobody sees read one that somebody does
            const uint32_t to = lds_at + (uint32_t)(buf * S::STAGE), kto = to + ins * S::KP, vto = to + S::KBLK + ins * S::VP;
            int64_t off;
            if constexpr (LAYOUT == KVRT_LAYOUT_CONTIG) {
                const int64_t base = head + (int64_t)key0 * D;
                const uint32_t at = (uint32_t)(key - key0) * (2 * D);
                if constexpr (OF_K) shared_dma<ONCE>(kg + base, at + 16 * (c ^ S::kx(sub)), kto);
                if constexpr (OF_V) shared_dma<ONCE>(vg + base, at + 16 * c, vto);
                continue;
            } else if constexpr (LAYOUT == KVRT_LAYOUT_RING) {
                int rr = ring0 + (key - key0);
                if (a.kv.rows >= kSharedKeys) rr = rr >= a.kv.rows ? rr - a.kv.rows : rr;  // wraps once at most
                else rr %= a.kv.rows;
                off = head + (int64_t)rr * D;
            } else {
                int page = r >= 16 ? page1 : page0;
                if (D == 512 || a.kv.block_shift < 4) page = __shfl(window, (key >> a.kv.block_shift) - win_page);
                off = page_row_offset(a.kv, page, u.kvh, key, D);
                bad |= off < 0;
                off = off < 0 ? 0 : off;
            }
            if constexpr (OF_K) shared_dma<ONCE>(kg + off + 8 * (c ^ S::kx(sub)), kto);
            if constexpr (OF_V) shared_dma<ONCE>(vg + off + 8 * c, vto);
        }
    };

    auto stage = [&](auto of_k, auto of_v, int x, int buf) __attribute__((always_inline)) {
        if (LAYOUT != KVRT_LAYOUT_PAGED && u.once) stage_as(std::true_type{}, of_k, of_v, x, buf);
        else stage_as(std::false_type{}, of_k, of_v, x, buf);
    };

    // ---- one tile
    // K: key row col (and + 16), chunk 4 c + grp; V: key row 4 grp + s16 / 4 (and + 16), dims
    // 4 (s16 % 4) .. + 3 of a block
    const int s16 = lane & 15, vrow = 4 * grp + (s16 >> 2);
    constexpr int H = 16 / S::IPB * 2 * D;  // bytes from row r to r + 16 (D 512: 16 instructions)
    const int kadr = (col % S::IPB) * S::KP + (col / S::IPB) * 2 * D + 16 * grp, kx = 16 * S::kx(col / S::IPB);
    const int vadr = (vrow % S::IPB) * S::VP + (vrow / S::IPB) * 2 * D + 8 * (s16 & 3) + 32 * b0;
    uint4 ph[RS], pl[RS];  // a tile's weights, high and low terms
    // V^T of 16 dims: this lane's dim 16 b + col, keys 16 h + 4 grp + 0 .. 3
    auto vop = [&](const uint8_t *vt, int b) __attribute__((always_inline)) {
        uint2 v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            v[h] = lds_read_tr16(reinterpret_cast<const uint16_t *>(vt + vadr + 32 * b + h * (D == 512 ? 16 * S::VP : H)));
        return make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
    };
    // The weights of tile x; whether all queries see all of it.
    auto weigh = [&](int x, int buf) __attribute__((always_inline)) {
        const uint8_t *kt = lds + buf * S::STAGE;
        f32x4_t sc[RS][2];
#pragma unroll
        for (int s = 0; s < RS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[s][h] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 k = *reinterpret_cast<const uint4 *>(kt + kadr + ((64 * c) ^ kx) + h * (D == 512 ? 16 * S::KP : H));
#pragma unroll
                for (int s = 0; s < RS; ++s) sc[s][h] = mfma_bf16(k, qop[s][c], sc[s][h]);
            }
        __builtin_amdgcn_sched_barrier(0);
        int key0;
        const Segment g = where(x, key0);
        const bool own = x >= u.pre.tiles;
        const int plen = own ? plen_o : plen_p;
        const bool whole = key0 >= g.all_lo && key0 + kSharedKeys <= g.all_hi && key0 >= plen;
        uint32_t word = ~0u;  // bit k: key0 + k passes the slot's mask
        if (key0 < plen) word = (uint32_t)__builtin_amdgcn_readlane((int)(own ? pw_o : pw_p), (key0 >> 5) & (kPrefixWords - 1));
#pragma unroll
        for (int s = 0; s < RS; ++s) {
            const int at = pos[s] + g.off;
            settle(sc[s][0], sc[s][1]);
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = sc[s][i / 4][i % 4];
            if (made) {
                if (a.cap != 0.f) {
                    cap_scores<8>(t, fabsf(a.inv_cap), a.cap);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) t[i] *= fabsf(a.scale);
                }
                if (a.slopes) {
                    const float far = (float)(key0 + 4 * grp - at);  // below 2^24 in earnest, and rounded beyond
#pragma unroll
                    for (int i = 0; i < 8; ++i) t[i] = fmaf(slope[s], far + (float)(16 * (i / 4) + i % 4), t[i]);
                }
            }
            if (!whole) {
                // bit k: key0 + k is seen by this row
                const int hi = min(max(min(at, g.last) - key0 + 1, 0), 32);
                const int lo = min(max(max(a.window > 0 ? at - a.window + 1 : 0, g.lo) - key0, 0), 32);
                uint32_t vis = word & (hi >= 32 ? ~0u : (1u << hi) - 1u) & (lo >= 32 ? 0u : ~0u << lo);
                vis >>= 4 * grp;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) t[4 * h + i] = (vis >> (16 * h + i)) & 1u ? t[4 * h + i] : -INFINITY;
            }
            float top = max3(max3(max3(t[0], t[1], t[2]), t[3], t[4]), max3(t[5], t[6], t[7]), t[7]);
            top = pair<OpMax, 32>(pair<OpMax, 16>(top * unit));
            const float mn = top > m[s] + kRescaleSlack ? top : m[s];
            if (__any(mn != m[s])) {
                const float corr = __builtin_amdgcn_exp2f(m[s] - mn);
                l[s] *= corr;
#pragma unroll
                for (int b = 0; b < NB; ++b) o[s][b] *= corr;
                m[s] = mn;
            }
            uint32_t hiw[4], low[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = __builtin_amdgcn_exp2f(fmaf(t[2 * i], unit, -m[s]));
                const float x1 = __builtin_amdgcn_exp2f(fmaf(t[2 * i + 1], unit, -m[s]));
                l[s] += x0 + x1;
                hiw[i] = pack_bf16x2(x0, x1);
                low[i] = pack_bf16x2(x0 - bf16_lo(hiw[i]), x1 - bf16_hi(hiw[i]));
            }
            ph[s] = make_uint4(hiw[0], hiw[1], hiw[2], hiw[3]);
            pl[s] = make_uint4(low[0], low[1], low[2], low[3]);
        }
        return whole;
    };
    // Whether V of a tile that some query does not see whole holds NaN or infinities: 0 * NaN is
    // not 0, so that its products are made one by one (add_odd).
    auto look = [&](int buf) __attribute__((always_inline)) {
        const uint8_t *vt = lds + buf * S::STAGE + S::KBLK;
        u16x2_t most = {0, 0};
#pragma clang loop unroll_count(2)
        for (int b = 0; b < NB; ++b) {
            const uint4 v = vop(vt, b);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
        }
        return __any(most[0] >= 0x7f80 || most[1] >= 0x7f80) != 0;
    };
    auto add = [&](int buf) __attribute__((always_inline)) {
        const uint8_t *vt = lds + buf * S::STAGE + S::KBLK;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint4 v = vop(vt, b);
#pragma unroll
            for (int s = 0; s < RS; ++s) o[s][b] = mfma_bf16(v, ph[s], o[s][b]);
#pragma unroll
            for (int s = 0; s < RS; ++s) o[s][b] = mfma_bf16(v, pl[s], o[s][b]);
        }
    };
    auto add_odd = [&](int buf) __attribute__((always_inline)) {
        const uint8_t *vt = lds + buf * S::STAGE + S::KBLK;
#pragma clang loop unroll(disable)
        for (int k = 0; k < kSharedKeys; ++k) {
            const int at = 2 * (k >> 4) + ((k >> 1) & 1), from = 16 * ((k >> 2) & 3) + col;
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                const uint4 hs = ph[s], ls = pl[s];
                const uint32_t hw = at < 2 ? (at == 0 ? hs.x : hs.y) : at == 2 ? hs.z : hs.w;
                const uint32_t lw = at < 2 ? (at == 0 ? ls.x : ls.y) : at == 2 ? ls.z : ls.w;
                const float p = __shfl(k & 1 ? bf16_hi(hw) + bf16_hi(lw) : bf16_lo(hw) + bf16_lo(lw), from);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(
                        vt + (k % S::IPB) * S::VP + (k / S::IPB) * 2 * D + 32 * (b0 + b) + 8 * grp);
                    const float x[4] = {bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)};
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[s][b][i] = p == 0.f ? o[s][b][i] : fmaf(p, x[i], o[s][b][i]);
                    __builtin_amdgcn_sched_barrier(0);  // (one block's values at a time: registers)
                }
            }
        }
    };

    const int n = u.x1 - u.x0;
    constexpr int PER = 2 * S::IPW;  // a wave's DMAs of a tile
    // With two stages (head_dim 512) K and V travel apart: a tile's K from when the last but
    // one's was read, its V half a tile later, so that both have a tile and a half under way (4
    // sessions of 8192 rows, 8 KV heads: 114 -> 107 us; 8 behind 8192 29.9 -> 27.3). On pages,
    // where every row's page would be looked up twice, together (116 us; apart 140).
    constexpr bool APART = NS == 2 && LAYOUT != KVRT_LAYOUT_PAGED;
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    if (n > 0) {
        if constexpr (APART) {
            stage(yes, no, u.x0, 0);
            stage(no, yes, u.x0, 0);
            if (n > 1) stage(yes, no, u.x0 + 1, 1);
        } else {
#pragma unroll
            for (int i = 0; i < NS - 1; ++i)
                if (i < n) stage(yes, yes, u.x0 + i, i);
        }
        // The queries travel beside the first tiles' bytes and are waited for here (a decode
        // step of 16 windowed sessions 7.5 -> 7.1 us, 16 paged ones 28.9 -> 27.2).
#pragma unroll
        for (int s = 0; s < RS; ++s) {
            asm volatile("" : "+v"(pos[s]), "+v"(slope[s]));
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint4 &x = qop[s][c];
                x = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
                asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w));
            }
        }
        // (add_odd stands outside the loop that all other tiles stay in: beside it in one loop,
        // the accumulators were copied at every tile)
        for (int i = 0, buf = 0;; ++i) {
            bool odd = false;
            for (; i < n; ++i) {
                const bool more = i + 1 < n;
                bool whole = true;
                if constexpr (APART) {
                    if (more) wait_vmem<PER>();  // V of tile i and K of the next may be under way
                    else wait_vmem<PER / 2>();
                    __syncthreads();             // every wave's K of tile i has landed, V of tile i - 1 is read
                    if (more) stage(no, yes, u.x0 + i + 1, buf ^ 1);
                    if (some) whole = weigh(u.x0 + i, buf);
                    if (more) wait_vmem<PER>();  // K and V of the next
                    else wait_vmem<0>();
                    __syncthreads();             // every wave's V of tile i has landed, its K is read
                    if (i + 2 < n) stage(yes, no, u.x0 + i + 2, buf);
                } else {
                    wait_vmem_steps<PER, NS - 2>(n - 1 - i);  // this wave's part of tile i has landed
                    __syncthreads();                          // every wave's has, and tile i - 1 is read
                    if (i + NS - 1 < n) stage(yes, yes, u.x0 + i + NS - 1, buf == 0 ? NS - 1 : buf - 1);
                    if (some) whole = weigh(u.x0 + i, buf);
                }
                if (some) {
                    odd = !whole && look(buf);
                    if (odd) break;
                    add(buf);
                }
                buf = buf == NS - 1 ? 0 : buf + 1;
            }
            if (!odd) break;
            add_odd(buf);
            buf = buf == NS - 1 ? 0 : buf + 1;
        }
    }
    if (bad) a.err[0] = 1;
    // A seen infinity times a weight's two terms is NaN where the low one is 0 or below (inf * 0,
    // inf - inf), and the infinity by definition. Outputs that are not numbers, of rows whose
    // scores are, are added up again with whole weights and stored over. The rows of block s:
    auto odd_rows = [&](int s) __attribute__((always_inline)) {
        float none[4] = {};  // one NaN where an output is no number
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) none[i] = fmaf(o[s][b][i], 0.f, none[i]);
        none[0] += none[1] + (none[2] + none[3]);
        const uint64_t odd = __ballot(none[0] != none[0] && l[s] == l[s]);
        const int left = u.nrows - 16 * (WIDE ? wave + 4 * s : 0);
        return (uint32_t)(odd | odd >> 16 | odd >> 32 | odd >> 48) & (left >= 16 ? 0xffffu : (1u << max(left, 0)) - 1u);
    };
#pragma unroll
    for (int s = 0; s < RS; ++s) l[s] = pair<OpSum, 32>(pair<OpSum, 16>(l[s]));
    if (a.parts == 1 && a.out == a.q) {  // (the same for all units: answers go where the queries are)
        uint32_t odd = 0;
#pragma unroll
        for (int s = 0; s < RS; ++s) odd |= odd_rows(s);
        if (odd != 0) *again = 1;
        __syncthreads();  // (and every wave has read its last tile)
        if (*again != 0) {
            for (int i = 8 * threadIdx.x; i < u.nrows * D; i += 8 * 256) {
                int item, rem, qr, hr;
                udivmod_uniform(u.row0 + i / D, per_item, item, rem);
                udivmod_uniform(rem, a.group, qr, hr);
                const uint16_t *from =
                    a.q + (((int64_t)item * (a.kv.kv_heads * a.group) + u.kvh * a.group + hr) * a.qn + qr) * D + i % D;
                *reinterpret_cast<uint4 *>(lds + 2 * i) = *reinterpret_cast<const uint4 *>(from);
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        const int r = 16 * (WIDE ? wave + 4 * s : 0) + col;
        const float sum = l[s];
        if (r >= u.nrows) continue;
        const int f = u.row0 + r;
        if (a.parts == 1) {
            int item, rem, qr, hr;
            udivmod_uniform(f, per_item, item, rem);
            udivmod_uniform(rem, a.group, qr, hr);
            const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
            uint16_t *dst =
                a.out + (((int64_t)item * (a.kv.kv_heads * a.group) + u.kvh * a.group + hr) * a.qn + qr) * D + 4 * grp;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                *reinterpret_cast<uint2 *>(dst + 16 * (b0 + b)) = make_uint2(
                    pack_bf16x2(o[s][b][0] * inv, o[s][b][1] * inv), pack_bf16x2(o[s][b][2] * inv, o[s][b][3] * inv));
        } else {
            const int64_t at = ((int64_t)u.kvh * a.n_items * per_item + f) * a.parts + u.part;
            float *dst = a.part_o + at * D + 4 * grp;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                *reinterpret_cast<float4 *>(dst + 16 * (b0 + b)) = make_float4(o[s][b][0], o[s][b][1], o[s][b][2], o[s][b][3]);
            if (grp == 0 && b0 == 0) a.part_ml[at] = make_float2(m[s], sum);
        }
    }
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        uint32_t left = odd_rows(s);
        if (__builtin_expect_with_probability(left == 0, 1, 0.9999)) continue;
        wait_vmem<0>();  // the rows' first answers are stored
        for (; left != 0; left &= left - 1) {
            const int c = __builtin_ctz(left);
            row_again<D, LAYOUT, 16 * NB>(u, reinterpret_cast<const uint16_t *>(lds), u.row0 + 16 * (WIDE ? wave + 4 * s : 0) + c,
                                          16 * b0, __shfl(m[s], c), __shfl(l[s], c), lane);
        }
    }
}

template <int D, int LAYOUT>
__global__ __launch_bounds__(256, D == 64 ? 3 : D == 128 ? 2 : 1) void shared_attend_kernel(SharedArgs a) {
    using S = SharedShape<D>;
    constexpr int TILE = shared_tile(D);
    __shared__ __align__(16) uint8_t lds[S::STAGES * S::STAGE];
    __shared__ int again;  // rows are added up again
    static_assert(TILE * D * 2 <= S::STAGES * S::STAGE, "a unit's queries fit the stages");
    if (threadIdx.x == 0) again = 0;
    const int lane = threadIdx.x & 63;
    const int hkv = a.kv.kv_heads, per_item = a.group * a.qn;
    const int capacity = a.capacity;
    const auto length = [&](int slot) __attribute__((always_inline)) {
        return min(max(a.len.lens[(int64_t)slot * a.len.stride + a.len.offset], 0), capacity);
    };
    SharedUnit u;
    u.lens = length(a.slots[min(lane, a.n_items - 1)]);
    const int prefix = a.prefix_slot >= 0 ? __builtin_amdgcn_readfirstlane(length(a.prefix_slot)) : 0;
    // KV heads are the least significant: workgroups of one head land on one XCD when
    // there are eight, and share its L2
    int at, splits;
    udivmod_uniform(blockIdx.x, hkv, at, u.kvh);
    const bool pre = at < a.pre_tiles * a.pre_splits;
    int ks, tile, minpos, maxpos;
    if (pre) {
        splits = a.pre_splits;
        udivmod_uniform(at, splits, tile, ks);
        u.row0 = tile * TILE;
        u.nrows = min(a.n_items * per_item - u.row0, TILE);
        u.part = ks;
        // (lanes past the items hold the last one's length)
        minpos = wave_total(wave_scan(u.lens, INT32_MAX, [](int x, int y) { return min(x, y); })) - a.qn;
        maxpos = wave_total(wave_scan(u.lens, INT32_MIN, [](int x, int y) { return max(x, y); })) - 1;
        u.pre = segment_of(a.prefix_slot, prefix, prefix, minpos, maxpos, a.window);
        u.own = segment_of(a.prefix_slot, 0, 0, 0, -1, 0);
    } else {
        int item, rem;
        at -= a.pre_tiles * a.pre_splits;
        if (a.own_per > 0) {
            // sessions of unequal length: each takes a range of own_per tiles after another
            const int t = lane < a.n_items ? segment_of(0, u.lens, 0, u.lens - a.qn, u.lens - 1, a.window).tiles : 0;
            const auto add = [](int x, int y) { return x + y; };
            int per = a.own_per;
            int mine = lane < a.n_items ? max(1, (t + per - 1) / per) : 0;
            int sum = wave_scan(mine, 0, add);
            if (wave_total(sum) > a.own_wgs || __any(mine > a.own_splits)) {
                // more of them than the launch and its partials were made for (a replay on longer
                // sessions): n sessions take at most total / per + n ranges
                const int all = wave_total(wave_scan(t, 0, add)), spare = a.own_wgs - a.n_items;
                const int top = wave_total(wave_scan(t, 0, [](int x, int y) { return max(x, y); }));
                per = max(max((top + a.own_splits - 1) / a.own_splits, spare > 0 ? (all + spare - 1) / spare : top), 1);
                mine = lane < a.n_items ? max(1, (t + per - 1) / per) : 0;
                sum = wave_scan(mine, 0, add);
            }
            const uint64_t past = __ballot(sum > at);
            if (past == 0) return;
            item = __builtin_ctzll(past);
            const int first = item == 0 ? 0 : __builtin_amdgcn_readlane(sum, item - 1);
            splits = __builtin_amdgcn_readlane(sum, item) - first;
            ks = at - first;
            tile = 0;
            if (ks == splits - 1) {  // parts that this session does not have
                const int none = a.own_splits - splits;
                for (int i = threadIdx.x; i < none * per_item; i += 256)
                    a.part_ml[((int64_t)u.kvh * a.n_items * per_item + item * per_item + i / none) * a.parts + a.pre_splits +
                              splits + i % none] = make_float2(kNegBig, 0.f);
            }
        } else {
            splits = a.own_splits;
            udivmod_uniform(at, splits * a.own_tiles, item, rem);
            udivmod_uniform(rem, splits, tile, ks);
        }
        u.row0 = item * per_item + tile * TILE;
        u.nrows = min(per_item - tile * TILE, TILE);
        u.part = a.pre_splits + ks;
        const int len = __builtin_amdgcn_readlane(u.lens, item);
        int qf, ql, ignore;
        udivmod_uniform(tile * TILE, a.group, qf, ignore);
        udivmod_uniform(tile * TILE + u.nrows - 1, a.group, ql, ignore);
        minpos = len - a.qn + qf;
        maxpos = len - a.qn + ql;
        u.own = segment_of(a.slots[item], len, 0, minpos, maxpos, a.window);
        u.pre = segment_of(a.prefix_slot, a.joined ? prefix : 0, prefix, minpos, maxpos, a.window);
    }
    // In calls that outgrow the last cache, rows that one unit reads pass the caches by (64
    // sessions behind 4096 rows 55.9 -> 52.0 us a call, 4 of 8192 at head_dim 512 106 -> 97). In
    // smaller ones the next call finds them there (8 of 8 rows behind 8192 at 512 27.7 us, 29.2
    // past the caches), as other units find what several read (16 behind 4096 28 and 32).
    u.once = LAYOUT != KVRT_LAYOUT_PAGED && a.large && (pre ? a.pre_tiles == 1 : a.own_tiles == 1 && !a.joined);
    const int tiles = u.pre.tiles + u.own.tiles, per = (tiles + splits - 1) / splits;
    u.x0 = min(ks * per, tiles);
    u.x1 = min(u.x0 + per, tiles);
    if (u.nrows <= 16) shared_unit<D, LAYOUT, 0>(a, u, lds, &again);
    else if (TILE == 64 || u.nrows <= 64) shared_unit<D, LAYOUT, 1>(a, u, lds, &again);
    else shared_unit<D, LAYOUT, TILE / 64>(a, u, lds, &again);
}

// Joins the partials of every row. A row's parts are dealt to GROUPS groups of D / 4
// threads, so that few rows of many parts take one or two round trips of loads (kAhead
// parts a thread at a time), and the groups' sums are added in group order.
template <int D, int GROUPS>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a) {
    constexpr int LANES = D / 4, ROWS = 256 / (LANES * GROUPS), kAhead = 8;
    __shared__ float4 so[GROUPS > 1 ? 256 : 1];
    __shared__ float2 sml[GROUPS > 1 ? 256 : 1];
    const int per_item = a.group * a.qn, lane = threadIdx.x % LANES, group = threadIdx.x / LANES % GROUPS;
    const int64_t rows = (int64_t)a.n_items * per_item;
    const int64_t at = (int64_t)blockIdx.x * ROWS + threadIdx.x / (LANES * GROUPS);
    const bool live = at < rows * a.kv.kv_heads;
    const int kvh = live ? (int)(at / rows) : 0, f = live ? (int)(at - kvh * rows) : 0, d = 4 * lane;
    const int n = live ? a.parts : 0;
    float M = kNegBig, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto take = [&](const float2(&ml)[kAhead], const float4(&x)[kAhead]) __attribute__((always_inline)) {
        float top = M;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) top = fmaxf(top, ml[i].x);
        const float c = __builtin_amdgcn_exp2f(M - top);
        sum *= c;
        o = make_float4(o.x * c, o.y * c, o.z * c, o.w * c);
        M = top;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (ml[i].x == kNegBig && ml[i].y == 0.f) continue;  // it saw no key
            const float w = __builtin_amdgcn_exp2f(ml[i].x - M);
            sum = fmaf(ml[i].y, w, sum);
            o = make_float4(fmaf(x[i].x, w, o.x), fmaf(x[i].y, w, o.y), fmaf(x[i].z, w, o.z), fmaf(x[i].w, w, o.w));
        }
    };
    float2 ml[kAhead];
    float4 x[kAhead];
    for (int p0 = group; p0 < n; p0 += kAhead * GROUPS) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t p = at * n + min(p0 + i * GROUPS, n - 1);
            ml[i] = a.part_ml[p];
            x[i] = *reinterpret_cast<const float4 *>(a.part_o + p * D + d);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (p0 + i * GROUPS >= n) ml[i] = make_float2(kNegBig, 0.f);
        take(ml, x);
    }
    if constexpr (GROUPS > 1) {
        so[threadIdx.x] = o;
        sml[threadIdx.x] = make_float2(M, sum);
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int g0 = 1; g0 < GROUPS; g0 += kAhead) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int g = threadIdx.x + min(g0 + i, GROUPS - 1) * LANES;
                ml[i] = g0 + i < GROUPS ? sml[g] : make_float2(kNegBig, 0.f);
                x[i] = so[g];
            }
            take(ml, x);
        }
    }
    if (!live) return;
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    int item, rem, qr, hr;
    udivmod_uniform(f, per_item, item, rem);
    udivmod_uniform(rem, a.group, qr, hr);
    uint16_t *dst = a.out + (((int64_t)item * (a.kv.kv_heads * a.group) + kvh * a.group + hr) * a.qn + qr) * D + d;
    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

template <int D, int GROUPS>
static hipError_t launch_shared_join(const SharedArgs &a, hipStream_t s) {
    if constexpr (GROUPS > 1)  // as many groups as leave each a batch of eight parts
        if (a.parts <= 8 * (GROUPS / 2)) return launch_shared_join<D, GROUPS / 2>(a, s);
    constexpr int ROWS = 1024 / (D * GROUPS);
    const int64_t rows = (int64_t)a.n_items * a.group * a.qn * a.kv.kv_heads;
    hipLaunchKernelGGL((shared_join_kernel<D, GROUPS>), dim3((unsigned)((rows + ROWS - 1) / ROWS)), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int D>
static hipError_t launch_shared_dim(const SharedArgs &a, hipStream_t s) {
    const int units = (a.pre_tiles * a.pre_splits +
                       (a.own_per > 0 ? a.own_wgs : a.n_items * a.own_tiles * a.own_splits)) * a.kv.kv_heads;
    switch (a.kv.layout) {
        case KVRT_LAYOUT_CONTIG:
            hipLaunchKernelGGL((shared_attend_kernel<D, KVRT_LAYOUT_CONTIG>), dim3(units), dim3(256), 0, s, a);
            break;
        case KVRT_LAYOUT_RING:
            hipLaunchKernelGGL((shared_attend_kernel<D, KVRT_LAYOUT_RING>), dim3(units), dim3(256), 0, s, a);
            break;
        case KVRT_LAYOUT_PAGED:
            hipLaunchKernelGGL((shared_attend_kernel<D, KVRT_LAYOUT_PAGED>), dim3(units), dim3(256), 0, s, a);
            break;
        default: return hipErrorInvalidValue;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.parts == 1) return e;
    return launch_shared_join<D, (D == 512 ? 2 : D == 256 ? 4 : 8)>(a, s);
}

}  // namespace kvrt
