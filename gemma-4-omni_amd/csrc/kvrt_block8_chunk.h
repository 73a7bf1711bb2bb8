// kvrt_block8_chunk.h — attention of many query rows per request over 8-bit pages.
//
// The mathematics is kvrt_block8_attend.hip's (codes as fp16, the V scale in the
// exponent); here 32 rows of a (request, KV head) lie on one wave and a workgroup's
// eight waves share the keys: 32-key blocks are converted to fp16 once, into LDS, and
// each wave takes per block
//   S^T (32 keys x 32 rows) = K Q^T     D/16    v_mfma_f32_32x32x16_f16
//   softmax per row (fp32, base 2)
//   O^T (D x 32) += V^T P^T             2 D/32  v_mfma_f32_32x32x16_f16
// A row tile is 64, 128 or 256 rows at D <= 128 and 128 beyond, where two waves share a
// row block's head dims (its Q and O fill two waves' registers). Its RW row blocks are
// fewer where the request's last tile has fewer rows; the RB / RW waves of a row block
// take the staged blocks in turn and are combined through LDS at the end. With few tiles the
// keys are also divided over `splits` workgroups, joined by a second launch.
//
// Bound by its vector and matrix instructions, which the two waves of a SIMD overlap only
// in part: at D 128 over 5600 keys counters show vector issue on half of all cycles and
// LDS on a quarter. Steps are therefore as long as LDS allows (fewer barriers), and nothing
// in a step waits for a load of its own. That serves long contexts: looking pages up a
// step ahead and a third staged step took the sliding chunk (four of 291 rows, window 512,
// D 256) from 33 to 37 us and the talker's (512 rows over 1400 keys) from 44 to 46.
// Measured, this kernel and the join of its splits: 4 requests of 512 rows, 16 heads over 8,
// D 128: 46 us over 1400 keys, 155 us over 5600 (0.58 PFLOP/s); 4 of 291, 8 heads over 1,
// D 256: 125 + 9 us over 4678 keys; one of 512, 16 heads over 2, D 512: 131 + 15 us over
// 4096.
//
// Lane layouts (32x32x16): A[row l%32][k 8(l/32)+j], B[k 8(l/32)+j][col l%32],
// D[row 8(i/4) + 4(l/32) + i%4][col l%32].
#pragma once

#include "kvrt_block8_rows.h"

namespace kvrt {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// LDS rows: K pitched so that 16 consecutive rows' 16-byte chunks lie on all 64 banks,
// V so that 4 rows' 64 bytes do (the transposed reads).
template <int D>
struct ChunkShape {
    static constexpr int NW = 8;                 // waves
    static constexpr int DS = D >= 256 ? 2 : 1;  // waves that share a row block's head dims
    static constexpr int RB = NW / DS;           // row blocks at most
    static constexpr int NBLK = D <= 128 ? 4 : 1;  // 32-key blocks of a step
    static constexpr int RMIN = RB / NBLK;                       // row blocks at least (waves past the blocks idle)
    static constexpr int KEYS = 32 * NBLK;
    static constexpr int SLOTS = D <= 128 ? 2 : D == 256 ? 3 : 1;  // steps whose K and V lie in LDS
    static constexpr int KP = 2 * D + 16, VP = 2 * D + 64;  // bytes
    static constexpr int PASSES = KEYS * D / (NW * 1024);   // 16-code chunks per thread of K (and of V)
    static constexpr int KSLOT = KEYS * KP, VSLOT = KEYS * VP, VBASE = SLOTS * KSLOT, BUF = VBASE + SLOTS * VSLOT;
    // codes wait for their step in LDS instead of in registers (D 512 has none left)
    static constexpr bool DMA = D == 512;
    static constexpr int RAW = DMA ? 2 * KEYS * D : 16;
    static constexpr int QL = D == 512 ? 3 : 0;  // ... nor for the last of the Q operands
    static constexpr int SX = DS > 1 ? NW * 4096 : 16;  // scores the waves of a row block exchange
};

// Calls f(integral_constant<int, u>) for u = U .. N - 1.
template <int U, int N>
struct ChunkFor {
    template <class F>
    __device__ __forceinline__ static void run(F &&f) {
        if constexpr (U < N) {
            f(std::integral_constant<int, U>{});
            ChunkFor<U + 1, N>::run(f);
        }
    }
};

struct ChunkScale {
    float k, log_v, inv_v, ok;
};

__device__ __forceinline__ f32x16_t mfma32_f16(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                  0);
}

// Sixteen codes as 32 bytes of fp16.
template <int CODE>
__device__ __forceinline__ void write_f16(uint8_t *dst, uint4 w) {
    uint4 a, b;
    codes_to_f16<CODE>(w.x, a.x, a.y);
    codes_to_f16<CODE>(w.y, a.z, a.w);
    codes_to_f16<CODE>(w.z, b.x, b.y);
    codes_to_f16<CODE>(w.w, b.z, b.w);
    *reinterpret_cast<uint4 *>(dst) = a;
    *reinterpret_cast<uint4 *>(dst + 16) = b;
}

// Tiles of `size` rows of the request.
__device__ __forceinline__ int tiles_of(const Block8AttendArgs &a, const Rows &r, int size) {
    return (r.count * a.group + size - 1) / size;
}

// The request that has tile u of all requests', its first tile; false past the last.
// Every thread of the workgroup calls.
template <int NW>
__device__ __forceinline__ bool tile_request(const Block8AttendArgs &a, int size, int u, int &req, int &before,
                                             bool &bad) {
    const int lane = threadIdx.x & 63;
    if (a.n <= 64) {
        int tiles = 0;
        if (lane < a.n) tiles = tiles_of(a, load_rows(a, lane, 0, size, bad), size);
        int inc = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(inc, d);
            if (lane >= d) inc += y;
        }
        const uint64_t past = __ballot(inc > u);
        if (past == 0) return false;
        req = __builtin_ctzll(past);
        before = __builtin_amdgcn_readlane(inc - tiles, req);
        return true;
    }
    __shared__ int lds[2 * NW], found[2];
    int at = 0;
    bool have = false;
    for (int base = 0; base < a.n && !have; base += 64 * NW) {
        const int i = base + threadIdx.x;
        const int tiles = i < a.n ? tiles_of(a, load_rows(a, i, 0, size, bad), size) : 0;
        int sum, top;
        const int first = at + scan_wg<NW>(tiles, lds, sum, top);
        at += sum;
        if (first <= u && u < first + tiles) found[0] = i, found[1] = first;
        have = u < at;
    }
    if (!have) return false;
    __syncthreads();
    req = __builtin_amdgcn_readfirstlane(found[0]);
    before = __builtin_amdgcn_readfirstlane(found[1]);
    return true;
}

// Key ranges the tile's keys are divided over (of at most a.splits).
template <int D>
__device__ __forceinline__ int splits_of(const Block8AttendArgs &a, const Rows &r) {
    const int steps = (r.kend - r.kstart / 32 * 32 + ChunkShape<D>::KEYS - 1) / ChunkShape<D>::KEYS;
    return min(a.splits, max(1, steps));
}

template <int CODE, int D>
__global__ __launch_bounds__(64 * ChunkShape<D>::NW) void block8_chunk_kernel(Block8AttendArgs a) {
    using C = ChunkShape<D>;
    constexpr int NW = C::NW, DS = C::DS, DW = D / DS;  // head dims of a wave
    constexpr int NB = DW / 32, NBLK = C::NBLK, KEYS = C::KEYS, PASSES = C::PASSES;
    __shared__ __align__(16) uint8_t lds[C::BUF];
    __shared__ __align__(16) ChunkScale scales[4][2 * NBLK];
    __shared__ float2 sml[C::RMIN < C::RB ? NW * 32 : 1];
    __shared__ __align__(16) uint8_t sx[C::SX], raw[C::RAW];
    __shared__ uint4 ql[C::QL ? NW * C::QL * 64 : 1];
    constexpr int NQ = DW / 16, QR = NQ - C::QL;  // Q operands, those in registers
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    // grid (head, split, tile): heads lie on XCDs of their own where they are 8
    const int size = 32 * a.row_waves;
    const int head = blockIdx.x, split = blockIdx.y, u = blockIdx.z;
    bool bad = false;
    int req, before;
    const bool mine = tile_request<NW>(a, size, u, req, before, bad);
    if (bad) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
    if (!mine) return;
    bool ignore = false;
    Rows r = load_rows(a, req, 0, size, ignore);
    const int tile = tiles_of(a, r, size) - 1 - (u - before);  // most keys first
    r = uniform(rows_of(a, r.start, r.count, r.length, tile, size));
    const int splits = splits_of<D>(a, r);
    if (split >= splits) return;

    int RW = C::RMIN;
    while (32 * RW < r.n) RW *= 2;
    const int KS = C::RB / RW;
    const int ds = wave & (DS - 1), rw = (wave / DS) & (RW - 1), part = wave / DS / RW;
    const int row0 = size * tile + 32 * rw, rows = r.count * a.group;
    const bool wlive = 32 * rw < r.n, valid = wlive && row0 + col < rows;
    const int row = valid ? row0 + col : size * tile;
    const int qr = row / a.group, hr = row - qr * a.group;
    const int base = r.length - r.count, pos = base + qr;
    // positions of this wave's first and last query
    const int wfirst = base + row0 / a.group, wlast = base + (min(rows, row0 + 32) - 1) / a.group;

    // the split's keys: steps [s0, s1) of KEYS from k0 on
    const int k0 = r.kstart / 32 * 32;
    const int steps = (r.kend - k0 + KEYS - 1) / KEYS;
    const int s0 = steps * split / splits, s1 = steps * (split + 1) / splits;

    // Q^T operands: lane (row col, half) holds dims 16c + 8half + 0..7 of its row, scaled
    // by a power of two so that the row's largest element lies in [2^14, 2^15)
    uint4 qop[QR];
    float qscale;
    {
        const uint16_t *q = a.q + (int64_t)(r.start + qr) * a.q_row + (int64_t)(head * a.group + hr) * a.q_head + 8 * half +
                            ds * DW;
        uint4 qraw[NQ];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
            const uint4 w = *reinterpret_cast<const uint4 *>(q + 16 * c);  // (lanes without a row: the tile's first)
            qraw[c] = w;
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, max(ws[i] & 0x7fffu, (ws[i] >> 16) & 0x7fffu));
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        if constexpr (DS > 1) {  // the row's largest element over both waves' dims
            uint32_t *tops = reinterpret_cast<uint32_t *>(sx);
            if (half == 0) tops[wave * 32 + col] = top;
            __syncthreads();
            top = max(top, tops[(wave ^ 1) * 32 + col]);
            __syncthreads();
        }
        const int shift = 14 + 127 - (int)max(top >> 7, 1u);
        const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
        qscale = fabsf(a.scale_log2) * ldexpf(1.0f, -shift);
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
            const uint32_t ws[4] = {qraw[c].x ^ flip, qraw[c].y ^ flip, qraw[c].z ^ flip, qraw[c].w ^ flip};
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = pack_f16(ldexpf(bf16_lo(ws[i]), shift), ldexpf(bf16_hi(ws[i]), shift));
            if (c < QR) qop[c < QR ? c : 0] = make_uint4(x[0], x[1], x[2], x[3]);
            else ql[(wave * C::QL + c - QR) * 64 + lane] = make_uint4(x[0], x[1], x[2], x[3]);
        }
    }

    float m = kNegBig, l = 0.f;
    f32x16_t o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] = 0.f;

    // ---- staging
    constexpr int LPR = D / 16, RPP = 64 * NW / LPR, RPWV = 64 / LPR;  // lanes per row, rows per pass and per wave of it
    const int srow = threadIdx.x / LPR, schunk = threadIdx.x % LPR;
    uint4 kr[C::DMA ? 1 : PASSES], vr[C::DMA ? 1 : PASSES];
    bool kok[PASSES], vok[PASSES];  // on mapped pages
    int ids = 0;
    const uint32_t raw_at = lds_addr(raw) + wave * PASSES * 2048;  // this wave's [pass][K, V][lane]
    // scales of 16-key block sblk of the next step, and the page of the step after it: its
    // entry is loaded a step before it is looked up. (All lanes load, a few store: loads
    // under a condition are copied behind it, which waits for them.)
    const int sblk = threadIdx.x & (2 * NBLK - 1);
    float next_k = 0.f, next_v = 0.f;
    int next_id = 0;
    bool unmapped = false, next_ok = false;
    auto load_scale_id = [&](int s) __attribute__((always_inline)) {
        next_id = a.table[(int64_t)req * a.table_stride + (min(k0 + s * KEYS + 16 * sblk, r.kend - 1) >> a.p.shift)];
    };
    // The pages of a step's passes, pass p's in lane p: a wave's rows of a pass lie in one
    // 16-key block, so on one page. A vector load, since waits for LDS reads do not include it.
    auto load_ids = [&](int s) __attribute__((always_inline)) {
        const int key = k0 + s * KEYS + (lane & (PASSES - 1)) * RPP + wave * RPWV;
        ids = a.table[(int64_t)req * a.table_stride + (min(key, r.kend - 1) >> a.p.shift)];
    };
    // Codes of step s to registers (D 512: to LDS). Nothing here may read them: that would
    // wait for the load in front of the step's work (one request of 512 rows, D 512, 4096
    // keys: 238 us for 136, when that was changed).
    auto fetch = [&](auto v_c, int s, int ids) __attribute__((always_inline)) {
        constexpr bool V = decltype(v_c)::value;
        const uint8_t *codes = V ? a.p.v : a.p.k;
        const int key0 = k0 + s * KEYS;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int wkey = key0 + p * RPP + wave * RPWV, id = __builtin_amdgcn_readlane(ids, p);
            const bool ok = (unsigned)id < (unsigned)a.p.pages;
            const int64_t at = ((((int64_t)(ok ? id : 0) * a.p.kv_heads + head) << a.p.shift) + (wkey & (a.p.block - 1))) * D;
            const uint32_t lane_at = 16 * lane;  // a wave's rows are contiguous
            if constexpr (C::DMA) {
                dma_load16_cached(codes + at + lane_at, raw_at + p * 2048 + (V ? 1024 : 0));
            } else {
                (V ? vr[p] : kr[p]) = *reinterpret_cast<const uint4 *>(codes + at + lane_at);
            }
            (V ? vok[p] : kok[p]) = ok;
        }
    };
    auto fetch_scales = [&](int s) __attribute__((always_inline)) {
        const int key = k0 + s * KEYS + 16 * sblk;
        next_ok = (unsigned)next_id < (unsigned)a.p.pages;
        unmapped |= !next_ok && key < r.kend && key + 16 > r.kstart;
        const int64_t at = (int64_t)(next_ok ? next_id : 0) * a.p.kv_heads + head;
        next_v = a.p.v_scale[at];
        next_k = a.p.k_scale[at];
        load_scale_id(s + 1);
    };
    // one pass of a step's K or V to LDS as fp16; keys nobody sees (before the window, past
    // the last, on unmapped pages) as zeros
    auto stage = [&](auto v_c, auto p_c, int slot, int s) __attribute__((always_inline)) {
        constexpr bool V = decltype(v_c)::value;
        constexpr int p = decltype(p_c)::value;
        uint8_t *to = lds + (V ? C::VBASE + slot * C::VSLOT : slot * C::KSLOT);
        const int rr = p * RPP + srow;
        uint4 w;
        const int wkey = k0 + s * KEYS + p * RPP + wave * RPWV, key = k0 + s * KEYS + rr;
        const bool ok = V ? vok[p] : kok[p];
        if constexpr (C::DMA) {
            if (p == 0) wait_vmem<0>();  // a lane reads what it fetched itself
            w = reinterpret_cast<const uint4 *>(raw)[(wave * PASSES + p) * 128 + (V ? 64 : 0) + lane];
        } else {
            w = V ? vr[p] : kr[p];
        }
        if (__builtin_amdgcn_readfirstlane(!ok || wkey + RPWV > r.kend || wkey < r.kstart)) {
            const bool data = ok && key < r.kend && key >= r.kstart;
            w = data ? w : make_uint4(0, 0, 0, 0);
        }
        write_f16<CODE>(to + rr * (V ? C::VP : C::KP) + 32 * schunk, w);
        if constexpr (C::DMA)
            if (p == PASSES - 1) wait_lds();  // read before the next step's codes land there
    };
    auto stage_scales = [&](int s) __attribute__((always_inline)) {
        if (threadIdx.x < 2 * NBLK) {
            const float v = scale_in_range(next_v);
            scales[s & 3][sblk] = ChunkScale{scale_in_range(next_k), __builtin_amdgcn_logf(v), __builtin_amdgcn_rcpf(v),
                                             next_ok ? 1.f : 0.f};
        }
    };
    auto stage_all = [&](auto v_c, int slot, int s) __attribute__((always_inline)) {
        ChunkFor<0, PASSES>::run([&](auto p_c) __attribute__((always_inline)) { stage(v_c, p_c, slot, s); });
    };
    constexpr std::false_type kK{};
    constexpr std::true_type kV{};

    // ---- one 32-key block, in steps of one MFMA: operands are read PK (PV) steps ahead;
    // sched_barrier holds that order
    const int kadr = col * C::KP + 16 * half + 2 * ds * DW;
    const int s16 = lane & 15;
    const int vadr = C::VBASE + (4 * half + (s16 >> 2)) * C::VP + 32 * ((lane >> 4) & 1) + 8 * (s16 & 3) + 2 * ds * DW;
    constexpr int NP = 2 * NB, PK = D == 512 ? 2 : NQ, PV = D == 512 ? 2 : NP;
    auto qk = [&](f32x16_t &s, int slot, int blk) __attribute__((always_inline)) {
        const uint8_t *kl = lds + slot * C::KSLOT + blk * 32 * C::KP + kadr;
        uint4 x[PK];
#pragma unroll
        for (int c = 0; c < PK; ++c) x[c] = *reinterpret_cast<const uint4 *>(kl + 32 * c);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
        __builtin_amdgcn_sched_barrier(0);
        ChunkFor<0, NQ>::run([&](auto c_c) __attribute__((always_inline)) {
            constexpr int c = decltype(c_c)::value;
            s = mfma32_f16(x[c % PK], c < QR ? qop[c < QR ? c : 0] : ql[(wave * C::QL + c - QR) * 64 + lane], s);
            if constexpr (c + PK < NQ) x[c % PK] = *reinterpret_cast<const uint4 *>(kl + 32 * (c + PK));
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    uint32_t w[8];  // the weights: of 16 keys in w[0 .. 3], of the next 16 in w[4 .. 7]
    auto pv = [&](int slot, int blk) __attribute__((always_inline)) {
        const uint8_t *vl = lds + slot * C::VSLOT + blk * 32 * C::VP + vadr;
        auto vop = [&](int u) __attribute__((always_inline)) {
            const uint8_t *p = vl + 16 * (u / NB) * C::VP + 64 * (u % NB);
            const uint2 lo = lds_read_tr16(reinterpret_cast<const uint16_t *>(p));
            const uint2 hi = lds_read_tr16(reinterpret_cast<const uint16_t *>(p + 8 * C::VP));
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        };
        uint4 x[PV];
#pragma unroll
        for (int u = 0; u < PV; ++u) x[u] = vop(u);
        __builtin_amdgcn_sched_barrier(0);
        ChunkFor<0, NP>::run([&](auto u_c) __attribute__((always_inline)) {
            constexpr int u = decltype(u_c)::value, h = u / NB;
            o[u % NB] = mfma32_f16(x[u % PV], make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]), o[u % NB]);
            if constexpr (u + PV < NP) x[u % PV] = vop(u + PV);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto mask = [&](f32x16_t &s, int key0, const ChunkScale (&sc)[2]) __attribute__((always_inline)) {
        const bool whole = key0 + 32 <= min(r.kend, wfirst + 1) && (a.window <= 0 || key0 > wlast - a.window) &&
                           sc[0].ok + sc[1].ok == 2.f;
        if (__builtin_amdgcn_readfirstlane(whole)) return;
        const int low = a.window > 0 ? pos - a.window : -1, high = min(pos, r.kend - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int lo = sc[h].ok != 0.f ? low : high;  // (then nothing lies between them)
#pragma unroll
            for (int i = 8 * h; i < 8 * h + 8; ++i) {
                const int key = key0 + 8 * (i >> 2) + 4 * half + (i & 3);
                s[i] = key > lo && key <= high ? s[i] : -INFINITY;
            }
        }
    };
    // the running max over s (the exponents are s * cf + log2(v scale))
    float cf[2];
    auto take_max = [&](const f32x16_t &s, const ChunkScale (&sc)[2]) __attribute__((always_inline)) {
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            cf[h] = fmaxf(qscale * sc[h].k, 1e-37f);  // above 0, so that a masked score stays one
            float t = s[8 * h];
#pragma unroll
            for (int i = 1; i < 8; ++i) t = fmaxf(t, s[8 * h + i]);
            top = fmaxf(top, fmaf(t, cf[h], sc[h].log_v));
        }
        top = pair<OpMax, 32>(top);
        const float mn = top > m + kRescaleSlack ? top : m;
        if (__any(mn != m)) {
            const float corr = __builtin_amdgcn_exp2f(m - mn);
            l *= corr;
#pragma unroll
            for (int b = 0; b < NB; ++b) o[b] *= corr;
            m = mn;
        }
    };
    auto soft = [&](const f32x16_t &s, const ChunkScale (&sc)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float d = sc[h].log_v + (kWeightShift - m);
            float sum = 0.f;  // in fp32: a page of small values has weights that fp16 drops but the sum needs
#pragma unroll
            for (int j = 4 * h; j < 4 * h + 4; ++j) {
                const float e0 = __builtin_amdgcn_exp2f(fmaf(s[2 * j], cf[h], d));
                const float e1 = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], cf[h], d));
                sum += e0 + e1;
                w[j] = pack_f16(e0, e1);
            }
            l = fmaf(sum, sc[h].inv_v, l);
            if (D == 512) __builtin_amdgcn_sched_barrier(0);
        }
    };
    // whether some row of the wave sees some of keys first .. first + 31
    auto sees = [&](int first) __attribute__((always_inline)) {
        return wlive && first <= wlast && first < r.kend && (a.window <= 0 || first + 32 > wfirst - a.window + 1);
    };
    // s to the weights w (DS > 1: s is this wave's half, the other's is in sx)
    f32x16_t sc;
    const int kx = wave * 256 + lane;
    auto give_scores = [&]() __attribute__((always_inline)) {
        if constexpr (DS > 1)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                reinterpret_cast<float4 *>(sx)[kx + g * 64] = make_float4(sc[4 * g], sc[4 * g + 1], sc[4 * g + 2], sc[4 * g + 3]);
    };
    auto weights = [&](int s, int blk) __attribute__((always_inline)) {
        if constexpr (DS > 1) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 x = reinterpret_cast<const float4 *>(sx)[(kx ^ 256) + g * 64];
                sc[4 * g] += x.x, sc[4 * g + 1] += x.y, sc[4 * g + 2] += x.z, sc[4 * g + 3] += x.w;
                if (D == 512 && g == 1) __builtin_amdgcn_sched_barrier(0);
            }
        }
        const ChunkScale two[2] = {scales[s & 3][2 * blk], scales[s & 3][2 * blk + 1]};
        mask(sc, k0 + s * KEYS + 32 * blk, two);
        take_max(sc, two);
        soft(sc, two);
    };

    if (s0 < s1) {
        load_ids(s0);
        load_scale_id(s0);
        int now = ids;
        load_ids(s0 + 1);
        fetch(kK, s0, now);
        fetch(kV, s0, now);
        fetch_scales(s0);
        if constexpr (C::SLOTS == 3) {
            // Four waves work on the matrix cores (M: P V of a block, then K Q^T of the next)
            // while the four beside them on the same SIMDs do a softmax (V), and the other
            // way round; a barrier ends each phase. In V the codes of K two steps ahead and
            // of V one step ahead are staged: with three slots no slot is written that a
            // wave one phase behind still reads, and what a wave one phase ahead reads is
            // whole.
            int past = ids;  // pages of the step whose V is fetched next
            load_ids(s0 + 2);
            stage_all(kK, 0, s0);
            stage_scales(s0);
            fetch(kK, s0 + 1, past);
            fetch_scales(s0 + 1);
            stage_all(kV, 0, s0);
            fetch(kV, s0 + 1, past);
            stage_all(kK, 1, s0 + 1);
            stage_scales(s0 + 1);
            past = ids;
            load_ids(s0 + 3);
            fetch(kK, s0 + 2, past);
            fetch_scales(s0 + 2);
            __syncthreads();
            const bool behind = wave >= NW / 2;
            if (behind) __syncthreads();
            int slot = 0;
            bool live = part == 0 && sees(k0 + s0 * KEYS);
            if (live) {
                qk(sc, 0, 0);
                give_scores();
            }
            __syncthreads();
            for (int s = s0; s < s1; ++s) {
                const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot1 == 2 ? 0 : slot1 + 1;
                if (live) weights(s, 0);
                stage_all(kV, slot1, s + 1);
                fetch(kV, s + 2, past);
                stage_all(kK, slot2, s + 2);
                stage_scales(s + 2);
                past = ids;
                load_ids(s + 4);  // looked up a step later
                fetch(kK, s + 3, past);
                fetch_scales(s + 3);
                __syncthreads();
                if (live) pv(slot, 0);
                live = part == 0 && s + 1 < s1 && sees(k0 + (s + 1) * KEYS);
                if (live) {
                    qk(sc, slot1, 0);
                    give_scores();
                }
                __syncthreads();
                slot = slot1;
            }
            if (!behind) __syncthreads();
        } else if constexpr (C::SLOTS == 2) {
            // the waves run freely within a step: one's matrix work lies beside another's
            // softmax without being told to
            auto stage_step = [&](int slot, int s) __attribute__((always_inline)) {
                stage_all(kK, slot, s);
                stage_all(kV, slot, s);
                stage_scales(s);
            };
            stage_step(0, s0);
            __syncthreads();
            for (int s = s0; s < s1; ++s) {
                const int slot = (s - s0) & 1;
                if (s + 1 < s1) {
                    now = ids;
                    load_ids(s + 2);
                    fetch(kK, s + 1, now);
                    fetch(kV, s + 1, now);
                    fetch_scales(s + 1);
                }
                for (int blk = part; blk < NBLK; blk += KS) {
                    if (!sees(k0 + s * KEYS + 32 * blk)) continue;
                    qk(sc, slot, blk);
                    weights(s, blk);
                    pv(slot, blk);
                }
                if (s + 1 < s1) stage_step(slot ^ 1, s + 1);
                __syncthreads();
            }
        } else {
            for (int s = s0; s < s1; ++s) {
                if (s > s0) __syncthreads();  // the last step's blocks are read
                stage_all(kK, 0, s);
                stage_all(kV, 0, s);
                stage_scales(s);
                if (s + 1 < s1) {
                    now = ids;
                    load_ids(s + 2);
                    fetch(kK, s + 1, now);
                    fetch(kV, s + 1, now);
                    fetch_scales(s + 1);
                }
                __syncthreads();
                const bool live = part == 0 && sees(k0 + s * KEYS);
                if (live) {
                    qk(sc, 0, 0);
                    give_scores();
                }
                __syncthreads();
                if (live) {
                    weights(s, 0);
                    pv(0, 0);
                }
            }
        }
    }
    if (unmapped) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
    l = pair<OpSum, 32>(l);

    // ---- the answer, or this split's partial
    const int64_t slot = ((int64_t)u * a.p.kv_heads + head) * a.splits + split;
    // this lane's row again: kept over the loop it would cost registers that the loop needs
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int ecol = ln & 31, ehalf = ln >> 5, erow = row0 + ecol;
    const bool evalid = wlive && erow < rows;
    const int eq = (evalid ? erow : 0) / a.group, eh = (evalid ? erow : 0) - eq * a.group;
    uint16_t *const out = a.out + (int64_t)(r.start + eq) * a.o_row + (int64_t)(head * a.group + eh) * a.o_head;
    auto store4 = [&](int b, int g, float4 x, float inv) __attribute__((always_inline)) {
        const int d = ds * DW + 32 * b + 8 * g + 4 * ehalf;
        if (splits == 1) {
            *reinterpret_cast<uint2 *>(out + d) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
        } else {
            *reinterpret_cast<float4 *>(a.part_o + (slot * size + 32 * rw + ecol) * D + d) = x;
        }
    };
    if (KS == 1) {
        if (!evalid) return;
        const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                store4(b, g, make_float4(o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]), inv);
        if (splits > 1 && ehalf == 0 && ds == 0) a.part_ml[slot * size + 32 * rw + ecol] = make_float2(m, l);
        return;
    }
    if constexpr (C::RMIN < C::RB) {
    // combine the parts of each row block, BS 32-dim blocks at a time
    constexpr int BS0 = C::BUF / (NW * 4096), BS = BS0 >= NB ? NB : BS0 >= 8 ? 8 : BS0 >= 4 ? 4 : BS0 >= 2 ? 2 : 1;
    static_assert(BS * NW * 4096 <= C::BUF && NB % BS == 0, "the waves' blocks fit the buffers");
    __syncthreads();  // every wave is done with the buffers
    if (ehalf == 0) sml[wave * 32 + ecol] = make_float2(m, l);
    __syncthreads();
    float M = kNegBig, sum = 0.f;
    for (int p = 0; p < KS; ++p) M = fmaxf(M, sml[((p * RW + rw) * DS + ds) * 32 + ecol].x);
    for (int p = 0; p < KS; ++p) {
        const float2 x = sml[((p * RW + rw) * DS + ds) * 32 + ecol];
        sum = fmaf(x.y, __builtin_amdgcn_exp2f(x.x - M), sum);
    }
    const float f = __builtin_amdgcn_exp2f(m - M), inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    float4 *xl = reinterpret_cast<float4 *>(lds);  // [wave][block][g][lane]
#pragma unroll
    for (int b0 = 0; b0 < NB; b0 += BS) {
        if (b0 > 0) __syncthreads();
#pragma unroll
        for (int b = 0; b < BS; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                xl[((wave * BS + b) * 4 + g) * 64 + ln] = make_float4(o[b0 + b][4 * g] * f, o[b0 + b][4 * g + 1] * f,
                                                                     o[b0 + b][4 * g + 2] * f, o[b0 + b][4 * g + 3] * f);
        __syncthreads();
        for (int e = part; e < 4 * BS; e += KS) {
            float4 x = xl[((rw * DS + ds) * BS * 4 + e) * 64 + ln];
            for (int p = 1; p < KS; ++p) {
                const float4 y = xl[(((p * RW + rw) * DS + ds) * BS * 4 + e) * 64 + ln];
                x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
            }
            if (evalid) store4(b0 + e / 4, e % 4, x, inv);
        }
    }
    if (splits > 1 && part == 0 && ds == 0 && ehalf == 0 && evalid) a.part_ml[slot * size + 32 * rw + ecol] = make_float2(M, sum);
    }
}

// Joins the splits of a row, in their order: a row's D/4 threads each take four
// elements; grid (head, row group, tile). Four partials at a time, for many waves on a
// CU: with sixteen (172 registers) it took 17 us for 2328 rows of D 256 in 3 splits.
template <int D>
__global__ __launch_bounds__(256) void block8_chunk_join_kernel(Block8AttendArgs a) {
    constexpr int LANES = D / 4, ROWS = 256 / LANES;
    const int size = 32 * a.row_waves, head = blockIdx.x, u = blockIdx.z;
    int req, before;
    bool ignore = false;
    if (!tile_request<4>(a, size, u, req, before, ignore)) return;
    Rows r = load_rows(a, req, 0, size, ignore);
    const int tile = tiles_of(a, r, size) - 1 - (u - before);
    r = rows_of(a, r.start, r.count, r.length, tile, size);
    const int splits = splits_of<D>(a, r), rr = blockIdx.y * ROWS + threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES);
    if (splits == 1 || rr >= r.n) return;
    const int64_t slot0 = ((int64_t)u * a.p.kv_heads + head) * a.splits;
    float M = kNegBig, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    join_partials<4>(splits, [&](int p, float2 &ml, float4 &y) __attribute__((always_inline)) {
        const int64_t at = (slot0 + p) * size + rr;
        ml = a.part_ml[at];
        y = *reinterpret_cast<const float4 *>(a.part_o + at * D + d);
    }, M, sum, x);
    store_out(a, r, head, size * tile + rr, d, x, sum);
}

template <int CODE, int D>
static hipError_t launch_chunk(const Block8AttendArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((block8_chunk_kernel<CODE, D>), dim3(a.p.kv_heads, a.splits, a.tiles),
                       dim3(64 * ChunkShape<D>::NW), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    const int rows = std::min(32 * a.row_waves, a.group * a.max_q), per = 1024 / D;
    hipLaunchKernelGGL((block8_chunk_join_kernel<D>), dim3(a.p.kv_heads, (rows + per - 1) / per, a.tiles), dim3(256), 0, s,
                       a);
    return hipGetLastError();
}

}  // namespace kvrt
