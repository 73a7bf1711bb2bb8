// kvrt_block8_attend.hip — attention of packed query rows over 8-bit pages with one
// scale per (page, KV head).
//
// The rows of a (request, KV head) are its q heads x queries, query first (row r:
// query r / g, head r % g); a tile is 16 of them. Per 32 keys one wave computes,
// with codes as fp16 (exact) and every query row scaled by a power of two to fp16's
// upper range (exact to 2^-38 of the row's largest element):
//   S^T (16 keys x 16 rows) = K Q^T        2 * D/32 v_mfma_f32_16x16x32_f16
//   t = S * k_scale * scale + log2(v_scale)
//   p = 2^(t - m)            m: running max of t per row
//   l += p / v_scale         O^T (D x 16) += V^T P^T   D/16 v_mfma_f32_16x16x32_f16
// and out = O / l: the page's V scale lives in the exponent, so P and the codes stay
// within fp16 whatever the scales, and one exponential serves both sums. m moves
// lazily (kRescaleSlack), and p carries a factor 2^7 that cancels: weights down to
// 2^-21 of the largest keep fp16's full 11 bits (2^-12 relative).
//
// Long contexts are bound by HBM, short ones by a chain of launch, division of the keys
// (2.5 us), first loads (2.5-3 us) and, where a head's keys lie over several workgroups,
// their join (3-4.5 us in the launch, 7 us for D 512's larger parts in a second one);
// beside those a 32-key tile costs a wave about 0.5 us at D 128, 1 us at D 256, of vector
// work. Measured: 64 requests to 8100 keys, 16 heads over 8, D 128: 117 us (5.2 TB/s);
// four of 4100 keys 15.7 us; one of 512 keys, 8 heads over 1, D 256: 11.4 us; four of
// 8192 with two rows, D 512: 18.3 + 7.1 us.
//
// Lane layouts (16x16x32): A[row l%16][k 8(l/16)+j], B[k 8(l/16)+j][col l%16],
// D[row 4(l/16)+i][col l%16]. The products' inner indices are free: K and Q order
// head dims so that a lane's 16 bytes of a key row are two operands, and keys are
// ordered in P V so that a lane's own weights are its operand: k = 8(l/16)+j is key
// 16(j/4) + 4(l/16) + j%4. V is read row by row, D/16 bytes per lane, and
// transposed in registers by byte permutes.
#include <algorithm>
#include <map>
#include <mutex>
#include <utility>

#include "kvrt_block8_rows.h"

namespace kvrt {

namespace {

constexpr int kTileKeys = 32, kUnitTiles = 4;  // a unit of division: one 32-key tile per wave

// Units of a head of the request. Rows without keys are one too: their zeros have to
// be written.
__device__ __forceinline__ int units_of(const Rows &r) {
    const int tiles = (r.kend + kTileKeys - 1) / kTileKeys - r.kstart / kTileKeys;
    return r.n == 0 ? 0 : max(1, (tiles + kUnitTiles - 1) / kUnitTiles);
}

// How the units of all requests' heads (request, head, unit order) are divided:
// workgroup w has units [w * per, (w + 1) * per). The host keeps their number
// below 2^31.
struct Division {
    int total, per;
};
__device__ __forceinline__ Division divide(const Block8AttendArgs &a, int units, int most) {
    Division d;
    d.total = units * a.p.kv_heads;
    d.per = (d.total + a.wgs - 1) / a.wgs;
    // n units in a row lie over at most (n - 1) / per + 2 workgroups, no head's over more
    // than one may join (join_most >= 2)
    if (a.join_all) d.per = max(d.per, (most + a.join_most - 2) / (a.join_most - 1));
    return d;
}

// N dwords of a lane from p (N = 1, 2, 4, 8; p aligned to min(4 N, 16) bytes).
template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t *p, uint32_t (&w)[N]) {
    if constexpr (N == 1) {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(p + 4 * i);
            w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
    }
}

__device__ __forceinline__ f32x4_t mfma16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4_t c) {
    const u32x4_t x = {a[0], a[1], a[2], a[3]}, y = {b[0], b[1], b[2], b[3]};
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x), __builtin_bit_cast(f16x8_t, y), c, 0, 0,
                                                  0);
}

// Q^T of a row tile as fp16 operands: lane (row l%16, group l/16) holds for step c
// the dims 64(c/2) + 16(l/16) + 8(c%2) + 0..7 of its row, scaled by 2^shift so that
// the row's largest element lies in [2^14, 2^15). back: 2^-shift. Lanes without a row
// are given another's: loads that only some lanes make are a divergent region, and
// the registers are too full for one.
template <int D>
__device__ __forceinline__ void load_query(const uint16_t *row, uint32_t flip, uint32_t (&op)[D / 32][4],
                                           float &back) {
    const int grp = (threadIdx.x & 63) >> 4;
    uint4 raw[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
        raw[c] = *reinterpret_cast<const uint4 *>(row + 64 * (c / 2) + 16 * grp + 8 * (c % 2));
    uint32_t top = 0;  // largest exponent field (with mantissa: bits of |x|)
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    // 2^(e - 127) <= largest < 2^(e - 126); subnormal rows count as e = 1
    const int e = (int)max(top >> 7, 1u);
    const int shift = 14 + 127 - e;
    back = ldexpf(1.0f, -shift);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        const uint32_t w[4] = {raw[c].x ^ flip, raw[c].y ^ flip, raw[c].z ^ flip, raw[c].w ^ flip};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            op[c][i] = pack_f16(ldexpf(bf16_lo(w[i]), shift), ldexpf(bf16_hi(w[i]), shift));
    }
}

}  // namespace

template <int CODE, int D>
__global__ __launch_bounds__(256) void block8_attend_kernel(Block8AttendArgs a) {
    constexpr int NB = D / 16;    // 16-dim blocks of the output
    constexpr int KC = D / 64;    // 16-byte chunks of a key row per lane
    constexpr int VW = D / 64;    // dwords of a V row per lane
    constexpr int PITCH = D + 4;  // floats of an output row in LDS: 16 rows on 16 different bank quadruples
    __shared__ __align__(16) float so[4 * 16 * PITCH];
    __shared__ float2 sml[4 * 16];
    __shared__ int scan_lds[8], found[2];
    __shared__ uint32_t arrived;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    constexpr int tile = 0;  // a head's rows are one tile
    const int wg = blockIdx.x;

    // this workgroup's units [u, uend), the request of the first and the units before it
    bool bad = false, unmapped = false;
    Division div;
    int req, before, u;
    Rows mine{};  // of request `lane`, where there are at most 64
    if (a.n <= 64) {
        int units = 0;
        if (lane < a.n) {
            mine = load_rows(a, lane, tile, 16, bad);
            units = units_of(mine);
        }
        int inc = units, top = units;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(inc, d);
            if (lane >= d) inc += y;
            top = max(top, __shfl_xor(top, d));
        }
        div = divide(a, __builtin_amdgcn_readlane(inc, 63), __builtin_amdgcn_readfirstlane(top));
        u = wg * div.per;
        const int end = inc * a.p.kv_heads;
        const uint64_t past = __ballot(end > u);
        if (past == 0) {
            if (bad) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
            return;
        }
        req = __builtin_ctzll(past);
        before = __builtin_amdgcn_readlane(end - units * a.p.kv_heads, req);
    } else {
        int all = 0, most = 0;
        for (int base = 0; base < a.n; base += 256) {
            const int i = base + threadIdx.x;
            int sum, top;
            scan_wg<4>(i < a.n ? units_of(load_rows(a, i, tile, 16, bad)) : 0, scan_lds, sum, top);
            all += sum;
            most = max(most, top);
        }
        div = divide(a, all, most);
        u = wg * div.per;
        if (u < div.total) {
            int at = 0;
            for (int base = 0; base < a.n; base += 256) {
                const int i = base + threadIdx.x;
                const int units = i < a.n ? units_of(load_rows(a, i, tile, 16, bad)) * a.p.kv_heads : 0;
                int sum, top;
                const int first = at + scan_wg<4>(units, scan_lds, sum, top);
                at += sum;
                if (first <= u && u < first + units) found[0] = i, found[1] = first;
            }
            __syncthreads();
        } else {
            if (bad) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
            return;
        }
        req = __builtin_amdgcn_readfirstlane(found[0]);
        before = __builtin_amdgcn_readfirstlane(found[1]);
    }
    if (bad) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
    const int uend = min(div.total, u + div.per);
    const float scale = fabsf(a.scale_log2);
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const ConstInts table = (ConstInts)(uintptr_t)a.table;
    const ConstFloats k_scale = (ConstFloats)(uintptr_t)a.p.k_scale, v_scale = (ConstFloats)(uintptr_t)a.p.v_scale;

    while (u < uend) {
        Rows r;
        if (a.n <= 64) {
            r = rows_of(a, __builtin_amdgcn_readlane(mine.start, req), __builtin_amdgcn_readlane(mine.count, req),
                        __builtin_amdgcn_readlane(mine.length, req), tile, 16);
        } else {
            bool ignore = false;
            r = load_rows(a, req, tile, 16, ignore);
        }
        r = uniform(r);
        const int units = units_of(r);
        if (u >= before + units * a.p.kv_heads) {
            before += units * a.p.kv_heads;
            ++req;
            continue;
        }
        const int head = (u - before) / units;
        const int seg = before + head * units;  // the head's first unit
        const int ua = u - seg, ub = min(units, uend - seg);
        const int first_tile = r.kstart / kTileKeys;
        const int t_end = min(first_tile + ub * kUnitTiles, (r.kend + kTileKeys - 1) / kTileKeys);
        const int t_begin = first_tile + ua * kUnitTiles + wave;

        // this lane's row (a column of S^T and O^T)
        const bool valid = col < r.n;
        const int row = 16 * tile + (valid ? col : 0);
        const int qr = row / a.group, hr = row - qr * a.group;
        const int pos = r.length - r.count + qr;

        if (t_begin < t_end) {
            // keys every row of the tile sees
            const int all_lo = a.window > 0 ? r.last - a.window + 1 : 0, all_hi = min(r.first + 1, r.kend);
            const ConstInts entries = table + (int64_t)req * a.table_stride;
            const int64_t head_bytes = (int64_t)a.p.block * D;
            uint32_t kc[2][KC][4], vc[2][4][VW];
            float ks[2], vs[2];
            bool ok[2];
            int page[2], ids[2];
            // the table's entries for a tile's two 16-key halves; past the range the last key's
            auto load_ids = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) ids[h] = entries[min(t * kTileKeys + 16 * h, r.kend - 1) >> a.p.shift];
            };
            auto take_pages = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    ok[h] = (unsigned)ids[h] < (unsigned)a.p.pages;
                    page[h] = ok[h] ? ids[h] : 0;
                }
            };
            // byte offset of a half's 16 rows of this head
            auto half_at = [&](int t, int h) __attribute__((always_inline)) {
                return ((int64_t)page[h] * a.p.kv_heads + head) * head_bytes +
                       (int64_t)((t * kTileKeys + 16 * h) & (a.p.block - 1)) * D;
            };
            auto load_k = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t *p = a.p.k + half_at(t, h) + (uint32_t)(col * D + 16 * grp);
#pragma unroll
                    for (int c = 0; c < KC; ++c) load_dwords<4>(p + 64 * c, kc[h][c]);
                    ks[h] = k_scale[(int64_t)page[h] * a.p.kv_heads + head];
                }
            };
            auto load_v = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t *p = a.p.v + half_at(t, h) + (uint32_t)(4 * grp * D + col * (D / 16));
#pragma unroll
                    for (int j = 0; j < 4; ++j) load_dwords<VW>(p + j * D, vc[h][j]);
                    vs[h] = v_scale[(int64_t)page[h] * a.p.kv_heads + head];
                }
            };
            load_ids(t_begin);
            uint32_t qop[D / 32][4];
            float back;
            take_pages();
            load_k(t_begin);
            load_v(t_begin);
            load_query<D>(a.q + (int64_t)(r.start + qr) * a.q_row + (int64_t)(head * a.group + hr) * a.q_head, flip, qop,
                          back);
            load_ids(min(t_begin + kUnitTiles, t_end - 1));
            const float qscale = scale * back;
            float m = kNegBig, l = 0.f;
            f32x4_t o[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) o[b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

            for (int t = t_begin; t < t_end; t += kUnitTiles) {
                // past the last tile: read again, not used
                const int next = min(t + kUnitTiles, t_end - 1), after = min(t + 2 * kUnitTiles, t_end - 1);
                // scores
                f32x4_t s[2];
                float lv[2], inv_vs[2], cf[2];
                bool good[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[h] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
                        uint32_t x[2][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            codes_to_f16<CODE>(kc[h][c][e], x[e / 2][2 * (e % 2)], x[e / 2][2 * (e % 2) + 1]);
                        s[h] = mfma16(x[0], qop[2 * c], s[h]);
                        s[h] = mfma16(x[1], qop[2 * c + 1], s[h]);
                    }
                    const float v = scale_in_range(vs[h]);
                    lv[h] = __builtin_amdgcn_logf(v);
                    inv_vs[h] = __builtin_amdgcn_rcpf(v);  // within 1 ulp
                    cf[h] = qscale * scale_in_range(ks[h]);
                    good[h] = ok[h];
                }
                take_pages();
                load_k(next);
                load_ids(after);
                // t = S * cf + lv, masked where a row does not see the key
                const int key0 = t * kTileKeys;
                const bool whole = key0 >= all_lo && key0 + kTileKeys <= all_hi && good[0] && good[1];
                float w[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[h][i] = fmaf(s[h][i], cf[h], lv[h]);
                if (!whole) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        unmapped |= !good[h] && key0 + 16 * h < r.kend && key0 + 16 * h + 16 > r.kstart;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = key0 + 16 * h + 4 * grp + i;
                            const bool seen = good[h] && key <= pos && key < r.kend && (a.window <= 0 || key > pos - a.window);
                            w[h][i] = seen ? w[h][i] : -INFINITY;
                            // rows that nobody sees may hold anything: 0 * NaN is not 0
                            const bool data = good[h] && key >= r.kstart && key < r.kend;
#pragma unroll
                            for (int e = 0; e < VW; ++e) vc[h][i][e] = data ? vc[h][i][e] : 0u;
                        }
                    }
                }
                float top = fmaxf(fmaxf(fmaxf(w[0][0], w[0][1]), fmaxf(w[0][2], w[0][3])),
                                  fmaxf(fmaxf(w[1][0], w[1][1]), fmaxf(w[1][2], w[1][3])));
                top = pair<OpMax, 32>(pair<OpMax, 16>(top));
                const float mn = top > m + kRescaleSlack ? top : m;
                if (__any(mn != m)) {
                    const float corr = __builtin_amdgcn_exp2f(m - mn);
                    l *= corr;
#pragma unroll
                    for (int b = 0; b < NB; ++b) o[b] *= corr;
                    m = mn;
                }
                uint32_t p[4];
                const float mo = kWeightShift - m;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(w[h][i] + mo);
                    l = fmaf((e[0] + e[1]) + (e[2] + e[3]), inv_vs[h], l);
                    p[2 * h] = pack_f16(e[0], e[1]);
                    p[2 * h + 1] = pack_f16(e[2], e[3]);
                }
                // O^T += V^T P^T: key pairs of four dims at a time
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    uint32_t x[4][4];  // [dim][key pair]
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t w0 = vc[h][2 * j][e], w1 = vc[h][2 * j + 1][e];
                            codes_to_f16<CODE>(__builtin_amdgcn_perm(w1, w0, 0x05010400u), x[0][2 * h + j], x[1][2 * h + j]);
                            codes_to_f16<CODE>(__builtin_amdgcn_perm(w1, w0, 0x07030602u), x[2][2 * h + j], x[3][2 * h + j]);
                        }
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[4 * e + d] = mfma16(x[d], p, o[4 * e + d]);
                }
                load_v(next);
            }
            l = pair<OpSum, 32>(pair<OpSum, 16>(l));
            if (valid) {
                if (grp == 0) sml[wave * 16 + col] = make_float2(m, l);
                float *dst = so + (wave * 16 + col) * PITCH + 4 * grp * NB;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int b = 0; b < NB; b += 4)
                        *reinterpret_cast<float4 *>(dst + i * NB + b) =
                            make_float4(o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]);
            }
        }
        __syncthreads();
        // join the waves that had keys: four elements of a row per thread
        const int parts = min(max(t_end - (t_begin - wave), 0), 4);
        const bool begins = ua == 0, ends = ub == units;
        const int w0 = seg / div.per, count = (seg + units - 1) / div.per - w0 + 1;  // workgroups of the head
        const bool here = a.counters && count <= a.join_most;                         // joined in this launch
        const int64_t slot0 = 0;
        for (int e = threadIdx.x; e < r.n * (D / 4); e += 256) {
            const int rr = e / (D / 4), d = 4 * (e % (D / 4));
            float M = kNegBig, sum = 0.f;
            for (int w = 0; w < parts; ++w) M = fmaxf(M, sml[w * 16 + rr].x);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = 0; w < parts; ++w) {
                const float2 ml = sml[w * 16 + rr];
                const float f = __builtin_amdgcn_exp2f(ml.x - M);
                const float4 y = *reinterpret_cast<const float4 *>(so + (w * 16 + rr) * PITCH + d);
                sum = fmaf(ml.y, f, sum);
                x = make_float4(fmaf(y.x, f, x.x), fmaf(y.y, f, x.y), fmaf(y.z, f, x.z), fmaf(y.w, f, x.w));
            }
            if (begins && ends) {
                store_out(a, r, head, 16 * tile + rr, d, x, sum);
            } else {
                // partial 0: the head's keys began in an earlier workgroup, 1: they begin here
                const int64_t slot = slot0 + 2 * wg + (begins ? 1 : 0);
                float *po = a.part_o + (slot * 16 + rr) * D + d;
                float2 *pm = a.part_ml + slot * 16 + rr;
                if (here) {
                    store_agent(reinterpret_cast<float2 *>(po), make_float2(x.x, x.y));
                    store_agent(reinterpret_cast<float2 *>(po + 2), make_float2(x.z, x.w));
                    if (d == 0) store_agent(pm, make_float2(M, sum));
                } else {
                    *reinterpret_cast<float4 *>(po) = x;
                    if (d == 0) *pm = make_float2(M, sum);
                }
            }
        }
        if (here && !(begins && ends)) {
            // the last of the head's workgroups to arrive joins their partials, in
            // workgroup order; it leaves the counter at zero
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's partials are stored
            __syncthreads();
            uint32_t *counter = a.counters + w0;
            if (threadIdx.x == 0) arrived = arrive_agent(counter);
            __syncthreads();
            if (arrived == (uint32_t)count - 1) {
                if (threadIdx.x == 0) clear_agent(counter);
                for (int e = threadIdx.x; e < r.n * (D / 4); e += 256) {
                    const int rr = e / (D / 4), d = 4 * (e % (D / 4));
                    float M = kNegBig, sum = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    join_partials(count, [&](int p, float2 &ml, float4 &y) __attribute__((always_inline)) {
                        const int64_t at = (slot0 + 2 * (w0 + p) + (p == 0 ? 1 : 0)) * 16 + rr;
                        ml = load_agent(a.part_ml + at);
                        const float2 lo = load_agent(reinterpret_cast<const float2 *>(a.part_o + at * D + d));
                        const float2 hi = load_agent(reinterpret_cast<const float2 *>(a.part_o + at * D + d + 2));
                        y = make_float4(lo.x, lo.y, hi.x, hi.y);
                    }, M, sum, x);
                    store_out(a, r, head, 16 * tile + rr, d, x, sum);
                }
            }
        }
        u = seg + ub;
        if (u < uend) __syncthreads();  // the sums are read before the next head's are written
    }
    if (unmapped) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
}

// Joins the partials of heads that the launch did not join (more workgroups shared them
// than one joins, or the call has no arrival counters): one workgroup per (request, KV
// head, row). Up to kFlat partials in their order, as the launch does; beyond, in GROUPS
// interleaved orders that are then joined.
constexpr int kFlat = 32;

template <int D>
__global__ __launch_bounds__(256) void block8_join_kernel(Block8AttendArgs a) {
    constexpr int LANES = D / 4, GROUPS = 256 / LANES;
    __shared__ int scan_lds[8];
    __shared__ float4 so[256];
    __shared__ float2 sml[256];
    constexpr int tile = 0;
    const int rr = blockIdx.y, head = blockIdx.x % a.p.kv_heads, req = blockIdx.x / a.p.kv_heads;
    bool bad = false;
    const Rows r = load_rows(a, req, tile, 16, bad);
    if (rr >= r.n) return;
    // units before the request, all, and the most of a head
    int all = 0, before = 0, most = 0;
    for (int base = 0; base < a.n; base += 256) {
        const int i = base + threadIdx.x;
        const int mine = i < a.n ? units_of(load_rows(a, i, tile, 16, bad)) : 0;
        int sum, less, top, ignore;
        scan_wg<4>(mine, scan_lds, sum, top);
        scan_wg<4>(i < req ? mine : 0, scan_lds, less, ignore);
        all += sum;
        before += less;
        most = max(most, top);
    }
    const Division div = divide(a, all, most);
    const int units = units_of(r), seg = before * a.p.kv_heads + head * units;
    const int w0 = seg / div.per, count = (seg + units - 1) / div.per - w0 + 1;
    if (count == 1 || (a.counters && count <= a.join_most)) return;
    const int group = threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES);
    const int groups = count <= kFlat ? 1 : GROUPS;
    float M = kNegBig, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (group < groups) {
        const int64_t slot0 = 2 * w0;
        join_partials((count - group + groups - 1) / groups, [&](int p, float2 &ml, float4 &y) __attribute__((always_inline)) {
            const int i = p * groups + group;
            const int64_t at = (slot0 + 2 * i + (i == 0 ? 1 : 0)) * 16 + rr;
            ml = a.part_ml[at];
            y = *reinterpret_cast<const float4 *>(a.part_o + at * D + d);
        }, M, sum, x);
    }
    if (groups > 1) {
        so[threadIdx.x] = x;
        sml[threadIdx.x] = make_float2(M, sum);
        __syncthreads();
        if (group != 0) return;
        M = kNegBig, sum = 0.f;
        x = make_float4(0.f, 0.f, 0.f, 0.f);
        join_partials(GROUPS, [&](int p, float2 &ml, float4 &y) __attribute__((always_inline)) {
            ml = sml[p * LANES + threadIdx.x];
            y = so[p * LANES + threadIdx.x];
        }, M, sum, x);
    } else if (group != 0) {
        return;
    }
    store_out(a, r, head, 16 * tile + rr, d, x, sum);
}

template <int CODE, int D>
static hipError_t launch_attend(const Block8AttendArgs &a, bool join, hipStream_t s) {
    hipLaunchKernelGGL((block8_attend_kernel<CODE, D>), dim3(a.wgs), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !join) return e;
    const int rows = (int)std::min<int64_t>(16, (int64_t)a.group * a.max_q);
    hipLaunchKernelGGL((block8_join_kernel<D>), dim3(a.n * a.p.kv_heads, rows), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int CODE>
static hipError_t launch_attend_code(const Block8AttendArgs &a, int head_dim, bool join, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_attend<CODE, 64>(a, join, s);
        case 128: return launch_attend<CODE, 128>(a, join, s);
        case 256: return launch_attend<CODE, 256>(a, join, s);
        case 512: return launch_attend<CODE, 512>(a, join, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_block8_attend(const Block8AttendArgs &a, int dtype, int head_dim, bool join, hipStream_t s) {
    return dtype == KVRT_INT8 ? launch_attend_code<KVRT_INT8>(a, head_dim, join, s)
                              : launch_attend_code<KVRT_E4M3>(a, head_dim, join, s);
}

// ---- arrival counters ---------------------------------------------------------------
//
// Zero at load and between launches. Calls on one stream run in order and share a
// slice. So do the calls that one capture records on one stream; their slice is the
// graph's for good, since it may be replayed beside anything else (a graph does not
// overlap itself). Eager streams have slices of their own kind, which captures cannot use
// up. Without a slice calls join in a second launch instead, and so do calls on
// hipStreamPerThread: that handle names another stream in each thread. Measured in graphs
// of 50 calls, with and without: four requests of up to 1500 keys 8.5 and 10.9 us, of
// 4159 keys 14.4 and 17.7, one request of 8100 keys and 63 of 100 18.2 and 24.2.
constexpr int kCaptureSlices = 448, kStreamSlices = 64;
static __device__ uint32_t block8_counters[(kCaptureSlices + kStreamSlices) * kBlock8MaxWgs];

uint32_t *block8_counter_slice(hipStream_t s) try {
    struct Device {
        uint32_t *base = nullptr;
        std::map<hipStream_t, int> streams;
        std::map<std::pair<unsigned long long, hipStream_t>, int> captures;  // by capture id, which is unique
    };
    static std::mutex mu;
    static std::map<int, Device> devices;
    if (s == hipStreamPerThread) return nullptr;
    int dev = 0;
    unsigned long long id = 0;
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess) e = hipStreamIsCapturing(s, &cs);
    if (e == hipSuccess && cs != hipStreamCaptureStatusNone) e = hipStreamGetCaptureInfo(s, &cs, &id);
    if (e != hipSuccess || cs == hipStreamCaptureStatusInvalidated) {
        (void)hipGetLastError();  // the launch that follows reports its own errors
        return nullptr;
    }
    std::lock_guard<std::mutex> lock(mu);
    Device &d = devices[dev];
    if (!d.base) {  // the first call may be a captured one, and the lookup may load the module
        hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
        void *at = nullptr;
        if (hipThreadExchangeStreamCaptureMode(&mode) != hipSuccess) return nullptr;
        e = hipGetSymbolAddress(&at, HIP_SYMBOL(block8_counters));
        (void)hipThreadExchangeStreamCaptureMode(&mode);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            return nullptr;
        }
        d.base = static_cast<uint32_t *>(at);
    }
    const auto slice = [&](auto &of, auto key, int first, int most) -> uint32_t * {
        const auto got = of.find(key);
        if (got == of.end() && (int)of.size() >= most) return nullptr;
        const int i = got != of.end() ? got->second : static_cast<int>(of.size());
        if (got == of.end()) of.emplace(key, i);
        return d.base + (size_t)(first + i) * kBlock8MaxWgs;
    };
    if (cs == hipStreamCaptureStatusActive) return slice(d.captures, std::make_pair(id, s), 0, kCaptureSlices);
    return slice(d.streams, s, kCaptureSlices, kStreamSlices);
} catch (...) {  // no memory for an entry
    return nullptr;
}

}  // namespace kvrt
