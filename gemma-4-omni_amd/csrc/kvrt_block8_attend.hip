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
// Lane layouts (16x16x32): A[row l%16][k 8(l/16)+j], B[k 8(l/16)+j][col l%16],
// D[row 4(l/16)+i][col l%16]. The products' inner indices are free: K and Q order
// head dims so that a lane's 16 bytes of a key row are two operands, and keys are
// ordered in P V so that a lane's own weights are its operand: k = 8(l/16)+j is key
// 16(j/4) + 4(l/16) + j%4. V is read row by row, D/16 bytes per lane, and
// transposed in registers by byte permutes.
#include "kvrt_block8.h"

namespace kvrt {

namespace {

constexpr int kTileKeys = 32, kUnitTiles = 4;  // a unit of division: one 32-key tile per wave
constexpr float kWeightShift = 7.f;

// A request as one row tile sees it.
struct Rows {
    int start, count;  // packed rows
    int length;        // keys
    int n;             // rows of the tile (0: none)
    int first, last;   // positions of its first and last query
    int kend;          // keys [kstart, kend) can be seen by some row
    int kstart;
};

__device__ __forceinline__ Rows rows_of(const Block8AttendArgs &a, int i, int tile, bool &bad) {
    Rows r;
    const int cap = a.width << a.p.shift;
    const int len = a.lengths[i], s0 = a.starts[i];
    const int64_t m = a.granted ? (int64_t)a.granted[i] : (int64_t)a.starts[i + 1] - s0;
    r.length = min(max(len, 0), cap);
    r.start = (int)min((int64_t)max(s0, 0), a.rows);
    r.count = (int)min(min(max(m, (int64_t)0), (int64_t)a.max_q), a.rows - r.start);
    bad |= r.length != len || r.start != s0 || r.count != m;
    const int all = r.count * a.group;
    r.n = min(max(all - 16 * tile, 0), 16);
    const int base = r.length - r.count;  // below 0: rows before the first key see nothing
    r.first = base + 16 * tile / a.group;
    r.last = base + (16 * tile + max(r.n, 1) - 1) / a.group;
    r.kend = r.n > 0 ? min(max(r.last + 1, 0), r.length) : 0;
    r.kstart = a.window > 0 ? min(max(r.first - a.window + 1, 0), r.kend) : 0;
    return r;
}
__device__ __forceinline__ int tiles_of(const Rows &r) {
    return (r.kend + kTileKeys - 1) / kTileKeys - r.kstart / kTileKeys;
}
// Rows without keys are one unit too: their zeros have to be written.
__device__ __forceinline__ int units_of(const Rows &r) {
    return r.n == 0 ? 0 : max(1, (tiles_of(r) + kUnitTiles - 1) / kUnitTiles);
}

// Running sum over the workgroup's 256 threads (exclusive) and the total.
__device__ __forceinline__ int64_t scan256(int64_t x, int64_t *lds, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(inc, d);
        if (lane >= d) inc += y;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = inc;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += lds[w];
        total += lds[w];
    }
    return before + inc - x;
}

// The units of all requests' heads for one row tile, in request, head, unit order.
__device__ __forceinline__ int64_t units_total(const Block8AttendArgs &a, int tile, int64_t *lds, bool &bad) {
    int64_t all = 0;
    for (int base = 0; base < a.n; base += 256) {
        const int i = base + threadIdx.x;
        int64_t sum;
        scan256(i < a.n ? units_of(rows_of(a, i, tile, bad)) : 0, lds, sum);
        all += sum;
    }
    return all * a.p.kv_heads;
}
// The request of unit u and the units before it. Every thread of the workgroup calls.
__device__ __forceinline__ void request_at(const Block8AttendArgs &a, int tile, int64_t u, int64_t *lds, int &req,
                                           int64_t &before) {
    bool bad = false;
    int64_t all = 0;
    __shared__ int64_t found[2];
    for (int base = 0; base < a.n; base += 256) {
        const int i = base + threadIdx.x;
        const int64_t mine = i < a.n ? (int64_t)units_of(rows_of(a, i, tile, bad)) * a.p.kv_heads : 0;
        int64_t sum;
        const int64_t at = all + scan256(mine, lds, sum);
        all += sum;
        if (at <= u && u < at + mine) {
            found[0] = i;
            found[1] = at;
        }
    }
    __syncthreads();
    req = __builtin_amdgcn_readfirstlane((int)found[0]);
    before = found[1];
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

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
}

// Q^T of a row tile as fp16 operands: lane (row l%16, group l/16) holds for step c
// the dims 64(c/2) + 16(l/16) + 8(c%2) + 0..7 of its row, scaled by 2^shift so that
// the row's largest element lies in [2^14, 2^15). back: 2^-shift.
template <int D>
__device__ __forceinline__ void load_query(const uint16_t *row, bool valid, uint32_t flip, uint32_t (&op)[D / 32][4],
                                           float &back) {
    const int grp = (threadIdx.x & 63) >> 4;
    uint4 raw[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        raw[c] = valid ? *reinterpret_cast<const uint4 *>(row + 64 * (c / 2) + 16 * grp + 8 * (c % 2))
                       : make_uint4(0, 0, 0, 0);
    }
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
    constexpr int NB = D / 16;   // 16-dim blocks of the output
    constexpr int KC = D / 64;   // 16-byte chunks of a key row per lane
    constexpr int VW = D / 64;   // dwords of a V row per lane
    __shared__ float4 so[4 * NB * 64];
    __shared__ float2 sml[4 * 16];
    __shared__ int64_t scan_lds[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int tile = blockIdx.y, wg = blockIdx.x;
    bool bad = false;
    const int64_t total = units_total(a, tile, scan_lds, bad);
    if (bad) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
    const int64_t per = (total + a.wgs - 1) / a.wgs;
    int64_t u = wg * per;
    const int64_t uend = min(total, u + per);
    if (u >= uend) return;
    int req;
    int64_t before;
    request_at(a, tile, u, scan_lds, req, before);
    const float scale = fabsf(a.scale_log2);
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    bool unmapped = false;

    while (u < uend) {
        bool ignore = false;
        const Rows r = rows_of(a, req, tile, ignore);
        const int units = units_of(r);
        if (u >= before + (int64_t)units * a.p.kv_heads) {
            before += (int64_t)units * a.p.kv_heads;
            ++req;
            continue;
        }
        const int head = (int)((u - before) / units);
        const int64_t seg = before + (int64_t)head * units;  // the head's first unit
        const int ua = (int)(u - seg), ub = (int)min((int64_t)units, uend - seg);
        const int first_tile = r.kstart / kTileKeys;
        const int t_end = min(first_tile + ub * kUnitTiles, (r.kend + kTileKeys - 1) / kTileKeys);
        const int t_begin = first_tile + ua * kUnitTiles + wave;

        // this lane's row (a column of S^T and O^T)
        const bool valid = col < r.n;
        const int row = 16 * tile + (valid ? col : 0);
        const int qr = row / a.group, hr = row - qr * a.group;
        const int pos = r.length - r.count + qr;
        uint32_t qop[D / 32][4];
        float back;
        load_query<D>(a.q + (int64_t)(r.start + qr) * a.q_row + (int64_t)(head * a.group + hr) * a.q_head, valid, flip, qop,
                      back);
        const float qscale = scale * back;

        float m = kNegBig, l = 0.f;
        f32x4_t o[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

        if (t_begin < t_end) {
            // keys every row of the tile sees
            const int all_lo = a.window > 0 ? r.last - a.window + 1 : 0, all_hi = min(r.first + 1, r.kend);
            const int32_t *entries = a.table + (int64_t)req * a.table_stride;
            const int64_t head_bytes = (int64_t)a.p.block * D;
            // the pages of a tile's two 16-key halves; past the range the last key's
            auto page_of = [&](int t, int h) __attribute__((always_inline)) {
                const int key = min(t * kTileKeys + 16 * h, r.kend - 1);
                return entries[key >> a.p.shift];
            };
            // byte offset of a half's 16 rows of this head
            auto half_at = [&](int page, int t, int h) __attribute__((always_inline)) {
                return ((int64_t)page * a.p.kv_heads + head) * head_bytes +
                       (int64_t)((t * kTileKeys + 16 * h) & (a.p.block - 1)) * D;
            };
            uint32_t kc[2][KC][4], vc[2][4][VW];
            float ks[2], vs[2];
            bool ok[2];
            int page[2];
            auto take_pages = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int p = page_of(t, h);
                    ok[h] = (unsigned)p < (unsigned)a.p.pages;
                    page[h] = ok[h] ? p : 0;
                }
            };
            auto load_k = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t *p = a.p.k + half_at(page[h], t, h) + col * D + 16 * grp;
#pragma unroll
                    for (int c = 0; c < KC; ++c) load_dwords<4>(p + 64 * c, kc[h][c]);
                    ks[h] = a.p.k_scale[(int64_t)page[h] * a.p.kv_heads + head];
                }
            };
            auto load_v = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t *p = a.p.v + half_at(page[h], t, h) + 4 * grp * D + col * (D / 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) load_dwords<VW>(p + j * D, vc[h][j]);
                    vs[h] = a.p.v_scale[(int64_t)page[h] * a.p.kv_heads + head];
                }
            };
            take_pages(t_begin);
            load_k(t_begin);
            load_v(t_begin);
            for (int t = t_begin; t < t_end; t += kUnitTiles) {
                const int next = min(t + kUnitTiles, t_end - 1);  // past the last: read again, not used
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
                    inv_vs[h] = 1.0f / v;
                    cf[h] = qscale * scale_in_range(ks[h]);
                    good[h] = ok[h];
                }
                take_pages(next);
                load_k(next);
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
                    for (int h = 0; h < 2; ++h)
                        unmapped |= !good[h] && key0 + 16 * h < r.kend && key0 + 16 * h + 16 > r.kstart;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
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
        }

        // combine the four waves: each scales its part to the rows' common max, and
        // sums and stores a quarter of the dims
        __syncthreads();  // the last segment's sums are read
        if (grp == 0) sml[wave * 16 + col] = make_float2(m, l);
        __syncthreads();
        float M = kNegBig, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w * 16 + col].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 x = sml[w * 16 + col];
            sum = fmaf(x.y, __builtin_amdgcn_exp2f(x.x - M), sum);
        }
        const float f = __builtin_amdgcn_exp2f(m - M);
#pragma unroll
        for (int b = 0; b < NB; ++b)
            so[(wave * NB + b) * 64 + lane] = make_float4(o[b][0] * f, o[b][1] * f, o[b][2] * f, o[b][3] * f);
        __syncthreads();
        constexpr int MB = NB / 4;  // blocks of this wave: MB wave .. MB wave + MB - 1
        float4 x[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            x[b] = so[(MB * wave + b) * 64 + lane];
#pragma unroll
            for (int w = 1; w < 4; ++w) {
                const float4 y = so[(w * NB + MB * wave + b) * 64 + lane];
                x[b] = make_float4(x[b].x + y.x, x[b].y + y.y, x[b].z + y.z, x[b].w + y.w);
            }
        }
        const bool begins = ua == 0, ends = ub == units;
        if (begins && ends) {
            if (valid) {
                const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
                uint16_t *out = a.out + (int64_t)(r.start + qr) * a.o_row + (int64_t)(head * a.group + hr) * a.o_head +
                                4 * grp * NB + MB * wave;
#pragma unroll
                for (int b = 0; b < MB; ++b) {
                    out[b] = f32_to_bf16(x[b].x * inv);
                    out[NB + b] = f32_to_bf16(x[b].y * inv);
                    out[2 * NB + b] = f32_to_bf16(x[b].z * inv);
                    out[3 * NB + b] = f32_to_bf16(x[b].w * inv);
                }
            }
        } else {
            // slot 0: the rows' keys began in an earlier workgroup, 1: they begin here
            const int64_t slot = ((int64_t)tile * a.wgs + wg) * 2 + (begins ? 1 : 0);
            float4 *po = reinterpret_cast<float4 *>(a.part_o) + (slot * NB + MB * wave) * 64 + lane;
#pragma unroll
            for (int b = 0; b < MB; ++b) po[b * 64] = x[b];
            if (wave == 0 && grp == 0) a.part_ml[slot * 16 + col] = make_float2(M, sum);
        }
        u = seg + ub;
    }
    if (unmapped) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
}

// Joins the partials of the rows whose keys several workgroups had: one workgroup
// per (request, KV head, row tile), in workgroup order.
template <int D>
__global__ __launch_bounds__(256) void block8_join_kernel(Block8AttendArgs a) {
    constexpr int NB = D / 16, MB = NB / 4;
    __shared__ int64_t scan_lds[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int tile = blockIdx.y, head = blockIdx.x % a.p.kv_heads, req = blockIdx.x / a.p.kv_heads;
    bool bad = false;
    const Rows r = rows_of(a, req, tile, bad);
    if (r.n == 0) return;
    // units before the request, and all
    int64_t all = 0, before = 0;
    for (int base = 0; base < a.n; base += 256) {
        const int i = base + threadIdx.x;
        const int64_t mine = i < a.n ? units_of(rows_of(a, i, tile, bad)) : 0;
        int64_t sum, less;
        scan256(mine, scan_lds, sum);
        scan256(i < req ? mine : 0, scan_lds, less);
        all += sum;
        before += less;
    }
    const int64_t per = (all * a.p.kv_heads + a.wgs - 1) / a.wgs;
    const int units = units_of(r);
    const int64_t seg = before * a.p.kv_heads + (int64_t)head * units;
    const int w0 = (int)(seg / per), w1 = (int)((seg + units - 1) / per);
    if (w0 == w1) return;
    auto slot_at = [&](int w) { return ((int64_t)tile * a.wgs + w) * 2 + (w == w0 ? 1 : 0); };
    float M = kNegBig;
    for (int w = w0; w <= w1; ++w) M = fmaxf(M, a.part_ml[slot_at(w) * 16 + col].x);
    float sum = 0.f;
    float4 x[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) x[b] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = w0; w <= w1; ++w) {
        const int64_t slot = slot_at(w);
        const float2 ml = a.part_ml[slot * 16 + col];
        const float f = __builtin_amdgcn_exp2f(ml.x - M);
        sum = fmaf(ml.y, f, sum);
        const float4 *po = reinterpret_cast<const float4 *>(a.part_o) + (slot * NB + MB * wave) * 64 + lane;
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const float4 y = po[b * 64];
            x[b] = make_float4(fmaf(y.x, f, x[b].x), fmaf(y.y, f, x[b].y), fmaf(y.z, f, x[b].z), fmaf(y.w, f, x[b].w));
        }
    }
    if (col >= r.n) return;
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    const int row = 16 * tile + col, qr = row / a.group, hr = row - qr * a.group;
    uint16_t *out = a.out + (int64_t)(r.start + qr) * a.o_row + (int64_t)(head * a.group + hr) * a.o_head + 4 * grp * NB +
                    MB * wave;
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        out[b] = f32_to_bf16(x[b].x * inv);
        out[NB + b] = f32_to_bf16(x[b].y * inv);
        out[2 * NB + b] = f32_to_bf16(x[b].z * inv);
        out[3 * NB + b] = f32_to_bf16(x[b].w * inv);
    }
}

template <int CODE, int D>
static hipError_t launch_attend(const Block8AttendArgs &a, int tiles, hipStream_t s) {
    hipLaunchKernelGGL((block8_attend_kernel<CODE, D>), dim3(a.wgs, tiles), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.wgs == 1) return e;
    hipLaunchKernelGGL((block8_join_kernel<D>), dim3(a.n * a.p.kv_heads, tiles), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int CODE>
static hipError_t launch_attend_code(const Block8AttendArgs &a, int head_dim, int tiles, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_attend<CODE, 64>(a, tiles, s);
        case 128: return launch_attend<CODE, 128>(a, tiles, s);
        case 256: return launch_attend<CODE, 256>(a, tiles, s);
        case 512: return launch_attend<CODE, 512>(a, tiles, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_block8_attend(const Block8AttendArgs &a, int dtype, int head_dim, int tiles, hipStream_t s) {
    return dtype == KVRT_INT8 ? launch_attend_code<KVRT_INT8>(a, head_dim, tiles, s)
                              : launch_attend_code<KVRT_E4M3>(a, head_dim, tiles, s);
}

}  // namespace kvrt
