// kvrt_block8.hip — 8-bit pages with one scale per (page, KV head): page tables and
// slot maps from request lengths, rows coded into pages, the padded batch read
// back, and the C entry points.
#include <algorithm>
#include <cmath>

#include "kvrt_block8.h"

namespace kvrt {

// ---- page tables and slot maps --------------------------------------------------
//
// With m_i mapped pages and c_i = ceil((len_i + new_i) / block) needed ones,
// request i releases max(0, m_i - c_i) pages and wants max(0, c_i - m_i). The free
// pages are a stack: the k-th released page (in request order, a request's
// pages in order) lands on free[top - 1 - k], top = count + all released, and
// the k-th wanted one is taken from there, so nothing but two running sums
// orders the requests and every request works on its own: no atomics, one
// result. A request is granted while the running sum of wanted pages is within
// top.
//
// Latency bounds it: few bytes, but sums over all requests before any page has its
// place. One workgroup keeps those on one CU without a second launch; the slot map,
// which any thread finds by itself, takes a launch of its own from 4096 rows on.
// Measured: 4 requests of two rows 4.7 us, 256 requests with 16608 rows 7.7 + 5.3 us.

// Sum of x over the workgroup's threads before this one, and the sum over all.
__device__ __forceinline__ int64_t scan_add(int64_t x, int64_t *lds, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
    int64_t inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(inc, d);
        if (lane >= d) inc += y;
    }
    __syncthreads();  // lds is free again
    if (lane == 63) lds[wave] = inc;
    __syncthreads();
    int64_t before = 0, sum = 0;
    for (int w = 0; w < waves; ++w) {
        if (w < wave) before += lds[w];
        sum += lds[w];
    }
    total = sum;
    return before + inc - x;
}

// What a request asks for. `start` and the sums that follow are its running sums.
struct PageAsk {
    int len, add, mapped, need;
    bool fits;
};
__device__ __forceinline__ PageAsk page_ask(const Block8TablesArgs &a, int i, int mapped) {
    PageAsk r;
    r.len = a.lengths[i];
    r.add = a.new_rows[i];
    r.mapped = min(max(mapped, 0), a.max_pages);
    const int64_t total = (int64_t)r.len + r.add;
    r.fits = r.len >= 0 && r.add >= 0 && r.mapped == mapped && r.len <= (int64_t)r.mapped << a.shift &&
             total <= (int64_t)a.max_pages << a.shift;
    r.need = r.fits ? (int)((total + a.block - 1) >> a.shift) : r.mapped;
    return r;
}

// work: [0, n) wanted pages before the request (-1: refused), [n, 2n) its mapped
// pages before the call, [2n, 3n) its kept rows, 3n: top of the stack
// before anything is taken.
__device__ __forceinline__ int slot_of(const Block8TablesArgs &a, int i, int64_t t, int start, bool &bad) {
    const int before = a.work[i];
    if (before < 0) return -1;
    const int was = a.work[a.n + i];
    const int64_t pos = a.work[2 * a.n + i] + (t - start);
    const int j = (int)(pos >> a.shift);
    const int top = a.work[3 * a.n];
    const int page = j < was ? a.table[(int64_t)i * a.max_pages + j] : a.free_pages[top - 1 - (before + j - was)];
    if ((unsigned)page >= (unsigned)a.pool_pages) {
        bad = true;
        return -1;
    }
    return (page << a.shift) + (int)(pos & (a.block - 1));
}

// The request of packed row t: the last one that starts at or before t.
__device__ __forceinline__ int request_of(const int32_t *starts, int n, int64_t t) {
    int lo = 0, hi = n;  // starts[lo] <= t < starts[hi] or hi == n
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// New entries of the tables and the slot map, one thread each.
__device__ void fill_tables(const Block8TablesArgs &a, int64_t first, int64_t step) {
    bool bad = false;
    const int last = a.starts[a.n];
    for (int64_t t = first; t < a.rows; t += step) {
        int slot = -1;
        if (t < last) {
            const int i = request_of(a.starts, a.n, t);
            slot = slot_of(a, i, t, a.starts[i], bad);
            // the first row of a page that was not mapped, or the request's first row
            // past its mapped pages, brings the page into the table
            const int was = a.work[a.n + i];
            const int64_t pos = a.work[2 * a.n + i] + (t - a.starts[i]);
            if (a.work[i] >= 0 && (pos & (a.block - 1)) == 0 && (pos >> a.shift) >= was)
                a.table[(int64_t)i * a.max_pages + (pos >> a.shift)] =
                    a.free_pages[a.work[3 * a.n] - 1 - (a.work[i] + (int)(pos >> a.shift) - was)];
        }
        a.slot_map[t] = slot;
    }
    if (bad) raise(a.status, KVRT_BLOCK_BAD_INDEX);
}

// Page j of a request that keeps `need` pages goes back to the stack; its released
// pages begin with number k0.
__device__ __forceinline__ void give_back(const Block8TablesArgs &a, int32_t *row, int j, int page, int need, int64_t k0,
                                          int64_t top) {
    const int64_t at = top - 1 - (k0 + j - need);
    if (at >= 0) a.free_pages[at] = page;
    row[j] = -1;
}

// The pages of requests that release many: a wave to a request, eight pages a lane
// at a time. Up to kFewPages a thread does by itself, eight at a time: 32 of 256 requests
// that release 32 pages each take 11.3 us so, 20.6 a wave to a request.
constexpr int kFewPages = 64;
__device__ void give_back_many(const Block8TablesArgs &a, int64_t top) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    for (int base = wave; base < a.n; base += 64 * waves) {
        const int i = base + waves * lane;
        int need = 0, was = 0, k0 = 0;
        if (i < a.n && a.work[i] >= 0) {
            need = a.mapped[i];
            was = a.work[a.n + i];
            k0 = a.work[3 * a.n + 1 + i];
        }
        for (uint64_t many = __ballot(was - need > kFewPages); many; many &= many - 1) {
            const int l = __builtin_ctzll(many);
            const int end = __builtin_amdgcn_readlane(was, l), first = __builtin_amdgcn_readlane(need, l),
                      k = __builtin_amdgcn_readlane(k0, l);
            int32_t *row = a.table + (int64_t)(base + waves * l) * a.max_pages;
            for (int j0 = first; j0 < end; j0 += 512) {
                int page[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int j = j0 + 64 * u + lane;
                    page[u] = j < end ? row[j] : 0;
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int j = j0 + 64 * u + lane;
                    if (j < end) give_back(a, row, j, page[u], first, k, top);
                }
            }
        }
    }
}

// One workgroup: the running sums over all requests, the released pages, and,
// where the call is small (FILL), the new entries too.
template <bool FILL>
__global__ __launch_bounds__(1024) void block8_tables_kernel(Block8TablesArgs a) {
    __shared__ int64_t lds[16];
    const int tid = threadIdx.x, threads = blockDim.x;
    int raised = 0;
    int64_t start0 = 0, gone0 = 0;
    const int count = min(max(a.free_count[0], 0), a.pool_pages);
    if (count != a.free_count[0]) raised |= KVRT_BLOCK_BAD_INDEX;
    // released pages first: they count for this call's requests
    for (int base = 0; base < a.n; base += threads) {
        const int i = base + tid;
        PageAsk r{0, 0, 0, 0, false};
        if (i < a.n) r = page_ask(a, i, a.mapped[i]);
        int64_t sum;
        const int64_t start = start0 + scan_add(i < a.n ? max(r.add, 0) : 0, lds, sum);
        start0 += sum;
        const bool fits = r.fits && start + r.add <= a.rows;
        const int gone = fits ? max(r.mapped - r.need, 0) : 0;
        const int64_t k0 = gone0 + scan_add(gone, lds, sum);
        gone0 += sum;
        if (i >= a.n) continue;
        a.starts[i] = (int)min(start, a.rows);
        a.work[i] = fits ? 0 : -1;
        a.work[a.n + i] = r.mapped;
        a.work[2 * a.n + i] = (int)min((int64_t)max(r.len, 0), (int64_t)r.mapped << a.shift);
        if (!fits) raised |= KVRT_BLOCK_BAD_INDEX;
        a.work[3 * a.n + 1 + i] = (int)k0;
    }
    const int64_t top = min(count + gone0, (int64_t)a.pool_pages);
    if (top != count + gone0) raised |= KVRT_BLOCK_BAD_INDEX;
    int64_t want0 = 0, taken0 = 0;
    bool many = false;
    for (int base = 0; base < a.n; base += threads) {
        const int i = base + tid;
        bool fits = false;
        PageAsk r{0, 0, 0, 0, false};
        if (i < a.n) {
            r = page_ask(a, i, a.mapped[i]);
            fits = a.work[i] == 0;
        }
        const int want = fits ? max(r.need - r.mapped, 0) : 0;
        int64_t sum;
        const int64_t before = want0 + scan_add(want, lds, sum);
        want0 += sum;
        const bool ok = fits && (want == 0 || before + want <= top);
        scan_add(ok ? want : 0, lds, sum);
        taken0 += sum;
        if (i >= a.n) continue;
        if (fits && !ok) raised |= KVRT_BLOCK_NO_PAGES;
        int32_t *row = a.table + (int64_t)i * a.max_pages;
        if (ok && r.need < r.mapped) {
            const int64_t k0 = a.work[3 * a.n + 1 + i];
            if (r.mapped - r.need > kFewPages) many = true;
            else
                for (int j0 = r.need; j0 < r.mapped; j0 += 8) {
                    int page[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) page[u] = j0 + u < r.mapped ? row[j0 + u] : 0;
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (j0 + u < r.mapped) give_back(a, row, j0 + u, page[u], r.need, k0, top);
                }
        }
        a.work[i] = ok ? (int)before : -1;
        a.mapped[i] = ok ? r.need : r.mapped;
        a.granted[i] = ok ? r.add : 0;
        a.out_lengths[i] = a.work[2 * a.n + i] + (ok ? r.add : 0);
    }
    if (tid == 0) {
        a.starts[a.n] = (int)min(start0, a.rows);
        a.work[3 * a.n] = (int)top;
        a.free_count[0] = (int)(top - taken0);
    }
    if (raised) raise(a.status, raised);
    if (__syncthreads_or(many)) {
        give_back_many(a, top);
        if constexpr (FILL) __syncthreads();
    }
    if constexpr (FILL) {
        fill_tables(a, tid, threads);
    }
}

__global__ __launch_bounds__(256) void block8_fill_kernel(Block8TablesArgs a) {
    fill_tables(a, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

hipError_t launch_block8_tables(const Block8TablesArgs &a, hipStream_t s) {
    const int threads = a.n <= 16 && a.rows <= 256 ? 64 : a.n <= 256 && a.rows <= 1024 ? 256 : 1024;
    if (a.rows <= 4096) {
        hipLaunchKernelGGL(block8_tables_kernel<true>, dim3(1), dim3(threads), 0, s, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(block8_tables_kernel<false>, dim3(1), dim3(threads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t wgs = (a.rows + 255) / 256;
    hipLaunchKernelGGL(block8_fill_kernel, dim3((unsigned)(wgs < 4096 ? wgs : 4096)), dim3(256), 0, s, a);
    return hipGetLastError();
}

// ---- append -----------------------------------------------------------------------
//
// One wave codes one run (rows of consecutive slots in one page) of one head of K
// or V: the largest magnitude over the run, the scale, the codes before the run
// anew where the scale grew, then the new codes. A run is found from the slot map
// alone: a slot that does not follow its predecessor, or is a page's first row,
// begins one. Latency is what it costs, so what a run needs is loaded at once: its
// rows (held in registers, up to kHeld of a lane), the scale, and the slots of 64 rows.
// Rows read twice, a slot at a time, took 15.6 us for 6872 rows of 16 requests, 8 heads of
// D 128; this takes 13.6 (3.1 TB/s), and 20 with 16 rows held (232 registers, 2 waves).
constexpr int kHeld = 4;
template <int CODE, int D>
__global__ __launch_bounds__(256) void block8_append_kernel(Block8AppendArgs a) {
    constexpr int LPR = D / 8, RPI = 64 / LPR;  // lanes per row (8 values each), rows per instruction
    const int lane = threadIdx.x & 63;
    const int64_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int kinds = 2 * a.p.kv_heads;
    const int kind = (int)(wave % kinds), kv = kind & 1, head = kind >> 1;
    const int64_t t0 = wave / kinds * a.chunk;
    if (t0 >= a.rows) return;
    const int64_t slots = (int64_t)a.p.pages << a.p.shift;
    int raised = 0;
    const int64_t t = t0 + lane;
    const int slot = t < a.rows ? a.slots[t] : -1;
    int prev = __shfl_up(slot, 1);
    if (lane == 0) prev = t0 > 0 ? a.slots[t0 - 1] : -2;
    const bool in = slot >= 0 && slot < slots;
    const bool follows = in && prev == slot - 1 && (slot & (a.p.block - 1)) != 0;
    if (lane < a.chunk && slot >= 0 && !in) raised |= KVRT_BLOCK_BAD_INDEX;
    uint64_t heads = __ballot(in && !follows && lane < a.chunk);  // rows that begin a run
    const uint64_t more = __ballot(follows);
    const int r0 = lane / LPR, d0 = 8 * (lane % LPR);
    while (heads) {
        const int b = __builtin_ctzll(heads);
        heads &= heads - 1;
        const int s0 = __builtin_amdgcn_readlane(slot, b);
        const int page = s0 >> a.p.shift, off = s0 & (a.p.block - 1);
        // the run's length: rows after b as long as their slots follow
        int run = 1 + __builtin_ctzll(~(more >> (b + 1)));  // (zeros are shifted in: b < chunk <= 16)
        if (b + run == 64)
            for (int base = run; base < a.p.block - off; base += 64) {
                const int j = base + lane;
                const bool on = j < a.p.block - off && t0 + b + j < a.rows && a.slots[t0 + b + j] == s0 + j;
                const uint64_t off_bits = ~__ballot(on);
                const int got = off_bits ? __builtin_ctzll(off_bits) : 64;
                run += got;
                if (got < 64) break;
            }
        const uint16_t *x = a.x[kv] + (t0 + b) * a.row[kv] + head * a.head[kv] + d0;
        float *sp = (kv ? a.p.v_scale : a.p.k_scale) + (int64_t)page * a.p.kv_heads + head;
        const float was = *sp;
        uint8_t *codes = (kv ? a.p.v : a.p.k) + ((((int64_t)page * a.p.kv_heads + head) << a.p.shift)) * D;
        uint4 held[kHeld];
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            held[u] = make_uint4(0, 0, 0, 0);
            if (u * RPI < run && r0 + u * RPI < run)
                held[u] = *reinterpret_cast<const uint4 *>(x + (int64_t)(r0 + u * RPI) * a.row[kv]);
        }
        // the largest finite magnitude
        float amax = 0.f;
        auto largest = [&](uint4 w) __attribute__((always_inline)) {
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float m = fabsf(h ? bf16_hi(ws[i]) : bf16_lo(ws[i]));
                    const bool fin = m < INFINITY;
                    if (!fin) raised |= KVRT_BLOCK_NOT_FINITE;
                    amax = fin ? fmaxf(amax, m) : amax;
                }
            }
        };
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (u * RPI < run) largest(held[u]);
        for (int r = r0 + kHeld * RPI; r < run; r += RPI)
            largest(*reinterpret_cast<const uint4 *>(x + (int64_t)r * a.row[kv]));
        amax = group_max<64>(amax);
        float scale = scale_in_range(amax / kCodeTop<CODE>);
        if (off > 0) {
            const float old = scale_in_range(was);
            scale = fmaxf(scale, old);
            if (scale > old) {
                const float r = old / scale;
                for (int e = lane * 16; e < off * D; e += 64 * 16) {
                    uint4 w = *reinterpret_cast<const uint4 *>(codes + e);
                    uint32_t *ws = &w.x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float c[4];
                        codes_to_f32<CODE>(ws[i], c);
#pragma unroll
                        for (int j = 0; j < 4; ++j) c[j] *= r;
                        ws[i] = f32_to_codes<CODE>(c);
                    }
                    *reinterpret_cast<uint4 *>(codes + e) = w;
                }
            }
        }
        if (lane == 0) *sp = scale;
        const float inv = 1.0f / scale;
        auto code = [&](int r, uint4 w) __attribute__((always_inline)) {
            const float lo[4] = {bf16_lo(w.x) * inv, bf16_hi(w.x) * inv, bf16_lo(w.y) * inv, bf16_hi(w.y) * inv};
            const float hi[4] = {bf16_lo(w.z) * inv, bf16_hi(w.z) * inv, bf16_lo(w.w) * inv, bf16_hi(w.w) * inv};
            *reinterpret_cast<uint2 *>(codes + (off + r) * D + d0) =
                make_uint2(f32_to_codes<CODE>(lo), f32_to_codes<CODE>(hi));
        };
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (u * RPI < run && r0 + u * RPI < run) code(r0 + u * RPI, held[u]);
        for (int r = r0 + kHeld * RPI; r < run; r += RPI)
            code(r, *reinterpret_cast<const uint4 *>(x + (int64_t)r * a.row[kv]));
    }
    if (raised) raise(a.p.status, raised);
}

template <int CODE>
static hipError_t launch_append(const Block8AppendArgs &a, int head_dim, hipStream_t s) {
    const int64_t waves = (a.rows + a.chunk - 1) / a.chunk * 2 * a.p.kv_heads;
    const dim3 grid((unsigned)((waves + 3) / 4)), wg(256);
    switch (head_dim) {
        case 64: hipLaunchKernelGGL((block8_append_kernel<CODE, 64>), grid, wg, 0, s, a); break;
        case 128: hipLaunchKernelGGL((block8_append_kernel<CODE, 128>), grid, wg, 0, s, a); break;
        case 256: hipLaunchKernelGGL((block8_append_kernel<CODE, 256>), grid, wg, 0, s, a); break;
        case 512: hipLaunchKernelGGL((block8_append_kernel<CODE, 512>), grid, wg, 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_block8_append(const Block8AppendArgs &a, int dtype, int head_dim, hipStream_t s) {
    return dtype == KVRT_INT8 ? launch_append<KVRT_INT8>(a, head_dim, s) : launch_append<KVRT_E4M3>(a, head_dim, s);
}

// ---- gather -----------------------------------------------------------------------
//
// x = code * scale, rounded once. 16 codes per lane: a lane reads 16 bytes and writes 32
// (bf16) or 64 (fp32), and HBM bounds it: 16 requests of 430 rows padded to 512, 8 heads
// of D 128 take 11.5 us (4.1 TB/s); two rows of four requests, 3.4 us, are latency.
template <int CODE, int D, bool FP32>
__global__ __launch_bounds__(256) void block8_gather_kernel(Block8GatherArgs a) {
    constexpr int LPR = D / 16, RPW = 256 / LPR;  // lanes per row, rows per workgroup
    const int item = blockIdx.z, head = blockIdx.y >> 1, kv = blockIdx.y & 1;
    const int row = blockIdx.x * RPW + threadIdx.x / LPR, d0 = 16 * (threadIdx.x % LPR);
    const int cap = a.width << a.p.shift;
    const int length = a.lengths[item], start = a.start_pos ? a.start_pos[item] : 0;
    bool bad = length < 0 || length > cap || start < 0;
    const int L = min(max(length, 0), cap);
    const int64_t pos = (int64_t)max(start, 0) + row;
    if (row >= a.lmax) return;
    const bool valid = start >= 0 && pos < L;
    uint4 w = make_uint4(0, 0, 0, 0);
    float scale = 0.f;
    bool zero = true;
    if (valid) {
        const int page = a.table[item * a.table_stride + (pos >> a.p.shift)];
        if ((unsigned)page < (unsigned)a.p.pages) {
            const int64_t ph = (int64_t)page * a.p.kv_heads + head;
            const uint8_t *codes = (kv ? a.p.v : a.p.k) + ((ph << a.p.shift) + (pos & (a.p.block - 1))) * D;
            w = load_stream16(codes + d0);
            scale = scale_in_range((kv ? a.p.v_scale : a.p.k_scale)[ph]);
            zero = false;
        } else {
            bad = true;
        }
    }
    float x[16];
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float c[4];
        codes_to_f32<CODE>(ws[i], c);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = zero ? 0.f : c[j] * scale;
    }
    const int64_t at = item * a.item[kv] + head * a.head[kv] + row * a.row[kv] + d0;
    if constexpr (FP32) {
        float *o = static_cast<float *>(a.out[kv]) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4 *>(o + 4 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
        uint16_t *o = static_cast<uint16_t *>(a.out[kv]) + at;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4 *>(o + 8 * i) =
                make_uint4(pack_bf16x2(x[8 * i], x[8 * i + 1]), pack_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                           pack_bf16x2(x[8 * i + 4], x[8 * i + 5]), pack_bf16x2(x[8 * i + 6], x[8 * i + 7]));
    }
    if (a.mask && blockIdx.y == 0 && d0 == 0) {
        const int64_t m = item * a.mask_stride + row;
        if (a.mask_dtype == KVRT_BOOL) static_cast<uint8_t *>(a.mask)[m] = valid ? 1 : 0;
        else if (a.mask_dtype == KVRT_FP32) static_cast<float *>(a.mask)[m] = valid ? 0.f : -3.4028234663852886e38f;
        else static_cast<uint16_t *>(a.mask)[m] = valid ? (uint16_t)0 : (uint16_t)0xff7f;  // bf16 finfo.min
    }
    if (bad) raise(a.p.status, KVRT_BLOCK_BAD_INDEX);
}

template <int CODE, int D>
static hipError_t launch_gather_dim(const Block8GatherArgs &a, hipStream_t s) {
    constexpr int RPW = 256 / (D / 16);
    const dim3 grid((a.lmax + RPW - 1) / RPW, 2 * a.p.kv_heads, a.n), wg(256);
    if (a.fp32) hipLaunchKernelGGL((block8_gather_kernel<CODE, D, true>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((block8_gather_kernel<CODE, D, false>), grid, wg, 0, s, a);
    return hipGetLastError();
}

template <int CODE>
static hipError_t launch_gather(const Block8GatherArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_gather_dim<CODE, 64>(a, s);
        case 128: return launch_gather_dim<CODE, 128>(a, s);
        case 256: return launch_gather_dim<CODE, 256>(a, s);
        case 512: return launch_gather_dim<CODE, 512>(a, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_block8_gather(const Block8GatherArgs &a, int dtype, int head_dim, hipStream_t s) {
    return dtype == KVRT_INT8 ? launch_gather<KVRT_INT8>(a, head_dim, s) : launch_gather<KVRT_E4M3>(a, head_dim, s);
}

// ---- checks of the C entry points ---------------------------------------------------

static bool aligned(const void *p, uintptr_t to) { return p && (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

static int block_shift(int block) {
    for (int s = 4; s <= 7; ++s)
        if (block == 1 << s) return s;
    return -1;
}

static bool view_of(const kvrt_block8 *p, Block8View &v) {
    if (!p || (p->dtype != KVRT_INT8 && p->dtype != KVRT_E4M3) || p->pages <= 0 || p->kv_heads < 1 || p->kv_heads > 64)
        return false;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256 && p->head_dim != 512) return false;
    const int shift = block_shift(p->block);
    if (shift < 0 || (int64_t)p->pages * p->kv_heads * p->block >= (int64_t)1 << 31) return false;
    if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->k_scale, 4) || !aligned(p->v_scale, 4) ||
        !aligned(p->status, 4))
        return false;
    v = Block8View{static_cast<uint8_t *>(p->k), static_cast<uint8_t *>(p->v), p->k_scale, p->v_scale, p->status,
                   p->pages, p->kv_heads, p->block, shift};
    return true;
}

// A tensor of that type and rank with a contiguous last dimension, rows aligned to
// `align` bytes and no negative size or stride. Empty ones need no data.
static bool strided(const kvrt_tensor *t, int dtype, int elem, int ndim, int align) {
    if (!t || t->dtype != dtype || t->ndim != ndim) return false;
    bool empty = false;
    for (int i = 0; i < ndim; ++i) {
        if (t->dims[i] < 0) return false;
        empty |= t->dims[i] == 0;
    }
    if (empty) return true;
    if (!aligned(t->data, align) || (t->dims[ndim - 1] > 1 && t->strides[ndim - 1] != 1)) return false;
    for (int i = 0; i < ndim - 1; ++i)
        if (t->strides[i] < 0 || (t->dims[i] > 1 && (t->strides[i] * elem) % align != 0)) return false;
    return true;
}

// Strides that put no element at two places of the shape (outputs).
static bool disjoint(const kvrt_tensor *t) {
    int64_t reach = 1;  // elements below the dimensions seen so far, by rising stride
    bool used[KVRT_MAX_RANK] = {};
    for (int k = 0; k < t->ndim; ++k) {
        int best = -1;
        for (int i = 0; i < t->ndim; ++i)
            if (!used[i] && (best < 0 || t->strides[i] < t->strides[best])) best = i;
        used[best] = true;
        if (t->dims[best] <= 1) continue;
        if (t->strides[best] < reach) return false;
        reach = t->strides[best] * (t->dims[best] - 1) + reach;
    }
    return true;
}

// Limits of a table, for the calls that build it and those that read it: requests are a
// grid dimension; kernels add a step of keys, and subtract windows and row counts, in 32
// bits.
constexpr int64_t kTableRequests = 65535, kTablePositions = (int64_t)1 << 30;

static bool table_ok(const kvrt_tensor *t, int shift, int64_t &n, int64_t &width) {
    if (!strided(t, KVRT_INT32, 4, 2, 4)) return false;
    n = t->dims[0];
    width = t->dims[1];
    return n <= kTableRequests && width <= kTablePositions >> shift;
}

constexpr int64_t kMaxRows = (int64_t)1 << 30, kJoinBytes = 48 << 10;
constexpr int64_t kGridWgs = (1 << 24) - 1;  // workgroups of 256 threads whose threads 32 bits count

// How a call's rows and keys are divided.
struct AttendPlan {
    bool chunk;           // more than 16 query rows per KV head
    int wgs;              // decode: workgroups the keys are divided over
    int64_t most;         // decode: units of 128 keys that a head of one request has at most
    int row_waves, splits;
    int64_t tiles;        // chunk: row tiles at most
    uint64_t part_rows;   // rows of partials in the workspace
};
static AttendPlan attend_plan(int kv_heads, int shift, int head_dim, int64_t n, int64_t width, int64_t rows, int64_t group,
                              int64_t max_q) {
    AttendPlan p{};
    width = std::max<int64_t>(width, 1);  // a table without columns has rows to be zeroed
    p.chunk = group * max_q > 16;
    if (!p.chunk) {
        // as many workgroups as run at a time: their registers (135, 140, 223 and 400) allow
        // 3, 3, 2 and 1 per CU. A fourth at D 64 waits for a place: 64 requests to 4000 keys, 16
        // heads over 8, took 45.6 us with it and take 38.2.
        const int64_t round = 256 * (head_dim <= 128 ? 3 : head_dim == 256 ? 2 : 1);
        p.most = ((width << shift) + 127) / 128 + 1;
        p.wgs = (int)std::max<int64_t>(1, std::min(n * kv_heads * p.most, round));
        p.part_rows = p.wgs == 1 ? 0 : (uint64_t)p.wgs * 2 * 16;
        return p;
    }
    // The most rows per tile (each shares the keys' conversion) that still leave a
    // workgroup per CU, then the keys divided as far as that takes. Every request's last
    // tile may be a partial one.
    const int least = head_dim <= 128 ? 2 : 4;  // row blocks that keep every wave busy
    for (p.row_waves = head_dim <= 128 ? 8 : 4;; p.row_waves /= 2) {
        const int64_t size = 32 * p.row_waves;
        p.tiles = std::min((rows * group + size - 1) / size + n - 1, n * ((group * max_q + size - 1) / size));
        if (p.row_waves == least || p.tiles * kv_heads >= 256) break;
    }
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(16, 256 / (p.tiles * kv_heads)));
    p.part_rows = p.splits == 1 ? 0 : (uint64_t)p.tiles * kv_heads * p.splits * 32 * p.row_waves;
    return p;
}
static uint64_t part_bytes(uint64_t rows, int head_dim) { return rows * (4 * head_dim + 8); }

}  // namespace kvrt

using namespace kvrt;

extern "C" {

int kvrt_block_tables_update_async(const kvrt_block_tables *t, const int32_t *lengths, const int32_t *new_rows,
                                   int64_t rows, int32_t *starts, int32_t *slot_map, int32_t *out_lengths,
                                   int32_t *granted, void *stream) {
    if (!t || t->n < 1 || t->n > kTableRequests || t->max_pages < 1 || t->pool_pages < 1) return KVRT_EINVAL;
    const int shift = block_shift(t->block);
    const int64_t limit = (int64_t)1 << 31;
    if (shift < 0 || (int64_t)t->n * t->max_pages >= limit || t->max_pages > kTablePositions >> shift ||
        (int64_t)t->pool_pages * t->block >= limit || rows < 0 || rows > kMaxRows)
        return KVRT_EINVAL;
    for (const void *p : {(const void *)t->table, (const void *)t->mapped, (const void *)t->free_pages,
                          (const void *)t->free_count, (const void *)t->work, (const void *)t->status,
                          (const void *)lengths, (const void *)new_rows, (const void *)starts,
                          (const void *)out_lengths, (const void *)granted})
        if (!aligned(p, 4)) return KVRT_EINVAL;
    if (rows > 0 && !aligned(slot_map, 4)) return KVRT_EINVAL;
    const Block8TablesArgs a{t->table, t->mapped, t->free_pages, t->free_count, t->work, t->status,
                             t->n, t->max_pages, t->pool_pages, t->block, shift,
                             lengths, new_rows, rows, starts, slot_map, out_lengths, granted};
    return launch_block8_tables(a, static_cast<hipStream_t>(stream)) == hipSuccess ? KVRT_OK : KVRT_EDEVICE;
}

int kvrt_block8_append_async(const kvrt_block8 *pages, const kvrt_tensor *k, const kvrt_tensor *v,
                             const int32_t *slot_map, void *stream) {
    Block8AppendArgs a{};
    if (!view_of(pages, a.p) || !strided(k, KVRT_BF16, 2, 3, 16) || !strided(v, KVRT_BF16, 2, 3, 16))
        return KVRT_EINVAL;
    for (const kvrt_tensor *x : {k, v})
        if (x->dims[0] != k->dims[0] || x->dims[1] != pages->kv_heads || x->dims[2] != pages->head_dim)
            return KVRT_EINVAL;
    a.rows = k->dims[0];
    if (a.rows == 0) return KVRT_OK;
    if (a.rows > kMaxRows || !aligned(slot_map, 4)) return KVRT_EINVAL;
    a.slots = slot_map;
    const kvrt_tensor *x[2] = {k, v};
    for (int i = 0; i < 2; ++i) {
        a.x[i] = static_cast<const uint16_t *>(x[i]->data);
        a.row[i] = x[i]->strides[0];
        a.head[i] = x[i]->strides[1];
    }
    a.chunk = a.rows * 2 * pages->kv_heads <= 4096 ? 1 : 16;
    if ((a.rows + a.chunk - 1) / a.chunk * 2 * pages->kv_heads > 4 * kGridWgs) return KVRT_EINVAL;
    const hipError_t e = launch_block8_append(a, pages->dtype, pages->head_dim, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? KVRT_OK : KVRT_EDEVICE;
}

int kvrt_block8_gather_async(const kvrt_block8 *pages, const kvrt_tensor *table, const int32_t *lengths,
                             const int32_t *start_pos, const kvrt_tensor *out_k, const kvrt_tensor *out_v,
                             const kvrt_tensor *mask, void *stream) {
    Block8GatherArgs a{};
    int64_t n, width;
    if (!view_of(pages, a.p) || !table_ok(table, a.p.shift, n, width)) return KVRT_EINVAL;
    if (!out_k || (out_k->dtype != KVRT_BF16 && out_k->dtype != KVRT_FP32)) return KVRT_EINVAL;
    const int elem = out_k->dtype == KVRT_FP32 ? 4 : 2;
    if (!strided(out_k, out_k->dtype, elem, 4, 16) || !strided(out_v, out_k->dtype, elem, 4, 16)) return KVRT_EINVAL;
    const int64_t lmax = out_k->dims[2];
    for (const kvrt_tensor *o : {out_k, out_v})
        if (o->dims[0] != n || o->dims[1] != pages->kv_heads || o->dims[2] != lmax || o->dims[3] != pages->head_dim)
            return KVRT_EINVAL;
    if (mask) {
        const int bytes = mask->dtype == KVRT_BOOL ? 1 : mask->dtype == KVRT_FP32 ? 4 : mask->dtype == KVRT_BF16 ? 2 : 0;
        if (!bytes || !strided(mask, mask->dtype, bytes, 2, bytes) || mask->dims[0] != n || mask->dims[1] != lmax)
            return KVRT_EINVAL;
    }
    if (n == 0 || lmax == 0) return KVRT_OK;
    if (lmax > kGridWgs * (4096 / pages->head_dim) || !disjoint(out_k) || !disjoint(out_v) || (mask && !disjoint(mask))) return KVRT_EINVAL;
    if (!aligned(lengths, 4) || (start_pos && !aligned(start_pos, 4)) || (width > 0 && !table->data))
        return KVRT_EINVAL;
    a.table = static_cast<const int32_t *>(table->data);
    a.table_stride = table->strides[0];
    a.lengths = lengths;
    a.start_pos = start_pos;
    a.n = (int)n;
    a.width = (int)width;
    a.lmax = (int)lmax;
    const kvrt_tensor *o[2] = {out_k, out_v};
    for (int i = 0; i < 2; ++i) {
        a.out[i] = o[i]->data;
        a.item[i] = o[i]->strides[0];
        a.head[i] = o[i]->strides[1];
        a.row[i] = o[i]->strides[2];
    }
    a.fp32 = elem == 4;
    a.mask = mask ? mask->data : nullptr;
    a.mask_dtype = mask ? mask->dtype : 0;
    a.mask_stride = mask ? mask->strides[0] : 0;
    const hipError_t e = launch_block8_gather(a, pages->dtype, pages->head_dim, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? KVRT_OK : KVRT_EDEVICE;
}

uint64_t kvrt_block8_attend_work(const kvrt_block8 *pages, int64_t n, int64_t width, int64_t rows, int64_t hq,
                                 int32_t max_q) {
    Block8View v;
    if (!view_of(pages, v) || n <= 0 || width < 0 || rows <= 0 || hq <= 0 || hq % pages->kv_heads != 0 || max_q <= 0)
        return 0;
    const AttendPlan p = attend_plan(v.kv_heads, v.shift, pages->head_dim, n, width, rows, hq / v.kv_heads, max_q);
    return part_bytes(p.part_rows, pages->head_dim);
}

int kvrt_block8_attend_async(const kvrt_block8 *pages, const kvrt_tensor *q, const kvrt_tensor *table,
                             const int32_t *lengths, const int32_t *starts, const int32_t *granted,
                             const kvrt_tensor *out, float scale, int32_t window, int32_t max_q, void *work,
                             uint64_t work_bytes, void *stream) {
    Block8AttendArgs a{};
    int64_t n, width;
    if (!view_of(pages, a.p) || !table_ok(table, a.p.shift, n, width)) return KVRT_EINVAL;
    if (!strided(q, KVRT_BF16, 2, 3, 16) || !strided(out, KVRT_BF16, 2, 3, 16)) return KVRT_EINVAL;
    for (int i = 0; i < 3; ++i)
        if (out->dims[i] != q->dims[i]) return KVRT_EINVAL;
    const int64_t hq = q->dims[1];
    if (q->dims[2] != pages->head_dim || hq < 1 || hq % pages->kv_heads != 0 || hq / pages->kv_heads > 64)
        return KVRT_EINVAL;
    if (!std::isfinite(scale) || window < 0 || max_q < 0 || q->dims[0] > kMaxRows) return KVRT_EINVAL;
    if (hq / pages->kv_heads * max_q >= (int64_t)1 << 30) return KVRT_EINVAL;  // rows of a head are numbered in 32 bits
    if (q->dims[0] == 0 || n == 0 || max_q == 0) return KVRT_OK;
    if (!disjoint(out) || !aligned(lengths, 4) || !aligned(starts, 4) || (granted && !aligned(granted, 4)) ||
        (width > 0 && !table->data))
        return KVRT_EINVAL;
    a.group = (int)(hq / pages->kv_heads);
    const AttendPlan plan = attend_plan(a.p.kv_heads, a.p.shift, pages->head_dim, n, width, q->dims[0], a.group, max_q);
    const int64_t heads = n * pages->kv_heads;
    if (!plan.chunk && plan.most * heads >= (int64_t)1 << 31) return KVRT_EINVAL;  // units are numbered in 32 bits
    if (plan.chunk && plan.tiles > 65535) return KVRT_EINVAL;                      // row tiles are a grid dimension
    if (plan.part_rows > 0 && (!aligned(work, 16) || work_bytes < part_bytes(plan.part_rows, pages->head_dim)))
        return KVRT_EINVAL;
    a.part_o = static_cast<float *>(work);
    a.part_ml = reinterpret_cast<float2 *>(static_cast<float *>(work) + plan.part_rows * pages->head_dim);
    a.wgs = plan.wgs;
    a.row_waves = plan.row_waves;
    a.tiles = (int)plan.tiles;
    a.splits = plan.splits;
    a.q = static_cast<const uint16_t *>(q->data);
    a.out = static_cast<uint16_t *>(out->data);
    a.q_row = q->strides[0];
    a.q_head = q->strides[1];
    a.o_row = out->strides[0];
    a.o_head = out->strides[1];
    a.table = static_cast<const int32_t *>(table->data);
    a.table_stride = table->strides[0];
    a.lengths = lengths;
    a.starts = starts;
    a.granted = granted;
    a.rows = q->dims[0];
    a.n = (int)n;
    a.width = (int)width;
    a.max_q = max_q;
    a.window = window >= width << a.p.shift ? 0 : window;  // (a window past the table's keys is none)
    a.scale_log2 = scale * 1.4426950408889634f;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (plan.chunk)
        return launch_block8_chunk(a, pages->dtype, pages->head_dim, st) == hipSuccess ? KVRT_OK : KVRT_EDEVICE;
    // Joined inside the launch: heads whose partials the last workgroup reads in a few
    // loads. Where that many workgroups per head fill the card, or a head never has
    // more, all are; else a second launch joins the others. The division follows the
    // shape alone; without arrival counters the second launch joins every head.
    bool join = false;
    a.join_most = 1;
    if (a.wgs > 1) {
        const int64_t rows = std::min<int64_t>(16, (int64_t)a.group * max_q);
        a.join_most = (int)std::min<int64_t>(32, kJoinBytes / (rows * pages->head_dim * 4));
        a.join_all = plan.most > a.join_most && heads * (a.join_most - 1) >= 512;
        a.counters = a.join_most > 1 ? block8_counter_slice(st) : nullptr;
        join = !a.counters || (plan.most > a.join_most && !a.join_all);
    }
    const hipError_t e = launch_block8_attend(a, pages->dtype, pages->head_dim, join, st);
    return e == hipSuccess ? KVRT_OK : KVRT_EDEVICE;
}

}  // extern "C"
