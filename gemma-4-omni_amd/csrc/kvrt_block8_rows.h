// kvrt_block8_rows.h — what the attention kernels over 8-bit pages share: requests
// and their row tiles, fp16 weights, the joining of partials.
#pragma once

#include "kvrt_block8.h"

namespace kvrt {

// Weights carry a factor 2^7 into fp16, which the division by their sum takes out.
constexpr float kWeightShift = 7.f;

// A request as one row tile sees it: `size` rows of a KV head's q heads x queries,
// query first (row r: query r / g, head r % g).
struct Rows {
    int start, count;  // packed rows
    int length;        // keys
    int n;             // rows of the tile (0: none)
    int first, last;   // positions of its first and last query
    int kend;          // keys [kstart, kend) can be seen by some row
    int kstart;
};

__device__ __forceinline__ Rows rows_of(const Block8AttendArgs &a, int start, int count, int length, int tile,
                                        int size) {
    Rows r;
    r.start = start;
    r.count = count;
    r.length = length;
    r.n = min(max(count * a.group - size * tile, 0), size);
    const int base = length - count;  // below 0: rows before the first key see nothing
    r.first = base + size * tile / a.group;
    r.last = base + (size * tile + max(r.n, 1) - 1) / a.group;
    r.kend = r.n > 0 ? min(max(r.last + 1, 0), length) : 0;
    r.kstart = a.window > 0 ? min(max(r.first - a.window + 1, 0), r.kend) : 0;
    return r;
}
// Request i from its words; what is out of range is brought into it and reported.
__device__ __forceinline__ Rows load_rows(const Block8AttendArgs &a, int i, int tile, int size, bool &bad) {
    const int cap = a.width << a.p.shift;
    const int len = a.lengths[i], s0 = a.starts[i];
    const int64_t m = a.granted ? (int64_t)a.granted[i] : (int64_t)a.starts[i + 1] - s0;
    const int length = min(max(len, 0), cap);
    const int start = (int)min((int64_t)max(s0, 0), a.rows);
    const int count = (int)min(min(max(m, (int64_t)0), (int64_t)a.max_q), a.rows - start);
    bad |= length != len || start != s0 || count != m;
    return rows_of(a, start, count, length, tile, size);
}
// The same, in scalar registers (every lane holds the same request).
__device__ __forceinline__ Rows uniform(Rows r) {
    r.start = __builtin_amdgcn_readfirstlane(r.start);
    r.count = __builtin_amdgcn_readfirstlane(r.count);
    r.length = __builtin_amdgcn_readfirstlane(r.length);
    r.n = __builtin_amdgcn_readfirstlane(r.n);
    r.first = __builtin_amdgcn_readfirstlane(r.first);
    r.last = __builtin_amdgcn_readfirstlane(r.last);
    r.kend = __builtin_amdgcn_readfirstlane(r.kend);
    r.kstart = __builtin_amdgcn_readfirstlane(r.kstart);
    return r;
}

// Running sum over the workgroup's NW waves (exclusive), the sum and the largest. lds
// holds 2 NW words.
template <int NW>
__device__ __forceinline__ int scan_wg(int x, int *lds, int &total, int &most) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = x, top = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(inc, d);
        if (lane >= d) inc += y;
        top = max(top, __shfl_xor(top, d));
    }
    __syncthreads();
    if (lane == 63) lds[wave] = inc, lds[NW + wave] = top;
    __syncthreads();
    int before = 0;
    total = 0, most = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < wave) before += lds[w];
        total += lds[w];
        most = max(most, lds[NW + w]);
    }
    return before + inc - x;
}

// Keys' words that nothing in the launch writes: uniform ones load as scalars.
typedef const __attribute__((address_space(4))) int32_t *ConstInts;
typedef const __attribute__((address_space(4))) float *ConstFloats;

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
}

// Joins partials p = 0 .. n - 1 of four output elements of a row, in their order,
// B at a time: ld(p, ml, o) reads one. The decode launch that makes the partials and its
// join kernel both use it, with the same B, so both give the same bits.
template <int B = 16, class Ld>
__device__ __forceinline__ void join_partials(int n, Ld ld, float &M, float &sum, float4 &o) {
    for (int p0 = 0; p0 < n; p0 += B) {
        float2 ml[B];
        float4 x[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            ml[i] = make_float2(kNegBig, 0.f);
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p0 + i < n) ld(p0 + i, ml[i], x[i]);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < B; ++i) top = fmaxf(top, ml[i].x);
        const float c = __builtin_amdgcn_exp2f(M - top);
        sum *= c;
        o = make_float4(o.x * c, o.y * c, o.z * c, o.w * c);
        M = top;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const float f = __builtin_amdgcn_exp2f(ml[i].x - M);
            sum = fmaf(ml[i].y, f, sum);
            o = make_float4(fmaf(x[i].x, f, o.x), fmaf(x[i].y, f, o.y), fmaf(x[i].z, f, o.z), fmaf(x[i].w, f, o.w));
        }
    }
}

// Four elements of a row of the answer: dims d .. d + 3 of row `row` of the head.
__device__ __forceinline__ void store_out(const Block8AttendArgs &a, const Rows &r, int head, int row, int d, float4 o,
                                          float sum) {
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    const int qr = row / a.group, hr = row - qr * a.group;
    uint16_t *out = a.out + (int64_t)(r.start + qr) * a.o_row + (int64_t)(head * a.group + hr) * a.o_head + d;
    *reinterpret_cast<uint2 *>(out) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

}  // namespace kvrt
