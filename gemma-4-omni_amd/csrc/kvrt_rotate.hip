// kvrt_rotate.hip — query, key and value heads normed and rotated in one pass.
//
// Per token and head, x of head_dim D:
//   y = x * w / sqrt(mean(x^2) + eps)                    where the head's kind is normed
//   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)         for each of F pairs of dims
// with c, s = scaling * cos, sin of position[axis of the pair] * inv_freq; pairs are
// (i, i + F) or (2i, 2i + 1), dims from 2F on pass, value heads are not rotated. Sums,
// angles and products in fp32 and better, one rounding to bf16 at the end.
//
// An angle is kept in turns, as a 64-bit fraction: the table holds inv_freq / 2 pi mod 1
// in units of 2^-64, and position times that, mod 2^64, drops whole turns exactly. Its
// high word (two 32-bit products, one where an fp64 product and its reduction take five
// instructions) is within 2^-32 turns for positions up to 2^31, and the hardware's sine
// and cosine take turns.
//
// A row's D / 16 lanes hold 16 dims each: both members of 8 pairs, so nothing is
// exchanged between lanes but the sum of squares, and a lane reads and writes 16 bytes
// twice. A group of lanes takes `per` heads of one kind and token: their rows are loaded
// at once and share sines, cosines and weights.
//
// What bounds it: long prompts the bytes (4 x 4096 tokens of 16 + 8 heads of 128: 201 MB in
// 39 us, 5.2 TB/s; a copy of 1 GiB reaches 5.1), short calls the launch: 2.8 us for one token.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "kvrt.h"
#include "kvrt_device.h"

namespace kvrt {

namespace {

constexpr int kKinds = 3;  // query, key, value heads
constexpr int kMaxAxes = 4;
// Lanes of a launch of one head per group up to which that is what a group takes, about a
// round of the card's lanes; past it the sines that four heads share count. us a call of one
// and of four heads a group (head_dim 128, 16 + 8 heads): 4 thousand lanes 3.3 and 4.3, 131
// thousand 4.5 and 4.9, 197 thousand 5.6 and 5.3, 1 million 18.1 and 13.0; the other dims
// cross at the same place.
constexpr int64_t kOneHeadLanes = 160 * 1024;
// Calls past that store around the L2, whose 32 MB would be written back after the last lane
// has ended, and calls of more than this many lanes (32 bytes each, in and out) load around it
// too, so that what was read does not push the answers out of the last cache. us a call, and
// of it and a reader of its query heads, head_dim 128, 16 + 8 heads, by MB of answers:
//   plain 8.4 6.4 / 11.0, 25 12.2 / 18.4, 101 46.1 / 65.9, 403 162 / 246
//   stores around 5.7 / 10.2, 10.7 / 18.4, 43.0 / 67.2, 154 / 254
//   stores and loads 5.8 / 10.4, 10.2 / 19.0, 43.1 / 64.9, 149 / 238
constexpr int64_t kLargeLanes = 1024 * 1024;

struct RotateArgs {
    const uint16_t *src[kKinds];
    uint16_t *dst[kKinds];
    int64_t s_item[kKinds], s_head[kKinds], s_row[kKinds];  // strides, elements
    int64_t d_item[kKinds], d_head[kKinds], d_row[kKinds];
    int heads[kKinds];
    int chunks[kKinds];      // groups of `per` heads (0: the kind is absent)
    const float *weight[2];  // [D] or null: ones
    const uint64_t *turns;   // [F]
    const uint8_t *axis;     // [F] or null: all 0
    const void *pos;
    int64_t p_axis, p_item, p_row;
    int pos64, axes;
    int rows;                // per item
    int freqs;
    int norm;                // bit per kind
    uint32_t groups;         // tokens * chunks of all kinds
    float eps, scaling;
};

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void widen(u32x4_t x, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(x[i]), f[2 * i + 1] = bf16_hi(x[i]);
}
__device__ __forceinline__ u32x4_t narrow(const float *f) {
    return (u32x4_t){pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
}

// Position p on axis `axis` of a token.
__device__ __forceinline__ int position(const RotateArgs &a, int axis, int item, int row) {
    const int64_t at = axis * a.p_axis + item * a.p_item + row * a.p_row;
    return a.pos64 ? (int)static_cast<const int64_t *>(a.pos)[at] : static_cast<const int32_t *>(a.pos)[at];
}

}  // namespace

// PASS: a kind of heads that is not normed has dims that do not turn. (4 x 291 tokens of 10 heads of
// 512, normed: 6.9 us, 7.2 in the other variant.)
template <int D, int PER, bool ADJACENT, bool LARGE, bool PASS>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
    constexpr int LANES = D / 16;
    const uint32_t group = (blockIdx.x * 256u + threadIdx.x) / LANES;
    if (group >= a.groups) return;  // whole groups of lanes: nothing is exchanged between groups
    const int j = threadIdx.x % LANES;
    const uint32_t all = a.chunks[0] + a.chunks[1] + a.chunks[2];
    const int token = group / all, chunk = group - token * all;
    const int item = (uint32_t)token / (uint32_t)a.rows, row = token - item * a.rows;
    const bool is_q = chunk < a.chunks[0], is_k = !is_q && chunk < a.chunks[0] + a.chunks[1];
    const int h0 = PER * (chunk - (is_q ? 0 : is_k ? a.chunks[0] : a.chunks[0] + a.chunks[1]));
    const int heads = is_q ? a.heads[0] : is_k ? a.heads[1] : a.heads[2];
    const auto pick = [&](const auto(&x)[kKinds]) __attribute__((always_inline)) { return is_q ? x[0] : is_k ? x[1] : x[2]; };
    // this lane's dims: lo .. lo + 7 and hi .. hi + 7
    const int f0 = 8 * j;
    const bool pairs = f0 < a.freqs, turned = pairs && (is_q || is_k);
    int lo, hi;
    if (ADJACENT) {
        lo = 16 * j, hi = lo + 8;
    } else {
        lo = pairs ? f0 : a.freqs + f0;
        hi = pairs ? a.freqs + f0 : D / 2 + f0;
    }
    const int64_t s_head = pick(a.s_head), d_head = pick(a.d_head);
    const uint16_t *src = pick(a.src) + item * pick(a.s_item) + row * pick(a.s_row) + h0 * s_head;
    uint16_t *dst = pick(a.dst) + item * pick(a.d_item) + row * pick(a.d_row) + h0 * d_head;
    u32x4_t x[PER][2];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const uint16_t *p = src + min(u, heads - 1 - h0) * s_head;  // past the last head: the last once more
        const auto *one = reinterpret_cast<const u32x4_t *>(p + lo), *two = reinterpret_cast<const u32x4_t *>(p + hi);
        if constexpr (LARGE) {
            x[u][0] = __builtin_nontemporal_load(one);
            x[u][1] = __builtin_nontemporal_load(two);
        } else {
            x[u][0] = *one;
            x[u][1] = *two;
        }
    }
    const bool normed = (a.norm >> (is_q ? 0 : is_k ? 1 : 2)) & 1;
    const float *weight = is_q ? a.weight[0] : is_k ? a.weight[1] : nullptr;
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 1.f;
    if (normed && weight) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 y = *reinterpret_cast<const float4 *>(weight + (i < 2 ? lo : hi - 8) + 4 * i);
            w[4 * i] = y.x, w[4 * i + 1] = y.y, w[4 * i + 2] = y.z, w[4 * i + 3] = y.w;
        }
    }
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
    if (turned) {
        int p[kMaxAxes];
        p[0] = position(a, 0, item, row);
#pragma unroll
        for (int e = 1; e < kMaxAxes; ++e) p[e] = a.axes > e ? position(a, e, item, row) : p[0];
        uint2 ax = make_uint2(0u, 0u);
        if (a.axis) ax = *reinterpret_cast<const uint2 *>(a.axis + f0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint64_t t = a.turns[f0 + i];
            const uint32_t e = ((i < 4 ? ax.x : ax.y) >> (8 * (i & 3))) & 0xffu;
            const int at = e == 0 ? p[0] : e == 1 ? p[1] : e == 2 ? p[2] : p[3];
            // high word of at * t mod 2^64, at as a signed number
            const uint32_t low = (uint32_t)t, high = (uint32_t)(t >> 32);
            const uint32_t turn = (uint32_t)at * high + __umulhi((uint32_t)at, low) - (at < 0 ? low : 0u);
            const float r = (float)(int32_t)turn * 0x1p-32f;  // in [-1/2, 1/2]
            c[i] = __builtin_amdgcn_cosf(r) * a.scaling;
            s[i] = __builtin_amdgcn_sinf(r) * a.scaling;
        }
    }
    // PASS: dims that neither turn nor are normed leave as they came; computed (c = 1, s = 0) they
    // would be NaN beside an infinity. (A mask: told of a condition, the compiler branches.)
    uint32_t same = turned || normed ? 0u : ~0u;
    if constexpr (PASS) asm volatile("" : "+v"(same));
    const auto out = [&](u32x4_t from, const float *to) __attribute__((always_inline)) {
        if constexpr (PASS) return (from & same) | (narrow(to) & ~same);
        else return narrow(to);
    };
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        float y[16];
        widen(x[u][0], y);
        widen(x[u][1], y + 8);
        if (normed) {
            const auto mean = [&](float eps) __attribute__((always_inline)) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) sum = fmaf(y[i], y[i], sum);
                return fmaf(group_sum<LANES>(sum), 1.0f / D, eps);
            };
            float m = mean(a.eps);
            // where squares leave fp32's range, x and eps are taken by a power of two (exact, and
            // the quotient the same)
            const float by = m < 0x1p-100f ? 0x1p100f : m > 0x1p100f ? 0x1p-70f : 1.f;
            if (__any(by != 1.f)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] *= by;
                m = mean(a.eps * by * by);
            }
            const float inv = __builtin_amdgcn_rsqf(m);  // within 1 ulp
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] *= inv * w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float &one = ADJACENT ? y[2 * i] : y[i], &two = ADJACENT ? y[2 * i + 1] : y[8 + i];
            const float t = one;
            one = fmaf(t, c[i], -(two * s[i]));
            two = fmaf(two, c[i], t * s[i]);
        }
        if (h0 + u < heads) {
            auto *one = reinterpret_cast<u32x4_t *>(dst + u * d_head + lo), *two = reinterpret_cast<u32x4_t *>(dst + u * d_head + hi);
            if constexpr (PER > 1) {
                __builtin_nontemporal_store(out(x[u][0], y), one);
                __builtin_nontemporal_store(out(x[u][1], y + 8), two);
            } else {
                *one = out(x[u][0], y);
                *two = out(x[u][1], y + 8);
            }
        }
    }
}

namespace {

template <int D>
hipError_t launch_rotate(RotateArgs &a, int64_t tokens, int per, bool large, bool adjacent, bool pass, hipStream_t s) {
    int all = 0;
    for (int i = 0; i < kKinds; ++i) all += a.chunks[i] = (a.heads[i] + per - 1) / per;
    a.groups = (uint32_t)(tokens * all);
    const dim3 grid((unsigned)((tokens * all * (D / 16) + 255) / 256));
    const auto launch = [&](auto per_c, auto large_c, auto adjacent_c, auto pass_c) {
        hipLaunchKernelGGL((rotate_kernel<D, decltype(per_c)::value, decltype(adjacent_c)::value, decltype(large_c)::value,
                                          decltype(pass_c)::value>),
                           grid, dim3(256), 0, s, a);
    };
    const std::true_type yes{};
    const std::false_type no{};
    const auto order = [&](auto per_c, auto large_c) {
        if (adjacent && pass) launch(per_c, large_c, yes, yes);
        else if (adjacent) launch(per_c, large_c, yes, no);
        else if (pass) launch(per_c, large_c, no, yes);
        else launch(per_c, large_c, no, no);
    };
    if (per == 1) order(std::integral_constant<int, 1>{}, no);
    else if (!large) order(std::integral_constant<int, 4>{}, no);
    else order(std::integral_constant<int, 4>{}, yes);
    return hipGetLastError();
}

bool aligned_to(const void *p, size_t to) { return p && reinterpret_cast<uintptr_t>(p) % to == 0; }

// Heads [n, H, Q, D]: bf16, last dim contiguous, 16-byte aligned rows; `out`: no row written twice.
bool heads_ok(const kvrt_tensor *t, bool out) {
    if (!t || t->dtype != KVRT_BF16 || t->ndim != 4) return false;
    for (int i = 0; i < 4; ++i)
        if (t->dims[i] < 0 || t->dims[i] > INT32_MAX) return false;
    for (int i = 0; i < 4; ++i)
        if (t->dims[i] == 0) return true;
    if (!aligned_to(t->data, 16) || t->strides[3] != 1) return false;
    for (int i = 0; i < 3; ++i)
        if (t->dims[i] > 1 && (t->strides[i] < (out ? 1 : 0) || t->strides[i] % 8 != 0)) return false;
    return true;
}

}  // namespace

}  // namespace kvrt

using namespace kvrt;

extern "C" {

int kvrt_rotation_turns(const double *inv_freq, int32_t n, uint64_t *turns) {
    if (n < 0 || (n > 0 && (!inv_freq || !turns))) return KVRT_EINVAL;
    for (int i = 0; i < n; ++i)
        if (!std::isfinite(inv_freq[i])) return KVRT_EINVAL;
    for (int i = 0; i < n; ++i) {
        // whole turns drop; what is left, in [0, 1), times 2^64 is rounded to a whole
        // number (1 - 2^-54 and above to 2^64, a whole turn)
        const long double t = (long double)inv_freq[i] / 6.283185307179586476925286766559005768L;
        const long double f = std::round((t - std::floor(t)) * 0x1p64L);
        turns[i] = f >= 0x1p64L ? 0u : (uint64_t)f;
    }
    return KVRT_OK;
}

int kvrt_rotate_heads_async(const kvrt_rotation *rot, const kvrt_tensor *q, const kvrt_tensor *k, const kvrt_tensor *v,
                            const kvrt_tensor *positions, const kvrt_tensor *out_q, const kvrt_tensor *out_k,
                            const kvrt_tensor *out_v, void *stream) {
    const kvrt_tensor *in[kKinds] = {q, k, v}, *out[kKinds] = {out_q, out_k, out_v}, *shape = nullptr;
    if (!rot || (rot->head_dim != 64 && rot->head_dim != 128 && rot->head_dim != 256 && rot->head_dim != 512))
        return KVRT_EINVAL;
    const int D = rot->head_dim;
    if (rot->n_freq < 0 || rot->n_freq % 8 != 0 || 2 * rot->n_freq > D || rot->n_axes < 1 || rot->n_axes > kMaxAxes ||
        rot->norm < 0 || rot->norm > 7 || (rot->adjacent != 0 && rot->adjacent != 1) || !(rot->eps >= 0.f) ||
        !std::isfinite(rot->eps) || !std::isfinite(rot->scaling))
        return KVRT_EINVAL;
    if (rot->n_freq > 0 && (!aligned_to(rot->turns, 8) || (rot->axis ? !aligned_to(rot->axis, 8) : rot->n_axes > 1)))
        return KVRT_EINVAL;
    for (const float *w : {rot->q_weight, rot->k_weight})
        if (w && !aligned_to(w, 16)) return KVRT_EINVAL;
    RotateArgs a{};
    int64_t heads = 0;
    for (int i = 0; i < kKinds; ++i) {
        if (!in[i] != !out[i]) return KVRT_EINVAL;
        if (!in[i]) continue;
        if (!heads_ok(in[i], false) || !heads_ok(out[i], true) || in[i]->dims[3] != D) return KVRT_EINVAL;
        for (int e = 0; e < 4; ++e)
            if (out[i]->dims[e] != in[i]->dims[e]) return KVRT_EINVAL;
        if (shape && (shape->dims[0] != in[i]->dims[0] || shape->dims[2] != in[i]->dims[2])) return KVRT_EINVAL;
        shape = in[i];
        a.src[i] = static_cast<const uint16_t *>(in[i]->data);
        a.dst[i] = static_cast<uint16_t *>(out[i]->data);
        a.s_item[i] = in[i]->strides[0], a.s_head[i] = in[i]->strides[1], a.s_row[i] = in[i]->strides[2];
        a.d_item[i] = out[i]->strides[0], a.d_head[i] = out[i]->strides[1], a.d_row[i] = out[i]->strides[2];
        a.heads[i] = (int)in[i]->dims[1];
        heads += a.heads[i];
    }
    if (!shape) return KVRT_EINVAL;
    const int64_t n = shape->dims[0], rows = shape->dims[2];
    // 32 bits count a launch's threads (n, rows and heads are below 2^31)
    if (n > 0 && rows > 0 && heads > 0 && (n > INT32_MAX / rows || n * rows > (int64_t)(UINT32_MAX - 255) / (heads * (D / 16))))
        return KVRT_EINVAL;
    if (rot->n_freq > 0) {
        const kvrt_tensor *p = positions;
        if (!p || p->ndim != 3 || (p->dtype != KVRT_INT32 && p->dtype != KVRT_INT64) || p->dims[0] != rot->n_axes ||
            p->dims[1] != n || p->dims[2] != rows)
            return KVRT_EINVAL;
        a.pos64 = p->dtype == KVRT_INT64;
        if (n > 0 && rows > 0 && !aligned_to(p->data, a.pos64 ? 8 : 4)) return KVRT_EINVAL;
        for (int i = 0; i < 3; ++i)
            if (p->strides[i] < 0) return KVRT_EINVAL;
        a.pos = p->data;
        a.p_axis = p->strides[0], a.p_item = p->strides[1], a.p_row = p->strides[2];
    }
    if (n == 0 || rows == 0 || heads == 0) return KVRT_OK;
    a.weight[0] = rot->q_weight, a.weight[1] = rot->k_weight;
    a.turns = rot->turns;
    a.axis = rot->axis;
    a.axes = rot->n_axes;
    a.rows = (int)rows;
    a.freqs = rot->n_freq;
    a.norm = rot->norm;
    a.eps = rot->eps;
    a.scaling = rot->scaling;
    const int64_t tokens = n * rows;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t lanes = tokens * heads * (D / 16);
    const int per = lanes <= kOneHeadLanes ? 1 : 4;
    const bool large = lanes > kLargeLanes;
    const bool adj = rot->adjacent != 0;
    bool pass = false;
    for (int i = 0; i < kKinds; ++i) pass |= a.heads[i] > 0 && !(rot->norm >> i & 1) && (i == 2 || 2 * rot->n_freq < D);
    hipError_t e;
    switch (D) {
        case 64: e = launch_rotate<64>(a, tokens, per, large, adj, pass, s); break;
        case 128: e = launch_rotate<128>(a, tokens, per, large, adj, pass, s); break;
        case 256: e = launch_rotate<256>(a, tokens, per, large, adj, pass, s); break;
        default: e = launch_rotate<512>(a, tokens, per, large, adj, pass, s); break;
    }
    return e == hipSuccess ? KVRT_OK : KVRT_EDEVICE;
}

}  // extern "C"
