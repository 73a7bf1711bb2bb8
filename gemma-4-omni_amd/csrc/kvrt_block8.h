// kvrt_block8.h — shared by the kernels of 8-bit pages with one scale per (page,
// KV head) and by their C entry points: arguments, code conversions, page lookup.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kvrt.h"
#include "kvrt_wave.h"

namespace kvrt {

constexpr float kScaleLow = 0x1p-64f, kScaleHigh = 0x1p32f;  // range of a page's scale

// One layer's coded pages as the kernels see them. A page's rows of one head are
// contiguous: (page * kv_heads + head) * block * D bytes from k or v.
struct Block8View {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    int32_t *status;
    int pages, kv_heads, block, shift;  // shift: log2(block)
};

struct Block8TablesArgs {
    int32_t *table, *mapped, *free_pages, *free_count, *work, *status;
    int n, max_pages, pool_pages, block, shift;
    const int32_t *lengths, *new_rows;
    int64_t rows;
    int32_t *starts, *slot_map, *out_lengths, *granted;
};

struct Block8AppendArgs {
    Block8View p;
    const uint16_t *x[2];      // K, V rows
    int64_t row[2], head[2];   // their strides, elements
    const int32_t *slots;
    int64_t rows;
    int chunk;                 // slots one wave looks through
};

struct Block8GatherArgs {
    Block8View p;
    const int32_t *table, *lengths, *start_pos;
    int64_t table_stride;
    int n, width, lmax;
    void *out[2];
    int64_t item[2], head[2], row[2];  // strides, elements
    int fp32;
    void *mask;
    int mask_dtype;
    int64_t mask_stride;
};

struct Block8AttendArgs {
    Block8View p;
    const uint16_t *q;
    uint16_t *out;
    int64_t q_row, q_head, o_row, o_head;  // strides, elements
    const int32_t *table, *lengths, *starts, *granted;
    int64_t table_stride, rows;            // packed rows of q
    int n, width, group, max_q, window;
    int wgs;                               // workgroups the keys are divided over (each row tile)
    int join_most;                         // partials of a head that one workgroup may join (sets the division)
    int join_all;                          // divide so that no head has more
    float scale_log2;                      // scale * log2(e)
    float *part_o;                         // partials of divided heads [tile][wg][2][16 rows][D]
    float2 *part_ml;                       // their (max, sum) [tile][wg][2][16]
    uint32_t *counters;                    // arrivals [wg], zero between launches; none: a second launch joins
    // chunks (kvrt_block8_chunk.h): tiles of 32 * row_waves rows, at most `tiles` of them,
    // keys divided over `splits` workgroups; partials [tile][head][split][row][D]
    int row_waves, tiles, splits;
};

constexpr int kBlock8MaxWgs = 1024;  // workgroups the keys are divided over, at most

hipError_t launch_block8_tables(const Block8TablesArgs &a, hipStream_t s);
hipError_t launch_block8_append(const Block8AppendArgs &a, int dtype, int head_dim, hipStream_t s);
hipError_t launch_block8_gather(const Block8GatherArgs &a, int dtype, int head_dim, hipStream_t s);
hipError_t launch_block8_attend(const Block8AttendArgs &a, int dtype, int head_dim, bool join, hipStream_t s);
hipError_t launch_block8_chunk(const Block8AttendArgs &a, int dtype, int head_dim, hipStream_t s);
// kBlock8MaxWgs zeroed arrival counters for a call on that stream; nullptr: none left
// (the call then joins in a second launch: same division, same order, same bits).
uint32_t *block8_counter_slice(hipStream_t s);

// ---- codes ----------------------------------------------------------------------
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Four codes of a word as fp16, exactly: x = codes 0, 1, y = codes 2, 3.
// int8: with its sign bit flipped a code is c + 128 in 0 .. 255, as low mantissa
// bits under the exponent of 1024 the number 1152 + c; one subtraction leaves c.
// (e4m3 values, their subnormals included, are normal or subnormal fp16 numbers.)
template <int CODE>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t &x, uint32_t &y) {
    if constexpr (CODE == KVRT_INT8) {
        const f16x2_t off = {(_Float16)1152.f, (_Float16)1152.f};
        w ^= 0x80808080u;
        const uint32_t a = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u);
        const uint32_t b = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
        x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, a) - off);
        y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, b) - off);
    } else {
        x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
        y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
}

// The same as floats.
template <int CODE>
__device__ __forceinline__ void codes_to_f32(uint32_t w, float (&x)[4]) {
    if constexpr (CODE == KVRT_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
    } else {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
    }
}

template <int CODE>
constexpr float kCodeTop = CODE == KVRT_INT8 ? 127.f : 448.f;

// Four values in units of the scale to codes: nearest, ties to even, clamped to
// the largest code; NaN becomes 0.
template <int CODE>
__device__ __forceinline__ uint32_t f32_to_codes(const float (&x)[4]) {
    float c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = fminf(fmaxf(x[i], -kCodeTop<CODE>), kCodeTop<CODE>);
        c[i] = x[i] != x[i] ? 0.f : c[i];
    }
    if constexpr (CODE == KVRT_INT8) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)rintf(c[i]) & 0xffu) << (8 * i);
        return w;
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
    }
}

// A scale as it is used, whatever the word holds (NaN: the lowest).
__device__ __forceinline__ float scale_in_range(float s) { return fminf(fmaxf(s, kScaleLow), kScaleHigh); }

__device__ __forceinline__ void raise(int32_t *status, int bit) { atomicOr(status, bit); }

}  // namespace kvrt
