// kvrt_shared_chunk.hip — chunks behind a shared prefix (kvrt_prefill.h, SHARED) at head_dim
// 64 and 128, and their dispatch.
//
// The prefill's tiles as they are: 32 rows of (query, head) a wave on 32x32 matrix
// instructions, online softmax, P in two bf16 terms. Keys are numbered in whole blocks of 32,
// the prefix first, so that the only new work of a block is whose slot it lies in, and, where
// asked for, the scores' cap and bias. A tile that ends with NaN in a row whose scores are
// numbers met NaN or infinities in V, and is computed again row by row.
// Measured: 4 x 512 queries of 16 heads of 128 behind 1400 rows and 577 to 700 of their own 52 us
// a call, 575 TFLOP/s with P counted once (on the tiles of kvrt_shared_kernel.h, which calls with
// masks take, 80); on pages 58; with an infinity in the prefix's V 4.7 ms. 2 x 291 capped ones
// over 2000 24.5, not capped 20.3. The matrix cores work for 50 % of the waves' life and vector
// instructions for 51 %: two waves on a SIMD that follow each other. The capped chunk has one
// wave on a SIMD, 17 % matrix, 35 % vector instructions and 36 % waits.
#include "kvrt_prefill.h"

namespace kvrt {

hipError_t launch_shared_chunk(const SharedChunkArgs &a, int head_dim, hipStream_t s) {
    const int rw = a.row_waves, ks = a.key_parts;
    hipError_t e = hipErrorInvalidValue;
    const auto shapes = [&](auto d_c) {
        constexpr int D = decltype(d_c)::value;
        if (rw == 4 && ks == 1) return launch_prefill_shape<D, 4, 1, 2>(a, s);
        if (rw == 2 && ks == 2) return launch_prefill_shape<D, 2, 2, 2>(a, s);
        if (rw == 2 && ks == 4) return launch_prefill_shape<D, 2, 4, 2>(a, s);
        if (rw == 1 && ks == 4 && a.kv.layout == KVRT_LAYOUT_CONTIG)
            return launch_prefill_layout<D, 1, 4, 2, KVRT_LAYOUT_CONTIG>(a, s);
        if (rw == 1 && ks == 4 && a.kv.layout == KVRT_LAYOUT_RING)
            return launch_prefill_layout<D, 1, 4, 2, KVRT_LAYOUT_RING>(a, s);
        return hipErrorInvalidValue;
    };
    if (head_dim == 64) e = shapes(std::integral_constant<int, 64>{});
    else if (head_dim == 128) e = shapes(std::integral_constant<int, 128>{});
    else e = launch_shared_chunk_wide(a, head_dim, s);
    return e != hipSuccess || a.n_ksplit == 1 ? e : launch_prefill_merge(a, head_dim, s);
}

}  // namespace kvrt
