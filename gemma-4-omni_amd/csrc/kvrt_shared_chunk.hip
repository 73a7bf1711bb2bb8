// kvrt_shared_chunk.hip — chunks behind a shared prefix (kvrt_prefill.h, SHARED) at head_dim
// 64 and 128, and their dispatch.
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
