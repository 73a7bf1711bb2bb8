// kvrt_shared_chunk_wide.hip — chunks behind a shared prefix (kvrt_prefill.h, SHARED) at
// head_dim 256 and 512, whose output accumulators live in AGPRs.
#include "kvrt_prefill.h"

namespace kvrt {

hipError_t launch_shared_chunk_wide(const SharedChunkArgs &a, int head_dim, hipStream_t s) {
    const int rw = a.row_waves, ks = a.key_parts;
    if (head_dim == 256) {
        if (rw == 4 && ks == 1) return launch_prefill_shape<256, 4, 1, 2>(a, s);
        if (rw == 2 && ks == 2) return launch_prefill_shape<256, 2, 2, 2>(a, s);
    }
    if (head_dim == 512 && rw == 4 && ks == 1) return launch_prefill_shape<512, 4, 1, 2>(a, s);
    return hipErrorInvalidValue;
}

}  // namespace kvrt
