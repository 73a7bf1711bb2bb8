// kvrt_block8_chunk_wide.hip — chunk attention over 8-bit pages, head_dim 256 (output
// accumulators in AGPRs: one wave per SIMD has more registers than VGPRs).
#include <algorithm>

#include "kvrt_block8_chunk.h"

namespace kvrt {

hipError_t launch_block8_chunk_wide(const Block8AttendArgs &a, int dtype, int head_dim, hipStream_t s) {
    if (head_dim != 256) return hipErrorInvalidValue;
    return dtype == KVRT_INT8 ? launch_chunk<KVRT_INT8, 256>(a, s) : launch_chunk<KVRT_E4M3, 256>(a, s);
}

}  // namespace kvrt
