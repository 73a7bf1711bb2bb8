// kvrt_block8_chunk.hip — chunk attention over 8-bit pages: instantiations.
#include <algorithm>

#include "kvrt_block8_chunk.h"

namespace kvrt {

template <int CODE>
static hipError_t launch_chunk_code(const Block8AttendArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_chunk<CODE, 64>(a, s);
        case 128: return launch_chunk<CODE, 128>(a, s);
        case 256: return launch_chunk<CODE, 256>(a, s);
        case 512: return launch_chunk<CODE, 512>(a, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_block8_chunk(const Block8AttendArgs &a, int dtype, int head_dim, hipStream_t s) {
    return dtype == KVRT_INT8 ? launch_chunk_code<KVRT_INT8>(a, head_dim, s) : launch_chunk_code<KVRT_E4M3>(a, head_dim, s);
}

}  // namespace kvrt
