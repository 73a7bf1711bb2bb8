// kvrt_block8_chunk.hip — chunk attention over 8-bit pages, head_dim 64, 128 and 512
// (MFMA results in ordinary registers).
#include <algorithm>

#include "kvrt_block8_chunk.h"

namespace kvrt {

hipError_t launch_block8_chunk(const Block8AttendArgs &a, int dtype, int head_dim, hipStream_t s) {
    const bool i8 = dtype == KVRT_INT8;
    switch (head_dim) {
        case 64: return i8 ? launch_chunk<KVRT_INT8, 64>(a, s) : launch_chunk<KVRT_E4M3, 64>(a, s);
        case 128: return i8 ? launch_chunk<KVRT_INT8, 128>(a, s) : launch_chunk<KVRT_E4M3, 128>(a, s);
        case 256: return launch_block8_chunk_wide(a, dtype, head_dim, s);
        case 512: return i8 ? launch_chunk<KVRT_INT8, 512>(a, s) : launch_chunk<KVRT_E4M3, 512>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace kvrt
