// kvrt_shared_wide.hip — shared-prefix attention (kvrt_shared_kernel.h) at head_dim 256 and 512.
#include "kvrt_shared_kernel.h"

namespace kvrt {

hipError_t launch_shared_wide(const SharedArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
        case 256: return launch_shared_dim<256>(a, s);
        case 512: return launch_shared_dim<512>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace kvrt
