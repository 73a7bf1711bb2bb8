// kvrt_shared.hip — shared-prefix attention (kvrt_shared_kernel.h) at head_dim 64 and 128.
#include "kvrt_shared_kernel.h"

namespace kvrt {

hipError_t launch_shared(const SharedArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_shared_dim<64>(a, s);
        case 128: return launch_shared_dim<128>(a, s);
        default: return launch_shared_wide(a, head_dim, s);
    }
}

}  // namespace kvrt
