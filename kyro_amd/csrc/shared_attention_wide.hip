// Attention over shared prefixes, bf16 at head dims 160, 192, 224 and 256.
#include "shared_attention.hpp"

namespace kyro {

hipError_t launch_shared_wide(const SharedArgs& s, hipStream_t stream) {
    switch (s.a.D) {
        case 160: launch_shared_dim<true, 160>(s, stream); break;
        case 192: launch_shared_dim<true, 192>(s, stream); break;
        case 224: launch_shared_dim<true, 224>(s, stream); break;
        case 256: launch_shared_dim<true, 256>(s, stream); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace kyro
