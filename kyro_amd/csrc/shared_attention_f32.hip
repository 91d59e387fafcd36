// Attention over shared prefixes, f32.
#include "shared_attention.hpp"

namespace kyro {

hipError_t launch_shared_f32(const SharedArgs& s, hipStream_t stream) {
    switch (s.a.D) {
        case 64: launch_shared_dim<false, 64>(s, stream); break;
        case 80: launch_shared_dim<false, 80>(s, stream); break;
        case 96: launch_shared_dim<false, 96>(s, stream); break;
        case 112: launch_shared_dim<false, 112>(s, stream); break;
        case 128: launch_shared_dim<false, 128>(s, stream); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace kyro
