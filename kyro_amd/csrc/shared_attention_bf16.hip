// Attention over shared prefixes, bf16 up to head dim 128.
#include "shared_attention.hpp"

namespace kyro {

hipError_t launch_shared_bf16(const SharedArgs& s, hipStream_t stream) {
    switch (s.a.D) {
        case 64: launch_shared_dim<true, 64>(s, stream); break;
        case 80: launch_shared_dim<true, 80>(s, stream); break;
        case 96: launch_shared_dim<true, 96>(s, stream); break;
        case 112: launch_shared_dim<true, 112>(s, stream); break;
        case 128: launch_shared_dim<true, 128>(s, stream); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace kyro
