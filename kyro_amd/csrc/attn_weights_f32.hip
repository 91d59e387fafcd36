// The f32 instances of the attention-weight kernels, in a file of their own so that they compile beside the
// bf16 ones.
#define KYRO_WEIGHTS_F32 1
#include "attn_weights.hip"
