// The kernel of prefill_attention.hip over the lists of shared_attention.hip, in bf16 up to head dim 128, in a translation
// unit of its own so that it compiles in parallel.
#define KYRO_PREFILL_UNIT 3
#include "prefill_attention.hip"
