// The kernel of prefill_attention.hip over the lists of shared_attention.hip, in f32, in a translation
// unit of its own so that it compiles in parallel.
#define KYRO_PREFILL_UNIT 5
#include "prefill_attention.hip"
