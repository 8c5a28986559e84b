// gla_prefill_sinks.hip -- batched causal prefill in a sliding window whose rows also see
// the first positions of their sequence (sinks): gla_prefill.hip in its SINKS mode.
#define GLA_PREFILL_MODE 1
#include "gla_prefill.hip"
