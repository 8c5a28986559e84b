// gla_prefill_sinks.hip -- batched causal prefill in a sliding window whose rows also see
// the first positions of their sequence (sinks): the prefill's code with the sinks'
// tiles in its lists. A translation unit of its own, so that both compile side by side.
#define GLA_PREFILL_SINKS 1
#include "gla_prefill.hip"
