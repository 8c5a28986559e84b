// gla_decode_prefix.hip -- the part of a batch's decode that groups of its sequences have in
// common, as one matrix product a group: gla_prefill.hip in its PREFIX mode.
#define GLA_PREFILL_MODE 2
#include "gla_prefill.hip"
