#include "attention_short.cuh"

namespace b200c {
int attention_short_forward_f16(const AttnArgs &a) { return as_dispatch<__half, AS_FORWARD>(a); }
int attention_short_dq_f16(const AttnArgs &a) { return as_dispatch<__half, AS_DQ>(a); }
int attention_short_dkv_f16(const AttnArgs &a) { return as_dispatch<__half, AS_DKV>(a); }
}  // namespace b200c
