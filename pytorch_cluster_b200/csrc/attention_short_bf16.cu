#include "attention_short.cuh"

namespace b200c {
int attention_short_forward_bf16(const AttnArgs &a) { return as_dispatch<__nv_bfloat16, AS_FORWARD>(a); }
int attention_short_dq_bf16(const AttnArgs &a) { return as_dispatch<__nv_bfloat16, AS_DQ>(a); }
int attention_short_dkv_bf16(const AttnArgs &a) { return as_dispatch<__nv_bfloat16, AS_DKV>(a); }
}  // namespace b200c
