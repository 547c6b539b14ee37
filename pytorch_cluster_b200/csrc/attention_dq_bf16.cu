#include "attention_tensor_inst.cuh"
#include "attention_tensor_launch.h"

namespace b200c {
int attention_tensor_dq_bf16(const AttnArgs &a) { return at_dispatch<AtQueriesCall, __nv_bfloat16>(a); }
}  // namespace b200c
