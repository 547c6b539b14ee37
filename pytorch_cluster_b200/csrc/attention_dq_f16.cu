#include "attention_tensor_inst.cuh"
#include "attention_tensor_launch.h"

namespace b200c {
int attention_tensor_dq_f16(const AttnArgs &a) { return at_dispatch<AtQueriesCall, __half>(a); }
}  // namespace b200c
