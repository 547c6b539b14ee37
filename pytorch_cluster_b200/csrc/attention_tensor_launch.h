// Launches of the attention kernels for 16-bit types, one translation unit per type and direction (they compile in
// parallel).
#pragma once

#include "attention.cuh"

namespace b200c {

int attention_tensor_forward_bf16(const AttnArgs &a);
int attention_tensor_forward_f16(const AttnArgs &a);
int attention_tensor_dq_bf16(const AttnArgs &a);
int attention_tensor_dq_f16(const AttnArgs &a);
int attention_tensor_dkv_bf16(const AttnArgs &a);
int attention_tensor_dkv_f16(const AttnArgs &a);

int attention_short_forward_bf16(const AttnArgs &a);
int attention_short_forward_f16(const AttnArgs &a);
int attention_short_dq_bf16(const AttnArgs &a);
int attention_short_dq_f16(const AttnArgs &a);
int attention_short_dkv_bf16(const AttnArgs &a);
int attention_short_dkv_f16(const AttnArgs &a);

}  // namespace b200c
