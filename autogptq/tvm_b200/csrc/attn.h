// The parts of b200gptq_attn.
#pragma once

#include <cuda_runtime.h>

#include "../../../include/b200gptq.h"

namespace b200gptq {

struct AttnSplit { int own, prefix; };      // runs that the keys of a sequence's own cache and of the prefix are cut into

bool attn_pdl_enabled();

AttnSplit attn_rows_split(const b200gptq_attn_args& a);
int attn_rows_dispatch(const b200gptq_attn_args& a, float* part, const AttnSplit& s, cudaStream_t stream);

}  // namespace b200gptq
