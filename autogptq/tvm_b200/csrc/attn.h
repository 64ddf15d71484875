// The parts of b200gptq_attn.
#pragma once

#include <cuda_runtime.h>

#include "../../../include/b200gptq.h"

namespace b200gptq {

// How a call is carried out.  tiles: one launch of the tcgen05 kernel.  Otherwise the rows kernel takes each sequence's own keys in `own` runs, and the
// prefix goes before it in `parts` runs (sums in scratch), by the tcgen05 kernel (prefix_tiles) or by the rows kernel.
struct AttnPlan { bool tiles, prefix_tiles; int own, parts; };

constexpr int kAttnMaxSplit = 8, kAttnRowsKeys = 128, kAttnTilesKeys = 64;      // CTAs of a cluster, keys that all warps of a CTA take at once (rows kernel), keys per unit (tcgen05)

bool attn_pdl_enabled();

int attn_rows_dispatch(const b200gptq_attn_args& a, float* part, const AttnPlan& p, cudaStream_t stream);
bool attn_tiles_maps(const b200gptq_attn_args& a, bool prefix);
int attn_tiles_dispatch(const b200gptq_attn_args& a, cudaStream_t stream);
int attn_tiles_prefix(const b200gptq_attn_args& a, float* part, int parts, cudaStream_t stream);

}  // namespace b200gptq
