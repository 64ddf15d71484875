// The parts of b200gptq_attn.
#pragma once

#include <cuda_runtime.h>

#include "../../../include/b200gptq.h"

namespace b200gptq {

// How a call is carried out.  tiles: one launch of the tcgen05 kernel.  Otherwise the rows kernel takes each sequence's own keys, with `own` CTAs of `warps`
// warps per tile of rows; the prefix is among them, or goes before in `parts` runs (sums in scratch), by the tcgen05 kernel (prefix_tiles) or by the rows kernel.
struct AttnPlan { bool tiles, prefix_tiles; int own, warps, parts; };

constexpr int kAttnMaxSplit = 8;         // CTAs of a cluster (rows kernel)
constexpr int kAttnMaxParts = 64;        // runs of a prefix
constexpr int kAttnTilesKeys = 64;       // keys of a unit (tcgen05 kernel)

bool attn_pdl_enabled();

int attn_rows_dispatch(const b200gptq_attn_args& a, float* part, const AttnPlan& p, cudaStream_t stream);
bool attn_tiles_maps(const b200gptq_attn_args& a, bool prefix);
int attn_tiles_dispatch(const b200gptq_attn_args& a, cudaStream_t stream);
int attn_tiles_prefix(const b200gptq_attn_args& a, float* part, int parts, cudaStream_t stream);

}  // namespace b200gptq
