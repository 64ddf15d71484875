// The parts of b200gptq_attn_cache.
#pragma once

#include "attn.cuh"
#include "attn.h"

namespace b200gptq {

constexpr int kAttn4MaxSplit = 8;        // CTAs of a cluster
constexpr int kAttn4Warps = 8;           // of a CTA; each has scratch for two (sequence, key head, tile of rows) that it does a part of

// The queries, positions and sizes as b200gptq_attn has them (without caches), and the cache.
struct Attn4Args {
    b200gptq_attn_args attn;
    b200gptq_cache4 cache;
};
struct Attn4Divisors { Divisor row_tiles, kv_heads, group; };

// How a call is carried out.  read: the rows that are seen are read back into scratch and the tcgen05 kernel of b200gptq_attn takes them.  Otherwise the rows kernel, with
// 8 * tiles8 rows of Q per tile, with even runs of all keys for the warps of `ctas` CTAs (flat) or with 2^split_bits CTAs for each tile.
struct Attn4Plan { bool read, flat; int tiles8, split_bits, ctas; };

int attn4_rows_dispatch(const Attn4Args& a, float* part, const Attn4Plan& p, cudaStream_t stream);
// The rows of the cache that any query sees, into k, v [batch, kv_heads, rows, hd] (cache4.cu).  Where `rows` is less than the cache has, which a window allows, rows behind the sinks move
// up so that the last one that is seen is the last there is, and `pos` gets the positions of token 0 among them.
int attn4_read_back(const Attn4Args& a, void* k, void* v, int rows, int64_t* pos, cudaStream_t stream);

}  // namespace b200gptq
