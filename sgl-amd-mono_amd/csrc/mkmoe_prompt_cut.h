// How the attention of a prompt's tokens is cut (mkmoe_prompt.hip), and which of its two cuts a call takes.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/mkmoe.h"

namespace mkmoe_latent {

// The attention's cuts, by the waves of a workgroup, W = 4 or 8: 32 W query rows a query tile, 8 W cached tokens a
// turn, and as many equal shares of the work as two or one workgroups a CU
constexpr int kMaxShares = 512;
constexpr __host__ __device__ int shares_of(int waves) { return 2048 / waves; }
constexpr __host__ __device__ int rows_of(int waves) { return 32 * waves; }
constexpr __host__ __device__ int key_shift(int waves) { return waves == 8 ? 6 : 5; }
constexpr int kKeys = 64;           // a sequence's packed rows are a multiple of so many
// What starting and storing a query tile takes, in turns of keys (5, 8, 12: ragged prompts' step 183, 179, 179 us)
constexpr int kItemSetup = 8;

inline int64_t packed_rows(int32_t context) { return ((int64_t)context + kKeys - 1) & -(int64_t)kKeys; }

// 8 waves a workgroup read the keys and values half as often, 4 (two workgroups a CU) run one's start and end under the
// other's turns. So 4 for short prompts and chunks, unless the cached tokens may be many: by the mean query tokens of a
// sequence and what bounds its length, the table's width and its part of max_context, for the host does not know the lengths
// (4 and 8 waves, us a call, 16 to 64 heads: 193 tokens over 700 38 and 44; 512 and
// 2048 tokens alone 43 and 47, 100 and 100; 16 ragged prompts of up to 500 70 and 78, of up to 1000 209 and 224; 8 of up to 300
// over 3000 144 and 157; 4 of up to 1024 over 4096 293 and 294; 512 over 16384 185 and 179; 300 over 65000 615 and 592; 8191 alone
// 769 and 742). 0: neither cut counts the call's units of work in 32 bits (8 waves have a quarter as many)
inline int prompt_waves(const mkmoe_latent_prompt_io& io) {
  const int64_t cap = packed_rows(io.max_context), table = (int64_t)io.max_pages * io.cache.page_size;
  auto countable = [&](int waves) {
    const int64_t units = ((table < cap ? table : cap) >> key_shift(waves)) + 1 + kItemSetup;
    return ((int64_t)io.tokens / rows_of(waves) + io.seqs) * io.heads * units <= 0x3fffffff;
  };
  if (!countable(8)) return 0;
  const int64_t context = io.max_context / io.seqs;
  return countable(4) && io.tokens / io.seqs <= 2048 && (context < table ? context : table) <= 32768 ? 4 : 8;
}

}  // namespace mkmoe_latent
