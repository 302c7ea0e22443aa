// What the plan, the CUDA-core kernel and the tensor-core kernel of the
// attention behind shared prefixes share.
//
// A plan is int32 words:
//   tokens [tokens][4]  prefix keys [p0, p1) and own keys [lo, hi) that the
//                       token sees, as places in the two slot arrays; lo and
//                       hi never decrease from token to token
//   items  [items][8]   PrefixItem: a run of tokens x a range of prefix keys
//                       and a range of own keys, one block per KV head
//   join   [n][4]       token, first entry, entries, 0: the tokens whose
//                       result is spread over several items (or none)
//   list   [entries]    per join token the places of its partial results
#pragma once

#include "common.cuh"

namespace cs {

constexpr int kPrefixTile = 128;  // query rows of a tile, and the plan's unit of keys

struct PrefixItem {
  int32_t tok0, ntok;
  int32_t a0, a1;  // prefix keys
  int32_t b0, b1;  // own keys
  int32_t part;    // first place of its partial results; -1: writes the output
  int32_t pad;
  int64_t steps() const {
    return ((int64_t)a1 - a0 + kPrefixTile - 1) / kPrefixTile +
           ((int64_t)b1 - b0 + kPrefixTile - 1) / kPrefixTile;
  }
};
static_assert(sizeof(PrefixItem) == 32, "plan words");

// the tensor-core kernel (prefix_sm100.cu); CS_ERR_UNSUPPORTED when the
// pool's layout does not fit its loads
int prefix_attn_sm100(const cs_prefix_params& p, const cs_prefix_plan_info& info,
                      const int32_t* plan, void* workspace, cudaStream_t stream);

}  // namespace cs
