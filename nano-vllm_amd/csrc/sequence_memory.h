// sequence_memory.h -- what sequences remember, moved as a whole: blocks of a paged cache and states of slots, copied in every
// layer together: a launch takes six sets of arrays (a pool of keys and values is two), and as many pieces as a grid has room for.
#pragma once

#include <vector>

#include "nvllm_internal.h"

namespace nvllm {

// `count` arrays of slots, `stride` bytes apart: slot s of array i lies at base + i * stride + s * slot_bytes.
struct SlotArrays {
    void* base;
    size_t slot_bytes;
    size_t stride;
    int count;
};
// slot to[i] <- slot from[i] in every array, as if all were read before any is written.  0, or a refusal of include/nvllm.h
// (nothing is enqueued then).
int copy_slots(const std::vector<SlotArrays>& arrays, int n_slots, const int* from, const int* to, int n);

// ops_api.hip: the arrays of a pool's blocks; empty: not a pool of this library, or memory that a later manager has
std::vector<SlotArrays> pool_arrays(const KVCacheManager* mgr);
// sequence_memory.hip: one of a shared block's users lets go of it; false: it has one user only
bool drop_shared_block(const KVCacheManager* mgr, int block);
void forget_shared_blocks(const int* stack);   // the manager with this free stack is gone

// Is the library stream being captured?  (Entry points whose arguments are host arrays refuse that: a replay would read what the
// arrays' staging holds by then.)
bool stream_is_captured();

}  // namespace nvllm
