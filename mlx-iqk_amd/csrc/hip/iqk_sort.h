// Sorting pairs by a small key, for the calls that need it beside iqk_sort.
#ifndef IQK_SORT_H
#define IQK_SORT_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace iqk {

constexpr int64_t kSortMaxExperts = 1024;

// How pairs are sorted: by `blocks` workgroups of `share` pairs each; where a launch before
// counts the shares, into a workspace of `words`, 16-byte aligned.
struct SortPlan {
    int64_t blocks, share, words;
};
SortPlan sort_plan(int64_t pairs, int64_t experts);

// Pair p has the key ids[p / per_id], experts where that is outside [0, experts).
struct SortCall {
    const void *ids;
    bool wide;           // 64-bit ids
    int64_t pairs, experts, per_token, per_id;
    uint32_t *work;
    int32_t *offsets;    // [experts + 1]: the pairs of lower keys
    int32_t *sorted_ids; // [pairs] each slot's key, or null
    int32_t *tokens;     // [pairs] each slot's p / per_token
    int32_t *slots;      // [pairs] each pair's slot, or null
};
int sort_launch(const SortCall &c, hipStream_t stream);

}  // namespace iqk

#endif  // IQK_SORT_H
