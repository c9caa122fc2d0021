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

constexpr int64_t kSortTile = 64;

// Pair p has the key ids[p / per_id], experts where that is outside [0, experts).  Its outputs are
// the lists of iqk_sort, or each key's pairs in tiles of their own.
struct SortCall {
    const void *ids;
    bool wide;            // 64-bit ids
    int64_t pairs, experts, per_token, per_id;
    uint32_t *work;
    int32_t *offsets, *sorted_ids, *tokens, *slots;
    void *tiles;          // null, or u32 [n_tiles][4]: key, -, pairs (0: none), -
    uint32_t *tile_pairs; // [n_tiles][kSortTile], those past a tile's pairs unwritten
    int64_t n_tiles;      // at least sort_tiles(pairs, experts)
};

// Tiles that any ids fill at most: every key may end in a part of one.
inline int64_t sort_tiles(int64_t pairs, int64_t experts) {
    const int64_t most = pairs / kSortTile + experts + 1;
    return most < pairs ? most : pairs;
}

int sort_launch(const SortCall &c, hipStream_t stream);

}  // namespace iqk

#endif  // IQK_SORT_H
