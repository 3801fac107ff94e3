// The stable counting sort of slots by key behind ascq_expert_sort; ascq_low_rank_add groups its rows by adapter with it.
#ifndef ASCQ_EXPERTS_CUH_
#define ASCQ_EXPERTS_CUH_

#include "ascq_internal.h"

namespace ascq {

constexpr int kMaxSortKeys = 1024;

// Enqueues the sort on `st`: counts[e] = slots with key e; rowOfSlot[s] = position of slot s, -1 for a slot without a key;
// slotOfRow[r] = slot at position r, -1 behind the last one.  A number outside [0, keys) is no key if `outside` is -1, else it
// counts as the key `outside`, and so does that number itself.  rowOfSlot or slotOfRow may be null.  The caller has checked
// 1 <= keys <= kMaxSortKeys and 0 < slots < 2^31.
ascq_status launch_key_sort(int64_t* counts, int32_t* rowOfSlot, int32_t* slotOfRow, const void* ids, bool ids64, int64_t slots, int keys, int outside,
                            ::CUstream_st* st);

}  // namespace ascq
#endif  // ASCQ_EXPERTS_CUH_
