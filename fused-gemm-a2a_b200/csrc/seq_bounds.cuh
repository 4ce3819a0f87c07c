// Boundaries of packed sequences. `cu` holds n + 1 offsets into the token axis (cu[0] is read as 0) that
// a user's program keeps in device memory; they are never read on the host, so every kernel clamps them
// to [0, tokens] and stays inside its tensors whatever they hold. Rows at and behind the last offset
// belong to no sequence. A null `cu` is one sequence of all rows.
#pragma once
#include <cstdint>

namespace fga {

__device__ __forceinline__ int seq_bound(const int* cu, int i, int n, int tokens) {
  if (i <= 0) return 0;
  if (cu == nullptr) return tokens;
  return min(max(__ldg(cu + min(i, n)), 0), tokens);
}

// The sequence that holds `row` (the last one that starts at or before it, so that empty sequences are
// skipped), or n when the row lies behind the last sequence.
__device__ __forceinline__ int seq_of_row(const int* cu, int n, int tokens, int row) {
  if (cu == nullptr) return 0;
  int lo = 0, hi = n;  // the answer is the largest i in [0, n] with bound(i) <= row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (seq_bound(cu, mid, n, tokens) <= row)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

}  // namespace fga
