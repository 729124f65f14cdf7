// Grids past what one launch carries.
#pragma once
#include <cstdint>

namespace fdm {

// A launch holds fewer than 2^32 threads.  launch(first, count) is called for `blocks` blocks of `threads` threads, in order, in as few pieces as that allows
// (one, in all but huge calls); `first` is a multiple of 8, so that a block keeps its XCD.  Ends with the first result that is not 0, and returns it.
template <typename F>
int launch_pieces(int64_t blocks, int threads, F&& launch) {
  const int64_t most = ((int64_t)0xffffffff / threads) & ~(int64_t)7;
  for (int64_t first = 0; first < blocks; first += most) {
    const int rc = launch(first, (unsigned)(blocks - first < most ? blocks - first : most));
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace fdm
