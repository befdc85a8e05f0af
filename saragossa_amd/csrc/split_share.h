// How many splits may share a launch's pages, on the host and in a host test.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace skv {

// A kernel's share of its pages begins at split * pages / splits, in 32 bits: the most splits whose product with `pages`, or a tile's
// few pages more, has them. 256 up to 2^24 pages (2^28 rows), 63 of 2^26, the most that a layer has. (The product in 64 bits, or taken apart
// behind a branch that no shorter context takes, was 0.1 to 0.3 us of every launch.)
inline size_t most_splits(size_t pages) { return UINT32_MAX / (pages + 4096); }

} // namespace skv
