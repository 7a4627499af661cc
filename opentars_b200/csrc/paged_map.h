// TMA maps of the paged cache's pools (host side).
#pragma once
#include <cuda.h>

#include "serve.h"

namespace tc {

// A 16-bit pool [pages][heads][slots][head dim] (strides of the cache, in any order) in boxes of 64
// elements x `rows` slots of one head and page, 128-byte swizzle; false when the driver has no encoder.
bool make_map_pool(CUtensorMap* m, const KvCache& c, const void* pool, int rows);

}  // namespace tc
