// A layer's keys and values in pages, as the kernels see it.
#pragma once

#include "page_table.cuh"

namespace psx {

struct PagedCacheView {
    PageTableView table;
    char *keys, *values;  // (num_pages, kv_heads, page_size, head_dim)
    int32_t kv_heads, head_dim;
};

}  // namespace psx
