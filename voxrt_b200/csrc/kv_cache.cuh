// Argument checks shared by the cache's entry points.
#pragma once
#include "common.h"

namespace vxg {

vxg_status cache_check(const vxg_kv_cache* c);
// The host-side part of a batch: `a` (lengths or starts) and `cu` are device arrays, checked by the kernels.
vxg_status cache_batch_check(const vxg_kv_cache* c, const int* table, int n_seq, int max_pages, const int* a,
                             const int* cu, int total);

}  // namespace vxg
