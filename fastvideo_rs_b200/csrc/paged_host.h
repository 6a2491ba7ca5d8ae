// Host checks shared by the entries over a paged K/V cache (paged_kv.cu).
#pragma once
#include "../../include/fv_sdpa.h"

namespace fvpg {
struct Pool;
struct Batch;
// Validates the cache and the batch and turns them into the kernels' form; FV_DECLINED without sequences or rows.
int check_paged(const char* what, const fv_paged_kv* kv, const fv_paged_batch* b, int rows, Pool* pool, Batch* batch, int* dev);
}  // namespace fvpg
