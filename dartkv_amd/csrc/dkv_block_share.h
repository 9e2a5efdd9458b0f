// What block_tables.hip and block_share.hip share.
#pragma once
#include <hip/hip_runtime.h>

#include "dkv_capi_util.h"

namespace dkv {

constexpr int kMaxRequests = 8190;

// The checks of every call on a block cache's tables.
static inline int check_block_tables(const dkv_block_tables_args& a, const char* where) {
  DKV_CHECK(a.requests >= 1 && a.requests <= kMaxRequests, DKV_ERR_INVALID, "%s: requests must be in 1..%d", where,
            kMaxRequests);
  DKV_CHECK(a.block_size >= 16 && a.block_size <= 256 && (a.block_size & (a.block_size - 1)) == 0, DKV_ERR_INVALID,
            "%s: block_size must be 16, 32, 64, 128 or 256", where);
  DKV_CHECK(a.max_blocks >= 1 && a.max_blocks * a.block_size < (1ll << 31) && a.blocks >= 1 && a.blocks < (1ll << 31),
            DKV_ERR_INVALID, "%s: bad block counts", where);
  DKV_CHECK(a.table && a.lengths && a.free && a.state, DKV_ERR_INVALID, "%s: NULL pointer", where);
  return DKV_OK;
}

// dkv_release_blocks of a state with shares (block_share.hip).
int release_shared(const dkv_block_tables_args& args, hipStream_t stream);

}  // namespace dkv
