// What the kernels of dkv_block_attention share.
#pragma once
#include <stdint.h>

#include "dkv_prompt_tile.h"

namespace dkv {

// The chunk kernel (blocks_chunk.hip): the requests of more than p.skip_rows query rows.
int launch_block_chunks(const PromptParams& p, int64_t rows_bound, bool bf16, void* stream);

}  // namespace dkv
