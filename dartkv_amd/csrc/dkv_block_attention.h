// What the kernels of dkv_block_attention share.
#pragma once
#include <stdint.h>

#include "dkv_prompt_tile.h"

namespace dkv {

// The chunk kernel (block_chunks.hip): the requests of more than p.skip_rows query rows, of rows_bound rows in all.
int64_t block_chunks_workspace_bytes(const PromptParams& p, int64_t rows_bound, bool bf16);
int launch_block_chunks(PromptParams p, int64_t rows_bound, bool bf16, void* workspace, void* stream);

}  // namespace dkv
