// Attention of long chunks of new tokens over e4m3 blocks: the tile kernel of dkv_prompt_tile.h with its keys and
// values converted into LDS, for the requests that block_attention.hip leaves.
#include "dkv_block_attention.h"
#include "dkv_capi_util.h"

namespace dkv {

namespace {

template <int DP, bool BF, int WAVES>
void launch(const PromptParams& p, int64_t rows_bound, hipStream_t stream) {
  const int64_t tiles = (rows_bound + 32 * WAVES - 1) / (32 * WAVES) + p.R;
  hipLaunchKernelGGL((prompt::prompt_tiles<DP, BF, WAVES, true>), dim3((unsigned)(tiles * p.H)), dim3(64 * WAVES),
                     prompt::lds_bytes(DP, !BF), stream, p);
}

template <bool BF>
void launch_dim(const PromptParams& p, int64_t rows_bound, hipStream_t stream) {
  if (p.D <= 64)
    launch<64, BF, 4>(p, rows_bound, stream);
  else if (p.D <= 128)
    launch<128, BF, 4>(p, rows_bound, stream);
  else
    launch<256, BF, 4>(p, rows_bound, stream);
}

}  // namespace

int launch_block_chunks(const PromptParams& p, int64_t rows_bound, bool bf16, void* stream) {
  DKV_CHECK((rows_bound / 128 + p.R + 1) * p.H < (1ll << 31), DKV_ERR_INVALID, "dkv_block_attention: too many tokens");
  bf16 ? launch_dim<true>(p, rows_bound, (hipStream_t)stream) : launch_dim<false>(p, rows_bound, (hipStream_t)stream);
  return dkv_check_launch("dkv_block_attention");
}

}  // namespace dkv
