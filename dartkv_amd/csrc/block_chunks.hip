// Attention of long chunks of new tokens over e4m3 blocks: the tile kernel of dkv_prompt_tile.h with its keys and
// values converted into LDS, for the requests that block_attention.hip leaves.
#include "dkv_block_attention.h"
#include "dkv_capi_util.h"

namespace dkv {

namespace {

struct Plan {
  int waves, splits;
  int64_t grid;  // workgroups of one part
};

Plan plan_of(const PromptParams& p, int64_t rows_bound, bool bf16) {
  auto grid_of = [&](int64_t rows) { return ((rows_bound + rows - 1) / rows + p.R) * p.H; };
  Plan plan;
  plan.waves = bf16 && p.D > 64 && p.D <= 128 && grid_of(256) >= 256 ? 8 : 4;
  plan.grid = grid_of(32 * plan.waves);
  const int DP = p.D <= 64 ? 64 : p.D <= 128 ? 128 : 256;
  plan.splits = prompt::splits_for(plan.grid, (int64_t)p.max_blocks << p.bs_shift, prompt::keys_of(DP, !bf16));
  return plan;
}

template <int DP, bool BF, int WAVES>
void launch(const PromptParams& p, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((prompt::prompt_tiles<DP, BF, WAVES, true>), dim3((unsigned)(grid * p.splits)), dim3(64 * WAVES),
                     prompt::lds_bytes(DP, !BF), stream, p);
  if (p.splits > 1)
    hipLaunchKernelGGL((prompt::prompt_merge<32 * WAVES, prompt::keys_of(DP, !BF), BF, true>),
                       dim3((unsigned)(grid * WAVES)), dim3(256), 0, stream, p);
}

template <bool BF>
void launch_dim(const PromptParams& p, const Plan& plan, hipStream_t stream) {
  if (p.D <= 64)
    launch<64, BF, 4>(p, plan.grid, stream);
  else if (p.D > 128)
    launch<256, BF, 4>(p, plan.grid, stream);
  else if constexpr (BF)
    plan.waves == 8 ? launch<128, BF, 8>(p, plan.grid, stream) : launch<128, BF, 4>(p, plan.grid, stream);
  else
    launch<128, BF, 4>(p, plan.grid, stream);
}

}  // namespace

int64_t block_chunks_workspace_bytes(const PromptParams& p, int64_t rows_bound, bool bf16) {
  const Plan plan = plan_of(p, rows_bound, bf16);
  return prompt::record_bytes(plan.grid, plan.splits, 32 * plan.waves, p.D);
}

int launch_block_chunks(PromptParams p, int64_t rows_bound, bool bf16, void* workspace, void* stream) {
  const Plan plan = plan_of(p, rows_bound, bf16);
  DKV_CHECK(plan.grid * 16 < (1ll << 31), DKV_ERR_INVALID, "dkv_block_attention: too many tokens");
  p.splits = plan.splits;
  p.records = (float*)workspace;
  p.stats = p.records + plan.grid * plan.splits * 32 * plan.waves * p.D;
  bf16 ? launch_dim<true>(p, plan, (hipStream_t)stream) : launch_dim<false>(p, plan, (hipStream_t)stream);
  return dkv_check_launch("dkv_block_attention");
}

}  // namespace dkv
