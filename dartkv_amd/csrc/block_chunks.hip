// Attention of long chunks of new tokens over e4m3 blocks: the tile kernel of dkv_prompt_tile.h with its keys and
// values converted into LDS, for the requests that block_attention.hip leaves.
#include "dkv_block_attention.h"
#include "dkv_capi_util.h"

namespace dkv {

namespace {

struct Plan {
  int waves, groups, splits;
  int64_t grid;  // workgroups of one part
  int rows() const { return 32 * waves / groups; }
};

// As for prompts; split weights (fp16, head_dim over 64) have the registers for four waves.
Plan plan_of(const PromptParams& p, int64_t rows_bound, bool bf16) {
  auto grid_of = [&](int64_t rows) { return prompt::tiles_of(rows_bound, p.R, rows) * p.H; };
  Plan plan = {4, 1, 1, grid_of(128)};
  if (p.D <= (bf16 ? 128 : 64) && plan.grid <= 256)
    plan.waves = 8, plan.groups = 2;
  else if (bf16 && p.D > 64 && p.D <= 128 && grid_of(256) >= 256)
    plan.waves = 8, plan.grid = grid_of(256);
  const int DP = p.D <= 64 ? 64 : p.D <= 128 ? 128 : 256;
  plan.splits = prompt::splits_for(plan.grid, (int64_t)p.max_blocks << p.bs_shift,
                                   plan.groups * prompt::keys_of(DP, !bf16), p.R == 1, 6);
  return plan;
}

template <int DP, bool BF, int WAVES, int GROUPS>
void launch(const PromptParams& p, int64_t grid, hipStream_t stream) {
  constexpr int keys = GROUPS * prompt::keys_of(DP, !BF), rows = 32 * WAVES / GROUPS;
  hipLaunchKernelGGL((prompt::prompt_tiles<DP, BF, WAVES, true, GROUPS>), dim3((unsigned)(grid * p.splits)),
                     dim3(64 * WAVES), prompt::lds_bytes(DP, prompt::keys_of(DP, !BF), GROUPS), stream, p);
  if (p.splits > 1)
    hipLaunchKernelGGL((prompt::prompt_merge<rows, keys, BF, true>), dim3((unsigned)(grid * (rows / 32))), dim3(256), 0,
                       stream, p);
}

template <bool BF>
void launch_dim(const PromptParams& p, const Plan& plan, hipStream_t stream) {
  if (p.D > 128)
    launch<256, BF, 4, 1>(p, plan.grid, stream);
  else if (p.D <= 64)
    plan.groups == 2 ? launch<64, BF, 8, 2>(p, plan.grid, stream) : launch<64, BF, 4, 1>(p, plan.grid, stream);
  else if constexpr (BF)
    plan.groups == 2  ? launch<128, BF, 8, 2>(p, plan.grid, stream)
    : plan.waves == 8 ? launch<128, BF, 8, 1>(p, plan.grid, stream)
                      : launch<128, BF, 4, 1>(p, plan.grid, stream);
  else
    launch<128, BF, 4, 1>(p, plan.grid, stream);
}

}  // namespace

int64_t block_chunks_workspace_bytes(const PromptParams& p, int64_t rows_bound, bool bf16) {
  const Plan plan = plan_of(p, rows_bound, bf16);
  return prompt::record_bytes(plan.grid, plan.splits, plan.rows(), p.D);
}

int launch_block_chunks(PromptParams p, int64_t rows_bound, bool bf16, void* workspace, void* stream) {
  const Plan plan = plan_of(p, rows_bound, bf16);
  DKV_CHECK(plan.grid * 16 < (1ll << 31), DKV_ERR_INVALID, "dkv_block_attention: too many tokens");
  p.splits = plan.splits;
  p.records = (float*)workspace;
  p.stats = p.records + plan.grid * plan.splits * plan.rows() * p.D;
  bf16 ? launch_dim<true>(p, plan, (hipStream_t)stream) : launch_dim<false>(p, plan, (hipStream_t)stream);
  return dkv_check_launch("dkv_block_attention");
}

}  // namespace dkv
