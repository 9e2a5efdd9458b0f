// Attention over whole prompts (dkv_prompt_attention): the host's checks and choice of tile.
#include "dkv_capi_util.h"
#include "dkv_prompt_tile.h"

using namespace dkv;

namespace {

template <int DP, bool BF, int WAVES, int GROUPS, int KEYS = prompt::keys_of(DP, false)>
int launch(const PromptParams& p, int64_t grid, hipStream_t stream) {
  [[maybe_unused]] constexpr int keys = GROUPS * KEYS, rows = 32 * WAVES / GROUPS;
  hipLaunchKernelGGL((prompt::prompt_tiles<DP, BF, WAVES, false, GROUPS, KEYS>), dim3((unsigned)(grid * p.splits)),
                     dim3(64 * WAVES), prompt::lds_bytes(DP, KEYS, GROUPS), stream, p);
  if constexpr (KEYS == prompt::keys_of(DP, false)) {  // (pairs come in one part)
    if (p.splits > 1)
      hipLaunchKernelGGL((prompt::prompt_merge<rows, keys, BF, false>), dim3((unsigned)(grid * (rows / 32))), dim3(256),
                         0, stream, p);
  }
  return dkv_check_launch("dkv_prompt_attention");
}

struct Plan {
  int waves, groups, splits;
  bool pairs;    // workgroups of 64 rows, two on a CU
  int64_t grid;  // workgroups of one part
  int rows() const { return 32 * waves / groups; }
};

template <bool BF>
int launch_dim(const PromptParams& p, const Plan& plan, hipStream_t stream) {
  if (p.D > 128) return launch<256, BF, 4, 1>(p, plan.grid, stream);
  if (p.D <= 64)
    return plan.groups == 2 ? launch<64, BF, 8, 2>(p, plan.grid, stream) : launch<64, BF, 4, 1>(p, plan.grid, stream);
  if (plan.pairs) return launch<128, BF, 4, 2, 32>(p, plan.grid, stream);
  if (plan.groups == 2) return launch<128, BF, 8, 2>(p, plan.grid, stream);
  return plan.waves == 8 ? launch<128, BF, 8, 1>(p, plan.grid, stream) : launch<128, BF, 4, 1>(p, plan.grid, stream);
}

// Eight waves share each tile's copies in LDS for long sequences (one of 16,384 tokens: 1.99 ms, four waves 2.03); with
// shorter ones two workgroups of four on a CU hide each other's start and end (16 of 64 to 4,096: 920 us, eight waves
// 937; one of 6,464, six heads a KV head: 274 and 284).  head_dim 64 gains more from three waves a SIMD (fp16, six
// heads a KV head: 179 us, eight waves 207), and over 128 the accumulators leave one.  No more workgroups of 128 rows
// than CUs: eight waves in two groups (one of 1,024 tokens: 22.6 us, one group 25.2).  Of a causal triangle half of
// those workgroups end early: workgroups of 64 rows and tiles of 32 keys, two on a CU, a long one with a short one
// (20.4 us; one of 512 tokens 16.0 -> 13.5, one of 2,048 with 16 heads 35 -> 32).  Where the tiles are about equally
// long the larger ones are as good or better (1,024 tokens that all see all: 24.5, in pairs 27; 512 behind 7,680: 84 and
// 104).
Plan plan_of(const dkv_prompt_attention_args& a) {
  const int64_t G = a.Hq / a.Hkv;
  auto grid_of = [&](int64_t bm) {
    if (!a.q_starts) return a.requests * ((a.q_tokens * G + bm - 1) / bm) * a.Hkv;
    return prompt::tiles_of(a.q_tokens * G, a.requests + (a.fill ? 1 : 0), bm) * a.Hkv;
  };
  Plan plan = {4, 1, 1, false, grid_of(128)};
  const bool triangle = a.causal && a.k_tokens <= 2 * a.q_tokens;
  if (triangle && a.D > 64 && a.D <= 128 && plan.grid >= 128 && plan.grid <= 256)
    return {4, 2, 1, true, grid_of(64)};
  if (a.D <= 128 && plan.grid <= 256)
    plan.waves = 8, plan.groups = 2;
  else if (a.D > 64 && a.D <= 128 && grid_of(256) >= 512 && (a.q_starts ? a.q_tokens / a.requests : a.q_tokens) >= 8192)
    plan.waves = 8, plan.grid = grid_of(256);
  plan.splits = prompt::splits_for(plan.grid, a.k_tokens, plan.groups * prompt::keys_of(a.D <= 128 ? 128 : 256, false),
                                   !a.q_starts || a.requests == 1, 10);
  return plan;
}

int check_prompt(const dkv_prompt_attention_args& a) {
  DKV_CHECK(a.dtype == kF16 || a.dtype == kBF16, DKV_ERR_DTYPE, "dkv_prompt_attention: tensors must be bf16 or fp16");
  DKV_CHECK(a.Hkv >= 1 && a.Hq >= a.Hkv && a.Hq % a.Hkv == 0 && a.Hq < (1 << 20), DKV_ERR_INVALID,
            "dkv_prompt_attention: query heads must be divisible by KV heads");
  DKV_CHECK(a.D >= 8 && a.D <= 256 && a.D % 8 == 0, DKV_ERR_INVALID,
            "dkv_prompt_attention: head_dim must be a multiple of 8 up to 256");
  DKV_CHECK(a.requests >= 1 && a.requests < (1 << 24) && a.q_tokens >= 0 && a.k_tokens >= 0, DKV_ERR_INVALID,
            "dkv_prompt_attention: bad counts");
  const int64_t G = a.Hq / a.Hkv;
  DKV_CHECK(a.q_tokens < (1ll << 31) / G - 1024 && a.k_tokens < (1ll << 31) - 1024, DKV_ERR_INVALID,
            "dkv_prompt_attention: too many tokens");
  return DKV_OK;
}

}  // namespace

extern "C" int64_t dkv_prompt_attention_workspace_bytes(const dkv_prompt_attention_args* args) {
  if (!args || check_prompt(*args) != DKV_OK) return 0;
  const Plan plan = plan_of(*args);
  return prompt::record_bytes(plan.grid, plan.splits, plan.rows(), args->D);
}

extern "C" int dkv_prompt_attention(const dkv_prompt_attention_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_prompt_attention: args is NULL");
  const dkv_prompt_attention_args& a = *args;
  const int rc = check_prompt(a);
  if (rc != DKV_OK) return rc;
  DKV_CHECK((a.q_starts == nullptr) == (a.k_starts == nullptr), DKV_ERR_INVALID,
            "dkv_prompt_attention: query and key starts come together");
  // (the fp32 factor must not be 0: a hidden key's logit would be -inf * 0)
  DKV_CHECK(a.scale >= 1e-37 && a.scale < 1e30, DKV_ERR_INVALID, "dkv_prompt_attention: scale must be in 1e-37 to 1e30");
  if (a.q_tokens == 0) return DKV_OK;
  DKV_CHECK(a.query && a.out && (a.k_tokens == 0 || (a.keys && a.values)), DKV_ERR_INVALID,
            "dkv_prompt_attention: NULL pointer");
  DKV_CHECK((((uintptr_t)a.query | (uintptr_t)a.keys | (uintptr_t)a.values |
              (uintptr_t)(2 * (a.q_sb | a.q_st | a.q_sh | a.k_sb | a.k_st | a.k_sh | a.v_sb | a.v_st | a.v_sh))) & 15) ==
                    0 &&
                (((uintptr_t)a.out | (uintptr_t)(2 * (a.o_sb | a.o_st | a.o_sh))) & 7) == 0,
            DKV_ERR_INVALID, "dkv_prompt_attention: rows must be 16-byte aligned (output rows 8-byte)");
  // offsets within a stage of up to 128 keys are 31-bit
  DKV_CHECK(a.k_st >= 0 && a.v_st >= 0 && a.k_st < (1 << 23) && a.v_st < (1 << 23), DKV_ERR_INVALID,
            "dkv_prompt_attention: token strides of keys and values must be under 2^23 elements");
  PromptParams p = {};
  p.q = a.query, p.k = a.keys, p.v = a.values, p.o = a.out;
  p.q_sb = a.q_sb, p.q_st = a.q_st, p.q_sh = a.q_sh, p.k_sb = a.k_sb, p.k_st = a.k_st, p.k_sh = a.k_sh;
  p.v_sb = a.v_sb, p.v_st = a.v_st, p.v_sh = a.v_sh, p.o_sb = a.o_sb, p.o_st = a.o_st, p.o_sh = a.o_sh;
  p.q_starts = a.q_starts, p.k_starts = a.k_starts;
  p.R = (int32_t)a.requests, p.H = (int32_t)a.Hkv, p.G = (int32_t)(a.Hq / a.Hkv), p.D = (int32_t)a.D;
  p.q_tokens = a.q_tokens, p.k_tokens = a.k_tokens;
  p.c = (float)(a.scale * 1.4426950408889634);
  p.causal = a.causal ? 1 : 0, p.fill = a.fill && a.q_starts ? 1 : 0, p.skip_rows = 0;
  const Plan plan = plan_of(a);
  DKV_CHECK(plan.grid * 16 < (1ll << 31), DKV_ERR_INVALID, "dkv_prompt_attention: too many tokens");
  p.splits = plan.splits, p.pairs = plan.pairs ? 1 : 0;
  if (plan.splits > 1) {
    DKV_CHECK(a.workspace && ((uintptr_t)a.workspace & 15) == 0 &&
                  a.workspace_bytes >= prompt::record_bytes(plan.grid, plan.splits, plan.rows(), a.D),
              DKV_ERR_INVALID, "dkv_prompt_attention: workspace too small");
    p.records = (float*)a.workspace;
    p.stats = p.records + plan.grid * plan.splits * plan.rows() * a.D;
  }
  return a.dtype == kBF16 ? launch_dim<true>(p, plan, (hipStream_t)stream)
                          : launch_dim<false>(p, plan, (hipStream_t)stream);
}
