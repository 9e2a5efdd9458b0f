// New keys and values into the e4m3 blocks of a block cache (dkv_append_blocks).
//
// A block of bs tokens of one KV head has one scale for its keys and one for its values, 2^e with e the least that
// brings the largest magnitude so far under e4m3's 448 (e in [-120, 121], -120 for a block of zeros).  A token's code is
// e4m3(x / 2^e), half to even: x / 2^e is exact, so each value is rounded once.  When new tokens raise e, the codes
// already in the block are multiplied by the exact power of two and rounded again; that only moves codes that become
// subnormal (a value of the block's largest over 2^14 or less), so a value is off by at most half a step at its own
// size or one step of the block's smallest.  With scales that are not powers of two every growth would round all
// codes again.
//
// One wave has one run (the tokens of a call that lie in one block, next to each other) of one KV head's keys or
// values: it finds the run from the slots alone.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_capi_util.h"
#include "dkv_device.h"

using namespace dkv;

namespace {

constexpr int kMinExponent = -120, kMaxExponent = 121;
constexpr int kThreads = 256;

typedef float f32x2 __attribute__((ext_vector_type(2)));

struct AppendParams {
  const void* src[2];  // keys, values
  int64_t st[2], sh[2];
  uint8_t* codes[2];
  float* scale[2];
  const int64_t* slots;
  uint32_t* nonfinite;
  int64_t T, blocks;
  int32_t H, D, shift, span, dtype;
};

// Eight elements at `at` (element index, a multiple of 8 elements from an aligned base).
template <int SRC>
__device__ __forceinline__ void load8(const void* src, int64_t at, float (&x)[8]) {
  if constexpr (SRC == kF32) {
    const float4 a = *(const float4*)((const float*)src + at), b = *(const float4*)((const float*)src + at + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 w = *(const uint4*)((const uint16_t*)src + at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (SRC == kBF16) {
        x[2 * i] = u2f(u[i] << 16), x[2 * i + 1] = u2f(u[i] & 0xffff0000u);
      } else {
        x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)u[i]);
        x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[i] >> 16));
      }
    }
  }
}

__device__ __forceinline__ int exponent_for(float amax) {
  int k;
  const float f = frexpf(amax, &k);  // amax = f 2^k, f in [1/2, 1); 448 = 7/8 2^9
  const int e = k - 9 + (f > 0.875f ? 1 : 0);
  return e < kMinExponent ? kMinExponent : e > kMaxExponent ? kMaxExponent : e;
}

__device__ __forceinline__ float pow2(int e) { return u2f((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int v = 0;
    v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, v, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, v, true);
    w[i] = (uint32_t)v;
  }
  return make_uint2(w[0], w[1]);
}

template <int SRC>
__global__ void __launch_bounds__(kThreads) block_append(AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kinds = 2 * p.H;
  const int64_t first = unit / kinds * p.span;
  if (first >= p.T) return;
  const int kind = (int)(unit % kinds), which = kind & 1, h = kind >> 1;
  const int64_t stop = first + p.span < p.T ? first + p.span : p.T;
  const int bs = 1 << p.shift;
  const int lpr = p.D >> 3, rpp = 64 / lpr;  // lanes of a row, rows of a pass
  const int my_row = lane / lpr, my_ch = (lane % lpr) * 8;
  const bool active = my_row < rpp;

  for (int64_t t = first; t < stop; ++t) {
    const int64_t slot = p.slots[t];
    if (slot < 0 || (slot >> p.shift) >= p.blocks) continue;
    const int64_t block = slot >> p.shift;
    if (t > 0 && p.slots[t - 1] >= 0 && (p.slots[t - 1] >> p.shift) == block) continue;  // inside a run
    int n = 0;  // tokens of the run
    while (n < bs) {
      const int64_t at = t + n + lane;
      const bool same = n + lane < bs && at < p.T && p.slots[at] >= 0 && (p.slots[at] >> p.shift) == block;
      const uint64_t mask = ~__ballot(same);
      const int more = mask ? __builtin_ctzll(mask) : 64;
      n += more;
      if (more < 64) break;
    }
    const int held = (int)(slot & (bs - 1));
    const void* src = p.src[which];
    const int64_t base = t * p.st[which] + h * p.sh[which] + my_ch;
    float amax = 0.f;
    bool bad = false;
    for (int row = 0; row < n; row += rpp) {
      const int r = row + my_row;
      if (active && r < n) {
        float x[8];
        load8<SRC>(src, base + r * p.st[which], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = fabsf(x[i]);
          if (a < __builtin_inff())
            amax = fmaxf(amax, a);
          else
            bad = true;
        }
      }
    }
    amax = wave_max(amax);
    if (p.nonfinite && __any(bad) && lane == 0) *p.nonfinite = 1;
    float* scale = p.scale[which] + block * p.H + h;
    const float before = *scale;
    float now = pow2(amax > 0.f ? exponent_for(amax) : kMinExponent);
    if (held > 0) now = fmaxf(now, before);
    uint8_t* codes = p.codes[which] + (block * p.H + h) * (int64_t)bs * p.D + my_ch;
    if (held > 0 && now != before) {  // the block's earlier codes at the new scale
      const float f = before / now;
      for (int row = 0; row < held; row += rpp) {
        const int r = row + my_row;
        if (active && r < held) {
          uint2* at = (uint2*)(codes + (int64_t)r * p.D);
          const uint2 w = *at;
          const uint32_t u[2] = {w.x, w.y};
          float x[8];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], false);
            const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], true);
            x[4 * i] = a[0], x[4 * i + 1] = a[1], x[4 * i + 2] = b[0], x[4 * i + 3] = b[1];
          }
          *at = codes8(x, f);
        }
      }
    }
    const float inv = 1.f / now;
    for (int row = 0; row < n; row += rpp) {
      const int r = row + my_row;
      if (active && r < n) {
        float x[8];
        load8<SRC>(src, base + r * p.st[which], x);
        const int at = (int)(p.slots[t + r] & (bs - 1));
        *(uint2*)(codes + (int64_t)at * p.D) = codes8(x, inv);
      }
    }
    if (lane == 0 && (held == 0 || now != before)) *scale = now;
  }
}

}  // namespace

extern "C" int dkv_append_blocks(const dkv_append_blocks_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_append_blocks: args is NULL");
  const dkv_append_blocks_args& a = *args;
  DKV_CHECK(a.dtype == kF32 || a.dtype == kF16 || a.dtype == kBF16, DKV_ERR_DTYPE,
            "dkv_append_blocks: keys and values must be bf16, fp16 or fp32");
  DKV_CHECK(a.H >= 1 && a.H < (1 << 20) && a.D >= 16 && a.D <= 512 && a.D % 16 == 0, DKV_ERR_INVALID,
            "dkv_append_blocks: head_dim must be a multiple of 16 up to 512");
  DKV_CHECK(a.block_size >= 16 && a.block_size <= 256 && (a.block_size & (a.block_size - 1)) == 0, DKV_ERR_INVALID,
            "dkv_append_blocks: block_size must be 16, 32, 64, 128 or 256");
  DKV_CHECK(a.tokens >= 0 && a.blocks >= 1, DKV_ERR_INVALID, "dkv_append_blocks: bad counts");
  if (a.tokens == 0) return DKV_OK;
  DKV_CHECK(a.keys && a.values && a.slots && a.key_codes && a.value_codes && a.key_scale && a.value_scale,
            DKV_ERR_INVALID, "dkv_append_blocks: NULL pointer");
  const int64_t esize = a.dtype == kF32 ? 4 : 2;
  DKV_CHECK((((uintptr_t)a.keys | (uintptr_t)a.values | (uintptr_t)(a.k_st * esize) | (uintptr_t)(a.k_sh * esize) |
              (uintptr_t)(a.v_st * esize) | (uintptr_t)(a.v_sh * esize) | (uintptr_t)a.key_codes |
              (uintptr_t)a.value_codes) & 15) == 0,
            DKV_ERR_INVALID, "dkv_append_blocks: rows must be 16-byte aligned");
  AppendParams p = {{a.keys, a.values}, {a.k_st, a.v_st}, {a.k_sh, a.v_sh}, {a.key_codes, a.value_codes},
                    {a.key_scale, a.value_scale}, a.slots, a.nonfinite, a.tokens, a.blocks,
                    (int32_t)a.H, (int32_t)a.D, __builtin_ctzll((uint64_t)a.block_size), 1, (int32_t)a.dtype};
  // few tokens: one wave for each of them; many: a wave looks through 64 for the runs that begin there
  p.span = a.tokens * a.H <= 16384 ? 1 : 64;
  const int64_t units = (a.tokens + p.span - 1) / p.span * 2 * a.H;
  const int64_t grid = (units + kThreads / 64 - 1) / (kThreads / 64);
  DKV_CHECK(grid < (1ll << 31), DKV_ERR_INVALID, "dkv_append_blocks: too many tokens");
  if (a.dtype == kF32)
    hipLaunchKernelGGL(block_append<kF32>, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, p);
  else if (a.dtype == kF16)
    hipLaunchKernelGGL(block_append<kF16>, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(block_append<kBF16>, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, p);
  return dkv_check_launch("dkv_append_blocks");
}
