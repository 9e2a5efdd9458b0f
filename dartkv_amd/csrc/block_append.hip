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
// One wave has one run (the tokens of a call that follow each other in one block) of one KV head's keys or values: it
// finds the runs that begin among its 64 tokens (one, where there are few) from the slots alone.  A block's rows are
// read once, all at once (64 registers for 64 rows of 128 in 16 bits), and stay there until the scale is known.
// Bound: memory, 3 bytes an element from 16 bits.  86,000 tokens of 8 KV heads of 128 in bf16: 102 us, 5.2 TB/s (242 us
// with two passes over the rows, one load at a time); 64 tokens, one for each of 64 blocks: 4.4 us.
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

// Rows of a run that stay in registers between the scale and the codes: all 64 of a block for head_dim 128 in 16 bits.
template <int SRC>
constexpr int kHeld = SRC == kF32 ? 8 : 16;  // passes of 64 / (D / 8) rows

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));

template <int SRC>
struct Raw {  // eight elements as they are
  static constexpr int kWords = SRC == kF32 ? 2 : 1;
  u32x4 w[kWords];
  __device__ __forceinline__ void load(const char* at) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = ((const u32x4*)at)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = (u32x4){0, 0, 0, 0};
  }
  // `top`: the largest magnitude's bits so far (magnitudes order as their bits do, infinities and NaN above all; two
  // maxima of 16 bits each).
  __device__ __forceinline__ void largest(uint32_t& top) const {
#pragma unroll
    for (int i = 0; i < 4 * kWords; ++i) {
      const uint32_t u = w[i / 4][i % 4];
      if constexpr (SRC == kF32) {
        top = (u & 0x7fffffffu) > top ? u & 0x7fffffffu : top;
      } else {
        top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, top),
                                                                     __builtin_bit_cast(ushort2v, u & 0x7fff7fffu)));
      }
    }
  }
  // The registers hold something unknown from here: what was made of them is not kept.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (SRC == kF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = u2f(w[i / 4][i % 4]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = w[0][i];
        if constexpr (SRC == kBF16) {
          x[2 * i] = u2f(u << 16), x[2 * i + 1] = u2f(u & 0xffff0000u);
        } else {
          x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)u);
          x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
        }
      }
    }
  }
};

// The magnitude that `largest` found.
template <int SRC>
__device__ __forceinline__ float magnitude(uint32_t top) {
  if constexpr (SRC == kF32) return u2f(top);
  const uint32_t u = (top & 0xffffu) > (top >> 16) ? top & 0xffffu : top >> 16;
  if constexpr (SRC == kBF16) return u2f(u << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}

template <int SRC>
__global__ void __launch_bounds__(kThreads) block_append(AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kinds = 2 * p.H;
  const int64_t first = unit / kinds * p.span;
  if (first >= p.T) return;
  const int kind = (int)(unit % kinds), which = kind & 1, h = kind >> 1;
  const int bs = 1 << p.shift;
  const int lpr = p.D >> 3, rpp = 64 / lpr;  // lanes of a row, rows of a pass
  const int my_row = lane / lpr, my_ch = (lane % lpr) * 8;
  const bool active = my_row < rpp;
  const void* src = p.src[which];
  constexpr int kSize = SRC == kF32 ? 4 : 2;
  const uint32_t my_at = (uint32_t)((my_row * p.st[which] + my_ch) * kSize), my_code = my_row * p.D + my_ch;

  // the runs that begin among this wave's tokens
  const int64_t mine = first + lane;
  const int64_t slot = mine < p.T ? p.slots[mine] : -1, prev = mine > 0 && mine < p.T ? p.slots[mine - 1] : -1;
  const bool in = slot >= 0 && (slot >> p.shift) < p.blocks;
  const bool goes_on = prev >= 0 && prev + 1 == slot && (slot & (bs - 1)) != 0;
  uint64_t runs = __ballot(lane < p.span && in && !goes_on);

  while (runs) {
    const int l = __builtin_ctzll(runs);
    runs &= runs - 1;
    const int64_t t = first + l;
    const int64_t begin = ((int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(slot >> 32), l) << 32) |
                          (uint32_t)__builtin_amdgcn_readlane((int)slot, l);
    const int64_t block = begin >> p.shift;
    const int held = (int)(begin & (bs - 1));
    const int most = bs - held;  // tokens of the run, found from the slots that follow each other
    int n = 1;
    while (n < most) {
      const int64_t at = t + n + lane;
      const bool same = n + lane < most && at < p.T && p.slots[at] == begin + n + lane;
      const uint64_t others = ~__ballot(same);
      const int more = others ? __builtin_ctzll(others) : 64;
      n += more;
      if (more < 64) break;
    }
    // rows of a pass: a wave-uniform address and this lane's offset
    const char* base = (const char*)src + (t * p.st[which] + h * p.sh[which]) * kSize;
    const int64_t pass = rpp * p.st[which] * kSize;
    float* scale = p.scale[which] + block * p.H + h;
    const float before = held > 0 ? *scale : 0.f;
    Raw<SRC> raw[kHeld<SRC>];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kHeld<SRC>; ++i) {
      const int r = i * rpp + my_row;
      raw[i].zero();
      if (active && r < n) raw[i].load(base + i * pass + my_at);
    }
#pragma unroll
    for (int i = 0; i < kHeld<SRC>; ++i) {
      raw[i].largest(top);
      raw[i].forget();
    }
    for (int row = kHeld<SRC> * rpp; row < n; row += rpp) {
      const int r = row + my_row;
      if (active && r < n) {
        Raw<SRC> more;
        more.load(base + (int64_t)row * p.st[which] * kSize + my_at);
        more.largest(top);
      }
    }
    float amax = magnitude<SRC>(top);
    if (__any(!(amax < __builtin_inff()))) {  // the largest of the finite ones
      amax = 0.f;
      if (p.nonfinite && lane == 0) *p.nonfinite = 1;
#pragma unroll 1
      for (int row = 0; row < n; row += rpp) {
        const int r = row + my_row;
        if (active && r < n) {
          float x[8];
          Raw<SRC> again;
          again.load(base + (int64_t)row * p.st[which] * kSize + my_at);
          again.get(x);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (fabsf(x[i]) < __builtin_inff()) amax = fmaxf(amax, fabsf(x[i]));
        }
      }
    }
    amax = wave_max(amax);
    float now = pow2(amax > 0.f ? exponent_for(amax) : kMinExponent);
    if (held > 0) now = fmaxf(now, before);
    uint8_t* codes = p.codes[which] + (block * p.H + h) * (int64_t)bs * p.D;
    if (held > 0 && now != before) {  // the block's earlier codes at the new scale
      const float f = before / now;
      for (int row = 0; row < held; row += rpp) {
        const int r = row + my_row;
        if (active && r < held) {
          uint2* at = (uint2*)(codes + row * p.D + my_code);
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
    codes += (int64_t)held * p.D;
#pragma unroll
    for (int i = 0; i < kHeld<SRC>; ++i) {
      const int r = i * rpp + my_row;
      float x[8];
      raw[i].get(x);
      if (active && r < n) *(uint2*)(codes + i * rpp * p.D + my_code) = codes8(x, inv);
    }
    for (int row = kHeld<SRC> * rpp; row < n; row += rpp) {
      const int r = row + my_row;
      if (active && r < n) {
        float x[8];
        Raw<SRC> more;
        more.load(base + (int64_t)row * p.st[which] * kSize + my_at);
        more.get(x);
        *(uint2*)(codes + row * p.D + my_code) = codes8(x, inv);
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
  DKV_CHECK(a.k_st >= 0 && a.v_st >= 0 && a.k_st < (1 << 23) && a.v_st < (1 << 23), DKV_ERR_INVALID,
            "dkv_append_blocks: token strides must be under 2^23 elements");
  AppendParams p = {{a.keys, a.values}, {a.k_st, a.v_st}, {a.k_sh, a.v_sh}, {a.key_codes, a.value_codes},
                    {a.key_scale, a.value_scale}, a.slots, a.nonfinite, a.tokens, a.blocks,
                    (int32_t)a.H, (int32_t)a.D, __builtin_ctzll((uint64_t)a.block_size), 1, (int32_t)a.dtype};
  // Few tokens: one wave for each of them; many: a wave looks through 64 for the runs that begin there.  16 x 5,354 tokens
  // of 8 heads: 103 us, a wave for each 424; 2,048 requests' single tokens: 31 us a wave for each, 112 through 64.  The
  // bound takes many tokens for prompts': single tokens of more requests than that, each a run, pay for it (4,096: 112
  // us, a wave for each 58).
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
