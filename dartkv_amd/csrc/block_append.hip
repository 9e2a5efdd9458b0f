// New keys and values into the e4m3 blocks of a block cache (dkv_append_blocks), and the same for keys that are normed
// and turned on their way, with their queries (dkv_append_rotated_blocks).
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
//
// Keys that are normed and turned are so in those registers, before the scale.  43,000 tokens of 32 + 8 + 8 heads of 128:
// 234 us, 150 of them the queries' launch at a copy's rate; the append's part waits for its angles at three waves a SIMD.
// 64 single tokens with their queries: 6.8 us in one launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_capi_util.h"
#include "dkv_rotate.h"

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
  uint32_t groups;  // workgroups of the launch
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
  __device__ __forceinline__ void set(const float (&x)[8]) {
    Words<SRC, 8> words;
    words.set(x);
#pragma unroll
    for (int i = 0; i < 4 * kWords; ++i) w[i / 4][i % 4] = words.w[i];
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

enum Turn { kStays, kHalves, kNeighbours };  // which channels of a key turn with each other

// Keys of a pass, as they go into the blocks: normed, turned by their tokens' angles and rounded to their type, as
// rotate_heads gives them.  A lane has eight channels of its row, whose sums go over `lanes` lanes (a power of two; those
// behind head_dim hold zeros); the partners of halves are in a lane of their own.
template <int SRC, Turn TURN>
struct KeyTurner {
  const RotateParams& r;
  int lane, lanes, ch;
  bool turns, second;
  float w[8];

  __device__ __forceinline__ KeyTurner(const RotateParams* rotation, int lane, int lanes, int ch)
      : r(*rotation), lane(lane), lanes(lanes), ch(ch) {
    turns = ch < 2 * r.half, second = TURN == kHalves && ch >= r.half;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f;
    if (r.side[1].w && ch < r.D) load_any<8>(r.side[1].w, ch, r.w_dtype, w);
  }
  struct Angles {
    float c[TURN == kNeighbours ? 4 : 8], s[TURN == kNeighbours ? 4 : 8];
    bool none;
  };
  // Token t's angles, where `real` says that it is one.
  __device__ __forceinline__ Angles angles(int64_t t, bool real) const {
    Angles x;
    const int64_t at = real ? angles_at(r, (uint32_t)t) : kNoToken;
    x.none = at == kNoToken;
#pragma unroll
    for (float& c : x.c) c = 1.f;
#pragma unroll
    for (float& s : x.s) s = 0.f;
    if (turns) load_angles(r, at, TURN == kNeighbours ? ch / 2 : second ? ch - r.half : ch, x.c, x.s);
    return x;
  }
  __device__ __forceinline__ void turn(Raw<SRC>& raw, const Angles& angle) const {
    float x[8];
    raw.get(x);
    const float f = r.side[1].w ? norm_factor(row_sum(sum_of_squares(x), lanes), r.inv_d, r.eps) : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = angle.none ? 0.f : x[i] * (f * w[i]);
    if constexpr (TURN == kNeighbours) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float a = x[i], b = x[i + 1], c = angle.c[i / 2], s = angle.s[i / 2];
        x[i] = fmaf(a, c, -(b * s)), x[i + 1] = fmaf(b, c, a * s);
      }
    } else {
      const int partner = turns ? (second ? lane - r.half / 8 : lane + r.half / 8) : lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __shfl(x[i], partner, 64);
        if (turns) x[i] = fmaf(x[i], angle.c[i], second ? y * angle.s[i] : -(y * angle.s[i]));
      }
    }
    raw.set(x);
  }
  // The row of token t.
  __device__ __forceinline__ void turn(Raw<SRC>& raw, int64_t t, bool real) const { turn(raw, angles(t, real)); }
  // The rows of several passes (token t + i * rpp, `row` of `n` tokens).  (The angles of two passes at once: 252 us in place
  // of 234 for 43,000 tokens, as the registers then leave two waves a SIMD.)
  template <int N>
  __device__ __forceinline__ void turn_all(Raw<SRC> (&raw)[N], int64_t t, int row, int rpp, int n, bool active) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * rpp < n) turn(raw[i], t + i * rpp + row, active && i * rpp + row < n);
  }
};

template <int SRC>
struct KeyTurner<SRC, kStays> {
  __device__ __forceinline__ KeyTurner(const RotateParams*, int, int, int) {}
  __device__ __forceinline__ void turn(Raw<SRC>&, int64_t, bool) const {}
  template <int N>
  __device__ __forceinline__ void turn_all(Raw<SRC> (&)[N], int64_t, int, int, int, bool) const {}
};

// Wave `unit`'s runs.
template <int SRC, Turn TURN>
__device__ __forceinline__ void append_runs(const AppendParams& p, const RotateParams* rotation, int64_t unit) {
  const int lane = threadIdx.x & 63;
  const int kinds = 2 * p.H;
  const int64_t first = unit / kinds * p.span;
  if (first >= p.T) return;
  const int kind = (int)(unit % kinds), which = kind & 1, h = kind >> 1;
  const int bs = 1 << p.shift;
  const int lpr = TURN == kStays ? p.D >> 3 : rotation->lanes * 2, rpp = 64 / lpr;  // lanes of a row, rows of a pass
  const int my_row = lane / lpr, my_ch = (lane % lpr) * 8;
  const bool active = my_row < rpp && (TURN == kStays || my_ch < p.D);
  const void* src = p.src[which];
  constexpr int kSize = SRC == kF32 ? 4 : 2;
  const bool turned = TURN != kStays && which == 0;
  const KeyTurner<SRC, TURN> turner(rotation, lane, lpr, my_ch);
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
    if (turned) turner.turn_all(raw, t, my_row, rpp, n, active);
#pragma unroll
    for (int i = 0; i < kHeld<SRC>; ++i) {
      raw[i].largest(top);
      raw[i].forget();
    }
    for (int row = kHeld<SRC> * rpp; row < n; row += rpp) {
      const int r = row + my_row;
      Raw<SRC> more;
      more.zero();
      if (active && r < n) more.load(base + (int64_t)row * p.st[which] * kSize + my_at);
      if (turned) turner.turn(more, t + r, active && r < n);
      more.largest(top);
    }
    float amax = magnitude<SRC>(top);
    if (__any(!(amax < __builtin_inff()))) {  // the largest of the finite ones
      amax = 0.f;
      if (p.nonfinite && lane == 0) *p.nonfinite = 1;
#pragma unroll 1
      for (int row = 0; row < n; row += rpp) {
        const int r = row + my_row;
        float x[8];
        Raw<SRC> again;
        again.zero();
        if (active && r < n) again.load(base + (int64_t)row * p.st[which] * kSize + my_at);
        if (turned) turner.turn(again, t + r, active && r < n);
        again.get(x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (fabsf(x[i]) < __builtin_inff()) amax = fmaxf(amax, fabsf(x[i]));
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
      float x[8];
      Raw<SRC> more;
      more.zero();
      if (active && r < n) more.load(base + (int64_t)row * p.st[which] * kSize + my_at);
      if (turned) turner.turn(more, t + r, active && r < n);
      more.get(x);
      if (active && r < n) *(uint2*)(codes + row * p.D + my_code) = codes8(x, inv);
    }
    if (lane == 0 && (held == 0 || now != before)) *scale = now;
  }
}

template <int SRC>
__global__ void __launch_bounds__(kThreads) block_append(AppendParams p) {
  append_runs<SRC, kStays>(p, nullptr, (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

// The workgroups of the append, then those of the queries' rows.
template <int SRC, Turn TURN>
__global__ void __launch_bounds__(kThreads) block_append_rotated(AppendParams p, RotateParams r) {
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x < p.groups)
    append_runs<SRC, TURN>(p, &r, (int64_t)blockIdx.x * (kThreads / 64) + wave);
  else
    rotate_rows<SRC, 8, TURN == kNeighbours, 1, 1>(r, r.side[0], (blockIdx.x - p.groups) * (kThreads / 64) + wave);
}

int append_params(const dkv_append_blocks_args& a, const char* where, AppendParams& p) {
  DKV_CHECK(a.dtype == kF32 || a.dtype == kF16 || a.dtype == kBF16, DKV_ERR_DTYPE,
            "%s: keys and values must be bf16, fp16 or fp32", where);
  DKV_CHECK(a.H >= 1 && a.H < (1 << 20) && a.D >= 16 && a.D <= 512 && a.D % 16 == 0, DKV_ERR_INVALID,
            "%s: head_dim must be a multiple of 16 up to 512", where);
  DKV_CHECK(a.block_size >= 16 && a.block_size <= 256 && (a.block_size & (a.block_size - 1)) == 0, DKV_ERR_INVALID,
            "%s: block_size must be 16, 32, 64, 128 or 256", where);
  DKV_CHECK(a.tokens >= 0 && a.blocks >= 1, DKV_ERR_INVALID, "%s: bad counts", where);
  p = {};
  if (a.tokens == 0) return DKV_OK;
  DKV_CHECK(a.keys && a.values && a.slots && a.key_codes && a.value_codes && a.key_scale && a.value_scale,
            DKV_ERR_INVALID, "%s: NULL pointer", where);
  const int64_t esize = a.dtype == kF32 ? 4 : 2;
  DKV_CHECK((((uintptr_t)a.keys | (uintptr_t)a.values | (uintptr_t)(a.k_st * esize) | (uintptr_t)(a.k_sh * esize) |
              (uintptr_t)(a.v_st * esize) | (uintptr_t)(a.v_sh * esize) | (uintptr_t)a.key_codes |
              (uintptr_t)a.value_codes) & 15) == 0,
            DKV_ERR_INVALID, "%s: rows must be 16-byte aligned", where);
  DKV_CHECK(a.k_st >= 0 && a.v_st >= 0 && a.k_st < (1 << 23) && a.v_st < (1 << 23), DKV_ERR_INVALID,
            "%s: token strides must be under 2^23 elements", where);
  p = {{a.keys, a.values}, {a.k_st, a.v_st}, {a.k_sh, a.v_sh}, {a.key_codes, a.value_codes},
       {a.key_scale, a.value_scale}, a.slots, a.nonfinite, a.tokens, a.blocks,
       (int32_t)a.H, (int32_t)a.D, __builtin_ctzll((uint64_t)a.block_size), 1, (int32_t)a.dtype};
  // Few tokens: one wave for each of them; many: a wave looks through 64 for the runs that begin there.  16 x 5,354 tokens
  // of 8 heads: 103 us, a wave for each 424; 2,048 requests' single tokens: 31 us a wave for each, 112 through 64.  The
  // bound takes many tokens for prompts': single tokens of more requests than that, each a run, pay for it (4,096: 112
  // us, a wave for each 58).
  p.span = a.tokens * a.H <= 16384 ? 1 : 64;
  const int64_t units = (a.tokens + p.span - 1) / p.span * 2 * a.H;
  const int64_t grid = (units + kThreads / 64 - 1) / (kThreads / 64);
  DKV_CHECK(grid < kGridLimit, DKV_ERR_INVALID, "%s: too many tokens", where);
  p.groups = (uint32_t)grid;
  return DKV_OK;
}

template <int SRC>
void launch_rotated(const AppendParams& p, const RotateParams& r, bool next, hipStream_t stream) {
  const dim3 grid(p.groups + r.side[0].groups), block(kThreads);
  if (next)
    hipLaunchKernelGGL((block_append_rotated<SRC, kNeighbours>), grid, block, 0, stream, p, r);
  else
    hipLaunchKernelGGL((block_append_rotated<SRC, kHalves>), grid, block, 0, stream, p, r);
}

}  // namespace

extern "C" int dkv_append_blocks(const dkv_append_blocks_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_append_blocks: args is NULL");
  AppendParams p;
  const int rc = append_params(*args, "dkv_append_blocks", p);
  if (rc != DKV_OK || p.T == 0) return rc;
  const dim3 grid(p.groups);
  if (p.dtype == kF32)
    hipLaunchKernelGGL(block_append<kF32>, grid, dim3(kThreads), 0, (hipStream_t)stream, p);
  else if (p.dtype == kF16)
    hipLaunchKernelGGL(block_append<kF16>, grid, dim3(kThreads), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(block_append<kBF16>, grid, dim3(kThreads), 0, (hipStream_t)stream, p);
  return dkv_check_launch("dkv_append_blocks");
}

extern "C" int dkv_append_rotated_blocks(const dkv_append_blocks_args* args, const dkv_rotate_heads_args* rotation,
                                         void* stream) {
  const char* where = "dkv_append_rotated_blocks";
  DKV_CHECK(args != nullptr && rotation != nullptr, DKV_ERR_INVALID, "%s: args is NULL", where);
  const dkv_rotate_heads_args& a = *rotation;
  AppendParams p;
  int rc = append_params(*args, where, p);
  if (rc != DKV_OK) return rc;
  RotateParams r;
  rc = rotate_params(a, where, r);
  if (rc != DKV_OK) return rc;
  DKV_CHECK(a.batch == 1 && a.tokens == args->tokens && a.Hkv == args->H && a.D == args->D && a.dtype == args->dtype,
            DKV_ERR_INVALID, "%s: queries and keys must have the same tokens, head_dim and type", where);
  DKV_CHECK(a.half % 8 == 0, DKV_ERR_UNSUPPORTED, "%s: turned channels must be a multiple of 16", where);
  if (p.T == 0) return DKV_OK;
  DKV_CHECK(a.query && a.q_out && a.positions && (a.half == 0 || (a.cos && a.sin)), DKV_ERR_INVALID, "%s: NULL pointer",
            where);
  DKV_CHECK((int64_t)p.groups + r.side[0].groups < kGridLimit, DKV_ERR_INVALID, "%s: too many tokens", where);
  // Queries of many rows have a launch of their own: beside the append's 168 registers too few of them are in flight.
  if (r.steps > 1) {
    RotateParams queries = r;
    queries.side[1].groups = 0;
    launch_rotate_heads(queries, (int)a.dtype, 8, a.interleaved != 0, (hipStream_t)stream);
    r.side[0].groups = 0;
  }
  if (p.dtype == kF32)
    launch_rotated<kF32>(p, r, a.interleaved != 0, (hipStream_t)stream);
  else if (p.dtype == kF16)
    launch_rotated<kF16>(p, r, a.interleaved != 0, (hipStream_t)stream);
  else
    launch_rotated<kBF16>(p, r, a.interleaved != 0, (hipStream_t)stream);
  return dkv_check_launch(where);
}
