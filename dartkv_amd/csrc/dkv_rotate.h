// Norm and rotation of query and key heads: what rotate.hip and block_append.hip share (gfx950, wave64).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_capi_util.h"
#include "dkv_device.h"

namespace dkv {

// VEC elements of type DT next to each other, as they lie in memory.
template <int DT, int VEC>
struct Words {
  static constexpr int kBytes = VEC * (DT == kF32 ? 4 : 2);
  uint32_t w[kBytes < 4 ? 1 : kBytes / 4];

  __device__ __forceinline__ void load(const void* at) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        const uint4 u = ((const uint4*)at)[i];
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 u = *(const uint2*)at;
      w[0] = u.x, w[1] = u.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *(const uint32_t*)at;
    } else {
      w[0] = *(const uint16_t*)at;
    }
  }
  __device__ __forceinline__ void store(void* at) const {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        ((uint4*)at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (kBytes == 8) {
      *(uint2*)at = make_uint2(w[0], w[1]);
    } else if constexpr (kBytes == 4) {
      *(uint32_t*)at = w[0];
    } else {
      *(uint16_t*)at = (uint16_t)w[0];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t& u : w) u = 0;
  }
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (DT == kF32) {
        x[i] = u2f(w[i]);
      } else {
        const uint32_t u = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
        x[i] = DT == kBF16 ? u2f(u << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)u);
      }
    }
  }
  __device__ __forceinline__ void set(const float (&x)[VEC]) {
    zero();
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (DT == kF32) {
        w[i] = f2u(x[i]);
      } else {
        const uint16_t u = DT == kBF16 ? __builtin_bit_cast(uint16_t, (__bf16)x[i])
                                       : __builtin_bit_cast(uint16_t, (_Float16)x[i]);
        w[i / 2] |= (uint32_t)u << (i & 1 ? 16 : 0);
      }
    }
  }
};

template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* base, int64_t index, float (&x)[VEC]) {
  Words<DT, VEC> words;
  words.load((const char*)base + index * (DT == kF32 ? 4 : 2));
  words.get(x);
}

// The same of a type that is known at run time (one for the launch).
template <int VEC>
__device__ __forceinline__ void load_any(const void* base, int64_t index, int dt, float (&x)[VEC]) {
  if (dt == kBF16)
    load_vec<kBF16>(base, index, x);
  else if (dt == kF16)
    load_vec<kF16>(base, index, x);
  else
    load_vec<kF32>(base, index, x);
}

// The sum over the `lanes` (a power of two) lanes that share a row, in each of them.
__device__ __forceinline__ float row_sum(float v, int lanes) {
  for (int off = lanes >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// 1 / sqrt(mean(x^2) + eps), rounded about once more than each of its steps.
__device__ __forceinline__ float norm_factor(float squares, float inv_d, float eps) {
  return rsqrtf(fmaf(squares, inv_d, eps));
}

// (Of each VEC channels first, then their sums: halves of D = 8 * 2^k channels are added in the order of row_sum over
// lanes of eight, and a key comes out the same wherever it is normed.)
template <int VEC>
__device__ __forceinline__ float sum_of_squares(const float (&x)[VEC]) {
  float sum = x[0] * x[0];
#pragma unroll
  for (int i = 1; i < VEC; ++i) sum = fmaf(x[i], x[i], sum);
  return sum;
}

constexpr int kMaxRotateDim = 256;

// Of queries or keys.
struct RotateSide {
  const char *x, *g;
  char* out;
  const void* w;
  void* dw;
  float* sums;  // [groups][D]
  int64_t x_sb, x_st, x_sh, g_sb, g_st, g_sh, o_sb, o_st, o_sh;
  uint32_t H, rows, groups;
};

struct RotateParams {
  RotateSide side[2];
  const void *cos, *sin, *positions;
  int64_t c_sb, c_st, table_rows;
  uint32_t T;  // tokens of a batch
  int32_t D, half, lanes, rows_shift, wide, w_dtype, c_dtype, steps;
  float eps, inv_d;
};

template <int VEC, bool NEXT>
struct RotateUnit {
  int a, b, angle;
  bool any, both, turns;
  __device__ __forceinline__ RotateUnit(int u, int D, int half) {
    turns = u * VEC < half;
    angle = u * VEC;
    if (NEXT) {
      a = 2 * u * VEC, b = a + VEC;
    } else if (turns) {
      a = u * VEC, b = half + a;
    } else {
      a = 2 * u * VEC, b = a + VEC;  // 2 half + 2 (u - half / VEC) VEC
    }
    any = a < D, both = b < D;
  }
};

// Turns the pairs of a unit by the angles c, s (BACK: back).
template <int VEC, bool NEXT, bool BACK>
__device__ __forceinline__ void turn(float (&a)[VEC], float (&b)[VEC], const float (&c)[VEC], const float (&s)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float* p = NEXT ? (2 * i < VEC ? &a[2 * i] : &b[2 * i - VEC]) : &a[i];
    float* q = NEXT ? (2 * i + 1 < VEC ? &a[2 * i + 1] : &b[2 * i + 1 - VEC]) : &b[i];
    const float x = *p, y = *q, sin = BACK ? -s[i] : s[i];
    *p = fmaf(x, c[i], -(y * sin));
    *q = fmaf(y, c[i], x * sin);
  }
}

// Where token n's angles lie: kNoAngles for a position outside the table, kNoToken for a negative one.
constexpr int64_t kNoAngles = -1, kNoToken = -2;

__device__ __forceinline__ int64_t angles_at(const RotateParams& p, uint32_t n) {
  const int64_t position = p.wide ? ((const int64_t*)p.positions)[n] : ((const int32_t*)p.positions)[n];
  return position < 0 ? kNoToken : position < p.table_rows ? position * p.c_st : kNoAngles;
}

// A lane's row of a step: the token and head, and where its angles lie.
struct RotateRow {
  int64_t b, t, h, angles;
  bool real;
  __device__ __forceinline__ RotateRow(const RotateParams& p, const RotateSide& side, uint32_t row) {
    real = row < side.rows;
    const uint32_t at = real ? row : 0;
    const uint32_t n = at / side.H;
    h = at - n * side.H;
    b = p.T ? n / p.T : 0;
    t = p.T ? n - (uint32_t)b * p.T : n;
    angles = p.positions ? angles_at(p, n) : b * p.c_sb + t * p.c_st;
  }
};

template <int VEC>
__device__ __forceinline__ void load_angles(const RotateParams& p, int64_t angles, int at, float (&c)[VEC],
                                            float (&s)[VEC]) {
  if (angles >= 0) {
    load_any<VEC>(p.cos, angles + at, p.c_dtype, c);
    load_any<VEC>(p.sin, angles + at, p.c_dtype, s);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = s[i] = angles == kNoToken ? 0.f : __builtin_nanf("");
  }
}

// Wave `wave` of a side's rows: p.steps times 64 / p.lanes rows of them, N of those steps at once, so that N rows' loads
// are in flight; a step whose tokens are those of the one before has its angles already.  K: units of a lane, 64 apart.
template <int DT, int VEC, bool NEXT, int K, int N>
__device__ __forceinline__ void rotate_rows(const RotateParams& p, const RotateSide& side, uint32_t wave) {
  const int lane = threadIdx.x & 63, u = lane & (p.lanes - 1);
  constexpr int kSize = DT == kF32 ? 4 : 2;

  float wa[K][VEC], wb[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
#pragma unroll
    for (int i = 0; i < VEC; ++i) wa[k][i] = wb[k][i] = 1.f;
    if (side.w && unit.any) load_any<VEC>(side.w, unit.a, p.w_dtype, wa[k]);
    if (side.w && unit.both) load_any<VEC>(side.w, unit.b, p.w_dtype, wb[k]);
  }
  for (int step = 0; step < p.steps; step += N) {
    const uint32_t first = (wave * p.steps + step) << p.rows_shift;
    if (first >= side.rows) return;
    Words<DT, VEC> ra[N][K], rb[N][K];
    float c[N][K][VEC], s[N][K][VEC];
    int64_t angles[N];
    char* out[N];
    bool real[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const RotateRow row(p, side, first + (n << p.rows_shift) + (lane >> (6 - p.rows_shift)));
      const char* x = side.x + (row.b * side.x_sb + row.t * side.x_st + row.h * side.x_sh) * kSize;
      out[n] = side.out + (row.b * side.o_sb + row.t * side.o_st + row.h * side.o_sh) * kSize;
      angles[n] = row.angles, real[n] = row.real;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
        ra[n][k].zero(), rb[n][k].zero();
        if (unit.any) ra[n][k].load(x + unit.a * kSize);
        if (unit.both) rb[n][k].load(x + unit.b * kSize);
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (n == 0 || __any(angles[n] != angles[n - 1])) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
          if (unit.turns) load_angles<VEC>(p, angles[n], unit.angle, c[n][k], s[n][k]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) c[n][k][i] = c[n - 1][k][i], s[n][k][i] = s[n - 1][k][i];
        }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float a[K][VEC], b[K][VEC], squares = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        ra[n][k].get(a[k]), rb[n][k].get(b[k]);
        squares += sum_of_squares(a[k]) + sum_of_squares(b[k]);
      }
      const float r = side.w ? norm_factor(row_sum(squares, p.lanes), p.inv_d, p.eps) : 1.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[k][i] *= r * wa[k][i], b[k][i] *= r * wb[k][i];
        if (angles[n] == kNoToken) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) a[k][i] = b[k][i] = 0.f;
        }
        if (unit.turns) turn<VEC, NEXT, false>(a[k], b[k], c[n][k], s[n][k]);
        ra[n][k].set(a[k]), rb[n][k].set(b[k]);
        if (real[n] && unit.any) ra[n][k].store(out[n] + unit.a * kSize);
        if (real[n] && unit.both) rb[n][k].store(out[n] + unit.b * kSize);
      }
    }
  }
}

// Steps of a wave that are in flight together where there are many rows (32,768 tokens of 32 + 8 heads of 128 in bf16: one
// 155 us, two 149, four 201, whose registers leave two waves a SIMD).
constexpr int kRotateSteps = 2;

// How a row lies over lanes.  (32,768 tokens of 32 + 8 heads in bf16, forward: 128 channels in halves 133 us, 5.1 TB/s; 72
// in halves, so that 36 angles go two at a time, 200, 1.9 TB/s; 96 with 12 angles 215; 80 with 15, one at a time, 520.)
struct RotateShape {
  int vec, lanes, rows_shift;
};

static inline RotateShape rotate_shape(int64_t D, int64_t half) {
  RotateShape s;
  s.vec = half % 8 == 0 ? 8 : half % 2 == 0 ? 2 : 1;
  const int64_t units = (D / s.vec + 1) / 2;  // (at most 128: two a lane)
  s.lanes = 1;
  while (s.lanes < units && s.lanes < 64) s.lanes *= 2;
  s.rows_shift = __builtin_ctz(64 / s.lanes);
  return s;
}

static inline int check_rotate(const dkv_rotate_heads_args& a, const char* where) {
  DKV_CHECK(a.dtype == kF32 || a.dtype == kF16 || a.dtype == kBF16, DKV_ERR_DTYPE,
            "%s: queries and keys must be bf16, fp16 or fp32", where);
  DKV_CHECK((a.angle_dtype == kF32 || a.angle_dtype == kF16 || a.angle_dtype == kBF16) &&
                (a.weight_dtype == kF32 || a.weight_dtype == kF16 || a.weight_dtype == kBF16),
            DKV_ERR_DTYPE, "%s: weights, cos and sin must be bf16, fp16 or fp32", where);
  DKV_CHECK(a.D >= 8 && a.D <= kMaxRotateDim && a.D % 8 == 0, DKV_ERR_INVALID, "%s: head_dim must be a multiple of 8 up to %d",
            where, kMaxRotateDim);
  DKV_CHECK(a.half >= 0 && 2 * a.half <= a.D, DKV_ERR_INVALID, "%s: more turned channels than head_dim", where);
  DKV_CHECK(a.Hq >= 1 && a.Hkv >= 1 && a.batch >= 0 && a.tokens >= 0 && a.Hq < (1 << 20) && a.Hkv < (1 << 20),
            DKV_ERR_INVALID, "%s: bad counts", where);
  DKV_CHECK(a.batch < (1ll << 31) && a.tokens < (1ll << 31) &&
                a.batch * a.tokens < (1ll << 31) / (a.Hq > a.Hkv ? a.Hq : a.Hkv),
            DKV_ERR_INVALID, "%s: 2^31 rows or more", where);
  DKV_CHECK(a.eps >= 0 && a.eps < 1e30, DKV_ERR_INVALID, "%s: eps must not be negative", where);
  return DKV_OK;
}

constexpr int64_t kManyWaves = 16384;  // steps of a call from which on a wave makes several

// Workgroups (of four waves) and parameters of a forward pass; pointers are looked at for their alignment alone.
static inline int rotate_params(const dkv_rotate_heads_args& a, const char* where, RotateParams& p) {
  const int rc = check_rotate(a, where);
  if (rc != DKV_OK) return rc;
  const int64_t esize = a.dtype == kF32 ? 4 : 2;
  DKV_CHECK((((uintptr_t)a.query | (uintptr_t)a.keys | (uintptr_t)a.q_out | (uintptr_t)a.k_out | (uintptr_t)a.q_grad |
              (uintptr_t)a.k_grad | (uintptr_t)a.q_weight | (uintptr_t)a.k_weight |
              (uintptr_t)(esize * (a.q_sb | a.q_st | a.q_sh | a.k_sb | a.k_st | a.k_sh | a.qo_sb | a.qo_st | a.qo_sh |
                                   a.ko_sb | a.ko_st | a.ko_sh | a.qg_sb | a.qg_st | a.qg_sh | a.kg_sb | a.kg_st |
                                   a.kg_sh))) & 15) == 0,
            DKV_ERR_INVALID, "%s: rows and weights must be 16-byte aligned", where);
  const RotateShape s = rotate_shape(a.D, a.half);
  const int64_t csize = a.angle_dtype == kF32 ? 4 : 2, need = s.vec * csize > 16 ? 16 : s.vec * csize;
  DKV_CHECK(a.half == 0 || (((uintptr_t)a.cos | (uintptr_t)a.sin | (uintptr_t)(csize * (a.c_sb | a.c_st))) & (need - 1)) == 0,
            DKV_ERR_INVALID, "%s: rows of cos and sin must be aligned to %d bytes", where, (int)need);
  DKV_CHECK(!a.positions || a.table_rows >= 0, DKV_ERR_INVALID, "%s: bad table of angles", where);
  p = {};
  p.side[0] = {(const char*)a.query, (const char*)a.q_grad, (char*)a.q_out, a.q_weight, nullptr, nullptr,
               a.q_sb, a.q_st, a.q_sh, a.qg_sb, a.qg_st, a.qg_sh, a.qo_sb, a.qo_st, a.qo_sh, (uint32_t)a.Hq};
  p.side[1] = {(const char*)a.keys, (const char*)a.k_grad, (char*)a.k_out, a.k_weight, nullptr, nullptr,
               a.k_sb, a.k_st, a.k_sh, a.kg_sb, a.kg_st, a.kg_sh, a.ko_sb, a.ko_st, a.ko_sh, (uint32_t)a.Hkv};
  p.cos = a.cos, p.sin = a.sin, p.positions = a.positions;
  p.c_sb = a.c_sb, p.c_st = a.c_st, p.table_rows = a.table_rows, p.wide = a.wide_positions != 0;
  p.T = a.batch > 1 ? (uint32_t)a.tokens : 0;
  p.D = (int32_t)a.D, p.half = (int32_t)a.half, p.lanes = s.lanes, p.rows_shift = s.rows_shift;
  p.w_dtype = (int32_t)a.weight_dtype, p.c_dtype = (int32_t)a.angle_dtype;
  p.eps = (float)a.eps, p.inv_d = 1.f / (float)a.D;
  const int64_t rows = a.batch * a.tokens * (a.Hq + a.Hkv);
  p.steps = rows >> s.rows_shift < kManyWaves ? 1 : kRotateSteps;
  const int64_t per_group = (4ll * p.steps) << s.rows_shift;
  for (RotateSide& side : p.side) {
    side.rows = (uint32_t)(a.batch * a.tokens * side.H);
    side.groups = (uint32_t)((side.rows + per_group - 1) / per_group);
  }
  return DKV_OK;
}

// The forward pass of what `p` says (rotate.hip).
void launch_rotate_heads(const RotateParams& p, int dtype, int vec, bool next, hipStream_t stream);

}  // namespace dkv
