// RMS norm of query and key heads and their rotation by the token's position, in one pass, and its gradients
// (dkv_rotate_heads, dkv_rotate_heads_backward).
//
// A head's row x of D channels becomes n = x r w with r = 1 / sqrt(mean(x^2) + eps), and the pairs (a, b) of its first
// 2 * half channels turn by their angle: a' = a c - b s, b' = b c + a s.  Backward, with g the gradient of the result:
// h = the pairs of g turned back (a: g_a c + g_b s, b: g_b c - g_a s), y = x r, dw = sum over rows of h y,
// dx = r (h w - y mean(h w y)).
//
// A lane holds one unit of a row: VEC channels and their VEC partners (behind the turned ones: the next VEC), so a
// pair is always in one lane and only the row's sums go through other lanes.  VEC is 8 (16-byte loads of 16-bit
// channels) where half and D allow it, else 2 or 1.  Everything is fp32 between the load and the one rounding at the end.
//
// Bound by memory: 32,768 tokens of 32 + 8 heads of 128 in bf16 148 us, 4.6 TB/s read and written as a copy; backward of
// 8,192 tokens 54 us (4.7 TB/s).  The weights' gradients are added in one order: by a lane over its rows, by lanes, waves,
// and the at most 1,024 workgroups' sums by a second launch with all of them in flight (4 us; 20 one load after another).
// One token: 3.5 us.  (3,001 tokens of 14 + 2 heads of 80 in fp16: forward 7, backward 15 us.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_capi_util.h"
#include "dkv_rotate.h"

using namespace dkv;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxDim = kMaxRotateDim;
constexpr int kMaxGroups = 1024;  // workgroups of a backward pass, each with its sums of the weights' gradients


template <int DT, int VEC, bool NEXT, int K, int N>
__global__ void __launch_bounds__(kThreads) rotate_heads(RotateParams p) {
  const bool keys = blockIdx.x >= p.side[0].groups;
  const uint32_t group = blockIdx.x - (keys ? p.side[0].groups : 0);
  rotate_rows<DT, VEC, NEXT, K, N>(p, p.side[keys], group * kWaves + (threadIdx.x >> 6));
}

template <int DT, int VEC, bool NEXT, int K>
__global__ void __launch_bounds__(kThreads) rotate_backward(RotateParams p) {
  const bool keys = blockIdx.x >= p.side[0].groups;
  const RotateSide& side = p.side[keys];
  const uint32_t group = blockIdx.x - (keys ? p.side[0].groups : 0);
  const int lane = threadIdx.x & 63, u = lane & (p.lanes - 1);
  const uint32_t wave = group * kWaves + (threadIdx.x >> 6);
  constexpr int kSize = DT == kF32 ? 4 : 2;

  float wa[K][VEC], wb[K][VEC], da[K][VEC], db[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
#pragma unroll
    for (int i = 0; i < VEC; ++i) wa[k][i] = wb[k][i] = 1.f, da[k][i] = db[k][i] = 0.f;
    if (side.w && unit.any) load_any<VEC>(side.w, unit.a, p.w_dtype, wa[k]);
    if (side.w && unit.both) load_any<VEC>(side.w, unit.b, p.w_dtype, wb[k]);
  }
  for (int step = 0; step < p.steps; ++step) {
    // (waves take turns, so that what they add up is spread over the tokens)
    const uint64_t first = ((uint64_t)step * side.groups * kWaves + wave) << p.rows_shift;
    if (first >= side.rows) break;
    const RotateRow row(p, side, (uint32_t)first + (lane >> (6 - p.rows_shift)));
    const char* x = side.x + (row.b * side.x_sb + row.t * side.x_st + row.h * side.x_sh) * kSize;
    const char* g = side.g + (row.b * side.g_sb + row.t * side.g_st + row.h * side.g_sh) * kSize;
    char* out = side.out + (row.b * side.o_sb + row.t * side.o_st + row.h * side.o_sh) * kSize;
    const bool given = row.real && row.angles != kNoToken;  // (else the row has no part in the result)
    Words<DT, VEC> ra[K], rb[K], ga[K], gb[K];
    float c[K][VEC], s[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
      ra[k].zero(), rb[k].zero(), ga[k].zero(), gb[k].zero();
      if (unit.any && given) ga[k].load(g + unit.a * kSize);
      if (unit.both && given) gb[k].load(g + unit.b * kSize);
      if (side.w && unit.any && given) ra[k].load(x + unit.a * kSize);
      if (side.w && unit.both && given) rb[k].load(x + unit.b * kSize);
      if (unit.turns) load_angles<VEC>(p, row.angles, unit.angle, c[k], s[k]);
    }
    float a[K][VEC], b[K][VEC], ha[K][VEC], hb[K][VEC], squares = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
      ra[k].get(a[k]), rb[k].get(b[k]), ga[k].get(ha[k]), gb[k].get(hb[k]);
      if (unit.turns && given) turn<VEC, NEXT, true>(ha[k], hb[k], c[k], s[k]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) squares = fmaf(a[k][i], a[k][i], fmaf(b[k][i], b[k][i], squares));
    }
    if (side.w) {
      const float sum = row_sum(squares, p.lanes), r = given ? norm_factor(sum, p.inv_d, p.eps) : 0.f;
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          a[k][i] *= r, b[k][i] *= r;
          da[k][i] = fmaf(ha[k][i], a[k][i], da[k][i]), db[k][i] = fmaf(hb[k][i], b[k][i], db[k][i]);
          ha[k][i] *= wa[k][i], hb[k][i] *= wb[k][i];
          dot = fmaf(ha[k][i], a[k][i], fmaf(hb[k][i], b[k][i], dot));
        }
      }
      const float mean = row_sum(dot, p.lanes) * p.inv_d;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          ha[k][i] = r * fmaf(-a[k][i], mean, ha[k][i]);
          hb[k][i] = r * fmaf(-b[k][i], mean, hb[k][i]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
      ga[k].set(ha[k]), gb[k].set(hb[k]);
      if (row.real && unit.any) ga[k].store(out + unit.a * kSize);
      if (row.real && unit.both) gb[k].store(out + unit.b * kSize);
    }
  }
  if (!side.dw) return;
  // the weights' gradients: over the wave's rows, then the waves, in a fixed order
  __shared__ float sums[kWaves][kMaxDim];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const RotateUnit<VEC, NEXT> unit(u + 64 * k, p.D, p.half);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      for (int off = p.lanes; off < 64; off <<= 1) {
        da[k][i] += __shfl_xor(da[k][i], off, 64);
        db[k][i] += __shfl_xor(db[k][i], off, 64);
      }
      if (lane < p.lanes && unit.any) sums[threadIdx.x >> 6][unit.a + i] = da[k][i];
      if (lane < p.lanes && unit.both) sums[threadIdx.x >> 6][unit.b + i] = db[k][i];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += kThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += sums[w][d];
    side.sums[(int64_t)group * p.D + d] = sum;
  }
}

// The workgroups' sums of the weights' gradients: 16 channels a workgroup, 64 threads each, whose loads are all in flight.
__global__ void __launch_bounds__(1024) rotate_weights(RotateParams p) {
  const RotateSide& side = p.side[blockIdx.y];
  const int column = threadIdx.x & 15, part = threadIdx.x >> 4, d = blockIdx.x * 16 + column;
  __shared__ float sums[64][17];
  float sum = 0.f;
  if (d < p.D && side.dw) {
    float x[kMaxGroups / 64];
#pragma unroll
    for (int i = 0; i < kMaxGroups / 64; ++i) {
      const uint32_t g = part + 64 * i;
      x[i] = g < side.groups ? side.sums[(int64_t)g * p.D + d] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kMaxGroups / 64; ++i) sum += x[i];
  }
  sums[part][column] = sum;
  __syncthreads();
  if (part == 0 && d < p.D && side.dw) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) sum += sums[i][column];
    dev_store(side.dw, d, sum, p.w_dtype);
  }
}

int64_t rows_of(const dkv_rotate_heads_args& a, int side) { return a.batch * a.tokens * (side ? a.Hkv : a.Hq); }

// Workgroups of a side in a backward pass: as many as the rows fill, at most kMaxGroups.
int64_t backward_groups(const dkv_rotate_heads_args& a, int side) {
  const RotateShape s = rotate_shape(a.D, a.half);
  const int64_t per_group = (int64_t)kWaves << s.rows_shift;
  const int64_t groups = (rows_of(a, side) + per_group - 1) / per_group;
  return groups > kMaxGroups ? kMaxGroups : groups;
}

template <int DT, int VEC, int K>
void launch_rotate(const RotateParams& p, bool next, bool backward, hipStream_t stream) {
  const dim3 grid(p.side[0].groups + p.side[1].groups), block(kThreads);
  if (backward) {
    if (next)
      hipLaunchKernelGGL((rotate_backward<DT, VEC, true, K>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((rotate_backward<DT, VEC, false, K>), grid, block, 0, stream, p);
  } else if (p.steps == 1) {
    if (next)
      hipLaunchKernelGGL((rotate_heads<DT, VEC, true, K, 1>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((rotate_heads<DT, VEC, false, K, 1>), grid, block, 0, stream, p);
  } else {
    constexpr int N = kRotateSteps;
    if (next)
      hipLaunchKernelGGL((rotate_heads<DT, VEC, true, K, N>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((rotate_heads<DT, VEC, false, K, N>), grid, block, 0, stream, p);
  }
}

template <int DT>
void launch_vec(const RotateParams& p, int vec, bool next, bool backward, hipStream_t stream) {
  if (vec == 8)
    launch_rotate<DT, 8, 1>(p, next, backward, stream);
  else if (vec == 2)
    launch_rotate<DT, 2, 1>(p, next, backward, stream);
  else
    launch_rotate<DT, 1, 2>(p, next, backward, stream);
}

int run_rotate(const dkv_rotate_heads_args& a, bool backward, const char* where, hipStream_t stream) {
  RotateParams p;
  const int rc = rotate_params(a, where, p);
  if (rc != DKV_OK) return rc;
  if (a.batch * a.tokens == 0) return DKV_OK;
  DKV_CHECK(a.query && a.keys && a.q_out && a.k_out && (a.half == 0 || (a.cos && a.sin)) &&
                (!backward || (a.q_grad && a.k_grad)),
            DKV_ERR_INVALID, "%s: NULL pointer", where);
  const RotateShape s = rotate_shape(a.D, a.half);
  DKV_CHECK(backward || (int64_t)p.side[0].groups + p.side[1].groups < kGridLimit, DKV_ERR_INVALID,
            "%s: more rows than a launch holds", where);
  if (backward) {
    p.steps = 1;
    for (int i = 0; i < 2; ++i) {
      p.side[i].groups = (uint32_t)backward_groups(a, i);
      const int64_t per_turn = (int64_t)p.side[i].groups * kWaves << s.rows_shift;
      const int32_t steps = (int32_t)((p.side[i].rows + per_turn - 1) / per_turn);
      p.steps = steps > p.steps ? steps : p.steps;
    }
  }
  const bool weights = backward && (a.q_weight_grad || a.k_weight_grad);
  if (weights) {
    DKV_CHECK((!a.q_weight_grad || a.q_weight) && (!a.k_weight_grad || a.k_weight), DKV_ERR_INVALID,
              "%s: the gradient of a weight that is not there", where);
    DKV_CHECK(a.workspace && ((uintptr_t)a.workspace & 15) == 0 &&
                  a.workspace_bytes >= dkv_rotate_heads_backward_workspace_bytes(&a),
              DKV_ERR_INVALID, "%s: workspace too small", where);
    p.side[0].dw = a.q_weight_grad, p.side[1].dw = a.k_weight_grad;
    p.side[0].sums = (float*)a.workspace;
    p.side[1].sums = p.side[0].sums + p.side[0].groups * a.D;
  }
  const bool next = a.interleaved != 0;
  if (a.dtype == kF32)
    launch_vec<kF32>(p, s.vec, next, backward, stream);
  else if (a.dtype == kF16)
    launch_vec<kF16>(p, s.vec, next, backward, stream);
  else
    launch_vec<kBF16>(p, s.vec, next, backward, stream);
  if (weights)
    hipLaunchKernelGGL(rotate_weights, dim3((unsigned)((a.D + 15) / 16), 2), dim3(1024), 0, stream, p);
  return dkv_check_launch(where);
}

}  // namespace

namespace dkv {

void launch_rotate_heads(const RotateParams& p, int dtype, int vec, bool next, hipStream_t stream) {
  if (dtype == kF32)
    launch_vec<kF32>(p, vec, next, false, stream);
  else if (dtype == kF16)
    launch_vec<kF16>(p, vec, next, false, stream);
  else
    launch_vec<kBF16>(p, vec, next, false, stream);
}

}  // namespace dkv

extern "C" int64_t dkv_rotate_heads_backward_workspace_bytes(const dkv_rotate_heads_args* args) {
  if (!args || check_rotate(*args, "dkv_rotate_heads_backward") != DKV_OK) return 0;
  return (backward_groups(*args, 0) + backward_groups(*args, 1)) * args->D * 4;
}

extern "C" int dkv_rotate_heads(const dkv_rotate_heads_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_rotate_heads: args is NULL");
  return run_rotate(*args, false, "dkv_rotate_heads", (hipStream_t)stream);
}

extern "C" int dkv_rotate_heads_backward(const dkv_rotate_heads_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_rotate_heads_backward: args is NULL");
  return run_rotate(*args, true, "dkv_rotate_heads_backward", (hipStream_t)stream);
}
