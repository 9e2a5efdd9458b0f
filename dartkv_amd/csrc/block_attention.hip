// Attention of each request's new tokens over its cache in e4m3 blocks (dkv_block_attention): few query rows.
//
// o[i] = sum_j softmax_j(scale q[i].k[j]) v[j] over the keys j < len - n + 1 + i of the request, k = code *
// kscale[block, head], v = code * vscale[block, head].
//
// Bound: the cache's bytes, 2 D per key and KV head; one wave reads 32 keys and values (64 D bytes) while it computes
// the 32 before: eight waves a CU keep 64 KB in flight at head_dim 128, 32 KB at 64, and the four that fit at 256 64 KB.
// 64 requests of 2,048 to 32,768 tokens, 8 KV heads of 128: 397 us, 5.7 TB/s (a copy reaches 4.7), and 7 to join the
// shares.  64 requests of 16,000, the whole call: head_dim 64 198 us, 5.3 TB/s; 128 372 us, 5.6; 256 710 us, 5.9; 16 of
// 8,000: 3.7, 4.8 and 4.5 TB/s.  One request of 4,000: 9 us, the chain of loads from the lengths to the keys, and 6.
//
// Work.  The requests' 32-key tiles are one line of units per KV head, cut into equal shares: a wave takes its
// share, whatever requests it covers, so ragged lengths leave no wave waiting for another.  A wave writes the
// result of a request that lies wholly in its share; of the first and the last, of which it has a part, it writes a
// record (m, l, o[D]) that block_merge joins.
//
// Matrix layout.  Both products are v_mfma_f32_16x16x32 with the query rows (row t * G + g: token t, head g of the
// KV head) as columns.  S^T = K Q^T: lane (key, group g) of a 16-key half tile reads DP / 4 contiguous channels of
// its key, so a step's 32 channels are 8 of each group's.  Its accumulators hold keys 4 g + 0..3 of row lane % 16,
// and O^T = V^T P^T takes P^T from there: slot j of group g is key 4 g + j of the first half tile (j < 4) or key
// 4 g + j - 4 of the second.  V is read in token order, DP / 16 contiguous channels per lane and token, and
// transposed in registers (byte pairs converted, then v_perm).  Nothing goes through LDS.
//
// Numerics.  Codes are exact in bf16 and fp16; the key scale goes into the logit's factor, the value scale (a power
// of two) into p, and p is split into two bf16 parts (16 bits of p: the products with V then lose nothing that a
// 16-bit result shows; the second product's cost is hidden behind the memory).  m, l and o are fp32; m is raised
// only when a logit exceeds it by more than 2^8.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_block_attention.h"
#include "dkv_capi_util.h"

using namespace dkv;
using namespace dkv::prompt;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kUnit = 32;       // keys of a unit of work
constexpr int kMinShare = 2;    // units of a wave at least
constexpr int kThreads = 256;

struct BlockParams {
  PromptParams a;
  float* records;  // [2 * workers][H][record_rows][D + 2]
  int32_t workers, rows;  // rows: the most of a request
  int32_t tile, record_rows;  // rows of a tile (16 NT), and of a record
};

struct Work {
  int n, rows, length, units;
  int64_t q0;
};

__device__ __forceinline__ int key_units(int length) {  // (a request without keys writes zeros)
  return length ? (length + kUnit - 1) / kUnit : 1;
}

// A request's new tokens and units (none when it has no rows, or more than this kernel takes).
__device__ __forceinline__ Work work_of(const BlockParams& bp, int r) {
  const PromptParams& p = bp.a;
  Work w = {0, 0, 0, 0, 0};
  if (r >= p.R) return w;
  int64_t a = r, b = r + 1;
  if (p.q_starts) a = p.q_starts[r], b = p.q_starts[r + 1];
  a = a < 0 ? 0 : a > p.q_tokens ? p.q_tokens : a;
  b = b < a ? a : b > p.q_tokens ? p.q_tokens : b;
  int64_t length = p.lengths[r];
  const int64_t most = (int64_t)p.max_blocks << p.bs_shift;
  length = length < 0 ? 0 : length > most ? most : length;
  w.q0 = a, w.n = (int)(b - a), w.length = (int)length;
  const int64_t rows = (b - a) * p.G;
  if (rows > bp.rows) return w;
  w.rows = (int)rows;
  w.units = (w.rows + bp.tile - 1) / bp.tile * key_units(w.length);
  return w;
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)(((uint64_t)uniform((uint32_t)(x >> 32)) << 32) | uniform((uint32_t)x));
}

__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(x, off, 64);
    if (lane >= off) x += up;
  }
  return x;
}

__device__ __forceinline__ int64_t share_of(int64_t total, int workers) {
  const int64_t s = (total + workers - 1) / workers;
  return s < kMinShare ? kMinShare : s;
}

template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0,
                                                  0);
}

// Two codes (the low or high half of w) as two 16-bit floats.
template <bool BF, bool HI>
__device__ __forceinline__ uint32_t two(uint32_t w) {
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
}

// LDS traffic of this wave before and after stays in program order.
__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 1 in each byte of w that is e4m3's NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u; }

template <int DP>
struct Unit {
  typedef uint32_t dwords __attribute__((ext_vector_type(DP / 64)));
  u32x4 k[2][DP / 64];  // 16-key halves; DP / 4 channels of one key
  dwords v[8];          // eight tokens; DP / 16 channels
  float ks[2], vs[2];
};

template <int DP, bool BF, int NT>
__global__ void __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) block_decode(BlockParams bp) {
  const PromptParams& p = bp.a;
  constexpr int KC = DP / 64;  // 16-byte pieces of a lane's key, dwords of a lane's value
  constexpr int KS = DP / 32, NB = DP / 16;
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + uniform(threadIdx.x >> 6);
  const int h = (int)(wave % p.H);
  const int worker = (int)(wave / p.H);
  if (worker >= bp.workers) return;
  __shared__ int32_t first_nan[kThreads / 64][DP];
  int32_t* first = first_nan[threadIdx.x >> 6];

  if (p.fill && p.q_starts) {  // rows behind the last request, then those before the first
    const int64_t end = clamped(p.q_starts[p.R], 0, p.q_tokens), begin = clamped(p.q_starts[0], 0, end);
    for (int64_t i = end + worker; i < p.q_tokens + begin; i += bp.workers) {
      const int64_t t = i < p.q_tokens ? i : i - p.q_tokens;
      for (int c = lane; c < p.G * p.D; c += 64)
        ((uint16_t*)p.o)[t * p.o_st + (h * p.G + c / p.D) * p.o_sh + c % p.D] = 0;
    }
  }

  // all units, then the request that this wave's first lies in
  Work mine = work_of(bp, lane);
  int scan = wave_scan(mine.units, lane);
  int64_t total = uniform(__shfl(scan, 63, 64));
  for (int b = 64; b < p.R; b += 64) {
    int x = work_of(bp, b + lane).units;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    total += uniform(x);
  }
  const int64_t share = share_of(total, bp.workers);
  int64_t unit = worker * share;
  const int64_t stop = unit + share < total ? unit + share : total;
  if (unit >= stop) return;
  int base = 0, lane_r = 0;
  int64_t before = 0;  // units before request `base`
  for (;;) {
    const uint64_t hit = __ballot(before + scan > unit);
    if (hit) {
      lane_r = __builtin_ctzll(hit);
      break;
    }
    before += uniform(__shfl(scan, 63, 64));
    base += 64;
    if (base >= p.R) return;  // (lengths beyond what any pool holds)
    mine = work_of(bp, base + lane);
    scan = wave_scan(mine.units, lane);
  }

  while (unit < stop) {
    // the request's part in this share (its units are not 0)
    const int r = uniform(base + lane_r);
    const int units = uniform(__shfl(mine.units, lane_r, 64));
    const int all_rows = uniform(__shfl(mine.rows, lane_r, 64));
    const int length = uniform(__shfl(mine.length, lane_r, 64));
    const int n = uniform(__shfl(mine.n, lane_r, 64));
    const int64_t q0 = (int64_t)uniform((uint32_t)__shfl((int)mine.q0, lane_r, 64));
    const int64_t start = before + uniform(__shfl(scan, lane_r, 64)) - units;
    const int key_units_r = uniform(key_units(length));
    const int tile = uniform((int)(unit - start) / key_units_r);
    const int64_t tile_start = start + (int64_t)tile * key_units_r;
    const int u0 = (int)(unit - tile_start);
    const int u1 = (int)((stop < tile_start + key_units_r ? stop : tile_start + key_units_r) - tile_start);
    const int row0 = tile * 16 * NT, rows = min(all_rows - row0, 16 * NT);
    const int nt = NT == 1 ? 1 : (rows + 15) / 16;

    u32x4 q[NT][KS];
    int limit[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = row0 + t * 16 + i16;
      const int token = row / p.G, head = h * p.G + row % p.G;
      const char* src = (const char*)p.q + 2 * ((q0 + token) * p.q_st + head * p.q_sh);
      limit[t] = row < all_rows ? length - n + 1 + token : 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int ch = g * (DP / 4) + s * 8;
        q[t][s] = (u32x4){0, 0, 0, 0};
        if (row < all_rows && ch < p.D) q[t][s] = *(const u32x4*)(src + 2 * ch);
      }
    }
    const int min_limit = length - n + 1 + row0 / p.G;

    f32x4 o[NT][NB];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -3.402823466e38f, l[t] = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) o[t][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }

    // 64 of the request's blocks and their scales, one per lane
    int cached = -64, my_block = 0;
    float my_ks = 0.f, my_vs = 0.f;
    auto fetch_blocks = [&](int first) {
      cached = first;
      const int at = first + lane < p.max_blocks ? first + lane : p.max_blocks - 1;
      const int id = p.table[(int64_t)r * p.max_blocks + at];
      const bool good = (uint32_t)id < (uint64_t)p.blocks;
      my_block = good ? id : 0;
      my_ks = p.kscale[(int64_t)my_block * p.H + h];
      my_vs = p.vscale[(int64_t)my_block * p.H + h];
      if (!good) my_ks = __builtin_nanf(""), my_vs = 1.f;  // a row that sees a bad entry is NaN
    };
    bool nans = false;
    // This lane's bytes of a half tile.  Channels behind head_dim read the first ones' bytes: their key operands are set
    // to 0 where they are used (a select beside the load would wait for it), their values' sums are not stored.
    const bool behind = p.D < DP;
    uint32_t kat[KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) kat[c] = i16 * p.D + (g * (DP / 4) + c * 16 < p.D ? g * (DP / 4) + c * 16 : 0);
    const uint32_t vat = 4 * g * p.D + (i16 * NB < p.D ? i16 * NB : 0);
    auto place = [&](int key, int s, int& at) {  // the byte of a half tile's first key in the codes
      at = ((key + 16 * s) >> p.bs_shift) - cached;
      const int id = uniform(__builtin_amdgcn_readlane(my_block, at));
      return (((int64_t)id * p.H + h) * (1 << p.bs_shift) + ((key + 16 * s) & ((1 << p.bs_shift) - 1))) * p.D;
    };
    auto load_keys = [&](Unit<DP>& x, int u) {
      const int key = u * kUnit;
      const int last_block = (key + 16) >> p.bs_shift;
      if (last_block >= cached + 64 || (key >> p.bs_shift) < cached || cached < 0) fetch_blocks(key >> p.bs_shift);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        int at;
        const uint8_t* kp = p.kc + place(key, s, at);
        x.ks[s] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_ks), at));
#pragma unroll
        for (int c = 0; c < KC; ++c) x.k[s][c] = *(const u32x4*)(kp + kat[c]);
      }
    };
    auto load_values = [&](Unit<DP>& x, int u) {  // after the unit's keys
      const int key = u * kUnit;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        int at;
        const uint8_t* vp = p.vc + place(key, s, at);
        x.vs[s] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_vs), at));
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[4 * s + j] = *(const typename Unit<DP>::dwords*)(vp + j * p.D + vat);
      }
    };
    auto products = [&](const Unit<DP>& x, f32x4 (&scores)[NT][2]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4 kf[KS];
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          const uint32_t a = x.k[s][c / 2][2 * (c % 2)], b = x.k[s][c / 2][2 * (c % 2) + 1];
          kf[c] = (u32x4){two<BF, false>(a), two<BF, true>(a), two<BF, false>(b), two<BF, true>(b)};
          if (behind && g * (DP / 4) + c * 8 >= p.D) kf[c] = (u32x4){0, 0, 0, 0};
        }
        const float f = p.c * x.ks[s];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (NT > 1 && t >= nt) break;
          f32x4 sc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KS; ++c) sc = mfma16<BF>(kf[c], q[t][c], sc);
#pragma unroll
          for (int e = 0; e < 4; ++e) scores[t][s][e] = sc[e] * f;
        }
        __builtin_amdgcn_sched_barrier(0);  // (one half's operands in registers at a time)
      }
    };
    auto sums = [&](const Unit<DP>& x, f32x4 (&scores)[NT][2], int u) {
      const int key = u * kUnit;
      u32x4 hi[NT], lo[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (NT > 1 && t >= nt) break;
        f32x4 (&sc)[2] = scores[t];
        if (key + kUnit > min_limit) {
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key + 16 * s + 4 * g + e >= limit[t]) sc[s][e] = -__builtin_inff();
        }
        float top = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) top = fmaxf(top, fmaxf(sc[0][e], sc[1][e]));
        if (__any(top > m[t] + 8.f)) {
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float up = fmaxf(m[t], top), f = __builtin_amdgcn_exp2f(m[t] - up);
          m[t] = up, l[t] *= f;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][b][e] *= f;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float w[4], rest[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float e2 = __builtin_amdgcn_exp2f(sc[s][e] - m[t]);
            l[t] += e2;
            w[e] = e2 * x.vs[s];
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t pair = pack2<true>(w[2 * e], w[2 * e + 1]);
            hi[t][2 * s + e] = pair;
            rest[2 * e] = w[2 * e] - u2f(pair << 16);
            rest[2 * e + 1] = w[2 * e + 1] - u2f(pair & 0xffff0000u);
            lo[t][2 * s + e] = pack2<true>(rest[2 * e], rest[2 * e + 1]);
          }
        }
      }
      const bool tail = key + kUnit > length;
      // Where drafted tokens hide keys from each other, 0 * NaN must not reach the rows that do not see a NaN code: such
      // codes become 0 here, and the first key of each channel that has one is kept; a row sees the keys before its
      // limit, so it sees one exactly if that key is before it (e4m3 has no infinities).
      bool any_nan = false;
      if (n > 1 && key + kUnit > min_limit) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int c = 0; c < KC; ++c) any_nan |= nan_bytes(x.v[j][c]) != 0;
        any_nan = __any(any_nan);
        if (any_nan) {
          if (!nans)
            for (int c = lane; c < DP; c += 64) first[c] = 0x7fffffff;
          nans = true;
          lds_order();
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < KC; ++c)
              for (uint32_t is = nan_bytes(x.v[j][c]); is; is &= is - 1)
                atomicMin(&first[i16 * NB + 4 * c + (__builtin_ctz(is) >> 3)], key + 16 * (j / 4) + 4 * g + j % 4);
        }
      }
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        u32x4 vf[4];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          uint32_t a = x.v[j][c], b = x.v[j + 1][c];
          if (tail) {
            const int tok = key + 16 * (j / 4) + 4 * g + j % 4;
            a = tok < length ? a : 0u;
            b = tok + 1 < length ? b : 0u;
          }
          if (any_nan) a &= ~(nan_bytes(a) * 0xffu), b &= ~(nan_bytes(b) * 0xffu);
          const uint32_t a0 = two<true, false>(a), a1 = two<true, true>(a);
          const uint32_t b0 = two<true, false>(b), b1 = two<true, true>(b);
          vf[0][j / 2] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
          vf[1][j / 2] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
          vf[2][j / 2] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
          vf[3][j / 2] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (NT > 1 && t >= nt) break;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            o[t][4 * c + b] = mfma16<true>(vf[b], hi[t], o[t][4 * c + b]);
            o[t][4 * c + b] = mfma16<true>(vf[b], lo[t], o[t][4 * c + b]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    if (length > 0) {
      f32x4 scores[NT][2];
      if constexpr (NT == 1) {
        Unit<DP> even, odd;
        auto load = [&](Unit<DP>& x, int u) { load_keys(x, u), load_values(x, u); };
        auto compute = [&](const Unit<DP>& x, int u) { products(x, scores), sums(x, scores, u); };
        load(even, u0);
        for (int u = u0; u < u1; u += 2) {
          if (u + 1 < u1) load(odd, u + 1);
          compute(even, u);
          if (u + 1 >= u1) break;
          if (u + 2 < u1) load(even, u + 2);
          compute(odd, u + 1);
        }
      } else {
        // The accumulators of more rows leave no room for a second unit: the next keys are read once the products
        // have used these, the next values after the sums.
        Unit<DP> x;
        load_keys(x, u0), load_values(x, u0);
        for (int u = u0; u < u1; ++u) {
          products(x, scores);
          if (u + 1 < u1) load_keys(x, u + 1);
          sums(x, scores, u);
          if (u + 1 < u1) load_values(x, u + 1);
        }
      }
    }

    if (nans) {
      lds_order();
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = first[(4 * g + e) * NB + b];
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (key < limit[t]) o[t][b][e] = __builtin_nanf("");
        }
    }

    // lane (row, g) has channels (4 g + e) * NB + b of its row
    const bool whole = u0 == 0 && u1 == key_units_r;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (NT > 1 && t >= nt) break;
      const int row = t * 16 + i16;
      l[t] += __shfl_xor(l[t], 16, 64);
      l[t] += __shfl_xor(l[t], 32, 64);
      if (row >= rows) continue;
      if (whole) {
        const float inv = l[t] == 0.f ? 0.f : 1.f / l[t];
        const int token = (row0 + row) / p.G, head = h * p.G + (row0 + row) % p.G;
        uint16_t* dst = (uint16_t*)p.o + (q0 + token) * p.o_st + head * p.o_sh;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ch = (4 * g + e) * NB;
          if (ch >= p.D) continue;
#pragma unroll
          for (int b = 0; b < NB; b += 2)
            *(uint32_t*)(dst + ch + b) = pack2<BF>(o[t][b][e] * inv, o[t][b + 1][e] * inv);
        }
      } else {
        float* rec = bp.records +
                     ((((int64_t)worker * 2 + (u0 == 0 ? 1 : 0)) * p.H + h) * bp.record_rows + row) * (p.D + 2);
        if (g == 0) rec[0] = m[t], rec[1] = l[t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ch = (4 * g + e) * NB;
          if (ch >= p.D) continue;
#pragma unroll
          for (int b = 0; b < NB; b += 2) *(f32x2*)(rec + 2 + ch + b) = (f32x2){o[t][b][e], o[t][b + 1][e]};
        }
      }
    }

    // the next tile, or the next request with units
    unit = tile_start + u1;
    if (unit < stop && unit == start + units) {
      uint64_t after = lane_r == 63 ? 0 : __ballot(mine.units > 0) >> (lane_r + 1) << (lane_r + 1);
      while (!after) {
        before += uniform(__shfl(scan, 63, 64));
        base += 64;
        if (base >= p.R) return;
        mine = work_of(bp, base + lane);
        scan = wave_scan(mine.units, lane);
        after = __ballot(mine.units > 0);
      }
      lane_r = __builtin_ctzll(after);
    }
  }
}

// Joins the records of the requests that several waves had, a row of a request and KV head at a time: by one wave, or
// (WIDE) by a workgroup's four where there are few rows, so that all of a long request's records are in flight.
template <bool BF, bool WIDE>
__global__ void __launch_bounds__(kThreads) block_merge(BlockParams bp) {
  const PromptParams& p = bp.a;
  constexpr int kAhead = 8;  // records in flight of a wave, each a round trip to memory that other XCDs have written
  __shared__ float part[WIDE ? 4 : 1][256];
  __shared__ float sums[4], tops[4];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t unit = WIDE ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int h = (int)(unit % p.H), row = (int)(unit / p.H % bp.rows);
  const int r = (int)(unit / p.H / bp.rows);
  if (r >= p.R) return;
  const Work w = work_of(bp, r);
  if (row >= w.rows) return;
  int64_t total = 0, start = 0;
  for (int base = 0; base < p.R; base += 64) {
    int x = work_of(bp, base + lane).units;
    int y = base + lane < r ? x : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64), y += __shfl_xor(y, off, 64);
    total += x, start += y;
  }
  const int64_t share = share_of(uniform64(total), bp.workers);
  start = uniform64(start);
  const int key_units_r = uniform(key_units(w.length)), place = row % bp.tile;
  start += (int64_t)(row / bp.tile) * key_units_r;
  const int w0 = uniform((int)(start / share)), w1 = uniform((int)((start + key_units_r - 1) / share));
  if (w0 == w1) return;
  float m = -3.402823466e38f, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int kStep = WIDE ? 4 : 1;
  for (int x0 = w0 + (WIDE ? wave : 0); x0 <= w1; x0 += kStep * kAhead) {
    float rm[kAhead], rl[kAhead];
    f32x2 v[kAhead][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int x = x0 + kStep * i <= w1 ? x0 + kStep * i : x0;
      const int slot = x == w0 ? 1 : 0;  // a part that begins the request, or goes on with it
      const float* rec = bp.records + ((((int64_t)x * 2 + slot) * p.H + h) * bp.record_rows + place) * (p.D + 2);
      rm[i] = x0 + kStep * i <= w1 ? rec[0] : -__builtin_inff(), rl[i] = rec[1];
#pragma unroll
      for (int c = 0; c < 2; ++c)
        v[i][c] = *(const f32x2*)(rec + 2 + (2 * (lane + 64 * c) < p.D ? 2 * (lane + 64 * c) : 0));
    }
    float up = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) up = fmaxf(up, rm[i]);
    const float f0 = __builtin_amdgcn_exp2f(m - up);
    m = up, l *= f0;
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] *= f0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float f = __builtin_amdgcn_exp2f(rm[i] - up);
      l += rl[i] * f;
#pragma unroll
      for (int c = 0; c < 2; ++c) acc[2 * c] += v[i][c][0] * f, acc[2 * c + 1] += v[i][c][1] * f;
    }
  }
  const int token = row / p.G, head = h * p.G + row % p.G;
  uint16_t* dst = (uint16_t*)p.o + (w.q0 + token) * p.o_st + head * p.o_sh;
  if constexpr (!WIDE) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (2 * (lane + 64 * c) < p.D)
        *(uint32_t*)(dst + 2 * (lane + 64 * c)) = pack2<BF>(acc[2 * c] * inv, acc[2 * c + 1] * inv);
  } else {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (2 * (lane + 64 * c) < p.D) {
        part[wave][2 * (lane + 64 * c)] = acc[2 * c];
        part[wave][2 * (lane + 64 * c) + 1] = acc[2 * c + 1];
      }
    }
    if (lane == 0) sums[wave] = l, tops[wave] = m;
    __syncthreads();
    const float up = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    float f[4], all = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __builtin_amdgcn_exp2f(tops[i] - up), all += sums[i] * f[i];
    const float inv = all == 0.f ? 0.f : 1.f / all;
    for (int c = 2 * threadIdx.x; c < p.D; c += 2 * kThreads) {
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) a += part[i][c] * f[i], b += part[i][c + 1] * f[i];
      *(uint32_t*)(dst + c) = pack2<BF>(a * inv, b * inv);
    }
  }
}

template <int DP, bool BF>
void launch_decode(const BlockParams& bp, hipStream_t stream) {
  const int64_t waves = (int64_t)bp.workers * bp.a.H;
  const dim3 grid((unsigned)((waves + 3) / 4));
  if (bp.tile == 16)
    hipLaunchKernelGGL((block_decode<DP, BF, 1>), grid, dim3(kThreads), 0, stream, bp);
  else if constexpr (DP <= 128)
    hipLaunchKernelGGL((block_decode<DP, BF, 2>), grid, dim3(kThreads), 0, stream, bp);
  // one wave a row where that gives the CUs eight each (16 requests of four tokens, 32 rows a KV head: 19.7 us with
  // four waves a row), else four (one request of 4,000 tokens: 64 records in two rounds)
  const int64_t rows = (int64_t)bp.a.R * bp.rows * bp.a.H;
  if (rows >= 2048)
    hipLaunchKernelGGL((block_merge<BF, false>), dim3((unsigned)((rows + 3) / 4)), dim3(kThreads), 0, stream, bp);
  else
    hipLaunchKernelGGL((block_merge<BF, true>), dim3((unsigned)rows), dim3(kThreads), 0, stream, bp);
}

// Waves of a KV head: two for each of 1,024 SIMDs, resident at once; head_dims over 128 leave one, and two rounds.
int workers_for(int64_t H) {
  const int64_t w = (2048 + H - 1) / H;
  return (int)(w < 1 ? 1 : w);
}

// Rows of a request that this kernel takes: all up to 64, in tiles of 16 or (two accumulators of 16, which head_dims
// over 128 leave no registers for) 32 that each read the keys; else those of at most 16 rows.
int rows_for(int64_t max_tokens, int64_t G) { return max_tokens <= 64 / G ? (int)(max_tokens * G) : 16; }

int64_t most_tokens(const dkv_block_attention_args& a) {
  const int64_t most = a.max_tokens < a.tokens ? a.max_tokens : a.tokens;
  return most < 1 ? 1 : most;
}

int check_blocks(const dkv_block_attention_args& a) {
  DKV_CHECK(a.dtype == kF16 || a.dtype == kBF16, DKV_ERR_DTYPE, "dkv_block_attention: the query must be bf16 or fp16");
  DKV_CHECK(a.Hkv >= 1 && a.Hq >= a.Hkv && a.Hq % a.Hkv == 0 && a.Hq < (1 << 20), DKV_ERR_INVALID,
            "dkv_block_attention: query heads must be divisible by the cache's KV heads");
  DKV_CHECK(a.D >= 16 && a.D <= 256 && a.D % 16 == 0, DKV_ERR_INVALID,
            "dkv_block_attention: head_dim must be a multiple of 16 up to 256");
  DKV_CHECK(a.block_size >= 16 && a.block_size <= 256 && (a.block_size & (a.block_size - 1)) == 0, DKV_ERR_INVALID,
            "dkv_block_attention: block_size must be 16, 32, 64, 128 or 256");
  DKV_CHECK(a.requests >= 1 && a.tokens >= 0 && a.blocks >= 1 && a.max_blocks >= 1 && a.max_tokens >= 1,
            DKV_ERR_INVALID, "dkv_block_attention: bad counts");
  DKV_CHECK(a.tokens < (1ll << 31) / (a.Hq / a.Hkv) - 1024 && a.max_blocks < ((1ll << 31) - 1024) / a.block_size &&
                a.blocks < (1ll << 31) && a.requests < (1 << 24) && a.requests * 64 * a.Hkv < (1ll << 31),
            DKV_ERR_INVALID, "dkv_block_attention: too many tokens");
  return DKV_OK;
}

BlockParams params_of(const dkv_block_attention_args& a) {
  BlockParams bp = {};
  PromptParams& p = bp.a;
  p.q = a.query, p.o = a.out;
  p.q_st = a.q_st, p.q_sh = a.q_sh, p.o_st = a.o_st, p.o_sh = a.o_sh;
  p.q_starts = a.starts;
  p.R = (int32_t)a.requests, p.H = (int32_t)a.Hkv, p.G = (int32_t)(a.Hq / a.Hkv), p.D = (int32_t)a.D;
  p.q_tokens = a.tokens;
  p.c = (float)(a.scale * 1.4426950408889634);
  p.causal = 1, p.fill = a.fill ? 1 : 0, p.splits = 1;
  p.kc = a.key_codes, p.vc = a.value_codes, p.kscale = a.key_scale, p.vscale = a.value_scale;
  p.table = a.table, p.lengths = a.lengths, p.blocks = a.blocks, p.max_blocks = (int32_t)a.max_blocks;
  p.bs_shift = __builtin_ctzll((uint64_t)a.block_size);
  bp.workers = workers_for(a.Hkv), bp.rows = rows_for(most_tokens(a), p.G);
  bp.tile = bp.rows > 16 && p.D <= 128 ? 32 : 16;
  bp.record_rows = bp.rows < bp.tile ? bp.rows : bp.tile;
  return bp;
}

int64_t workspace_of(const dkv_block_attention_args& a, const BlockParams& bp) {
  const int64_t few = 2 * (int64_t)bp.workers * a.Hkv * bp.record_rows * (a.D + 2) * 4;
  if (most_tokens(a) <= bp.rows / bp.a.G) return few;
  const int64_t many = block_chunks_workspace_bytes(bp.a, a.tokens * bp.a.G, a.dtype == kBF16);
  return few > many ? few : many;  // (one after the other on the stream)
}

}  // namespace

extern "C" int64_t dkv_block_attention_workspace_bytes(const dkv_block_attention_args* args) {
  if (!args || check_blocks(*args) != DKV_OK) return 0;
  return workspace_of(*args, params_of(*args));
}

extern "C" int dkv_block_attention(const dkv_block_attention_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_block_attention: args is NULL");
  const dkv_block_attention_args& a = *args;
  const int bad = check_blocks(a);
  if (bad != DKV_OK) return bad;
  DKV_CHECK(a.starts || a.tokens == a.requests, DKV_ERR_INVALID,
            "dkv_block_attention: without starts every request has one token");
  // (the fp32 factor must not be 0: a hidden key's logit would be -inf * 0)
  DKV_CHECK(a.scale >= 1e-37 && a.scale < 1e30, DKV_ERR_INVALID, "dkv_block_attention: scale must be in 1e-37 to 1e30");
  if (a.tokens == 0) return DKV_OK;
  DKV_CHECK(a.query && a.out && a.key_codes && a.value_codes && a.key_scale && a.value_scale && a.table && a.lengths,
            DKV_ERR_INVALID, "dkv_block_attention: NULL pointer");
  DKV_CHECK((((uintptr_t)a.query | (uintptr_t)(2 * a.q_st) | (uintptr_t)(2 * a.q_sh) | (uintptr_t)a.key_codes |
              (uintptr_t)a.value_codes) & 15) == 0 &&
                (((uintptr_t)a.out | (uintptr_t)(2 * a.o_st) | (uintptr_t)(2 * a.o_sh)) & 7) == 0,
            DKV_ERR_INVALID, "dkv_block_attention: query rows must be 16-byte aligned, output rows 8-byte");
  BlockParams bp = params_of(a);
  PromptParams& p = bp.a;
  DKV_CHECK(a.workspace && ((uintptr_t)a.workspace & 15) == 0 && a.workspace_bytes >= workspace_of(a, bp),
            DKV_ERR_INVALID, "dkv_block_attention: workspace too small");
  bp.records = (float*)a.workspace;
  const bool bf = a.dtype == kBF16;
  const hipStream_t s = (hipStream_t)stream;
  if (a.D <= 64)
    bf ? launch_decode<64, true>(bp, s) : launch_decode<64, false>(bp, s);
  else if (a.D <= 128)
    bf ? launch_decode<128, true>(bp, s) : launch_decode<128, false>(bp, s);
  else
    bf ? launch_decode<256, true>(bp, s) : launch_decode<256, false>(bp, s);
  const int rc = dkv_check_launch("dkv_block_attention");
  if (rc != DKV_OK || most_tokens(a) <= bp.rows / p.G) return rc;
  p.skip_rows = bp.rows, p.fill = 0;
  if (!a.starts) p.q_tokens = 1, p.q_sb = a.q_st, p.o_sb = a.o_st;  // a batch of one token each
  return launch_block_chunks(p, a.tokens * p.G, bf, a.workspace, stream);
}
