// Attention of a tile of query rows over a request's keys (gfx950, wave64): the kernel of prompt_attention
// (16-bit keys and values, prompt.hip) and of block_attention's long chunks (e4m3 blocks, block_chunks.hip).
//
// Rows.  The query heads of a KV head are rows of one problem: row t * G + g is token t of head h * G + g, so a
// tile of BM rows reads its keys once for all G heads, and a causal tile of 128 rows masks no more than 128 / G
// tokens' diagonal.  Row t * G + g sees the first t + 1 + (nk - nq) keys (all nk without the causal mask).
//
// One pass over the keys, 64 at a time, with a running maximum m and sum l (fp32) per row:
//   s = c q.k (c = scale log2 e), p = 2^(s - m), l += p, o += p v, and o, l times 2^(m - m') when m grows.
// m is only raised when a row's maximum exceeds it by more than 8 (2^8: p stays within bf16 and fp16, and l and
// o are sums of the same p), so most tiles scale nothing.  fp16 has 2^7 p in place of p, which cancels in o / l: up to
// 2^15 of its 2^16, and normal from p = 2^-21 on (bare weights were subnormal under 2^-14 and 0 under 2^-25, while l had
// them whole: beside a dominant key 2^20 times as heavy the others' sum was 3 % off).
//
// Matrix layout.  Both products are v_mfma_f32_32x32x16 with the query row in the column of the result:
// S^T = K Q^T puts keys 8 (i / 4) + 4 half + i % 4 (i < 16) of 32 in lane (row, half)'s accumulators, and
// O^T = V^T P^T takes P^T's 16 keys of a step from the same lane: step ks, slot j is key 16 ks + 8 (j / 4) +
// 4 half + j % 4, accumulator 8 (ks % 2) + j.  So P never leaves its lane, a row's maximum takes one exchange
// between the wave's halves, and its scale one value per lane.  V^T's operand has four keys of one channel per
// ds_read_b64_tr_b16: V stays in token order in LDS.
//
// LDS.  Rows of 2 DP bytes in chunks of 16, chunk c of row r at c ^ swizzle(r): sixteen consecutive rows' reads
// of one chunk (K) and four consecutive rows' reads of four chunks (V) fall in different banks (no conflicts counted).
// Two buffers of 64 keys (32 where registers are short); the next tile's copies are in flight while a tile is computed,
// one barrier a tile.
//
// Fewer bits.  l sums p in fp32; for the second product p is rounded to the operands' type (prompts, and chunks under bf16
// queries), half a step each.  In bf16 that takes the error from 1.6e-3 of the result's norm, which is the result's own
// rounding, to 2.1e-3.  p in two bf16 parts, as chunks under fp16 queries have it, leaves 1.6e-3 and costs half of all
// products again: 16,384 tokens 2,740 us in place of 1,980, 16 ragged prompts 977 and 752, 1,024 tokens 32.7 and 26.7.
//
// Bound and measured.  16,384 tokens of 32 query heads of 128, bf16: 1.95-2.01 ms, 1.1 PFLOP/s.  Matrix units busy 53 % of
// the cycles, vector units 46 %, LDS 27 %, at 1.78-1.91 GHz (counters and times of the same launches); a 16,384^3 matrix
// product keeps the matrix units busy 72 % at 1.81 GHz, 1.37 PFLOP/s.  So it is the exponentials and maxima between the
// products that hold it, not the clock.  Ragged prompts of 64 to 4,096 tokens: 45 % busy, the vector units the same: about
// 18 key tiles a workgroup, whose start and end cost about four.  A single short prompt is bound by its last tiles and
// about 8 us of start and end.  Chunks over blocks: 35 % and 39 % busy at 2.1 GHz, as a stage's conversion into LDS stands
// between two barriers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_device.h"

namespace dkv {

struct PromptParams {
  const void *q, *k, *v;
  void* o;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh;  // strides in elements
  const int32_t *q_starts, *k_starts;  // [R + 1], or NULL: every request has q_tokens (k_tokens)
  int32_t R, H, G, D;
  int64_t q_tokens, k_tokens;  // rows of the packed tensors, or of each request
  float c;                     // scale * log2(e)
  int32_t causal, fill;        // fill: rows behind the last request and before the first become 0
  // e4m3 blocks
  const uint8_t *kc, *vc;       // [blocks][H][bs][D]
  const float *kscale, *vscale;  // [blocks][H]
  const int32_t *table, *lengths;
  int64_t blocks;
  int32_t max_blocks, bs_shift;
  int32_t skip_rows;  // requests of at most this many rows are another kernel's
  // A tile's keys in up to `splits` parts of at least kMinPart key tiles, where there are few workgroups: each leaves a
  // record, o [BM][D] and (m, l) [BM], that prompt_merge joins.
  int32_t splits;
  int32_t pairs;  // two workgroups share a CU: the second half of a request's tiles are its shortest, shortest first
  float *records, *stats;
};

namespace prompt {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) void lds_void;

// Keys of a tile: 64; 32 where the accumulators (head_dims over 128) or the split weights (fp16 queries over blocks)
// leave no registers for more.
constexpr int keys_of(int DP, bool split) { return DP <= (split ? 64 : 128) ? 64 : 32; }
// LDS of a workgroup: two buffers of keys and values, the blocks' scales, the careful pass's first keys.
constexpr int lds_bytes(int DP, int keys, int groups) { return 4 * groups * keys * 2 * DP + 64 + 8 * DP; }

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0,
                                                  0);
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, half2v));
}

// The other half's value of the same row.
__device__ __forceinline__ float other_half(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

template <int DP>
__device__ __forceinline__ int swizzle(int row) {
  if constexpr (DP == 64)
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else
    return ((row & 3) << 2) | ((row >> 2) & 3);
}

// 64 x 16 bytes, lane l's from byte `offset` of the buffer to LDS address lds + 16 l; zeros outside the buffer.
// From inline assembly, so that the compiler does not wait for it before the other buffer's reads.
__device__ __forceinline__ void buffer_to_lds(u32x4 rsrc, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds" ::"v"(offset), "s"(lds),
               "s"(rsrc)
               : "memory");
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// A buffer descriptor of `bytes` bytes at `base` (both wave-uniform).
__device__ __forceinline__ u32x4 buffer(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  return (u32x4){uniform((uint32_t)a), uniform((uint32_t)(a >> 32)) & 0xffffu, uniform(bytes), 0x00027000u};
}

constexpr int kMinPart = 8;

// Key tiles of a part, and how many parts there are.
struct Parts {
  int per, count;
};
__device__ __forceinline__ Parts parts_of(int limit, int keys, int splits) {
  const int n = (limit + keys - 1) / keys;
  const int per = max((n + splits - 1) / splits, kMinPart);
  return {per, max(1, (n + per - 1) / per)};
}

// Which request and row tile a workgroup has.
struct Tile {
  int request;  // -1: none
  int tile, rows;
  int nq, nk;
  int64_t q0, k0;  // first tokens
};

__device__ __forceinline__ int64_t clamped(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// The requests' tiles one after the other, those of more keys first (up to 64 requests; else in their order), found
// by a wave's scan over the requests: the longest work begins first, and what begins last is short.  Rows to fill are one
// more request without keys, from the last request's end round to the first's start.
template <int BM, bool BLOCKS>
__device__ __forceinline__ Tile find_tile(const PromptParams& p, int64_t index) {
  Tile t = {-1, 0, 0, 0, 0, 0, 0};
  const int lane = threadIdx.x & 63;
  const int64_t most = (int64_t)p.max_blocks << p.bs_shift;
  if (!p.q_starts) {
    const int rows = (int)p.q_tokens * p.G, tiles = (rows + BM - 1) / BM;
    const bool across = p.pairs;  // every request's longest tiles first
    if (index >= (int64_t)tiles * p.R) return t;
    const int r = (int)(across ? index % p.R : index / tiles);
    const int nk = BLOCKS ? (int)clamped(p.lengths[r], 0, most) : (int)p.k_tokens;
    t = {r, (int)(across ? index / p.R : index - (int64_t)r * tiles), rows, (int)p.q_tokens, nk, 0, 0};
    return t;
  }
  int64_t before = 0;
  const int total = p.R + (p.fill ? 1 : 0);
  for (int base = 0; base < total; base += 64) {
    int r = base + lane;
    int64_t a = 0, b = 0, ka = 0, kb = 0;
    if (r < total) {  // (never outside the tensors, whatever the starts say)
      a = clamped(p.q_starts[r], 0, p.q_tokens);
      b = r < p.R ? clamped(p.q_starts[r + 1], a, p.q_tokens) : p.q_tokens + clamped(p.q_starts[0], 0, a);
      if (r < p.R) {
        if constexpr (BLOCKS) {
          kb = clamped(p.lengths[r], 0, most);
        } else {
          ka = clamped(p.k_starts[r], 0, p.k_tokens);
          kb = clamped(p.k_starts[r + 1], ka, p.k_tokens);
        }
      }
    }
    int rows = (int)(b - a) * p.G, nk = (int)(kb - ka);
    if (rows <= p.skip_rows && r < p.R) rows = 0;
    if (total > 1 && total <= 64) {  // lane i takes the request of the i-th most keys
      int rank = 0;
      for (int i = 0; i < total; ++i) {
        const int other = __builtin_amdgcn_readlane(nk, i);
        rank += other > nk || (other == nk && i < lane) ? 1 : 0;
      }
      if (lane >= total) rank = lane;
      r = __builtin_amdgcn_ds_permute(4 * rank, r);
      rows = __builtin_amdgcn_ds_permute(4 * rank, rows), nk = __builtin_amdgcn_ds_permute(4 * rank, nk);
      a = __builtin_amdgcn_ds_permute(4 * rank, (int)a), b = __builtin_amdgcn_ds_permute(4 * rank, (int)b);
      ka = __builtin_amdgcn_ds_permute(4 * rank, (int)ka);
    }
    const int tiles = (rows + BM - 1) / BM;
    int sum = tiles;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int up = __shfl_up(sum, off, 64);
      if (lane >= off) sum += up;
    }
    const uint64_t hit = __ballot(before + sum > index);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      t.request = __builtin_amdgcn_readlane(r, l);
      t.rows = __builtin_amdgcn_readlane(rows, l), t.nk = __builtin_amdgcn_readlane(nk, l);
      t.tile = (int)(index - before) - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
      t.q0 = __builtin_amdgcn_readlane((int)a, l), t.k0 = __builtin_amdgcn_readlane((int)ka, l);
      t.nq = __builtin_amdgcn_readlane((int)b, l) - (int)t.q0;
      return t;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return t;
}

// A tile of the rows to fill, which go round the end of the packed tensor: a way of its own, so that the kernel around it
// keeps its registers (head_dim 256: 4 % of a prompt's time with the wrap in every tile's addresses).
template <int BM>
__device__ __forceinline__ void fill_tile(const PromptParams& p, const Tile& t, int h) {
  const int pieces = p.D / 4;
  for (int i = threadIdx.x; i < BM * pieces; i += blockDim.x) {
    const int row = t.tile * BM + i / pieces;
    if (row >= t.rows) return;
    int64_t at = t.q0 + row / p.G;
    if (at >= p.q_tokens) at -= p.q_tokens;
    *(u32x2*)((uint16_t*)p.o + at * p.o_st + (h * p.G + row % p.G) * p.o_sh + i % pieces * 4) = (u32x2){0, 0};
  }
}

// A product adds 0 * v for a key that its row does not see, or whose weight is too small for its type, which is NaN where
// v is an infinity or a NaN.  Where a tile's result is not finite, it is computed again with such values set to 0 in LDS,
// and what they do is added at the end: a row sees the keys before its limit, so it sees one exactly if the channel's
// first one is before it.
// first[ch] is the first key with an infinity or NaN, first[DP + ch] with a negative infinity or NaN.
template <int DP, int KEYS, bool BF, int THREADS>
__device__ __forceinline__ void set_apart(char* lv, int j, int32_t* first) {
  constexpr uint32_t kExp = BF ? 0x7f80u : 0x7c00u;
  for (int at = threadIdx.x; at < KEYS * DP; at += THREADS) {
    const int row = at / DP, ch = at % DP;
    uint16_t* place = (uint16_t*)(lv + row * 2 * DP + (((ch >> 3) ^ swizzle<DP>(row)) << 4)) + (ch & 7);
    const uint32_t x = *place;
    if ((x & kExp) == kExp) {
      const bool nan = (x & 0x7fffu) > kExp;
      if (nan || !(x & 0x8000u)) atomicMin(&first[ch], j + row);
      if (nan || (x & 0x8000u)) atomicMin(&first[DP + ch], j + row);
      *place = 0;
    }
  }
}

// Copies of 16-bit keys and values: straight from memory to LDS.
template <int DP, int WAVES, int kKeys>
struct DenseSource {
  const char *k, *v;
  int64_t kst, vst;  // bytes
  int nk, valid;     // valid: bytes of a row
  uint32_t koff[kKeys * DP / 512 / WAVES], voff[kKeys * DP / 512 / WAVES];
  static constexpr int kCopies = kKeys * DP / 512 / WAVES;  // of a wave, for keys and for values
  static constexpr int kRowBytes = 2 * DP;

  __device__ __forceinline__ void init(const PromptParams& p, const Tile& t, int h) {
    const int64_t b = p.k_starts ? 0 : t.request;
    k = (const char*)p.k + 2 * (b * p.k_sb + t.k0 * p.k_st + h * p.k_sh);
    v = (const char*)p.v + 2 * (b * p.v_sb + t.k0 * p.v_st + h * p.v_sh);
    kst = 2 * p.k_st, vst = 2 * p.v_st, nk = t.nk, valid = 2 * p.D;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = (i * WAVES + wave) * 1024 + lane * 16;  // LDS byte of the tile
      const int row = at / kRowBytes, chunk = ((at % kRowBytes) >> 4) ^ swizzle<DP>(row);
      const bool in = chunk * 16 < valid;
      koff[i] = in ? (uint32_t)(row * kst) + chunk * 16 : 0x80000000u;
      voff[i] = in ? (uint32_t)(row * vst) + chunk * 16 : 0x80000000u;
    }
  }
  // Start the copies of keys [j, j + 64) to the LDS tiles at lk and lv.
  __device__ __forceinline__ void issue(int j, uint32_t lk, uint32_t lv) {
    const int left = nk - j < kKeys ? nk - j : kKeys;
    const u32x4 rk = buffer(k + j * kst, (uint32_t)((left - 1) * kst) + valid);
    const u32x4 rv = buffer(v + j * vst, (uint32_t)((left - 1) * vst) + valid);
    const int wave = uniform(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) buffer_to_lds(rk, koff[i], lk + (i * WAVES + wave) * 1024);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) buffer_to_lds(rv, voff[i], lv + (i * WAVES + wave) * 1024);
  }
};

// Keys and values held in e4m3 blocks: read into registers while the tile before is computed, then converted into
// LDS.  bf16 queries: codes times their scale (exact), fp16 queries: keys as bare fp16 codes (a scaled value may
// leave fp16's range), whose scale goes to the logits, and values as scaled bf16.
template <int DP, bool BF, int WAVES, int kKeys>
struct BlockSource {
  static constexpr int kChunks = kKeys * DP / 16 / (64 * WAVES);  // 16 codes each, of a thread
  static constexpr int kRowBytes = 2 * DP;
  const PromptParams& p;
  const int32_t* table;
  int h, nk;
  int id[kChunks];
  u32x4 k[kChunks], v[kChunks];
  float ks[kChunks], vs[kChunks];
  enum { kCodes, kNothing, kBad };
  int what[kChunks];

  __device__ __forceinline__ BlockSource(const PromptParams& p_, int request, int h_, int nk_)
      : p(p_), table(p_.table + (int64_t)request * p_.max_blocks), h(h_), nk(nk_) {}
  __device__ __forceinline__ static int row_of(int i) { return (threadIdx.x + i * 64 * WAVES) / (DP / 16); }
  __device__ __forceinline__ static int chunk_of(int i) { return (threadIdx.x + i * 64 * WAVES) % (DP / 16); }
  // The blocks of keys [j, j + 64), asked for a tile ahead.
  __device__ __forceinline__ void blocks(int j) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int at = (j + row_of(i)) >> p.bs_shift;
      id[i] = table[at < p.max_blocks ? at : p.max_blocks - 1];
    }
  }
  // (What a load brings is not looked at here: that would wait for it.)
  __device__ __forceinline__ void issue(int j) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int key = j + row_of(i), ch = 16 * chunk_of(i);
      const bool in = key < nk && ch < p.D, good = (uint32_t)id[i] < (uint64_t)p.blocks;
      const int64_t bh = (int64_t)(good ? id[i] : 0) * p.H + h;
      const int64_t off = ((bh << p.bs_shift) + (key & ((1 << p.bs_shift) - 1))) * p.D + (in ? ch : 0);
      k[i] = *(const u32x4*)(p.kc + off), v[i] = *(const u32x4*)(p.vc + off);
      ks[i] = p.kscale[bh], vs[i] = p.vscale[bh];
      what[i] = !in ? kNothing : good ? kCodes : kBad;
    }
  }
  template <bool AS_BF>
  __device__ __forceinline__ static void convert(u32x4 w, float scale, u32x4& a, u32x4& b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t lo, hi;
      if constexpr (AS_BF) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], scale, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], scale, true));
      } else {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, true));
      }
      if (i < 2)
        a[2 * i] = lo, a[2 * i + 1] = hi;
      else
        b[2 * i - 4] = lo, b[2 * i - 3] = hi;
    }
  }
  // The tile read last to LDS: keys, values and (fp16) the scale of every 16 keys.
  __device__ __forceinline__ void finish(char* lk, char* lv, float* lscale) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int row = row_of(i), chunk = chunk_of(i);
      const int a = row * kRowBytes + (((2 * chunk) ^ swizzle<DP>(row)) << 4);
      const int b = row * kRowBytes + (((2 * chunk + 1) ^ swizzle<DP>(row)) << 4);
      u32x4 x, y;
      if (what[i] != kCodes) {
        const uint32_t fill = what[i] == kBad ? 0x7f7f7f7fu : 0u;  // NaN: a bad entry shows
        k[i] = (u32x4){fill, fill, fill, fill}, v[i] = (u32x4){0, 0, 0, 0};
      }
      convert<BF>(k[i], ks[i], x, y);
      *(u32x4*)(lk + a) = x, *(u32x4*)(lk + b) = y;
      convert<true>(v[i], vs[i], x, y);
      *(u32x4*)(lv + a) = x, *(u32x4*)(lv + b) = y;
      if (!BF && chunk == 0 && row % 16 == 0) lscale[row / 16] = ks[i];
    }
  }
};

// GROUPS 2: half of the waves have a stage's first kKeys keys, the other half its second for the same rows, and their
// sums are joined at the end: two waves a SIMD where a launch has no more workgroups than CUs.  KEYS: keys of a tile.
template <int DP, bool BF, int WAVES, bool BLOCKS, int GROUPS, int KEYS = keys_of(DP, BLOCKS && !BF)>
__global__ void __launch_bounds__(64 * WAVES, DP <= 64 && !BLOCKS && GROUPS == 1 ? 3 : DP <= 128 ? 2 : 1)
    prompt_tiles(PromptParams p) {
  constexpr int BM = 32 * WAVES / GROUPS, KS = DP / 16, CB = DP / 32, kKeys = KEYS, T2 = kKeys / 32;
  constexpr int kStage = GROUPS * kKeys, kRowBytes = 2 * DP, kTileBytes = kStage * kRowBytes;
  extern __shared__ __attribute__((aligned(1024))) char lds[];  // K, V, K, V
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6) % (WAVES / GROUPS), half = lane >> 5;
  const int group = GROUPS == 1 ? 0 : uniform(threadIdx.x >> 6) / (WAVES / GROUPS);

  const int h = (int)(blockIdx.x % p.H), part = (int)(blockIdx.x / p.H % p.splits);
  Tile t = find_tile<BM, BLOCKS>(p, blockIdx.x / p.H / p.splits);
  if (t.request < 0) return;
  t.request = uniform(t.request), t.tile = uniform(t.tile), t.rows = uniform(t.rows), t.nq = uniform(t.nq);
  t.nk = uniform(t.nk), t.q0 = uniform((uint32_t)t.q0), t.k0 = uniform((uint32_t)t.k0);
  {
    const int tiles = (t.rows + BM - 1) / BM, late = t.tile - (tiles + 1) / 2;
    t.tile = p.pairs && late >= 0 ? late : tiles - 1 - t.tile;  // the longest tiles first
  }
  if (t.request == p.R) {
    if (part == 0) fill_tile<BM>(p, t, h);
    return;
  }
  const int nk = t.nk;

  // this lane's row, how many keys it sees, and its query in the products' operand layout
  const int row = t.tile * BM + wave * 32 + (lane & 31);
  const bool real = row < t.rows;
  const int token = row / p.G, head = h * p.G + row % p.G;
  const int64_t qb = p.q_starts ? 0 : t.request;
  auto limit_of = [&](int tok) {
    int n = p.causal ? tok + 1 + nk - t.nq : nk;
    return n < 0 ? 0 : n > nk ? nk : n;
  };
  const int limit = real ? limit_of(token) : 0;
  const int last_row = min(t.tile * BM + BM, t.rows) - 1;
  const Parts parts = parts_of(uniform(limit_of(last_row / p.G)), kStage, p.splits);
  if (part >= parts.count) return;
  const int part_first = part * parts.per * kStage;
  const int tile_limit = min(uniform(limit_of(last_row / p.G)), part_first + parts.per * kStage);
  const int wave_first = min(t.tile * BM + wave * 32, t.rows - 1), wave_last = min(wave_first + 31, t.rows - 1);
  const bool wave_real = t.tile * BM + wave * 32 < t.rows;
  const int wave_min = uniform(limit_of(wave_first / p.G));
  const int wave_max = wave_real ? uniform(limit_of(wave_last / p.G)) : 0;

  f32x16 o[CB];
  float m, l;

  // LDS bytes of this lane's operand chunks within a tile
  int kaddr[KS], vaddr[CB][2];
  {
    const int key = lane & 31;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kaddr[ks] = key * kRowBytes + (((2 * ks + half) ^ swizzle<DP>(key)) << 4);
    const int L = lane & 15;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int r = 8 * s + 4 * half + (L >> 2);
        const int chunk = 4 * cb + 2 * ((lane >> 4) & 1) + ((L & 3) >> 1);
        vaddr[cb][s] = r * kRowBytes + ((chunk ^ swizzle<DP>(r)) << 4) + 8 * (L & 1);
      }
  }
  const uint32_t lds0 = uniform((uint32_t)(uintptr_t)(lds_void*)lds);

  DenseSource<DP, WAVES, kStage> dense;
  BlockSource<DP, BF, WAVES, kStage> blocks(p, t.request, h, nk);
  float* lscale = (float*)(lds + 4 * kTileBytes);  // [2][8]
  if constexpr (!BLOCKS) {
    dense.init(p, t, h);
    if (tile_limit > 0) dense.issue(part_first, lds0, lds0 + kTileBytes);
  }

  u32x4 q[KS];
  {
    const char* src = (const char*)p.q + 2 * (qb * p.q_sb + (t.q0 + token) * p.q_st + head * p.q_sh);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int ch = 16 * ks + 8 * half;
      q[ks] = (u32x4){0, 0, 0, 0};
      if (real && ch < p.D) q[ks] = *(const u32x4*)(src + 2 * ch);
    }
    // They are there before the loop: a load that may still be out in it makes the compiler wait in every tile for all
    // memory traffic, the copies among it (a prompt of 16,384 tokens: 2.16 ms, 2.07 with this).
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(q[ks]));
  }
  int32_t* first = (int32_t*)(lds + 4 * kTileBytes + 64);  // [2][DP], of the careful pass
  bool careful = false;  // (the same for the whole workgroup)
  for (;;) {
    m = -3.402823466e38f, l = 0.f;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[cb][i] = 0.f;
    if (tile_limit > 0) {
      if constexpr (BLOCKS) {
        blocks.blocks(part_first);
        blocks.issue(part_first);
        blocks.blocks(part_first + kStage);
        blocks.finish(lds, lds + kTileBytes, lscale);
      } else if (careful) {
        dense.issue(part_first, lds0, lds0 + kTileBytes);
      }
    }
    int buf = 0;
    for (int j = part_first; j < tile_limit; j += kStage) {
      // this wave's copies are done, then everybody's; and everybody has read the other buffer
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const int at = buf * 2 * kTileBytes;
      const float* ls = lscale + 8 * buf + 4 * group;
      buf ^= 1;
      const int next = buf * 2 * kTileBytes;
      const bool more = j + kStage < tile_limit;
      const int jg = j + group * kKeys;  // this wave's keys
      if (more) {
        if constexpr (BLOCKS) {
          blocks.issue(j + kStage);
          blocks.blocks(j + 2 * kStage);
        } else {
          dense.issue(j + kStage, lds0 + next, lds0 + next + kTileBytes);
        }
      }
      if (careful) {
        set_apart<DP, kStage, BF || BLOCKS, 64 * WAVES>(lds + at + kTileBytes, j, first);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
      if (jg < wave_max) {
      const char* lk = lds + at + group * kKeys * kRowBytes;
      const char* lv = lk + kTileBytes;

      f32x16 s[T2];
#pragma unroll
      for (int t2 = 0; t2 < T2; ++t2)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t2][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int t2 = 0; t2 < T2; ++t2)
          s[t2] = mfma32<BF>(*(const u32x4*)(lk + kaddr[ks] + t2 * 32 * kRowBytes), q[ks], s[t2]);
      {  // three steps of operands ahead of the matrix instructions
        constexpr int kMfma = 0x8, kRead = 0x100;
        __builtin_amdgcn_sched_group_barrier(kRead, 3 * T2, 0);
#pragma unroll
        for (int ks = 0; ks < KS - 3; ++ks) {
          __builtin_amdgcn_sched_group_barrier(kMfma, T2, 0);
          __builtin_amdgcn_sched_group_barrier(kRead, T2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, 3 * T2, 0);
      }
      if constexpr (BLOCKS && !BF) {
#pragma unroll
        for (int t2 = 0; t2 < T2; ++t2)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t2][i] *= ls[2 * t2 + i / 8];
      }
      if (jg + kKeys > wave_min) {
#pragma unroll
        for (int t2 = 0; t2 < T2; ++t2)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (jg + 32 * t2 + 8 * (i / 4) + 4 * half + i % 4 >= limit) s[t2][i] = -__builtin_inff();
      }
      float top = s[0][0];  // of this lane's half of the row's keys
#pragma unroll
      for (int t2 = 0; t2 < T2; ++t2)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t2][i]);
      top *= p.c;
      if (__any(top > m + 8.f)) {
        top = fmaxf(top, other_half(top));
        const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - up);
        m = up, l *= f;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[cb][i] *= f;
      }
      constexpr bool kSplit = BLOCKS && !BF;  // p as two bf16 parts: an fp16 result shows one rounding to bf16
      // Step ks: the weights of 16 keys, p = 2^(s c - m) in the operand type, and their products with the values.  A
      // step's matrix instructions run beside the exponentials and the operands' reads of the step after.
      u32x4 pk[2], rest[2], a[2][CB];
      auto values = [&](int ks) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          union {
            short4v part[2];
            u32x4 whole;
          } x;
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2)
            x.part[s2] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_short4*)(lds_void*)(lv + vaddr[cb][s2] + ks * 16 * kRowBytes));
          a[ks & 1][cb] = x.whole;
        }
      };
      float lift = -m;
      if constexpr (!BF && !BLOCKS) lift = 7.f - m;
      auto weights = [&](int ks) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = 8 * (ks % 2) + 2 * i;
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks / 2][at], p.c, lift));
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks / 2][at + 1], p.c, lift));
          l += x, l += y;
          const uint32_t pair = pack2<BF || BLOCKS>(x, y);
          pk[ks & 1][i] = pair;
          if constexpr (kSplit) rest[ks & 1][i] = pack2<true>(x - u2f(pair << 16), y - u2f(pair & 0xffff0000u));
        }
      };
      constexpr bool kAhead = !BLOCKS && DP > 64;  // (not where registers are short: the blocks' loads, three waves a SIMD)
      if constexpr (kAhead) values(0);
      weights(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < 2 * T2; ++ks) {
        if constexpr (!kAhead) values(ks);
        if (ks + 1 < 2 * T2) {
          if constexpr (kAhead) values(ks + 1);
          weights(ks + 1);
        }
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          o[cb] = mfma32<BF || BLOCKS>(a[ks & 1][cb], pk[ks & 1], o[cb]);
          if constexpr (kSplit) o[cb] = mfma32<true>(a[ks & 1][cb], rest[ks & 1], o[cb]);
        }
        if (ks + 1 < 2 * T2) {
          constexpr int kMfma = 0x8, kValu = 0x2, kRead = 0x100;
#pragma unroll
          for (int i = 0; i < CB; ++i) {
            __builtin_amdgcn_sched_group_barrier(kMfma, kSplit ? 2 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
            __builtin_amdgcn_sched_group_barrier(kValu, (kSplit ? 44 : 28) / CB, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      }
      if constexpr (BLOCKS)
        if (more) blocks.finish(lds + next, lds + next + kTileBytes, lscale + 8 * buf);
    }
    if (careful) break;
    float zero = 0.f;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(o[cb][i], 0.f, zero);
    if (!__syncthreads_or(real && zero != 0.f)) break;  // (NaN is not 0)
    careful = true;
    for (int i = threadIdx.x; i < 2 * DP; i += 64 * WAVES) first[i] = 0x7fffffff;
  }

  if constexpr (GROUPS == 2) {
    // the second group's sums through LDS (its stages are no longer used), a register of all lanes at a time
    float* other = (float*)lds + wave * 64 * (16 * CB + 2) + lane;
    __syncthreads();
    if (group == 1) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) other[64 * (16 * cb + i)] = o[cb][i];
      other[64 * 16 * CB] = m, other[64 * (16 * CB + 1)] = l;
    }
    __syncthreads();
    if (group == 1) return;
    const float m1 = other[64 * 16 * CB], up = fmaxf(m, m1);
    const float f0 = __builtin_amdgcn_exp2f(m - up), f1 = __builtin_amdgcn_exp2f(m1 - up);
    m = up, l = l * f0 + other[64 * (16 * CB + 1)] * f1;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[cb][i] = o[cb][i] * f0 + other[64 * (16 * cb + i)] * f1;
  }
  if (careful) {
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int ch = 32 * cb + 8 * (i / 4) + 4 * half + i % 4;
        if (first[ch] < limit) o[cb][i] += __builtin_inff();
        if (first[DP + ch] < limit) o[cb][i] -= __builtin_inff();
      }
  }
  l += other_half(l);
  if (!real) return;
  if (parts.count > 1) {
    const int64_t at = (int64_t)blockIdx.x * BM + wave * 32 + (lane & 31);
    if (half == 0) *(f32x2*)(p.stats + 2 * at) = (f32x2){m, l};
    float* rec = p.records + at * p.D;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ch = 32 * cb + 8 * i + 4 * half;
        if (ch < p.D)
          *(f32x4*)(rec + ch) = (f32x4){o[cb][4 * i], o[cb][4 * i + 1], o[cb][4 * i + 2], o[cb][4 * i + 3]};
      }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* dst = (char*)p.o + 2 * (qb * p.o_sb + (t.q0 + token) * p.o_st + head * p.o_sh);
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ch = 32 * cb + 8 * i + 4 * half;
      const u32x2 w = {pack2<BF>(o[cb][4 * i] * inv, o[cb][4 * i + 1] * inv),
                       pack2<BF>(o[cb][4 * i + 2] * inv, o[cb][4 * i + 3] * inv)};
      if (ch < p.D) *(u32x2*)(dst + 2 * ch) = w;
    }
}

// A part's sum at the weight of its maximum: an infinity stays one however small that is.
__device__ __forceinline__ float weighted(float x, float f) { return __builtin_isfinite(x) ? x * f : x; }

// Joins the parts' records of a tile: a workgroup has 32 of its rows, a wave one at a time.
template <int BM, int KEYS, bool BF, bool BLOCKS>
__global__ void __launch_bounds__(256) prompt_merge(PromptParams p) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int sub = (int)(blockIdx.x % (BM / 32)), h = (int)(blockIdx.x / (BM / 32) % p.H);
  const int64_t index = blockIdx.x / (BM / 32) / p.H;
  Tile t = find_tile<BM, BLOCKS>(p, index);
  if (t.request < 0) return;
  t.request = uniform(t.request), t.tile = uniform(t.tile), t.rows = uniform(t.rows), t.nq = uniform(t.nq);
  t.nk = uniform(t.nk), t.q0 = uniform((uint32_t)t.q0);
  t.tile = (t.rows + BM - 1) / BM - 1 - t.tile;
  const int last_row = min(t.tile * BM + BM, t.rows) - 1;
  int limit = p.causal ? last_row / p.G + 1 + t.nk - t.nq : t.nk;
  limit = limit < 0 ? 0 : limit > t.nk ? t.nk : limit;
  const Parts parts = parts_of(limit, KEYS, p.splits);
  if (parts.count == 1) return;
  const int64_t qb = p.q_starts ? 0 : t.request;
  for (int i = wave; i < 32; i += 4) {
    const int place = sub * 32 + i, row = t.tile * BM + place;
    if (row >= t.rows) return;
    float m = -3.402823466e38f, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int x0 = 0; x0 < parts.count; x0 += 4) {
      f32x2 ml[4], v[4][2];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int part = x0 + x < parts.count ? x0 + x : x0;
        const int64_t at = ((index * p.splits + part) * p.H + h) * BM + place;
        ml[x] = *(const f32x2*)(p.stats + 2 * at);
        if (x0 + x >= parts.count) ml[x] = (f32x2){-__builtin_inff(), 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int ch = 2 * (lane + 64 * c);
          v[x][c] = *(const f32x2*)(p.records + at * p.D + (ch < p.D ? ch : 0));
        }
      }
      float up = m;
#pragma unroll
      for (int x = 0; x < 4; ++x) up = fmaxf(up, ml[x][0]);
      const float f0 = __builtin_amdgcn_exp2f(m - up);
      m = up, l *= f0;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] = weighted(acc[c], f0);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (ml[x][1] == 0.f) continue;  // no key seen
        const float f = __builtin_amdgcn_exp2f(ml[x][0] - up);
        l += ml[x][1] * f;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          acc[2 * c] += weighted(v[x][c][0], f), acc[2 * c + 1] += weighted(v[x][c][1], f);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* dst = (uint16_t*)p.o + qb * p.o_sb + (t.q0 + row / p.G) * p.o_st + (h * p.G + row % p.G) * p.o_sh;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int ch = 2 * (lane + 64 * c);
      if (ch < p.D) *(uint32_t*)(dst + ch) = pack2<BF>(acc[2 * c] * inv, acc[2 * c + 1] * inv);
    }
  }
}

// Parts for a launch of `grid` workgroups over at most `keys` keys, where not every one of 256 CUs has a workgroup: the
// least time in tiles, where a workgroup's start and end cost about as much as four and joining the parts as `join`
// (fewer for blocks, whose tiles are converted and take longer).  `even`: equally long tiles, in whole rounds of the
// card; else about three quarters of the longest's length, and the short fill the gaps that the long leave.
// (Always two workgroups a CU is worse where one round becomes two or three: 2,000 tokens of 16 heads, all seeing all,
// 252 workgroups, 40 us and 66; 300 tokens behind 7,892, head_dim 64, 50 and 71.)
inline int splits_for(int64_t grid, int64_t keys, int tile_keys, bool even, int join) {
  const int64_t n = (keys + tile_keys - 1) / tile_keys;
  int best = 1;
  int64_t least = 0;
  for (int s = 1; s <= 16 && grid < 256 && (s == 1 || n > (int64_t)(s - 1) * kMinPart); ++s) {
    // 256ths of a round
    const int64_t fill = even ? (grid * s + 255) / 256 * 256 : grid * s < 342 ? 256 : grid * s * 3 / 4;
    const int64_t cost = fill * ((n + s - 1) / s + 4) + (s > 1 ? 256 * join : 0);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return best;
}
// Tiles of `bm` rows of R sequences of `rows` rows together, at most.
inline int64_t tiles_of(int64_t rows, int64_t R, int64_t bm) { return (rows + R * (bm - 1)) / bm; }
inline int64_t record_bytes(int64_t grid, int splits, int rows, int64_t D) {
  return splits > 1 ? grid * splits * rows * (D + 2) * 4 : 0;
}

}  // namespace prompt
}  // namespace dkv
