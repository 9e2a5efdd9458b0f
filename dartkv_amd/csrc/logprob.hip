// Log probabilities of given tokens, the entropy and the most likely alternatives of rows of logits, and the gradient
// of the logits (dkv_token_logprobs, dkv_token_logprobs_backward).
//
// With any m, z = (x - m) log2(e), s = sum 2^z and t = sum 2^z z:  log p(v) = (x_v - m) - ln s and
// H = ln s - ln(2) t / s.  One pass: a thread keeps (m, s, t) of what it has read; m is raised to the maximum after 1, 2,
// 4, .. steps, and when s leaves 2^16, by d in units of z: s becomes 2^-d s and t becomes 2^-d (t - d s).  (Beyond, x - m
// and ln s would cancel more digits than m itself has.  So m is not the row's maximum.)  x - m is taken before the factor,
// so a row at the type's lowest value is a row of equals.  Masked logits are -inf, where 2^z z is NaN: steps with one, once
// that shows, and those at a row's ends are computed with z from -200 on.
//
// Alternatives: a wave keeps the 64 largest keys it has seen sorted over its lanes (key: the value in an order of
// integers, then the inverted index, so the lower index wins among equals).  Only what exceeds a bound goes on to a buffer
// in LDS; 64 of them are sorted and merged at once.  The bound is the k-th largest of the lanes' maxima after 1, 2, 4, ..
// steps, or of the keys kept.  Lanes exchange by permutations within the vector unit, not through LDS.
//
// Bound by memory: 4,096 rows of 151,936 in bf16 213 to 218 us (5.7 TB/s), with five alternatives 227 to 246, 8,192 with twenty
// 485 (5.1 TB/s); 4,096 of 32,003 53 us (5.0 TB/s).  Before, by vector instructions: a maximum and a careful product for
// every element 326 us.  64 rows of 151,936 with twenty alternatives take 24 us in 16 parts each, a chain of sorting steps
// and a second launch that joins them.  Nine tenths of 4,096 x 151,936 masked: 293 us in place of 218, with five
// alternatives 329 in place of 227, and 575 where rows begin with the mask: every -inf is a candidate until there are five
// others.
//
// Backward, with g the gradient of the given token's log probability (and of the alternatives', each at its own index),
// G their sum and h the entropy's: dx_v = sum of the g at v - p_v (G + h (log p_v + H)).  One read and one write: 97 us
// for 4,096 rows of 32,003 in bf16 (5.4 TB/s).  Logits that do not begin as their gradient within 16 bytes are read one by
// one (rows cut out of 32,016: 80 us more).
#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "dkv_capi_util.h"
#include "dkv_device.h"

using namespace dkv;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxTop = 64;
constexpr int kPartChunks = 4;  // of a thread, in the smallest part of a row
constexpr int kDeep = 2;  // chunks of 16 bytes a thread computes on, while as many are on their way
constexpr float kLog2E = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

struct LogprobParams {
  const char* logits;
  const void* tokens;
  float *logprobs, *entropy, *stats, *top_logprobs;
  int64_t* top_tokens;
  float* records;      // [rows][splits]: (m, s, t, 0)
  uint64_t* lists;     // [rows][splits][top]
  int64_t stride;      // bytes of a row
  int64_t chunks;      // of a split, a multiple of kThreads
  int32_t V, splits, top, wide;
  uint32_t rows;
};

struct Sums {
  float m, s, t;
};

// (2^z is 0 before z is -200)
__device__ __forceinline__ float finite(float z) { return fmaxf(z, -200.f); }

__device__ __forceinline__ void raise(Sums& a, float m) {
  const float d = fminf((m - a.m) * kLog2E, 300.f), f = __builtin_amdgcn_exp2f(-d);
  a.t = f * (a.t - d * a.s), a.s *= f, a.m = m;
}

__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  raise(a, m), raise(b, m);
  return {m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ Sums wave_join(Sums a) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    a = join(a, {__shfl_xor(a.m, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.t, off, 64)});
  return a;
}

// An order of integers in which NaN is the least (0: nothing) and -0 equals 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = f2u(x + 0.f);
  return x != x ? 0u : (u >> 31 ? ~u : u | 0x80000000u);
}
constexpr uint32_t kLowest = 0x007fffffu;  // of -inf
__device__ __forceinline__ float value_of(uint32_t order) { return u2f(order >> 31 ? order ^ 0x80000000u : ~order); }

__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  const uint32_t order = order_of(x);
  return order ? (uint64_t)order << 32 | (uint32_t)~index : 0;
}

__device__ __forceinline__ uint64_t shuffle(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32 | (uint32_t)__shfl((int)v, lane, 64);
}

// Lane ^ STRIDE's value, without a way through LDS: permutations within four, mirrors and rotations within rows of 16, and
// swaps of rows and halves.
template <int STRIDE>
__device__ __forceinline__ uint32_t across(uint32_t v, int lane) {
  const auto dpp = [](uint32_t x, auto control) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(control)::value, 0xf, 0xf, true);
  };
  if constexpr (STRIDE == 1) return dpp(v, std::integral_constant<int, 0xb1>());
  if constexpr (STRIDE == 2) return dpp(v, std::integral_constant<int, 0x4e>());
  if constexpr (STRIDE == 4)  // lane ^ 7, then ^ 3
    return dpp(dpp(v, std::integral_constant<int, 0x141>()), std::integral_constant<int, 0x1b>());
  if constexpr (STRIDE == 8) return dpp(v, std::integral_constant<int, 0x128>());
  if constexpr (STRIDE == 16) {
    const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? both[0] : both[1];
  }
  if constexpr (STRIDE == 32) {
    const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? both[0] : both[1];
  }
}
template <int STRIDE>
__device__ __forceinline__ uint64_t across(uint64_t v, int lane) {
  return (uint64_t)across<STRIDE>((uint32_t)(v >> 32), lane) << 32 | across<STRIDE>((uint32_t)v, lane);
}

// One step of a sorting network: the larger goes to the lower lane, in lanes with SIZE set to the higher one.
template <int SIZE, int STRIDE, typename T>
__device__ __forceinline__ T exchange(T v, int lane) {
  const T other = across<STRIDE>(v, lane);
  return (v > other) == (((lane & STRIDE) == 0) == ((lane & SIZE) == 0)) ? v : other;
}

template <int SIZE, int STRIDE, typename T>
__device__ __forceinline__ T exchanges(T v, int lane) {
  if constexpr (STRIDE > 0) return exchanges<SIZE, STRIDE / 2>(exchange<SIZE, STRIDE>(v, lane), lane);
  return v;
}

template <typename T, int SIZE = 2>
__device__ __forceinline__ T sort_lanes(T v, int lane) {  // the largest in lane 0
  v = exchanges<SIZE, SIZE / 2>(v, lane);
  if constexpr (SIZE < 64) return sort_lanes<T, 2 * SIZE>(v, lane);
  return v;
}

// The 64 largest of two sorted lists, sorted.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, uint64_t b, int lane) {
  const uint64_t other = shuffle(b, 63 - lane);
  return exchanges<64, 32>(a > other ? a : other, lane);
}

// What a wave keeps of the largest it has seen.
struct Best {
  uint64_t list = 0;   // sorted over the lanes
  uint64_t bound = 0;  // keys up to it are not wanted
  float least = -INFINITY;  // its value
  int waiting = 0;

  __device__ __forceinline__ void raise_bound(uint64_t key) {
    bound = key > bound ? key : bound;
    least = bound ? value_of((uint32_t)(bound >> 32)) : -INFINITY;
  }
  // Every lane with `wanted` adds its key to the buffer of 128, which is merged when it holds 64.
  __device__ __forceinline__ void add(uint64_t key, uint64_t* buffer, int top, int lane) {
    const bool wanted = key > bound;
    const uint64_t mask = __ballot(wanted);
    if (mask == 0) return;
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    if (wanted) buffer[waiting + before] = key;
    waiting += __builtin_popcountll(mask);
    if (waiting >= 64) flush(buffer, top, lane);
  }
  __device__ __forceinline__ void flush(uint64_t* buffer, int top, int lane) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t first = lane < waiting ? buffer[lane] : 0, rest = 64 + lane < waiting ? buffer[64 + lane] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    list = merge_lists(list, sort_lanes(first, lane), lane);
    waiting = waiting > 64 ? waiting - 64 : 0;
    if (lane < waiting) buffer[lane] = rest;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    raise_bound(shuffle(list, top - 1));
  }
};

template <int DT>
struct Chunk {  // 16 bytes of a row
  static constexpr int kElements = DT == kF32 ? 4 : 8;
  static constexpr int kSize = DT == kF32 ? 4 : 2;
  uint32_t w[4];
  // Chunk c of the row that begins `off` elements behind an aligned address; -inf outside the row.
  __device__ __forceinline__ void load(const char* aligned, int64_t c, int off, int64_t V) {
    const int64_t first = c * kElements - off;
    const char* at = aligned + c * 16;
    if (first >= 0 && first + kElements <= V) {
      const uint4 u = *(const uint4*)at;
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = DT == kF32 ? 0xff800000u : DT == kBF16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
      for (int i = 0; i < kElements; ++i) {
        if (first + i < 0 || first + i >= V) continue;
        if (DT == kF32)
          w[i] = *(const uint32_t*)(at + 4 * i);
        else
          w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | (uint32_t) * (const uint16_t*)(at + 2 * i) << 16
                           : (w[i / 2] & 0xffff0000u) | *(const uint16_t*)(at + 2 * i);
      }
    }
  }
  // Element `lane` of lane l's chunk (lanes from kElements on: something else).
  __device__ __forceinline__ float of_lane(int l, int lane) const {
    uint32_t u = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t word = (uint32_t)__builtin_amdgcn_readlane((int)w[i], l);
      if ((DT == kF32 ? lane : lane >> 1) == i) u = word;
    }
    if (DT == kF32) return u2f(u);
    const uint32_t half = lane & 1 ? u >> 16 : u & 0xffffu;
    return DT == kBF16 ? u2f(half << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)half);
  }
  __device__ __forceinline__ float get(int i) const {
    if (DT == kF32) return u2f(w[i]);
    if (DT == kBF16) return u2f(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2]));
  }
};

// A row as a split's wave reads it: kDeep chunks of each lane at a time, a workgroup's chunks next to each other.
template <int DT, int THREADS>  // THREADS: of a row's part
struct Group {
  static constexpr int E = Chunk<DT>::kElements;
  Chunk<DT> chunk[kDeep];
  bool whole;  // for the wave: nothing but the row
  // The group of chunks c + i * THREADS (c: this lane's); what is not the row's or the split's is -inf.
  __device__ __forceinline__ void load(const char* aligned, int64_t c, int lane, int64_t stop, int off, int64_t V) {
    const int64_t first = c - lane, last = first + 63 + (kDeep - 1) * THREADS;
    whole = first * E >= off && last < stop && (last + 1) * E - off <= V;
    if (whole) {
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const uint4 u = *(const uint4*)(aligned + (c + i * THREADS) * 16);
        chunk[i].w[0] = u.x, chunk[i].w[1] = u.y, chunk[i].w[2] = u.z, chunk[i].w[3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const bool in = c + i * THREADS < stop;
        chunk[i].load(aligned, in ? c + i * THREADS : 0, off, in ? V : -1);
      }
    }
  }
  // The registers hold something unknown from here: what was made of them is not kept.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(chunk[i].w[j]));
  }
  __device__ __forceinline__ void largest(float (&top)[kDeep]) const {
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      top[i] = chunk[i].get(0);
#pragma unroll
      for (int j = 1; j < E; ++j) top[i] = fmaxf(top[i], chunk[i].get(j));
    }
  }
  // (A step's terms are added before they come to the others: the entropy of 4,096 x 151,936 is 0.5e-7 off in place of the
  // 3.9e-7 of one long sum, for 1 % of the time.)
  __device__ __forceinline__ void add(Sums& a) const {
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float z = (chunk[i].get(j) - a.m) * kLog2E, e = __builtin_amdgcn_exp2f(z);
        s += e, t = fmaf(e, z, t);
      }
    }
    a.s += s, a.t += t;
  }
  __device__ __forceinline__ void add_careful(Sums& a) const {
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float z = (chunk[i].get(j) - a.m) * kLog2E, e = __builtin_amdgcn_exp2f(z);
        s += e, t = fmaf(e, finite(z), t);
      }
    }
    a.s += s, a.t += t;
  }
};

__device__ __forceinline__ int64_t token_of(const LogprobParams& p, uint32_t row) {
  return p.wide ? ((const int64_t*)p.tokens)[row] : ((const int32_t*)p.tokens)[row];
}

// The results of a row from its sums and the sorted list (a wave).
template <int DT>
__device__ __forceinline__ void finish(const LogprobParams& p, uint32_t row, Sums sums, uint64_t list, int lane) {
  const float ln_s = logf(sums.s);
  const bool empty = sums.s == 0.f;
  if (lane == 0) {
    const int64_t token = token_of(p, row);
    float logp = 0.f;  // (of a negative token)
    if (token >= p.V) {
      logp = __builtin_nanf("");
    } else if (token >= 0) {
      const char* at = p.logits + row * p.stride + token * Chunk<DT>::kSize;
      const float x = dev_load(at, 0, DT);
      logp = empty ? -INFINITY : (x - sums.m) - ln_s;
    }
    p.logprobs[row] = logp;
    p.entropy[row] = empty ? 0.f : ln_s - kLn2 * sums.t / sums.s;
    if (p.stats) p.stats[2 * (int64_t)row] = sums.m, p.stats[2 * (int64_t)row + 1] = log2f(sums.s);
  }
  if (lane < p.top) {
    const int64_t at = (int64_t)row * p.top + lane;
    const float x = value_of((uint32_t)(list >> 32));
    p.top_tokens[at] = list ? (int64_t)(uint32_t)~(uint32_t)list : -1;
    p.top_logprobs[at] = empty ? -INFINITY : list ? (x - sums.m) - ln_s : __builtin_nanf("");
  }
}

// WAVES of a workgroup share a part of a row: all four, or each has a row of its own.
template <int DT, bool TOP, int WAVES>
__global__ void __launch_bounds__(kThreads) logprob_rows(LogprobParams p) {
  constexpr int E = Chunk<DT>::kElements;
  __shared__ Sums wave_sums[kWaves];
  __shared__ uint64_t buffers[TOP ? kWaves : 1][TOP ? 128 : 1];
  __shared__ uint32_t shared_bound;
  constexpr int kPart = 64 * WAVES;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, thread = threadIdx.x & (kPart - 1);
  const uint32_t part = WAVES == 1 ? blockIdx.x * kWaves + wave : blockIdx.x;
  const uint32_t row = part / p.splits, split = part - row * p.splits;
  if (WAVES == 1 && row >= p.rows) return;
  const char* base = p.logits + row * p.stride;
  const int off = (int)((uintptr_t)base & 15) / Chunk<DT>::kSize;
  const char* aligned = base - off * Chunk<DT>::kSize;
  const int64_t all = ((int64_t)p.V + off + E - 1) / E;
  const int64_t stop = (split + 1) * p.chunks < all ? (split + 1) * p.chunks : all;
  uint64_t* buffer = buffers[TOP ? wave : 0];

  Sums sums = {-FLT_MAX, 0.f, 0.f};
  Best best;
  float seen = -INFINITY;  // the largest of this lane
  int steps = 0, refresh = 1;
  if constexpr (TOP) {
    if (WAVES > 1) {
      if (threadIdx.x == 0) shared_bound = 0;
      __syncthreads();
    }
  }
  Group<DT, kPart> next;
  int64_t c0 = split * p.chunks + thread;
  if (c0 - lane < stop) next.load(aligned, c0, lane, stop, off, p.V);
  for (; c0 - lane < stop; c0 += kDeep * kPart) {
    Group<DT, kPart> group = next;
    if (c0 - lane + kDeep * kPart < stop) next.load(aligned, c0 + kDeep * kPart, lane, stop, off, p.V);
    float top[kDeep], most = -INFINITY;
    if constexpr (TOP) {
      group.largest(top);
#pragma unroll
      for (int i = 0; i < kDeep; ++i) most = fmaxf(most, top[i]);
    }
    // Steps 0, 1, 3, 7, .., ends of rows, steps with a -inf and those that s grows too much in take the careful way, which
    // raises m before.  (With the first alone the entropy was 1.4 times as far off.)
    Sums sum = sums;
    bool careful = (steps & (steps + 1)) == 0 || !group.whole;
    if (!careful) {
      group.add(sum);
      careful = !__all(sum.s < 0x1p16f && sum.t == sum.t);
    }
    if (careful) {
      group.forget();
      if constexpr (!TOP) {
        group.largest(top);
#pragma unroll
        for (int i = 0; i < kDeep; ++i) most = fmaxf(most, top[i]);
      }
      if (most > sums.m) raise(sums, most);
      group.add_careful(sums);
    } else {
      sums = sum;
    }
    ++steps;
    if constexpr (TOP) {
      seen = fmaxf(seen, most);
      if (steps == refresh) {  // after 1, 2, 4, .. steps
        // at least top values are as large as the top-th largest of the lanes' maxima, so the row's top-th is; each wave's
        // bound serves the others
        refresh *= 2;
        const uint32_t sorted = sort_lanes(order_of(seen), lane);
        uint32_t kth = (uint32_t)__builtin_amdgcn_readlane((int)sorted, p.top - 1);
        if (WAVES > 1 && lane == 0) kth = max(kth, atomicMax(&shared_bound, kth));
        kth = (uint32_t)__builtin_amdgcn_readfirstlane((int)kth);
        if (kth > kLowest) best.raise_bound(((uint64_t)kth << 32) - 1);
      }
      if (__any(most >= best.least)) {
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
          uint64_t lanes = __ballot(top[i] >= best.least);
          const int64_t c = c0 + i * kPart;
          if (__builtin_popcountll(lanes) > 4) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
              const int64_t index = c * E - off + j;
              const bool real = c < stop && index >= 0 && index < p.V;
              best.add(real ? key_of(group.chunk[i].get(j), (uint32_t)index) : 0, buffer, p.top, lane);
            }
          } else {
            while (lanes) {  // lane j takes element j of that lane's chunk
              const int l = __builtin_ctzll(lanes);
              lanes &= lanes - 1;
              const float x = group.chunk[i].of_lane(l, lane);
              const int64_t from = c - lane + l, index = from * E - off + lane;
              const bool real = lane < E && from < stop && index >= 0 && index < p.V;
              best.add(real ? key_of(x, (uint32_t)index) : 0, buffer, p.top, lane);
            }
          }
        }
      }
    }
  }
  if constexpr (TOP) best.flush(buffer, p.top, lane);
  sums = wave_join(sums);
  if constexpr (WAVES > 1) {
    if constexpr (TOP) buffer[lane] = best.list;
    if (lane == 0) wave_sums[wave] = sums;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      sums = join(sums, wave_sums[w]);
      if constexpr (TOP) best.list = merge_lists(best.list, buffers[w][lane], lane);
    }
  }
  if (p.splits == 1) {
    finish<DT>(p, row, sums, best.list, lane);
  } else {
    if (lane == 0) *(float4*)(p.records + 4 * (int64_t)part) = make_float4(sums.m, sums.s, sums.t, 0.f);
    if (lane < p.top) p.lists[(int64_t)part * p.top + lane] = best.list;
  }
}

// The parts of a row joined by the waves of a workgroup: each takes every WAVES-th part, then they meet in pairs.
template <int DT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) logprob_join(LogprobParams p) {
  __shared__ Sums wave_sums[WAVES];
  __shared__ uint64_t lists[WAVES][64];
  const uint32_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t first = (int64_t)row * p.splits;
  Sums sums = {-FLT_MAX, 0.f, 0.f};
  for (int i = threadIdx.x; i < p.splits; i += 64 * WAVES) {
    const float4 r = *(const float4*)(p.records + 4 * (first + i));
    sums = join(sums, {r.x, r.y, r.z});
  }
  uint64_t list = 0;
  if (p.top)
    for (int i = wave; i < p.splits; i += WAVES)
      list = merge_lists(list, lane < p.top ? p.lists[(first + i) * p.top + lane] : 0, lane);
  sums = wave_join(sums);
  if (lane == 0) wave_sums[wave] = sums;
  if (p.top) {
#pragma unroll
    for (int half = WAVES / 2; half > 0; half /= 2) {
      if (wave >= half && wave < 2 * half) lists[wave][lane] = list;
      __syncthreads();
      if (wave < half) list = merge_lists(list, lists[wave + half][lane], lane);
    }
  } else {
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) sums = join(sums, wave_sums[w]);
  finish<DT>(p, row, sums, list, lane);
}

struct GradParams {
  const char* logits;
  char* out;
  const void* tokens;
  const float *stats, *entropy, *g_logprobs, *g_entropy, *g_top;
  const int64_t* top_tokens;
  int64_t stride, out_stride;  // bytes
  int64_t chunks;
  int32_t V, splits, top, wide;
};

template <int DT>
__global__ void __launch_bounds__(kThreads) logprob_backward(GradParams p) {
  constexpr int E = Chunk<DT>::kElements, kSize = Chunk<DT>::kSize;
  __shared__ float at_value[kMaxTop + 1];
  __shared__ int64_t at_index[kMaxTop + 1];
  const uint32_t row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
  const int64_t token = p.wide ? ((const int64_t*)p.tokens)[row] : ((const int32_t*)p.tokens)[row];
  const float m = p.stats[2 * (int64_t)row], log2_s = p.stats[2 * (int64_t)row + 1];
  const bool empty = log2_s == -INFINITY;
  const float entropy = p.entropy[row], h = p.g_entropy ? p.g_entropy[row] : 0.f;
  const float g = p.g_logprobs && token >= 0 && token < p.V ? p.g_logprobs[row] : 0.f;
  float sum = g;
  if (threadIdx.x == 0) at_index[0] = token, at_value[0] = g;
  if (p.g_top) {
    for (int i = threadIdx.x; i < p.top; i += kThreads) {
      at_index[1 + i] = p.top_tokens[(int64_t)row * p.top + i];
      at_value[1 + i] = p.g_top[(int64_t)row * p.top + i];
    }
  }
  __syncthreads();
  const int points = p.g_top ? 1 + p.top : 1;
  for (int i = 1; i < points; ++i) sum += at_value[i];

  const char* base = p.logits + row * p.stride;
  char* out = p.out + row * p.out_stride;
  const int off = (int)((uintptr_t)out & 15) / kSize;
  const bool alike = (((uintptr_t)base ^ (uintptr_t)out) & 15) == 0;
  const int64_t all = ((int64_t)p.V + off + E - 1) / E;
  const int64_t start = split * p.chunks, stop = start + p.chunks < all ? start + p.chunks : all;
  const auto gradient = [&](float x) {
    const float z = fmaf(x - m, kLog2E, -log2_s), prob = __builtin_amdgcn_exp2f(z);  // log2 p
    return empty ? 0.f : -prob * fmaf(h, fmaf(finite(z), kLn2, entropy), sum);
  };
  for (int64_t c = start + threadIdx.x; c < stop; c += kThreads) {
    const int64_t first = c * E - off;
    float x[E];
    if (alike) {
      Chunk<DT> chunk;
      chunk.load(base - off * kSize, c, off, p.V);
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] = chunk.get(j);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] = first + j >= 0 && first + j < p.V ? dev_load(base, first + j, DT) : -INFINITY;
    }
    if (first >= 0 && first + E <= p.V) {
      uint32_t w[4] = {};
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float y = gradient(x[j]);
        if (DT == kF32) {
          w[j] = f2u(y);
        } else {
          const uint16_t u = DT == kBF16 ? __builtin_bit_cast(uint16_t, (__bf16)y) : __builtin_bit_cast(uint16_t, (_Float16)y);
          w[j / 2] |= (uint32_t)u << (j & 1 ? 16 : 0);
        }
      }
      *(uint4*)(out + first * kSize) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (first + j >= 0 && first + j < p.V) dev_store(out, first + j, gradient(x[j]), DT);
    }
  }
  // the points with a gradient of their own, behind the workgroup's other stores
  __syncthreads();
  const int64_t from = start * E - off, to = stop * E - off;
  for (int i = threadIdx.x; i < points; i += kThreads) {
    const int64_t v = at_index[i];
    if (v < 0 || v >= p.V || v < from || v >= to) continue;
    float delta = 0.f;
    bool again = false;
    for (int j = 0; j < points; ++j) {
      if (at_index[j] != v) continue;
      again |= j < i;  // (the first of equals writes)
      delta += at_value[j];
    }
    if (!again) dev_store(out, v, empty ? 0.f : delta + gradient(dev_load(base, v, DT)), DT);
  }
}

// Rows from which on each has one wave in place of four: 4,096 x 32,003 with twenty alternatives 91 us in place of 120,
// 65,536 x 1,000 42 and 113, 2,048 x 32,000 with five 45 and 45; 1,024 x 151,936, which leave the card half empty, 98 and
// 58.
constexpr int64_t kManyRows = 2048;

// Parts of a row: enough workgroups for the card (four a CU) where there are few rows, none smaller than kPartChunks steps
// of a thread (1,024 x 151,936: 58 us whole, 65 in two parts; 64 with twenty alternatives: 24 in 16 and in 19).
int64_t parts_of(int64_t rows, int64_t V, int64_t dtype, int least) {
  const int64_t E = dtype == kF32 ? 4 : 8, chunks = (V + 2 * E - 1) / E;
  const int64_t most = (chunks + (int64_t)least * kThreads - 1) / ((int64_t)least * kThreads);
  const int64_t want = (1024 + rows - 1) / rows;
  return want < most ? want : most;
}

int64_t chunks_of(int64_t V, int64_t dtype, int64_t parts) {
  const int64_t E = dtype == kF32 ? 4 : 8, chunks = (V + 2 * E - 1) / E;  // (a row may begin within a chunk)
  const int64_t each = (chunks + parts - 1) / parts;
  return (each + kThreads - 1) / kThreads * kThreads;
}

// Rows of a launch.
constexpr int64_t kMaxRows = kGridLimit / 2;

// Rows in several calls of about as many, none of so few that they would be read in parts.
template <typename Call>
int in_turns(const dkv_token_logprobs_args& a, Call call) {
  const int64_t turns = (a.rows + kMaxRows - 1) / kMaxRows, each = (a.rows + turns - 1) / turns;
  const int64_t esize = a.dtype == kF32 ? 4 : 2;
  for (int64_t first = 0; first < a.rows; first += each) {
    dkv_token_logprobs_args part = a;
    part.rows = a.rows - first < each ? a.rows - first : each;
    part.logits = (const char*)a.logits + first * a.stride * esize;
    part.tokens = (const char*)a.tokens + first * (a.wide_tokens ? 8 : 4);
    if (a.logprobs) part.logprobs = a.logprobs + first;
    if (a.entropy) part.entropy = a.entropy + first;
    if (a.stats) part.stats = a.stats + 2 * first;
    if (a.top_logprobs) part.top_logprobs = a.top_logprobs + first * a.top;
    if (a.top_tokens) part.top_tokens = a.top_tokens + first * a.top;
    const int rc = call(part, first);
    if (rc != DKV_OK) return rc;
  }
  return DKV_OK;
}

int check_logprobs(const dkv_token_logprobs_args& a, const char* where) {
  DKV_CHECK(a.dtype == kF32 || a.dtype == kF16 || a.dtype == kBF16, DKV_ERR_DTYPE,
            "%s: logits must be bf16, fp16 or fp32", where);
  DKV_CHECK(a.rows >= 0 && a.rows < (1ll << 31) && a.vocab >= 1 && a.vocab < (1ll << 31) - 64, DKV_ERR_INVALID,
            "%s: bad counts", where);
  DKV_CHECK(a.top >= 0 && a.top <= kMaxTop && a.top <= a.vocab, DKV_ERR_INVALID,
            "%s: top must be at most %d, and at most the row's size", where, kMaxTop);
  return DKV_OK;
}

}  // namespace

extern "C" int64_t dkv_token_logprobs_workspace_bytes(const dkv_token_logprobs_args* args) {
  if (!args || check_logprobs(*args, "dkv_token_logprobs") != DKV_OK || args->rows == 0) return 0;
  const int64_t parts = parts_of(args->rows, args->vocab, args->dtype, kPartChunks);
  return parts == 1 ? 0 : args->rows * parts * (16 + 8 * args->top);
}

extern "C" int dkv_token_logprobs(const dkv_token_logprobs_args* args, void* stream) {
  const char* where = "dkv_token_logprobs";
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "%s: args is NULL", where);
  const dkv_token_logprobs_args& a = *args;
  const int rc = check_logprobs(a, where);
  if (rc != DKV_OK) return rc;
  if (a.rows == 0) return DKV_OK;
  DKV_CHECK(a.logits && a.tokens && a.logprobs && a.entropy && (a.top == 0 || (a.top_logprobs && a.top_tokens)),
            DKV_ERR_INVALID, "%s: NULL pointer", where);
  const int64_t esize = a.dtype == kF32 ? 4 : 2;
  DKV_CHECK(((uintptr_t)a.logits & (esize - 1)) == 0 && a.stride >= 0, DKV_ERR_INVALID, "%s: bad rows", where);
  if (a.rows > kMaxRows)
    return in_turns(a, [&](const dkv_token_logprobs_args& part, int64_t) { return dkv_token_logprobs(&part, stream); });
  LogprobParams p = {};
  p.logits = (const char*)a.logits, p.tokens = a.tokens;
  p.logprobs = a.logprobs, p.entropy = a.entropy, p.stats = a.stats;
  p.top_logprobs = a.top_logprobs, p.top_tokens = a.top_tokens;
  p.stride = a.stride * esize, p.V = (int32_t)a.vocab, p.top = (int32_t)a.top, p.wide = a.wide_tokens != 0;
  p.rows = (uint32_t)a.rows;
  const int64_t parts = parts_of(a.rows, a.vocab, a.dtype, kPartChunks);
  p.splits = (int32_t)parts, p.chunks = chunks_of(a.vocab, a.dtype, parts);
  if (parts > 1) {
    DKV_CHECK(a.workspace && ((uintptr_t)a.workspace & 15) == 0 &&
                  a.workspace_bytes >= dkv_token_logprobs_workspace_bytes(&a),
              DKV_ERR_INVALID, "%s: workspace too small", where);
    p.records = (float*)a.workspace;
    p.lists = (uint64_t*)(p.records + 4 * a.rows * parts);
  }
  const dim3 grid((unsigned)(a.rows * parts)), block(kThreads);
  const hipStream_t s = (hipStream_t)stream;
  const bool alone = parts == 1 && a.rows >= kManyRows;
  const dim3 fewer((unsigned)((a.rows + kWaves - 1) / kWaves));
#define DKV_LOGPROBS(DT)                                                         \
  do {                                                                           \
    if (alone && p.top)                                                          \
      hipLaunchKernelGGL((logprob_rows<DT, true, 1>), fewer, block, 0, s, p);    \
    else if (alone)                                                              \
      hipLaunchKernelGGL((logprob_rows<DT, false, 1>), fewer, block, 0, s, p);   \
    else if (p.top)                                                              \
      hipLaunchKernelGGL((logprob_rows<DT, true, kWaves>), grid, block, 0, s, p);  \
    else                                                                         \
      hipLaunchKernelGGL((logprob_rows<DT, false, kWaves>), grid, block, 0, s, p); \
    if (parts > 1) hipLaunchKernelGGL((logprob_join<DT, 8>), dim3((unsigned)a.rows), dim3(512), 0, s, p); \
  } while (0)
  if (a.dtype == kF32)
    DKV_LOGPROBS(kF32);
  else if (a.dtype == kF16)
    DKV_LOGPROBS(kF16);
  else
    DKV_LOGPROBS(kBF16);
#undef DKV_LOGPROBS
  return dkv_check_launch(where);
}

extern "C" int dkv_token_logprobs_backward(const dkv_token_logprobs_args* args, const dkv_token_logprobs_grads* grads,
                                           void* stream) {
  const char* where = "dkv_token_logprobs_backward";
  DKV_CHECK(args != nullptr && grads != nullptr, DKV_ERR_INVALID, "%s: args is NULL", where);
  const dkv_token_logprobs_args& a = *args;
  const int rc = check_logprobs(a, where);
  if (rc != DKV_OK) return rc;
  if (a.rows == 0) return DKV_OK;
  DKV_CHECK(a.logits && a.tokens && a.stats && a.entropy && grads->out && (!grads->top_logprobs || a.top == 0 || a.top_tokens),
            DKV_ERR_INVALID, "%s: NULL pointer", where);
  const int64_t esize = a.dtype == kF32 ? 4 : 2;
  DKV_CHECK((((uintptr_t)a.logits | (uintptr_t)grads->out) & (esize - 1)) == 0 && a.stride >= 0 &&
                grads->stride >= a.vocab,
            DKV_ERR_INVALID, "%s: bad rows", where);
  if (a.rows > kMaxRows)
    return in_turns(a, [&](const dkv_token_logprobs_args& part, int64_t first) {
      dkv_token_logprobs_grads g = *grads;
      if (g.logprobs) g.logprobs += first;
      if (g.entropy) g.entropy += first;
      if (g.top_logprobs) g.top_logprobs += first * a.top;
      g.out = (char*)g.out + first * g.stride * esize;
      return dkv_token_logprobs_backward(&part, &g, stream);
    });
  GradParams p = {};
  p.logits = (const char*)a.logits, p.out = (char*)grads->out, p.tokens = a.tokens;
  p.stats = a.stats, p.entropy = a.entropy;
  p.g_logprobs = grads->logprobs, p.g_entropy = grads->entropy;
  p.top = (int32_t)a.top, p.g_top = a.top ? grads->top_logprobs : nullptr, p.top_tokens = a.top_tokens;
  p.stride = a.stride * esize, p.out_stride = grads->stride * esize;
  p.V = (int32_t)a.vocab, p.wide = a.wide_tokens != 0;
  const int64_t parts = parts_of(a.rows, a.vocab, a.dtype, 1);
  p.splits = (int32_t)parts, p.chunks = chunks_of(a.vocab, a.dtype, parts);
  const dim3 grid((unsigned)(a.rows * parts)), block(kThreads);
  if (a.dtype == kF32)
    hipLaunchKernelGGL(logprob_backward<kF32>, grid, block, 0, (hipStream_t)stream, p);
  else if (a.dtype == kF16)
    hipLaunchKernelGGL(logprob_backward<kF16>, grid, block, 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(logprob_backward<kBF16>, grid, block, 0, (hipStream_t)stream, p);
  return dkv_check_launch(where);
}
