// Blocks of a block cache that several requests hold: requests that become copies of others, what goes back to the stack,
// blocks that move together, and the copies of their contents (dkv_fork_blocks, dkv_release_blocks with shares,
// dkv_compact_blocks, dkv_copy_blocks).
//
// shares[b] counts the holders of block b beside one, so tables without forks need no more than zeros.  A row that lets go
// of b takes 1 off; b is free when that makes it -1.  Which of several rows does that last is not in one order, that it
// happens is: the freed blocks are then found by looking through the shares, and go onto the stack by their numbers (the
// lowest on top), so results do not depend on the order of the atomics.
//
// fork: rows change all at once, so a first launch gathers the new rows into the workspace and counts their blocks'
// new holders, a second one writes them and takes the old rows' off; an entry that stays the same (the common beginning
// of beams) is not counted at all.  A third launch collects what is free and changes the lengths.  A thread has one column
// of kRows rows, whose loads are all in flight, and counts equal blocks below each other (samples of one prompt) at once:
// 256 rows of 1,000 blocks, 32 of a prompt, released in 10 us (18 with an atomic for each entry) and forked in 15 (21).
// Where the table is small, one workgroup does all of it in one launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_block_share.h"

using namespace dkv;

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 16;                   // of a thread's column
constexpr int kCollect = 1024;              // threads of a collecting workgroup
constexpr int kEach = 16;                   // blocks that one of them looks at
constexpr int kSegment = kEach * kCollect;
constexpr int64_t kSmallTable = 16 * 1024;  // entries
constexpr int64_t kMaxCompact = 1ll << 20;  // blocks: a bit each in LDS

enum : int32_t { kNoBlocks = 1, kRowFull = 2, kBadCount = 4, kBadSource = 16 };

struct ShareParams {
  int32_t *table, *lengths, *free, *state, *shares, *copies;
  const int32_t *sources, *tokens;  // tokens NULL: all
  int32_t *rows, *counts;           // workspace: [R][max_blocks], [groups]
  int64_t blocks;
  int32_t R, max_blocks, shift, groups;
};

__device__ __forceinline__ int32_t blocks_of(int32_t tokens, int shift) {
  return (int32_t)(((int64_t)tokens + (1 << shift) - 1) >> shift);
}

// What a call makes of a row: how many tokens and blocks it had and keeps.
struct Change {
  int32_t source, before, after, old, now, bad;
  bool any;
};

// `length(r)`: a row's length before the call.
template <bool FORK, typename Length>
__device__ __forceinline__ Change change_of(const ShareParams& p, int r, Length length) {
  Change c;
  c.source = FORK ? p.sources[r] : r;
  c.before = length(r);
  c.bad = 0, c.any = false;
  if (FORK && c.source == -1) return c;
  if (FORK && (c.source < 0 || c.source >= p.R)) {
    c.bad = kBadSource;
    return c;
  }
  const int32_t whole = FORK ? length(c.source) : c.before;
  int32_t n = p.tokens ? p.tokens[r] : whole;
  if (c.before < 0 || whole < 0 || (FORK && n < 0)) {
    c.bad = kBadCount;
    return c;
  }
  n = n < 0 ? 0 : n > whole ? whole : n;
  c.after = FORK ? n : whole - n;
  c.old = blocks_of(c.before, p.shift), c.now = blocks_of(c.after, p.shift);
  if (c.old > p.max_blocks || blocks_of(whole, p.shift) > p.max_blocks)
    c.bad = kRowFull;
  else
    c.any = true;
  return c;
}

// What a call makes of kRows rows, from `first` on, in LDS; threads of a column share it.
struct Changes {
  int32_t source[kRows], old[kRows], now[kRows];  // source -1: nothing changes
  template <bool FORK>
  __device__ __forceinline__ void load(const ShareParams& p, int first) {
    const int i = threadIdx.x, r = first + i;
    if (i < kRows) {
      Change c = {};
      if (r < p.R) c = change_of<FORK>(p, r, [&](int q) { return p.lengths[q]; });
      source[i] = c.any ? c.source : -1;
      old[i] = c.any ? c.old : 0, now[i] = c.any ? c.now : 0;
    }
    __syncthreads();
  }
};

// Equal blocks after each other, counted at once.
struct Run {
  int32_t block = -1, count = 0;
  __device__ __forceinline__ void add(const ShareParams& p, int32_t b, int sign) {
    if (b != block) {
      flush(p, sign);
      block = b, count = 0;
    }
    ++count;
  }
  __device__ __forceinline__ void flush(const ShareParams& p, int sign) {
    if (count && block >= 0 && block < p.blocks) atomicAdd(&p.shares[block], sign * count);
    count = 0;
  }
};

// kRows rows a workgroup of x, columns in turns over y.
__global__ void __launch_bounds__(kThreads) fork_gather(ShareParams p) {
  __shared__ Changes rows;
  const int first = blockIdx.x * kRows;
  if (blockIdx.y == 0 && threadIdx.x < kRows && first + (int)threadIdx.x < p.R) {
    const Change c = change_of<true>(p, first + threadIdx.x, [&](int q) { return p.lengths[q]; });
    if (c.bad) atomicOr(&p.state[1], c.bad);
  }
  rows.load<true>(p, first);
  int most = 0;
  for (int i = 0; i < kRows; ++i) most = rows.now[i] > most ? rows.now[i] : most;
  for (int j = blockIdx.y * kThreads + threadIdx.x; j < most; j += gridDim.y * kThreads) {
    int32_t block[kRows], mine[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      block[i] = j < rows.now[i] ? p.table[(int64_t)rows.source[i] * p.max_blocks + j] : -1;
      mine[i] = j < rows.now[i] && j < rows.old[i] ? p.table[(int64_t)(first + i) * p.max_blocks + j] : -1;
    }
    Run run;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (j < rows.now[i]) {
        p.rows[(int64_t)(first + i) * p.max_blocks + j] = block[i];
        if (block[i] != mine[i]) run.add(p, block[i], 1);
      }
    }
    run.flush(p, 1);
  }
}

// The rows' entries as they are now; what they held before goes.
template <bool FORK>
__global__ void __launch_bounds__(kThreads) share_apply(ShareParams p) {
  __shared__ Changes rows;
  const int first = blockIdx.x * kRows;
  if (!FORK && blockIdx.y == 0 && threadIdx.x < kRows && first + (int)threadIdx.x < p.R) {
    const Change c = change_of<FORK>(p, first + threadIdx.x, [&](int q) { return p.lengths[q]; });
    if (c.bad) atomicOr(&p.state[1], c.bad);
  }
  rows.load<FORK>(p, first);
  int begin = FORK ? 0 : p.max_blocks, most = 0;
  for (int i = 0; i < kRows; ++i) {
    const int end = rows.old[i] > rows.now[i] ? rows.old[i] : rows.now[i];
    most = end > most ? end : most;
    if (!FORK && rows.now[i] < rows.old[i]) begin = rows.now[i] < begin ? rows.now[i] : begin;
  }
  for (int j = begin + blockIdx.y * kThreads + threadIdx.x; j < most; j += gridDim.y * kThreads) {
    int32_t before[kRows], now[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t at = (int64_t)(first + i) * p.max_blocks + j;
      const bool gone = j < rows.old[i] && (FORK || j >= rows.now[i]);
      before[i] = gone ? p.table[at] : -1;
      now[i] = FORK && j < rows.now[i] ? p.rows[at] : -1;
    }
    Run run;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (before[i] != now[i]) {
        p.table[(int64_t)(first + i) * p.max_blocks + j] = now[i];
        if (before[i] >= 0) run.add(p, before[i], -1);
      }
    }
    run.flush(p, -1);
  }
}

__device__ __forceinline__ int4 load_shares(const ShareParams& p, int64_t at) {  // (0 behind the last)
  if (at + 4 <= p.blocks) return *(const int4*)(p.shares + at);
  int4 v = {0, 0, 0, 0};
  if (at < p.blocks) v.x = p.shares[at];
  if (at + 1 < p.blocks) v.y = p.shares[at + 1];
  if (at + 2 < p.blocks) v.z = p.shares[at + 2];
  return v;
}

__device__ __forceinline__ int freed(const int4& v) { return (v.x < 0) + (v.y < 0) + (v.z < 0) + (v.w < 0); }

// The sum of `v` over the workgroup's threads, and over those before this one.
template <int THREADS>
__device__ __forceinline__ int scan(int v, int& before, int32_t* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(sum, off, 64);
    if (lane >= off) sum += up;
  }
  __syncthreads();  // (what was in sums has been read)
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  int all = 0;
  before = sum - v;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += sums[w];
    all += sums[w];
  }
  return all;
}

// How many blocks became free in each segment.
__global__ void __launch_bounds__(kCollect) share_count(ShareParams p) {
  __shared__ int32_t sums[kCollect / 64];
  int n = 0, before;
  const int64_t start = (int64_t)blockIdx.x * kSegment;
  for (int i = 0; i < kSegment; i += 4 * kCollect) n += freed(load_shares(p, start + i + 4 * threadIdx.x));
  n = scan<kCollect>(n, before, sums);
  if (threadIdx.x == 0) p.counts[blockIdx.x] = n;
}

// Free blocks of this workgroup's segment onto the stack, the highest first; returns how many became free in all, and
// whether the stack has room for them.
__device__ __forceinline__ int64_t collect(const ShareParams& p, int64_t count, int32_t* sums, bool& fits) {
  const int tid = threadIdx.x;
  const int64_t start = (int64_t)blockIdx.x * kSegment;
  int64_t above = 0, gone = 0;  // freed blocks of the segments behind this one, and all
  int4 v[kEach / 4];
  if (p.groups > 1) {
    int part = 0, all = 0, ignored;
    for (int g = tid; g < p.groups; g += kCollect) {
      all += p.counts[g];
      if (g > (int)blockIdx.x) part += p.counts[g];
    }
    above = scan<kCollect>(part, ignored, sums);
    gone = scan<kCollect>(all, ignored, sums);
  }
  int mine = 0, before;
#pragma unroll
  for (int i = 0; i < kEach / 4; ++i) v[i] = load_shares(p, start + kEach * tid + 4 * i);
#pragma unroll
  for (const int4& x : v) mine += freed(x);
  const int all = scan<kCollect>(mine, before, sums);
  if (p.groups == 1) gone = all;
  fits = count >= 0 && count + gone <= p.blocks;
  if (mine) {
    int64_t at = count + above + all - before;  // (behind this thread's place on the stack)
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) {
      const int32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t block = start + kEach * tid + 4 * i + j;
        if (x[j] < 0) {
          p.shares[block] = 0;
          if (fits) p.free[--at] = (int32_t)block;
        }
      }
    }
  }
  return gone;
}

// The lengths and the stack's count, by one workgroup behind everything else; lens: the lengths before.
template <bool FORK>
__device__ __forceinline__ void settle(const ShareParams& p, const int32_t* lens, int64_t count, int64_t gone, bool fits) {
  for (int r = threadIdx.x; r < p.R; r += kCollect) {
    const Change c = change_of<FORK>(p, r, [&](int i) { return lens[i]; });
    if (c.any && c.after != c.before) p.lengths[r] = c.after;
  }
  if (threadIdx.x == 0) {
    if (fits)
      p.state[0] = (int32_t)(count + gone);
    else
      p.state[1] |= kNoBlocks;
    p.state[2] = 0;
  }
}

// The last workgroup changes the stack's count and the lengths.
template <bool FORK>
__global__ void __launch_bounds__(kCollect) share_collect(ShareParams p) {
  extern __shared__ int32_t lens[];  // [R]
  __shared__ int32_t sums[kCollect / 64], last;
  const int64_t count = p.state[0];
  bool fits;
  const int64_t gone = collect(p, count, sums, fits);
  __syncthreads();
  if (p.groups > 1) {
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(&p.state[2], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.groups - 1;
    __syncthreads();
    if (!last) return;
  }
  for (int r = threadIdx.x; r < p.R; r += kCollect) lens[r] = p.lengths[r];
  __syncthreads();
  settle<FORK>(p, lens, count, gone, fits);
}

// All of it by one workgroup, where table and pool are small: a thread's entries stay in registers, and the order of what
// is added and taken off does not matter before the shares are looked through.
template <bool FORK>
__global__ void __launch_bounds__(kCollect) share_small(ShareParams p) {
  extern __shared__ int32_t lens[];  // [R], then what the rows become: [R] sources, old and new blocks
  __shared__ int32_t sums[kCollect / 64];
  int32_t *source = lens + p.R, *old = source + p.R, *now = old + p.R;
  const int tid = threadIdx.x;
  const int64_t count = p.state[0];
  for (int r = tid; r < p.R; r += kCollect) lens[r] = p.lengths[r];
  __syncthreads();
  for (int r = tid; r < p.R; r += kCollect) {
    const Change c = change_of<FORK>(p, r, [&](int i) { return lens[i]; });
    if (c.bad) atomicOr(&p.state[1], c.bad);
    source[r] = c.any ? c.source : -1, old[r] = c.any ? c.old : 0, now[r] = c.any ? c.now : 0;
  }
  __syncthreads();
  constexpr int kEntries = kSmallTable / kCollect;
  const uint32_t entries = (uint32_t)p.R * p.max_blocks;
  int32_t before[kEntries], after[kEntries];
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    before[i] = after[i] = -1;
    const uint32_t at = tid + i * kCollect, r = at / p.max_blocks, j = at - r * p.max_blocks;
    if (at < entries) {
      if ((int)j < old[r] && (FORK || (int)j >= now[r])) before[i] = p.table[at];
      if (FORK && (int)j < now[r]) after[i] = p.table[(int64_t)source[r] * p.max_blocks + j];
    }
  }
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    if (before[i] == after[i]) continue;
    if (after[i] >= 0 && after[i] < p.blocks) atomicAdd(&p.shares[after[i]], 1);
    if (before[i] >= 0 && before[i] < p.blocks) atomicSub(&p.shares[before[i]], 1);
  }
  __threadfence();  // (the shares are read by other threads)
  __syncthreads();  // (and the table has been read)
#pragma unroll
  for (int i = 0; i < kEntries; ++i)
    if (before[i] != after[i]) p.table[tid + i * kCollect] = after[i];
  bool fits;
  const int64_t gone = collect(p, count, sums, fits);
  settle<FORK>(p, lens, count, gone, fits);
}

// ---- compaction ----

// Which blocks move where, by one workgroup: free ones as bits in LDS, then those above and below the count in use.
// rows[0 ..]: the new number of block n + i at rows[i]; counts[0]: how many move, -1 where the stack is not one.
__global__ void __launch_bounds__(kCollect) compact_plan(ShareParams p) {
  extern __shared__ uint32_t bits[];  // [blocks / 32], set where free
  __shared__ int32_t sums[kCollect / 64], hole_before[kCollect], mover_before[kCollect], bad;
  const int tid = threadIdx.x;
  const int64_t count = p.state[0], blocks = p.blocks;
  const int words = (int)((blocks + 31) / 32);
  if (tid == 0) bad = count < 0 || count > blocks;
  for (int i = tid; i < words; i += kCollect) bits[i] = 0;
  __syncthreads();
  if (!bad) {
    for (int64_t i = tid; i < count; i += kCollect) {
      const int32_t block = p.free[i];
      if (block < 0 || block >= blocks)
        bad = 1;
      else
        atomicOr(&bits[block >> 5], 1u << (block & 31));
    }
  }
  __syncthreads();
  const int64_t used = blocks - count;
  // each thread's words: bits of free blocks below `used`, of used ones from there on
  const int each = (words + kCollect - 1) / kCollect, begin = tid * each, end = begin + each < words ? begin + each : words;
  const auto holes = [&](int w) {
    const int64_t first = (int64_t)w * 32;
    return first >= used ? 0u : first + 32 <= used ? bits[w] : bits[w] & ((1u << (used - first)) - 1);
  };
  const auto movers = [&](int w) {
    const int64_t first = (int64_t)w * 32;
    if (first + 32 <= used) return 0u;
    uint32_t x = ~bits[w];
    if (first < used) x &= ~((1u << (used - first)) - 1);
    if (first + 32 > blocks) x &= (1u << (blocks - first)) - 1;
    return x;
  };
  int n_holes = 0, n_movers = 0, hole_at, mover_at;
  if (!bad) {
    for (int w = begin; w < end; ++w) n_holes += __builtin_popcount(holes(w)), n_movers += __builtin_popcount(movers(w));
  }
  const int all_holes = scan<kCollect>(n_holes, hole_at, sums), all_movers = scan<kCollect>(n_movers, mover_at, sums);
  const bool fits = !bad && all_holes == all_movers;
  if (tid == 0) {
    p.counts[0] = fits ? all_movers : -1;
    if (!fits) p.state[1] |= kNoBlocks;
  }
  if (!fits) return;
  // (at most half of the blocks move: fewer are in use above the count than are free below it)
  hole_before[tid] = hole_at, mover_before[tid] = mover_at;
  __syncthreads();
  // the place of `block` among the bits of its kind
  const auto rank = [&](int64_t block, const int32_t* before, auto bits_of) {
    const int word = (int)(block >> 5), owner = word / each;
    int n = before[owner] + __builtin_popcount(bits_of(word) & ((1u << (block & 31)) - 1));
    for (int w = owner * each; w < word; ++w) n += __builtin_popcount(bits_of(w));
    return n;
  };
  for (int64_t block = tid; block < used && all_holes; block += kCollect)
    if (bits[block >> 5] >> (block & 31) & 1) p.copies[3 * (int64_t)rank(block, hole_before, holes) + 1] = (int32_t)block;
  __threadfence();
  __syncthreads();
  for (int64_t block = used + tid; block < blocks && all_movers; block += kCollect) {
    if (bits[block >> 5] >> (block & 31) & 1) continue;
    int32_t* entry = p.copies + 3 * (int64_t)rank(block, mover_before, movers);
    const int32_t to = entry[1];
    entry[0] = (int32_t)block, entry[2] = 1 << p.shift;
    p.rows[block - used] = to;
    if (p.shares) p.shares[to] = p.shares[block], p.shares[block] = 0;
  }
}

// Tables, stack and the copies' end follow.
__global__ void __launch_bounds__(kThreads) compact_apply(ShareParams p) {
  const int64_t me = (int64_t)blockIdx.x * kThreads + threadIdx.x, all = (int64_t)gridDim.x * kThreads;
  const int32_t moved = p.counts[0];
  const int64_t listed = p.blocks / 2, from = moved < 0 ? 0 : moved;
  for (int64_t i = 3 * from + me; i < 3 * listed; i += all) p.copies[i] = -1;
  if (moved < 0) return;
  const int64_t count = p.state[0], used = p.blocks - count;
  for (int64_t i = me; i < count; i += all) p.free[i] = (int32_t)(p.blocks - 1 - i);
  const int64_t entries = (int64_t)p.R * p.max_blocks;
  for (int64_t i = me; i < entries; i += all) {
    const int32_t block = p.table[i];
    if (block >= used && block < p.blocks) p.table[i] = p.rows[block - used];
  }
}

// ---- copies of blocks ----

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CopyParams {
  const int32_t* copies;
  uint8_t *codes[2];
  float* scale[2];
  int64_t stride[2], scale_stride[2];  // of a layer
  int64_t count, blocks;
  int32_t H, bs, D, heads;
  uint32_t across;
};

// Workgroup x + p.across * y: p.heads KV heads' keys or values of a layer for each y, entries x, x + p.across, .. of
// 64 p.across at a time: a lane looks at each.
__global__ void __launch_bounds__(kThreads) block_copy(CopyParams p) {
  const int lane = threadIdx.x & 63;
  const uint32_t pieces = (p.H + p.heads - 1) / p.heads;
  const uint32_t y = blockIdx.x / p.across, x = blockIdx.x - y * p.across;
  const uint32_t piece = y % pieces, rest = y / pieces, which = rest & 1, layer = rest >> 1;
  const int first = piece * p.heads, heads = p.H - first < p.heads ? p.H - first : p.heads;
  const int64_t part = (int64_t)p.bs * p.D;
  uint8_t* codes = p.codes[which] + layer * p.stride[which] + first * part;
  float* scale = p.scale[which] + layer * p.scale_stride[which] + first;
  for (int64_t base = x; base < p.count; base += 64ll * p.across) {
    const int64_t mine = base + (int64_t)lane * p.across;
    int32_t from = -1, to = -1, tokens = 0;
    if (mine < p.count) from = p.copies[3 * mine], to = p.copies[3 * mine + 1], tokens = p.copies[3 * mine + 2];
    uint64_t real = __ballot(from >= 0 && from < p.blocks && to >= 0 && to < p.blocks && from != to);
    while (real) {
      const int l = __builtin_ctzll(real);
      real &= real - 1;
      const int64_t source = __builtin_amdgcn_readlane(from, l), target = __builtin_amdgcn_readlane(to, l);
      const int32_t n = __builtin_amdgcn_readlane(tokens, l);
      const uint32_t units = (uint32_t)(n < 0 ? 0 : n > p.bs ? p.bs : n) * p.D / 16, all = units * heads;
      const char* src = (const char*)codes + source * p.H * part;
      char* dst = (char*)codes + target * p.H * part;
      if ((int)threadIdx.x < heads) scale[target * p.H + threadIdx.x] = scale[source * p.H + threadIdx.x];
      constexpr int kDeep = 8;
      for (uint32_t i = threadIdx.x; i < all; i += kDeep * kThreads) {
        u32x4 data[kDeep];
        uint32_t at[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
          const uint32_t u = i + k * kThreads, h = u / units;
          at[k] = h * (uint32_t)part + (u - h * units) * 16;
          if (u < all) data[k] = *(const u32x4*)(src + at[k]);
        }
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
          if (i + k * kThreads < all) *(u32x4*)(dst + at[k]) = data[k];
      }
    }
  }
}

int64_t groups_of(int64_t blocks) { return (blocks + kSegment - 1) / kSegment; }

int64_t rows_bytes(const dkv_block_tables_args& a) {
  const int64_t entries = a.requests * a.max_blocks, most = entries > a.blocks ? entries : a.blocks;
  return (4 * most + 15) / 16 * 16;
}

int share_params(const dkv_block_tables_args& a, const char* where, ShareParams& p) {
  const int rc = check_block_tables(a, where);
  if (rc != DKV_OK) return rc;
  DKV_CHECK(a.workspace && ((uintptr_t)a.workspace & 15) == 0 && a.workspace_bytes >= dkv_share_workspace_bytes(&a),
            DKV_ERR_INVALID, "%s: workspace too small", where);
  DKV_CHECK(((uintptr_t)a.shares & 15) == 0, DKV_ERR_INVALID, "%s: shares must be 16-byte aligned", where);
  p = {};
  p.table = a.table, p.lengths = a.lengths, p.free = a.free, p.state = a.state, p.shares = a.shares;
  p.copies = a.copies, p.sources = a.sources, p.tokens = a.tokens;
  p.rows = (int32_t*)a.workspace;
  p.counts = (int32_t*)((char*)a.workspace + rows_bytes(a));
  p.blocks = a.blocks, p.R = (int32_t)a.requests, p.max_blocks = (int32_t)a.max_blocks;
  p.shift = __builtin_ctzll((uint64_t)a.block_size);
  p.groups = (int32_t)groups_of(a.blocks);
  return DKV_OK;
}

dim3 row_grid(const ShareParams& p) {
  const int64_t x = (p.R + kRows - 1) / kRows;
  int64_t y = ((int64_t)p.max_blocks + kThreads - 1) / kThreads;
  const int64_t most = 4096 / x;  // workgroups of columns that no row has end at once, but are not free
  y = y > most ? most : y;
  return dim3((unsigned)x, (unsigned)y);
}

// One workgroup does everything where tables and pool are few, as the launches then cost more than their work: a step of
// 64 beams of 63 blocks (release, fork, reserve, copy) 36 us, 28 of them kernels, and 42 with three launches in place of one.
bool small(const ShareParams& p) { return (int64_t)p.R * p.max_blocks <= kSmallTable && p.groups == 1; }

template <bool FORK>
void launch_collect(const ShareParams& p, hipStream_t stream) {
  if (p.groups > 1) hipLaunchKernelGGL(share_count, dim3(p.groups), dim3(kCollect), 0, stream, p);
  hipLaunchKernelGGL(share_collect<FORK>, dim3(p.groups), dim3(kCollect), 4 * p.R, stream, p);
}

}  // namespace

namespace dkv {

int release_shared(const dkv_block_tables_args& args, hipStream_t stream) {
  ShareParams p;
  const int rc = share_params(args, "dkv_release_blocks", p);
  if (rc != DKV_OK) return rc;
  if (small(p)) {
    hipLaunchKernelGGL(share_small<false>, dim3(1), dim3(kCollect), 16 * p.R, stream, p);
  } else {
    hipLaunchKernelGGL(share_apply<false>, row_grid(p), dim3(kThreads), 0, stream, p);
    launch_collect<false>(p, stream);
  }
  return dkv_check_launch("dkv_release_blocks");
}

}  // namespace dkv

extern "C" int64_t dkv_share_workspace_bytes(const dkv_block_tables_args* args) {
  if (!args || args->requests < 1 || args->max_blocks < 1 || args->blocks < 1) return 0;
  return rows_bytes(*args) + 4 * groups_of(args->blocks);
}

extern "C" int dkv_fork_blocks(const dkv_block_tables_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_fork_blocks: args is NULL");
  ShareParams p;
  const int rc = share_params(*args, "dkv_fork_blocks", p);
  if (rc != DKV_OK) return rc;
  DKV_CHECK(p.shares && p.sources, DKV_ERR_INVALID, "dkv_fork_blocks: NULL pointer");
  const hipStream_t s = (hipStream_t)stream;
  if (small(p)) {
    hipLaunchKernelGGL(share_small<true>, dim3(1), dim3(kCollect), 16 * p.R, s, p);
  } else {
    hipLaunchKernelGGL(fork_gather, row_grid(p), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL(share_apply<true>, row_grid(p), dim3(kThreads), 0, s, p);
    launch_collect<true>(p, s);
  }
  return dkv_check_launch("dkv_fork_blocks");
}

extern "C" int dkv_compact_blocks(const dkv_block_tables_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_compact_blocks: args is NULL");
  ShareParams p;
  const int rc = share_params(*args, "dkv_compact_blocks", p);
  if (rc != DKV_OK) return rc;
  DKV_CHECK(p.copies || args->blocks < 2, DKV_ERR_INVALID, "dkv_compact_blocks: NULL pointer");
  DKV_CHECK(args->blocks <= kMaxCompact, DKV_ERR_UNSUPPORTED, "dkv_compact_blocks: at most %lld blocks",
            (long long)kMaxCompact);
  const hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(compact_plan, dim3(1), dim3(kCollect), 4 * ((args->blocks + 31) / 32), s, p);
  const int64_t entries = args->requests * args->max_blocks, most = entries > 2 * args->blocks ? entries : 2 * args->blocks;
  int64_t groups = (most + 4 * kThreads - 1) / (4 * kThreads);
  groups = groups > 2048 ? 2048 : groups;
  hipLaunchKernelGGL(compact_apply, dim3((unsigned)groups), dim3(kThreads), 0, s, p);
  return dkv_check_launch("dkv_compact_blocks");
}

extern "C" int dkv_copy_blocks(const dkv_copy_blocks_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_copy_blocks: args is NULL");
  const dkv_copy_blocks_args& a = *args;
  DKV_CHECK(a.block_size >= 16 && a.block_size <= 256 && (a.block_size & (a.block_size - 1)) == 0, DKV_ERR_INVALID,
            "dkv_copy_blocks: block_size must be 16, 32, 64, 128 or 256");
  DKV_CHECK(a.D >= 16 && a.D <= 512 && a.D % 16 == 0, DKV_ERR_INVALID,
            "dkv_copy_blocks: head_dim must be a multiple of 16 up to 512");
  DKV_CHECK(a.count >= 0 && a.layers >= 1 && a.blocks >= 1 && a.blocks < (1ll << 31) && a.H >= 1 &&
                a.layers < (1 << 20) && a.H < (1 << 20) && 2 * a.layers * a.H < (1ll << 30),
            DKV_ERR_INVALID, "dkv_copy_blocks: bad counts");
  if (a.count == 0) return DKV_OK;
  DKV_CHECK(a.copies && a.key_codes && a.value_codes && a.key_scale && a.value_scale, DKV_ERR_INVALID,
            "dkv_copy_blocks: NULL pointer");
  DKV_CHECK((((uintptr_t)a.key_codes | (uintptr_t)a.value_codes | (uintptr_t)a.key_stride | (uintptr_t)a.value_stride) & 15) == 0,
            DKV_ERR_INVALID, "dkv_copy_blocks: codes must be 16-byte aligned");
  CopyParams p = {a.copies, {a.key_codes, a.value_codes}, {a.key_scale, a.value_scale}, {a.key_stride, a.value_stride},
                  {a.key_scale_stride, a.value_scale_stride}, a.count, a.blocks, (int32_t)a.H, (int32_t)a.block_size,
                  (int32_t)a.D, 1, 1};
  // 32 KiB of a whole block for a workgroup (at most kThreads heads, whose scales its threads copy)
  const int64_t heads = 32768 / (a.block_size * a.D);
  p.heads = (int32_t)(heads < 1 ? 1 : heads > a.H ? a.H : heads);
  const int64_t y = 2 * a.layers * ((a.H + p.heads - 1) / p.heads);
  int64_t x = 65536 / y < 1 ? 1 : 65536 / y;
  x = x > a.count ? a.count : x;
  DKV_CHECK(x * y < kGridLimit, DKV_ERR_INVALID, "dkv_copy_blocks: too many layers and heads");
  p.across = (uint32_t)x;
  hipLaunchKernelGGL(block_copy, dim3((unsigned)(x * y)), dim3(kThreads), 0, (hipStream_t)stream, p);
  return dkv_check_launch("dkv_copy_blocks");
}
