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
// of beams) is not counted at all.  A third launch collects what is free and changes the lengths.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_block_share.h"

using namespace dkv;

namespace {

constexpr int kThreads = 256;
constexpr int kCollect = 1024;              // threads of a collecting workgroup
constexpr int kSegment = 16 * 1024;         // blocks that one of them looks through
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

__device__ __forceinline__ void let_go(const ShareParams& p, int32_t block) {
  if (block >= 0 && block < p.blocks) atomicSub(&p.shares[block], 1);
}

// The new rows, and their blocks' new holders.  One row a workgroup of x, columns in turns over y.
__global__ void __launch_bounds__(kThreads) fork_gather(ShareParams p) {
  const int r = blockIdx.x;
  const Change c = change_of<true>(p, r, [&](int i) { return p.lengths[i]; });
  if (c.bad && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(&p.state[1], c.bad);
  if (!c.any) return;
  const int32_t *from = p.table + (int64_t)c.source * p.max_blocks, *mine = p.table + (int64_t)r * p.max_blocks;
  int32_t* to = p.rows + (int64_t)r * p.max_blocks;
  for (int j = blockIdx.y * kThreads + threadIdx.x; j < c.now; j += gridDim.y * kThreads) {
    const int32_t block = from[j];
    to[j] = block;
    if ((j >= c.old || mine[j] != block) && block >= 0 && block < p.blocks) atomicAdd(&p.shares[block], 1);
  }
}

// The rows' new entries; what they held before goes.
template <bool FORK>
__global__ void __launch_bounds__(kThreads) share_apply(ShareParams p) {
  const int r = blockIdx.x;
  const Change c = change_of<FORK>(p, r, [&](int i) { return p.lengths[i]; });
  if (!FORK && c.bad && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(&p.state[1], c.bad);
  if (!c.any) return;
  int32_t* mine = p.table + (int64_t)r * p.max_blocks;
  const int32_t* to = p.rows + (int64_t)r * p.max_blocks;
  const int most = c.old > c.now ? c.old : c.now;
  for (int j = (FORK ? 0 : c.now) + blockIdx.y * kThreads + threadIdx.x; j < most; j += gridDim.y * kThreads) {
    const int32_t before = j < c.old ? mine[j] : -1, now = FORK && j < c.now ? to[j] : -1;
    if (before == now) continue;
    mine[j] = now;
    let_go(p, before);
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

// Free blocks onto the stack, the highest first; the last workgroup changes the stack's count and the lengths.
template <bool FORK>
__global__ void __launch_bounds__(kCollect) share_collect(ShareParams p) {
  extern __shared__ int32_t lens[];  // [R]
  __shared__ int32_t sums[kCollect / 64], last;
  const int tid = threadIdx.x;
  const int64_t count = p.state[0];
  const int64_t start = (int64_t)blockIdx.x * kSegment;
  int64_t above = 0, gone = 0;  // freed blocks of the segments behind this one, and all
  int4 v[kSegment / 4 / kCollect];
  if (p.groups > 1) {
    int part = 0, all = 0, ignored;
    for (int g = tid; g < p.groups; g += kCollect) {
      all += p.counts[g];
      if (g > (int)blockIdx.x) part += p.counts[g];
    }
    above = scan<kCollect>(part, ignored, sums);
    gone = scan<kCollect>(all, ignored, sums);
  }
#pragma unroll
  for (int i = 0; i < kSegment / 4 / kCollect; ++i) v[i] = load_shares(p, start + i * 4 * kCollect + 4 * tid);
  if (p.groups == 1) {
    int n = 0, ignored;
#pragma unroll
    for (const int4& x : v) n += freed(x);
    gone = scan<kCollect>(n, ignored, sums);
  }
  const bool fits = count >= 0 && count + gone <= p.blocks;
#pragma unroll
  for (int i = kSegment / 4 / kCollect - 1; i >= 0; --i) {
    int before;
    const int mine = freed(v[i]);
    const int all = scan<kCollect>(mine, before, sums);
    if (mine) {
      int64_t at = count + above + all - before;  // (behind this thread's place on the stack)
      const int64_t block = start + i * 4 * kCollect + 4 * tid;
      const int32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (x[j] < 0) {
          p.shares[block + j] = 0;
          if (fits) p.free[--at] = (int32_t)(block + j);
        }
      }
    }
    above += all;
  }
  __syncthreads();
  if (p.groups > 1) {
    if (tid == 0)
      last = __hip_atomic_fetch_add(&p.state[2], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.groups - 1;
    __syncthreads();
    if (!last) return;
  }
  for (int r = tid; r < p.R; r += kCollect) lens[r] = p.lengths[r];
  __syncthreads();
  for (int r = tid; r < p.R; r += kCollect) {
    const Change c = change_of<FORK>(p, r, [&](int i) { return lens[i]; });
    if (c.any && c.after != c.before) p.lengths[r] = c.after;
  }
  if (tid == 0) {
    if (fits)
      p.state[0] = (int32_t)(count + gone);
    else
      p.state[1] |= kNoBlocks;
    p.state[2] = 0;
  }
}

// ---- compaction ----

// Which blocks move where, by one workgroup: free ones as bits in LDS, then those above and below the count in use.
// rows[0 ..]: the new number of block n + i at rows[i]; counts[0]: how many move, -1 where the stack is not one.
__global__ void __launch_bounds__(kCollect) compact_plan(ShareParams p) {
  extern __shared__ uint32_t bits[];  // [blocks / 32], set where free
  __shared__ int32_t sums[kCollect / 64], bad;
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
  for (int w = begin; w < end; ++w)
    for (uint32_t x = holes(w); x; x &= x - 1) p.copies[3 * (int64_t)hole_at++ + 1] = w * 32 + __builtin_ctz(x);
  __syncthreads();
  const int32_t size = 1 << p.shift;
  for (int w = begin; w < end; ++w) {
    for (uint32_t x = movers(w); x; x &= x - 1) {
      const int32_t from = w * 32 + __builtin_ctz(x), to = p.copies[3 * (int64_t)mover_at + 1];
      p.copies[3 * (int64_t)mover_at] = from, p.copies[3 * (int64_t)mover_at + 2] = size;
      ++mover_at;
      p.rows[from - used] = to;
      if (p.shares) p.shares[to] = p.shares[from], p.shares[from] = 0;
    }
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

struct CopyParams {
  const int32_t* copies;
  uint8_t *codes[2];
  float* scale[2];
  int64_t stride[2], scale_stride[2];  // of a layer
  int64_t count, blocks;
  int32_t H, bs, D;
};

// One KV head's keys or values of a layer for each workgroup of y, entries x, x + X, .. of 64 X at a time: a lane looks
// at each.
__global__ void __launch_bounds__(kThreads) block_copy(CopyParams p) {
  const int lane = threadIdx.x & 63;
  const uint32_t h = blockIdx.y % p.H, rest = blockIdx.y / p.H, which = rest & 1, layer = rest >> 1;
  const int64_t part = (int64_t)p.bs * p.D;
  uint8_t* codes = p.codes[which] + layer * p.stride[which] + h * part;
  float* scale = p.scale[which] + layer * p.scale_stride[which] + h;
  for (int64_t base = blockIdx.x; base < p.count; base += 64ll * gridDim.x) {
    const int64_t mine = base + (int64_t)lane * gridDim.x;
    int32_t from = -1, to = -1, tokens = 0;
    if (mine < p.count) from = p.copies[3 * mine], to = p.copies[3 * mine + 1], tokens = p.copies[3 * mine + 2];
    uint64_t real = __ballot(from >= 0 && from < p.blocks && to >= 0 && to < p.blocks && from != to);
    while (real) {
      const int l = __builtin_ctzll(real);
      real &= real - 1;
      const int32_t source = __builtin_amdgcn_readlane(from, l), target = __builtin_amdgcn_readlane(to, l);
      const int32_t n = __builtin_amdgcn_readlane(tokens, l);
      const int32_t bytes = (n < 0 ? 0 : n > p.bs ? p.bs : n) * p.D;
      const uint4* src = (const uint4*)(codes + (int64_t)source * p.H * part);
      uint4* dst = (uint4*)(codes + (int64_t)target * p.H * part);
      const int units = bytes / 16;
      for (int i = threadIdx.x; i < units; i += 2 * kThreads) {
        const uint4 a = src[i];
        if (i + kThreads < units) {
          const uint4 b = src[i + kThreads];
          dst[i + kThreads] = b;
        }
        dst[i] = a;
      }
      if (threadIdx.x == 0) scale[(int64_t)target * p.H] = scale[(int64_t)source * p.H];
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

// Columns of a row over workgroups: 2,048 a workgroup.
dim3 row_grid(const ShareParams& p) {
  int64_t y = ((int64_t)p.max_blocks + 8 * kThreads - 1) / (8 * kThreads);
  y = y > 64 ? 64 : y;
  return dim3((unsigned)p.R, (unsigned)y);
}

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
  hipLaunchKernelGGL(share_apply<false>, row_grid(p), dim3(kThreads), 0, stream, p);
  launch_collect<false>(p, stream);
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
  hipLaunchKernelGGL(fork_gather, row_grid(p), dim3(kThreads), 0, s, p);
  hipLaunchKernelGGL(share_apply<true>, row_grid(p), dim3(kThreads), 0, s, p);
  launch_collect<true>(p, s);
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
                2 * a.layers * a.H < 65536,
            DKV_ERR_INVALID, "dkv_copy_blocks: bad counts");
  if (a.count == 0) return DKV_OK;
  DKV_CHECK(a.copies && a.key_codes && a.value_codes && a.key_scale && a.value_scale, DKV_ERR_INVALID,
            "dkv_copy_blocks: NULL pointer");
  DKV_CHECK((((uintptr_t)a.key_codes | (uintptr_t)a.value_codes | (uintptr_t)a.key_stride | (uintptr_t)a.value_stride) & 15) == 0,
            DKV_ERR_INVALID, "dkv_copy_blocks: codes must be 16-byte aligned");
  CopyParams p = {a.copies, {a.key_codes, a.value_codes}, {a.key_scale, a.value_scale}, {a.key_stride, a.value_stride},
                  {a.key_scale_stride, a.value_scale_stride}, a.count, a.blocks, (int32_t)a.H, (int32_t)a.block_size,
                  (int32_t)a.D};
  const int64_t y = 2 * a.layers * a.H;
  int64_t x = 65536 / y < 1 ? 1 : 65536 / y;
  x = x > a.count ? a.count : x;
  hipLaunchKernelGGL(block_copy, dim3((unsigned)x, (unsigned)y), dim3(kThreads), 0, (hipStream_t)stream, p);
  return dkv_check_launch("dkv_copy_blocks");
}
