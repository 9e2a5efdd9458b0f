// Block tables and slot maps of a block cache from its requests' lengths (dkv_reserve_blocks, dkv_release_blocks).
//
// State on the GPU: table [R][max_blocks] (a request's blocks in order, -1 behind the last), lengths [R], the
// free blocks free[0 .. state[0]) as a stack, state[1] the status, state[2] the ticket of a running call.
//
// reserve: request r gets n_r new tokens behind its lengths[r].  With need_r = ceil((len + n) / bs) - ceil(len / bs)
// and P_r, N_r the sums of need and n over the requests before r, its j-th new block is free[state[0] - 1 - (P_r +
// j)] and its i-th new token has slot block * bs + (len + i) % bs at place N_r + i of the slot map.
// release: the last d_r tokens of each request go; its blocks from ceil((len - d) / bs) on return to the stack at
// state[0] + sum(gone) - 1 - (P_r + j): a release of what a reserve gave restores the stack exactly.
//
// One launch.  Every workgroup makes the prefix sums over all requests in LDS for itself (12 bytes a request) and
// writes its share of the slots and of the moved blocks, whose requests it finds in the sums by bisection; what all of
// them read (lengths, the stack's count) is changed by the last workgroup to finish, which the ticket tells.  It needs
// no fence: the others have only read what it changes, and nothing that they wrote is read (with fences a reserve of
// 400,000 slots took 38 us).  Bound: latency, a load of the lengths, one of the blocks and the ticket's round trip after
// each other.  256 requests, a token each: 4.2 us; 128 requests, 400,000 tokens: 10.6 us, their release 5.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_capi_util.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 8190;  // 12 bytes each of 160 KiB of LDS
constexpr int kSlots = 4;  // of a thread, where there are many

struct TablesParams {
  int32_t *table, *lengths, *free, *state;
  const int32_t* tokens;  // [R]; NULL (release): everything
  int64_t* slots;
  int32_t* starts;
  int64_t total, blocks;
  int32_t R, max_blocks, shift;
};

enum : int32_t { kNoBlocks = 1, kRowFull = 2, kBadCount = 4, kBadTotal = 8 };

__device__ __forceinline__ int64_t blocks_of(int64_t tokens, int shift) {
  return (tokens + (1 << shift) - 1) >> shift;
}

struct Row {
  int32_t length, moved, old, count;  // tokens before, tokens added or dropped, first block moved, blocks moved
};

template <bool RESERVE>
__device__ __forceinline__ Row row_of(const TablesParams& p, int r, int32_t& bad) {
  Row x;
  x.length = p.lengths[r];
  const int64_t length = x.length < 0 ? 0 : x.length;
  int64_t n = p.tokens ? p.tokens[r] : length;
  if constexpr (RESERVE) {
    if (n < 0 || x.length < 0) bad |= kBadCount, n = 0;
    if (n > p.total) bad |= kBadTotal, n = 0;
    const int64_t now = blocks_of(length + n, p.shift);
    if (now > p.max_blocks) bad |= kRowFull;
    x.old = (int32_t)blocks_of(length, p.shift);
    x.count = (int32_t)(now - x.old);
  } else {
    n = n < 0 ? 0 : n > length ? length : n;
    x.old = (int32_t)blocks_of(length - n, p.shift);
    x.count = (int32_t)(blocks_of(length, p.shift) - x.old);
    if (x.old + x.count > p.max_blocks) bad |= kRowFull;
  }
  x.moved = (int32_t)n;
  return x;
}

// Prefix sums, of blocks and of tokens; they stop at 2^32 - 1, which is more than any call can have.
struct Sum {
  uint32_t blocks, tokens;
};
__device__ __forceinline__ Sum operator+(Sum a, Sum b) {
  return {__builtin_elementwise_add_sat(a.blocks, b.blocks), __builtin_elementwise_add_sat(a.tokens, b.tokens)};
}

// The last request whose sum is at most i.
template <bool TOKENS>
__device__ __forceinline__ int find(const Sum* sums, int R, uint32_t i) {
  int lo = 0, hi = R - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((TOKENS ? sums[mid].tokens : sums[mid].blocks) <= i)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <bool RESERVE, int SLOTS>  // SLOTS: of a thread
__global__ void __launch_bounds__(kThreads) block_tables(TablesParams p) {
  extern __shared__ Sum sums[];                // [R + 1]: before each request
  int32_t* lens = (int32_t*)(sums + p.R + 1);  // [R]: the lengths before
  __shared__ Sum wave_sum[2][4];
  __shared__ int32_t flags, last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) flags = 0;
  const int64_t count = p.state[0];

  Sum running = {0, 0};
  int32_t bad = 0;
  for (int base = 0; base < p.R; base += kThreads) {
    const int r = base + tid;
    Sum x = {0, 0};
    if (r < p.R) {
      const Row row = row_of<RESERVE>(p, r, bad);
      x = {(uint32_t)row.count, (uint32_t)row.moved};
      lens[r] = row.length;
    }
    Sum sum = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const Sum up = {(uint32_t)__shfl_up((int)sum.blocks, off, 64), (uint32_t)__shfl_up((int)sum.tokens, off, 64)};
      if (lane >= off) sum = sum + up;
    }
    Sum before = {(uint32_t)__shfl_up((int)sum.blocks, 1, 64), (uint32_t)__shfl_up((int)sum.tokens, 1, 64)};
    if (lane == 0) before = {0, 0};
    Sum* wsum = wave_sum[base / kThreads & 1];
    if (lane == 63) wsum[wave] = sum;
    __syncthreads();
    before = before + running;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before = before + wsum[w];
      running = running + wsum[w];
    }
    if (r < p.R) sums[r] = before;
  }
  if (tid == 0) sums[p.R] = running;
  if (bad) atomicOr(&flags, bad);
  __syncthreads();
  bad = flags;
  const int64_t used = running.blocks, moved = running.tokens;
  if (count < 0 || count > p.blocks) bad |= kNoBlocks;
  if (RESERVE && used > count) bad |= kNoBlocks;
  if (!RESERVE && count + used > p.blocks) bad |= kNoBlocks;
  if (RESERVE && moved > p.total) bad |= kBadTotal;
  const bool fits = bad == 0;
  const int64_t me = (int64_t)blockIdx.x * kThreads + tid, all = (int64_t)gridDim.x * kThreads;

  if constexpr (RESERVE) {
    for (int64_t i = me; i <= p.R; i += all) p.starts[i] = fits ? (int32_t)sums[i].tokens : 0;
    const int mask = (1 << p.shift) - 1;
    for (int64_t at = me * SLOTS; at < p.total; at += all * SLOTS) {
      int64_t slot[SLOTS];
      int r = fits && at < moved ? find<true>(sums, p.R, (uint32_t)at) : 0;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        slot[i] = -1;
        if (fits && at + i < moved) {
          if (i > 0)
            while (sums[r + 1].tokens <= at + i) ++r;
          const int64_t position = lens[r] + (at + i - sums[r].tokens);
          const int32_t block = (int32_t)(position >> p.shift), old = (int32_t)blocks_of(lens[r], p.shift);
          const int32_t id = block < old ? p.table[(int64_t)r * p.max_blocks + block]
                                         : p.free[count - 1 - ((int64_t)sums[r].blocks + block - old)];
          slot[i] = ((int64_t)id << p.shift) + (position & mask);
        }
      }
      if (SLOTS > 1 && at + SLOTS <= p.total) {
#pragma unroll
        for (int i = 0; i + 1 < SLOTS; i += 2) *(longlong2*)(p.slots + at + i) = make_longlong2(slot[i], slot[i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
          if (at + i < p.total) p.slots[at + i] = slot[i];
      }
    }
  }
  // the blocks, in the stack's order
  if (fits) {
    for (int64_t i = me; i < used; i += all) {
      const int r = find<false>(sums, p.R, (uint32_t)i);
      const int64_t j = i - sums[r].blocks, length = lens[r];
      const int64_t old = RESERVE ? blocks_of(length, p.shift)
                                  : blocks_of(length - (int64_t)(sums[r + 1].tokens - sums[r].tokens), p.shift);
      int32_t* entry = p.table + (int64_t)r * p.max_blocks + old + j;
      if constexpr (RESERVE) {
        *entry = p.free[count - 1 - i];
      } else {
        p.free[count + used - 1 - i] = *entry;
        *entry = -1;
      }
    }
  }

  // the last workgroup changes what the others read
  __syncthreads();
  if (gridDim.x > 1) {
    if (tid == 0)
      last = __hip_atomic_fetch_add(&p.state[2], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
  }
  if (fits) {
    for (int r = tid; r < p.R; r += kThreads) {
      const int32_t n = (int32_t)(sums[r + 1].tokens - sums[r].tokens);
      if (n) p.lengths[r] = lens[r] + (RESERVE ? n : -n);
    }
    if constexpr (RESERVE)
      for (int64_t i = count - used + tid; i < count; i += kThreads) p.free[i] = -1;
  }
  if (tid == 0) {
    if (fits) p.state[0] = (int32_t)(RESERVE ? count - used : count + used);
    if (bad) p.state[1] |= bad;
    p.state[2] = 0;
  }
}

int check_tables(const dkv_block_tables_args& a, const char* where, TablesParams& p) {
  DKV_CHECK(a.requests >= 1 && a.requests <= kMaxRequests, DKV_ERR_INVALID, "%s: requests must be in 1..%d", where,
            kMaxRequests);
  DKV_CHECK(a.block_size >= 16 && a.block_size <= 256 && (a.block_size & (a.block_size - 1)) == 0, DKV_ERR_INVALID,
            "%s: block_size must be 16, 32, 64, 128 or 256", where);
  DKV_CHECK(a.max_blocks >= 1 && a.max_blocks * a.block_size < (1ll << 31) && a.blocks >= 1 && a.blocks < (1ll << 31),
            DKV_ERR_INVALID, "%s: bad block counts", where);
  DKV_CHECK(a.table && a.lengths && a.free && a.state, DKV_ERR_INVALID, "%s: NULL pointer", where);
  p = {a.table, a.lengths, a.free, a.state, a.tokens, a.slots, a.starts, a.total, a.blocks,
       (int32_t)a.requests, (int32_t)a.max_blocks, __builtin_ctzll((uint64_t)a.block_size)};
  return DKV_OK;
}

}  // namespace

extern "C" int dkv_reserve_blocks(const dkv_block_tables_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_reserve_blocks: args is NULL");
  TablesParams p;
  const int rc = check_tables(*args, "dkv_reserve_blocks", p);
  if (rc != DKV_OK) return rc;
  DKV_CHECK(args->tokens && args->starts && (args->slots || args->total == 0), DKV_ERR_INVALID,
            "dkv_reserve_blocks: NULL pointer");
  DKV_CHECK(args->total >= 0 && args->total < (1ll << 31), DKV_ERR_INVALID, "dkv_reserve_blocks: bad total");
  DKV_CHECK(((uintptr_t)args->slots & 15) == 0, DKV_ERR_INVALID, "dkv_reserve_blocks: slots must be 16-byte aligned");
  const int lds = 12 * p.R + 8;
  if (args->total <= 4 * kThreads) {
    const int64_t groups = args->total > kThreads ? (args->total + kThreads - 1) / kThreads : 1;
    hipLaunchKernelGGL((block_tables<true, 1>), dim3((unsigned)groups), dim3(kThreads), lds, (hipStream_t)stream, p);
  } else {
    int64_t groups = (args->total + kSlots * kThreads - 1) / (kSlots * kThreads);
    groups = groups > 512 ? 512 : groups;
    hipLaunchKernelGGL((block_tables<true, kSlots>), dim3((unsigned)groups), dim3(kThreads), lds, (hipStream_t)stream, p);
  }
  return dkv_check_launch("dkv_reserve_blocks");
}

extern "C" int dkv_release_blocks(const dkv_block_tables_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_release_blocks: args is NULL");
  TablesParams p;
  const int rc = check_tables(*args, "dkv_release_blocks", p);
  if (rc != DKV_OK) return rc;
  int64_t groups = (p.blocks + 4 * kThreads - 1) / (4 * kThreads);  // (at most that many blocks return)
  groups = groups > 16 ? 16 : groups;
  hipLaunchKernelGGL((block_tables<false, 1>), dim3((unsigned)groups), dim3(kThreads), 12 * p.R + 8, (hipStream_t)stream, p);
  return dkv_check_launch("dkv_release_blocks");
}
