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
// One launch.  Every workgroup makes the prefix sums over all requests in LDS for itself (8 bytes a request) and
// writes its share of the slots and of the table's rows; what all of them read (lengths, the stack's count) is
// changed by the last workgroup to finish, which the ticket tells.  Bound: the latency of reading the lengths and
// of the ticket's round trip; a second launch for the update would cost as much again.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_capi_util.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 8190;  // prefix sums of 8 bytes a request in 64 KiB of LDS
constexpr int kSlotsPerGroup = 1024;

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

template <bool RESERVE>
__global__ void __launch_bounds__(kThreads) block_tables(TablesParams p) {
  extern __shared__ int64_t sums[];  // [R + 1]: (tokens before) << 32 | blocks before
  __shared__ int64_t wave_sum[4];
  __shared__ int32_t flags, last;
  __shared__ unsigned long long all_tokens, all_blocks;  // the sums' halves may overflow, these do not
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) flags = 0, all_tokens = 0, all_blocks = 0;
  __syncthreads();

  int64_t running = 0, my_tokens = 0, my_blocks = 0;
  int32_t bad = 0;
  for (int base = 0; base < p.R; base += kThreads) {
    const int r = base + tid;
    int64_t x = 0;
    if (r < p.R) {
      const Row row = row_of<RESERVE>(p, r, bad);
      x = ((int64_t)row.moved << 32) + row.count;
      my_tokens += row.moved, my_blocks += row.count;
    }
    int64_t sum = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t up = __shfl_up(sum, off, 64);
      if (lane >= off) sum += up;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int64_t before = running;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += wave_sum[w];
      running += wave_sum[w];
    }
    if (r < p.R) sums[r] = before + sum - x;
    __syncthreads();
  }
  if (tid == 0) sums[p.R] = running;
  if (bad) atomicOr(&flags, bad);
  if (my_tokens) atomicAdd(&all_tokens, (unsigned long long)my_tokens);
  if (my_blocks) atomicAdd(&all_blocks, (unsigned long long)my_blocks);
  const int64_t count = p.state[0];
  __syncthreads();
  bad = flags;
  const int64_t used = (int64_t)all_blocks, moved = (int64_t)all_tokens;
  if (count < 0 || count > p.blocks) bad |= kNoBlocks;
  if (RESERVE && used > count) bad |= kNoBlocks;
  if (!RESERVE && count + used > p.blocks) bad |= kNoBlocks;
  if (RESERVE && moved > p.total) bad |= kBadTotal;
  const bool fits = bad == 0;

  if constexpr (RESERVE) {
    for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i <= p.R; i += (int64_t)gridDim.x * kThreads)
      p.starts[i] = fits ? (int32_t)(sums[i] >> 32) : 0;
    for (int64_t at = (int64_t)blockIdx.x * kSlotsPerGroup + tid; at < p.total; at += (int64_t)gridDim.x * kSlotsPerGroup) {
      const int64_t stop = at - tid + kSlotsPerGroup;
      for (int64_t i = at; i < stop && i < p.total; i += kThreads) {
        int64_t slot = -1;
        if (fits && i < moved) {
          int lo = 0, hi = p.R - 1;  // the last request that starts at or before i
          while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((sums[mid] >> 32) <= i)
              lo = mid;
            else
              hi = mid - 1;
          }
          const int64_t position = p.lengths[lo] + (i - (sums[lo] >> 32));
          const int32_t block = (int32_t)(position >> p.shift);
          const int32_t old = (int32_t)blocks_of(p.lengths[lo], p.shift);
          const int32_t id = block < old ? p.table[(int64_t)lo * p.max_blocks + block]
                                         : p.free[count - 1 - ((int32_t)sums[lo] + block - old)];
          slot = ((int64_t)id << p.shift) + (position & ((1 << p.shift) - 1));
        }
        p.slots[i] = slot;
      }
    }
  }
  // the table's rows, one for each wave in turn
  if (fits) {
    for (int r = blockIdx.x * 4 + wave; r < p.R; r += gridDim.x * 4) {
      const int32_t before = (int32_t)sums[r], n = (int32_t)sums[r + 1] - before;
      if (n == 0) continue;
      int32_t ignored = 0;
      const Row row = row_of<RESERVE>(p, r, ignored);
      int32_t* entry = p.table + (int64_t)r * p.max_blocks + row.old;
      for (int j = lane; j < n; j += 64) {
        if constexpr (RESERVE) {
          entry[j] = p.free[count - 1 - (before + j)];
        } else {
          p.free[count + used - 1 - (before + j)] = entry[j];
          entry[j] = -1;
        }
      }
    }
  }

  // the last workgroup changes what the others read
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(&p.state[2], 1) == (int32_t)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (fits) {
    for (int r = tid; r < p.R; r += kThreads) {
      int32_t n = (int32_t)((sums[r + 1] >> 32) - (sums[r] >> 32));
      if (n) p.lengths[r] += RESERVE ? n : -n;
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
  int64_t groups = (args->total + kSlotsPerGroup - 1) / kSlotsPerGroup;
  groups = groups < 1 ? 1 : groups > 1024 ? 1024 : groups;
  hipLaunchKernelGGL(block_tables<true>, dim3((unsigned)groups), dim3(kThreads), 8 * (p.R + 1), (hipStream_t)stream, p);
  return dkv_check_launch("dkv_reserve_blocks");
}

extern "C" int dkv_release_blocks(const dkv_block_tables_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_release_blocks: args is NULL");
  TablesParams p;
  const int rc = check_tables(*args, "dkv_release_blocks", p);
  if (rc != DKV_OK) return rc;
  int64_t groups = (p.R + 63) / 64;
  groups = groups > 128 ? 128 : groups;
  hipLaunchKernelGGL(block_tables<false>, dim3((unsigned)groups), dim3(kThreads), 8 * (p.R + 1), (hipStream_t)stream, p);
  return dkv_check_launch("dkv_release_blocks");
}
