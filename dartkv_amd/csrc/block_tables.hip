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
// 400,000 slots took 38 us).  With shares (blocks that several requests hold) a request that writes into a block of others
// gets a copy of it first: of the writers of a block those whose rank among them, in the requests' order, is below the
// block's shares; the last workgroup changes those entries and the shares.  Bound: latency, a load of the lengths, one of
// the blocks and the ticket's round trip after each other.  256 requests, a token each: 4.2 us (10 where all write into
// shared blocks); 128 requests, 400,000 tokens: 10.6 us, their release 5.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkv_block_share.h"
#include "dkv_capi_util.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = dkv::kMaxRequests;  // 12 bytes each of 160 KiB of LDS (16 with shares)
constexpr int kFewWriters = 512;  // requests whose ranks are counted one by one
constexpr int kSlots = 4;  // of a thread, where there are many

struct TablesParams {
  int32_t *table, *lengths, *free, *state;
  const int32_t* tokens;  // [R]; NULL (release): everything
  int64_t* slots;
  int32_t* starts;
  int64_t total, blocks;
  int32_t R, max_blocks, shift;
  int32_t *shares, *copies, *positions;
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

// Sorts `n` keys in LDS, the least first.  Each merge first compares mirrored places, then those `stride` apart, always
// the lesser to the lower place; what lies behind the last would be larger than all, so pairs with it are left out.
__device__ __forceinline__ void sort_keys(uint64_t* keys, int n) {
  for (int size = 1; 1 << (size - 1) < n; ++size) {
    for (int stride = size; stride > 0; --stride) {
      // pair i of the step: the lower place is in the first half of its group of 2^stride
      const int half = 1 << (stride - 1), pairs = (n >> stride) * half + half;
      for (int i = threadIdx.x; i < pairs; i += kThreads) {
        const int group = i >> (stride - 1) << stride, at = i & (half - 1), low = group + at;
        const int high = stride == size ? group + 2 * half - 1 - at : low + half;
        if (high >= n) continue;
        const uint64_t a = keys[low], b = keys[high];
        if (a > b) keys[low] = b, keys[high] = a;
      }
      __syncthreads();
    }
  }
}

// The blocks that requests have to copy: copied[r] is the shared block that request r writes into, or -1 where it does
// not, or is the last of all its holders.  `keys`: LDS of 8 bytes a request.  Many writers' ranks come from sorting them by
// block and request (8,190 requests: a reserve of 395 us in place of 1,600 where each looks at all before it, 1,024: 51 and
// 56; 256 do that in 4).
__device__ __forceinline__ void find_copies(const TablesParams& p, int32_t* copied, uint64_t* keys) {
  static_assert((kMaxRequests + kThreads - 1) / kThreads <= 32, "a bit for each of a thread's requests");
  __shared__ int32_t any;
  if (threadIdx.x == 0) any = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < p.R; r += kThreads) {
    const int32_t length = p.lengths[r], column = length >> p.shift;
    int32_t block = -1;
    if (p.tokens[r] > 0 && length > 0 && (length & ((1 << p.shift) - 1)) != 0 && column < p.max_blocks) {
      block = p.table[(int64_t)r * p.max_blocks + column];
      if (block < 0 || block >= p.blocks || p.shares[block] <= 0) block = -1;
    }
    copied[r] = block;
    keys[r] = block >= 0 ? (uint64_t)(uint32_t)block << 32 | (uint32_t)r : ~0ull;
    if (block >= 0) any = 1;
  }
  __syncthreads();
  if (!any) return;
  if (p.R > kFewWriters) {
    sort_keys(keys, p.R);
    for (int i = threadIdx.x; i < p.R; i += kThreads) {
      const uint64_t key = keys[i];
      if (key == ~0ull) break;
      const uint32_t block = (uint32_t)(key >> 32);
      int lo = 0, hi = i;  // the block's first writer
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if ((uint32_t)(keys[mid] >> 32) < block)
          lo = mid + 1;
        else
          hi = mid;
      }
      if (i - lo >= p.shares[block]) copied[(uint32_t)key] = -1;
    }
    __syncthreads();
    return;
  }
  uint32_t keeps = 0;
  for (int r = threadIdx.x, i = 0; r < p.R; r += kThreads, ++i) {
    const int32_t block = copied[r];
    if (block < 0) continue;
    int32_t rank = 0;
    int q = 0;
#pragma unroll 4
    for (; q + 4 <= r; q += 4) {
      const int4 four = *(const int4*)(copied + q);
      rank += (four.x == block) + (four.y == block) + (four.z == block) + (four.w == block);
    }
    for (; q < r; ++q) rank += copied[q] == block;
    if (rank >= p.shares[block]) keeps |= 1u << i;
  }
  __syncthreads();
  for (int r = threadIdx.x, i = 0; r < p.R; r += kThreads, ++i)
    if (keeps >> i & 1) copied[r] = -1;
  __syncthreads();
}

// The copies, in the requests' order, and the entries and shares that they change.
__device__ __forceinline__ void make_copies(const TablesParams& p, const Sum* sums, const int32_t* lens,
                                            const int32_t* copied, int64_t count, bool fits) {
  __shared__ int32_t wave_count[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int running = 0;
  for (int base = 0; base < p.R; base += kThreads) {
    const int r = base + tid;
    const bool copy = fits && r < p.R && copied[r] >= 0;
    const uint64_t mask = __ballot(copy);
    int32_t* counts = wave_count[base / kThreads & 1];
    if (lane == 0) counts[wave] = __builtin_popcountll(mask);
    __syncthreads();
    int before = running + __builtin_popcountll(mask & ((1ull << lane) - 1));
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += counts[w];
      running += counts[w];
    }
    if (copy) {
      const int32_t id = p.free[count - 1 - sums[r].blocks];
      p.table[(int64_t)r * p.max_blocks + (lens[r] >> p.shift)] = id;
      atomicSub(&p.shares[copied[r]], 1);
      int32_t* entry = p.copies + 3 * (int64_t)before;
      entry[0] = copied[r], entry[1] = id, entry[2] = lens[r] & ((1 << p.shift) - 1);
    }
  }
  for (int i = 3 * running + tid; i < 3 * p.R; i += kThreads) p.copies[i] = -1;
  __syncthreads();  // (the stack is read before it is cleared)
}

template <bool RESERVE, int SLOTS, bool SHARED>  // SLOTS: of a thread
__global__ void __launch_bounds__(kThreads) block_tables(TablesParams p) {
  extern __shared__ __attribute__((aligned(16))) Sum sums[];  // [R + 1]: before each request
  int32_t* lens = (int32_t*)(sums + p.R + 1);  // [R]: the lengths before
  int32_t* copied = lens + p.R;                // [R] (SHARED), 16-byte aligned
  copied += -(2 * (p.R + 1) + p.R) & 3;
  __shared__ Sum wave_sum[2][4];
  __shared__ int32_t flags, last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) flags = 0;
  const int64_t count = p.state[0];

  if constexpr (SHARED) find_copies(p, copied, (uint64_t*)sums);
  Sum running = {0, 0};
  int32_t bad = 0;
  for (int base = 0; base < p.R; base += kThreads) {
    const int r = base + tid;
    Sum x = {0, 0};
    if (r < p.R) {
      const Row row = row_of<RESERVE>(p, r, bad);
      x = {(uint32_t)row.count + (SHARED && copied[r] >= 0), (uint32_t)row.moved};
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
      int32_t place[SLOTS];
      int r = fits && at < moved ? find<true>(sums, p.R, (uint32_t)at) : 0;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        slot[i] = place[i] = -1;
        if (fits && at + i < moved) {
          if (i > 0)
            while (sums[r + 1].tokens <= at + i) ++r;
          const int64_t position = lens[r] + (at + i - sums[r].tokens);
          const int32_t block = (int32_t)(position >> p.shift), old = (int32_t)blocks_of(lens[r], p.shift);
          const int copy = SHARED && copied[r] >= 0;  // (its tokens lie in block old - 1 and those behind it)
          const int32_t id = block < old - copy ? p.table[(int64_t)r * p.max_blocks + block]
                                                : p.free[count - 1 - ((int64_t)sums[r].blocks + block - (old - copy))];
          slot[i] = ((int64_t)id << p.shift) + (position & mask), place[i] = (int32_t)position;
        }
      }
      if (SLOTS > 1 && at + SLOTS <= p.total) {
#pragma unroll
        for (int i = 0; i + 1 < SLOTS; i += 2) *(longlong2*)(p.slots + at + i) = make_longlong2(slot[i], slot[i + 1]);
        if constexpr (SLOTS == 4)
          if (p.positions) *(int4*)(p.positions + at) = make_int4(place[0], place[1], place[2], place[3]);
      } else {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
          if (at + i < p.total) p.slots[at + i] = slot[i];
        if (p.positions) {
#pragma unroll
          for (int i = 0; i < SLOTS; ++i)
            if (at + i < p.total) p.positions[at + i] = place[i];
        }
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
      if (SHARED && copied[r] >= 0 && j == 0) continue;  // (others read that entry)
      int32_t* entry = p.table + (int64_t)r * p.max_blocks + old + j - (SHARED && copied[r] >= 0);
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
  if constexpr (SHARED) make_copies(p, sums, lens, copied, count, fits);
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
  const int rc = dkv::check_block_tables(a, where);
  if (rc != DKV_OK) return rc;
  p = {a.table, a.lengths, a.free, a.state, a.tokens, a.slots, a.starts, a.total, a.blocks,
       (int32_t)a.requests, (int32_t)a.max_blocks, __builtin_ctzll((uint64_t)a.block_size), a.shares, a.copies, a.positions};
  return DKV_OK;
}

template <bool SHARED>
void launch_reserve(const TablesParams& p, hipStream_t stream) {
  const int lds = (SHARED ? 16 : 12) * p.R + (SHARED ? 24 : 8);
  if (p.total <= 4 * kThreads) {
    const int64_t groups = p.total > kThreads ? (p.total + kThreads - 1) / kThreads : 1;
    hipLaunchKernelGGL((block_tables<true, 1, SHARED>), dim3((unsigned)groups), dim3(kThreads), lds, stream, p);
  } else {
    int64_t groups = (p.total + kSlots * kThreads - 1) / (kSlots * kThreads);
    groups = groups > 512 ? 512 : groups;
    hipLaunchKernelGGL((block_tables<true, kSlots, SHARED>), dim3((unsigned)groups), dim3(kThreads), lds, stream, p);
  }
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
  DKV_CHECK((((uintptr_t)args->slots | (uintptr_t)args->positions) & 15) == 0, DKV_ERR_INVALID,
            "dkv_reserve_blocks: slots and positions must be 16-byte aligned");
  if (p.shares) {
    DKV_CHECK(p.copies, DKV_ERR_INVALID, "dkv_reserve_blocks: NULL pointer");
    launch_reserve<true>(p, (hipStream_t)stream);
  } else {
    launch_reserve<false>(p, (hipStream_t)stream);
  }
  return dkv_check_launch("dkv_reserve_blocks");
}

extern "C" int dkv_release_blocks(const dkv_block_tables_args* args, void* stream) {
  DKV_CHECK(args != nullptr, DKV_ERR_INVALID, "dkv_release_blocks: args is NULL");
  TablesParams p;
  const int rc = check_tables(*args, "dkv_release_blocks", p);
  if (rc != DKV_OK) return rc;
  if (args->shares) return dkv::release_shared(*args, (hipStream_t)stream);
  int64_t groups = (p.blocks + 4 * kThreads - 1) / (4 * kThreads);  // (at most that many blocks return)
  groups = groups > 16 ? 16 : groups;
  hipLaunchKernelGGL((block_tables<false, 1, false>), dim3((unsigned)groups), dim3(kThreads), 12 * p.R + 8, (hipStream_t)stream, p);
  return dkv_check_launch("dkv_release_blocks");
}
