// Requests that share pool slots, and the moving of slots (gfx950): new requests over the slots of another or over copies of them, the release of
// requests' tokens, and compaction.  No counterpart in the reference, whose slots have reference counts too (loongserve/common/longserve_mem_manager.py:61-88) but whose
// lists count a slot that is named twice once, so that requests that share tokens cannot be freed together.
//
// All of it is whole numbers and rows as bytes.  What bounds it: rows, HBM (two copies of 6500 tokens in 32 layers of 8 heads of 128, 3.3 GB there and back, 533 us, 6.2 TB/s, in 8 bits
// with their exponents 302, 5.7; half of 60000 slots in use, 12 layers, compacted: 1.43 GB, 306 us, 4.7 TB/s, a large copy's rate); the rest, launch latency and a few MB of tables and counts
// (eight forks of 2999 tokens 3.7 us, a release of 100 tokens 2.4 and of 128 requests 11.4 + 3.8, the plan of a compaction 5.3 for 5000 slots and 10.4 for 60000).  Counts change by integer atomics, whose order does not change a result.
#include "common.hip.h"

namespace lsattn {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kCUs = 256;

// ------------------------------------------------------------------------------------------------ fork
struct ForkParams {
  int32_t* table;
  int64_t max_seq_len;
  int32_t most;  // positions that the call takes of a request: max_len_in_batch, at most max_seq_len
  const int32_t* src;
  const int32_t* dst;
  const int32_t* len;
  int32_t n, num_reqs;
  int32_t* state;
  int32_t size;
};
__device__ __forceinline__ int fork_len(const ForkParams& p, int i) {
  const int n = p.len[i];
  return p.dst[i] < 0 || p.dst[i] >= p.num_reqs ? 0 : n < p.most ? n : p.most;
}
constexpr int kNoSlot = 0x7fffffff;  // as the table's unused entries
// A thread has a position of a fork.  Forks of one request that stand next to each other count as one addition per token, made by the first of them: many samples of one
// question would otherwise queue at the same words.  Positions of a source that is no row of the table name no slot: what the fork's row held before may be others' tokens by now.
// Nor do those whose slot is free: nobody holds it, and a count that began here would be one that the allocator's number of free slots has not seen.  (Counts that are not zero stay so within the
// call, and zeros stay zeros, so that it does not matter when a thread looks.)
__global__ __launch_bounds__(kThreads) void fork_share_kernel(ForkParams p) {
  const int i = blockIdx.y, pos = (int)(blockIdx.x * kThreads + threadIdx.x), lane = threadIdx.x & 63;
  const int src = p.src[i], mine = fork_len(p, i);
  int slot = -1;
  const bool valid_src = src >= 0 && src < p.num_reqs;
  const bool leads = i == 0 || p.src[i - 1] != src;
  if (pos < mine) {
    slot = valid_src ? p.table[(int64_t)src * p.max_seq_len + pos] : kNoSlot;
    if ((uint32_t)slot < (uint32_t)p.size && p.state[slot] == 0) slot = kNoSlot;
    p.table[(int64_t)p.dst[i] * p.max_seq_len + pos] = slot;
  }
  if (!leads || !valid_src) return;
  int refs = 0;
  for (int k0 = i; k0 < p.n; k0 += 64) {  // the run's lengths, one per lane
    const int k = k0 + lane;
    const bool same = k < p.n && p.src[k] == src;
    const int len = same ? fork_len(p, k) : 0;
    const uint64_t ends = __builtin_amdgcn_ballot_w64(!same);
    const int run = ends ? __builtin_ctzll(ends) : 64;
    for (int j = 0; j < run; j++) refs += __builtin_amdgcn_readlane(len, j) > pos;
    if (run < 64) break;
  }
  if (refs == 0) return;
  if (pos >= mine) {  // (a longer fork behind the first)
    slot = p.table[(int64_t)src * p.max_seq_len + pos];
    if ((uint32_t)slot < (uint32_t)p.size && p.state[slot] == 0) slot = kNoSlot;
  }
  if ((uint32_t)slot < (uint32_t)p.size) atomicAdd(p.state + slot, refs);
}

// ------------------------------------------------------------------------------------------------ rows
struct RowsParams {
  char* rows;  // [layers, slots, row]
  int64_t layer_stride, slot_stride;  // bytes
  int32_t pieces, lanes_shift;        // pieces of a row; log2 of the lanes that take one
  int32_t num_slots;
};
// `row_of(i, src, dst)`: the slots of the workgroup's row i (dst: -1 where a target has none), false if it has none.
template <typename Piece, int ROWS, int TARGETS, typename F> __device__ __forceinline__ void move_rows(const RowsParams& p, int layer, F row_of) {
  const int lanes = 1 << p.lanes_shift, sub = threadIdx.x & (lanes - 1);
  char* const base = p.rows + layer * p.layer_stride;
  for (int i = threadIdx.x >> p.lanes_shift; i < ROWS; i += kThreads >> p.lanes_shift) {
    int src, dst[TARGETS];
    if (!row_of(i, src, dst)) continue;
    const Piece* from = (const Piece*)(base + (int64_t)src * p.slot_stride);
#pragma unroll 4
    for (int x = sub; x < p.pieces; x += lanes) {
      const Piece v = from[x];
#pragma unroll
      for (int t = 0; t < TARGETS; t++)
        if (dst[t] >= 0) ((Piece*)(base + (int64_t)dst[t] * p.slot_stride))[x] = v;
    }
  }
}

struct CopyParams {
  ForkParams f;
  RowsParams r, scales;
  const int64_t* index;
  const int32_t* start;
  int64_t num_index;
};
constexpr int kCopyRows = 16;
// grid (positions, forks, layers).  FORKS of one source that stand next to each other read it together where there are more than a few (us, alone | four together, 32 layers of 8 heads: 8 copies of 2000 tokens
// 677 | 502, of 300 114 | 92, 4 of 2000 336 | 281; but 4 of 300 61 | 65, 8 of 20 11 | 23, where a workgroup's chain of loads and stores counts, and 2 of 6500 526 | 535).
constexpr int kCopyTogether = 4;
constexpr int64_t kTogetherFromTokens = 2048;
template <int FORKS> __global__ __launch_bounds__(kThreads) void fork_copy_kernel(CopyParams p) {
  const int i = blockIdx.y, pos0 = (int)blockIdx.x * kCopyRows;
  [[maybe_unused]] const int lane = threadIdx.x & 63;
  const int req = p.f.src[i];
  if constexpr (FORKS > 1) {
    int in_run = 0;  // the forks of the source right in front of this one
    for (int k1 = i; k1 > 0; k1 -= 64) {
      const int k = k1 - 1 - lane;
      const uint64_t ends = __builtin_amdgcn_ballot_w64(k < 0 || p.f.src[k] != req);
      in_run += ends ? __builtin_ctzll(ends) : 64;
      if (ends) break;
    }
    if (in_run % FORKS) return;
  }
  int len[FORKS], most = 0;
  int64_t start[FORKS];
#pragma unroll
  for (int f = 0; f < FORKS; f++) {
    const bool with = i + f < p.f.n && (f == 0 || (len[f - 1] >= 0 && p.f.src[i + f] == req));
    len[f] = with ? fork_len(p.f, i + f) : -1;
    len[f] = with && len[f] < 0 ? 0 : len[f];
    start[f] = with ? p.start[i + f] : 0;
    most = len[f] > most ? len[f] : most;
  }
  if (pos0 >= most) return;
  const bool known = req >= 0 && req < p.f.num_reqs;
  const int32_t* const src_row = p.f.table + (int64_t)req * p.f.max_seq_len;
  auto target = [&](int64_t first, int n, int pos) -> int {  // the slot of a position, -1 if there is none
    const int64_t at = first + pos;
    const int64_t d = pos < n && at >= 0 && at < p.num_index ? p.index[at] : -1;
    return d >= 0 && d < p.r.num_slots ? (int)d : -1;
  };
  if (blockIdx.z == 0 && threadIdx.x < kCopyRows) {
    const int pos = pos0 + threadIdx.x;
#pragma unroll
    for (int f = 0; f < FORKS; f++) {
      const int d = target(start[f], len[f], pos);
      if (pos < len[f]) p.f.table[(int64_t)p.f.dst[i + f] * p.f.max_seq_len + pos] = known && d >= 0 ? d : kNoSlot;
    }
  }
  if (!known) return;
  auto row_of = [&](int k, int& src, int (&dst)[FORKS]) {
    const int pos = pos0 + k;
    if (pos >= most) return false;
    src = src_row[pos];
    if ((uint32_t)src >= (uint32_t)p.r.num_slots) return false;
#pragma unroll
    for (int f = 0; f < FORKS; f++) dst[f] = target(start[f], len[f], pos);
    return true;
  };
  move_rows<u32x4, kCopyRows, FORKS>(p.r, blockIdx.z, row_of);
  if (p.scales.rows) move_rows<uint8_t, kCopyRows, FORKS>(p.scales, blockIdx.z, row_of);
}

// ------------------------------------------------------------------------------------------------ release
struct ReleaseParams {
  const int32_t* table;
  int64_t max_seq_len;
  int32_t most;  // as ForkParams::most
  const int32_t* req;
  const int32_t* len;
  int32_t n, num_reqs;
  int32_t* state;
  int32_t size;
  int32_t blocks;  // of kThreads positions per request
  int32_t* sums;   // (freed, wrong) of every workgroup
  int64_t* cells;
};
// Tokens of request i.
__device__ __forceinline__ int release_len(const ReleaseParams& p, int i) { return p.len[i] < p.most ? p.len[i] : p.most; }
// `refs` references less on a slot.  A count does not fall below zero: what is too much is given back and counts as wrong.  (Of any number of threads one sees the count end: what is given back
// was below zero.)
template <int SCOPE> __device__ __forceinline__ int release_refs(const ReleaseParams& p, int slot, int refs) {
  return __hip_atomic_fetch_sub(p.state + slot, refs, __ATOMIC_RELAXED, SCOPE);
}
template <int SCOPE> __device__ __forceinline__ void release_seen(const ReleaseParams& p, int slot, int refs, int old, int& freed, int& wrong) {
  const int had = old > 0 ? old : 0;
  if (had && had <= refs) freed++;
  if (had < refs) {
    __hip_atomic_fetch_add(p.state + slot, refs - had, __ATOMIC_RELAXED, SCOPE);
    wrong += refs - had;
  }
}
template <int SCOPE> __device__ __forceinline__ void release_one(const ReleaseParams& p, int i, int pos, int& freed, int& wrong) {
  const int req = p.req[i];
  if (pos >= release_len(p, i)) return;
  const int slot = req >= 0 && req < p.num_reqs ? p.table[(int64_t)req * p.max_seq_len + pos] : -1;
  if ((uint32_t)slot >= (uint32_t)p.size) wrong++;
  else release_seen<SCOPE>(p, slot, 1, release_refs<SCOPE>(p, slot, 1), freed, wrong);
}
template <int THREADS> __device__ __forceinline__ void sum_group(int& a, int& b) {
  __shared__ int sh[2][THREADS / 64];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) a += __shfl_xor(a, d, 64), b += __shfl_xor(b, d, 64);
  if ((threadIdx.x & 63) == 0) sh[0][threadIdx.x >> 6] = a, sh[1][threadIdx.x >> 6] = b;
  __syncthreads();
  a = b = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; w++) a += sh[0][w], b += sh[1][w];
}
// (the cells may lie in host memory)
__device__ __forceinline__ void tell(int64_t* cells, int64_t freed, int64_t wrong) {
  __hip_atomic_store(cells, freed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  __hip_atomic_store(cells + 1, wrong, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
__global__ __launch_bounds__(kThreads) void release_kernel(ReleaseParams p) {
  int freed = 0, wrong = 0;
  release_one<__HIP_MEMORY_SCOPE_AGENT>(p, blockIdx.y, (int)(blockIdx.x * kThreads + threadIdx.x), freed, wrong);
  sum_group<kThreads>(freed, wrong);
  if (threadIdx.x == 0) {
    int32_t* s = p.sums + 2 * ((int64_t)blockIdx.y * p.blocks + blockIdx.x);
    s[0] = freed, s[1] = wrong;
  }
}
// Many requests: a lane has a request, a wave 64 of them and kRun positions.  Requests that share tokens share them at the same positions, so lanes that name one slot there are counted and the
// first of them makes one change: an atomic on a slot that lies anywhere costs a transaction of its own, and a search's branches name most slots many times (128 requests, 560000 tokens
// on 69000 slots: 20.5 us with an atomic each, 11.4 so; a wave of sixteen positions, one atomic behind the other, 26).  Two lanes in a row that are alone with their slots end the counting:
// behind the shared part everybody is.  A call, a thread per token | a lane per request, us: forks of one parent's 3000 tokens, 24 21.0 | 21.2, 32 21.2 | 20.6, 64 25 | 21, 256 46 | 30; of eight
// parents of 300 to 8000, 24 22.2 | 23.1, 128 37 | 26; requests that share nothing (1000 tokens each) 64 20.0 | 21.1, 256 28.0 | 28.3.
constexpr int kRun = 4;
constexpr int64_t kColumnsFromRequests = 32;
__global__ __launch_bounds__(kThreads) void release_columns_kernel(ReleaseParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = blockIdx.y * 64 + lane;
  const int pos0 = ((int)blockIdx.x * (kThreads / 64) + wave) * kRun;
  int len = 0, req = -1, freed = 0, wrong = 0;
  if (i < p.n) len = release_len(p, i), req = p.req[i];
  const bool known = req >= 0 && req < p.num_reqs;
  const int32_t* const row = p.table + (int64_t)(known ? req : 0) * p.max_seq_len;
  int slot[kRun];
  if (known && pos0 + kRun <= len) {
    typedef int Four __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int k = 0; k < kRun; k += 4) {
      const Four x = *(const Four*)(row + pos0 + k);
#pragma unroll
      for (int e = 0; e < 4; e++) slot[k + e] = x[e];
    }
  } else {
#pragma unroll
    for (int k = 0; k < kRun; k++) slot[k] = known && pos0 + k < len ? row[pos0 + k] : -1;
  }
  int refs[kRun], old[kRun];
#pragma unroll
  for (int k = 0; k < kRun; k++) {
    const bool valid = (uint32_t)slot[k] < (uint32_t)p.size;
    wrong += pos0 + k < len && !valid;
    uint64_t left = __builtin_amdgcn_ballot_w64(valid);
    int alone = 0;
    refs[k] = valid ? 1 : 0;
    while (left && alone < 2) {
      const int l = __builtin_ctzll(left), s = __builtin_amdgcn_readlane(slot[k], l);
      const uint64_t same = __builtin_amdgcn_ballot_w64(valid && slot[k] == s) & left;
      const int count = __builtin_popcountll(same);
      left &= ~same;
      alone = count == 1 ? alone + 1 : 0;
      if ((same >> lane) & 1) refs[k] = lane == l ? count : 0;
    }
  }
  // all changes are under way before the first is looked at
#pragma unroll
  for (int k = 0; k < kRun; k++) {
    old[k] = 0;
    if (refs[k]) old[k] = release_refs<__HIP_MEMORY_SCOPE_AGENT>(p, slot[k], refs[k]);
  }
#pragma unroll
  for (int k = 0; k < kRun; k++)
    if (refs[k]) release_seen<__HIP_MEMORY_SCOPE_AGENT>(p, slot[k], refs[k], old[k], freed, wrong);
  sum_group<kThreads>(freed, wrong);
  if (threadIdx.x == 0) {
    int32_t* s = p.sums + 2 * ((int64_t)blockIdx.y * p.blocks + blockIdx.x);
    s[0] = freed, s[1] = wrong;
  }
}
__global__ __launch_bounds__(1024) void release_sum_kernel(ReleaseParams p, int64_t groups) {
  __shared__ int64_t sh[2][16];
  int64_t a = 0, b = 0;
  for (int64_t i = threadIdx.x; i < groups; i += 1024) a += p.sums[2 * i], b += p.sums[2 * i + 1];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) a += __shfl_xor(a, d, 64), b += __shfl_xor(b, d, 64);
  if ((threadIdx.x & 63) == 0) sh[0][threadIdx.x >> 6] = a, sh[1][threadIdx.x >> 6] = b;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; w++) a += sh[0][w], b += sh[1][w];
  tell(p.cells, a, b);
}
// Few tokens: one workgroup takes all of them and tells the counts itself.  Whoever sees those (the host, which may go on to another stream) finds the states changed: the atomics are the
// system's and have arrived in front of the barrier.
constexpr int64_t kOneGroupTokens = 4096;
__global__ __launch_bounds__(1024) void release_one_group_kernel(ReleaseParams p, int max_len) {
  int freed = 0, wrong = 0;
  for (int i = threadIdx.x; i < p.n * max_len; i += 1024) release_one<__HIP_MEMORY_SCOPE_SYSTEM>(p, i / max_len, i % max_len, freed, wrong);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  sum_group<1024>(freed, wrong);
  if (threadIdx.x == 0) tell(p.cells, freed, wrong);
}

// ------------------------------------------------------------------------------------------------ compact
// With U slots in use, the k-th free slot below U takes the k-th used slot from U on: as few moves as there are, and what moves keeps its order.
constexpr int kPlanThreads = 1024, kPlanSlots = kPlanThreads * 4;
struct CompactParams {
  int32_t* state;
  int32_t size, blocks;
  int32_t* used;    // [blocks] slots in use
  int32_t* header;  // [0] moves
  int32_t* hole;    // [size / 2 + 1]
  int32_t* source;
  int32_t* code;    // [size]: the new slot; -1 free; -2 - k: the k-th move's source
  int32_t* remap;
  int32_t* table;
  int64_t max_seq_len;
  const int32_t* req;
  const int32_t* len;
  int32_t n, num_reqs;
  RowsParams r, scales;
  int32_t move_wgs, table_blocks, layers, most;
};
__device__ __forceinline__ void load_states(const CompactParams& p, int64_t at, int (&s)[4]) {  // (past the end: free)
  if (at + 4 <= p.size) {
    typedef int Four __attribute__((ext_vector_type(4), aligned(4)));
    const Four x = *(const Four*)(p.state + at);
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = x[e];
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; e++) s[e] = at + e < p.size ? p.state[at + e] : 0;
}
__device__ __forceinline__ int count_group(int mine, int* sh) {  // over the workgroup; `sh`: for this count alone
  const int wave = __builtin_amdgcn_readlane(scan_sum(mine), 63);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = wave;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; w++) all += sh[w];
  return all;
}
__global__ __launch_bounds__(kPlanThreads) void compact_count_kernel(CompactParams p) {
  __shared__ int sh[kPlanThreads / 64];
  int s[4];
  load_states(p, (int64_t)blockIdx.x * kPlanSlots + 4 * threadIdx.x, s);
  const int all = count_group((s[0] != 0) + (s[1] != 0) + (s[2] != 0) + (s[3] != 0), sh);
  if (threadIdx.x == 0) p.used[blockIdx.x] = all;
}
// A pool of up to kLookBlocks workgroups' slots: each of them looks through all counts itself, a bit per slot, instead of waiting for a launch that counts (us a call, 1 layer, launch | look: 65536 slots
// 22.4 | 20.2, 5000 22.5 | 18.6 with the scales' launch gone, too).
constexpr int kLookBlocks = 16;
template <bool LOOK> __global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(CompactParams p) {
  __shared__ int sh[4][kPlanThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t at = (int64_t)blockIdx.x * kPlanSlots + 4 * threadIdx.x;
  int s[4], before = 0, all = 0, front = 0;
  load_states(p, at, s);
  if (LOOK) {
    uint64_t used = 0;  // bit 4 b + e: slot e of the thread's four in block b
#pragma unroll 4
    for (int b = 0; b < p.blocks; b++) {
      int t[4];
      load_states(p, (int64_t)b * kPlanSlots + 4 * threadIdx.x, t);
#pragma unroll
      for (int e = 0; e < 4; e++) used |= (uint64_t)(t[e] != 0) << (4 * b + e);
    }
    all = count_group(__builtin_popcountll(used), sh[0]);
    before = count_group(__builtin_popcountll(used & (((uint64_t)1 << 4 * (int)blockIdx.x) - 1)), sh[1]);
    // (all <= size: of block all / kPlanSlots the slots in front of it)
    const int border = all / kPlanSlots, rest = all - border * kPlanSlots - 4 * (int)threadIdx.x, bits = 4 * border + (rest < 0 ? 0 : rest < 4 ? rest : 4);
    front = count_group(__builtin_popcountll(bits < 64 ? used & (((uint64_t)1 << bits) - 1) : used), sh[2]);
  } else {
    for (int b = threadIdx.x; b < p.blocks; b += kPlanThreads) {
      const int n = p.used[b];
      before += b < (int)blockIdx.x ? n : 0;
      all += n;
    }
    before = count_group(before, sh[0]), all = count_group(all, sh[1]);
    // slots in use in front of slot `all`
    const int border = all / kPlanSlots;
    for (int b = threadIdx.x; b < border; b += kPlanThreads) front += p.used[b];
    int t[4];
    const int64_t bat = (int64_t)border * kPlanSlots + 4 * threadIdx.x;
    load_states(p, bat, t);
#pragma unroll
    for (int e = 0; e < 4; e++) front += bat + e < all && t[e] != 0;
    front = count_group(front, sh[2]);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.header[0] = all - front;
  // ranks
  const int mine = (s[0] != 0) + (s[1] != 0) + (s[2] != 0) + (s[3] != 0), up_to = scan_sum(mine);
  if (lane == 63) sh[3][wave] = up_to;
  __syncthreads();
  int rank = before + up_to - mine;  // used slots in front of the thread's first one
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; w++) rank += w < wave ? sh[3][w] : 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int64_t slot = at + e;
    if (slot >= p.size) break;
    const bool in_use = s[e] != 0;
    int code = in_use ? (int)slot : -1;
    if (slot < all && !in_use) p.hole[slot - rank] = (int)slot;
    if (slot >= all && in_use) {
      p.source[rank - front] = (int)slot;
      code = -2 - (rank - front);
    }
    p.code[slot] = code;
    if (code >= -1) p.remap[slot] = code;
    rank += in_use;
  }
}
// Workgroups that move rows (and the counts, with the first layer), those of a layer side by side, and behind them workgroups that rewrite the requests' table entries.
constexpr int kMoveRows = 16;
__global__ __launch_bounds__(kThreads) void compact_move_kernel(CompactParams p) {
  const int moves = p.header[0], layer = (int)blockIdx.x / p.move_wgs;
  if (layer < (p.layers ? p.layers : 1)) {
    for (int m0 = ((int)blockIdx.x - layer * p.move_wgs) * kMoveRows; m0 < moves; m0 += p.move_wgs * kMoveRows) {
      if (layer == 0 && threadIdx.x < kMoveRows && m0 + (int)threadIdx.x < moves) {
        const int src = p.source[m0 + threadIdx.x], dst = p.hole[m0 + threadIdx.x];
        p.state[dst] = p.state[src];
        p.state[src] = 0;
        p.remap[src] = dst;
      }
      auto move = [&](int k, int& src, int (&dst)[1]) {
        if (m0 + k >= moves) return false;
        src = p.source[m0 + k], dst[0] = p.hole[m0 + k];
        return true;
      };
      if (p.layers) move_rows<u32x4, kMoveRows, 1>(p.r, layer, move);
      if (p.scales.rows) move_rows<uint8_t, kMoveRows, 1>(p.scales, layer, move);
    }
    return;
  }
  const int x = (int)blockIdx.x - p.move_wgs * (p.layers ? p.layers : 1), i = x / p.table_blocks, pos = (x - i * p.table_blocks) * kThreads + threadIdx.x;
  const int req = p.req[i], len = p.len[i] < p.most ? p.len[i] : p.most;
  if (req < 0 || req >= p.num_reqs || pos >= len) return;
  int32_t* entry = p.table + (int64_t)req * p.max_seq_len + pos;
  const int slot = *entry;
  if ((uint32_t)slot >= (uint32_t)p.size) return;
  const int code = p.code[slot];
  if (code <= -2) *entry = p.hole[-2 - code];
}

// rows of `bytes` (16-byte pieces) by lanes that are a power of two, a wave at most
void set_rows(RowsParams& r, void* rows, int64_t layer_stride, int64_t slot_stride, int64_t pieces, int64_t num_slots) {
  r.rows = (char*)rows, r.layer_stride = layer_stride, r.slot_stride = slot_stride, r.num_slots = (int32_t)num_slots;
  r.pieces = (int32_t)pieces, r.lanes_shift = 0;
  while (r.lanes_shift < 6 && (1 << r.lanes_shift) < pieces) r.lanes_shift++;
}
// workgroups of a release: along the positions, and in all
struct ReleaseGroups {
  int64_t blocks, rows;
  int64_t all() const { return blocks * rows; }
};
ReleaseGroups release_groups(int64_t n, int64_t most) {
  if (n < kColumnsFromRequests) return ReleaseGroups{(most + kThreads - 1) / kThreads, n};
  constexpr int64_t positions = kThreads / 64 * kRun;
  return ReleaseGroups{(most + positions - 1) / positions, (n + 63) / 64};
}
bool rows_ok(const lsattn_pool_rows* r) {
  if (!r->rows) return r->num_layers == 0 && !r->scales;
  if (r->num_layers < 1 || r->num_layers > 65535 || r->row_bytes < 16 || r->row_bytes % 16 || r->row_bytes > 0x7fffffff || r->slot_stride_bytes < r->row_bytes ||
      r->slot_stride_bytes % 16 || r->layer_stride_bytes % 16 || ((uintptr_t)r->rows & 15) || r->num_slots < 1 || r->num_slots > 0x7fffffff)
    return false;
  return !r->scales || (r->scale_bytes >= 1 && r->scale_bytes <= 0x7fffffff && r->scale_slot_stride_bytes >= r->scale_bytes);
}

}  // namespace
}  // namespace lsattn

using namespace lsattn;

extern "C" int lsattn_fork_requests(int32_t* req_to_tokens, int64_t num_reqs, int64_t max_seq_len, const int32_t* src_req_idx, const int32_t* dst_req_idx,
                                    const int32_t* b_seq_len, int64_t n, int64_t max_len_in_batch, int32_t* mem_state, int64_t pool_size, void* stream) {
  if (!req_to_tokens || !src_req_idx || !dst_req_idx || !b_seq_len || !mem_state || num_reqs < 0 || max_seq_len < 0 || n < 0 || max_len_in_batch < 0 || pool_size < 0 ||
      num_reqs > 0x7fffffff || max_seq_len > 0x7fff0000 || n > 65535 || pool_size > 0x7fffffff)
    return LSATTN_ERR_INVALID_ARG;
  const int64_t most = max_len_in_batch < max_seq_len ? max_len_in_batch : max_seq_len;
  if (n == 0 || most == 0) return LSATTN_OK;
  const ForkParams p{req_to_tokens, max_seq_len, (int32_t)most, src_req_idx, dst_req_idx, b_seq_len, (int32_t)n, (int32_t)num_reqs, mem_state, (int32_t)pool_size};
  LSATTN_LAUNCH_KERNEL(fork_share_kernel, dim3((unsigned)((most + kThreads - 1) / kThreads), (unsigned)n), dim3(kThreads), 0, (hipStream_t)stream, p);
  return check_launch();
}

extern "C" int lsattn_copy_requests(const lsattn_copy_requests_args* a, const lsattn_pool_rows* rows, void* stream) {
  if (!a || !rows || !a->req_to_tokens || !a->src_req_idx || !a->dst_req_idx || !a->b_seq_len || !a->b_start_loc || !a->mem_index || !rows->rows || !rows_ok(rows))
    return LSATTN_ERR_INVALID_ARG;
  if (a->num_reqs < 0 || a->max_seq_len < 0 || a->n < 0 || a->max_len_in_batch < 0 || a->num_index < 0 || a->num_reqs > 0x7fffffff || a->max_seq_len > 0x7fff0000 ||
      a->n > 65535)
    return LSATTN_ERR_INVALID_ARG;
  const int64_t most = a->max_len_in_batch < a->max_seq_len ? a->max_len_in_batch : a->max_seq_len;
  if (a->n == 0 || most == 0) return LSATTN_OK;
  CopyParams p = {};
  p.f = ForkParams{a->req_to_tokens, a->max_seq_len, (int32_t)most, a->src_req_idx, a->dst_req_idx, a->b_seq_len, (int32_t)a->n, (int32_t)a->num_reqs, nullptr, 0};
  p.index = a->mem_index, p.start = a->b_start_loc, p.num_index = a->num_index;
  const dim3 grid((unsigned)((most + kCopyRows - 1) / kCopyRows), (unsigned)a->n, (unsigned)rows->num_layers);
  hipStream_t st = (hipStream_t)stream;
  set_rows(p.r, rows->rows, rows->layer_stride_bytes, rows->slot_stride_bytes, rows->row_bytes / 16, rows->num_slots);
  if (rows->scales) set_rows(p.scales, rows->scales, rows->scale_layer_stride_bytes, rows->scale_slot_stride_bytes, rows->scale_bytes, rows->num_slots);
  if (a->n >= kCopyTogether && a->n * most >= kTogetherFromTokens) LSATTN_LAUNCH_KERNEL(fork_copy_kernel<kCopyTogether>, grid, dim3(kThreads), 0, st, p);
  else LSATTN_LAUNCH_KERNEL(fork_copy_kernel<1>, grid, dim3(kThreads), 0, st, p);
  return check_launch();
}

extern "C" size_t lsattn_release_workspace_bytes(int64_t n, int64_t max_len_in_batch) {
  if (n <= 0 || max_len_in_batch <= 0 || n > 65535 || max_len_in_batch > 0x7fff0000 || n * max_len_in_batch <= kOneGroupTokens) return 0;
  // (enough for fewer requests, too, which may be more workgroups)
  const int64_t all = release_groups(n, max_len_in_batch).all(), fewer = n < kColumnsFromRequests ? 0 : release_groups(kColumnsFromRequests - 1, max_len_in_batch).all();
  return (size_t)((all > fewer ? all : fewer) * 8);
}

extern "C" int lsattn_release_requests(const int32_t* req_to_tokens, int64_t num_reqs, int64_t max_seq_len, const int32_t* b_req_idx, const int32_t* b_seq_len, int64_t n,
                                       int64_t max_len_in_batch, int32_t* mem_state, int64_t pool_size, int64_t* counts, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  if (!req_to_tokens || !b_req_idx || !b_seq_len || !mem_state || !counts || num_reqs < 0 || max_seq_len < 0 || n < 0 || max_len_in_batch < 0 || pool_size < 0 ||
      num_reqs > 0x7fffffff || max_seq_len > 0x7fff0000 || n > 65535 || pool_size > 0x7fffffff || max_len_in_batch > 0x7fff0000)
    return LSATTN_ERR_INVALID_ARG;
  const int64_t most = max_len_in_batch < max_seq_len ? max_len_in_batch : max_seq_len;
  const size_t need = lsattn_release_workspace_bytes(n, most);
  if (need && (!workspace || workspace_bytes < need)) return LSATTN_ERR_WORKSPACE;
  if (need && ((uintptr_t)workspace & 3)) return LSATTN_ERR_INVALID_ARG;
  ReleaseParams p{req_to_tokens, max_seq_len, (int32_t)most, b_req_idx, b_seq_len, (int32_t)n, (int32_t)num_reqs, mem_state, (int32_t)pool_size, 0, (int32_t*)workspace, counts};
  hipStream_t st = (hipStream_t)stream;
  if (!need) {
    LSATTN_LAUNCH_KERNEL(release_one_group_kernel, dim3(1), dim3(1024), 0, st, p, (int)most);
    return check_launch();
  }
  const ReleaseGroups g = release_groups(n, most);
  p.blocks = (int32_t)g.blocks;
  const dim3 grid((unsigned)g.blocks, (unsigned)g.rows);
  if (n < kColumnsFromRequests) LSATTN_LAUNCH_KERNEL(release_kernel, grid, dim3(kThreads), 0, st, p);
  else LSATTN_LAUNCH_KERNEL(release_columns_kernel, grid, dim3(kThreads), 0, st, p);
  if (hipPeekAtLastError() != hipSuccess) return check_launch();
  LSATTN_LAUNCH_KERNEL(release_sum_kernel, dim3(1), dim3(1024), 0, st, p, g.all());
  return check_launch();
}

extern "C" size_t lsattn_compact_workspace_bytes(int64_t pool_size) {
  if (pool_size <= 0 || pool_size > 0x7fff0000) return 0;
  const int64_t blocks = (pool_size + kPlanSlots - 1) / kPlanSlots;
  return (size_t)(4 * (4 + blocks + 2 * (pool_size / 2 + 1) + pool_size));
}

extern "C" int lsattn_compact_pool(const lsattn_compact_args* a, const lsattn_pool_rows* rows, void* stream) {
  if (!a || !rows || !rows_ok(rows) || (rows->rows && rows->num_slots < a->pool_size)) return LSATTN_ERR_INVALID_ARG;
  if (a->pool_size < 0 || a->pool_size > 0x7fff0000 || a->n < 0 || a->n > 65535 || a->max_len_in_batch < 0 || a->num_reqs < 0 || a->num_reqs > 0x7fffffff ||
      a->max_seq_len < 0 || a->max_seq_len > 0x7fff0000)
    return LSATTN_ERR_INVALID_ARG;
  if (a->pool_size == 0) return LSATTN_OK;
  if (!a->mem_state || !a->remap || (a->n && (!a->req_to_tokens || !a->b_req_idx || !a->b_seq_len))) return LSATTN_ERR_INVALID_ARG;
  if (!a->workspace || a->workspace_bytes < lsattn_compact_workspace_bytes(a->pool_size)) return LSATTN_ERR_WORKSPACE;
  if ((uintptr_t)a->workspace & 15) return LSATTN_ERR_INVALID_ARG;
  const int64_t most = a->max_len_in_batch < a->max_seq_len ? a->max_len_in_batch : a->max_seq_len;
  CompactParams p = {};
  p.state = a->mem_state, p.size = (int32_t)a->pool_size, p.blocks = (int32_t)((a->pool_size + kPlanSlots - 1) / kPlanSlots);
  p.header = (int32_t*)a->workspace, p.used = p.header + 4, p.hole = p.used + p.blocks, p.source = p.hole + (p.size / 2 + 1), p.code = p.source + (p.size / 2 + 1);
  p.remap = a->remap, p.table = a->req_to_tokens, p.max_seq_len = a->max_seq_len, p.req = a->b_req_idx, p.len = a->b_seq_len;
  p.n = (int32_t)a->n, p.num_reqs = (int32_t)a->num_reqs;
  p.table_blocks = (int32_t)((most + kThreads - 1) / kThreads), p.most = (int32_t)most;
  if ((int64_t)p.table_blocks * p.n > kMaxUnits - 0x400000) return LSATTN_ERR_INVALID_ARG;
  p.layers = (int32_t)rows->num_layers;
  const int64_t moves = p.size / 2, fill = p.layers ? (16 * kCUs + p.layers - 1) / p.layers : 4 * kCUs, by_moves = (moves + kMoveRows - 1) / kMoveRows;
  p.move_wgs = (int32_t)(by_moves < 1 ? 1 : by_moves < fill ? by_moves : fill);
  const unsigned move_wgs = (unsigned)(p.move_wgs * (p.layers ? p.layers : 1)), table_wgs = (unsigned)(p.table_blocks * p.n);
  hipStream_t st = (hipStream_t)stream;
  if (p.layers) set_rows(p.r, rows->rows, rows->layer_stride_bytes, rows->slot_stride_bytes, rows->row_bytes / 16, rows->num_slots);
  if (rows->scales) set_rows(p.scales, rows->scales, rows->scale_layer_stride_bytes, rows->scale_slot_stride_bytes, rows->scale_bytes, rows->num_slots);
  if (p.blocks <= kLookBlocks) {
    LSATTN_LAUNCH_KERNEL(compact_plan_kernel<true>, dim3(p.blocks), dim3(kPlanThreads), 0, st, p);
  } else {
    LSATTN_LAUNCH_KERNEL(compact_count_kernel, dim3(p.blocks), dim3(kPlanThreads), 0, st, p);
    if (hipPeekAtLastError() != hipSuccess) return check_launch();
    LSATTN_LAUNCH_KERNEL(compact_plan_kernel<false>, dim3(p.blocks), dim3(kPlanThreads), 0, st, p);
  }
  if (hipPeekAtLastError() != hipSuccess) return check_launch();
  LSATTN_LAUNCH_KERNEL(compact_move_kernel, dim3(move_wgs + table_wgs), dim3(kThreads), 0, st, p);
  return check_launch();
}
