// Attention for requests that share the first tokens of their contexts (gfx950, wave64).
//
// A group of requests names the same pool slots for its first P tokens.  For its query rows (a token and a query head each) the softmax over prefix and own
// tokens splits,
//   o = sum_j exp(s_j) v_j / sum_j exp(s_j),   j over the prefix, then over the request's own tokens,
// into partials with a log-sum-exp each, and the prefix's part is one product of all the group's rows with the same keys: every K/V row of the prefix is
// read once for 128 query rows and goes through the matrix pipe, where a decode kernel reads it once per request.
//
// Prefix part: a workgroup of four waves owns 128 rows of one KV head (a wave 32, as rows come: token by token, the query heads of the KV head side by side,
// whatever their number) and walks tiles of 64 keys of a share of the prefix:
//   * the work of all groups, (row tile, block of 64 keys) pairs, is dealt to the workgroups of a KV head on the device, whatever the groups' sizes and prefixes are (the host
//     does not know them): in equal shares, or in pieces that the row tiles of a group go through side by side (Deal); a workgroup leaves one fp32 partial per row tile it touches;
//   * K and V rows lie where the request table says.  Direct loads to LDS take an address per lane, so gathering them costs a multiplication per load; two stages,
//     16-byte chunks XORed with the row (prefill_small.hip says why); the slots of the tile after next are under way;
//   * the order of the keys in a tile does not matter without a causal mask: rows lie so that a lane's slots are neighbours in the table;
//   * entries of the table that name no slot, and positions past the prefix, are a mask of the tile; its V rows are cleared in LDS before they are used;
//   * scores transposed, S^T = K Q^T, so that P^T goes into O^T += V^T P^T from the lane that computed it.  fp16: P as fp16, 2^-11, which a 16-bit output rounds away for the most part
//     (2.9e-4 against 2.1e-4 with fp32 weights; a second part would be half as many products again), O divided by the sum of the very weights
//     that multiplied V; bfloat16: P in two parts, high and low, 2^-16 (8 bits alone would cost 1e-3 of O);
//   * the running maximum is raised where a lane's eight weights pass 2^15, and then set so that the largest is 2^9.
// Own tokens: the decode walk of pool_walk.hip.h from the prefix's end on, in the same launch (those workgroups wait for memory where the others keep the matrix
// pipe busy), equal shares of all requests' own tokens.  A second launch joins a request's partials.
//
// What bounds it, with the case that shows it (launches alone, without the one that joins, of a GPU that was idle before; hundreds of passes in a row raise the clock, and those that compute
// get 6 to 10% faster):
//   * few rows per group: reads, of which too few are under way.  24 requests in three groups and alone, 32/32 heads, 449 MB: 92 us, 4.9 TB/s (a streaming read: 7.0).  A group of 8 has 8 rows of
//     a tile's 128, which one wave of four multiplies while the tile's loads have been waited for;
//   * prefix and own tokens together, reads too: 64 requests behind 16384 tokens, 32/8 heads, up to 1500 own: 59 us (284 MB, 4.8 TB/s; the parts alone 35 and 42 us; 64 us, 4.4 TB/s, where
//     nothing of it is in the last-level cache);
//   * many rows, 64-wide bfloat16: vector work, then the matrix pipe, which runs beside it only in part (busy 54% and 30%): 160 requests in two groups, 28/4 heads: 66 us, 0.4 PFLOP/s of the
//     formula, a half more with the second part of P;
//   * many rows, 128-wide fp16: the products (0.9 PFLOP/s of whole row tiles as the prefix grows, 1.14 where nothing has to be loaded, 1.17 a large library product), and 17 us of start and end: prompts of
//     293 rows behind 6001 tokens 50 us, of which 6 are 28 MB of partials that all workgroups store at once.
// Tried and left out (timed while this was built; 128-wide heads, all 0.70 to 0.75 PFLOP/s before the tiles went side by side, as this form): four stages of 32 keys; operands read a step ahead, or all at once (decode 5 to
// 8% slower); eight waves of 256 rows, in alternating phases or not (no room beside it for the own tokens; prompts of
// 150 to 400 rows 0 to 8% slower, of 1200 2 to 4% faster, of 2500 behind 20000 tokens 10%); lines fetched into the L2 ahead (5%, few rows 30% slower); three and four waves per SIMD of
// the 64-wide form (equal, and slower for spills); sums and exponentials in independent batches, products of 32 x 32 for bfloat16 (equal).  Of 64-wide bfloat16 rows 16 exponentials take an eighth of
// a tile's time, the low parts of P a ninth, the reads from LDS nothing.
#include <type_traits>

#include "pool_walk.hip.h"

namespace lsattn {
namespace {

typedef __attribute__((address_space(3))) i16x4* lds_i16x4_ptr;

constexpr int kRows = 128;   // query rows of a workgroup of the prefix part
constexpr int kKeys = 64;    // keys of a tile
constexpr float kPrefixHead = 9.f;
constexpr int kPlanInts = 12;

struct SharedParams {
  PoolParams w;  // the pool, the table, the requests' own tokens and their shares; part_o / part_lse: the own parts
  int64_t q_st, q_sh;  // bytes
  const int32_t* g_start;
  const int32_t* g_size;
  const int32_t* g_req;
  const int32_t* g_prefix;
  int32_t groups, rows;  // rows of q
  int32_t most;          // a bound of the prefixes: longer ones are cut there
  int32_t near;          // whether every row lies within 2 GB of its head's first, slots and strides of 24 bits
  int32_t shares, parts; // of the prefix part, per KV head; partials of 128 rows per KV head
  int32_t ahead;         // whether the prefix part's waves come before those of the own tokens
  int32_t rounds;        // pieces that a workgroup takes at most (see Deal)
  int32_t xcds_shift;    // log2 of the XCDs that run a KV head's workgroups
  int32_t own_wgs;       // workgroups of the own tokens (prompts: of the plan), in front of those of the prefix part; a multiple of 8
  int32_t* plan;         // [batch, kPlanInts] where a request's partials lie, for the second launch
  float* pre_o;          // [hkv, parts, 128, D]
  float* pre_lse;        // [hkv, parts, 128], log2 domain
  FastDiv by_hkv, by_hq, by_group, by_pre_shares;
};

__device__ __forceinline__ const char* uniform_ptr(const char* ptr) {
  const uint64_t u = (uint64_t)ptr;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return (const char*)(((uint64_t)hi << 32) | lo);
}
// s_waitcnt vmcnt(N) (expcnt / lgkmcnt fields left at their maximum)
template <int N> __device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14)); }

// 64 groups at a time, one per lane.  Groups stand in ascending order of their rows; a row that two of them name belongs to the first, so that
// whatever the lists hold no row is counted twice.
struct Groups {
  int at;                    // the group of lane 0
  int lo, size, req, prefix; // of the lane's group: its rows, from lo on
  int end;                   // the end of the rows up to the lane's group
  int tiles, blocks;         // row tiles, blocks of keys
  int tiles_to, units_to;    // sums over the 64 up to the lane's group; a unit is a row tile with a block
  int pieces_to;             // as these, of the pieces of Deal
  __device__ __forceinline__ void look(const SharedParams& p, int g0, int end_before) {
    const int lane = threadIdx.x & 63, g = g0 + lane;
    at = g0;
    int start = 0, last = 0;
    req = 0, prefix = 0;
    if (g < p.groups) {
      start = p.g_start[g], last = p.g_size[g], req = p.g_req[g], prefix = p.g_prefix[g];
      start = start < 0 ? 0 : start < p.rows ? start : p.rows;
      last = last < 0 ? start : last < p.rows - start ? start + last : p.rows;
      prefix = prefix < 0 || req < 0 || req >= p.w.num_reqs ? 0 : prefix < p.most ? prefix : p.most;
    }
    end = scan_max(last);
    end = end > end_before ? end : end_before;
    const int below = __shfl_up(end, 1, 64);
    const int taken = lane ? below : end_before;
    lo = start > taken ? start : taken;
    size = last > lo ? last - lo : 0;
    blocks = (prefix + kKeys - 1) / kKeys;
    tiles = blocks ? (int)(((int64_t)size * p.w.group + kRows - 1) / kRows) : 0;
    tiles_to = scan_sum(tiles), units_to = scan_sum(tiles * blocks);
  }
  __device__ __forceinline__ int end_of_all() const { return __builtin_amdgcn_readlane(end, 63); }
  __device__ __forceinline__ int all_tiles() const { return __builtin_amdgcn_readlane(tiles_to, 63); }
  __device__ __forceinline__ int all_units() const { return __builtin_amdgcn_readlane(units_to, 63); }
};
// How the units are dealt to the workgroups of a KV head.
// A row tile reads all of its group's prefix, so the tiles of a group read the same rows, and where they do it at different times and the prefix is longer than an L2, each of
// them reads it from memory again (293 rows of 32/8 heads behind 24000 tokens: 90% of the L2's requests missed).  So where a group has more than one tile and it comes out even,
// the prefixes are cut into pieces of `cut` blocks for every tile of the group, the tiles of a piece side by side, and a workgroup takes a piece (or one of each round): the tiles go
// through it in step on one XCD, which reads it once (12% missed; us, without | with, both launches: 293 rows behind 1000 tokens 45 | 41, 6001 70 | 63, 20000 147 | 139; 150 behind 6001 54 | 46).
// "Even": no more than an eighth longer than equal shares, a piece's start and end counted (600 rows behind 6001 in three rounds of short pieces: 97 | 114).
// Else, in order of tiles and their blocks, `per` units each.
constexpr int kPieceCost = 4;  // blocks that a piece's start and its partials cost
struct Deal {
  int per, cut, pieces;
};
__device__ __forceinline__ Deal deal_of(const SharedParams& p, Groups& g) {  // `g`: at the first groups, and left there
  int total = g.all_units();
  if (p.groups > 64) {
    for (int g0 = 64; g0 < p.groups; g0 += 64) g.look(p, g0, g.end_of_all()), total += g.all_units();
    g.look(p, 0, 0);
  }
  Deal d;
  d.per = (int)div_by((uint32_t)(total + p.shares - 1), p.by_pre_shares);
  d.per = d.per < 1 ? 1 : d.per;
  d.cut = 0, d.pieces = total;
  if (!p.rounds) return d;
  const uint32_t longest = (uint32_t)__builtin_amdgcn_readlane(scan_max(g.tiles ? g.blocks : 0), 63);
  if (p.groups > 64 || __builtin_amdgcn_ballot_w64(g.tiles > 1) == 0 || longest >= 1u << 20) return d;
  for (int round = 1; round <= p.rounds; round++) {
    const uint32_t most = (uint32_t)round * p.shares;
    const int n = (int)(most * longest / (uint32_t)total);  // pieces of the longest prefix, if they all were as long
    for (int c = n; c > 0 && c > n - 3; c--) {
      const int cut = (int)((longest + c - 1) / (uint32_t)c);
      if (round * (cut + kPieceCost) * 8 > (d.per + kPieceCost) * 9) break;
      g.pieces_to = scan_sum(g.tiles * ((g.blocks + cut - 1) / cut));
      const int pieces = __builtin_amdgcn_readlane(g.pieces_to, 63);
      if (pieces <= (int)most) {
        d.cut = cut, d.pieces = pieces;
        return d;
      }
    }
  }
  return d;
}

// The group of row b (per lane; -1: none) and its numbers, looked up from the first groups on.
struct Membership {
  int lo, prefix, tile0, unit0, blocks;  // the group's first row, prefix, and the tiles and units of all groups in front of it
  int g;                                 // the group, of the last 64 that were looked through
  __device__ __forceinline__ void find(const SharedParams& p, Groups& g, int b) {
    lo = prefix = tile0 = unit0 = blocks = this->g = 0;
    if (p.groups <= 8) {  // (a trip to LDS takes as long as two of them)
      for (int n = 0; n < p.groups; n++) {
        const int s = __builtin_amdgcn_readlane(g.lo, n), sz = __builtin_amdgcn_readlane(g.size, n), t1 = __builtin_amdgcn_readlane(g.tiles, n);
        const int bl = __builtin_amdgcn_readlane(g.blocks, n), pr = __builtin_amdgcn_readlane(g.prefix, n);
        const int t0 = __builtin_amdgcn_readlane(g.tiles_to, n) - t1, u0 = __builtin_amdgcn_readlane(g.units_to, n) - t1 * bl;
        if (s <= b && b < s + sz) lo = s, prefix = pr, blocks = bl, tile0 = t0, unit0 = u0, this->g = n;
      }
      return;
    }
    int tiles = 0, units = 0;
    for (int g0 = 0;;) {
      int n = 0;  // groups of the 64 that end at b or in front of it
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        const int e = __shfl(g.end, n + d - 1, 64);
        n += e <= b ? d : 0;
      }
      const int e63 = __shfl(g.end, 63, 64);
      const bool here = n < 63 || e63 > b;  // (n counts up to 63)
      const int s = __shfl(g.lo, n, 64), sz = __shfl(g.size, n, 64), pr = __shfl(g.prefix, n, 64), bl = __shfl(g.blocks, n, 64);
      const int tt = __shfl(g.tiles_to, n, 64), t1 = __shfl(g.tiles, n, 64), ut = __shfl(g.units_to, n, 64);
      if (here && s <= b && b < s + sz) lo = s, prefix = pr, blocks = bl, tile0 = tiles + tt - t1, unit0 = units + ut - t1 * bl, this->g = n;
      tiles += g.all_tiles(), units += g.all_units();
      g0 += 64;
      if (g0 >= p.groups) break;
      g.look(p, g0, g.end_of_all());
    }
    if (p.groups > 64) g.look(p, 0, 0);
  }
};

// Where the prefix's partials of a row tile lie: n of them from `first` on, `step` apart.
struct Partials {
  int first, n, step;
};
__device__ __forceinline__ Partials partials_of(const Deal& d, int tile, int tile0, int unit0, int blocks, int tiles, int pieces0) {
  if (!blocks) return Partials{0, 0, 1};
  if (d.cut) return Partials{pieces0 + tile, (blocks + d.cut - 1) / d.cut, tiles};
  const uint32_t u0 = (uint32_t)(unit0 + tile * blocks), first = u0 / (uint32_t)d.per;
  return Partials{(int)first + tile0 + tile, (int)((u0 + blocks - 1) / (uint32_t)d.per - first) + 1, 1};
}

// What the launch that joins the partials has to know of a row of q (found again by each of its workgroups, this made that launch two to three times as long).
struct PlanRow {
  const Membership& m;
  const Deal& d;
  int tiles, pieces0;
  __device__ __forceinline__ PlanRow(const Membership& m, const Groups& g, const Deal& d) : m(m), d(d) {  // (by whole waves)
    tiles = __shfl(g.tiles, m.g, 64);
    pieces0 = d.cut ? __shfl(g.pieces_to - g.tiles * ((g.blocks + d.cut - 1) / d.cut), m.g, 64) : 0;
  }
  __device__ __forceinline__ void put(const SharedParams& p, int b, bool shares, int own0, int n_own) const {
    int32_t* const plan = p.plan + kPlanInts * (int64_t)b;
    *(u32x4*)plan = u32x4{(uint32_t)m.lo, (uint32_t)m.tile0, (uint32_t)m.unit0, shares ? (uint32_t)m.blocks : 0u};
    *(u32x4*)(plan + 4) = u32x4{(uint32_t)own0, (uint32_t)n_own, (uint32_t)d.per, (uint32_t)d.cut};
    *(u32x4*)(plan + 8) = u32x4{(uint32_t)tiles, (uint32_t)pieces0, 0u, 0u};
  }
};

// ------------------------------------------------------------------------------------------------ the prefix part
template <typename T, int D> constexpr int kPrefixLds = 2 * 2 * kKeys * D * 2 + 2 * 8;  // two stages of K and V tiles, their masks

// THROUGH: partials go through to memory as they are stored.  Of many rows the launch's end waits for less then (prompts of 293 rows behind 6001 tokens 67 -> 65 us); beside workgroups that
// still read, or of few rows, it waits for more (24 requests 96 -> 97.5 us).
template <typename T, int D, bool THROUGH> __device__ __forceinline__ void prefix_share(const SharedParams& p, char* lds, int kvh, int share) {
  constexpr bool HIGH_LOW = __is_same(T, BF16);
  constexpr int NP = HIGH_LOW ? 2 : 1;      // parts of P
  constexpr int KS = D / 32, NDB = D / 16;  // contraction steps of Q K^T; 16-wide blocks of the head
  constexpr int CPR = D / 8, RB = D * 2;    // 16-byte chunks and bytes of a row
  constexpr int TB = kKeys * RB;
  constexpr int RPI = 64 / CPR, NI = 16 / RPI;  // rows per load instruction; instructions for a wave's 16 rows of a tile
  constexpr int RPB = 256 / RB;
  constexpr int kMaskOff = 4 * TB;
  auto swz_k = [](int row) { return (row / RPB) & (CPR - 1); };
  auto swz_v = [](int row) { return ((row / RPB) & (CPR / 2 - 1)) << 1; };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int lds_base = (int)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  Groups gs;
  gs.look(p, 0, 0);
  const Deal deal = deal_of(p, gs);
  // units, or pieces, in the order in which they are dealt: from `at` on, up to `end`
  int at = deal.cut ? share : (int)((int64_t)share * deal.per < deal.pieces ? share * deal.per : deal.pieces);
  const int end = deal.cut || deal.pieces - at < deal.per ? deal.pieces : at + deal.per;
  int first = 0, tiles_before = 0;  // units and tiles in front of the 64 groups
  // the lane's row of its first load instruction, and its chunk of it, K and V (rows RPI apart differ in bits of their XOR that the lane's own row leaves free)
  const int j_row = lane / CPR;
  const uint32_t k_chunk = (uint32_t)(((lane % CPR) ^ swz_k(j_row)) * 16), v_chunk = (uint32_t)(((lane % CPR) ^ swz_v(j_row)) * 16);
  int kaddr[KS], vaddr[NDB];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) kaddr[ks] = lds_base + c * RB + (((4 * ks + g) & (CPR - 1)) ^ swz_k(c)) * 16;
#pragma unroll
  for (int db = 0; db < NDB; db++) {
    const int row = 4 * g + (c >> 2);
    vaddr[db] = lds_base + TB + row * RB + ((2 * db + ((c & 3) >> 1)) ^ swz_v(row)) * 16 + (c & 1) * 8;
  }
  const char* const kb = uniform_ptr(p.w.k + kvh * p.w.k_s1);
  const char* const vb = uniform_ptr(p.w.v + kvh * p.w.v_s1);
  const uint32_t k_s0 = (uint32_t)p.w.k_s0, v_s0 = (uint32_t)p.w.v_s0;
  const float scale = p.w.scale_log2;

  if (p.ahead) __builtin_amdgcn_s_setprio(3);
  while (at < end) {
    while (!deal.cut && at >= first + gs.all_units()) {  // (at < deal.pieces: a later group has some)
      first += gs.all_units(), tiles_before += gs.all_tiles();
      gs.look(p, gs.at + 64, gs.end_of_all());
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64((deal.cut ? gs.pieces_to : first + gs.units_to) > at));
    const int blocks = __builtin_amdgcn_readlane(gs.blocks, l), tiles = __builtin_amdgcn_readlane(gs.tiles, l);
    int tile, block0, nt, part;  // tiles of keys to walk
    if (deal.cut) {
      const int i = at - (__builtin_amdgcn_readlane(gs.pieces_to, l) - tiles * ((blocks + deal.cut - 1) / deal.cut)), chunk = i / tiles;
      tile = i - chunk * tiles, block0 = chunk * deal.cut, nt = blocks - block0 < deal.cut ? blocks - block0 : deal.cut, part = at;
    } else {
      const int unit0 = first + __builtin_amdgcn_readlane(gs.units_to, l) - tiles * blocks;
      tile = (at - unit0) / blocks, block0 = (at - unit0) - tile * blocks;
      nt = blocks - block0 < end - at ? blocks - block0 : end - at;
      part = share + tiles_before + __builtin_amdgcn_readlane(gs.tiles_to, l) - tiles + tile;
    }
    const int lo = __builtin_amdgcn_readlane(gs.lo, l), prefix = __builtin_amdgcn_readlane(gs.prefix, l);
    const int rows = __builtin_amdgcn_readlane(gs.size, l) * p.w.group;
    const int32_t* const row_slots = (const int32_t*)uniform_ptr((const char*)(p.w.table + (int64_t)__builtin_amdgcn_readlane(gs.req, l) * p.w.max_seq_len));
    const int row0 = tile * kRows + wave * 32;
    const bool active = row0 < rows;

    u32x4 qreg[2][KS];
    f32x4 oacc[2][NDB], l_pv[2];
    float m_run[2], l_run[2];
#pragma unroll
    for (int qb = 0; qb < 2; qb++) {
      int r = row0 + 16 * qb + c;
      r = r < rows ? r : rows - 1;
      const int tok = (int)div_by((uint32_t)r, p.by_group), h = kvh * p.w.group + r - tok * p.w.group;
      const char* src = p.w.q + (int64_t)(lo + tok) * p.q_st + (int64_t)h * p.q_sh + g * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) qreg[qb][ks] = *(const u32x4*)(src + ks * 64);
#pragma unroll
      for (int db = 0; db < NDB; db++) oacc[qb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
      l_pv[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[qb] = -INFINITY, l_run[qb] = 0.f;
    }
    typedef int Slots __attribute__((ext_vector_type(NI), aligned(4)));
    int slot[NI];
    // The slots of the lane's rows of tile t, neighbours in the table (LDS row 16 wave + RPI i + j is key 16 wave + NI j + i); positions past the prefix repeat its last one.
    // (the tile's place in the row is the wave's, with 64 bits: a row may be longer than 2^30 entries)
    const int of_tile = 16 * wave + NI * j_row;
    const uint32_t pos0 = (uint32_t)(block0 * kKeys + of_tile);
    auto load_slots = [&](int t) __attribute__((always_inline)) {
      const int start = (block0 + t) * kKeys;
      if (start + kKeys <= prefix) {  // (wave-uniform)
        const Slots x = *(const Slots*)(row_slots + start + of_tile);
#pragma unroll
        for (int i = 0; i < NI; i++) slot[i] = x[i];
      } else {
#pragma unroll
        for (int i = 0; i < NI; i++) slot[i] = row_slots[start + of_tile + i < prefix ? start + of_tile + i : prefix - 1];
      }
    };
    // The rows of tile t.  What stands here is issued by every wave for every tile, so the common case, all 64 keys there, is kept short: offsets of 32 bits where the pool allows
    // them (one full-rate multiplication each), and masks that are written only where they change.
    uint32_t masked = 0;  // stages whose mask is not all ones
    auto request = [&](int stage, int t) __attribute__((always_inline)) {
      const int dst = __builtin_amdgcn_readfirstlane(lds_base + stage * 2 * TB + wave * 16 * RB);
      bool ok = true;
#pragma unroll
      for (int i = 0; i < NI; i++) ok &= (uint32_t)slot[i] < (uint32_t)p.w.num_slots;
      const bool whole = (block0 + t + 1) * kKeys <= prefix && __builtin_amdgcn_ballot_w64(!ok) == 0;
      if (!whole || ((masked >> stage) & 1u)) {  // (wave-uniform)
        uint32_t there = 0;  // bit per LDS row of the wave
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const bool here = pos0 + t * kKeys + i < (uint32_t)prefix && (uint32_t)slot[i] < (uint32_t)p.w.num_slots;
          const uint64_t lanes = __builtin_amdgcn_ballot_w64(here);
#pragma unroll
          for (int j = 0; j < RPI; j++) there |= (uint32_t)((lanes >> (CPR * j)) & 1u) << (RPI * i + j);
          slot[i] = here ? slot[i] : 0;
        }
        if (lane == 0) *(uint16_t*)(lds + kMaskOff + stage * 8 + wave * 2) = (uint16_t)there;
        masked = whole ? masked & ~(1u << stage) : masked | 1u << stage;
      }
      auto send = [&](auto once) __attribute__((always_inline)) {
        if (p.near) {
#pragma unroll
          for (int i = 0; i < NI; i++) {
            const uint32_t ko = __umul24((uint32_t)slot[i], k_s0) + (k_chunk ^ (swz_k(RPI * i) * 16)), vo = __umul24((uint32_t)slot[i], v_s0) + (v_chunk ^ (swz_v(RPI * i) * 16));
            if (decltype(once)::value)
              asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4 nt\n\t"
                           "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5 nt" ::"s"(dst + i * 1024), "s"(dst + TB + i * 1024), "v"(ko), "v"(vo), "s"(kb), "s"(vb)
                           : "m0", "memory");
            else
              asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4\n\t"
                           "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5" ::"s"(dst + i * 1024), "s"(dst + TB + i * 1024), "v"(ko), "v"(vo), "s"(kb), "s"(vb)
                           : "m0", "memory");
          }
        } else {
#pragma unroll
          for (int i = 0; i < NI; i++) {
            const char* ka = kb + (uint64_t)(uint32_t)slot[i] * k_s0 + (k_chunk ^ (swz_k(RPI * i) * 16));
            const char* va = vb + (uint64_t)(uint32_t)slot[i] * v_s0 + (v_chunk ^ (swz_v(RPI * i) * 16));
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\t"
                         "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, off" ::"s"(dst + i * 1024), "s"(dst + TB + i * 1024), "v"(ka), "v"(va)
                         : "m0", "memory");
          }
        }
      };
      // (rows that one row tile reads are read once: nontemporal, 24 requests of 32/32 heads 105 -> 97 us; of a group of several tiles they come from the L2 for the others: 64 requests behind 32768
      // tokens 70 us, 77 with nontemporal loads)
      if (tiles == 1) send(std::true_type{});
      else send(std::false_type{});
    };
    __syncthreads();  // (the tiles of the segment before are done with)
    if (lane < 2) *(uint16_t*)(lds + kMaskOff + lane * 8 + wave * 2) = 0xffff;
    load_slots(0);
    request(0, 0);
    load_slots(1);
    auto step = [&](auto stage_tag, int t) __attribute__((always_inline)) {
      constexpr int S = decltype(stage_tag)::value;
      wait_loads<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (t + 1 < nt) {
        request(S ^ 1, t + 1);
        load_slots(t + 2);
      }
      const uint64_t mask64 = *(const uint64_t*)(lds + kMaskOff + S * 8);
      const uint32_t mask[2] = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)mask64), (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(mask64 >> 32))};
      if ((mask[0] & mask[1]) != 0xffffffffu) {  // (the same for the whole workgroup)
        // (what lies in the slot that was read in place of one that does not exist may be infinite or NaN, and 0 times that is NaN)
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const int r = RPI * i + j_row;
          if (!((mask[wave >> 1] >> (16 * (wave & 1) + r)) & 1u))
            *(u32x4*)(lds + S * 2 * TB + TB + wave * 16 * RB + i * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if (!active) return;
#pragma unroll
      for (int part32 = 0; part32 < 2; part32++) {
        u32x4 ka[2][KS];
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
          for (int ks = 0; ks < KS; ks++)
            ka[kk][ks] = *(const __attribute__((address_space(3))) u32x4*)(kaddr[ks] + S * 2 * TB + (32 * part32 + 16 * kk) * RB);
        f32x4 s[2][2];
#pragma unroll
        for (int qb = 0; qb < 2; qb++) s[qb][0] = s[qb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
          for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int qb = 0; qb < 2; qb++) s[qb][kk] = mfma<T>(ka[kk][ks], qreg[qb][ks], s[qb][kk]);
        if (mask[part32] != 0xffffffffu) {
          const uint32_t mine = mask[part32] >> (4 * g);
#pragma unroll
          for (int qb = 0; qb < 2; qb++)
#pragma unroll
            for (int e = 0; e < 8; e++) s[qb][e / 4][e % 4] = (mine >> (16 * (e / 4) + e % 4)) & 1u ? s[qb][e / 4][e % 4] : -INFINITY;
        }
        u32x4 pk[2][NP];
        float ps[2];
        auto compute_p = [&](int qb, float neg_m) __attribute__((always_inline)) {
          float pv[8];
#pragma unroll
          for (int e = 0; e < 8; e++) pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qb][e / 4][e % 4], scale, neg_m));
          ps[qb] = ((pv[0] + pv[1]) + (pv[2] + pv[3])) + ((pv[4] + pv[5]) + (pv[6] + pv[7]));
#pragma unroll
          for (int e = 0; e < 4; e++) {
            pk[qb][0][e] = pack2<T>(pv[2 * e], pv[2 * e + 1]);
            if constexpr (HIGH_LOW) {
              float a, b;
              unpack2<T>(pk[qb][0][e], a, b);
              pk[qb][NP - 1][e] = pack2<T>(pv[2 * e] - a, pv[2 * e + 1] - b);
            }
          }
        };
        bool over = false;
#pragma unroll
        for (int qb = 0; qb < 2; qb++) {
          compute_p(qb, -m_run[qb]);
          over |= !(ps[qb] < 32768.f);
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(over) != 0, 0)) {
#pragma unroll
          for (int qb = 0; qb < 2; qb++) {
            const float mx = fmaxf(fmaxf(fmaxf(s[qb][0][0], s[qb][0][1]), fmaxf(s[qb][0][2], s[qb][0][3])),
                                   fmaxf(fmaxf(s[qb][1][0], s[qb][1][1]), fmaxf(s[qb][1][2], s[qb][1][3])));
            const float m_new = fmaxf(m_run[qb], col_max(mx) * scale - kPrefixHead);
            const float alpha = exp2_diff(m_run[qb], m_new);
            l_run[qb] *= alpha;
            l_pv[qb] *= alpha;
#pragma unroll
            for (int db = 0; db < NDB; db++) oacc[qb][db] *= alpha;
            m_run[qb] = m_new;
            compute_p(qb, m_new == -INFINITY ? 0.f : -m_new);  // (a row that has seen no key: every weight is 0)
          }
        }
#pragma unroll
        for (int qb = 0; qb < 2; qb++) l_run[qb] += ps[qb];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int db = 0; db < NDB; db++) {
          const int va_at = vaddr[db] + S * 2 * TB + 32 * part32 * RB;
          const i16x4 xa = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr)va_at);
          const i16x4 xb = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr)(va_at + 16 * RB));
          const u32x2 wa = __builtin_bit_cast(u32x2, xa), wb = __builtin_bit_cast(u32x2, xb);
          const u32x4 va = u32x4{wa[0], wa[1], wb[0], wb[1]};
#pragma unroll
          for (int qb = 0; qb < 2; qb++)
#pragma unroll
            for (int n = 0; n < NP; n++) oacc[qb][db] = mfma<T>(va, pk[qb][n], oacc[qb][db]);
        }
        if constexpr (!HIGH_LOW) {
          constexpr uint32_t kOnes = 0x3C003C00u;
#pragma unroll
          for (int qb = 0; qb < 2; qb++) l_pv[qb] = mfma<T>(u32x4{kOnes, kOnes, kOnes, kOnes}, pk[qb][0], l_pv[qb]);
        }
      }
    };
    for (int t = 0; t < nt; t += 2) {
      step(std::integral_constant<int, 0>{}, t);
      if (t + 1 < nt) step(std::integral_constant<int, 1>{}, t + 1);
    }
    if (active && part < p.parts) {
#pragma unroll
      for (int qb = 0; qb < 2; qb++) {
        const float l_tot = col_sum(l_run[qb]);
        const float l_of_v = HIGH_LOW ? l_tot : l_pv[qb][0];
        const float inv = l_of_v == 0.f ? 0.f : 1.f / l_of_v;
        const int r = row0 + 16 * qb + c;
        if (r < rows) {
          const int64_t to = ((int64_t)kvh * p.parts + part) * kRows + (r - tile * kRows);
          float* dst = p.pre_o + to * D + 4 * g;
#pragma unroll
          for (int db = 0; db < NDB; db++) {
            if constexpr (THROUGH) store16_through(dst + 16 * db, oacc[qb][db] * inv);
            else *(f32x4*)(dst + 16 * db) = oacc[qb][db] * inv;
          }
          if (g == 0) p.pre_lse[to] = l_tot > 0.f ? m_run[qb] + __builtin_amdgcn_logf(l_tot) : (l_tot == l_tot ? -INFINITY : l_tot);
        }
      }
    }
    at += deal.cut ? p.shares : nt;
  }
}

// ------------------------------------------------------------------------------------------------ the requests' own tokens
// Blocks of own tokens of all requests, numbered request by request; 64 requests at a time, of which a lane has one each.  A request that is shorter than its group's prefix
// shares nothing.
struct OwnRequests {
  int first_request, len, req, n_own, units, up_to;
  Membership group;
  bool shares;  // whether it has its group's prefix
  __device__ __forceinline__ void look(const SharedParams& p, Groups& g, int b0) {
    const int lane = threadIdx.x & 63, b = b0 + lane;
    first_request = b0;
    len = req = n_own = 0;
    if (b < p.w.batch) n_own = visible(p.w, b, len, req);
    group.find(p, g, b);
    shares = group.prefix <= len;
    n_own -= shares && b < p.w.batch ? group.prefix : 0;
    units = (n_own + kBlock - 1) / kBlock;
    up_to = scan_sum(units);
  }
  __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(up_to, 63); }
};
__device__ __forceinline__ int per_own_share(const PoolParams& p, int total) {
  const int per = (int)div_by((uint32_t)(total + p.shares - 1), p.by_shares);
  return per < p.min_units ? p.min_units : per;
}

template <typename T, int D> __device__ __forceinline__ void own_share(const SharedParams& sp, char* lds, int share, int task) {
  const PoolParams& p = sp.w;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Groups gs;
  gs.look(sp, 0, 0);
  OwnRequests rs;
  rs.look(sp, gs, 0);
  int total = rs.all();
  if (p.batch > 64) {
    for (int b0 = 64; b0 < p.batch; b0 += 64) rs.look(sp, gs, b0), total += rs.all();
    rs.look(sp, gs, 0);
  }
  const int per_share = per_own_share(p, total);
  // Where every request's partials lie, for the launch that joins them: 64 requests per wave, by the first task's waves.
  if (task == 0) {
    const Deal deal = deal_of(sp, gs);
    for (int b0 = 0, before = 0; b0 < p.batch; b0 += 64) {
      if (rs.first_request != b0) rs.look(sp, gs, b0);
      const int b = b0 + (threadIdx.x & 63);
      const PlanRow row(rs.group, gs, deal);
      if ((b0 >> 6) % p.shares == share && b < p.batch) {
        const int u0 = before + rs.up_to - rs.units, s0 = u0 / per_share;
        row.put(sp, b, rs.shares, s0, rs.units ? (u0 + rs.units - 1) / per_share - s0 + 1 : 0);
      }
      before += rs.all();
    }
    if (rs.first_request) rs.look(sp, gs, 0);
  }
  if ((int64_t)share * per_share >= total) return;
  int at = share * per_share;
  const int end = total - at < per_share ? total : at + per_share;
  int first = 0;
  while (at >= first + rs.all()) {
    first += rs.all();
    rs.look(sp, gs, rs.first_request + 64);
  }
  int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(first + rs.up_to > at));
  first += __builtin_amdgcn_readlane(rs.up_to, l) - __builtin_amdgcn_readlane(rs.units, l);
  Walk<T, T, D> w(p, lds + wave * kWaveLds<T, D>);
  const int kvh = (int)div_by((uint32_t)task, p.by_sub), sg = task - kvh * p.sub_groups;
  const int h0 = kvh * p.group + sg * kHeads;
  const int nh = p.group - sg * kHeads < kHeads ? p.group - sg * kHeads : kHeads;
  for (;;) {
    const int b = rs.first_request + l, units = __builtin_amdgcn_readlane(rs.units, l), n_own = __builtin_amdgcn_readlane(rs.n_own, l);
    const int to = end - first < units ? end : first + units;
    if (to > at) {
      w.start(b, __builtin_amdgcn_readlane(rs.req, l), task, __builtin_amdgcn_readlane(rs.len, l), n_own);
      const int last = (to - first) * kBlock;
      w.run((at - first) * kBlock, last < n_own ? last : n_own, 1);
      w.join();
      if (w.c < nh) {
        const int64_t r0 = ((int64_t)(share + b) * p.hq + h0 + w.c);
        const float inv = w.l == 0.f ? 0.f : 1.f / w.l;
        float* dst = p.part_o + r0 * D;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int j = 0; j < D / 16; j += 4)
            *(f32x4*)(dst + (D / 16) * (4 * w.g + r) + j) = f32x4{w.acc[j][r], w.acc[j + 1][r], w.acc[j + 2][r], w.acc[j + 3][r]} * inv;
        if (w.g == 0) p.part_lse[r0] = w.l > 0.f ? w.m + __builtin_amdgcn_logf(w.l) : (w.l == w.l ? -INFINITY : w.l);  // (log2 domain)
      }
      at = to;
    }
    if (at >= end) return;
    first += units;
    if (++l == 64) rs.look(sp, gs, rs.first_request + 64), l = 0;
  }
}

// Workgroups of the own tokens first, four waves with a share each, then those of the prefix part.  Prompts (!OWN) have no such tokens here.
template <typename T, int D> constexpr int kSharedLds = kPrefixLds<T, D> > 4 * kWaveLds<T, D> ? kPrefixLds<T, D> : 4 * kWaveLds<T, D>;
template <typename T, int D, bool OWN>
__global__ __launch_bounds__(256, 2) void shared_prefix_kernel(SharedParams p) {
  __shared__ __attribute__((aligned(1024))) char lds[OWN ? kSharedLds<T, D> : kPrefixLds<T, D>];
  if ((int)blockIdx.x >= p.own_wgs) {
    const uint32_t x = blockIdx.x - p.own_wgs;  // (a multiple of 8)
    // ids are dealt to the XCDs round-robin; the workgroups of a KV head that run on one XCD take neighbouring shares
    const int i = (int)div_by(x, p.by_hkv), share = (i & ((1 << p.xcds_shift) - 1)) * (p.shares >> p.xcds_shift) + (i >> p.xcds_shift);
    prefix_share<T, D, !OWN>(p, lds, (int)x - i * p.w.hkv, share);
    return;
  }
  if constexpr (OWN) {
    const uint32_t x = blockIdx.x;
    const uint32_t unit = ((x & 7) * (p.own_wgs >> 3) + (x >> 3)) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int share = (int)div_by(unit, p.w.by_tasks), task = (int)(unit - (uint32_t)share * p.w.tasks);
    if (share < p.w.shares) own_share<T, D>(p, lds, share, task);
  } else {  // (prompts: these workgroups write the plan)
    Groups gs;
    gs.look(p, 0, 0);
    const Deal deal = deal_of(p, gs);
    for (int b0 = (int)blockIdx.x * 256; b0 < p.rows; b0 += p.own_wgs * 256) {
      const int b = b0 + threadIdx.x;
      Membership m;
      m.find(p, gs, b < p.rows ? b : p.rows - 1);
      const PlanRow row(m, gs, deal);
      if (b < p.rows) row.put(p, b, true, 0, 0);
    }
  }
}

// The partials of a request's row: those of its group's prefix, then those of its own tokens.
struct MergeRow {
  int n, n_pre, pre_step;
  int64_t pre_row, own_row;
  __device__ __forceinline__ MergeRow(const SharedParams& sp, int b, int h) {
    const int32_t* const plan = sp.plan + kPlanInts * (int64_t)b;
    const int kvh = (int)div_by((uint32_t)h, sp.by_group);
    const int r = (b - plan[0]) * sp.w.group + (h - kvh * sp.w.group), tile = r / kRows;
    const Partials pre = partials_of(Deal{plan[6], plan[7], 0}, tile, plan[1], plan[2], plan[3], plan[8], plan[9]);
    n_pre = pre.n, n = pre.n + plan[5], pre_step = pre.step * kRows;
    pre_row = ((int64_t)kvh * sp.parts + pre.first) * kRows + (r - tile * kRows), own_row = (int64_t)(plan[4] + b) * sp.w.hq + h;
  }
  __device__ __forceinline__ float lse(const SharedParams& sp, int i) const {
    return i < n_pre ? sp.pre_lse[pre_row + (int64_t)i * pre_step] : sp.w.part_lse[own_row + (int64_t)(i - n_pre) * sp.w.hq];
  }
  __device__ __forceinline__ const float* row(const SharedParams& sp, int i, int d) const {
    return i < n_pre ? sp.pre_o + (pre_row + (int64_t)i * pre_step) * d : sp.w.part_o + (own_row + (int64_t)(i - n_pre) * sp.w.hq) * d;
  }
};
// Maximum and sum over the wave, in every lane: within rows of 16 lanes by DPP, then of the four rows.
__device__ __forceinline__ float of_row(float v, int row) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16 * row)); }
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_mov<0xB1>(v)), v = fmaxf(v, dpp_mov<0x4E>(v)), v = fmaxf(v, dpp_mov<0x141>(v)), v = fmaxf(v, dpp_mov<0x140>(v));
  return fmaxf(fmaxf(of_row(v, 0), of_row(v, 1)), fmaxf(of_row(v, 2), of_row(v, 3)));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = sum_row16(v);
  return (of_row(v, 0) + of_row(v, 1)) + (of_row(v, 2) + of_row(v, 3));
}
// o = sum of a row's partials by their log-sum-exps, by WAVES waves a row: each of them finds all weights for itself, 64 at a time in its lanes, so that its rows' loads wait for no other, and
// takes every WAVES-th of the partials.
template <int D, int WAVES>
__global__ __launch_bounds__(256) void shared_decode_merge_kernel(SharedParams sp) {
  constexpr int W = D / 4, SL = 64 / W, kLoads = WAVES > 1 ? 4 : 8;
  const PoolParams& p = sp.w;
  __shared__ __attribute__((aligned(16))) float acc[WAVES > 1 ? WAVES - 1 : 1][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave & (WAVES - 1);
  const int i0 = (int)blockIdx.x * (4 / WAVES) + wave / WAVES;
  const int b = (int)div_by((uint32_t)i0, sp.by_hq), h = i0 - b * p.hq;
  if (b >= p.batch) return;  // (WAVES of 4: every workgroup has a row)
  const MergeRow m(sp, b, h);
  float M = -INFINITY;
  for (int i = lane; i < m.n; i += 64) M = fmaxf(M, m.lse(sp, i));
  M = wave_max(M);
  float L = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const int slice = lane / W, d = (lane & (W - 1)) * 4;
  for (int i1 = 0; i1 < m.n; i1 += 64) {
    const float weight = i1 + lane < m.n ? exp2_diff(m.lse(sp, i1 + lane), M) : 0.f;  // (NaN stays NaN)
    L += weight;
    const int n = m.n - i1 < 64 ? m.n - i1 : 64;
    for (int k0 = part * SL; k0 < n; k0 += kLoads * WAVES * SL) {  // (by the whole wave: a lane that has left the loop would hand out no weight)
      f32x4 x[kLoads];
#pragma unroll
      for (int u = 0; u < kLoads; u++) {
        const int k = k0 + u * WAVES * SL + slice;
        x[u] = *(const f32x4*)(m.row(sp, i1 + (k < n ? k : n - 1), D) + d);
      }
#pragma unroll
      for (int u = 0; u < kLoads; u++) {
        const int k = k0 + u * WAVES * SL + slice;
        const float w = __shfl(weight, k & 63, 64);
        if (k < n) sum += x[u] * w;
      }
    }
  }
  L = wave_sum(L);
#pragma unroll
  for (int x = 32; x >= W; x >>= 1)
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] += __shfl_xor(sum[e], x, 64);
  if constexpr (WAVES > 1) {
    if (part && slice == 0) *(f32x4*)&acc[part - 1][d] = sum;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int k = 0; k < WAVES - 1; k++) sum += *(const f32x4*)&acc[k][d];
  }
  if (slice) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t at = (int64_t)b * p.hq + h;
  store_elem4(p.o, p.o_dtype, at * D + d, sum * inv);
  if (d == 0) p.lse[at] = ln_of(M, L);
}

// The prompts' step: a row's partials by their log-sum-exps, folded into the running (o, m, l) as context_attention_fwd's kernels do
// (ring_context_flashattention_nopad.py:171-188).  D / 4 lanes have a (row, head); rows of no group, or whose prefix shows them no key, stay as they are.
struct FoldParams {
  char* o;
  int64_t o_st, o_sh;  // bytes
  float* m;
  float* l;
  int64_t ml_st, ml_sh;
};
template <typename T, int D> __global__ __launch_bounds__(256) void shared_prefix_fold_kernel(SharedParams sp, FoldParams f) {
  constexpr int W = D / 4;
  const int i = (int)blockIdx.x * (256 / W) + threadIdx.x / W, x = threadIdx.x & (W - 1);
  const int b = (int)div_by((uint32_t)i, sp.by_hq), h = i - b * sp.w.hq;
  if (b >= sp.rows) return;
  const MergeRow r(sp, b, h);
  if (!r.n) return;
  float M = -INFINITY;
  for (int j = x; j < r.n; j += W) M = fmaxf(M, r.lse(sp, j));
#pragma unroll
  for (int d = W / 2; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
  const int64_t ml = (int64_t)b * f.ml_st + (int64_t)h * f.ml_sh;
  const float m_old = f.m[ml], l_old = f.l[ml];
  const float top = fmaxf(M, m_old);
  float L = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int j = 0; j < r.n; j++) {
    const float w = exp2_diff(r.lse(sp, j), top);
    L += w;
    sum += *(const f32x4*)(r.row(sp, j, D) + 4 * x) * w;
  }
  if (L == 0.f) return;
  const float w_old = l_old * exp2_diff(m_old, top);
  uint16_t* o = (uint16_t*)(f.o + (int64_t)b * f.o_st + (int64_t)h * f.o_sh) + 4 * x;
  if (w_old != 0.f) {  // (a row in its start state may hold anything)
    const u32x2 old = *(const u32x2*)o;
    float x0, x1, x2, x3;
    unpack2<T>(old[0], x0, x1);
    unpack2<T>(old[1], x2, x3);
    sum += f32x4{x0, x1, x2, x3} * w_old;
    L += w_old;
  }
  sum *= 1.f / L;
  *(u32x2*)o = u32x2{pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3])};
  if (x == 0) f.m[ml] = top, f.l[ml] = L;
}

// Many rows: the prefixes as contiguous K/V for the prefill kernel, group g's from row g * most on.
struct GatherParams {
  char* k;
  char* v;           // [groups * most, hkv, D]; V of bfloat16 as the fp16 copy that the prefill kernel multiplies
  int32_t* list;     // [groups, most] slots
  int32_t* vectors;  // the six vectors of the step, [6, groups]
  int32_t most;      // as SharedParams::most
  FastDiv by_head_chunks;
};
// A group's slots in the table's order without the entries that name none, and the vectors of the step.  One workgroup per group, 4096 entries at a time.
__global__ __launch_bounds__(1024) void shared_prefix_list_kernel(SharedParams p, GatherParams a) {
  __shared__ int sums[2][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = blockIdx.x;
  Groups gs;
  for (int g0 = 0, end = 0;; g0 += 64, end = gs.end_of_all()) {
    gs.look(p, g0, end);
    if (g < g0 + 64) break;
  }
  const int l = g & 63, lo = __builtin_amdgcn_readlane(gs.lo, l), size = __builtin_amdgcn_readlane(gs.size, l);
  const int prefix = __builtin_amdgcn_readlane(gs.prefix, l);
  const int32_t* const slots = p.w.table + (int64_t)__builtin_amdgcn_readlane(gs.req, l) * p.w.max_seq_len;
  int32_t* const list = a.list + (int64_t)g * a.most;
  int count = 0, set = 0;
  for (int at = 0; at < prefix; at += 4096, set ^= 1) {
    int slot[4], mine = 0;
    bool ok[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = at + 4 * (int)threadIdx.x + e;
      slot[e] = i < prefix ? slots[i] : -1;
      ok[e] = (uint32_t)slot[e] < (uint32_t)p.w.num_slots;
      mine += ok[e];
    }
    int up_to = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int below = __shfl_up(up_to, d, 64);
      if (lane >= d) up_to += below;
    }
    if (lane == 63) sums[set][wave] = up_to;
    __syncthreads();
    int rank = count + up_to - mine;
#pragma unroll
    for (int w = 0; w < 16; w++) {
      rank += w < wave ? sums[set][w] : 0;
      count += sums[set][w];
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (ok[e]) list[rank++] = slot[e];
  }
  if (threadIdx.x == 0) {
    int32_t* v = a.vectors + g;
    v[0] = size ? lo : 0;             // q_b_start_loc
    v[p.groups] = size;               // q_b_seq_len
    v[2 * p.groups] = a.most;         // the rows' position: behind every key
    v[3 * p.groups] = g * a.most;     // kv_b_start_loc
    v[4 * p.groups] = count;          // kv_b_seq_len
    v[5 * p.groups] = 0;
  }
}
// A thread has 16 bytes of a row.
template <typename T> __global__ __launch_bounds__(256) void shared_prefix_gather_kernel(SharedParams p, GatherParams a, uint32_t head_chunks) {
  const uint32_t chunks = 2 * p.w.hkv * head_chunks;  // of a token
  const int g = blockIdx.y;
  const int32_t* const list = a.list + (int64_t)g * a.most;
  const int64_t total = (int64_t)a.vectors[4 * p.groups + g] * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const uint32_t t = (uint32_t)(i / chunks), x = (uint32_t)(i - (int64_t)t * chunks), hh = div_by(x, a.by_head_chunks), cc = x - hh * head_chunks;
    const bool is_v = hh >= (uint32_t)p.w.hkv;
    const uint32_t head = is_v ? hh - p.w.hkv : hh, slot = (uint32_t)list[t];
    const char* src = is_v ? p.w.v + (uint64_t)slot * (uint32_t)p.w.v_s0 + head * p.w.v_s1 : p.w.k + (uint64_t)slot * (uint32_t)p.w.k_s0 + head * p.w.k_s1;
    u32x4 v = *(const u32x4*)(src + cc * 16);
    if (__is_same(T, BF16) && is_v) {  // round toward zero: exact in fp16's normal range, larger magnitudes become +-65504
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float lo, hi;
        unpack2<BF16>(v[e], lo, hi);
        v[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
      }
    }
    *(u32x4*)((is_v ? a.v : a.k) + ((((int64_t)g * a.most + t) * p.w.hkv + head) * head_chunks + cc) * 16) = v;
  }
}

// ------------------------------------------------------------------------------------------------ the host's side
constexpr int64_t kPrefixWorkgroups = 2 * kCUs;  // at most
constexpr int kPlanWorkgroups = 8;  // in front of a prompts' step (a multiple of the XCDs)
constexpr int64_t kRounds = 3;  // pieces per workgroup, at most
constexpr int64_t kOwnWaves = 4 * kCUs;
constexpr int64_t kOwnMinUnits = 2;

// a bound of the prefixes that a table can hold
int64_t most_of(int64_t max_prefix, int64_t max_seq_len) { return max_prefix < max_seq_len ? max_prefix : max_seq_len; }

bool is_near(const PoolParams& w) {
  const int64_t last = (int64_t)w.num_slots - 1;
  return w.num_slots <= 1 << 24 && w.k_s0 < 1 << 24 && w.v_s0 < 1 << 24 && last * w.k_s0 < 0x7fff0000 && last * w.v_s0 < 0x7fff0000;
}
struct Plan {
  int64_t tiles, shares, parts, rounds, xcds_shift;  // prefix part, per KV head
  bool ahead;
  int64_t own_shares;
  int64_t pre_floats, own_floats, plan_ints;  // of the workspace
  int64_t all() const { return (pre_floats + own_floats + plan_ints) * 4; }
};
// `own`: the bound of a request's own tokens (0: no own part)
Plan plan_of(int64_t rows, int64_t groups, int64_t hq, int64_t hkv, int64_t d, int64_t max_prefix, int64_t max_own, bool decode) {
  Plan p;
  p.tiles = groups > 0 && max_prefix > 0 ? rows * (hq / hkv) / kRows + (groups < rows ? groups : rows) : 0;
  const int64_t units = p.tiles * ((max_prefix + kKeys - 1) / kKeys);
  const int64_t tasks = hkv * ((hq / hkv + kHeads - 1) / kHeads), own_units = decode ? rows * ((max_own + kBlock - 1) / kBlock) : 0;
  // The two parts of a decode step beside each other, where the groups fill their row tiles.  Blocks of own tokens and units of the prefix cost about the same, so their ratio says
  // which part is the longer one (us; 32/8 heads of 128 if not said):
  // * of 128-wide heads a SIMD holds two waves: one workgroup of each part per CU, not two of the prefix part, unless that has nearly all the work: 64 requests behind 16384 tokens, up to
  //   1500 own tokens 79 | 68, 200 54 | 52; behind 24000, 200 own 64 | 66.  Of 64-wide ones it holds three: always two (160 in two groups, 28/4 heads, up to 800 own tokens 76 | 96).
  //   Rows that do not fill a tile: what counts is loads in flight (24 in three groups, 32/32 heads, 105 | 113; 64 in four groups, up to 400 own tokens 80 | 94).
  // * the prefix part's waves come first, as long as it is not much the shorter one: each of its matrix instructions waits for a turn among the other part's vector work, which waits for memory
  //   all the same: 64 behind 16384 tokens, up to 1500 own 77 | 68; 160 in two groups, 28/4 of 64, up to 3000 own 95 | 89; but 64 behind 8192, up to 3000 own 88 | 93.
  const bool full = decode && rows * (hq / hkv) >= kRows * groups;
  const bool beside = full && d == 128 && own_units * tasks * 2 >= units * hkv;
  p.ahead = full && own_units * tasks <= units * hkv * 6;
  p.shares = (beside ? kCUs : kPrefixWorkgroups) / hkv;
  p.shares = p.shares < 1 ? 1 : p.shares;
  p.shares = p.shares < units ? p.shares : units < 1 ? 1 : units;
  p.xcds_shift = hkv % 8 == 0 ? 0 : hkv % 4 == 0 ? 1 : hkv % 2 == 0 ? 2 : 3;
  if (p.shares >> p.xcds_shift >= 8) p.shares = p.shares >> p.xcds_shift << p.xcds_shift;  // (as many on each of the XCDs, and not many fewer for it)
  else p.xcds_shift = 0;
  // (no group has more rows than there are; code that is not run is not fetched: a small launch is 1 us shorter)
  p.rounds = rows * (hq / hkv) <= kRows ? 0 : p.tiles * 6 <= kPrefixWorkgroups / hkv ? 1 : kRounds;
  auto parts = [&](int64_t shares) { return shares + p.tiles > p.rounds * shares ? shares + p.tiles : p.rounds * shares; };
  p.parts = parts(p.shares);
  // (room for the partials of the most workgroups that a launch of these sizes or smaller ones takes, so that a workspace for the largest sizes does for all)
  int64_t most_shares = kPrefixWorkgroups / hkv;
  most_shares = most_shares < 1 ? 1 : most_shares;
  most_shares = most_shares < units ? most_shares : units < 1 ? 1 : units;
  p.pre_floats = p.tiles ? hkv * parts(most_shares) * kRows * (d + 1) : 0;
  p.own_shares = 1, p.own_floats = 0, p.plan_ints = kPlanInts * rows;
  if (decode) {
    const int64_t by_waves = kOwnWaves / tasks, by_units = (own_units + kOwnMinUnits - 1) / kOwnMinUnits;
    p.own_shares = by_waves < by_units ? by_waves : by_units;
    p.own_shares = p.own_shares < 1 ? 1 : p.own_shares;
    p.own_floats = ((p.own_shares + rows) * hq * (d + 1) + 3) / 4 * 4;
  }
  return p;
}

// Rows from which the launch that joins them has a wave per row instead of four (us, four | one): 32 heads of 128, 4 requests 3.9 | 5.4, 32 6.5 | 5.8, 64 6.5 | 6.7, 160 12.5 | 7.0; 28 heads of
// 64, 16 requests 4.9 | 6.1, 64 5.8 | 5.8, 160 10.7 | 6.6.
constexpr int64_t kMergeByWaves = 4096;
template <typename T, int D> void launch_decode(const SharedParams& p, hipStream_t st) {
  const int64_t prefix = p.groups ? (int64_t)p.shares * p.w.hkv : 0;
  LSATTN_LAUNCH_KERNEL((shared_prefix_kernel<T, D, true>), dim3((unsigned)(p.own_wgs + prefix)), dim3(256), 0, st, p);
  if (hipPeekAtLastError() != hipSuccess) return;
  const int64_t rows = (int64_t)p.w.batch * p.w.hq;
  if (rows >= kMergeByWaves) LSATTN_LAUNCH_KERNEL((shared_decode_merge_kernel<D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
  else LSATTN_LAUNCH_KERNEL((shared_decode_merge_kernel<D, 4>), dim3((unsigned)rows), dim3(256), 0, st, p);
}

}  // namespace
}  // namespace lsattn

using namespace lsattn;

extern "C" size_t lsattn_shared_decode_workspace_bytes(int64_t batch, int64_t num_groups, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                                       int64_t max_prefix_len, int64_t max_own_len) {
  if (batch <= 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || (head_dim != 64 && head_dim != 128) ||
      max_prefix_len < 0 || max_own_len < 0 || batch > 65535 || num_groups > 0x7fffff00 || num_q_heads > 65535 || max_prefix_len > 0x7fffffff ||
      max_own_len > 0x7fffffff)  // (as the launch refuses)
    return 0;
  const Plan pl = plan_of(batch, num_groups, num_q_heads, num_kv_heads, head_dim, max_prefix_len, max_own_len, true);
  return (size_t)pl.all();
}

extern "C" int lsattn_shared_decode(const lsattn_shared_decode_args* a, void* stream) {
  if (!a || !a->q || !a->k || !a->v || !a->o || !a->lse || !a->req_to_tokens || !a->b_req_idx || !a->b_seqlen) return LSATTN_ERR_INVALID_ARG;
  if (a->batch < 0 || a->num_q_heads < 1 || a->num_kv_heads < 1 || a->num_slots < 1 || a->num_reqs < 0 || a->max_seq_len < 0 || a->num_groups < 0 ||
      a->max_prefix_len < 0 || a->max_own_len < 0)
    return LSATTN_ERR_INVALID_ARG;
  if (a->num_groups && (!a->g_start_loc || !a->g_size || !a->g_req_idx || !a->g_prefix_len)) return LSATTN_ERR_INVALID_ARG;
  if (a->num_q_heads % a->num_kv_heads || (a->head_dim != 128 && a->head_dim != 64)) return LSATTN_ERR_UNSUPPORTED;
  if (a->o_dtype != LSATTN_F32 && a->o_dtype != LSATTN_F16 && a->o_dtype != LSATTN_BF16) return LSATTN_ERR_UNSUPPORTED;
  if (a->dtype != LSATTN_F16 && a->dtype != LSATTN_BF16) return LSATTN_ERR_UNSUPPORTED;
  if ((a->k_stride_0 * 2) % 16 || (a->k_stride_1 * 2) % 16 || (a->v_stride_0 * 2) % 16 || (a->v_stride_1 * 2) % 16 ||
      (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->o) & 15))
    return LSATTN_ERR_INVALID_ARG;
  // (offsets are a slot times a stride of 32 bits)
  auto slot_stride = [](int64_t elements) { return elements >= 0 && elements <= 0x3fffffff; };
  if (!slot_stride(a->k_stride_0) || !slot_stride(a->v_stride_0)) return LSATTN_ERR_INVALID_ARG;
  if (a->batch > 65535 || a->num_q_heads > 65535 || a->max_seq_len > 0x7fff0000 || a->num_slots > 0x7fffffff || a->num_reqs > 0x7fffffff ||
      a->num_groups > 0x7fffff00 || a->max_prefix_len > 0x7fffffff || a->max_own_len > 0x7fffffff)
    return LSATTN_ERR_INVALID_ARG;
  if (!(a->sm_scale > 0.f)) return LSATTN_ERR_INVALID_ARG;
  if (a->batch == 0) return LSATTN_OK;
  const int64_t most = most_of(a->max_prefix_len, a->max_seq_len);
  const Plan pl = plan_of(a->batch, a->num_groups, a->num_q_heads, a->num_kv_heads, a->head_dim, most, a->max_own_len, true);
  if (!a->workspace || a->workspace_bytes < (size_t)pl.all()) return LSATTN_ERR_WORKSPACE;
  if ((uintptr_t)a->workspace & 15) return LSATTN_ERR_INVALID_ARG;
  // (units of both parts are numbered with 31 bits, and requests may be longer than the caller's bound)
  if (pl.tiles * ((most + kKeys - 1) / kKeys) > kMaxUnits - kPrefixWorkgroups ||
      a->batch * ((a->max_seq_len + kBlock - 1) / kBlock) > kMaxUnits - kOwnWaves || a->batch * a->num_q_heads > kMaxUnits)
    return LSATTN_ERR_INVALID_ARG;
  SharedParams p;
  PoolParams& w = p.w;
  w.q = (const char*)a->q, w.k = (const char*)a->k, w.v = (const char*)a->v;
  w.k_s0 = a->k_stride_0 * 2, w.k_s1 = a->k_stride_1 * 2, w.v_s0 = a->v_stride_0 * 2, w.v_s1 = a->v_stride_1 * 2;
  w.ks = w.vs = nullptr, w.ks_s0 = w.ks_s1 = w.vs_s0 = w.vs_s1 = 0;
  w.table = a->req_to_tokens, w.b_req = a->b_req_idx, w.b_len = a->b_seqlen, w.max_seq_len = a->max_seq_len;
  w.batch = (int32_t)a->batch, w.num_reqs = (int32_t)a->num_reqs, w.num_slots = (int32_t)a->num_slots;
  w.hq = (int32_t)a->num_q_heads, w.hkv = (int32_t)a->num_kv_heads, w.group = w.hq / w.hkv;
  w.sub_groups = (w.group + kHeads - 1) / kHeads, w.tasks = w.hkv * w.sub_groups;
  w.window = 0, w.sinks = 0;
  w.scale_log2 = a->sm_scale * kLog2e;
  w.o = (char*)a->o, w.o_dtype = a->o_dtype, w.lse = a->lse;
  w.by_tasks = fast_div((uint32_t)w.tasks), w.by_sub = fast_div((uint32_t)w.sub_groups);
  w.shares = (int32_t)pl.own_shares, w.by_shares = fast_div((uint32_t)pl.own_shares), w.min_units = (int32_t)kOwnMinUnits;
  p.pre_o = (float*)a->workspace, p.pre_lse = p.pre_o + (pl.pre_floats / (a->head_dim + 1)) * a->head_dim;
  w.part_o = p.pre_o + pl.pre_floats, w.part_lse = w.part_o + (pl.own_shares + w.batch) * w.hq * a->head_dim;
  p.plan = (int32_t*)(w.part_o + pl.own_floats);
  p.q_st = a->num_q_heads * a->head_dim * 2, p.q_sh = a->head_dim * 2;
  p.g_start = a->g_start_loc, p.g_size = a->g_size, p.g_req = a->g_req_idx, p.g_prefix = a->g_prefix_len;
  p.groups = pl.tiles ? (int32_t)a->num_groups : 0;
  p.rows = w.batch, p.most = (int32_t)most, p.near = is_near(w);
  p.shares = (int32_t)pl.shares, p.parts = (int32_t)pl.parts, p.rounds = (int32_t)pl.rounds, p.ahead = pl.ahead, p.xcds_shift = (int32_t)pl.xcds_shift, p.own_wgs = (int32_t)(((pl.own_shares * w.tasks + 3) / 4 + 7) / 8 * 8);
  p.by_hkv = fast_div((uint32_t)w.hkv), p.by_hq = fast_div((uint32_t)w.hq), p.by_group = fast_div((uint32_t)w.group), p.by_pre_shares = fast_div((uint32_t)pl.shares);
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == LSATTN_F16) {
    if (a->head_dim == 128) launch_decode<F16, 128>(p, st);
    else launch_decode<F16, 64>(p, st);
  } else {
    if (a->head_dim == 128) launch_decode<BF16, 128>(p, st);
    else launch_decode<BF16, 64>(p, st);
  }
  return check_launch();
}

namespace lsattn {
namespace {
// The prompts' step takes its rows itself where they are few, and hands contiguous K/V to the prefill kernel where its workgroups of 256 rows are a round and a half
// of the CUs and more. Microseconds, own kernel | prefill kernel (f16, 32/8 heads of 128, with the fills of m and l): prefix 6001 tokens: 293 rows 62 | 120, 600 97 | 120, 1200 161 | 211, 2500
// 301 | 341, 5000 594 | 518; 20000 tokens: 1200 455 | 564, 2500 965 | 954, 5000 1907 | 1448; five groups of 1200 rows behind 3000 435 | 331; 8/1 heads, 1200 rows behind 6001 76 | 112.
// Where a prefix has few rows of its own, laying it out costs more than it saves: 8192 rows behind 2000 tokens each, 32/8 heads, 32 groups 455 | 406, 64 591 | 538, 128 633 | 827;
// 32/32 heads, 16 groups 591 | 538, 32 596 | 827.
constexpr int64_t kGatherFromRows = kCUs * 3 / 2 * 256, kGatherFromGroupRows = 512;
bool gathers(int64_t rows, int64_t groups, int64_t hq, int64_t hkv) { return rows * hq >= kGatherFromRows && rows * (hq / hkv) >= groups * kGatherFromGroupRows; }
// the most rows that do not gather, 1 at least
int64_t most_direct_rows(int64_t groups, int64_t hq, int64_t hkv) {
  const int64_t group = hq / hkv, by_all = (kGatherFromRows + hq - 1) / hq, by_group = (groups * kGatherFromGroupRows + group - 1) / group;
  return (by_all > by_group ? by_all : by_group) - 1;
}
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
struct PromptBytes {
  int64_t k, list, vectors, all;
};
PromptBytes prompt_bytes(int64_t groups, int64_t hkv, int64_t d, int64_t most) {
  PromptBytes b;
  b.k = groups * most * hkv * d * 2, b.list = up16(groups * most * 4), b.vectors = up16(6 * groups * 4);
  b.all = 2 * b.k + b.list + b.vectors;
  return b;
}
}  // namespace
}  // namespace lsattn

extern "C" size_t lsattn_shared_prefill_workspace_bytes(int64_t rows, int64_t num_groups, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                                        int64_t max_prefix_len) {
  if (rows <= 0 || num_groups <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || (head_dim != 64 && head_dim != 128) ||
      max_prefix_len <= 0 || rows > 0x7fffff00 || num_groups > 65535 || num_q_heads > 65535 || max_prefix_len > 0x7fff0000)  // (as the launch refuses)
    return 0;
  // (fewer rows of as many groups may be taken the other way, whose room does not follow from this one's)
  const int64_t direct_most = most_direct_rows(num_groups, num_q_heads, num_kv_heads), direct_rows = rows < direct_most ? rows : direct_most;
  const int64_t direct = plan_of(direct_rows, num_groups, num_q_heads, num_kv_heads, head_dim, max_prefix_len, 0, false).all();
  const int64_t laid_out = gathers(rows, num_groups, num_q_heads, num_kv_heads) ? prompt_bytes(num_groups, num_kv_heads, head_dim, max_prefix_len).all : 0;
  return (size_t)(direct > laid_out ? direct : laid_out);
}

extern "C" int lsattn_shared_prefill(const lsattn_shared_prefill_args* a, void* stream) {
  if (!a || !a->q || !a->k || !a->v || !a->o || !a->m || !a->l || !a->req_to_tokens) return LSATTN_ERR_INVALID_ARG;
  if (a->rows < 0 || a->num_q_heads < 1 || a->num_kv_heads < 1 || a->num_slots < 1 || a->num_reqs < 0 || a->max_seq_len < 0 || a->num_groups < 0 ||
      a->max_prefix_len < 0 || a->max_group_rows < 0)
    return LSATTN_ERR_INVALID_ARG;
  if (a->num_groups && (!a->g_start_loc || !a->g_size || !a->g_req_idx || !a->g_prefix_len)) return LSATTN_ERR_INVALID_ARG;
  if (a->num_q_heads % a->num_kv_heads || (a->head_dim != 128 && a->head_dim != 64)) return LSATTN_ERR_UNSUPPORTED;
  if (a->dtype != LSATTN_F16 && a->dtype != LSATTN_BF16) return LSATTN_ERR_UNSUPPORTED;
  if (((a->k_stride_0 | a->k_stride_1 | a->v_stride_0 | a->v_stride_1 | a->q_stride_t | a->q_stride_h) % 8) || ((a->o_stride_t | a->o_stride_h) % 8) ||
      (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->o) & 15) || (((uintptr_t)a->m | (uintptr_t)a->l) & 3))
    return LSATTN_ERR_INVALID_ARG;
  auto slot_stride = [](int64_t elements) { return elements >= 0 && elements <= 0x3fffffff; };
  if (!slot_stride(a->k_stride_0) || !slot_stride(a->v_stride_0)) return LSATTN_ERR_INVALID_ARG;
  const int64_t group = a->num_q_heads / a->num_kv_heads;
  if (a->rows * group > 0x7fffff00 || a->num_q_heads > 65535 || a->max_seq_len > 0x7fff0000 || a->num_slots > 0x7fffffff || a->num_reqs > 0x7fffffff ||
      a->num_groups > 65535 || a->max_prefix_len > 0x7fff0000 || a->rows * a->num_q_heads > kMaxUnits)
    return LSATTN_ERR_INVALID_ARG;
  if (!(a->sm_scale > 0.f)) return LSATTN_ERR_INVALID_ARG;
  const int64_t most = most_of(a->max_prefix_len, a->max_seq_len);
  if (a->rows == 0 || a->num_groups == 0 || most == 0) return LSATTN_OK;
  // A workspace for more groups, which are not laid out, may be too small to lay out these: then they are taken as those would be.
  const PromptBytes pb = prompt_bytes(a->num_groups, a->num_kv_heads, a->head_dim, most);
  const bool lay_out = gathers(a->rows, a->num_groups, a->num_q_heads, a->num_kv_heads) && a->workspace_bytes >= (size_t)pb.all;
  const Plan pl = plan_of(a->rows, a->num_groups, a->num_q_heads, a->num_kv_heads, a->head_dim, most, 0, false);
  if (!a->workspace || (!lay_out && a->workspace_bytes < (size_t)pl.all())) return LSATTN_ERR_WORKSPACE;
  if ((uintptr_t)a->workspace & 15) return LSATTN_ERR_INVALID_ARG;
  SharedParams p = {};
  PoolParams& w = p.w;
  w.q = (const char*)a->q, w.k = (const char*)a->k, w.v = (const char*)a->v;
  w.k_s0 = a->k_stride_0 * 2, w.k_s1 = a->k_stride_1 * 2, w.v_s0 = a->v_stride_0 * 2, w.v_s1 = a->v_stride_1 * 2;
  w.table = a->req_to_tokens, w.max_seq_len = a->max_seq_len;
  w.num_reqs = (int32_t)a->num_reqs, w.num_slots = (int32_t)a->num_slots;
  w.hq = (int32_t)a->num_q_heads, w.hkv = (int32_t)a->num_kv_heads, w.group = (int32_t)group;
  w.scale_log2 = a->sm_scale * kLog2e;
  p.q_st = a->q_stride_t * 2, p.q_sh = a->q_stride_h * 2;
  p.g_start = a->g_start_loc, p.g_size = a->g_size, p.g_req = a->g_req_idx, p.g_prefix = a->g_prefix_len;
  p.groups = (int32_t)a->num_groups, p.rows = (int32_t)a->rows, p.most = (int32_t)most, p.near = is_near(w);
  p.by_hkv = fast_div((uint32_t)w.hkv), p.by_group = fast_div((uint32_t)group);
  hipStream_t st = (hipStream_t)stream;
  if (lay_out) {
    if (a->num_groups * most > 0x7fffff00) return LSATTN_ERR_INVALID_ARG;  // (rows of the gathered K/V)
    GatherParams g;
    char* at = (char*)a->workspace;
    g.k = at, g.v = at + pb.k, g.list = (int32_t*)(at + 2 * pb.k), g.vectors = (int32_t*)(at + 2 * pb.k + pb.list);
    g.most = (int32_t)most;
    const uint32_t head_chunks = (uint32_t)a->head_dim / 8;
    g.by_head_chunks = fast_div(head_chunks);
    LSATTN_LAUNCH_KERNEL(shared_prefix_list_kernel, dim3(p.groups), dim3(1024), 0, st, p, g);
    if (hipPeekAtLastError() != hipSuccess) return check_launch();
    const int64_t pieces = (most * 2 * w.hkv * head_chunks + 1023) / 1024, fill = 8 * kCUs / a->num_groups + 1;
    const dim3 grid((unsigned)(pieces < fill ? pieces : fill), (unsigned)a->num_groups);
    if (a->dtype == LSATTN_F16) LSATTN_LAUNCH_KERNEL((shared_prefix_gather_kernel<F16>), grid, dim3(256), 0, st, p, g, head_chunks);
    else LSATTN_LAUNCH_KERNEL((shared_prefix_gather_kernel<BF16>), grid, dim3(256), 0, st, p, g, head_chunks);
    if (hipPeekAtLastError() != hipSuccess) return check_launch();
    lsattn_prefill_args s = {};
    s.q = a->q, s.k = g.k, s.v = g.v;
    s.q_stride_t = a->q_stride_t, s.q_stride_h = a->q_stride_h;
    s.k_stride_t = s.v_stride_t = a->num_kv_heads * a->head_dim, s.k_stride_h = s.v_stride_h = a->head_dim;
    const int32_t* v = g.vectors;
    s.q_b_start_loc = v, s.q_b_seq_len = v + p.groups, s.q_first_token_global_idx = v + 2 * p.groups;
    s.kv_b_start_loc = v + 3 * p.groups, s.kv_b_seq_len = v + 4 * p.groups, s.kv_first_token_global_idx = v + 5 * p.groups;
    s.batch = p.groups, s.num_q_heads = w.hq, s.num_kv_heads = w.hkv, s.head_dim = (int32_t)a->head_dim, s.dtype = a->dtype, s.sp_peers = 1;
    const int64_t longest = a->max_group_rows < a->rows ? a->max_group_rows : a->rows;
    s.max_q_len = (int32_t)longest, s.sm_scale = a->sm_scale;
    s.o = a->o, s.o_stride_t = a->o_stride_t, s.o_stride_h = a->o_stride_h, s.o_dtype = a->dtype, s.v_is_f16 = a->dtype == LSATTN_BF16;
    s.m = a->m, s.l = a->l, s.ml_stride_t = a->ml_stride_t, s.ml_stride_h = a->ml_stride_h;
    s.total_q_rows = a->rows, s.total_kv_rows = a->num_groups * most, s.max_kv_len = (int32_t)most;
    return lsattn_prefill_step_merge(&s, stream);
  }
  if (pl.tiles * ((most + kKeys - 1) / kKeys) > kMaxUnits - kPrefixWorkgroups) return LSATTN_ERR_INVALID_ARG;  // (units are numbered with 31 bits)
  p.pre_o = (float*)a->workspace, p.pre_lse = p.pre_o + (pl.pre_floats / (a->head_dim + 1)) * a->head_dim;
  p.shares = (int32_t)pl.shares, p.parts = (int32_t)pl.parts, p.rounds = (int32_t)pl.rounds, p.ahead = pl.ahead, p.xcds_shift = (int32_t)pl.xcds_shift;
  p.by_pre_shares = fast_div((uint32_t)pl.shares), p.by_hq = fast_div((uint32_t)w.hq);
  p.plan = (int32_t*)(p.pre_o + pl.pre_floats), p.own_wgs = kPlanWorkgroups;
  FoldParams f;
  f.o = (char*)a->o, f.o_st = a->o_stride_t * 2, f.o_sh = a->o_stride_h * 2, f.m = a->m, f.l = a->l, f.ml_st = a->ml_stride_t, f.ml_sh = a->ml_stride_h;
  const unsigned fold_wgs = (unsigned)((a->rows * w.hq * (a->head_dim / 4) + 255) / 256);
  auto launch = [&](auto t, auto d) {
    constexpr int D = decltype(d)::value;
    LSATTN_LAUNCH_KERNEL((shared_prefix_kernel<decltype(t), D, false>), dim3((unsigned)(p.own_wgs + pl.shares * w.hkv)), dim3(256), 0, st, p);
    if (hipPeekAtLastError() != hipSuccess) return;
    LSATTN_LAUNCH_KERNEL((shared_prefix_fold_kernel<decltype(t), D>), dim3(fold_wgs), dim3(256), 0, st, p, f);
  };
  constexpr std::integral_constant<int, 128> d128{};
  constexpr std::integral_constant<int, 64> d64{};
  if (a->dtype == LSATTN_F16) a->head_dim == 128 ? launch(F16{}, d128) : launch(F16{}, d64);
  else a->head_dim == 128 ? launch(BF16{}, d128) : launch(BF16{}, d64);
  return check_launch();
}
