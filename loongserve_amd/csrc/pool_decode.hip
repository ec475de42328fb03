// Decode attention over the token-indexed pool with a sliding window and sinks, and over a pool held in 8 bits (gfx950, wave64).
//
// For request b with n tokens and query head h, over the positions j < n with j >= n - window or j < sinks (all, without a window):
//   s_j = scale * (q_h . k_j),   o = sum_j softmax(s)_j v_j,   LSE = log sum_j exp(s_j),
// where an e4m3 pool holds k_j and v_j as q * 2^e with one e per token and head.  n_vis visible tokens are numbered 0 .. n_vis - 1, sinks first, and the
// kernel walks those: a token outside the window costs nothing.
//
// What bounds it is HBM: (D + 1) bytes per K and V row of a head in 8 bits, 2 D in 16, against 2 D multiply-adds per query head
// for each.  Hence a row is read once for up to eight query heads of its KV head, and the vector work beside the matrix pipe is
// kept below what the memory leaves time for:
//   * a wave takes blocks of 32 tokens of one KV head.  Every load instruction takes whole rows (a row in two instructions of half a row each reads
//     a sixth slower): lane (g, c) = (lane / 16, lane % 16) has elements [c * D / 16, + D / 16) of V rows 4g .. 4g + 3 and 16 + 4g .. 16 + 4g + 3;
//     K rows are turned round in the wave's own LDS, from pieces of 16 bytes to the operands of the products;
//   * scores transposed, S^T = K Q^T with 16x16x32 MFMAs: the order of the head's elements along the contraction is whatever
//     the loads give, the query is read in the same one.  Column c of the product is query head c % 8, so the lane holds the
//     scores of eight tokens, 4g + r and 16 + 4g + r, of one head: the tokens whose V rows it has;
//   * O^T += V^T P^T with the V rows turned by byte permutes in registers: P^T goes into the product from the lane that
//     computed it, and every accumulator of a lane belongs to the head whose maximum and sum it keeps;
//   * P keeps more than 16 bits although the operands have 16: columns c and c + 8 of the product carry two parts of the same
//     head's P, high and low, and a second product a third part where the type is bfloat16 (8 bits each).  The parts are
//     added once, at the end;
//   * the scale of a token's V row goes into its weight: 2^(s + e) multiplies the e4m3 values as they are, and the reference that the weights are
//     taken relative to follows the maximum of s + e, so that they fit fp16 whatever the scales are.  The sum takes 2^s, relative to a reference that
//     follows the maximum of s: drawn from the weights instead it would lose a token whose s + e lies far below the largest (a V row of zeros beside one
//     of 2^61).  Both references are whole numbers, so 2^(their difference) is exact;
//   * the references are raised only when a score exceeds the maximum they were set by (by 8 log2 units, the sum's by 80): the accumulators
//     are seldom rescaled, and no exchange between lanes stands in the common path.
// Short contexts and windows: the waves of one workgroup share a (request, KV head) and meet in LDS (one launch).  Otherwise the blocks of
// all requests are dealt to the waves in equal shares, whatever the requests' lengths are (the host does not know them);
// a wave leaves one partial per request it touches, and a second launch merges them.
// Measured (32 / 8 heads of 128): 64 requests of 4096 .. 32768 tokens in 8 bits 408 us (5.9 TB/s), 96 behind a window of 16-bit rows 231 (6.2 TB/s); one request of 2047
// tokens 10.7, of 131072 55.
#include "common.hip.h"

namespace lsattn {
namespace {

struct E4M3 {};  // element tag of the pool

constexpr int kBlock = 32;       // tokens per step of a wave
// LDS of a wave: the byte offsets of a block's K rows and of its V rows, the factors of its scores, the exponents of its V rows
constexpr int kVOff = 256, kKScale = 512, kVExp = 640, kKRows = 768;  // (and the K rows of a block)
template <typename KV, int D> constexpr int kWaveLds = kKRows + kBlock * D * (__is_same(KV, E4M3) ? 1 : 2);
constexpr int kHeads = 8;        // query heads per task
constexpr int64_t kCUs = 256;
// The reference m of a head's weights is set to the maximum so far less kHead, and raised when a score exceeds it by kLag: weights
// of up to 2^15 (fp16 ends at 2^16), the largest 2^7 or more, so that the second part of a small fp16 weight does not run out of exponent.
constexpr float kHead = 7.f, kLag = 15.f;
// 8 bits: both references start here (finite, so that the scores of a block whose positions do not exist, -inf, leave them alone), and the sum's is raised where
// eight of its terms come to this (2^80 times 2^31 tokens stays a float, and so does what lies 2^-40 below the largest).
constexpr float kStart = -0x1p100f, kSumLimit = 0x1p80f;

struct PoolParams {
  const char* q;
  const char* k;
  const char* v;
  int64_t k_s0, k_s1, v_s0, v_s1;  // bytes
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t ks_s0, ks_s1, vs_s0, vs_s1;
  const int32_t* table;
  const int32_t* b_req;
  const int32_t* b_len;
  int64_t max_seq_len;
  int32_t batch, num_reqs, num_slots, hq, hkv, group, sub_groups, tasks;
  int32_t window, sinks;  // window 0: none
  float scale_log2;
  char* o;
  int32_t o_dtype;
  float* lse;
  float* part_o;    // [shares + batch, hq, D]
  float* part_lse;  // [shares + batch, hq]
  int32_t shares, min_units;
  FastDiv by_tasks, by_sub, by_shares;
};

__device__ __forceinline__ float xor16(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));
}
__device__ __forceinline__ float xor32(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, xor16(v));
  return fmaxf(v, xor32(v));
}
// (one instruction: from fmaxf the compiler makes three, which quiet signalling NaNs first)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float col_sum(float v) {
  v += xor16(v);
  return v + xor32(v);
}

template <typename T> __device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c);
template <> __device__ __forceinline__ f32x4 mfma<F16>(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma<BF16>(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two of the four e4m3 values of a word as 16-bit floats (exact)
template <typename T, bool HI> __device__ __forceinline__ uint32_t widen(uint32_t w);
template <> __device__ __forceinline__ uint32_t widen<F16, false>(uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)); }
template <> __device__ __forceinline__ uint32_t widen<F16, true>(uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)); }
template <> __device__ __forceinline__ uint32_t widen<BF16, false>(uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)); }
template <> __device__ __forceinline__ uint32_t widen<BF16, true>(uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)); }

// 2^e of an exponent byte (0, which no row written here has, is 2^-127)
__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte ? byte << 23 : 0x400000u); }

// The parts of eight P values: `hi` lanes give the first, the others the second (fp16: 2^-22 of the value is left out at most).  bfloat16, 8 bits a
// part: a third comes from the hi lanes in a product of its own, zero from the others; parts are cut off, not rounded, which leaves out 2^-23.
template <typename T> struct Parts;
template <> struct Parts<F16> {
  static constexpr int N = 1;
  static __device__ __forceinline__ void of(const float (&x)[8], bool hi, u32x4 (&out)[2]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t first = pack2<F16>(x[2 * e], x[2 * e + 1]);
      float a, b;  // x less its first part
      asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(a) : "v"(first), "v"(x[2 * e]));
      asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(first), "v"(x[2 * e + 1]));
      const uint32_t second = pack2<F16>(a, b);
      out[0][e] = hi ? first : second;
    }
  }
};
template <> struct Parts<BF16> {
  static constexpr int N = 2;
  static __device__ __forceinline__ float cut(float v) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t upper(float lo, float hi) { return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u); }
  static __device__ __forceinline__ void of(const float (&x)[8], bool hi, u32x4 (&out)[2]) {
    const uint32_t mine = hi ? 0xffffffffu : 0u;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float rest[2], third[2], first[2];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        rest[k] = x[2 * e + k] - cut(x[2 * e + k]);
        third[k] = rest[k] - cut(rest[k]);
        first[k] = hi ? x[2 * e + k] : rest[k];
      }
      out[0][e] = upper(first[0], first[1]);
      out[1][e] = upper(third[0], third[1]) & mine;
    }
  }
};

template <typename KV> struct PvOf { typedef KV type; };
template <> struct PvOf<E4M3> { typedef F16 type; };

// visible tokens of a request
__device__ __forceinline__ int visible(const PoolParams& p, int b, int& len, int& req) {
  len = p.b_len[b];
  req = p.b_req[b];
  if (len > p.max_seq_len) len = (int)p.max_seq_len;
  if (len < 0 || req < 0 || req >= p.num_reqs) len = 0;
  if (!p.window) return len;
  const int64_t most = (int64_t)p.window + p.sinks;
  return len < most ? len : (int)most;
}

// One wave's walk over blocks of visible tokens of one (request, KV head, up to eight query heads).
template <typename QT, typename KV, int D> struct Walk {
  typedef typename PvOf<KV>::type PV;
  static constexpr bool k8 = __is_same(KV, E4M3);
  static constexpr int KS = D / 32;               // contraction steps of Q K^T
  static constexpr int EV = D / 16;               // elements of a V row per lane
  static constexpr int CPR = k8 ? D / 16 : D / 8; // 16-byte pieces of a K row
  static constexpr int RPI = 64 / CPR;            // K rows per load instruction
  static constexpr int KI = kBlock / RPI;         // and instructions for a block
  static constexpr int VW = k8 ? EV / 4 : EV / 2; // words of a V row per lane
  static constexpr int ES = k8 ? 1 : 2;           // bytes per element

  const PoolParams& p;
  const int lane, g, c;
  char* const lds;
  u32x4 qf[KS];
  f32x4 acc[EV];  // acc[j][r] = O[head][EV * (4g + r) + j], of the parts of P in this lane's column
  float m, l;     // log2-domain maximum of the head; the lane's share of the sum
  float ml;       // (8 bits) what the sum is relative to

  __device__ __forceinline__ Walk(const PoolParams& p_, char* lds_wave)
      : p(p_), lane(threadIdx.x & 63), g(lane >> 4), c(lane & 15), lds(lds_wave) {}

  const char *kb, *vb;
  const uint8_t* sb;  // the lane's column of scales: K for lanes 0 .. 31, V for the others
  uint32_t s_s0, row_s0;  // and the bytes from one slot to the next there, and in the rows
  const int32_t* row;
  int sinks, skip, limit;

  // a task = one KV head and up to eight query heads of its group
  __device__ __forceinline__ void start(int b, int req, int task, int len, int n_vis) {
    const int kvh = (int)div_by((uint32_t)task, p.by_sub), sg = task - kvh * p.sub_groups;
    const int h0 = kvh * p.group + sg * kHeads;
    const int nh = p.group - sg * kHeads < kHeads ? p.group - sg * kHeads : kHeads;
    const int h = (c & 7) < nh ? (c & 7) : nh - 1;
    const char* q = p.q + ((int64_t)b * p.hq + h0 + h) * D * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      // (the order of the K loads below)
      const int d = k8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g;
      qf[ks] = *(const u32x4*)(q + d * 2);
    }
    kb = p.k + kvh * p.k_s1 + 16 * (lane & (CPR - 1));
    vb = p.v + kvh * p.v_s1 + c * EV * ES;
    if (k8) {
      sb = lane < 32 ? p.ks + kvh * p.ks_s1 : p.vs + kvh * p.vs_s1;
      s_s0 = (uint32_t)(lane < 32 ? p.ks_s0 : p.vs_s0);
    }
    row_s0 = (uint32_t)(lane < 32 ? p.k_s0 : p.v_s0);
    row = p.table + (int64_t)req * p.max_seq_len;
    sinks = p.window ? p.sinks : 0;
    skip = len - n_vis;
    m = k8 ? kStart : -INFINITY, ml = kStart, l = 0.f;
#pragma unroll
    for (int j = 0; j < EV; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // the slot of token `at` + lane % 32 (positions past the end repeat the last one)
  __device__ __forceinline__ int load_slot(int at) const {
    int i = at + (lane & 31);
    i = i < limit ? i : limit - 1;
    return row[i < sinks ? i : i + skip];
  }

  struct Rows {  // a block's K and V in flight
    u32x4 k[KI];
    uint32_t v[8][VW];
    uint32_t scale_byte;
    uint32_t there;  // bit i: token i of the block exists
  };

  // the rows of the block at `at`, whose slots the lanes have in `slot`; `next`: where the block after it starts, whose slots are asked for in front
  __device__ __forceinline__ void load_rows(Rows& r, int at, int& slot_of, int next) {
    int slot = slot_of;
    slot_of = load_slot(next);
    const bool ok = at + (lane & 31) < limit && (uint32_t)slot < (uint32_t)p.num_slots;
    r.there = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
    slot = ok ? slot : 0;
    if (k8) r.scale_byte = sb[(uint64_t)(uint32_t)slot * s_s0];
    *(uint64_t*)(lds + lane * 8) = (uint64_t)(uint32_t)slot * row_s0;
    __builtin_amdgcn_wave_barrier();
    uint64_t koff[KI], voff[8];
#pragma unroll
    for (int i = 0; i < KI; i++) koff[i] = *(const uint64_t*)(lds + (RPI * i + lane / CPR) * 8);
#pragma unroll
    for (int i = 0; i < 4; i++) *(u32x4*)(voff + 2 * i) = *(const u32x4*)(lds + kVOff + (i >> 1) * 128 + 32 * g + (i & 1) * 16);
    __builtin_amdgcn_wave_barrier();
    // Rows are read once and loaded so (nontemporal): on a pool that no cache holds yet a fifth to a quarter faster in 16 bits (64 requests behind a window of 4096,
    // 1.1 GB: 185 us, 235 without), 6 - 30 % in 8.  (the empty statements keep each 64-bit address next to its load instead of ten of them live at once)
#pragma unroll
    for (int i = 0; i < KI; i++) {
      asm volatile("" : "+v"(koff[i]));
      r.k[i] = __builtin_nontemporal_load((const u32x4*)(kb + koff[i]));
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      asm volatile("" : "+v"(voff[i]));
      const char* at_v = vb + voff[i];
      if constexpr (VW == 1) r.v[i][0] = __builtin_nontemporal_load((const uint32_t*)at_v);
      else if constexpr (VW == 2) *(u32x2*)r.v[i] = __builtin_nontemporal_load((const u32x2*)at_v);
      else *(u32x4*)r.v[i] = __builtin_nontemporal_load((const u32x4*)at_v);
    }
  }

  __device__ __forceinline__ void compute(Rows& rows) {
    // the K rows through LDS: pieces XORed with the row, so that neither side meets in the banks
    char* const k_lds = lds + kKRows;
#pragma unroll
    for (int i = 0; i < KI; i++) {
      const int row = RPI * i + lane / CPR;
      *(u32x4*)(k_lds + row * (CPR * 16) + (((lane & (CPR - 1)) ^ (row & (CPR - 1))) << 4)) = rows.k[i];
    }
    __builtin_amdgcn_wave_barrier();
    // scores of the lane's head with tokens 4g + r (s[0]) and 16 + 4g + r (s[1])
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    constexpr int PIECES = CPR / 4;  // pieces of a row per lane, the contraction's 16 (8 bits) or 8 elements each
#pragma unroll
    for (int w = 0; w < PIECES; w++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const u32x4 k = *(const u32x4*)(k_lds + (16 * t + c) * (CPR * 16) + (((4 * w + g) ^ (c & (CPR - 1))) << 4));
        if constexpr (k8) {
#pragma unroll
          for (int n = 0; n < 2; n++) {
            const u32x4 a = u32x4{widen<QT, false>(k[2 * n]), widen<QT, true>(k[2 * n]), widen<QT, false>(k[2 * n + 1]), widen<QT, true>(k[2 * n + 1])};
            s[t] = mfma<QT>(a, qf[2 * w + n], s[t]);
          }
        } else {
          s[t] = mfma<QT>(k, qf[w], s[t]);
        }
        if (t) __builtin_amdgcn_sched_barrier(0);
      }
    __builtin_amdgcn_wave_barrier();
    float x[8];  // the score in log2 units
    f32x4 ve[2];  // (8 bits) the exponent of the token's V row
    if constexpr (k8) {
      // (a position that does not exist has the exponent 0: what lies in the slot that was read in its place may be any byte)
      const uint32_t byte = (rows.there >> (lane & 31)) & 1u ? rows.scale_byte : 127u;
      *(float*)(lds + kKScale + lane * 4) = lane < 32 ? scale_of(byte) * p.scale_log2 : (float)((int)byte - 127);
      __builtin_amdgcn_wave_barrier();
      f32x4 kf[2];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        kf[t] = *(const f32x4*)(lds + kKScale + 64 * t + 16 * g);
        ve[t] = *(const f32x4*)(lds + kVExp + 64 * t + 16 * g);
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = s[e / 4][e % 4] * kf[e / 4][e % 4];
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = s[e / 4][e % 4] * p.scale_log2;
    }
    if (rows.there != 0xffffffffu) {  // (the same for every lane)
      const uint32_t mine = ((rows.there >> (4 * g)) & 15u) | ((rows.there >> (12 + 4 * g)) & 0xf0u);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool ok = (mine >> e) & 1u;
        x[e] = ok ? x[e] : -INFINITY;
#pragma unroll
        for (int w = 0; w < VW; w++) rows.v[e][w] = ok ? rows.v[e][w] : 0u;  // (what lies there may be infinite or NaN)
      }
    }
    auto largest = [](const float (&v)[8]) __attribute__((always_inline)) { return max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), fmaxf(v[6], v[7])); };
    if constexpr (k8) {
      // the arguments of the weights, s + e - m (e - m is exact, and so they are rounded where they are small), and the sum's terms, 2^(s - ml)
      float y[8], part;
      auto relative = [&]() __attribute__((always_inline)) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = x[e] + (ve[e / 4][e % 4] - m), w[e] = __builtin_amdgcn_exp2f(x[e] - ml);
        part = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      };
      relative();
      if (__builtin_amdgcn_ballot_w64(largest(y) > kLag || !(part < kSumLimit)) != 0) {
        float with_e[8];
#pragma unroll
        for (int e = 0; e < 8; e++) with_e[e] = x[e] + ve[e / 4][e % 4];
        const float m_new = fmaxf(m, floorf(col_max(largest(with_e))) - kHead), ml_new = fmaxf(ml, floorf(col_max(largest(x))));
        const float alpha = __builtin_amdgcn_exp2f(m - m_new);
        l *= __builtin_amdgcn_exp2f(ml - ml_new);
#pragma unroll
        for (int j = 0; j < EV; j++) acc[j] *= alpha;
        m = m_new, ml = ml_new;
        relative();
      }
      l += part;
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = __builtin_amdgcn_exp2f(y[e]);
    } else {
      const float mx = largest(x);
      if (__builtin_amdgcn_ballot_w64(mx > m + kLag) != 0) {
        const float m_new = fmaxf(m, col_max(mx) - kHead);
        const float alpha = exp2_diff(m, m_new);
        l *= alpha;
#pragma unroll
        for (int j = 0; j < EV; j++) acc[j] *= alpha;
        m = m_new;
      }
      const float m_safe = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = __builtin_amdgcn_exp2f(x[e] - m_safe);
      l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    }
    u32x4 pk[2];
    Parts<PV>::of(x, c < 8, pk);
    __builtin_amdgcn_sched_barrier(0);
    // V^T operands: element j of the eight tokens
#pragma unroll
    for (int w = 0; w < VW; w++) {
      if constexpr (k8) {
        u32x4 va[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const uint32_t lo = __builtin_amdgcn_perm(rows.v[2 * t + 1][w], rows.v[2 * t][w], 0x05010400u);
          const uint32_t hi = __builtin_amdgcn_perm(rows.v[2 * t + 1][w], rows.v[2 * t][w], 0x07030602u);
          va[0][t] = widen<PV, false>(lo);
          va[1][t] = widen<PV, true>(lo);
          va[2][t] = widen<PV, false>(hi);
          va[3][t] = widen<PV, true>(hi);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int n = 0; n < Parts<PV>::N; n++) acc[4 * w + j] = mfma<PV>(va[j], pk[n], acc[4 * w + j]);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        u32x4 va[2];
#pragma unroll
        for (int t = 0; t < 4; t++) {
          va[0][t] = __builtin_amdgcn_perm(rows.v[2 * t + 1][w], rows.v[2 * t][w], 0x05040100u);
          va[1][t] = __builtin_amdgcn_perm(rows.v[2 * t + 1][w], rows.v[2 * t][w], 0x07060302u);
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int n = 0; n < Parts<PV>::N; n++) acc[2 * w + j] = mfma<PV>(va[j], pk[n], acc[2 * w + j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // Visible tokens [from, to) in steps of `step` blocks; the first block exists.  The next block's rows are in flight while one is worked on (a lone
  // wave otherwise spends 2 us on a block, nearly all of it waiting), and the slots of the one after it.
  __device__ __forceinline__ void run(int from, int to, int step) {
    limit = to;
    step *= kBlock;
    Rows a, b;
    int slot = load_slot(from);
    load_rows(a, from, slot, from + step);
    // (loads without a condition around them: behind one the compiler would wait for all of them.  Past the end they repeat the last rows)
    for (int at = from; at < to; at += 2 * step) {
      load_rows(b, at + step, slot, at + 2 * step);
      __builtin_amdgcn_sched_barrier(0);
      compute(a);
      load_rows(a, at + 2 * step, slot, at + 3 * step);
      __builtin_amdgcn_sched_barrier(0);
      if (at + step < to) compute(b);
    }
  }

  // the parts of P together, and the sum over the head's lanes.  8 bits: O as the mean, m the log-sum-exp, a sum of 1 (0: nothing seen)
  __device__ __forceinline__ void join() {
#pragma unroll
    for (int j = 0; j < EV; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) acc[j][r] += dpp_mov<0x128>(acc[j][r]);  // row_ror:8
    l = col_sum(l);
    if constexpr (k8) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int up = l > 0.f ? (int)(m - ml) : 0;  // (whole numbers; the difference of the two may pass what a float's exponent takes)
#pragma unroll
      for (int j = 0; j < EV; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) acc[j][r] = __builtin_amdgcn_ldexpf(acc[j][r] * inv, up);
      m = l > 0.f ? ml + __builtin_amdgcn_logf(l) : -INFINITY;
      l = l > 0.f ? 1.f : l;
    }
  }
};

__device__ __forceinline__ void store_elem4(char* o, int dtype, int64_t at, const f32x4& v) {
  if (dtype == LSATTN_F32) *(f32x4*)((float*)o + at) = v;
  else if (dtype == LSATTN_F16) *(u32x2*)((uint16_t*)o + at) = u32x2{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3])};
  else *(u32x2*)((uint16_t*)o + at) = u32x2{pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3])};
}
__device__ __forceinline__ float ln_of(float m, float l) { return l > 0.f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : (l == l ? -INFINITY : l); }

// One workgroup per (task, request): its NW waves take every NW-th block and meet in LDS.  Four of them, so that two or three workgroups fill a CU (8 bits, 256
// requests of 512 tokens, 277 MB: 73 us, 86 with eight waves; a lone request of 512 as well, 8.4 and 9.9).
template <typename QT, typename KV, int D, int NW>
__global__ __launch_bounds__(NW * 64, (D == 128 && !__is_same(KV, E4M3) ? 2 : 3)) void pool_decode_direct_kernel(PoolParams p) {
  constexpr int ROW = D + 4;  // floats per head in LDS: O, maximum, sum (and a bank's shift)
  __shared__ __attribute__((aligned(16))) char lds[NW * (kHeads * ROW * 4 > kWaveLds<KV, D> ? kHeads * ROW * 4 : kWaveLds<KV, D>)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int task = blockIdx.x, b = blockIdx.y;
  const int kvh = (int)div_by((uint32_t)task, p.by_sub), sg = task - kvh * p.sub_groups;
  const int h0 = kvh * p.group + sg * kHeads;
  const int nh = p.group - sg * kHeads < kHeads ? p.group - sg * kHeads : kHeads;
  int len, req;
  const int n_vis = visible(p, b, len, req);
  Walk<QT, KV, D> w(p, lds + wave * kWaveLds<KV, D>);
  if (wave * kBlock < n_vis) {
    w.start(b, req, task, len, n_vis);
    w.run(wave * kBlock, n_vis, NW);
    w.join();
  } else {
    w.m = -INFINITY, w.l = 0.f;
  }
  __syncthreads();  // (the waves' slots and scales lie where the results go)
  float* const res = (float*)lds;
  if (w.c < nh) {
    float* mine = res + (wave * kHeads + w.c) * ROW;
    if (wave * kBlock < n_vis) {
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int j = 0; j < D / 16; j += 4)
          *(f32x4*)(mine + (D / 16) * (4 * w.g + r) + j) = f32x4{w.acc[j][r], w.acc[j + 1][r], w.acc[j + 2][r], w.acc[j + 3][r]};
    }
    if (w.g == 0) mine[D] = w.m, mine[D + 1] = w.l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * (D / 4); i += NW * 64) {
    const int h = i / (D / 4), d = (i & (D / 4 - 1)) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < NW; v++) M = fmaxf(M, res[(v * kHeads + h) * ROW + D]);
    float L = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; v++) {
      const float* r = res + (v * kHeads + h) * ROW;
      if (v * kBlock < n_vis) {
        const float f = exp2_diff(r[D], M);
        L += r[D + 1] * f;
        sum += *(const f32x4*)(r + d) * f;
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int64_t at = (int64_t)b * p.hq + h0 + h;
    store_elem4(p.o, p.o_dtype, at * D + d, sum * inv);
    if (d == 0) p.lse[at] = ln_of(M, L);
  }
}

// How the blocks of all requests are dealt: numbered request by request, per_share to a share.  Every wave counts them by itself, 64 requests at a
// time, of which a lane has one each; up to 64 requests are one look at their lengths.
struct Requests {
  int first_request, len, req, n_vis, units, up_to;  // up_to: units of the 64 up to the lane's request
  __device__ __forceinline__ void look(const PoolParams& p, int b0) {
    const int lane = threadIdx.x & 63;
    first_request = b0;
    n_vis = 0;
    if (b0 + lane < p.batch) n_vis = visible(p, b0 + lane, len, req);
    units = (n_vis + kBlock - 1) / kBlock;
    up_to = units;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int below = __shfl_up(up_to, d, 64);
      if (lane >= d) up_to += below;
    }
  }
  __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(up_to, 63); }
};
__device__ __forceinline__ int per_share_of(const PoolParams& p, int total) {
  const int per = (int)div_by((uint32_t)(total + p.shares - 1), p.by_shares);
  return per < p.min_units ? p.min_units : per;
}

// Four waves per workgroup, each with a share of its own of one task; the tasks of a share are neighbours, on one XCD.
template <typename QT, typename KV, int D>
__global__ __launch_bounds__(256, 2) void pool_decode_shares_kernel(PoolParams p) {
  __shared__ __attribute__((aligned(16))) char lds[4 * kWaveLds<KV, D>];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (ids go to the XCDs round-robin; gridDim.x is a multiple of 8)
  const uint32_t id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const uint32_t unit = id * 4 + wave;
  const int share = (int)div_by(unit, p.by_tasks), task = (int)(unit - (uint32_t)share * p.tasks);
  if (share >= p.shares) return;
  Requests rs;
  rs.look(p, 0);
  int total = rs.all();
  if (p.batch > 64) {
    for (int b0 = 64; b0 < p.batch; b0 += 64) rs.look(p, b0), total += rs.all();
    rs.look(p, 0);
  }
  const int per_share = per_share_of(p, total);
  int at = share * per_share;  // (up to shares - 1 more than there are units)
  const int end = total - at < per_share ? total : at + per_share;
  if (at >= end) return;
  // the request of the share's first unit (at < total: found before the batch ends)
  int first = 0;
  while (at >= first + rs.all()) {
    first += rs.all();
    rs.look(p, rs.first_request + 64);
  }
  int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(first + rs.up_to > at));
  first += __builtin_amdgcn_readlane(rs.up_to, l) - __builtin_amdgcn_readlane(rs.units, l);
  Walk<QT, KV, D> w(p, lds + wave * kWaveLds<KV, D>);
  const int kvh = (int)div_by((uint32_t)task, p.by_sub), sg = task - kvh * p.sub_groups;
  const int h0 = kvh * p.group + sg * kHeads;
  const int nh = p.group - sg * kHeads < kHeads ? p.group - sg * kHeads : kHeads;
  for (;;) {
    const int b = rs.first_request + l, units = __builtin_amdgcn_readlane(rs.units, l), n_vis = __builtin_amdgcn_readlane(rs.n_vis, l);
    const int to = end - first < units ? end : first + units;
    if (to > at) {
      w.start(b, __builtin_amdgcn_readlane(rs.req, l), task, __builtin_amdgcn_readlane(rs.len, l), n_vis);
      const int last = (to - first) * kBlock;
      w.run((at - first) * kBlock, last < n_vis ? last : n_vis, 1);
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
    if (++l == 64) rs.look(p, rs.first_request + 64), l = 0;
  }
}

// o = sum of a request's partials by their log-sum-exps: first the weights of all of them, by all threads, into LDS, then the rows, whose loads wait for nothing.
// W lanes read W * 4 elements of a row, the rows are dealt to the rest of the workgroup; D / 4 / W workgroups share a head (few requests: a lone workgroup draws 350
// rows in 9 us).
constexpr int kMaxShares = 4 * (int)kCUs;  // (kShareWaves)
template <int D, int W>
__global__ __launch_bounds__(256) void pool_decode_merge_kernel(PoolParams p) {
  constexpr int SL = 256 / W;
  __shared__ __attribute__((aligned(16))) float acc[SL][W * 4];
  __shared__ float weight[kMaxShares], part[8];
  const int h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Requests rs;
  int total = 0, first = 0, units = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    rs.look(p, b0);
    if (b >= b0 && b < b0 + 64) {
      units = __builtin_amdgcn_readlane(rs.units, b - b0);
      first = total + __builtin_amdgcn_readlane(rs.up_to, b - b0) - units;
    }
    total += rs.all();
  }
  const uint32_t per_share = (uint32_t)per_share_of(p, total);
  const int s0 = (int)((uint32_t)first / per_share), n = units ? (int)((uint32_t)(first + units - 1) / per_share) - s0 + 1 : 0;
  const float* lse = p.part_lse + ((int64_t)(s0 + b) * p.hq + h);
  float M = -INFINITY;
  for (int i = threadIdx.x; i < n; i += 256) {
    const float x = lse[(int64_t)i * p.hq];
    weight[i] = x;
    M = fmaxf(M, x);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
  if (lane == 0) part[wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  float L = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) {
    const float w = exp2_diff(weight[i], M);  // (NaN stays NaN)
    weight[i] = w;
    L += w;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) L += __shfl_xor(L, d, 64);
  if (lane == 0) part[4 + wave] = L;
  __syncthreads();
  L = (part[4] + part[5]) + (part[6] + part[7]);
  const int slice = threadIdx.x / W, d = (threadIdx.x & (W - 1)) * 4, d0 = (int)blockIdx.z * W * 4;
  const float* row = p.part_o + ((int64_t)(s0 + b) * p.hq + h) * D + d0 + d;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = slice; i < n; i += SL) {
    const f32x4 v = *(const f32x4*)(row + (int64_t)i * p.hq * D);
    sum += v * weight[i];  // (every row is finite unless the result is not)
  }
  *(f32x4*)&acc[slice][d] = sum;
  __syncthreads();
  if (slice) return;
#pragma unroll 8
  for (int i = 1; i < SL; i++) sum += *(const f32x4*)&acc[i][d];
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t at = (int64_t)b * p.hq + h;
  store_elem4(p.o, p.o_dtype, at * D + d0 + d, sum * inv);
  if (d0 + d == 0) p.lse[at] = ln_of(M, L);
}

constexpr int kDirectWaves = 4;
// A workgroup takes a whole (request, KV head) where the longest request's visible tokens are few for the workgroups there are.  Microseconds on a cold pool, a workgroup | shares,
// heads of 128, 8 bits (16 bits):
//   32/8: 1 request of 512 tokens 9.2 | 11.5 (11.0 | 13.1), 768 11.5 | 11.7 (13.6 | 13.1), 1024 13.8 | 11.9 (16.8 | 13.2); 16 of 768 13.4 | 15.5 (17.4 | 19.3), 1024 16.8 | 16.4 (21.4 | 21.2),
//   2048 30.3 | 23.5 (36.9 | 31.3); 32 of 512 13.6 | 18.4 (16.5 | 21.8), 1024 20.8 | 23.4 (27.5 | 32.4), 2048 36.3 | 36.4 (49.8 | 53.4); 64 of 2048 66.4 | 62.6 (94.4 | 96.8); 256 of 512
//   75.4 | 91.6 (105.7 | 124.1), 2048 259 | 244 (371 | 377)
//   8/1: 16 of 1024 13.7 | 13.4 (15.1 | 14.1); 256 of 1024 20.1 | 31.9 (29.0 | 41.9), 2048 34.2 | 46.2 (52.2 | 64.9)
//   32/32: 1 of 768 13.3 | 13.6 (14.2 | 13.5), 1024 15.5 | 13.9 (17.5 | 14.2); 32 of 1024 66.7 | 61.8 (92.1 | 93.5), 2048 127 | 113 (179 | 175); 64/4: 32 of 1024 19.3 | 23.8 (28.9 | 29.9),
//   2048 32.7 | 33.0 (52.2 | 46.1)
// Length and workgroups alone do not tell all of it: in 8 bits this rule takes the slower form for 2048 tokens of 64 and more requests (6 %) and of
// 32 with 32/32 heads (12 %; 1024 tokens 8 %), in 16 bits for 32 of 2048 with 64/4 (13 %).
// Waves that a launch of shares deals to: one per SIMD.  More leave shorter shares, whose starts and partials cost more than the loads in flight bring (microseconds, cold;
// 4 | 8 of a CU's waves): 8 bits 1 request of 32768 24.0 | 25.3, 32 of 8192 112 | 115, 64 of 4096 .. 32768 465 | 465, 32 of 8192 64-wide 86 | 94; 16 bits 8 behind
// 8192 52.4 | 55.2, 128 681 | 688.  Numbers that leave the SIMDs of a CU with unequal counts lose a fifth: 3 134, 5 154, 6 139 for the 32 when 4 took 116.
constexpr int64_t kShareWaves = 4 * kCUs;
constexpr int64_t kMinUnits = 2;

int64_t most_visible(int64_t max_len, int64_t window, int64_t sinks) { return window > 0 && window < max_len && sinks < max_len - window ? window + sinks : max_len; }
int64_t tasks_of(int64_t hq, int64_t hkv) { return hkv * ((hq / hkv + kHeads - 1) / kHeads); }
bool is_direct(int64_t batch, int64_t tasks, int64_t most) {
  const int64_t wgs = batch * tasks;
  return most <= (wgs >= kCUs ? 2048 : wgs >= kCUs / 4 ? 1024 : 768);
}
// shares of a launch that is not direct
int64_t shares_of(int64_t batch, int64_t tasks, int64_t most) {
  const int64_t units = batch * ((most + kBlock - 1) / kBlock);
  const int64_t by_waves = kShareWaves / tasks, by_units = (units + kMinUnits - 1) / kMinUnits;
  const int64_t n = by_waves < by_units ? by_waves : by_units;
  return n < 1 ? 1 : n;
}

template <typename QT, typename KV, int D> void launch(const PoolParams& p, bool direct, hipStream_t st) {
  if (direct) {
    LSATTN_LAUNCH_KERNEL((pool_decode_direct_kernel<QT, KV, D, kDirectWaves>), dim3(p.tasks, p.batch), dim3(kDirectWaves * 64), 0, st, p);
    return;
  }
  const int64_t wgs = ((int64_t)p.shares * p.tasks + 3) / 4;
  LSATTN_LAUNCH_KERNEL((pool_decode_shares_kernel<QT, KV, D>), dim3((unsigned)((wgs + 7) / 8 * 8)), dim3(256), 0, st, p);
  if (hipPeekAtLastError() != hipSuccess) return;
  if ((int64_t)p.hq * p.batch <= kCUs / 2) LSATTN_LAUNCH_KERNEL((pool_decode_merge_kernel<D, 8>), dim3(p.hq, p.batch, D / 32), dim3(256), 0, st, p);
  else LSATTN_LAUNCH_KERNEL((pool_decode_merge_kernel<D, D / 4>), dim3(p.hq, p.batch), dim3(256), 0, st, p);
}
template <typename QT, typename KV> void launch_d(const PoolParams& p, int64_t d, bool direct, hipStream_t st) {
  if (d == 128) launch<QT, KV, 128>(p, direct, st);
  else launch<QT, KV, 64>(p, direct, st);
}

}  // namespace
}  // namespace lsattn

using namespace lsattn;

extern "C" size_t lsattn_pool_attention_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                                        int64_t max_len_in_batch, int64_t window, int64_t sinks) {
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0 || max_len_in_batch <= 0 || window < 0 || sinks < 0 ||
      batch > 65535 || num_q_heads > 65535 || max_len_in_batch > 0x7fffffff)  // (as the launch refuses)
    return 0;
  const int64_t tasks = tasks_of(num_q_heads, num_kv_heads), most = most_visible(max_len_in_batch, window, sinks);
  if (is_direct(batch, tasks, most)) return 0;
  return (size_t)((shares_of(batch, tasks, most) + batch) * num_q_heads * (head_dim + 1) * 4);
}

extern "C" int lsattn_pool_attention(const lsattn_pool_attention_args* a, void* stream) {
  if (!a || !a->q || !a->k || !a->v || !a->o || !a->lse || !a->req_to_tokens || !a->b_req_idx || !a->b_seqlen) return LSATTN_ERR_INVALID_ARG;
  if (a->batch < 0 || a->num_q_heads < 1 || a->num_kv_heads < 1 || a->num_slots < 1 || a->num_reqs < 0 || a->max_seq_len < 0 || a->max_len_in_batch < 0 ||
      a->window < 0 || a->sinks < 0)
    return LSATTN_ERR_INVALID_ARG;
  if (a->num_q_heads % a->num_kv_heads || (a->head_dim != 128 && a->head_dim != 64)) return LSATTN_ERR_UNSUPPORTED;
  if (a->o_dtype != LSATTN_F32 && a->o_dtype != LSATTN_F16 && a->o_dtype != LSATTN_BF16) return LSATTN_ERR_UNSUPPORTED;
  if ((a->dtype != LSATTN_F16 && a->dtype != LSATTN_BF16) || (a->kv_dtype != a->dtype && a->kv_dtype != LSATTN_E4M3)) return LSATTN_ERR_UNSUPPORTED;
  const bool k8 = a->kv_dtype == LSATTN_E4M3;
  const int64_t es = k8 ? 1 : 2;
  if ((a->k_stride_0 * es) % 16 || (a->k_stride_1 * es) % 16 || (a->v_stride_0 * es) % 16 || (a->v_stride_1 * es) % 16 ||
      (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->o) & 15))
    return LSATTN_ERR_INVALID_ARG;
  if (k8 && (!a->k_scales || !a->v_scales)) return LSATTN_ERR_INVALID_ARG;
  // (offsets are a slot times a stride of 32 bits)
  auto slot_stride = [](int64_t bytes) { return bytes >= 0 && bytes <= 0x7fffffff; };
  if (!slot_stride(a->k_stride_0 * es) || !slot_stride(a->v_stride_0 * es) || (k8 && (!slot_stride(a->ks_stride_0) || !slot_stride(a->vs_stride_0))))
    return LSATTN_ERR_INVALID_ARG;
  if (a->batch > 65535 || a->num_q_heads > 65535 || a->max_seq_len > 0x7fff0000 || a->num_slots > 0x7fffffff || a->num_reqs > 0x7fffffff ||
      a->max_len_in_batch > 0x7fffffff)
    return LSATTN_ERR_INVALID_ARG;
  if (!(a->sm_scale > 0.f)) return LSATTN_ERR_INVALID_ARG;
  if (a->batch == 0) return LSATTN_OK;
  PoolParams p;
  p.q = (const char*)a->q, p.k = (const char*)a->k, p.v = (const char*)a->v;
  p.k_s0 = a->k_stride_0 * es, p.k_s1 = a->k_stride_1 * es, p.v_s0 = a->v_stride_0 * es, p.v_s1 = a->v_stride_1 * es;
  p.ks = a->k_scales, p.vs = a->v_scales;
  p.ks_s0 = a->ks_stride_0, p.ks_s1 = a->ks_stride_1, p.vs_s0 = a->vs_stride_0, p.vs_s1 = a->vs_stride_1;
  p.table = a->req_to_tokens, p.b_req = a->b_req_idx, p.b_len = a->b_seqlen, p.max_seq_len = a->max_seq_len;
  p.batch = (int32_t)a->batch, p.num_reqs = (int32_t)a->num_reqs, p.num_slots = (int32_t)a->num_slots;
  p.hq = (int32_t)a->num_q_heads, p.hkv = (int32_t)a->num_kv_heads, p.group = p.hq / p.hkv;
  p.sub_groups = (p.group + kHeads - 1) / kHeads, p.tasks = p.hkv * p.sub_groups;
  // (a window that holds every position a table can have is none)
  p.window = a->window >= a->max_seq_len ? 0 : (int32_t)a->window;
  p.sinks = a->sinks > a->max_seq_len ? (int32_t)a->max_seq_len : (int32_t)a->sinks;
  p.scale_log2 = a->sm_scale * kLog2e;
  p.o = (char*)a->o, p.o_dtype = a->o_dtype, p.lse = a->lse;
  p.by_tasks = fast_div((uint32_t)p.tasks), p.by_sub = fast_div((uint32_t)p.sub_groups);
  const int64_t most = most_visible(a->max_len_in_batch, a->window, a->sinks);
  const bool direct = is_direct(p.batch, p.tasks, most);
  p.part_o = nullptr, p.part_lse = nullptr, p.shares = 1, p.by_shares = fast_div(1), p.min_units = (int32_t)kMinUnits;
  if (!direct) {
    const int64_t shares = shares_of(p.batch, p.tasks, most), rows = shares + p.batch;
    if (!a->workspace || a->workspace_bytes < (size_t)(rows * p.hq * (a->head_dim + 1) * 4)) return LSATTN_ERR_WORKSPACE;
    if ((uintptr_t)a->workspace & 15) return LSATTN_ERR_INVALID_ARG;
    p.shares = (int32_t)shares, p.by_shares = fast_div((uint32_t)shares);
    if (a->batch * ((a->max_seq_len + kBlock - 1) / kBlock) > kMaxUnits - kMaxShares) return LSATTN_ERR_INVALID_ARG;  // (blocks are numbered with 31 bits)
    p.part_o = (float*)a->workspace, p.part_lse = p.part_o + rows * p.hq * a->head_dim;
  }
  hipStream_t st = (hipStream_t)stream;
  if (k8) {
    if (a->dtype == LSATTN_F16) launch_d<F16, E4M3>(p, a->head_dim, direct, st);
    else launch_d<BF16, E4M3>(p, a->head_dim, direct, st);
  } else {
    if (a->dtype == LSATTN_F16) launch_d<F16, F16>(p, a->head_dim, direct, st);
    else launch_d<BF16, BF16>(p, a->head_dim, direct, st);
  }
  return check_launch();
}
