// A wave's walk over tokens of a KV pool, for decode attention (pool_decode.hip says what it computes and how): the types, the arguments of a
// launch and the walk itself, which the kernels over whole contexts and windows (pool_decode.hip) and those over the tokens behind a shared prefix
// (shared_prefix.hip) run.
#pragma once
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

}  // namespace
}  // namespace lsattn
