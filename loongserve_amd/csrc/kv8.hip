// The KV pool held in 8 bits: rows quantised as they are written, and read back as 16-bit K/V (gfx950).
//
// A (token, head) row of D elements is kept as D e4m3 values and one exponent e (a byte, e + 127): x stands as q * 2^e with
//   e = the least integer with max |x| <= 448 * 2^e (448: the largest e4m3 value), at least -126,   q = e4m3(x * 2^-e).
// The scale is a power of two, so that x * 2^-e is exact and the rounding to e4m3 (to nearest, ties to even) is the only
// one: a value above 2^-6 * 2^e is off by at most 2^-4 of itself, smaller ones by at most 2^-10 * 2^e.  e comes from the
// exponent and three mantissa bits of the maximum, without a division.  Elements that are not finite become NaN and do not count
// in the maximum.  A scale per token because a slot is what this pool allocates: the neighbour of a slot may belong to
// another request, and a scale they shared would make one request's write change the other's values.
//
// Both kernels are bound by HBM: 2 + 1 bytes per element.  A thread takes 16 elements (16 bytes of the pool, 32 of the 16-bit
// rows), the D / 16 threads of a row are neighbours and exchange the maximum by DPP.  Measured: 16383 tokens of 64 heads of 128 written in 76 us (5.3 TB/s), 131072
// tokens of 16 heads read back in 159 us (5.1 TB/s); a copy of 2 GB runs at 4.96.
#include "common.hip.h"

namespace lsattn {
namespace {

template <int CTRL> __device__ __forceinline__ float max_dpp(float v) { return fmaxf(v, dpp_mov<CTRL>(v)); }
// maximum over each aligned group of N lanes (N = 1, 2, 4, 8)
template <int N> __device__ __forceinline__ float max_lanes(float v) {
  if (N > 1) v = max_dpp<0xB1>(v);   // quad_perm [1,0,3,2]
  if (N > 2) v = max_dpp<0x4E>(v);   // quad_perm [2,3,0,1]
  if (N > 4) v = max_dpp<0x141>(v);  // row_half_mirror
  return v;
}

struct Write8Params {
  const char* src;
  int64_t src_st, src_sh;  // bytes
  const void* dest_index;
  char* pool;
  int64_t pool_s0, pool_s1;
  uint8_t* scales;
  int64_t sc_s0, sc_s1;
  uint32_t pieces, heads;
  int64_t num_slots;
  FastDiv by_heads;
};

template <typename T, typename IT, int D>
__global__ __launch_bounds__(256) void kv_scatter_fp8_kernel(Write8Params p) {
  constexpr uint32_t LPR = D / 16;  // lanes per row
  const uint32_t gid = blockIdx.x * 256 + threadIdx.x;
  // (threads past the end repeat the last row and store nothing: no lane leaves before the exchange)
  const uint32_t piece = gid < p.pieces ? gid : p.pieces - LPR + (gid & (LPR - 1));
  const uint32_t row = piece / LPR, part = piece & (LPR - 1);
  const uint32_t t = div_by(row, p.by_heads), h = row - t * p.heads;
  const char* src = p.src + t * p.src_st + h * p.src_sh + part * 32;
  const u32x4 w0 = *(const u32x4*)src, w1 = *(const u32x4*)(src + 16);
  const int64_t slot = (int64_t)((const IT*)p.dest_index)[t];
  float x[16];
  unpack8<T>(w0, x);
  unpack8<T>(w1, x + 8);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const float a = fabsf(x[i]);
    const bool finite = a < INFINITY;  // (false for NaN)
    amax = fmaxf(amax, finite ? a : 0.f);
    x[i] = finite ? x[i] : __builtin_nanf("");
  }
  amax = max_lanes<(int)LPR>(amax);
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  int byte = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  byte = byte < 1 ? 1 : byte;
  const float inv = __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23);
  u32x4 q;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
    q[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, r, true);
  }
  if (gid >= p.pieces || slot < 0 || slot >= p.num_slots) return;
  *(u32x4*)(p.pool + slot * p.pool_s0 + h * p.pool_s1 + part * 16) = q;
  if (part == 0) p.scales[slot * p.sc_s0 + h * p.sc_s1] = (uint8_t)byte;
}

struct Read8Params {
  const char* pool;
  int64_t pool_s0, pool_s1;
  const uint8_t* scales;
  int64_t sc_s0, sc_s1;
  int64_t num_slots, num_reqs, max_seq_len, out_rows, max_len;
  const int32_t* req_to_tokens;
  const int32_t* b_req_idx;
  const int32_t* b_first;
  const int32_t* b_seq_len;
  const int32_t* b_start_loc;
  char* out;
  int64_t out_st, out_sh;  // bytes
  uint32_t heads, parts, rows_per_wg;  // parts: threads per token, heads * D / 16
  FastDiv by_parts;
};

// 2^e times an e4m3 value as 16 bits: one rounding (none in the normal range of the type).  What lies past the type's range (a row
// whose maximum rounded up to 65536, or to 2^128) becomes its largest value, NaN stays.
template <typename T> __device__ __forceinline__ uint32_t pack2_in_range(float a, float b) { return pack2<T>(a, b); }
template <> __device__ __forceinline__ uint32_t pack2_in_range<F16>(float a, float b) {
  a = fabsf(a) > 65504.f ? copysignf(65504.f, a) : a;
  b = fabsf(b) > 65504.f ? copysignf(65504.f, b) : b;
  return pack2<F16>(a, b);
}
// (bfloat16: infinities of a pair as the largest value)
__device__ __forceinline__ uint32_t finite_bf16(uint32_t w) {
  if ((w & 0x7fffu) == 0x7f80u) w -= 1;
  if ((w & 0x7fff0000u) == 0x7f800000u) w -= 0x10000u;
  return w;
}

template <typename T, int D>
__global__ __launch_bounds__(256) void kv_gather_fp8_kernel(Read8Params p) {
  constexpr uint32_t LPR = D / 16;
  const int64_t b = blockIdx.y;
  const int64_t len = p.b_seq_len[b] < p.max_len ? p.b_seq_len[b] : p.max_len;
  const int32_t first = p.b_first ? p.b_first[b] : 0, req = p.b_req_idx[b];
  const int64_t start = p.b_start_loc[b];
  const uint32_t rw = div_by(threadIdx.x, p.by_parts);
  // a workgroup takes rows_per_wg whole rows at a time where these have at most 256 pieces; longer rows take several steps
  for (uint32_t piece = p.parts < 256 ? threadIdx.x - rw * p.parts : threadIdx.x; piece < p.parts; piece += 256) {
    const int64_t i = (int64_t)blockIdx.x * p.rows_per_wg + (p.parts < 256 ? rw : 0);
    if ((p.parts < 256 && rw >= p.rows_per_wg) || i >= len || start + i < 0 || start + i >= p.out_rows) return;
    const uint32_t h = piece / LPR, part = piece & (LPR - 1);
    const int64_t pos = (int64_t)first + i;
    int64_t slot = -1;
    if (req >= 0 && req < p.num_reqs && pos >= 0 && pos < p.max_seq_len) slot = p.req_to_tokens[req * p.max_seq_len + pos];
    u32x4 o0 = {0, 0, 0, 0}, o1 = {0, 0, 0, 0};
    if (slot >= 0 && slot < p.num_slots) {
      const u32x4 w = *(const u32x4*)(p.pool + slot * p.pool_s0 + h * p.pool_s1 + part * 16);
      const uint32_t byte = p.scales[slot * p.sc_s0 + h * p.sc_s1];
      const float scale = __builtin_bit_cast(float, byte ? byte << 23 : 0x400000u);
      uint32_t r[8];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
        r[2 * k] = pack2_in_range<T>(lo[0] * scale, lo[1] * scale);
        r[2 * k + 1] = pack2_in_range<T>(hi[0] * scale, hi[1] * scale);
      }
      // (only rows of the largest exponent hold such; a look at every value costs 5 %)
      if (!__is_same(T, F16) && __builtin_amdgcn_ballot_w64(byte >= 247) != 0) {
#pragma unroll
        for (int k = 0; k < 8; k++) r[k] = finite_bf16(r[k]);
      }
      o0 = u32x4{r[0], r[1], r[2], r[3]};
      o1 = u32x4{r[4], r[5], r[6], r[7]};
    }
    char* dst = p.out + (start + i) * p.out_st + h * p.out_sh + part * 32;
    *(u32x4*)dst = o0;
    *(u32x4*)(dst + 16) = o1;
  }
}

bool head_dim_ok(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128; }

template <typename T, typename IT> void launch_write(const Write8Params& p, int64_t d, hipStream_t st) {
  const dim3 grid((p.pieces + 255) / 256), block(256);
  if (d == 128) LSATTN_LAUNCH_KERNEL((kv_scatter_fp8_kernel<T, IT, 128>), grid, block, 0, st, p);
  else if (d == 64) LSATTN_LAUNCH_KERNEL((kv_scatter_fp8_kernel<T, IT, 64>), grid, block, 0, st, p);
  else if (d == 32) LSATTN_LAUNCH_KERNEL((kv_scatter_fp8_kernel<T, IT, 32>), grid, block, 0, st, p);
  else LSATTN_LAUNCH_KERNEL((kv_scatter_fp8_kernel<T, IT, 16>), grid, block, 0, st, p);
}
template <typename T> void launch_read(const Read8Params& p, int64_t d, dim3 grid, hipStream_t st) {
  const dim3 block(256);
  if (d == 128) LSATTN_LAUNCH_KERNEL((kv_gather_fp8_kernel<T, 128>), grid, block, 0, st, p);
  else if (d == 64) LSATTN_LAUNCH_KERNEL((kv_gather_fp8_kernel<T, 64>), grid, block, 0, st, p);
  else if (d == 32) LSATTN_LAUNCH_KERNEL((kv_gather_fp8_kernel<T, 32>), grid, block, 0, st, p);
  else LSATTN_LAUNCH_KERNEL((kv_gather_fp8_kernel<T, 16>), grid, block, 0, st, p);
}

}  // namespace
}  // namespace lsattn

using namespace lsattn;

extern "C" int lsattn_kv_scatter_fp8(const lsattn_kv_scatter_fp8_args* a, void* stream) {
  if (!a || !a->src || !a->dest_index || !a->pool || !a->scales || a->num_tokens < 0 || a->num_heads < 1 || a->num_slots < 0)
    return LSATTN_ERR_INVALID_ARG;
  if (a->dtype != LSATTN_F16 && a->dtype != LSATTN_BF16) return LSATTN_ERR_UNSUPPORTED;
  if (!head_dim_ok(a->head_dim)) return LSATTN_ERR_UNSUPPORTED;
  if (a->dest_index_is_i64 != 0 && a->dest_index_is_i64 != 1) return LSATTN_ERR_INVALID_ARG;
  if (a->src_stride_t % 8 || a->src_stride_h % 8 || a->pool_stride_0 % 16 || a->pool_stride_1 % 16 ||
      (((uintptr_t)a->src | (uintptr_t)a->pool) & 15))
    return LSATTN_ERR_INVALID_ARG;
  const int64_t per_token = a->num_heads * (a->head_dim / 16);
  if (a->num_heads > kMaxUnits || per_token > kMaxUnits) return LSATTN_ERR_INVALID_ARG;
  hipStream_t st = (hipStream_t)stream;
  Write8Params p;
  p.src_st = a->src_stride_t * 2, p.src_sh = a->src_stride_h * 2;
  p.pool = (char*)a->pool, p.pool_s0 = a->pool_stride_0, p.pool_s1 = a->pool_stride_1;
  p.scales = a->scales, p.sc_s0 = a->scale_stride_0, p.sc_s1 = a->scale_stride_1;
  p.heads = (uint32_t)a->num_heads, p.num_slots = a->num_slots, p.by_heads = fast_div((uint32_t)a->num_heads);
  for (int64_t t0 = 0, slice = kMaxUnits / per_token; t0 < a->num_tokens; t0 += slice) {
    const int64_t n = a->num_tokens - t0 < slice ? a->num_tokens - t0 : slice;
    p.src = (const char*)a->src + t0 * p.src_st;
    p.dest_index = (const char*)a->dest_index + t0 * (a->dest_index_is_i64 ? 8 : 4);
    p.pieces = (uint32_t)(n * per_token);
    if (a->dtype == LSATTN_F16) {
      if (a->dest_index_is_i64) launch_write<F16, int64_t>(p, a->head_dim, st);
      else launch_write<F16, int32_t>(p, a->head_dim, st);
    } else {
      if (a->dest_index_is_i64) launch_write<BF16, int64_t>(p, a->head_dim, st);
      else launch_write<BF16, int32_t>(p, a->head_dim, st);
    }
  }
  return a->num_tokens > 0 ? check_launch() : LSATTN_OK;
}

extern "C" int lsattn_kv_gather_fp8(const lsattn_kv_gather_fp8_args* a, void* stream) {
  if (!a || !a->pool || !a->scales || !a->req_to_tokens || !a->b_req_idx || !a->b_seq_len || !a->b_start_loc || !a->out)
    return LSATTN_ERR_INVALID_ARG;
  if (a->batch < 0 || a->max_len_in_batch < 0 || a->num_heads < 1 || a->num_slots < 0 || a->num_reqs < 0 || a->max_seq_len < 0 || a->out_rows < 0)
    return LSATTN_ERR_INVALID_ARG;
  if (a->dtype != LSATTN_F16 && a->dtype != LSATTN_BF16) return LSATTN_ERR_UNSUPPORTED;
  if (!head_dim_ok(a->head_dim)) return LSATTN_ERR_UNSUPPORTED;
  if (a->out_stride_t % 8 || a->out_stride_h % 8 || a->pool_stride_0 % 16 || a->pool_stride_1 % 16 ||
      (((uintptr_t)a->out | (uintptr_t)a->pool) & 15))
    return LSATTN_ERR_INVALID_ARG;
  const int64_t parts = a->num_heads * (a->head_dim / 16);
  if (a->num_heads > kMaxUnits || parts > kMaxUnits || a->batch > 65535) return LSATTN_ERR_INVALID_ARG;
  if (a->batch == 0 || a->max_len_in_batch == 0) return LSATTN_OK;
  Read8Params p;
  p.pool = (const char*)a->pool, p.pool_s0 = a->pool_stride_0, p.pool_s1 = a->pool_stride_1;
  p.scales = a->scales, p.sc_s0 = a->scale_stride_0, p.sc_s1 = a->scale_stride_1;
  p.num_slots = a->num_slots, p.num_reqs = a->num_reqs, p.max_seq_len = a->max_seq_len, p.out_rows = a->out_rows, p.max_len = a->max_len_in_batch;
  p.req_to_tokens = a->req_to_tokens, p.b_req_idx = a->b_req_idx, p.b_first = a->b_first, p.b_seq_len = a->b_seq_len;
  p.b_start_loc = a->b_start_loc;
  p.out = (char*)a->out, p.out_st = a->out_stride_t * 2, p.out_sh = a->out_stride_h * 2;
  p.heads = (uint32_t)a->num_heads, p.parts = (uint32_t)parts;
  p.rows_per_wg = parts < 256 ? 256 / (uint32_t)parts : 1;
  p.by_parts = fast_div(p.parts);
  const int64_t wgs = (a->max_len_in_batch + p.rows_per_wg - 1) / p.rows_per_wg;
  if (wgs > 0x7fffffff) return LSATTN_ERR_INVALID_ARG;
  const dim3 grid((unsigned)wgs, (unsigned)a->batch);
  if (a->dtype == LSATTN_F16) launch_read<F16>(p, a->head_dim, grid, (hipStream_t)stream);
  else launch_read<BF16>(p, a->head_dim, grid, (hipStream_t)stream);
  return check_launch();
}
