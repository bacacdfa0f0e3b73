// Norm of each head's query and key rows and their rotation by position, in one pass. Part of kvq_int8.hip (included at
// its end: it shares the helpers above it).
#pragma once

namespace {

struct NormRopeArgs {
  const uint16_t* q;
  const uint16_t* k;
  uint16_t* qo;
  uint16_t* ko;
  const void* positions;
  const void* table;
  const void* qw;   // NULL: no norm
  const void* kw;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh, t_st, num_positions;
  int num_tokens, hq, heads, rd;   // heads: query heads, then key heads
  int groups;                      // groups of a token's heads, a wavefront each
  int per_wave;                    // heads that a wavefront takes, one after another for every row it holds
  int wide_pos, weight_bf16;
  float eps;
};

__device__ __forceinline__ float sum_quad(float x) {   // over each 4 lanes
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xf, 0xf, true));   // lanes 1 0 3 2
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xf, 0xf, true));   // 2 3 0 1
}
__device__ __forceinline__ float sum_half_row(float x) {   // over each 8 lanes
  x = sum_quad(x);
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, true));   // mirrored
}
__device__ __forceinline__ void eight(u32x4 w, float* o) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[2 * j] = bf16_lo(w[j]);
    o[2 * j + 1] = bf16_hi(w[j]);
  }
}
// 8 values at p[i ..], fp32 or bf16
__device__ __forceinline__ void eight_of(const void* p, bool bf16, int64_t i, float* o) {
  if (bf16) {
    eight(*reinterpret_cast<const u32x4*>((const uint16_t*)p + i), o);
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>((const float*)p + i), b = *reinterpret_cast<const f32x4*>((const float*)p + i + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j] = a[j];
      o[4 + j] = b[j];
    }
  }
}

// y = x / sqrt(mean x^2 + eps) * w; then (a, b) -> (a cos - b sin, b cos + a sin) for the pairs of the first rd channels,
// (i, i + rd / 2) or, INTER, (2 i, 2 i + 1); fp32 throughout, one rounding to bf16. A lane holds 8 pairs of a row, so a
// pair never leaves its lane, a row's mean is a sum over D / 16 lanes, and a token's cos and sin, which all of its heads
// share, are read once by the wavefront that takes them.
// Bound by memory: 16384 tokens of 32 + 8 heads of 128 (344 MB): 66 us, 5.2 TB/s, what a stream of as many bytes read as
// written reaches (5.3 .. 5.5). 32 tokens of 28 + 4 heads: 3.5 us, a launch.
template <int D, bool INTER, bool BF16_TABLE>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
  constexpr int LPR = D / 16, RPW = WAVE / LPR;   // lanes per row, rows per wavefront
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int item = blockIdx.x * 4 + wave;
  const int t = item / a.groups, h0 = (item - t * a.groups) * a.per_wave;
  if (t >= a.num_tokens) return;
  const int j = lane % LPR, row = lane / LPR;
  const int64_t pos = a.wide_pos ? ((const int64_t*)a.positions)[t] : (int64_t)((const int*)a.positions)[t];
  if (pos < 0 || pos >= a.num_positions) return;   // such a token's rows stay as they are
  const bool turn = 16 * j < a.rd;
  const int c0 = !INTER && turn ? 8 * j : 16 * j, c1 = !INTER && turn ? a.rd / 2 + 8 * j : 16 * j + 8;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  if (turn) {
    eight_of(a.table, BF16_TABLE, pos * a.t_st + 8 * j, cs);
    eight_of(a.table, BF16_TABLE, pos * a.t_st + a.rd / 2 + 8 * j, sn);
  }
  const int h1 = min(h0 + a.per_wave, a.heads);
  for (int h = h0 + row; h < h1; h += RPW) {
    const bool key = h >= a.hq;
    const uint16_t* x = key ? a.k + t * a.k_st + (h - a.hq) * a.k_sh : a.q + t * a.q_st + h * a.q_sh;
    uint16_t* o = key ? a.ko + t * a.ko_st + (h - a.hq) * a.ko_sh : a.qo + t * a.qo_st + h * a.qo_sh;
    float y[16];
    eight(*reinterpret_cast<const u32x4*>(x + c0), y);
    eight(*reinterpret_cast<const u32x4*>(x + c1), y + 8);
    if (a.qw) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) s = __builtin_fmaf(y[e], y[e], s);
      s = LPR == 8 ? sum_half_row(s) : sum_quad(s);
      const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(s, 1.f / D, a.eps));
      float w[16];
      eight_of(key ? a.kw : a.qw, a.weight_bf16, c0, w);
      eight_of(key ? a.kw : a.qw, a.weight_bf16, c1, w + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = y[e] * r * w[e];
    }
    float z[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int p0 = INTER ? 2 * e : e, p1 = INTER ? 2 * e + 1 : e + 8;
      // (lanes behind the rotated channels: cos 1, sin 0; an infinite value there must not meet the 0)
      z[p0] = turn ? __builtin_fmaf(-y[p1], sn[e], y[p0] * cs[e]) : y[p0];
      z[p1] = turn ? __builtin_fmaf(y[p0], sn[e], y[p1] * cs[e]) : y[p1];
    }
    *reinterpret_cast<u32x4*>(o + c0) = u32x4{pack_bf16x2_rne(z[0], z[1]), pack_bf16x2_rne(z[2], z[3]),
                                              pack_bf16x2_rne(z[4], z[5]), pack_bf16x2_rne(z[6], z[7])};
    *reinterpret_cast<u32x4*>(o + c1) = u32x4{pack_bf16x2_rne(z[8], z[9]), pack_bf16x2_rne(z[10], z[11]),
                                              pack_bf16x2_rne(z[12], z[13]), pack_bf16x2_rne(z[14], z[15])};
  }
}

}  // namespace

extern "C" {

int kvq_norm_rope(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, void* q_out,
                  int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh, int64_t num_tokens,
                  int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, const void* positions, int64_t position_bits,
                  const void* table, int64_t t_st, int64_t num_positions, int64_t rotary_dim, int64_t table_bf16,
                  const void* q_weight, const void* k_weight, int64_t weight_bf16, double eps, int64_t interleaved,
                  void* stream) {
  const char* nm = "norm_rope";
  if (head_dim != 64 && head_dim != 128) return fail("%s: head_dim must be 64 or 128, got %lld", nm, (long long)head_dim);
  if (num_tokens < 0 || num_tokens > INT32_MAX || num_q_heads < 0 || num_kv_heads < 0 || num_q_heads + num_kv_heads > 65535 ||
      num_positions < 0)
    return fail("%s: bad sizes", nm);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16)
    return fail("%s: rotary_dim must be a multiple of 16 up to head_dim, got %lld", nm, (long long)rotary_dim);
  if (position_bits != 32 && position_bits != 64) return fail("%s: positions must have 32 or 64 bits", nm);
  if (!(eps >= 0 && eps < INFINITY)) return fail("%s: eps must be finite and not negative", nm);
  if (num_tokens == 0 || num_q_heads + num_kv_heads == 0) { g_err.clear(); return KVQ_OK; }
  if ((num_q_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out)) || !positions || (rotary_dim && !table))
    return fail("%s: null pointer", nm);
  if (!q_weight != !k_weight) return fail("%s: both weights or none", nm);
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) ||
      (q_st | q_sh | k_st | k_sh | qo_st | qo_sh | ko_st | ko_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  if ((rotary_dim && (!aligned16(table) || t_st % 8)) || !aligned16(q_weight) || !aligned16(k_weight))
    return fail("%s: the table's rows and the weights must be 16-byte aligned", nm);
  NormRopeArgs a;
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.qo = (uint16_t*)q_out; a.ko = (uint16_t*)k_out;
  a.positions = positions; a.table = table; a.qw = q_weight; a.kw = k_weight;
  a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh; a.qo_st = qo_st; a.qo_sh = qo_sh; a.ko_st = ko_st; a.ko_sh = ko_sh;
  a.t_st = t_st; a.num_positions = num_positions;
  a.num_tokens = (int)num_tokens; a.hq = (int)num_q_heads; a.heads = (int)(num_q_heads + num_kv_heads); a.rd = (int)rotary_dim;
  a.wide_pos = position_bits == 64; a.weight_bf16 = weight_bf16 != 0; a.eps = (float)eps;
  const int rpw = head_dim == 128 ? 8 : 16;
  a.per_wave = rpw;
  a.groups = (a.heads + a.per_wave - 1) / a.per_wave;
  const int64_t items = num_tokens * a.groups;
  if (items > INT32_MAX - 3) return fail("%s: too many tokens and heads for one call", nm);
  const dim3 grid((unsigned)((items + 3) / 4));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  void (*kern)(NormRopeArgs) =
      head_dim == 128 ? (interleaved ? (table_bf16 ? norm_rope_kernel<128, true, true> : norm_rope_kernel<128, true, false>)
                                     : (table_bf16 ? norm_rope_kernel<128, false, true> : norm_rope_kernel<128, false, false>))
                      : (interleaved ? (table_bf16 ? norm_rope_kernel<64, true, true> : norm_rope_kernel<64, true, false>)
                                     : (table_bf16 ? norm_rope_kernel<64, false, true> : norm_rope_kernel<64, false, false>));
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a);
  return launched(nm);
}

}  // extern "C"
