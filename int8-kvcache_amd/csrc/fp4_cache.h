// The 4-bit cache: e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), two to a byte, the even channel's in the low
// half, and one exponent byte for each 32 channels of a row (page, slot, head), K and V apart; a cached value is
// code * 2^(byte - 127), exact in bf16; one instruction converts two of them. A row's scales are its own, so
// rows are written, moved and dropped one by one. Part of kvq_int8.hip (included at its end: it shares the helpers above it).
//
//   quant_fp4_kernel   quantize a step's new K/V rows into their slots
//   read_fp4_kernel    ranges of the requests' keys back to bf16 rows
//   fp4_pages_kernel   pages back to a contiguous bf16 cache
//   fp4_prefill_kernel attention of long queries over that
//   fp4_attn_kernel    attention of short queries
#pragma once

namespace {

constexpr int FP4_GROUP = 32;             // channels per exponent byte
constexpr int FP4_MIN_E = 27, FP4_MAX_E = 252;   // the exponent bytes that the write makes: 2^-100 .. 2^125

// a cache's exponent bytes: those of (page p, head h, slot n) are D / 32 bytes at p * sb + h * sh + n * D / 32
struct Fp4Scales {
  uint8_t* k;
  uint8_t* v;
  int64_t sb, sh;
};

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// 8 codes -> 8 bf16, times 2^(byte - 127) (byte << 23 as a float's bits; exact, the smallest products as subnormals)
__device__ __forceinline__ u32x4 fp4_to_bf16(uint32_t w, uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3))};
}
// exponent bytes that no write makes (a buffer that was never cleared) still give finite values
__device__ __forceinline__ uint32_t fp4_finite(uint32_t byte) { return min(byte, (uint32_t)FP4_MAX_E); }

// ------------------------------------------------------------------------------------------------
// Quantize rows into their slots. For the 32 values x of a group, t = max |x| (finite x):
//   e = floor(log2 t) - 2, one more where t 2^-e > 7, between -100 and 125;   code = the nearest of x 2^-e, ties to even, at
//   most 6: what lies above 6 is off by no more than the half step from 4 to 6
// infinities become 6, NaN 0. A lane holds 8 channels, so a group is 4 lanes and its maximum two exchanges within them.
// Bound by memory: each value is read once, 16 bytes a lane, and written once. 16384 tokens of 4 heads of 128, K and V (42 MB):
// 10.3 us, 4.1 TB/s; 32 tokens: 3.2 us, a launch and two dependent loads (slot, row).
// ------------------------------------------------------------------------------------------------
struct QuantFp4Args {
  const uint16_t* key;
  const uint16_t* value;
  uint8_t* kc;
  uint8_t* vc;
  const int64_t* slots;
  Fp4Scales s;
  int64_t key_st, key_sh, val_st, val_sh, kc_sb, kc_sn, kc_sh, vc_sb, vc_sn, vc_sh, num_slots;
  int num_tokens, heads, lbs;
};

__device__ __forceinline__ float max_quad(float x) {   // over each 4 lanes
  x = __builtin_fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xf, 0xf, true)));
  return __builtin_fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xf, 0xf, true)));
}
// a lane's 8 codes; byte: the group's exponent byte
__device__ __forceinline__ uint32_t fp4_codes8(u32x4 w, uint32_t& byte) {
  const float t = max_quad(absmax8(w));
  const int e = (int)((__float_as_uint(t) + 0x1fffffu) >> 23) - 2;   // a mantissa above 1.75 carries
  byte = (uint32_t)min(max(e, FP4_MIN_E), FP4_MAX_E);
  const float m = __uint_as_float((254u - byte) << 23);
  uint32_t codes = 0;
  auto clean = [&](float x) { return x == x ? x * m : 0.f; };
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, clean(bf16_lo(w[0])), clean(bf16_hi(w[0])), 1.f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, clean(bf16_lo(w[1])), clean(bf16_hi(w[1])), 1.f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, clean(bf16_lo(w[2])), clean(bf16_hi(w[2])), 1.f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, clean(bf16_lo(w[3])), clean(bf16_hi(w[3])), 1.f, 3);
}

template <int D>
__global__ __launch_bounds__(256) void quant_fp4_kernel(QuantFp4Args a) {
  constexpr int LPR = D / 8;              // lanes per row
  constexpr int RPB = 256 / LPR;          // (token, head) rows per workgroup
  const int64_t item = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  const int t = (int)(item / a.heads), h = (int)(item - (int64_t)t * a.heads), c = threadIdx.x % LPR;
  if (t >= a.num_tokens) return;
  const int64_t slot = a.slots[t];
  const u32x4 kw = *reinterpret_cast<const u32x4*>(a.key + t * a.key_st + h * a.key_sh + 8 * c);
  const u32x4 vw = *reinterpret_cast<const u32x4*>(a.value + t * a.val_st + h * a.val_sh + 8 * c);
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t page = slot >> a.lbs;
  const int off = (int)(slot & ((1 << a.lbs) - 1));
  uint32_t kb, vb;
  const uint32_t kq = fp4_codes8(kw, kb), vq = fp4_codes8(vw, vb);
  *reinterpret_cast<uint32_t*>(a.kc + page * a.kc_sb + off * a.kc_sn + h * a.kc_sh + 4 * c) = kq;
  *reinterpret_cast<uint32_t*>(a.vc + page * a.vc_sb + off * a.vc_sn + h * a.vc_sh + 4 * c) = vq;
  if (c % 4 == 0) {
    const int64_t at = page * a.s.sb + h * a.s.sh + off * (D / FP4_GROUP) + c / 4;
    a.s.k[at] = (uint8_t)kb;
    a.s.v[at] = (uint8_t)vb;
  }
}

// ------------------------------------------------------------------------------------------------
// Read ranges of keys back: request r's positions start[r] .. are rows cu_k[r] .. cu_k[r + 1] - 1 of k_out / v_out. One
// wavefront takes one aligned run of 16 positions (one page) of one head, as read_block_kernel does. Bound by memory: 33.5 MB
// of rows out of 8.9 MB of codes 9.6 us, 4.4 TB/s; 680 MB past the caches (NT: loads and stores that leave them alone) 131 us,
// 5.2 TB/s, what as many bytes read and written elsewhere reach.
// ------------------------------------------------------------------------------------------------
struct ReadFp4Args {
  const uint8_t* kc;
  const uint8_t* vc;
  uint16_t* ko;
  uint16_t* vo;
  const int* start;
  const int* cu_k;
  const int* block_table;
  Fp4Scales s;
  int64_t kc_sb, kc_sn, kc_sh, vc_sb, vc_sn, vc_sh, ko_st, ko_sh, vo_st, vo_sh, bt_stride;
  int num_seqs, num_rows, heads, num_blocks, lbs, items;
};

template <int D, bool NT>
__global__ __launch_bounds__(256) void read_fp4_kernel(ReadFp4Args a) {
  constexpr int LPR = D / 8, RPL = WAVE / LPR, N = 16 / RPL, SB = D / FP4_GROUP;
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int item = blockIdx.x * 4 + wave;
  if (item >= a.items) return;
  const int u = item / a.heads, h = item - u * a.heads;
  const SlotRequest q = request_of_slot(a.cu_k, a.start, a.num_seqs, 4, u, lane);
  const int r = q.r, row0 = q.cu0, n = min(q.cu1, a.num_rows) - row0, start = q.of;
  if (start < 0) return;
  const int b0 = ((start >> 4) + u - ((row0 >> 4) + 2 * r)) << 4;
  const int first = max(start, b0), last = min(start + n, b0 + 16);
  if (first >= last) return;
  int page = page_at(a.block_table, a.bt_stride, r, b0 >> a.lbs);
  page = page >= 0 && page < a.num_blocks ? page : 0;
  const int off = b0 & ((1 << a.lbs) - 1);
  const int row = lane / LPR, c = lane % LPR;
  const int64_t si = (int64_t)page * a.s.sb + (int64_t)h * a.s.sh + (int64_t)off * SB + c / 4;
  const uint8_t* kc = a.kc + (int64_t)page * a.kc_sb + (int64_t)off * a.kc_sn + (int64_t)h * a.kc_sh + 4 * c;
  const uint8_t* vc = a.vc + (int64_t)page * a.vc_sb + (int64_t)off * a.vc_sn + (int64_t)h * a.vc_sh + 4 * c;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = row + RPL * j, p = b0 + i;
    if (p < first || p >= last) continue;
    const int64_t t = row0 + p - start;
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(kc + (int64_t)i * a.kc_sn);
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(vc + (int64_t)i * a.vc_sn);
    const uint32_t kb = fp4_finite(a.s.k[si + i * SB]), vb = fp4_finite(a.s.v[si + i * SB]);
    u32x4* ko = reinterpret_cast<u32x4*>(a.ko + t * a.ko_st + (int64_t)h * a.ko_sh + 8 * c);
    u32x4* vo = reinterpret_cast<u32x4*>(a.vo + t * a.vo_st + (int64_t)h * a.vo_sh + 8 * c);
    if constexpr (NT) {
      const uint32_t k = __builtin_nontemporal_load(kp), v = __builtin_nontemporal_load(vp);
      __builtin_nontemporal_store(fp4_to_bf16(k, kb), ko);
      __builtin_nontemporal_store(fp4_to_bf16(v, vb), vo);
    } else {
      *ko = fp4_to_bf16(*kp, kb);
      *vo = fp4_to_bf16(*vp, vb);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Pages back to a contiguous bf16 cache [P, block_size, H, D] (as dequant_pages_kernel leaves it): page p is
// block_table[src_req[p], src_j[p]]. A lane converts 8 channels of one (slot, head), K or V by blockIdx.z; lanes in the order
// of the output. The prefill over it is the block-scaled cache's, whose weights leave room for large values: every scale 1.
// A chunk's queries are many per key, so that its keys are converted once, and not by each tile of queries. 3,533 keys of 8 heads
// (18 MB): 6.2 us, 3 TB/s.
// ------------------------------------------------------------------------------------------------
struct Fp4PagesArgs {
  const uint8_t* kc;
  const uint8_t* vc;
  uint16_t* ko;
  uint16_t* vo;
  f32x4* table;   // [H, P * block_size / 16]
  const int* block_table;
  const int* src_req;
  const int* src_j;
  Fp4Scales s;
  int64_t kc_sb, kc_sn, kc_sh, vc_sb, vc_sn, vc_sh, bt_stride;
  int heads, num_blocks, bs;
};
template <int D>
__global__ __launch_bounds__(256) void fp4_pages_kernel(Fp4PagesArgs a) {
  constexpr int LPR = D / 8;
  const int p = blockIdx.x;
  const int r = __builtin_amdgcn_readfirstlane(a.src_req[p]), j = __builtin_amdgcn_readfirstlane(a.src_j[p]);
  int page = __builtin_amdgcn_readfirstlane(a.block_table[(int64_t)r * a.bt_stride + j]);
  page = page >= 0 && page < a.num_blocks ? page : 0;
  const bool v = blockIdx.z != 0;
  const uint8_t* cache = v ? a.vc + (int64_t)page * a.vc_sb : a.kc + (int64_t)page * a.kc_sb;
  const int64_t sn = v ? a.vc_sn : a.kc_sn, sh = v ? a.vc_sh : a.kc_sh;
  const uint8_t* scale = (v ? a.s.v : a.s.k) + (int64_t)page * a.s.sb;
  if (!v) {
    const int nb16 = a.bs / 16, entries = a.heads * nb16;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < entries; i += 256 * gridDim.y)
      a.table[((int64_t)(i / nb16) * gridDim.x + p) * nb16 + i % nb16] = f32x4{1.f, 0.f, 1.f, 0.f};
  }
  u32x4* out = reinterpret_cast<u32x4*>((v ? a.vo : a.ko) + (int64_t)p * a.bs * a.heads * D);
  const int n = a.bs * a.heads * LPR;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < n; i += 256 * gridDim.y) {
    const int c = i % LPR, at = i / LPR, t = at / a.heads, h = at - t * a.heads;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(cache + t * sn + h * sh + 4 * c);
    out[i] = fp4_to_bf16(w, fp4_finite(scale[h * a.s.sh + t * (D / FP4_GROUP) + c / 4]));
  }
}

// The bf16 prefill over those pages. Its weights are a sum of two bf16, as the short queries' below, so that a row's accuracy does
// not depend on how many tokens its request has: 1.6e-3 against 64 bits, the output's own rounding, where one bf16 had 2.1e-3.
// The second product over V costs what it adds to the matrix cores' work, half as much again: 2 x 8,192 tokens of 32 / 8 heads x
// 128 1,260 us with the copy in place of 910, 700 tokens and 333 behind 2,167 keys 53.6 in place of 47.7.
template <int D, bool SPLIT>
__global__ __launch_bounds__(256, D == 64 ? 4 : 3) void fp4_prefill_kernel(PrefillArgs a) {
  prefill_body<D, PR_SRC_BF16_FP4, SPLIT>(a);
}

// ------------------------------------------------------------------------------------------------
// Attention of short queries: attn_kernel's plan and pieces. Per (request, kv head) and 32-key tile, log2 domain:
//   S    = K . q^T     v_mfma_f32_16x16x32_bf16: a lane's 32 (D = 64: 16) channels of a key lie in one group, so a conversion
//                      makes two codes and their exponent two bf16 operands, exactly; q as it is
//   e    = S scale     m: the row's largest e plus BLOCK_REF, raised where it lags by more than 8
//   P    = 2^(e - m),  l += P
//   O   += V^T . P     v_mfma_f32_16x16x32_bf16, twice: V's values as bf16 (exact), P as a sum of two bf16, cut off (2^-14
//                      of each weight; one bf16 was as far off as the output's own rounding, 2.3e-3 in all in place of 1.7e-3, and
//                      decode of 128 x 32768 keys 354 us in place of 364, verification of 64 x 8 tokens 51 in place of 56)
// A conversion leaves two channels of a key side by side; the product sums over what is side by side. Not PACK: v_perm pairs
// keys of a channel, two for four values. PACK (at most 8 (token, q head) rows per kv head): the rows are the columns 0 .. 7 and
// again 8 .. 15, and the product runs over (key, channel of the pair): P stands beside zeros, in columns 0 .. 7 for the even
// channel and in 8 .. 15 for the odd one. No value moves, and the accumulators are half as many.
// (The scaled MFMA takes the codes without a conversion, but sums products of 8-bit floats to 2^-13 of the largest of each few:
// scores were 7e-4 off.)
// Weights are kept below 2^-24 (BLOCK_REF), so that a sum over a million keys of V's largest values (6 2^125) stays finite.
//
// What bounds it, and the time (4 KV heads of 128, 7 q heads each):
//   decode, 128 requests of 32768 keys   364 us for 2.29 GB: 6.3 TB/s of the 6.9 that a plain stream reads (whole lines, below)
//   decode, 1 request of 4096 keys       9.3 us and 3.9 for the merge: latency of launch, plan, table, first tile and merge
//   64 requests of 8 tokens, 512 .. 8192 keys 49 us and 8 for the merge, for 89 MB: issue of vector instructions. Of a tile and
//                  16 rows it needs 64 conversions, 32 v_perm and some 100 others; two row tiles a wavefront share the first two
// 12 or 16 wavefronts to a workgroup, 3 or 4 to a SIMD, change neither of the last two (the third, when a weight was one bf16 and
// each row tile had a wavefront: 62 .. 64 us where 8 took 63).
// ------------------------------------------------------------------------------------------------
struct Fp4AttnArgs {
  AttnArgs a;   // (first: fresh_args)
  Fp4Scales s;
  float* lse;   // [tokens, q heads], or NULL
  int64_t lse_st;
  int apart;    // K and V rows are not side by side
};
static_assert(offsetof(Fp4AttnArgs, a) == 0 && sizeof(AttnArgs) % 8 == 0, "AttnArgs lead the kernel arguments");
__device__ __forceinline__ const Fp4AttnArgs& fresh_fp4() {
  auto* p = (const __attribute__((address_space(4))) void*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Fp4AttnArgs*)p;
}
constexpr float LN2 = 0.6931471805599453f;

// A wavefront's ring of tiles in LDS. A slot holds two halves of 16 keys, each its rows' K and V codes in 16-byte chunks (chunk
// p of row r: K's first, then V's), then the rows' exponent bytes, K's and V's (and 256 bytes in all, what a DMA of 4 bytes a lane
// writes).
constexpr int fp4_chunks(int d) { return d / 16; }                             // chunks of a row, K's and V's
constexpr int fp4_codes(int d) { return 16 * 16 * fp4_chunks(d); }             // bytes of a half's codes
constexpr int fp4_half(int d) { return fp4_codes(d) + 256; }
constexpr int fp4_slot(int d) { return 2 * fp4_half(d); }
constexpr int fp4_accs(int d, bool pack) { return pack ? d / 32 : d / 16; }
// what a lane hands over in the merge of key splits: accumulators, maximum, denominator
constexpr int fp4_merge_fields(int d, bool pack) { return 4 * fp4_accs(d, pack) + 2; }
// Wavefronts of a workgroup: what its registers and LDS leave room for. Segments that are not cut are shared by all of them.
constexpr int FP4_WAVES = 8;
// Tiles of a wavefront's ring. Up to 8 query rows a key's products are few and the loads are what it waits for. In segments that
// are cut, of few wavefronts: 4 (ragged decode, 96 requests of up to 32768 keys: 66 us; 2 slots, with twice the workgroups on a
// unit, 71). Whole ones: 2 (128 requests of 32768 keys 367 us, of 4096 74; 4 slots 374 and 76; the units are full either way and
// ask for less at once; 12 and 16 wavefronts of 2 slots: 370, 366). More rows: 2, where the products cover the loads and more
// workgroups fit (24 requests of 4 tokens: 24.3 us; 4 slots 26.5).
constexpr int fp4_slots(bool pack, bool cut) { return pack && cut ? 4 : 2; }
// The DMAs' cache policy: streaming (2) where K and V are read once; the wavefronts of several row tiles read the same lines
// (verification, 16 requests of 8 tokens: 23.6 us against 25.4; 24 of 4: 24.3 against 25.9; 64 of 8: 54.7 against 56.9; 64 of 4
// over 4096 keys each: 42.0 against 40.9).
constexpr int fp4_dma_aux(bool pack) { return pack ? 2 : 0; }

// 16 query rows as the MFMA's second operand: lane (n, g) holds row n's channels (D / 4) g + 8 s .. + 7 in step s.
template <int D>
struct Fp4Query {
  u32x4 raw[D / 32];
  bf16x8 op[D / 32];
  float odd;   // 0, or NaN where the row holds a NaN or an infinity: then its output is NaN too
  __device__ __forceinline__ void load(const uint16_t* row, bool real, int g) {
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      raw[s] = u32x4{0u, 0u, 0u, 0u};
      if (real) raw[s] = *reinterpret_cast<const u32x4*>(row + (D / 4) * g + 8 * s);
    }
  }
  __device__ __forceinline__ void make() {
    odd = 0.f;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      op[s] = *reinterpret_cast<bf16x8*>(&raw[s]);
#pragma unroll
      for (int j = 0; j < 4; ++j) odd = __builtin_fmaf(bf16_lo(raw[s][j]), 0.f, __builtin_fmaf(bf16_hi(raw[s][j]), 0.f, odd));
    }
    odd = group4_sum(odd);
  }
};
// what a float's upper half, as bf16, leaves of it (exact)
__device__ __forceinline__ float behind_bf16(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// S^T[key][row] of 16 keys and NR row tiles: lane (n, g) holds row n's keys 4 g + i. The keys are converted once.
template <int D, int NR>
__device__ __forceinline__ void fp4_scores(const uint32_t (&k)[D / 32], uint32_t byte, const Fp4Query<D> (&q)[NR], int b, f32x4 (&z)[NR][2]) {
#pragma unroll
  for (int t = 0; t < NR; ++t) z[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    const u32x4 w = fp4_to_bf16(k[s], byte);
#pragma unroll
    for (int t = 0; t < NR; ++t)
      z[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(&w), q[t].op[s], z[t][b], 0, 0, 0);
  }
}
// key_weights_kernel's loads: a streaming load of each lane's own `off` from a base that the wavefront shares, through a buffer
// descriptor. The base and `uni` stay in scalar registers, a lane's part is 32 bits (64-bit addresses take two vector registers
// and an addition a load).
template <typename T>
__device__ __forceinline__ T load_at(const uint8_t* base, uint32_t off, uint32_t uni) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, INT32_MAX, QC_RSRC_WORD3);
  if constexpr (sizeof(T) == 16) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b128(r, off, uni, QC_LOAD_AUX));
  else if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(r, off, uni, QC_LOAD_AUX));
  else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b8(r, off, uni, QC_LOAD_AUX));
}
// page p of `base`: strides are below 4 GiB (check_fp4)
__device__ __forceinline__ const uint8_t* page_base(const uint8_t* base, int p, uint32_t stride) {
  return base + (uint64_t)(uint32_t)p * stride;
}
// the lane's words of 16 keys' codes
template <int D>
__device__ __forceinline__ void load_k16(uint32_t (&k)[D / 32], const uint8_t* base, uint32_t off, uint32_t uni) {
  if constexpr (D == 128) {
    const u32x4 w = load_at<u32x4>(base, off, uni);
#pragma unroll
    for (int s = 0; s < 4; ++s) k[s] = w[s];
  } else {
    const u32x2 w = load_at<u32x2>(base, off, uni);
    k[0] = w.x;
    k[1] = w.y;
  }
}

// Where chunk p of row r of a half stands in LDS, in chunks. A DMA writes 64 chunks in the order of its lanes; which chunk a lane
// asks for is free. K and V rows side by side in memory (vLLM's views): a DMA takes 8 (D = 64: 16) whole rows, so that it asks for
// lines of 128 bytes (half lines, K's and V's in turn, stream at 5.9 TB/s, whole ones at 6.8). Apart: K's rows, then V's. The
// chunks of a row are swapped by the row (exclusive or), so that the reads below meet few banks twice.
template <int D>
__device__ __forceinline__ int fp4_place(bool apart, int r, int p) {
  constexpr int CH = fp4_chunks(D), H = CH / 2;
  return apart ? (p / H) * 16 * H + r * H + ((p % H) ^ ((r * H / 4) & (H - 1))) : r * CH + (p ^ (r & (CH - 1)));
}

// One wavefront's share of a piece: NR row tiles from row0 on, key tiles c_begin + ks, c_begin + ks + KS, .. below c_end.
template <int D, bool PACK, int NR, int S>
__device__ __forceinline__ void attend_fp4(int seq, int tok, int qlen, int seqlen, int kvh, int row0, int c_begin, int c_end,
                                           int ks, int KS, int part, int nparts, uint8_t* lds, int lane) {
  const Fp4AttnArgs& args = fresh_fp4();
  const AttnArgs& a = args.a;
  constexpr int RT = PACK ? 8 : 16;        // rows of a tile
  static_assert(!PACK || NR == 1, "at most 8 rows are one tile");
  constexpr int VT = D / 16, NA = fp4_accs(D, PACK), SB = D / FP4_GROUP;
  constexpr int SLOT = fp4_slot(D), HALF = fp4_half(D), CODES = fp4_codes(D), CH = fp4_chunks(D);
  constexpr int DMAS = CODES / 1024, OPS = 2 * (DMAS + 1);   // DMAs of a half's codes; vector memory operations of a tile
  static_assert(S * OPS < 64, "vmcnt range");
  const int G = PACK ? a.G >> 1 : a.G;     // (PACK: the plan counts 16 columns a tile, two a row)
  const bool active = row0 < qlen * G;
  const int num_blocks = a.num_blocks, lbs = a.lbs;
  const uint32_t c_sb = (uint32_t)a.k_sb, c_sn = (uint32_t)a.k_sn, s_sb = (uint32_t)args.s.sb;
  seq = __builtin_amdgcn_readfirstlane(seq);
  tok = __builtin_amdgcn_readfirstlane(tok);
  qlen = __builtin_amdgcn_readfirstlane(qlen);
  kvh = __builtin_amdgcn_readfirstlane(kvh);
  row0 = __builtin_amdgcn_readfirstlane(row0);
  c_begin = __builtin_amdgcn_readfirstlane(c_begin);
  c_end = __builtin_amdgcn_readfirstlane(c_end);
  part = __builtin_amdgcn_readfirstlane(part);
  nparts = __builtin_amdgcn_readfirstlane(nparts);
  ks = __builtin_amdgcn_readfirstlane(ks);
  KS = __builtin_amdgcn_readfirstlane(KS);
  const int n = lane & 15, g = lane >> 4;
  const int L = __builtin_amdgcn_readfirstlane(seqlen);
  if (L <= 0 || !active) c_end = c_begin;
  const int nt = c_begin + ks < c_end ? (c_end - c_begin - ks + KS - 1) / KS : 0;
  auto tile = [&](int j) { return c_begin + ks + j * KS; };
  const int* bt = a.block_table + (int64_t)seq * a.bt_stride;
  const int bs = 1 << lbs;
  auto div_g = [&](int x) { return G == 1 ? x : a.g_inv ? (int)__umulhi((unsigned)x, a.g_inv) : x / G; };

  int rtok[NR], rh[NR];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    const int R = row0 + RT * t + (n & (RT - 1));
    rtok[t] = div_g(R);
    rh[t] = R - rtok[t] * G;
  }
  const int lim_lo = L - qlen + 1 + __builtin_amdgcn_readfirstlane(div_g(row0));
  Fp4Query<D> q[NR];
  if (nt > 0) {
#pragma unroll
    for (int t = 0; t < NR; ++t)
      q[t].load(a.q + (int64_t)(tok + min(rtok[t], qlen - 1)) * a.q_st + (int64_t)(kvh * G + rh[t]) * a.q_sh, rtok[t] < qlen, g);
  }

  // ---- what each lane's DMAs ask for, beside a page and slot, and where it reads ----
  const bool apart = args.apart;
  const uint8_t* src[DMAS];
#pragma unroll
  for (int u = 0; u < DMAS; ++u) {
    const int at = 64 * u + lane;   // the place this lane's chunk goes to: fp4_place the other way round
    constexpr int H = CH / 2;
    int r, p;
    if (apart) {
      r = at / H % 16;
      p = at / (16 * H) * H + ((at % H) ^ ((r * H / 4) & (H - 1)));
    } else {
      r = at / CH;
      p = (at % CH) ^ (r & (CH - 1));
    }
    src[u] = (const uint8_t*)(p < H ? a.kc + (int64_t)kvh * a.k_sh : a.vc + (int64_t)kvh * a.v_sh) + (uint64_t)(r * c_sn) + 16 * (p % H);
  }
  // exponent bytes: 4 SB words of K's, as many of V's, then both again
  const uint8_t* ssrc = ((lane / (4 * SB)) % 2 ? args.s.v : args.s.k) + (int64_t)kvh * args.s.sh + 4 * (lane % (4 * SB));
  const uint32_t base = (uint32_t)(uintptr_t)lds;
  uint32_t kadr, vadr[4];
  {
    const int ch = g * (D / 8);   // byte of the row's K
    kadr = base + 16 * fp4_place<D>(apart, n, ch / 16) + ch % 16;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ch = n * (VT / 2);
    vadr[i] = base + 16 * fp4_place<D>(apart, 4 * g + i, CH / 2 + ch / 16) + ch % 16;
  }
  const uint32_t ksadr = base + CODES + n * SB + g * (D / 4) / FP4_GROUP, vsadr = base + CODES + 16 * SB + 4 * g * SB;
  const uint32_t vrot = 8 * (n * VT / FP4_GROUP) + 9;   // brings the byte of the lane's V channels to bits 23 .. 30

  // a tile's two page ids are asked for one tile ahead
  auto half_key = [&](int j, int b) { return min(tile(min(j, nt - 1)) * TILE + 16 * b, (L - 1) & ~15); };
  int next[2] = {0, 0};
  auto fetch = [&](int j) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
      next[b] = ((const __attribute__((address_space(4))) int*)bt)[__builtin_amdgcn_readfirstlane(half_key(j, b) >> lbs)];
  };
  auto load = [&](uint32_t slot, int j) {   // tile j, whose page ids are here; slot: its offset in the ring
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int id = __builtin_amdgcn_readfirstlane(next[b]), p = (unsigned)id < (unsigned)num_blocks ? id : 0;
      const uint32_t of = half_key(j, b) & (bs - 1);
      const uint64_t co = (uint64_t)(uint32_t)p * c_sb + of * c_sn, so = (uint64_t)(uint32_t)p * s_sb + of * SB;
      uint8_t* dst = lds + slot + b * HALF;
#pragma unroll
      for (int u = 0; u < DMAS; ++u)
        __builtin_amdgcn_global_load_lds((const void*)(src[u] + co), (__attribute__((address_space(3))) void*)(dst + 1024 * u), 16, 0, fp4_dma_aux(PACK));
      __builtin_amdgcn_global_load_lds((const void*)(ssrc + so), (__attribute__((address_space(3))) void*)(dst + CODES), 4, 0, fp4_dma_aux(PACK));
    }
  };

  if (nt > 0) {
    fetch(0);
#pragma unroll
    for (int j = 0; j < S - 1; ++j)
      if (j < nt) {
        load(j * SLOT, j);
        fetch(j + 1);
      }
#pragma unroll
    for (int t = 0; t < NR; ++t) q[t].make();
  } else {
#pragma unroll
    for (int t = 0; t < NR; ++t) q[t].odd = 0.f;
  }
  float rs[NR], m[NR], l[NR];
  int lim[NR];
  f32x4 acc[NR][NA];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    rs[t] = a.sm_log2 + q[t].odd;
    lim[t] = rtok[t] < qlen ? L - qlen + 1 + rtok[t] : L;
    m[t] = FP4_NO_SCORE;
    l[t] = 0.f;
#pragma unroll
    for (int c = 0; c < NA; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t pick = n >= 8 ? 0x03020c0cu : 0x0c0c0302u;   // PACK: a weight's upper half to where the column has it, beside 0

  // tile j, at `slot` of the ring (the reads' statements wait for themselves: the compiler sees neither the DMAs nor that they
  // are done)
  auto compute = [&](auto masked_t, uint32_t slot, int j) {
    constexpr bool MASKED = decltype(masked_t)::value;
    const int n0 = tile(j) * TILE;
    uint32_t kw[2][D / 32], ksw[2], v[8], vs[2][D / 32];
    if constexpr (D == 128) {
      u32x4 k0, k1;
      asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%c6\n\t"
                   "ds_read_u8 %2, %5\n\tds_read_u8 %3, %5 offset:%c6\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(k0), "=&v"(k1), "=&v"(ksw[0]), "=&v"(ksw[1]) : "v"(kadr + slot), "v"(ksadr + slot), "n"(HALF) : "memory");
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kw[0][i] = k0[i];
        kw[1][i] = k1[i];
      }
    } else {
      u32x2 k0, k1;
      asm volatile("ds_read_b64 %0, %4\n\tds_read_b64 %1, %4 offset:%c6\n\t"
                   "ds_read_u8 %2, %5\n\tds_read_u8 %3, %5 offset:%c6\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(k0), "=&v"(k1), "=&v"(ksw[0]), "=&v"(ksw[1]) : "v"(kadr + slot), "v"(ksadr + slot), "n"(HALF) : "memory");
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kw[0][i] = k0[i];
        kw[1][i] = k1[i];
      }
    }
    // ---- scores; key of (b, i) = n0 + 16 b + 4 g + i ----
    f32x4 z[NR][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) fp4_scores<D, NR>(kw[b], ksw[b], q, b, z);
    if constexpr (D == 128) {   // (while the products run)
      u32x4 x0, x1;
      asm volatile("ds_read_b32 %0, %10\n\tds_read_b32 %1, %11\n\tds_read_b32 %2, %12\n\t"
                   "ds_read_b32 %3, %13\n\tds_read_b32 %4, %10 offset:%c15\n\tds_read_b32 %5, %11 offset:%c15\n\t"
                   "ds_read_b32 %6, %12 offset:%c15\n\tds_read_b32 %7, %13 offset:%c15\n\tds_read_b128 %8, %14\n\t"
                   "ds_read_b128 %9, %14 offset:%c15\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]),
                     "=&v"(x0), "=&v"(x1)
                   : "v"(vadr[0] + slot), "v"(vadr[1] + slot), "v"(vadr[2] + slot), "v"(vadr[3] + slot), "v"(vsadr + slot), "n"(HALF) : "memory");
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vs[0][i] = x0[i];
        vs[1][i] = x1[i];
      }
    } else {
      u32x2 x0, x1;
      asm volatile("ds_read_u16 %0, %10\n\tds_read_u16 %1, %11\n\tds_read_u16 %2, %12\n\t"
                   "ds_read_u16 %3, %13\n\tds_read_u16 %4, %10 offset:%c15\n\tds_read_u16 %5, %11 offset:%c15\n\t"
                   "ds_read_u16 %6, %12 offset:%c15\n\tds_read_u16 %7, %13 offset:%c15\n\tds_read_b64 %8, %14\n\t"
                   "ds_read_b64 %9, %14 offset:%c15\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]),
                     "=&v"(x0), "=&v"(x1)
                   : "v"(vadr[0] + slot), "v"(vadr[1] + slot), "v"(vadr[2] + slot), "v"(vadr[3] + slot), "v"(vsadr + slot), "n"(HALF) : "memory");
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        vs[0][i] = x0[i];
        vs[1][i] = x1[i];
      }
    }
    fetch(j + S);   // (here: the statements above wait for every scalar load as well)
    // ---- online softmax ----
    float p[NR][2][4];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      bool ok[2][4];
      float tmax = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ok[b][i] = MASKED ? n0 + 16 * b + 4 * g + i < lim[t] : true;
          tmax = ok[b][i] ? __builtin_fmaxf(tmax, z[t][b][i]) : tmax;
        }
      tmax = __builtin_fmaf(group4_fmax(tmax), rs[t], BLOCK_REF);   // the reference that this tile asks for
      const bool raise = tmax > m[t] + ATTN_SLACK;
      const float mnew = raise ? tmax : m[t];
      const float alpha = __builtin_amdgcn_exp2f(m[t] - mnew);
      m[t] = mnew;
      l[t] *= alpha;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[t][b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[t][b][i], rs[t], -mnew));
          if (MASKED) p[t][b][i] = ok[b][i] ? p[t][b][i] : 0.f;
          l[t] += p[t][b][i];
        }
      if (__any(raise)) {
#pragma unroll
        for (int c = 0; c < NA; ++c) acc[t][c] *= alpha;
      }
    }
    // ---- PV: O^T[channel][row] += V^T . P^T ----
    float vsc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // the lane's byte as an exponent: the conversion reads no other bits of its scale (D = 64: two keys' bytes to a word)
      const uint32_t w = D == 128 ? vs[e / 4][e % 4] : vs[e / 4][e % 4 / 2];
      vsc[e] = __uint_as_float(__builtin_amdgcn_alignbit(w, w, D == 128 || e % 2 == 0 ? vrot : vrot + 16));
      // what lies behind the last key, and keys whose byte no write makes, are finite: they meet weights of 0 (in the tiles that
      // every row sees whole no weight is masked, and such a byte is its key's alone)
      if (MASKED)
        vsc[e] = n0 + 16 * (e / 4) + 4 * g + e % 4 < L
                     ? __uint_as_float(min(__float_as_uint(vsc[e]) & 0x7f800000u, (uint32_t)FP4_MAX_E << 23)) : 0.f;
    }
    if constexpr (PACK) {
      u32x4 pw[2], pl[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pw[b][i] = __builtin_amdgcn_perm(0, __float_as_uint(p[0][b][i]), pick);
          pl[b][i] = __builtin_amdgcn_perm(0, __float_as_uint(behind_bf16(p[0][b][i])), pick);
        }
      auto pair = [&](auto byte_t) {   // the channels 2 B and 2 B + 1 of the lane's
        constexpr int B = decltype(byte_t)::value;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[4 * b + i], vsc[4 * b + i], B));
          const bf16x8 x = *reinterpret_cast<bf16x8*>(&w);
          acc[0][B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, *reinterpret_cast<bf16x8*>(&pw[b]), acc[0][B], 0, 0, 0);
          acc[0][B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, *reinterpret_cast<bf16x8*>(&pl[b]), acc[0][B], 0, 0, 0);
        }
      };
      pair(std::integral_constant<int, 0>{});
      pair(std::integral_constant<int, 1>{});
      if constexpr (D == 128) {
        pair(std::integral_constant<int, 2>{});
        pair(std::integral_constant<int, 3>{});
      }
    } else {
      bf16x8 pop[NR], plo[NR];   // the MFMA's key 8 g + 4 b + i: key 16 b + 4 g + i
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        u32x4 pw, pl;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = p[t][i / 2][2 * (i % 2)], y = p[t][i / 2][2 * (i % 2) + 1];
          pw[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
          pl[i] = __builtin_amdgcn_perm(__float_as_uint(behind_bf16(y)), __float_as_uint(behind_bf16(x)), 0x07060302u);
        }
        pop[t] = *reinterpret_cast<bf16x8*>(&pw);
        plo[t] = *reinterpret_cast<bf16x8*>(&pl);
      }
      auto pair = [&](auto byte_t) {
        constexpr int B = decltype(byte_t)::value;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[e], vsc[e], B));
        u32x4 even, odd;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          even[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x05040100u);
          odd[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302u);
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          acc[t][2 * B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<bf16x8*>(&even), pop[t], acc[t][2 * B], 0, 0, 0);
          acc[t][2 * B + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<bf16x8*>(&odd), pop[t], acc[t][2 * B + 1], 0, 0, 0);
          acc[t][2 * B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<bf16x8*>(&even), plo[t], acc[t][2 * B], 0, 0, 0);
          acc[t][2 * B + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<bf16x8*>(&odd), plo[t], acc[t][2 * B + 1], 0, 0, 0);
        }
      };
      pair(std::integral_constant<int, 0>{});
      pair(std::integral_constant<int, 1>{});
      if constexpr (D == 128) {
        pair(std::integral_constant<int, 2>{});
        pair(std::integral_constant<int, 3>{});
      }
    }
  };

  // S - 1 tiles in flight. One body for whole tiles and one for those at some row's limit or at the end, whatever their place in
  // the ring: a piece is a few tiles, and the first pass through code costs more than the second (a body to each slot: 1 request
  // of 4096 keys 13.3 us against 12.7, 64 of 8 tokens 64 against 60, 128 of 32768 keys 359 against 361, when weights were one bf16).
  const int full_end = lim_lo > 0 ? lim_lo / TILE : 0;
  const int j_full = full_end > c_begin + ks ? (full_end - c_begin - ks + KS - 1) / KS : 0;
  uint32_t slot = 0, free = (S - 1) * SLOT;
  auto turn = [&] {
    free = slot;
    slot = slot + SLOT == S * SLOT ? 0 : slot + SLOT;
  };
  int j = 0;
#pragma unroll 1
  for (const int end = min(j_full, nt - (S - 1)); j < end; ++j) {
    load(free, j + S - 1);
    wait_vm<(S - 1) * OPS>();   // this wavefront's operations behind the tile's own
    compute(std::false_type{}, slot, j);
    turn();
  }
#pragma unroll 1
  for (; j < nt; ++j) {
    if (j + S - 1 < nt) {
      load(free, j + S - 1);
      wait_vm<(S - 1) * OPS>();
    } else {
      wait_vm<0>();
    }
    compute(std::true_type{}, slot, j);
    turn();
  }

  // ---- the key splits' merge, half of them into the other half at a time, one row tile after the other ----
#pragma unroll
  for (int t = 0; t < NR; ++t) l[t] = group4_sum(l[t]);
  if (KS > 1) {
    // (each wavefront hands over in its own ring, which is done with)
    constexpr int FIELDS = fp4_merge_fields(D, PACK);
    static_assert(FIELDS * WAVE * 4 <= S * SLOT, "merge fields in the ring");
    auto mem = [&](int k) { return reinterpret_cast<float*>(lds + (k - ks) * (a.rt / NR) * S * SLOT) + lane; };
    for (int half = KS, width = KS; width > 1; width = half) {
      half = (width + 1) / 2;
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        if (active && ks >= half && ks < width) {
          float* to = mem(ks);
#pragma unroll
          for (int c = 0; c < NA; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) to[(4 * c + i) * WAVE] = acc[t][c][i];
          to[(4 * NA) * WAVE] = m[t];
          to[(4 * NA + 1) * WAVE] = l[t];
        }
        __syncthreads();
        if (active && ks + half < width) {
          const float* from = mem(ks + half);
          const float mo = from[(4 * NA) * WAVE], M = __builtin_fmaxf(m[t], mo);
          const float w0 = __builtin_amdgcn_exp2f(m[t] - M), w1 = __builtin_amdgcn_exp2f(mo - M);
          l[t] = __builtin_fmaf(w1, from[(4 * NA + 1) * WAVE], l[t] * w0);
#pragma unroll
          for (int c = 0; c < NA; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][c][i] = __builtin_fmaf(w1, from[(4 * c + i) * WAVE], acc[t][c][i] * w0);
          m[t] = M;
        }
        __syncthreads();
      }
    }
  }
  if (ks > 0 || !active) return;
  // ---- the end of a piece: bf16 out of a whole segment, or the fp32 partial of a cut one ----
  const Fp4AttnArgs& f = fresh_fp4();
  const AttnArgs& o = f.a;
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    // x: the lane's consecutive channels from ch on. Not PACK: acc[c][i] is channel (D/4) g + (D/16) i + c. PACK: acc[c][i] is
    // channel (D/4) g + (D/16) i + 2 c, or the one behind it in columns 8 .. 15: the row's two lanes exchange, and take i < 2
    // and i >= 2.
    constexpr int OPL = PACK ? D / 8 : D / 4;
    float x[OPL];
    int ch = (D / 4) * g;
    if constexpr (PACK) {
      const bool hi = n >= 8;
      ch += hi ? D / 8 : 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < NA; ++c) {
          const float give = hi ? acc[t][c][i] : acc[t][c][i + 2], got = ror8(give), mine = hi ? acc[t][c][i + 2] : acc[t][c][i];
          x[VT * i + 2 * c] = hi ? got : mine;
          x[VT * i + 2 * c + 1] = hi ? mine : got;
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < VT; ++c) x[VT * i + c] = acc[t][c][i];
    }
    if (rtok[t] >= qlen) continue;
    const int qt = tok + rtok[t], head = kvh * G + rh[t];
    float lse = __builtin_fmaf(m[t], LN2, __builtin_amdgcn_logf(l[t]) * LN2);
    if (l[t] != l[t]) {   // (a denominator that is no number would not tell the merge that the row was cut)
      lse = NAN;
      l[t] = 1.f;
#pragma unroll
      for (int e = 0; e < OPL; ++e) x[e] = NAN;
    }
    const bool first = g == 0 && (!PACK || n < 8);
    if (nparts == 1) {
      if (first) {
        if (o.max_splits > 1 && qt < o.cut_rows) o.segm_sum[(int64_t)qt * o.seg_st + (int64_t)head * o.seg_sh] = -1.f;
        if (f.lse) f.lse[(int64_t)qt * f.lse_st + head] = lse;
      }
      const float inv = l[t] > 0.f ? 1.f / l[t] : 0.f;
      uint32_t w[OPL / 2];
#pragma unroll
      for (int e = 0; e < OPL / 2; ++e) w[e] = pack_bf16x2_rne(x[2 * e] * inv, x[2 * e + 1] * inv);
      u32x4* op = reinterpret_cast<u32x4*>(o.out + (int64_t)qt * o.o_st + (int64_t)head * o.o_sh + ch);
#pragma unroll
      for (int u = 0; u < OPL / 8; ++u) op[u] = u32x4{w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]};
    } else {
      const int64_t sidx = (int64_t)qt * o.seg_st + (int64_t)head * o.seg_sh + part;
      if (first) {
        o.segm_max[sidx] = m[t];
        o.segm_sum[sidx] = part == nparts - 1 ? last_piece_sum(l[t]) : l[t];
      }
      float* sp = o.segm_out + sidx * D + ch;
#pragma unroll
      for (int u = 0; u < OPL / 4; ++u)
        reinterpret_cast<float4*>(sp)[u] = float4{x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]};
    }
  }
}

template <int D, bool PACK, int NR, int S>
__global__ __launch_bounds__(WAVE * FP4_WAVES) __attribute__((amdgpu_waves_per_eu(1, 2))) void fp4_attn_kernel(Fp4AttnArgs args) {
  touch_args();
  const AttnArgs& a = args.a;
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int rw = a.rt / NR, ksplit = a.ksplit, kspl = wave / rw, rtile = NR * (wave - kspl * rw);
  extern __shared__ __attribute__((aligned(1024))) uint8_t fp4_lds[];
  uint8_t* ring = fp4_lds + wave * S * fp4_slot(D);
  int solo = 0;
  walk_pieces(a, lane, [&](int r, const ReqWork& w, int kvh, int rg, int c0, int c1, int part, int nparts) {
    const int row0 = (rg * a.rt + rtile) * (PACK ? 8 : 16);
    // (a piece for all key splits, or a short one for one of them: one call, the code is long)
    const bool all = ksplit > 1 && c1 - c0 >= a.coop;
    if (all || solo % ksplit == kspl)
      attend_fp4<D, PACK, NR, S>(r, w.tok, w.qlen, w.len, kvh, row0, c0, c1, all ? kspl : 0, all ? ksplit : 1, part, nparts, ring, lane);
    if (!all) ++solo;
  });
}

template <int D>
auto fp4_attn_of(bool pack, bool cut, int nr) -> void (*)(Fp4AttnArgs) {
  if (pack) return cut ? fp4_attn_kernel<D, true, 1, fp4_slots(true, true)> : fp4_attn_kernel<D, true, 1, fp4_slots(true, false)>;
  return nr == 1 ? fp4_attn_kernel<D, false, 1, fp4_slots(false, true)> : fp4_attn_kernel<D, false, 2, fp4_slots(false, true)>;
}

// split_reduce_kernel, with the rows' log-sum-exp
template <int D>
__global__ __launch_bounds__(WAVE * RED_WAVES) void fp4_reduce_kernel(AttnArgs a, float* lse, int64_t lse_st) {
  const int lane = threadIdx.x & (WAVE - 1);
  const int seq = blockIdx.x;
  const int h = blockIdx.y * RED_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int tok = a.cu_q[seq], qlen = a.cu_q[seq + 1] - tok;
  if (h >= a.G * a.hkv || qlen <= 0 || qlen > a.qmax) return;
  const int rows = min(qlen, a.cut_rows - tok);
  for (int t = blockIdx.z; t < rows; t += gridDim.z)
    merge_row<D, true>(a, tok, t, h, lane, lse ? lse + (int64_t)(tok + t) * lse_st + h : nullptr);
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
// What every call on a 4-bit cache checks; 0, or the error after fail().
int check_fp4(const char* nm, int64_t num_blocks, int64_t block_size, int64_t heads, int64_t head_dim, const void* kc,
              int64_t k_sb, int64_t k_sn, int64_t k_sh, const void* vc, int64_t v_sb, int64_t v_sn, int64_t v_sh,
              const void* ks, const void* vs, int64_t s_sb, int64_t s_sh) {
  if (head_dim != 64 && head_dim != 128) return fail("%s: head_dim must be 64 or 128, got %lld", nm, (long long)head_dim);
  if (block_size < 16 || !pow2(block_size) || block_size > (1 << 24))
    return fail("%s: block_size must be a power of two >= 16", nm);
  if (heads <= 0 || heads > 65535 || num_blocks <= 0 || num_blocks > INT32_MAX) return fail("%s: bad sizes", nm);
  if (!kc || !vc || !ks || !vs) return fail("%s: null pointer", nm);
  if (!aligned16(kc) || !aligned16(vc) || (k_sb | k_sn | k_sh | v_sb | v_sn | v_sh) % 16)
    return fail("%s: cache rows must be 16-byte aligned (base pointers and strides)", nm);
  if (!aligned16(ks) || !aligned16(vs) || (s_sb | s_sh) % 16)
    return fail("%s: scales must be 16-byte aligned (base pointers and strides)", nm);
  if (k_sn < 0 || v_sn < 0 || block_size * k_sn > INT32_MAX || block_size * v_sn > INT32_MAX)
    return fail("%s: page too large for 32-bit lane offsets", nm);
  if ((k_sb | v_sb | s_sb) >> 32) return fail("%s: pages 4 GiB apart or more", nm);
  return 0;
}

}  // namespace

extern "C" {

int kvq_quant_fp4_cache(const void* key, int64_t key_st, int64_t key_sh, const void* value, int64_t val_st, int64_t val_sh,
                        uint8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, uint8_t* v_cache, int64_t vc_sb,
                        int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads,
                        int64_t head_dim, uint8_t* k_scale, uint8_t* v_scale, int64_t s_sb, int64_t s_sh,
                        const int64_t* slot_mapping, int64_t num_tokens, void* stream) {
  const char* nm = "quant_fp4_cache";
  if (num_tokens < 0 || num_tokens > INT32_MAX) return fail("%s: bad sizes", nm);
  if (num_tokens == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_fp4(nm, num_blocks, block_size, num_heads, head_dim, k_cache, kc_sb, kc_sn, kc_sh, v_cache, vc_sb,
                               vc_sn, vc_sh, k_scale, v_scale, s_sb, s_sh)) return rc;
  if (!key || !value || !slot_mapping) return fail("%s: null pointer", nm);
  if (!aligned16(key) || !aligned16(value) || (key_st | key_sh | val_st | val_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  QuantFp4Args a;
  a.key = (const uint16_t*)key; a.value = (const uint16_t*)value; a.kc = k_cache; a.vc = v_cache; a.slots = slot_mapping;
  a.s = Fp4Scales{k_scale, v_scale, s_sb, s_sh};
  a.key_st = key_st; a.key_sh = key_sh; a.val_st = val_st; a.val_sh = val_sh;
  a.kc_sb = kc_sb; a.kc_sn = kc_sn; a.kc_sh = kc_sh; a.vc_sb = vc_sb; a.vc_sn = vc_sn; a.vc_sh = vc_sh;
  a.num_slots = num_blocks * block_size;
  a.num_tokens = (int)num_tokens; a.heads = (int)num_heads; a.lbs = log2i(block_size);
  const int64_t rpb = 256 / (head_dim / 8), blocks = (num_tokens * num_heads + rpb - 1) / rpb;
  if (blocks > INT32_MAX) return fail("%s: too many tokens and heads for one call", nm);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (head_dim == 128) hipLaunchKernelGGL(quant_fp4_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(quant_fp4_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  return launched(nm);
}

int kvq_read_fp4_cache(const uint8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, const uint8_t* v_cache,
                       int64_t vc_sb, int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads,
                       int64_t head_dim, const uint8_t* k_scale, const uint8_t* v_scale, int64_t s_sb, int64_t s_sh,
                       const int32_t* starts, const int32_t* cu_seqlens_k, const int32_t* block_table, int64_t bt_stride,
                       int64_t num_seqs, void* k_out, int64_t ko_st, int64_t ko_sh, void* v_out, int64_t vo_st, int64_t vo_sh,
                       int64_t num_rows, void* stream) {
  const char* nm = "read_fp4_cache";
  if (num_rows < 0 || num_seqs < 0 || num_rows > INT32_MAX || num_seqs > INT32_MAX / 4) return fail("%s: bad sizes", nm);
  if (num_rows == 0 || num_seqs == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_fp4(nm, num_blocks, block_size, num_heads, head_dim, k_cache, kc_sb, kc_sn, kc_sh, v_cache, vc_sb,
                               vc_sn, vc_sh, k_scale, v_scale, s_sb, s_sh)) return rc;
  if (!k_out || !v_out || !starts || !cu_seqlens_k || !block_table) return fail("%s: null pointer", nm);
  if (!aligned16(k_out) || !aligned16(v_out) || (ko_st | ko_sh | vo_st | vo_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  ReadFp4Args a;
  a.kc = k_cache; a.vc = v_cache; a.ko = (uint16_t*)k_out; a.vo = (uint16_t*)v_out;
  a.start = starts; a.cu_k = cu_seqlens_k; a.block_table = block_table;
  a.s = Fp4Scales{const_cast<uint8_t*>(k_scale), const_cast<uint8_t*>(v_scale), s_sb, s_sh};
  a.kc_sb = kc_sb; a.kc_sn = kc_sn; a.kc_sh = kc_sh; a.vc_sb = vc_sb; a.vc_sn = vc_sn; a.vc_sh = vc_sh;
  a.ko_st = ko_st; a.ko_sh = ko_sh; a.vo_st = vo_st; a.vo_sh = vo_sh; a.bt_stride = bt_stride;
  a.num_seqs = (int)num_seqs; a.num_rows = (int)num_rows; a.heads = (int)num_heads; a.num_blocks = (int)num_blocks;
  a.lbs = log2i(block_size);
  const int64_t items = block_slots(num_rows, num_seqs, 4) * num_heads;
  if (items > INT32_MAX - 3) return fail("%s: too many rows and heads for one call", nm);
  a.items = (int)items;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool nt = 5 * num_rows * num_heads * head_dim > READ_NT_BYTES;
  void (*kern)(ReadFp4Args) = head_dim == 128 ? (nt ? read_fp4_kernel<128, true> : read_fp4_kernel<128, false>)
                                              : (nt ? read_fp4_kernel<64, true> : read_fp4_kernel<64, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)((items + 3) / 4)), dim3(256), 0, st, a);
  return launched(nm);
}

int kvq_fp4_pages(const uint8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, const uint8_t* v_cache, int64_t vc_sb,
                  int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim,
                  const uint8_t* k_scale, const uint8_t* v_scale, int64_t s_sb, int64_t s_sh, void* k_out, void* v_out,
                  float* scales_out, const int32_t* block_table, int64_t bt_stride, const int32_t* src_req,
                  const int32_t* src_j, int64_t num_pages, void* stream) {
  const char* nm = "fp4_pages";
  if (num_pages < 0 || num_pages > INT32_MAX) return fail("%s: bad sizes", nm);
  if (num_pages == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_fp4(nm, num_blocks, block_size, num_heads, head_dim, k_cache, kc_sb, kc_sn, kc_sh, v_cache, vc_sb,
                               vc_sn, vc_sh, k_scale, v_scale, s_sb, s_sh)) return rc;
  if (!k_out || !v_out || !scales_out || !block_table || !src_req || !src_j) return fail("%s: null pointer", nm);
  if (!aligned16(k_out) || !aligned16(v_out) || !aligned16(scales_out))
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  if (2 * block_size * num_heads * head_dim > INT32_MAX) return fail("%s: page too large for 32-bit lane offsets", nm);
  Fp4PagesArgs a;
  a.kc = k_cache; a.vc = v_cache; a.ko = (uint16_t*)k_out; a.vo = (uint16_t*)v_out;
  a.table = reinterpret_cast<f32x4*>(scales_out); a.block_table = block_table; a.src_req = src_req; a.src_j = src_j;
  a.s = Fp4Scales{const_cast<uint8_t*>(k_scale), const_cast<uint8_t*>(v_scale), s_sb, s_sh};
  a.kc_sb = kc_sb; a.kc_sn = kc_sn; a.kc_sh = kc_sh; a.vc_sb = vc_sb; a.vc_sn = vc_sn; a.vc_sh = vc_sh; a.bt_stride = bt_stride;
  a.heads = (int)num_heads; a.num_blocks = (int)num_blocks; a.bs = (int)block_size;
  // few pages: each page over several workgroups
  const int64_t chunks = (block_size * num_heads * head_dim / 8 + 255) / 256;
  const int64_t slices = std::min<int64_t>(std::min<int64_t>(chunks, 65535), std::max<int64_t>(1, (int64_t)device_cus() * 8 / (2 * num_pages)));
  const dim3 grid((unsigned)num_pages, (unsigned)slices, 2);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (head_dim == 128) hipLaunchKernelGGL(fp4_pages_kernel<128>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(fp4_pages_kernel<64>, grid, dim3(256), 0, st, a);
  return launched(nm);
}

int kvq_fp4_prefill_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k_pages, const void* v_pages,
                              const float* page_scales, int64_t num_pages, int64_t block_size, int64_t num_kv_heads,
                              int64_t head_dim, void* out, int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q,
                              const int32_t* seq_lens, const int32_t* pages_table, int64_t pt_stride, int64_t num_q_heads,
                              const int32_t* tile_req, const int32_t* tile_row, int64_t num_tiles, int64_t rows_per_tile,
                              double softmax_scale, const int32_t* tile_piece, const int32_t* tile_slot, const int32_t* merge,
                              int64_t num_merge, float* part_out, float* part_ml, void* stream) {
  const char* nm = "fp4_prefill_attention";
  if (num_tiles < 0 || num_tiles > INT32_MAX || num_merge < 0 || num_merge > INT32_MAX) return fail("%s: bad sizes", nm);
  if (num_tiles == 0) { g_err.clear(); return KVQ_OK; }
  if (rows_per_tile != PR_ROWS) return fail("%s: work list tiles must be %d rows", nm, PR_ROWS);
  if (!tile_req || !tile_row || (tile_piece && !tile_slot)) return fail("%s: bad work list", nm);
  if (tile_piece && num_merge > 0 && (!merge || !part_out || !part_ml || !aligned16(merge) || !aligned16(part_out) ||
                                      !aligned16(part_ml)))
    return fail("%s: split work list needs 16-byte aligned merge list and partial buffers", nm);
  if (!(softmax_scale >= MIN_SOFTMAX_SCALE && softmax_scale <= MAX_SOFTMAX_SCALE))
    return fail("%s: softmax_scale must be positive and finite, from %g to %g", nm, MIN_SOFTMAX_SCALE, MAX_SOFTMAX_SCALE);
  if (const int rc = check_fp4(nm, num_pages, block_size, num_kv_heads, head_dim, k_pages, 0, 0, 0, v_pages, 0, 0, 0, page_scales,
                               page_scales, 0, 0)) return rc;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads || num_q_heads > 65535)
    return fail("%s: bad head counts Hq=%lld Hkv=%lld", nm, (long long)num_q_heads, (long long)num_kv_heads);
  if (!q || !out || !cu_seqlens_q || !seq_lens || !pages_table) return fail("%s: null pointer", nm);
  if (!aligned16(q) || !aligned16(out) || (q_st | q_sh | o_st | o_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  if (2 * block_size * num_kv_heads * head_dim > INT32_MAX)
    return fail("%s: page too large for 32-bit page / slot offsets", nm);
  PrefillArgs a;
  memset(&a, 0, sizeof(a));
  a.q = (const uint16_t*)q; a.kc = (const uint16_t*)k_pages; a.vc = (const uint16_t*)v_pages; a.out = (uint16_t*)out;
  a.cu_q = cu_seqlens_q; a.seq_lens = seq_lens; a.block_table = pages_table; a.tile_req = tile_req; a.tile_row = tile_row;
  a.tile_piece = tile_piece; a.tile_slot = tile_slot; a.part_out = part_out; a.part_ml = part_ml;
  a.q_st = q_st; a.q_sh = q_sh; a.o_st = o_st; a.o_sh = o_sh; a.bt_stride = pt_stride;
  a.k_sh = a.v_sh = head_dim;
  a.k_sn = a.v_sn = num_kv_heads * head_dim;
  a.k_sb = a.v_sb = block_size * a.k_sn;
  a.krow = a.vrow = (uint32_t)(2 * a.k_sn);
  a.kpage = a.vpage = (uint32_t)(2 * a.k_sb);
  a.contig = 1;
  a.sm_log2 = (float)(softmax_scale * 1.4426950408889634);
  a.G = (int)(num_q_heads / num_kv_heads); a.lbs = log2i(block_size); a.num_blocks = (int)num_pages;
  a.s_table = reinterpret_cast<const f32x4*>(page_scales);
  const dim3 grid((unsigned)num_tiles, (unsigned)num_kv_heads);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  void (*kern)(PrefillArgs) = head_dim == 128
      ? (tile_piece ? fp4_prefill_kernel<128, true> : fp4_prefill_kernel<128, false>)
      : (tile_piece ? fp4_prefill_kernel<64, true> : fp4_prefill_kernel<64, false>);
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a);
  const int rc = launched(nm);
  if (rc != KVQ_OK || !tile_piece || num_merge == 0) return rc;
  const dim3 mgrid((unsigned)num_merge, (unsigned)num_kv_heads, PR_ROWS / PR_MERGE_WAVES);
  const int4* ml = reinterpret_cast<const int4*>(merge);
  if (head_dim == 128) hipLaunchKernelGGL(prefill_merge_kernel<128>, mgrid, dim3(WAVE * PR_MERGE_WAVES), 0, st, a, ml);
  else hipLaunchKernelGGL(prefill_merge_kernel<64>, mgrid, dim3(WAVE * PR_MERGE_WAVES), 0, st, a, ml);
  return launched("fp4_prefill_attention: merge");
}

int kvq_fp4_decode_attention(const void* q, int64_t q_st, int64_t q_sh, const uint8_t* k_cache, int64_t k_sb, int64_t k_sn,
                             int64_t k_sh, const uint8_t* v_cache, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                             int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_dim,
                             const uint8_t* k_scale, const uint8_t* v_scale, int64_t s_sb, int64_t s_sh, void* out,
                             int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                             const int32_t* block_table, int64_t bt_stride, int64_t num_seqs, int64_t num_q_heads,
                             double softmax_scale, float* segm_out, float* segm_max, float* segm_sum, int64_t seg_st,
                             int64_t seg_sh, int64_t num_splits, int64_t segm_rows, float* lse, int64_t lse_st,
                             int64_t target_waves, int64_t max_query_len, int64_t qmax, void* stream) {
  const char* nm = "fp4_decode_attention";
  if (num_splits < 1 || num_splits > MAX_SPLITS) return fail("%s: at most %d split-KV segments", nm, MAX_SPLITS);
  if (num_seqs < 0 || num_seqs > INT32_MAX / 4 || max_query_len < 0 || qmax < 1 || target_waves < 0 || segm_rows < 0)
    return fail("%s: bad sizes", nm);
  if (num_seqs == 0) { g_err.clear(); return KVQ_OK; }
  if (!(softmax_scale >= MIN_SOFTMAX_SCALE && softmax_scale <= MAX_SOFTMAX_SCALE))
    return fail("%s: softmax_scale must be positive and finite, from %g to %g", nm, MIN_SOFTMAX_SCALE, MAX_SOFTMAX_SCALE);
  if (const int rc = check_fp4(nm, num_blocks, block_size, num_kv_heads, head_dim, k_cache, k_sb, k_sn, k_sh, v_cache, v_sb,
                               v_sn, v_sh, k_scale, v_scale, s_sb, s_sh)) return rc;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads || num_q_heads > 65535)
    return fail("%s: bad head counts Hq=%lld Hkv=%lld", nm, (long long)num_q_heads, (long long)num_kv_heads);
  if (!q || !out || !cu_seqlens_q || !seq_lens || !block_table) return fail("%s: null pointer", nm);
  if (!aligned16(q) || !aligned16(out) || (q_st | q_sh | o_st | o_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  if (num_splits > 1 && segm_rows > 0 && (!segm_out || !segm_max || !segm_sum || !aligned16(segm_out)))
    return fail("%s: split buffers missing or not 16-byte aligned", nm);
  if (k_sb != v_sb || k_sn != v_sn) return fail("%s: K and V caches must have the same page and slot strides", nm);
  const int G = (int)(num_q_heads / num_kv_heads);
  const int64_t maxq = std::min<int64_t>(std::max<int64_t>(max_query_len, 1), qmax), rows = (int64_t)G * maxq;
  if (rows > INT32_MAX / 4) return fail("%s: grid too large", nm);
  // the row tile: 8 rows where that holds all of a request's rows; else 16
  const bool pack = rows <= 8;
  const Tuning tune = read_tuning();
  const bool cut = num_splits > 1 && segm_rows > 0, few = num_seqs * num_kv_heads <= WIDE_SPLIT_PAIRS;
  // More rows than a tile holds: a wavefront to each tile of rows, or one to two of them, which loads and converts a key once for
  // both but keeps half as many wavefronts busy. Few pairs of a request and a KV head, cut, take the first (16 requests of 8 tokens,
  // 28 heads on 4: 23.6 us against 27.0), others the second (64 such requests: 54.7 against 62.4; 64 of 4096 keys, whole: 69
  // against 81).
  const int rt = rows <= 16 ? 1 : rows <= 32 ? 2 : MAX_ROW_TILES, nr = rt == 1 || (cut && few) ? 1 : 2, rw = rt / nr;
  const int most = cut && rt == 1 ? MAX_ROW_TILES : FP4_WAVES;
  const int ks_max = tune.ksplit ? std::max(1, std::min(FP4_WAVES, atoi(tune.ksplit)))
                     : !cut || few ? most : DEFAULT_KSPLIT;
  const int ks = std::max(1, std::min(ks_max, most / rw)), waves = rw * ks;
  Fp4AttnArgs b;
  b.s = Fp4Scales{const_cast<uint8_t*>(k_scale), const_cast<uint8_t*>(v_scale), s_sb, s_sh};
  b.lse = lse; b.lse_st = lse_st;
  b.apart = !(v_cache == k_cache + head_dim / 2 && k_sh == v_sh);
  AttnArgs& a = b.a;
  a.q = (const uint16_t*)q; a.kc = (const int8_t*)k_cache; a.vc = (const int8_t*)v_cache; a.out = (uint16_t*)out;
  a.segm_out = segm_out; a.segm_max = segm_max; a.segm_sum = segm_sum;
  a.cu_q = cu_seqlens_q; a.seq_lens = seq_lens; a.block_table = block_table;
  a.ks = a.vs = nullptr; a.ks_pc = a.vs_pc = 0;
  a.q_st = q_st; a.q_sh = q_sh; a.o_st = o_st; a.o_sh = o_sh;
  a.k_sb = k_sb; a.k_sn = k_sn; a.k_sh = k_sh; a.v_sb = v_sb; a.v_sn = v_sn; a.v_sh = v_sh;
  a.seg_st = seg_st; a.seg_sh = seg_sh; a.bt_stride = bt_stride;
  a.sm_log2 = (float)(softmax_scale * 1.4426950408889634);
  a.num_blocks = (int)num_blocks; a.lbs = log2i(block_size);
  a.G = pack ? 2 * G : G;   // the plan's rows: planes of rows where two share an MFMA
  a.g_inv = G > 1 && (G * std::min<int64_t>(qmax, INT32_MAX) + 64) < (1ll << 32) / G ? (unsigned)(((1ll << 32) + G - 1) / G) : 0u;
  a.qmax = (int)std::min<int64_t>(qmax, INT32_MAX);
  a.num_seqs = (int)num_seqs; a.hkv = (int)num_kv_heads;
  a.max_splits = (int)num_splits;
  a.cut_rows = num_splits > 1 ? (int)std::min<int64_t>(segm_rows, INT32_MAX) : 0;
  a.rt = rt; a.ksplit = ks; a.waves = waves;
  a.min_tiles = MIN_SPLIT_TILES;
  a.coop = coop_tiles(num_splits > 1, ks);
  a.xcd_order = tune.xcd_order ? atoi(tune.xcd_order) : 1;
  a.plan_fast_max = tune.plan_fast_max ? (int)std::max(1ll, std::min(PLAN_FAST_MAX, atoll(tune.plan_fast_max)))
                                       : (int)PLAN_FAST_MAX;
  a.seg_cost = seg_cost_units(tune, 0);
  const int slots = fp4_slots(pack, cut);
  const size_t lds = (size_t)waves * slots * fp4_slot((int)head_dim);
  void (*kern)(Fp4AttnArgs) = head_dim == 128 ? fp4_attn_of<128>(pack, cut, nr) : fp4_attn_of<64>(pack, cut, nr);
  const int64_t tw = target_waves > 0 ? target_waves
                     : cut            ? (int64_t)device_cus() * resident_waves((const void*)kern, WAVE * waves, lds)
                                      : (int64_t)device_cus() * waves;
  a.workers = (int)std::max<int64_t>(1, std::min<int64_t>(tw / waves, INT32_MAX));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(kern, dim3((unsigned)a.workers), dim3(WAVE * waves), lds, st, b);
  const int rc = launched(nm);
  if (rc != KVQ_OK || num_splits == 1 || a.cut_rows == 0) return rc;
  a.G = G;
  const dim3 rgrid((unsigned)num_seqs, (unsigned)((num_q_heads + RED_WAVES - 1) / RED_WAVES),
                   (unsigned)std::min<int64_t>(maxq, MERGE_Z));
  if (head_dim == 128) hipLaunchKernelGGL(fp4_reduce_kernel<128>, rgrid, dim3(WAVE * RED_WAVES), 0, st, a, lse, lse_st);
  else hipLaunchKernelGGL(fp4_reduce_kernel<64>, rgrid, dim3(WAVE * RED_WAVES), 0, st, a, lse, lse_st);
  return launched("fp4_decode_attention: merge");
}

}  // extern "C"
