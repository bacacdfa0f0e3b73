// The block-scaled INT8 cache: no calibrated scales, one fp32 scale for each block of 16 .. 128 consecutive positions
// of a page and kv head, K and V apart, made as the cache is written. Part of kvq_int8.hip (included at its end: it
// shares the helpers above it).
//
//   quant_block_kernel   quantize a step's new K/V into their blocks, raising scales (and requantizing) where needed
//   read_block_kernel    ranges of the requests' keys back to bf16 rows
//   block_attn_kernel    attention of short queries: scores on int8 MFMA, q in two int8 planes; bf16 MFMA for the values
//   block_verify_kernel, block_prefill_kernel   attention of many query rows (block_rows.h)
//
// A cached value is code * scale; attention is that of those values and the bf16 q. The codes are exact throughout. Rounded:
//   q        to a 15-bit integer of its row's largest where K stays int8 (block_attn_kernel, block_rows.h): 2^-15 of the largest
//            a channel, where K's codes are off by 2^-8 of theirs; bf16 as given where K's codes are copied as bf16
//   weights  to a sum of two bf16 (block_attn_kernel: 2^-14 of each, error against 64 bits 1.66e-3, the bf16 output's) or to
//            one (many rows: 2^-8, 2.0 to 2.3e-3; a second MFMA for every product there). Each weight keeps its own exponent:
//            as integers of a tile's scale the keys beside two of 95% of a row's attention and no V were 1.3 to 4.7% off.

#include "block_rows.h"

namespace {

constexpr int BLK_MIN = 16, BLK_MAX = 128;   // positions per scale
constexpr double MIN_SOFTMAX_SCALE = 1e-16, MAX_SOFTMAX_SCALE = 1e16;

// The request that holds slot u of a line on which request r starts at (cu[r] >> lg) + 2 r: as long as cu[r] counts
// rows of consecutive positions, r's rows touch at most (rows >> lg) + 2 aligned blocks of 2^lg positions, so its
// blocks fit before the next request's start wherever its first position lies in a block. A launch sizes its grid
// from the row count alone. 64-way search, the lanes a request each at the end, whose cu[r], cu[r + 1] and of[r] come
// with the same round trip to memory; uniform across the wavefront.
struct SlotRequest {
  int r, cu0, cu1, of;
};
__device__ __forceinline__ SlotRequest request_of_slot(const int* __restrict__ cu, const int* __restrict__ of, int num_seqs,
                                                       int lg, int u, int lane) {
  int lo = 0, n = num_seqs;
  while (n > WAVE) {
    const int step = (n + WAVE - 1) / WAVE, r = lo + lane * step;
    const bool in = lane * step < n && (cu[r] >> lg) + 2 * r <= u;
    // (the first probe always holds: request lo starts at or before u)
    lo += max(__builtin_popcountll(__ballot(in)) - 1, 0) * step;
    n = min(step, num_seqs - lo);
  }
  const int r = lo + min(lane, n - 1);
  const int c0 = cu[r], c1 = cu[r + 1], o = of[r];
  const int k = max(__builtin_popcountll(__ballot(lane < n && (c0 >> lg) + 2 * r <= u)) - 1, 0);
  return {__builtin_amdgcn_readfirstlane(lo) + k, __builtin_amdgcn_readlane(c0, k), __builtin_amdgcn_readlane(c1, k),
          __builtin_amdgcn_readlane(o, k)};
}
inline int64_t block_slots(int64_t rows, int64_t num_seqs, int lg) { return (rows >> lg) + 2 * num_seqs; }

__device__ __forceinline__ int page_at(const int* __restrict__ bt, int64_t bt_stride, int r, int page) {
  return __builtin_amdgcn_readfirstlane(bt[(int64_t)r * bt_stride + page]);
}

// ------------------------------------------------------------------------------------------------
// Quantize a step's new K / V rows into their blocks. Request r's new tokens are its last q_r positions; one item is
// one (request, block, head), whose W = block / 16 wavefronts take 16 positions each, K and V. With x the block's new
// values and s_old its scale if it holds earlier positions of the request (else 0):
//   s = max(s_old, fl(max |x| / 127), 1e-8);  new slots: sat127(rint(fl(x / s)));  old: rint(fl(code * fl(s_old / s)))
// The items of a call touch disjoint blocks, so nothing is shared between wavefronts of different items. Bound by memory for
// many tokens: 16,384 of 4 heads x 128 move 50 MB in 13.2 us (3.8 TB/s, graph); by its three dependent round trips for few:
// 32 requests' one token each 4.4 us. A second kernel for the scales would read the rows twice.
// ------------------------------------------------------------------------------------------------
struct QuantBlockArgs {
  const uint16_t* key;
  const uint16_t* value;
  int8_t* kc;
  int8_t* vc;
  float* ks;
  float* vs;
  const int* cu_q;
  const int* seq_lens;
  const int* block_table;
  int64_t key_st, key_sh, val_st, val_sh, kc_sb, kc_sn, kc_sh, vc_sb, vc_sn, vc_sh, s_sb, s_sh, s_sg, bt_stride;
  int num_seqs, num_tokens, heads, num_blocks, lbs, lg, items;
};

// largest finite |x| of 8 bf16
__device__ __forceinline__ float absmax8(u32x4 w) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = __builtin_fabsf(bf16_lo(w[j])), b = __builtin_fabsf(bf16_hi(w[j]));
    m = __builtin_fmaxf(m, a < INFINITY ? a : 0.f);
    m = __builtin_fmaxf(m, b < INFINITY ? b : 0.f);
  }
  return m;
}
__device__ __forceinline__ u32x2 codes8(u32x4 w, float s, float y) {
  float t[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t[2 * j] = code_magic(bf16_lo(w[j]), s, y);
    t[2 * j + 1] = code_magic(bf16_hi(w[j]), s, y);
  }
  return u32x2{pack_magic4(t[0], t[1], t[2], t[3]), pack_magic4(t[4], t[5], t[6], t[7])};
}
// 8 codes at another scale: rint(fl(code * ratio)), ratio <= 1
__device__ __forceinline__ u32x2 rescaled8(u32x2 c, float ratio) {
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = (float)(int8_t)(c[e / 4] >> (8 * (e % 4))) * ratio + QC_MAGIC;
  return u32x2{pack_magic4(t[0], t[1], t[2], t[3]), pack_magic4(t[4], t[5], t[6], t[7])};
}

template <int D, int W>
__global__ __launch_bounds__(WAVE * (W < 4 ? 4 : W)) void quant_block_kernel(QuantBlockArgs a) {
  constexpr int LPR = D / 8;              // lanes per row
  constexpr int RPL = WAVE / LPR;         // rows per load
  constexpr int N = 16 / RPL;             // loads per matrix and wavefront
  constexpr int WPB = W < 4 ? 4 : W;      // wavefronts per workgroup
  __shared__ float top[WPB][2];
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int item = blockIdx.x * (WPB / W) + wave / W, part = wave % W;
  // three dependent round trips to memory, no more: the request; its rows and the page id; the block as it is
  bool live = item < a.items;
  int h = 0, b0 = 0, first = 0, last = 0, page = 0, off = 0;
  int64_t tok0 = 0;
  const int row = lane / LPR, d0 = 8 * (lane % LPR);
  u32x4 kin[N], vin[N];
  u32x2 kold[N], vold[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    kin[j] = vin[j] = u32x4{0u, 0u, 0u, 0u};
    kold[j] = vold[j] = u32x2{0u, 0u};
  }
  if (live) {
    const int u = item / a.heads;
    h = item - u * a.heads;
    const SlotRequest q = request_of_slot(a.cu_q, a.seq_lens, a.num_seqs, a.lg, u, lane);
    const int p0 = q.of - (q.cu1 - q.cu0);                                 // first new position (negative ones: no slot)
    b0 = ((max(p0, 0) >> a.lg) + u - ((q.cu0 >> a.lg) + 2 * q.r)) << a.lg; // the item's block of the request's positions
    first = max(max(p0, 0), b0);                                           // its new positions: [first, last)
    last = min(p0 + min(q.cu1, a.num_tokens) - q.cu0, b0 + (1 << a.lg));
    tok0 = (int64_t)q.cu0 - p0;                                            // token of position p: tok0 + p
    live = first < last;
    if (live) {
      const int id = a.block_table[(int64_t)q.r * a.bt_stride + (b0 >> a.lbs)];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int p = b0 + 16 * part + row + RPL * j;
        if (p >= first && p < last) {
          kin[j] = *reinterpret_cast<const u32x4*>(a.key + (tok0 + p) * a.key_st + (int64_t)h * a.key_sh + d0);
          vin[j] = *reinterpret_cast<const u32x4*>(a.value + (tok0 + p) * a.val_st + (int64_t)h * a.val_sh + d0);
        }
      }
      page = __builtin_amdgcn_readfirstlane(id);
      live = page >= 0 && page < a.num_blocks;                             // a bad id: nothing is written
      page = live ? page : 0;
    }
    off = b0 & ((1 << a.lbs) - 1);                                         // the block's first slot of the page
  }
  int8_t* kc = a.kc + (int64_t)page * a.kc_sb + (int64_t)(off + 16 * part) * a.kc_sn + (int64_t)h * a.kc_sh + d0;
  int8_t* vc = a.vc + (int64_t)page * a.vc_sb + (int64_t)(off + 16 * part) * a.vc_sn + (int64_t)h * a.vc_sh + d0;
  const bool begun = live && first > b0;                                   // earlier positions of the request share the block
  float km = 0.f, vm = 0.f, ks_old = 0.f, vs_old = 0.f;
  float* ksp = a.ks + (int64_t)page * a.s_sb + (int64_t)h * a.s_sh + (int64_t)(off >> a.lg) * a.s_sg;
  float* vsp = a.vs + (int64_t)page * a.s_sb + (int64_t)h * a.s_sh + (int64_t)(off >> a.lg) * a.s_sg;
  if (begun) {
    ks_old = *ksp;
    vs_old = *vsp;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = row + RPL * j;
      if (b0 + 16 * part + i < first) {
        kold[j] = *reinterpret_cast<const u32x2*>(kc + (int64_t)i * a.kc_sn);
        vold[j] = *reinterpret_cast<const u32x2*>(vc + (int64_t)i * a.vc_sn);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    km = __builtin_fmaxf(km, absmax8(kin[j]));
    vm = __builtin_fmaxf(vm, absmax8(vin[j]));
  }
  km = wave_max(km);
  vm = wave_max(vm);
  if constexpr (W > 1) {   // the block's wavefronts agree on the maxima
    if (lane == 0) {
      top[wave][0] = km;
      top[wave][1] = vm;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; ++k) {
      km = __builtin_fmaxf(km, top[wave - part + k][0]);
      vm = __builtin_fmaxf(vm, top[wave - part + k][1]);
    }
  }
  if (!live) return;
  const float ks = __builtin_fmaxf(__builtin_fmaxf(km / 127.f, 1e-8f), ks_old);
  const float vs = __builtin_fmaxf(__builtin_fmaxf(vm / 127.f, 1e-8f), vs_old);
  if (lane == 0 && part == 0) {
    *ksp = ks;
    *vsp = vs;
  }
  const float ky = 1.f / ks, vy = 1.f / vs, kr = ks_old / ks, vr = vs_old / vs;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = row + RPL * j, p = b0 + 16 * part + i;
    u32x2* kp = reinterpret_cast<u32x2*>(kc + (int64_t)i * a.kc_sn);
    u32x2* vp = reinterpret_cast<u32x2*>(vc + (int64_t)i * a.vc_sn);
    if (p >= first && p < last) {
      *kp = codes8(kin[j], ks, ky);
      *vp = codes8(vin[j], vs, vy);
    } else if (begun && p < first) {
      if (ks > ks_old) *kp = rescaled8(kold[j], kr);
      if (vs > vs_old) *vp = rescaled8(vold[j], vr);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Read ranges of keys back: request r's positions start[r] .. are rows cu_k[r] .. cu_k[r + 1] - 1 of k_out / v_out,
// bf16_rne(code * scale). One wavefront takes one aligned run of 16 positions (one page, one scale) of one head. Bound by
// memory, two bytes written for each read: 16,384 keys of 4 heads x 128 9.9 us, 131,072 148 us (5.4 TB/s); 1,000 3.5 us (graph).
// ------------------------------------------------------------------------------------------------
struct ReadBlockArgs {
  const int8_t* kc;
  const int8_t* vc;
  uint16_t* ko;
  uint16_t* vo;
  const int* start;
  const int* cu_k;
  const int* block_table;
  BlockScales s;
  int64_t kc_sb, kc_sn, kc_sh, vc_sb, vc_sn, vc_sh, ko_st, ko_sh, vo_st, vo_sh, bt_stride;
  int num_seqs, num_rows, heads, num_blocks, lbs, items;
};

// NT: streaming loads and stores, for calls that move more than the last-level cache holds: 805 MB 159.5 -> 148.6 us (5.4
// TB/s), 767 MB 139.9 -> 131.3; below, what the rows' reader finds in the cache is worth more (100 MB 9.9 us and 12.1).
constexpr int64_t READ_NT_BYTES = 256ll << 20;
template <int D, bool NT>
__global__ __launch_bounds__(256) void read_block_kernel(ReadBlockArgs a) {
  constexpr int LPR = D / 8, RPL = WAVE / LPR, N = 16 / RPL;
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
  const int64_t si = (int64_t)page * a.s.sb + (int64_t)h * a.s.sh + (int64_t)(off >> a.s.lg) * a.s.sg;
  const float ks = a.s.ks[si], vs = a.s.vs[si];
  const int row = lane / LPR, d0 = 8 * (lane % LPR);
  const int8_t* kc = a.kc + (int64_t)page * a.kc_sb + (int64_t)off * a.kc_sn + (int64_t)h * a.kc_sh + d0;
  const int8_t* vc = a.vc + (int64_t)page * a.vc_sb + (int64_t)off * a.vc_sn + (int64_t)h * a.vc_sh + d0;
  float ksc[8], vsc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    ksc[e] = ks;
    vsc[e] = vs;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = row + RPL * j, p = b0 + i;
    if (p < first || p >= last) continue;
    const int64_t t = row0 + p - start;
    const u32x2* kp = reinterpret_cast<const u32x2*>(kc + (int64_t)i * a.kc_sn);
    const u32x2* vp = reinterpret_cast<const u32x2*>(vc + (int64_t)i * a.vc_sn);
    u32x4* ko = reinterpret_cast<u32x4*>(a.ko + t * a.ko_st + (int64_t)h * a.ko_sh + d0);
    u32x4* vo = reinterpret_cast<u32x4*>(a.vo + t * a.vo_st + (int64_t)h * a.vo_sh + d0);
    if constexpr (NT) {
      const u32x2 k = __builtin_nontemporal_load(kp), v = __builtin_nontemporal_load(vp);
      __builtin_nontemporal_store(dq8x(k.x, k.y, ksc), ko);
      __builtin_nontemporal_store(dq8x(v.x, v.y, vsc), vo);
    } else {
      const u32x2 k = *kp, v = *vp;
      *ko = dq8x(k.x, k.y, ksc);
      *vo = dq8x(v.x, v.y, vsc);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Attention of short queries: attn_kernel's plan, pieces and tiles (int8 MFMA on the K codes as they lie in the cache),
// with operands that keep what an int8 code would lose. Per (request, kv head) and 32-key tile, log2 domain:
//   S    = q16 . k_code            q16 = rint(q / sq), |q16| <= 16256 = 127 * 128: two int8 planes q16 = 128 hi + lo
//   e    = S sq scale k_scale      m: the row's largest e plus BLOCK_REF, raised where it lags by more than 8
//   P    = 2^(e - m + log2(v_scale))               the V scale rides in the exponent;  l += P / v_scale
//   O   += V^T . (Phi + Plo)       v_mfma_f32_16x16x32_bf16: V's codes as bf16 (exact), Phi = P truncated to bf16, Plo the rest
// so the scales cost one multiplication (K) and one addition (V) per 16-key half tile, not one per element, and O stays in
// the accumulators. A half tile lies in one block (blocks are 16 positions or more). A V code costs its lane one conversion
// and half a pack, as much as an integer product's transposing of V and adding of its sums to O.
// PACK: at most 8 (token, q head) rows per kv head: the hi parts (of q, of P) are the MFMA's columns 0 .. 7, the lo parts
// columns 8 .. 15, so both cost one MFMA, as one part of 16 rows does; lanes n and n + 8 hold the same row and exchange
// their half of S by a 16-lane rotation, and their halves of O at the end. Otherwise 16 rows and two MFMAs per product.
// Bound by memory for long contexts: 128 requests of 32,768 keys (28 / 4 heads x 128) 4.3 GB in 636 to 662 us, 6.5 to 6.77
// TB/s. 96 of 1 to 32,768 keys 101 us with the merge, 534 MB: fixed costs per piece. One of 4,096 13 us: the launches and one
// wave of pieces.
// ------------------------------------------------------------------------------------------------
struct BlockAttnArgs {
  AttnArgs a;   // (first: fresh_args)
  BlockScales s;
};
static_assert(offsetof(BlockAttnArgs, a) == 0 && sizeof(AttnArgs) % 8 == 0, "AttnArgs lead the kernel arguments");
__device__ __forceinline__ const BlockScales& fresh_scales() {
  auto* p = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const BlockScales*)(const void*)(p + offsetof(BlockAttnArgs, s));
}

__device__ __forceinline__ int ror8(int x) { return __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true); }
__device__ __forceinline__ float ror8(float x) { return __int_as_float(ror8(__float_as_int(x))); }

// the upper halves of two fp32: a pair of bf16 (exact where they hold 8 significant bits, else truncated)
__device__ __forceinline__ uint32_t bf16x2_upper(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

template <int D, int PF, bool PACK>
__device__ __forceinline__ void attend_blocks(int seq, int tok, int qlen, int seqlen, int kvh, int row0, int c_begin,
                                              int c_end, int ks, int KS, int rtile, int part, int nparts, float* lds,
                                              int lane) {
  const AttnArgs& a = fresh_args();
  const BlockScales& bs_ = fresh_scales();
  constexpr int RT = PACK ? 8 : 16;        // rows of this wavefront's tile
  constexpr int NP = PACK ? 1 : 2;         // planes in separate MFMAs
  constexpr int KPL = D / 4, KSTEPS = D / 64, VT = D / 16, VW = D / 64, OPL = D / 4;
  const int G = PACK ? a.G >> 1 : a.G;     // (PACK: the plan counts plane rows, two a row)
  const bool active = row0 < qlen * G;
  const int num_blocks = a.num_blocks, lbs = a.lbs, lg = bs_.lg;
  const int64_t k_sb = a.k_sb, k_sn = a.k_sn, v_sb = a.v_sb, v_sn = a.v_sn, s_sb = bs_.sb, s_sg = bs_.sg;
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

  const int R = row0 + (n & (RT - 1)), rtok = div_g(R), rh = R - rtok * G;
  const int lim_lo = L - qlen + 1 + __builtin_amdgcn_readfirstlane(div_g(row0));
  const int8_t* kbase = a.kc + (int64_t)kvh * a.k_sh;
  const int8_t* vbase = a.vc + (int64_t)kvh * a.v_sh;
  const int koff = n * (int)k_sn + g * KPL;
  const int voff = 4 * g * (int)v_sn + n * VT;
  const int vsn = (int)v_sn;
  // a tile's four scales, one load: lane l takes that of half l / 2 % 2, K (l even) or V
  const float* sbase = ((lane & 1) ? bs_.vs : bs_.ks) + (int64_t)kvh * bs_.sh;

  auto page_of = [&](int key) -> int {
    const int idx = __builtin_amdgcn_readfirstlane(key >> lbs);
    const int p = __builtin_amdgcn_readfirstlane(((const __attribute__((address_space(4))) int*)bt)[idx]);
    return (p >= 0 && p < num_blocks) ? p : 0;
  };
  struct Tile {
    KVTile<D> kv;
    float sc;
  };
  auto load = [&](Tile& r, int c) {
    const int n0 = c * TILE, n1 = n0 + 16;
    const int p0 = page_of(n0);
    const int p1 = n1 < L ? page_of(n1) : p0;
    const int o0 = n0 & (bs - 1), o1 = n1 < L ? (n1 & (bs - 1)) : o0;
    const int8_t* kb0 = kbase + (int64_t)p0 * k_sb + (int64_t)o0 * k_sn;
    const int8_t* kb1 = kbase + (int64_t)p1 * k_sb + (int64_t)o1 * k_sn;
    const int8_t* vb0 = vbase + (int64_t)p0 * v_sb + (int64_t)o0 * v_sn;
    const int8_t* vb1 = vbase + (int64_t)p1 * v_sb + (int64_t)o1 * v_sn;
    const int64_t s0 = (int64_t)p0 * s_sb + (int64_t)(o0 >> lg) * s_sg, s1 = (int64_t)p1 * s_sb + (int64_t)(o1 >> lg) * s_sg;
    r.sc = sbase[(lane & 2) ? s1 : s0];
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      r.kv.k[0][s] = ldk(reinterpret_cast<const i32x4*>(kb0 + koff + 16 * s));
      r.kv.k[1][s] = ldk(reinterpret_cast<const i32x4*>(kb1 + koff + 16 * s));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VW == 2) {
        const u32x2 w0 = ldv(reinterpret_cast<const u32x2*>(vb0 + voff + i * vsn));
        const u32x2 w1 = ldv(reinterpret_cast<const u32x2*>(vb1 + voff + i * vsn));
        r.kv.v[i][0] = w0.x; r.kv.v[i][1] = w0.y;
        r.kv.v[4 + i][0] = w1.x; r.kv.v[4 + i][1] = w1.y;
      } else {
        r.kv.v[i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(vb0 + voff + i * vsn));
        r.kv.v[4 + i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(vb1 + voff + i * vsn));
      }
    }
  };

  Tile ring[PF];
  // the q row is requested before the first tiles, and made two planes while they are in flight
  const bool qrow = rtok < qlen;
  u32x4 qraw[KPL / 8];
#pragma unroll
  for (int u = 0; u < KPL / 8; ++u) qraw[u] = u32x4{0u, 0u, 0u, 0u};
  if (qrow) {
    const u32x4* qp = reinterpret_cast<const u32x4*>(a.q + (int64_t)(tok + rtok) * a.q_st +
                                                     (int64_t)(kvh * G + rh) * a.q_sh + g * KPL);
#pragma unroll
    for (int u = 0; u < KPL / 8; ++u) qraw[u] = qp[u];
  }
  if (nt > 0) {
#pragma unroll
    for (int j = 0; j < PF - 1; ++j) load(ring[j], tile(min(j, nt - 1)));
  }
  i32x4 qop[NP][KSTEPS];
  float rs;
  {
    float x[KPL], amax = 0.f;
#pragma unroll
    for (int u = 0; u < KPL / 8; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[8 * u + 2 * j] = bf16_lo(qraw[u][j]);
        x[8 * u + 2 * j + 1] = bf16_hi(qraw[u][j]);
      }
#pragma unroll
    for (int e = 0; e < KPL; ++e) amax = __builtin_fmaxf(amax, __builtin_fabsf(x[e]));
    float odd = 0.f;   // 0, or NaN where the row holds a NaN or an infinity: then its output does too
#pragma unroll
    for (int e = 0; e < KPL; ++e) odd = __builtin_fmaf(x[e], 0.f, odd);
    amax = __builtin_fmaxf(group4_fmax(amax), 1e-30f);
    const float inv = Q16_MAX / amax;
    rs = amax / Q16_MAX * a.sm_log2 + group4_sum(odd);
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int e = 16 * s + 4 * w;
        int hi, lo;
        q_planes4(x[e], x[e + 1], x[e + 2], x[e + 3], inv, hi, lo);
        if constexpr (PACK) {
          qop[0][s][w] = n < 8 ? hi : lo;
        } else {
          qop[0][s][w] = hi;
          qop[NP - 1][s][w] = lo;
        }
      }
  }
  const int lim = rtok < qlen ? L - qlen + 1 + rtok : L;
  const int sh = n < 8 ? 7 : 0;            // PACK: this lane's plane of S
  const uint32_t drop = PACK && n < 8 ? 0u : 0xffff0000u;   // its part of P: what is left without these bits

  float m = -1e30f, l = 0.f;
  f32x4 acc[VT];
#pragma unroll
  for (int t = 0; t < VT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](auto masked_t, const Tile& tl, int c) {
    constexpr bool MASKED = decltype(masked_t)::value;
    const KVTile<D>& r = tl.kv;
    const int n0 = c * TILE;
    // ---- QK: S^T[key][row] of the tile's two 16-key halves ----
    int sc[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      i32x4 z[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        z[p] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) z[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(r.k[b][s], qop[p][s], z[p], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (PACK) {
          const int own = z[0][i] << sh;
          sc[b][i] = own + ror8(own);
        } else {
          sc[b][i] = (z[0][i] << 7) + z[NP - 1][i];
        }
      }
    }
    // ---- the halves' scales ----
    const float vfl = __builtin_fmaxf(tl.sc, MIN_V_SCALE);
    const float lg2 = __builtin_amdgcn_logf(vfl), rcp = __builtin_amdgcn_rcpf(vfl);
    auto of_lane = [](float x, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)); };
    const float f[2] = {rs * of_lane(tl.sc, 0), rs * of_lane(tl.sc, 2)};
    const float lv[2] = {of_lane(lg2, 1), of_lane(lg2, 3)}, iv[2] = {of_lane(rcp, 1), of_lane(rcp, 3)};
    // ---- online softmax; key of accumulator (b, i) = n0 + 16 b + 4 g + i ----
    bool ok[2][4];
    float tmax = -INFINITY;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      int mx = INT32_MIN;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ok[b][i] = MASKED ? n0 + 16 * b + 4 * g + i < lim : true;
        mx = ok[b][i] ? max(mx, sc[b][i]) : mx;
      }
      // (a dot product never reaches INT32_MIN: it marks a half without a visible key)
      const float tb = (float)mx * f[b];
      tmax = (MASKED && mx == INT32_MIN) ? tmax : __builtin_fmaxf(tmax, tb);
    }
    tmax = group4_fmax(tmax) + BLOCK_REF;    // the reference that this tile asks for
    const bool raise = tmax > m + ATTN_SLACK;
    const float mnew = raise ? tmax : m;
    const float alpha = __builtin_amdgcn_exp2f(m - mnew);
    m = mnew;
    float p[2][4], sum[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float e0 = lv[b] - mnew;
      sum[b] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf((float)sc[b][i], f[b], e0));
        if (MASKED) p[b][i] = ok[b][i] ? p[b][i] : 0.f;
        sum[b] += p[b][i];
      }
    }
    l = __builtin_fmaf(sum[0], iv[0], __builtin_fmaf(sum[1], iv[1], l * alpha));
    if (__any(raise)) {
#pragma unroll
      for (int t = 0; t < VT; ++t) acc[t] *= alpha;
    }
    // ---- PV: O^T[channel][row] += V^T . (Phi + Plo)^T, the MFMA's key 8 g + 4 b + i: key 16 b + 4 g + i ----
    bf16x8 pop[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      float x[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[b][i] = NP == 2 && k == 0 ? p[b][i] : p[b][i] - __uint_as_float(__float_as_uint(p[b][i]) & drop);
      u32x4 w = {bf16x2_upper(x[0][0], x[0][1]), bf16x2_upper(x[0][2], x[0][3]), bf16x2_upper(x[1][0], x[1][1]),
                 bf16x2_upper(x[1][2], x[1][3])};
      pop[k] = *reinterpret_cast<bf16x8*>(&w);
    }
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      auto code = [&](int j) { return (float)(int8_t)(r.v[j][t / 4] >> (8 * (t % 4))); };
      u32x4 w = {bf16x2_upper(code(0), code(1)), bf16x2_upper(code(2), code(3)), bf16x2_upper(code(4), code(5)),
                 bf16x2_upper(code(6), code(7))};
      const bf16x8 vop = *reinterpret_cast<bf16x8*>(&w);
#pragma unroll
      for (int k = 0; k < NP; ++k) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, pop[k], acc[t], 0, 0, 0);
    }
  };

  // the ring of attn_kernel: PF - 1 tiles in flight, loads past the end re-read the last tile
  if (nt > 0) {
    const int full_end = lim_lo > 0 ? lim_lo / TILE : 0;
    const int j_full = min(nt, full_end > c_begin + ks ? (full_end - c_begin - ks + KS - 1) / KS : 0);
    int j0 = 0;
    for (; j0 + PF <= j_full; j0 += PF) {
#pragma unroll
      for (int jj = 0; jj < PF; ++jj) {
        load(ring[(jj + PF - 1) % PF], tile(min(j0 + jj + PF - 1, nt - 1)));
        compute(std::false_type{}, ring[jj], tile(j0 + jj));
      }
    }
    for (; j0 < nt; j0 += PF) {
#pragma unroll
      for (int jj = 0; jj < PF; ++jj) {
        const int j = j0 + jj;
        if (j >= nt) break;
        load(ring[(jj + PF - 1) % PF], tile(min(j + PF - 1, nt - 1)));
        compute(std::true_type{}, ring[jj], tile(j));
      }
    }
  }

  // ---- epilogue: lane (n, g) holds channels (D/4) g + (D/16) i + t of its row in acc[t][i] ----
  l = group4_sum(l);
  if constexpr (PACK) {   // both planes of a row: lanes n and n + 8 end with the same sums
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] += ror8(acc[t][i]);
  }
  if (KS > 1) {   // attn_kernel's merge of the key splits
    static_assert(VT * 4 + 2 <= MERGE_FIELDS, "merge slot too small");
    auto slot = [&](int k) { return lds + (size_t)((k - 1) * a.rt + rtile) * MERGE_FIELDS * WAVE + lane; };
    if (ks > 0 && active) {
      float* sl = slot(ks);
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sl[(4 * t + i) * WAVE] = acc[t][i];
      sl[(4 * VT) * WAVE] = m;
      sl[(4 * VT + 1) * WAVE] = l;
    }
    __syncthreads();
    if (ks == 0 && active) {
      float M = m;
      for (int k = 1; k < KS; ++k) M = __builtin_fmaxf(M, slot(k)[(4 * VT) * WAVE]);
      const float w0 = __builtin_amdgcn_exp2f(m - M);
      l *= w0;
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] *= w0;
      for (int k = 1; k < KS; ++k) {
        const float* src = slot(k);
        const float wk = __builtin_amdgcn_exp2f(src[(4 * VT) * WAVE] - M);
        l = __builtin_fmaf(wk, src[(4 * VT + 1) * WAVE], l);
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(wk, src[(4 * t + i) * WAVE], acc[t][i]);
      }
      m = M;
    }
    __syncthreads();
  }
  if (ks > 0 || !active || rtok >= qlen || (PACK && n >= 8)) return;
  // ---- the end of a piece: bf16 out of a whole segment, or the fp32 partial of a cut one (as finish_segment) ----
  const AttnArgs& o = fresh_args();
  const int qt = tok + rtok, head = kvh * G + rh;
  if (l != l) {   // (a denominator that is no number would not tell the merge that the row was cut)
    l = 1.f;
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = NAN;
  }
  if (nparts == 1) {
    if (o.max_splits > 1 && qt < o.cut_rows && g == 0)
      o.segm_sum[(int64_t)qt * o.seg_st + (int64_t)head * o.seg_sh] = -1.f;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint32_t w[OPL / 2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < VT; t += 2) w[(VT * i + t) / 2] = pack_bf16x2(acc[t][i] * inv, acc[t + 1][i] * inv);
    u32x4* op = reinterpret_cast<u32x4*>(o.out + (int64_t)qt * o.o_st + (int64_t)head * o.o_sh + OPL * g);
#pragma unroll
    for (int u = 0; u < OPL / 8; ++u) op[u] = u32x4{w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]};
  } else {
    const int64_t sidx = (int64_t)qt * o.seg_st + (int64_t)head * o.seg_sh + part;
    if (g == 0) {
      o.segm_max[sidx] = m;
      o.segm_sum[sidx] = part == nparts - 1 ? last_piece_sum(l) : l;
    }
    float* sp = o.segm_out + sidx * D + OPL * g;
#pragma unroll
    for (int u = 0; u < OPL / 4; ++u) {
      const int c0 = 4 * u;
      reinterpret_cast<float4*>(sp)[u] = float4{acc[(c0 + 0) % VT][(c0 + 0) / VT], acc[(c0 + 1) % VT][(c0 + 1) / VT],
                                                acc[(c0 + 2) % VT][(c0 + 2) / VT], acc[(c0 + 3) % VT][(c0 + 3) / VT]};
    }
  }
}

// Two wavefronts a SIMD at head_dim 128, though the 163 registers that PACK needs leave room for three: those cut a batch into
// more pieces for nothing (the ragged batch 102 -> 118 us, 32 requests of 4,000 to 8,192 keys 42.4 -> 47.0), and with pieces
// for two but room for three the CUs that an earlier kernel leaves first take more than their share (48 decode rows behind
// two prompts' prefill 86.8 -> 89.2 us in all).
template <int D>
constexpr int BLOCK_ATTN_WAVES = D == 128 ? 2 : 8;
template <int D, int PF, bool PACK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, BLOCK_ATTN_WAVES<D>))) void block_attn_kernel(BlockAttnArgs args) {
  touch_args();
  const AttnArgs& a = args.a;
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int rt = a.rt, ksplit = a.ksplit, kspl = div_row_tiles(wave, rt), rtile = wave - kspl * rt;
  extern __shared__ float merge_lds[];
  int solo = 0;
  walk_pieces(a, lane, [&](int r, const ReqWork& w, int kvh, int rg, int c0, int c1, int part, int nparts) {
    const int row0 = (rg * rt + rtile) * (PACK ? 8 : 16);
    if (ksplit > 1 && c1 - c0 >= a.coop) {
      attend_blocks<D, PF, PACK>(r, w.tok, w.qlen, w.len, kvh, row0, c0, c1, kspl, ksplit, rtile, part, nparts, merge_lds, lane);
    } else {
      if (solo % ksplit == kspl)
        attend_blocks<D, PF, PACK>(r, w.tok, w.qlen, w.len, kvh, row0, c0, c1, 0, 1, rtile, part, nparts, merge_lds, lane);
      ++solo;
    }
  });
}

// ------------------------------------------------------------------------------------------------
// Many query rows (block_rows.h). block_verify_kernel: short queries of more rows than block_attn_kernel's tiles suit, on
// its plan, in pieces of 64 rows. block_prefill_kernel: the work lists of long queries, 128 rows an entry.
// 64 requests of 8 tokens, 512 to 8,192 keys (28 / 4 heads x 128): 46 us + 8.5 of the merge, 162 MB; the vector units are busy
// 48% of the cycles and the wavefronts wait for 31% of theirs. Not at a limit of its own: each wavefront reads the whole tile
// from LDS for 16 rows, and all of them convert V behind one barrier. 700 + 333 tokens (block_prefill_kernel, cut): 43 us + 7.5.
// ------------------------------------------------------------------------------------------------
constexpr int64_t BLOCK_VERIFY_ONE_GROUP = 128;   // (request, kv head) pairs of a cut batch from which one group is faster
template <int D, int KW>
__global__ __launch_bounds__(256 * KW, KW == 1 ? 3 : 2) void block_verify_kernel(BlockAttnArgs args) {
  touch_args();
  __shared__ __attribute__((aligned(1024))) RowsLds<D, 4> lds[KW];
  const int lane = threadIdx.x & (WAVE - 1), n = lane & 15, g = lane >> 4;
  walk_pieces(args.a, lane, [&](int r, const ReqWork& w, int kvh, int rg, int c0, int c1, int part, int nparts) {
    const AttnArgs& a = fresh_args();
    const BlockScales& s = fresh_scales();
    const RowsView v{a.q, a.kc + (int64_t)kvh * a.k_sh, a.vc + (int64_t)kvh * a.v_sh, a.block_table + (int64_t)r * a.bt_stride,
                     s.ks + (int64_t)kvh * s.sh, s.vs + (int64_t)kvh * s.sh, a.q_st, a.q_sh, a.k_sb, a.k_sn, a.v_sb, a.v_sn,
                     s.sb, s.sg, a.sm_log2, a.G, a.num_blocks, a.lbs, s.lg};
    attend_rows<D, 4, 1, KW>(v, lds, w.tok, w.qlen, w.len, kvh, 64 * rg, c0, w.len > 0 ? c1 : c0, min(w.len, c1 * PR_KEYS),
                      [&](int, int t, int hq, bool valid, float m, float l, const f32x4 (&acc)[D / 16]) {
      if (!valid) return;
      const AttnArgs& o = fresh_args();
      const int qt = w.tok + t;
      if (nparts == 1) {
        if (o.max_splits > 1 && qt < o.cut_rows && g == 0)
          o.segm_sum[(int64_t)qt * o.seg_st + (int64_t)hq * o.seg_sh] = -1.f;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        uint16_t* op = o.out + (int64_t)qt * o.o_st + (int64_t)hq * o.o_sh + 4 * g;
#pragma unroll
        for (int tt = 0; tt < D / 16; ++tt)
          *reinterpret_cast<u32x2*>(op + 16 * tt) = u32x2{pack_bf16x2_rne(acc[tt][0] * inv, acc[tt][1] * inv),
                                                          pack_bf16x2_rne(acc[tt][2] * inv, acc[tt][3] * inv)};
      } else {
        const int64_t sidx = (int64_t)qt * o.seg_st + (int64_t)hq * o.seg_sh + part;
        if (g == 0) {
          if (l != l) l = 1.f;   // (no number would not tell the merge that the row was cut; the accumulators are none either)
          o.segm_max[sidx] = m;
          o.segm_sum[sidx] = part == nparts - 1 ? last_piece_sum(l) : l;
        }
        float* sp = o.segm_out + sidx * D + 4 * g;
#pragma unroll
        for (int tt = 0; tt < D / 16; ++tt) *reinterpret_cast<f32x4*>(sp + 16 * tt) = acc[tt];
      }
    });
  });
}

// The bf16 prefill over a temporary cache of the codes and their scales' table (kvq_block_codes). 2 x 8,192 tokens of 32 / 8
// heads x 128 941 us, 1.17 PFLOP/s, the matrix cores busy 59% of the cycles (profiled alone; with the copy, 21 us, 960 to
// 1,028 us a call).
template <int D, bool SPLIT>
__global__ __launch_bounds__(256, 3) void block_codes_prefill_kernel(PrefillArgs a) {
  prefill_body<D, PR_SRC_BF16_BLOCK, SPLIT>(a);
}

struct BlockPrefillArgs {
  PrefillArgs p;
  BlockScales s;
};

// D = 128: eight wavefronts of one row block each (four of two leave the tile loop short of registers).
template <int D>
constexpr int BLOCK_PREFILL_WAVES = D == 128 ? 8 : 4;
template <int D, bool SPLIT>
__global__ __launch_bounds__(WAVE * BLOCK_PREFILL_WAVES<D>, 4) void block_prefill_kernel(BlockPrefillArgs args) {
  constexpr int NW = BLOCK_PREFILL_WAVES<D>, RB = PR_ROWS / (16 * NW);
  __shared__ __attribute__((aligned(1024))) RowsLds<D, NW> lds[1];
  const PrefillArgs& a = args.p;
  const BlockScales& s = args.s;
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), n = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.y, r = a.tile_req[blockIdx.x], row0 = a.tile_row[blockIdx.x];
  const int tok = a.cu_q[r], Q = a.cu_q[r + 1] - tok, L = a.seq_lens[r];
  const int t_last = min(Q - 1, (row0 + PR_ROWS - 1) / a.G);
  int kend = max(0, min(L, L - Q + 1 + t_last)), c_lo = 0, c_hi = (kend + PR_KEYS - 1) / PR_KEYS;
  if constexpr (SPLIT) {   // an equal share of the rows' tiles
    const int pp = a.tile_piece[blockIdx.x], nparts = pp >> 16, part = pp & 0xffff, each = c_hi / nparts, rem = c_hi % nparts;
    c_lo = part * each + min(part, rem);
    c_hi = c_lo + each + (part < rem ? 1 : 0);
    kend = min(kend, c_hi * PR_KEYS);
  }
  const RowsView v{a.q, (const int8_t*)a.kc + (int64_t)kvh * a.k_sh, (const int8_t*)a.vc + (int64_t)kvh * a.v_sh,
                   a.block_table + (int64_t)r * a.bt_stride, s.ks + (int64_t)kvh * s.sh, s.vs + (int64_t)kvh * s.sh, a.q_st,
                   a.q_sh, a.k_sb, a.k_sn, a.v_sb, a.v_sn, s.sb, s.sg, a.sm_log2, a.G, a.num_blocks, a.lbs, s.lg};
  bool piece = false;
  int pslot = 0;
  attend_rows<D, NW, RB, 1>(v, lds, tok, Q, L, kvh, row0, c_lo, c_hi, kend,
                        [&](int rb, int t, int hq, bool valid, float m, float l, const f32x4 (&acc)[D / 16]) {
    if constexpr (SPLIT) {
      if (rb == 0) {   // read here, not held through the tile loop
        int x = blockIdx.x;
        asm volatile("" : "+s"(x));
        piece = (a.tile_piece[x] >> 16) > 1;
        pslot = a.tile_slot[x];
      }
    }
    if (!valid) return;
    if (SPLIT && piece) {   // the accumulators as they are: the merge divides by the whole denominator
      const int64_t pr = ((int64_t)pslot * gridDim.y + kvh) * PR_ROWS + (wave * RB + rb) * 16 + n;
      if (g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * pr) = float2{m, l};
      float* prow = a.part_out + pr * D + 4 * g;
#pragma unroll
      for (int tt = 0; tt < D / 16; ++tt) *reinterpret_cast<f32x4*>(prow + 16 * tt) = acc[tt];
      return;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint16_t* op = a.out + (int64_t)(tok + t) * a.o_st + (int64_t)hq * a.o_sh + 4 * g;
#pragma unroll
    for (int tt = 0; tt < D / 16; ++tt)
      *reinterpret_cast<u32x2*>(op + 16 * tt) = u32x2{pack_bf16x2_rne(acc[tt][0] * inv, acc[tt][1] * inv),
                                                      pack_bf16x2_rne(acc[tt][2] * inv, acc[tt][3] * inv)};
  });
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
// What every call on a block-scaled cache checks; 0, or the error after fail().
int check_blocks(const char* nm, int64_t num_blocks, int64_t block_size, int64_t group, int64_t heads, int64_t head_dim,
                 const void* kc, int64_t k_sb, int64_t k_sn, int64_t k_sh, const void* vc, int64_t v_sb, int64_t v_sn,
                 int64_t v_sh) {
  if (head_dim != 64 && head_dim != 128) return fail("%s: head_dim must be 64 or 128, got %lld", nm, (long long)head_dim);
  if (block_size < 16 || !pow2(block_size) || block_size > (1 << 24))
    return fail("%s: block_size must be a power of two >= 16", nm);
  if (!pow2(group) || group < BLK_MIN || group > BLK_MAX || group > block_size)
    return fail("%s: positions per scale must be a power of two from %d to %d, at most block_size, got %lld", nm, BLK_MIN, BLK_MAX,
                (long long)group);
  if (heads <= 0 || heads > 65535 || num_blocks <= 0 || num_blocks > INT32_MAX) return fail("%s: bad sizes", nm);
  if (!kc || !vc || !aligned16(kc) || !aligned16(vc) || (k_sb | k_sn | k_sh | v_sb | v_sn | v_sh) % 16)
    return fail("%s: cache rows must be 16-byte aligned (base pointers and strides)", nm);
  return 0;
}
BlockScales block_scales(const float* ks, const float* vs, int64_t sb, int64_t sh, int64_t sg, int64_t group) {
  return BlockScales{ks, vs, sb, sh, sg, log2i(group)};
}

}  // namespace

extern "C" {

int kvq_quant_block_cache(const void* key, int64_t key_st, int64_t key_sh, const void* value, int64_t val_st,
                          int64_t val_sh, int64_t num_tokens, int8_t* k_cache, int64_t kc_sb, int64_t kc_sn,
                          int64_t kc_sh, int8_t* v_cache, int64_t vc_sb, int64_t vc_sn, int64_t vc_sh,
                          int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim, float* k_scale,
                          float* v_scale, int64_t s_sb, int64_t s_sh, int64_t s_sg, int64_t group,
                          const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                          int64_t bt_stride, int64_t num_seqs, void* stream) {
  const char* nm = "quant_block_cache";
  if (num_tokens < 0 || num_seqs < 0 || num_tokens > INT32_MAX || num_seqs > INT32_MAX / 4) return fail("%s: bad sizes", nm);
  if (num_tokens == 0 || num_seqs == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_blocks(nm, num_blocks, block_size, group, num_heads, head_dim, k_cache, kc_sb, kc_sn, kc_sh, v_cache,
                                  vc_sb, vc_sn, vc_sh)) return rc;
  if (!key || !value || !k_scale || !v_scale || !cu_seqlens_q || !seq_lens || !block_table) return fail("%s: null pointer", nm);
  if (!aligned16(key) || !aligned16(value) || (key_st | key_sh | val_st | val_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  QuantBlockArgs a;
  a.key = (const uint16_t*)key; a.value = (const uint16_t*)value; a.kc = k_cache; a.vc = v_cache; a.ks = k_scale; a.vs = v_scale;
  a.cu_q = cu_seqlens_q; a.seq_lens = seq_lens; a.block_table = block_table;
  a.key_st = key_st; a.key_sh = key_sh; a.val_st = val_st; a.val_sh = val_sh;
  a.kc_sb = kc_sb; a.kc_sn = kc_sn; a.kc_sh = kc_sh; a.vc_sb = vc_sb; a.vc_sn = vc_sn; a.vc_sh = vc_sh;
  a.s_sb = s_sb; a.s_sh = s_sh; a.s_sg = s_sg; a.bt_stride = bt_stride;
  a.num_seqs = (int)num_seqs; a.num_tokens = (int)num_tokens; a.heads = (int)num_heads; a.num_blocks = (int)num_blocks;
  a.lbs = log2i(block_size); a.lg = log2i(group);
  const int64_t items = block_slots(num_tokens, num_seqs, a.lg) * num_heads;
  if (items > INT32_MAX) return fail("%s: too many tokens and heads for one call", nm);
  a.items = (int)items;
  const int w = (int)(group / 16), wpb = w < 4 ? 4 : w;
  const dim3 grid((unsigned)((items + wpb / w - 1) / (wpb / w))), block(WAVE * wpb);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto d_t) {
    constexpr int D = decltype(d_t)::value;
    if (w == 1) hipLaunchKernelGGL((quant_block_kernel<D, 1>), grid, block, 0, st, a);
    else if (w == 2) hipLaunchKernelGGL((quant_block_kernel<D, 2>), grid, block, 0, st, a);
    else if (w == 4) hipLaunchKernelGGL((quant_block_kernel<D, 4>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((quant_block_kernel<D, 8>), grid, block, 0, st, a);
  };
  if (head_dim == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  return launched(nm);
}

int kvq_read_block_cache(const int8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, const int8_t* v_cache,
                         int64_t vc_sb, int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size,
                         int64_t num_heads, int64_t head_dim, const float* k_scale, const float* v_scale, int64_t s_sb,
                         int64_t s_sh, int64_t s_sg, int64_t group, const int32_t* starts, const int32_t* cu_seqlens_k,
                         const int32_t* block_table, int64_t bt_stride, int64_t num_seqs, void* k_out, int64_t ko_st,
                         int64_t ko_sh, void* v_out, int64_t vo_st, int64_t vo_sh, int64_t num_rows, void* stream) {
  const char* nm = "read_block_cache";
  if (num_rows < 0 || num_seqs < 0 || num_rows > INT32_MAX || num_seqs > INT32_MAX / 4) return fail("%s: bad sizes", nm);
  if (num_rows == 0 || num_seqs == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_blocks(nm, num_blocks, block_size, group, num_heads, head_dim, k_cache, kc_sb, kc_sn, kc_sh, v_cache,
                                  vc_sb, vc_sn, vc_sh)) return rc;
  if (!k_out || !v_out || !k_scale || !v_scale || !starts || !cu_seqlens_k || !block_table) return fail("%s: null pointer", nm);
  if (!aligned16(k_out) || !aligned16(v_out) || (ko_st | ko_sh | vo_st | vo_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  ReadBlockArgs a;
  a.kc = k_cache; a.vc = v_cache; a.ko = (uint16_t*)k_out; a.vo = (uint16_t*)v_out;
  a.start = starts; a.cu_k = cu_seqlens_k; a.block_table = block_table;
  a.s = block_scales(k_scale, v_scale, s_sb, s_sh, s_sg, group);
  a.kc_sb = kc_sb; a.kc_sn = kc_sn; a.kc_sh = kc_sh; a.vc_sb = vc_sb; a.vc_sn = vc_sn; a.vc_sh = vc_sh;
  a.ko_st = ko_st; a.ko_sh = ko_sh; a.vo_st = vo_st; a.vo_sh = vo_sh; a.bt_stride = bt_stride;
  a.num_seqs = (int)num_seqs; a.num_rows = (int)num_rows; a.heads = (int)num_heads; a.num_blocks = (int)num_blocks;
  a.lbs = log2i(block_size);
  const int64_t items = block_slots(num_rows, num_seqs, 4) * num_heads;
  if (items > INT32_MAX) return fail("%s: too many rows and heads for one call", nm);
  a.items = (int)items;
  const dim3 grid((unsigned)((items + 3) / 4));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool nt = 6 * num_rows * num_heads * head_dim > READ_NT_BYTES;
  void (*kern)(ReadBlockArgs) = head_dim == 128 ? (nt ? read_block_kernel<128, true> : read_block_kernel<128, false>)
                                                : (nt ? read_block_kernel<64, true> : read_block_kernel<64, false>);
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a);
  return launched(nm);
}

}  // extern "C"

namespace {

// What the two attention calls check.
int check_attention(const char* nm, const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                    int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                    int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_dim, const float* k_scale,
                    const float* v_scale, int64_t group, void* out, int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q,
                    const int32_t* seq_lens, const int32_t* block_table, int64_t num_q_heads, double softmax_scale) {
  // (times an unwritten block's least K scale, 1e-20, it has to stay a normal fp32 number: a masked score is multiplied by it)
  if (!(softmax_scale >= MIN_SOFTMAX_SCALE && softmax_scale <= MAX_SOFTMAX_SCALE))
    return fail("%s: softmax_scale must be positive and finite, from %g to %g", nm, MIN_SOFTMAX_SCALE, MAX_SOFTMAX_SCALE);
  if (const int rc = check_blocks(nm, num_blocks, block_size, group, num_kv_heads, head_dim, k_cache, k_sb, k_sn, k_sh, v_cache,
                                  v_sb, v_sn, v_sh)) return rc;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads || num_q_heads > 65535)
    return fail("%s: bad head counts Hq=%lld Hkv=%lld", nm, (long long)num_q_heads, (long long)num_kv_heads);
  if (!q || !out || !k_scale || !v_scale || !cu_seqlens_q || !seq_lens || !block_table) return fail("%s: null pointer", nm);
  if (!aligned16(q) || !aligned16(out) || (q_st | q_sh | o_st | o_sh) % 8)
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  return 0;
}
}  // namespace

extern "C" {

int kvq_block_decode_attention(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                               int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                               int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                               int64_t head_dim, const float* k_scale, const float* v_scale, int64_t s_sb, int64_t s_sh,
                               int64_t s_sg, int64_t group, void* out, int64_t o_st, int64_t o_sh,
                               const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                               int64_t bt_stride, int64_t num_seqs, int64_t num_q_heads, double softmax_scale,
                               float* segm_out, float* segm_max, float* segm_sum, int64_t seg_st, int64_t seg_sh,
                               int64_t num_splits, int64_t segm_rows, int64_t target_waves, int64_t max_query_len,
                               int64_t qmax, void* stream) {
  const char* nm = "block_decode_attention";
  if (num_splits < 1 || num_splits > MAX_SPLITS) return fail("%s: at most %d split-KV segments", nm, MAX_SPLITS);
  if (num_seqs < 0 || num_seqs > INT32_MAX / 4 || max_query_len < 0 || qmax < 1 || target_waves < 0 || segm_rows < 0)
    return fail("%s: bad sizes", nm);
  if (num_seqs == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_attention(nm, q, q_st, q_sh, k_cache, k_sb, k_sn, k_sh, v_cache, v_sb, v_sn, v_sh, num_blocks,
                                     block_size, num_kv_heads, head_dim, k_scale, v_scale, group, out, o_st, o_sh, cu_seqlens_q,
                                     seq_lens, block_table, num_q_heads, softmax_scale)) return rc;
  if (num_splits > 1 && segm_rows > 0 && (!segm_out || !segm_max || !segm_sum || !aligned16(segm_out)))
    return fail("%s: split buffers missing or not 16-byte aligned", nm);
  if (k_sn < 0 || v_sn < 0 || block_size * k_sn > INT32_MAX || block_size * v_sn > INT32_MAX)
    return fail("%s: page too large for 32-bit lane offsets", nm);
  const int G = (int)(num_q_heads / num_kv_heads);
  const int64_t maxq = std::min<int64_t>(std::max<int64_t>(max_query_len, 1), qmax), rows = (int64_t)G * maxq;
  if (rows > INT32_MAX / 4) return fail("%s: grid too large", nm);
  // the row tile: 8 rows, both planes in one MFMA, where that holds all of a request's rows; else 16
  const bool pack = rows <= 8;
  const int rt = (int)std::min<int64_t>(MAX_ROW_TILES, (rows + 15) / 16);
  const Tuning tune = read_tuning();
  // many rows (attn_rules.h) share each tile through LDS: one group of wavefronts a workgroup, three workgroups a CU, where
  // the batch is cut into enough pieces for that (us, one and two groups: 64 x 8 tokens of 28 / 4 heads at 512 to 8,192 keys
  // 72.0 and 78.9, 32 x 4 at 4,096 39.7 and 45.7, 64 x 8 of 32 / 8 80.4 and 87.5), else two groups that share a piece's
  // tiles (16 x 8 at 1,000 to 3,000 27.5 and 23.3, 64 decode rows of 32 / 1 41.8 and 38.1; whole segments 64 x 8 at 4,096
  // 103 and 77). KVQ_V32_KSPLIT sets the groups, KVQ_ROWS32=0 takes block_attn_kernel for every row count.
  const int64_t pairs = num_seqs * num_kv_heads;
  const bool cut = num_splits > 1 && segm_rows > 0;
  const bool many = verify_rows(rows, pairs, cut) && !(tune.rows32 && atoi(tune.rows32) == 0);
  const int kw = tune.v32_ksplit ? v32_key_splits(tune) : cut && pairs >= BLOCK_VERIFY_ONE_GROUP ? 1 : 2;
  const int ks_max = tune.ksplit ? std::max(1, std::min(MAX_ROW_TILES, atoi(tune.ksplit)))
                     : num_splits == 1 || num_seqs * num_kv_heads <= WIDE_SPLIT_PAIRS ? MAX_ROW_TILES : DEFAULT_KSPLIT;
  const int ks = many ? 1 : std::max(1, std::min(ks_max, MAX_ROW_TILES / rt)), waves = many ? 4 * kw : rt * ks;
  BlockAttnArgs b;
  b.s = block_scales(k_scale, v_scale, s_sb, s_sh, s_sg, group);
  AttnArgs& a = b.a;
  a.q = (const uint16_t*)q; a.kc = k_cache; a.vc = v_cache; a.out = (uint16_t*)out;
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
  a.rt = many ? 4 : rt; a.ksplit = ks; a.waves = waves;
  a.min_tiles = many ? MIN_SPLIT_TILES * kw : MIN_SPLIT_TILES;
  a.coop = coop_tiles(num_splits > 1, ks);
  a.xcd_order = tune.xcd_order ? atoi(tune.xcd_order) : 1;
  a.plan_fast_max = tune.plan_fast_max ? (int)std::max(1ll, std::min(PLAN_FAST_MAX, atoll(tune.plan_fast_max)))
                                       : (int)PLAN_FAST_MAX;
  a.seg_cost = seg_cost_units(tune, many ? 2 : 0);
  const size_t lds = many ? 0 : (size_t)(ks - 1) * rt * MERGE_FIELDS * WAVE * sizeof(float);
  void (*kern)(BlockAttnArgs) = many ? (head_dim == 128 ? (kw == 2 ? block_verify_kernel<128, 2> : block_verify_kernel<128, 1>)
                                     : (kw == 2 ? block_verify_kernel<64, 2> : block_verify_kernel<64, 1>))
                              : head_dim == 128 ? (pack ? block_attn_kernel<128, 2, true> : block_attn_kernel<128, 2, false>)
                                                : (pack ? block_attn_kernel<64, 2, true> : block_attn_kernel<64, 2, false>);
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
  if (head_dim == 128) hipLaunchKernelGGL((split_reduce_kernel<128, true>), rgrid, dim3(WAVE * RED_WAVES), 0, st, a);
  else hipLaunchKernelGGL((split_reduce_kernel<64, true>), rgrid, dim3(WAVE * RED_WAVES), 0, st, a);
  return launched("block_decode_attention: merge");
}

int kvq_block_prefill_attention(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                                int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                                int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                int64_t head_dim, const float* k_scale, const float* v_scale, int64_t s_sb, int64_t s_sh,
                                int64_t s_sg, int64_t group, void* out, int64_t o_st, int64_t o_sh,
                                const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                                int64_t bt_stride, int64_t num_q_heads, const int32_t* tile_req, const int32_t* tile_row,
                                int64_t num_tiles, int64_t rows_per_tile, double softmax_scale, const int32_t* tile_piece,
                                const int32_t* tile_slot, const int32_t* merge, int64_t num_merge, float* part_out,
                                float* part_ml, const void* k_codes, const void* v_codes, const float* code_scales,
                                int64_t num_pages, const int32_t* codes_table, int64_t ct_stride, void* stream) {
  const char* nm = "block_prefill_attention";
  if (num_tiles < 0 || num_tiles > INT32_MAX || num_merge < 0 || num_merge > INT32_MAX) return fail("%s: bad sizes", nm);
  if (num_tiles == 0) { g_err.clear(); return KVQ_OK; }
  if (rows_per_tile != PR_ROWS) return fail("%s: work list tiles must be %d rows", nm, PR_ROWS);
  if (!tile_req || !tile_row || (tile_piece && !tile_slot)) return fail("%s: bad work list", nm);
  if (tile_piece && num_merge > 0 && (!merge || !part_out || !part_ml || !aligned16(merge) || !aligned16(part_out) ||
                                      !aligned16(part_ml)))
    return fail("%s: split work list needs 16-byte aligned merge list and partial buffers", nm);
  if (const int rc = check_attention(nm, q, q_st, q_sh, k_cache, k_sb, k_sn, k_sh, v_cache, v_sb, v_sn, v_sh, num_blocks,
                                     block_size, num_kv_heads, head_dim, k_scale, v_scale, group, out, o_st, o_sh, cu_seqlens_q,
                                     seq_lens, block_table, num_q_heads, softmax_scale)) return rc;
  if (k_sn < 0 || v_sn < 0 || block_size * k_sn > INT32_MAX || block_size * v_sn > INT32_MAX)
    return fail("%s: page too large for 32-bit lane offsets", nm);
  if (k_codes && (!v_codes || !codes_table || !code_scales || !aligned16(code_scales) || num_pages <= 0 || num_pages > INT32_MAX || !aligned16(k_codes) || !aligned16(v_codes)))
    return fail("%s: bad temporary cache", nm);
  if (k_codes && 2 * block_size * num_kv_heads * head_dim > INT32_MAX)
    return fail("%s: page too large for 32-bit page / slot offsets", nm);
  BlockPrefillArgs b;
  b.s = block_scales(k_scale, v_scale, s_sb, s_sh, s_sg, group);
  PrefillArgs& a = b.p;
  a.q = (const uint16_t*)q; a.kc = (const uint16_t*)k_cache; a.vc = (const uint16_t*)v_cache; a.out = (uint16_t*)out;
  a.cu_q = cu_seqlens_q; a.seq_lens = seq_lens; a.block_table = block_table; a.tile_req = tile_req; a.tile_row = tile_row;
  a.tile_piece = tile_piece; a.tile_slot = tile_slot; a.part_out = part_out; a.part_ml = part_ml;
  a.q_st = q_st; a.q_sh = q_sh; a.o_st = o_st; a.o_sh = o_sh;
  a.k_sb = k_sb; a.k_sn = k_sn; a.k_sh = k_sh; a.v_sb = v_sb; a.v_sn = v_sn; a.v_sh = v_sh; a.bt_stride = bt_stride;
  a.sm_log2 = (float)(softmax_scale * 1.4426950408889634);
  a.G = (int)(num_q_heads / num_kv_heads); a.lbs = log2i(block_size); a.num_blocks = (int)num_blocks;
  a.kpage = a.vpage = a.krow = a.vrow = 0; a.contig = 0; a.ks = a.vs = nullptr; a.ks_pc = a.vs_pc = 0;   // (prefill_body's)
  a.s_table = reinterpret_cast<const f32x4*>(code_scales);
  if (k_codes) {   // the temporary cache's pages instead: bf16 [num_pages, block_size, H, D], contiguous
    a.kc = (const uint16_t*)k_codes; a.vc = (const uint16_t*)v_codes;
    a.block_table = codes_table; a.bt_stride = ct_stride; a.num_blocks = (int)num_pages;
    a.k_sh = a.v_sh = head_dim;
    a.k_sn = a.v_sn = num_kv_heads * head_dim;
    a.k_sb = a.v_sb = block_size * a.k_sn;
    a.krow = a.vrow = (uint32_t)(2 * a.k_sn);
    a.kpage = a.vpage = (uint32_t)(2 * a.k_sb);
    a.contig = 1;
  }
  const dim3 grid((unsigned)num_tiles, (unsigned)num_kv_heads);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  void (*kern)(BlockPrefillArgs) = head_dim == 128 ? (tile_piece ? block_prefill_kernel<128, true> : block_prefill_kernel<128, false>)
                                              : (tile_piece ? block_prefill_kernel<64, true> : block_prefill_kernel<64, false>);
  void (*codes_kern)(PrefillArgs) = head_dim == 128
      ? (tile_piece ? block_codes_prefill_kernel<128, true> : block_codes_prefill_kernel<128, false>)
      : (tile_piece ? block_codes_prefill_kernel<64, true> : block_codes_prefill_kernel<64, false>);
  if (k_codes) hipLaunchKernelGGL(codes_kern, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(kern, grid, dim3(WAVE * (head_dim == 128 ? BLOCK_PREFILL_WAVES<128> : BLOCK_PREFILL_WAVES<64>)), 0, st, b);
  const int rc = launched(nm);
  if (rc != KVQ_OK || !tile_piece || num_merge == 0) return rc;
  const dim3 mgrid((unsigned)num_merge, (unsigned)num_kv_heads, PR_ROWS / PR_MERGE_WAVES);
  const int4* ml = reinterpret_cast<const int4*>(merge);
  if (head_dim == 128) hipLaunchKernelGGL(prefill_merge_kernel<128>, mgrid, dim3(WAVE * PR_MERGE_WAVES), 0, st, a, ml);
  else hipLaunchKernelGGL(prefill_merge_kernel<64>, mgrid, dim3(WAVE * PR_MERGE_WAVES), 0, st, a, ml);
  return launched("block_prefill_attention: merge");
}

int kvq_block_codes(const int8_t* k_cache, int64_t k_sb, int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb,
                    int64_t v_sn, int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim,
                    const float* k_scale, const float* v_scale, int64_t s_sb, int64_t s_sh, int64_t s_sg, int64_t group,
                    void* k_out, void* v_out, float* scales_out, const int32_t* block_table, int64_t bt_stride,
                    const int32_t* src_req, const int32_t* src_j, int64_t num_pages, void* stream) {
  const char* nm = "block_codes";
  if (num_pages < 0 || num_pages > INT32_MAX) return fail("%s: bad sizes", nm);
  if (num_pages == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_blocks(nm, num_blocks, block_size, group, num_heads, head_dim, k_cache, k_sb, k_sn, k_sh, v_cache,
                                  v_sb, v_sn, v_sh)) return rc;
  if (!k_out || !v_out || !scales_out || !k_scale || !v_scale || !block_table || !src_req || !src_j) return fail("%s: null pointer", nm);
  if (!aligned16(k_out) || !aligned16(v_out) || !aligned16(scales_out))
    return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  return dequant_launch<true>(nm, k_cache, k_sb, k_sn, k_sh, v_cache, v_sb, v_sn, v_sh, num_blocks, block_size, num_heads,
                              head_dim, k_out, v_out, block_table, bt_stride, src_req, src_j, num_pages, nullptr, 0, nullptr, 0,
                              BlockCodes{block_scales(k_scale, v_scale, s_sb, s_sh, s_sg, group), reinterpret_cast<f32x4*>(scales_out)},
                              stream);
}

}  // extern "C"
