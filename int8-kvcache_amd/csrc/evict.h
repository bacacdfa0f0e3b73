// Eviction from a 4-bit cache by accumulated attention weight. Part of kvq_int8.hip (included at its end, after fp4_cache.h).
//
//   key_weights_kernel   adds what each cached key gets of a step's rows to its running sum
//   evict_kernel         chooses each request's and kv head's keys and moves them to the front of its pages
//   evict_lens_kernel    the lengths from then on, where they replace what evict_kernel reads
#pragma once

namespace {

// ------------------------------------------------------------------------------------------------
// w[r, h, j] += sum over the request's rows i (query tokens x the kv head's q heads) that see key j of 2^(s_ij - lse_i)
// The scores are fp4_attn_kernel's; K alone is read. Pieces of key tiles by attn_kernel's plan (rt is all of a request's row
// tiles, so a key's sum has one owner in a call: nothing is atomic, the result does not depend on the order of workgroups);
// a piece's tiles go round the workgroup's wavefronts. A wavefront holds RT row tiles' planes; more rows take another round
// over the piece's tiles, whose keys' sums the same lanes then add to again.
// Bound by memory: 16 requests of 16384 keys, 8 KV heads of 128, 8 tokens of 4 q heads: 58 us for 160 MB, of K's codes and the
// sums. Where K's and V's codes of a key share a line, the half that is V's comes along: 290 MB, 5.0 TB/s. A ragged batch of 24
// decoding requests: 6.7 us. Rings of 3 and 4 tiles, 8 wavefronts and loads without the streaming hint were all slower.
// ------------------------------------------------------------------------------------------------
struct KeyWeightArgs {
  AttnArgs a;   // (first: fresh_args)
  Fp4Scales s;
  const float* lse;
  float* w;
  int64_t lse_st, w_sr, w_sh;
  int cols;
};
static_assert(offsetof(KeyWeightArgs, a) == 0, "AttnArgs lead the kernel arguments");

// sum over each 16 lanes
__device__ __forceinline__ float sum_row(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, true));   // row_ror:8
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xf, 0xf, true));   // row_ror:4
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x122, 0xf, 0xf, true));   // row_ror:2
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x121, 0xf, 0xf, true));   // row_ror:1
}

constexpr int KW_WAVES = 4;
template <int D, int RT>
__global__ __launch_bounds__(WAVE * KW_WAVES) void key_weights_kernel(KeyWeightArgs args) {
  touch_args();
  constexpr int SB = D / FP4_GROUP;
  const AttnArgs& a = args.a;
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int n = lane & 15, g = lane >> 4;
  walk_pieces(a, lane, [&](int r, const ReqWork& w, int kvh, int, int c0, int c1, int, int) {
    const int L = __builtin_amdgcn_readfirstlane(w.len), qlen = __builtin_amdgcn_readfirstlane(w.qlen);
    const int tok = __builtin_amdgcn_readfirstlane(w.tok);
    if (L <= 0) return;
    const int G = a.G, bs = 1 << a.lbs;
    const int* bt = a.block_table + (int64_t)r * a.bt_stride;
    const uint8_t* kbase = (const uint8_t*)a.kc + (int64_t)kvh * a.k_sh;
    const uint8_t* sbase = args.s.k + (int64_t)kvh * args.s.sh;
    const uint32_t koff = n * (int)a.k_sn + (D / 8) * g, soff = n * SB + g * (D / 4) / FP4_GROUP;
    float* wrow = args.w + (int64_t)r * args.w_sr + (int64_t)kvh * args.w_sh;
    for (int row0 = 0; row0 < qlen * G; row0 += 16 * RT) {
      Fp4Query<D> q[RT];
      float f[RT], l2[RT];
      int lim[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int R = row0 + 16 * t + n, rtok = div_group(a, R), rh = R - rtok * G;
        const bool real = rtok < qlen;
        const int64_t at = tok + min(rtok, qlen - 1);
        q[t].load(a.q + at * a.q_st + (int64_t)(kvh * G + rh) * a.q_sh, real, g);
        q[t].make();
        const float l = args.lse[at * args.lse_st + kvh * G + rh];
        // a row whose log-sum-exp is no finite number adds nothing: it saw no key, or its weights are none
        const bool in = real && __builtin_fabsf(l) < INFINITY;
        f[t] = a.sm_log2;
        l2[t] = l * 1.4426950408889634f;
        lim[t] = in ? L - qlen + 1 + rtok : 0;
      }
      struct Tile {
        uint32_t k[2][D / 32];
        uint8_t ks[2];
        float w;      // the running sum of the lane's key (lanes n < 8: key 16 (n / 4) + 4 g + n % 4 of the tile)
      };
      const int own = 16 * (n >> 2) + 4 * g + (n & 3), count = n < 8 ? min(L, args.cols) : 0;
      auto load = [&](Tile& x, int c) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int key = min(c * TILE + 16 * b, (L - 1) & ~15);
          const int p = page_at(bt, 0, 0, key >> a.lbs), pg = (unsigned)p < (unsigned)a.num_blocks ? p : 0, of = key & (bs - 1);
          load_k16<D>(x.k[b], page_base(kbase, pg, (uint32_t)a.k_sb), koff, of * (uint32_t)a.k_sn);
          x.ks[b] = load_at<uint8_t>(page_base(sbase, pg, (uint32_t)args.s.sb), soff, of * SB);
        }
        x.w = c * TILE + own < count ? wrow[c * TILE + own] : 0.f;
      };
      auto add = [&](const Tile& x, int c) {
        float sum[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = 0.f;
        f32x4 z[RT][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) fp4_scores<D, RT>(x.k[b], x.ks[b], q, b, z);
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[t][b][i], f[t], -l2[t]));
              sum[4 * b + i] += c * TILE + 16 * b + 4 * g + i < lim[t] ? p : 0.f;
            }
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float s = sum_row(sum[i]);
          mine = n == i ? s : mine;
        }
        if (c * TILE + own < count) wrow[c * TILE + own] = x.w + mine;
      };
      Tile ring[2];
      int c = c0 + wave;
      if (c < c1) load(ring[0], c);
      for (; c < c1; c += 2 * KW_WAVES) {
        if (c + KW_WAVES < c1) load(ring[1], c + KW_WAVES);
        add(ring[0], c);
        if (c + KW_WAVES >= c1) break;
        if (c + 2 * KW_WAVES < c1) load(ring[0], c + 2 * KW_WAVES);
        add(ring[1], c + KW_WAVES);
      }
    }
  });
}

// ------------------------------------------------------------------------------------------------
// One workgroup per (request, kv head) with n keys of which it may hold m = keep < n. Kept: the last min(recent, m), and of the
// rest those of the m - recent largest sums, ties to the lowest position.
//   select   the sum at which the count is reached, by histograms of 12, 12 and 8 bits of its ordered bits; done as soon as a bin
//            is taken whole, with sums that differ after the second
//   list     the kept positions in order: a wavefront compares its share of the positions, 64 at a time, and lane u keeps the
//            64 answers of the u-th; so counts, ties and places are a scan over lanes and one over wavefronts
//   move     row i takes the row of the i-th kept position, which is i or later: rows are read into registers, in order, a
//            batch at a time, and written after a barrier, so that nothing is overwritten that is still to be read
// One workgroup: a choice needs all of a head's sums, its counts and places stay within the workgroup, and there is one launch.
// (Rows whose source lies at or behind m meet no destination and could be moved by any number of workgroups, in a launch more.)
// 64 requests of 1024 .. 32768 keys, 8 heads, to 2048 each (51 of them have more): 88 .. 103 us from box to box. In a pass that
// finds the rows moved already it takes 42: the choice, from 19 MB of sums that it reads two or three times (select, list) by one
// workgroup for the longest head. The rest are the moves, 225 MB read and written, some 4 TB/s, and the clearing of 16 MB of sums.
// 1 request of 4096 keys to 1024, 4 heads: 16 us, 9 of them the choice: latency of its passes and barriers.
// ------------------------------------------------------------------------------------------------
struct EvictArgs {
  uint8_t* kc;
  uint8_t* vc;
  Fp4Scales s;
  float* w;
  const int* seq_lens;
  const int* keep;
  const int* block_table;
  int* kept;
  int* new_lens;   // NULL: evict_lens_kernel writes them
  int64_t k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, w_sr, w_sh, bt_stride, kp_sr, kp_sh;
  int heads, num_blocks, lbs, cols, bt_cols, kept_cols, recent;
};
constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / WAVE;
constexpr int EV_BINS = 4096;
constexpr int EV_ROWS = 4;      // rows that a thread holds of a batch
constexpr int EV_AHEAD = 8;     // sums that a thread asks for at once
constexpr int EV_LIST = 4096;   // kept positions that are in LDS as well
constexpr int EV_PAGES = 4096;  // page ids that are in LDS as well
constexpr int EV_BLOCKS = WAVE; // blocks of 64 positions whose answers a wavefront holds

// order of the sums as unsigned numbers: NaN the largest, -0 as 0
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : u >> 31 ? ~u : u | 0x80000000u;
}

// request r's keys, and how many of them each kv head may hold
__device__ __forceinline__ int evict_keys_of(const EvictArgs& a, int r) {
  return min(max(a.seq_lens[r], 0), (int)min((int64_t)a.bt_cols << a.lbs, (int64_t)INT32_MAX));
}
__device__ __forceinline__ int evict_most_of(const EvictArgs& a, int r) { return min(max(a.keep[r], 0), a.kept_cols); }

// The lengths in a launch behind evict_kernel's, for a call whose new_lens is its seq_lens or keep: a head's workgroup may start
// after another of its request has ended, and reads both. (Elsewhere the first head's workgroup writes them: a launch less.)
__global__ __launch_bounds__(256) void evict_lens_kernel(EvictArgs a, int* new_lens, int num_seqs) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < num_seqs) new_lens[r] = min(evict_keys_of(a, r), evict_most_of(a, r));
}

template <int D>
__global__ __launch_bounds__(EV_THREADS) void evict_kernel(EvictArgs a) {
  constexpr int SB = D / FP4_GROUP, CH = D / 32;   // exponent bytes, 16-byte chunks of a row's codes
  __shared__ uint32_t bins[EV_BINS];
  __shared__ int list[EV_LIST], pages[EV_PAGES];
  __shared__ uint32_t wsum[2][EV_WAVES];
  __shared__ uint32_t found[3];
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int r = blockIdx.x / a.heads, h = blockIdx.x - r * a.heads;
  const int* bt = a.block_table + (int64_t)r * a.bt_stride;
  const int n = evict_keys_of(a, r), m = evict_most_of(a, r);
  int* kept = a.kept + (int64_t)r * a.kp_sr + (int64_t)h * a.kp_sh;
  float* w = a.w + (int64_t)r * a.w_sr + (int64_t)h * a.w_sh;
  if (a.new_lens && h == 0 && tid == 0) a.new_lens[r] = min(n, m);
  if (n <= m) {   // all of them stay where they are
    for (int i = tid; i < n; i += EV_THREADS) kept[i] = i;
    return;
  }
  const int used = min((n + (1 << a.lbs) - 1) >> a.lbs, EV_PAGES);
  for (int i = tid; i < used; i += EV_THREADS) pages[i] = bt[i];
  const int recent = min(a.recent, m), c = n - recent, need = m - recent;   // candidates: positions 0 .. c - 1; need < c
  // the lanes' sums at from + lane: a descriptor that ends with them, so that what lies behind reads as 0
  const auto desc = __builtin_amdgcn_make_buffer_rsrc(w, 0, 4 * min(c, a.cols), QC_RSRC_WORD3);
  auto sum_at = [&](int i) { return i < a.cols ? w[i] : 0.f; };
  // f(number of the block, its first position, the lane's key) for the blocks of 64 positions from, from + step, .. below end,
  // several loads under way; whole wavefronts
  auto walk = [&](int from, int end, int step, auto&& f) {
    for (int i0 = from, k = 0; i0 < end; i0 += EV_AHEAD * step, k += EV_AHEAD) {
      float x[EV_AHEAD];
#pragma unroll
      for (int u = 0; u < EV_AHEAD; ++u)
        x[u] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(desc, 4 * (i0 + u * step + lane), 0, 0));
#pragma unroll
      for (int u = 0; u < EV_AHEAD; ++u)
        if (i0 + u * step < end) f(k + u, i0 + u * step, ordered(x[u]));
    }
  };
  // sum of the wavefronts' numbers before this one's
  auto before = [&](uint32_t x, int k) {
    if (lane == 0) wsum[k][wave] = x;
    __syncthreads();
    const int incl = wave_incl_sum(lane < EV_WAVES ? (int)wsum[k][lane] : 0);
    return wave ? (uint32_t)__builtin_amdgcn_readlane(incl, wave - 1) : 0u;
  };
  // ---- select ----
  uint32_t edge = 0xffffffffu;   // keys above it are kept, and `ties` of those equal to it
  int ties = 0;
  if (need > 0) {
    uint32_t prefix = 0;
    int left = need;   // still to be found at or below the current bin
    bool whole = false;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 20 : pass == 1 ? 8 : 0, nb = pass == 2 ? 256 : EV_BINS;
      const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xfff00000u : 0xffffff00u;
      for (int i = tid; i < nb; i += EV_THREADS) bins[i] = 0;
      __syncthreads();
      walk(wave * WAVE, c, EV_THREADS, [&](int, int i0, uint32_t key) {
        const bool in = i0 + lane < c && (key & mask) == prefix;
        const uint64_t all = __ballot(in);
        if (all == 0) return;
        // (many alike, zeros of keys that were never looked at: one addition for those of the first lane's bin)
        const int bin = (key >> shift) & (nb - 1), lead = __builtin_ctzll(all), one = __builtin_amdgcn_readlane(bin, lead);
        const uint64_t same = __ballot(in && bin == one);
        if (lane == lead) atomicAdd(&bins[bin], (uint32_t)__builtin_popcountll(same));
        else if (in && bin != one) atomicAdd(&bins[bin], 1u);
      });
      __syncthreads();
      // the bin, counted from the largest, where the count reaches `left`: a thread has `per` bins
      const int per = nb / EV_THREADS > 0 ? nb / EV_THREADS : 1, top = nb - 1 - tid * per;
      uint32_t own = 0;
      if (top >= 0)
        for (int i = 0; i < per; ++i) own += bins[top - i];
      uint32_t incl = (uint32_t)wave_incl_sum((int)own);
      incl += before((uint32_t)__builtin_amdgcn_readlane((int)incl, WAVE - 1), pass & 1);
      if (top >= 0 && (int)incl >= left && (int)(incl - own) < left) {
        uint32_t done = incl - own;
        int b = top;
        while ((int)(done + bins[b]) < left) done += bins[b--];
        found[0] = (uint32_t)b;
        found[1] = done;
        found[2] = bins[b];
      }
      __syncthreads();
      prefix |= found[0] << shift;
      left -= (int)found[1];
      whole = (uint32_t)left == found[2];
      if (whole) break;
    }
    // a bin taken whole: every key from its first on; one number alone (the last pass): `left` of its ties
    edge = whole ? prefix - 1 : prefix;   // (prefix is not 0: a key is at least ordered(-inf))
    ties = whole ? 0 : left;
  }
  // ---- list: wavefront k has the candidates [k, k + 1) * share ----
  const int share = ((c + EV_WAVES - 1) / EV_WAVES + WAVE - 1) / WAVE * WAVE;
  const int from = min(wave * share, c), to = min(from + share, c);
  uint64_t ab = 0, em = 0;   // lane u's: which positions of block u are above the edge, or at it
  auto compare = [&](int i0, int end) {
    ab = em = 0;
    walk(i0, end, WAVE, [&](int k, int p0, uint32_t key) {
      const bool in = p0 + lane < end;
      const uint64_t x = __ballot(in && key > edge), y = ties ? __ballot(in && key == edge) : 0ull;
      ab = lane == k ? x : ab;
      em = lane == k ? y : em;
    });
  };
  constexpr int SPAN = EV_BLOCKS * WAVE;   // positions whose answers fit
  uint32_t cnt = 0, eq = 0;
  if (need > 0)
    for (int i0 = from; i0 < to; i0 += SPAN) {
      compare(i0, min(i0 + SPAN, to));
      cnt += __builtin_popcountll(ab);
      eq += __builtin_popcountll(em);
    }
  cnt = (uint32_t)__builtin_amdgcn_readlane(wave_incl_sum((int)cnt), WAVE - 1);
  eq = (uint32_t)__builtin_amdgcn_readlane(wave_incl_sum((int)eq), WAVE - 1);
  __syncthreads();   // (the last pass's numbers have been read)
  uint32_t at = before(cnt, 0), eq_at = before(eq, 1);
  at += min(eq_at, (uint32_t)ties);
  if (need > 0)
    for (int i0 = from; i0 < to; i0 += SPAN) {
      const int end = min(i0 + SPAN, to);
      if (to - from > SPAN) compare(i0, end);   // (else they are here)
      // of the positions at the edge, those before the `ties`-th
      const int e = __builtin_popcountll(em), e_incl = wave_incl_sum(e);
      int take = min(max(ties - (int)eq_at - (e_incl - e), 0), e);
      uint64_t rest = em;
      if (take < e)
        for (; take > 0; --take) rest &= rest - 1;
      else
        rest = 0;
      const uint64_t chosen = ab | (em & ~rest);
      const int num = __builtin_popcountll(chosen), incl = wave_incl_sum(num), first = (int)at + incl - num;
      for (int u = 0; u * WAVE < end - i0; ++u) {
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)chosen, u), hi = __builtin_amdgcn_readlane((int)(uint32_t)(chosen >> 32), u);
        const int slot = __builtin_amdgcn_readlane(first, u) + (int)__builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
        if ((lane < 32 ? lo >> lane : hi >> (lane - 32)) & 1) {
          const int i = i0 + u * WAVE + lane;
          kept[slot] = i;
          if (slot < EV_LIST) list[slot] = i;
        }
      }
      at += (uint32_t)__builtin_amdgcn_readlane(incl, WAVE - 1);
      eq_at += (uint32_t)__builtin_amdgcn_readlane(e_incl, WAVE - 1);
    }
  for (int i = tid; i < recent; i += EV_THREADS) {
    kept[need + i] = c + i;
    if (need + i < EV_LIST) list[need + i] = c + i;
  }
  __threadfence_block();
  __syncthreads();
  // ---- move ----
  auto page = [&](int i) { return (i >> a.lbs) < EV_PAGES ? pages[i >> a.lbs] : bt[i >> a.lbs]; };
  auto good = [&](int p) { return p >= 0 && p < a.num_blocks; };
  const int bs = 1 << a.lbs;
  constexpr int LPR = 2 * CH, RPB = EV_THREADS / LPR;   // lanes per row (K's chunks, then V's), rows per batch step
  const int ch = tid % LPR, row = tid / LPR;
  const bool v = ch >= CH;
  uint8_t* cache = v ? a.vc + (int64_t)h * a.v_sh : a.kc + (int64_t)h * a.k_sh;
  const int64_t sb = v ? a.v_sb : a.k_sb, sn = v ? a.v_sn : a.k_sn;
  uint8_t* scale = (v ? a.s.v : a.s.k) + (int64_t)h * a.s.sh;
  for (int b0 = 0; b0 < m; b0 += RPB * EV_ROWS) {
    i32x4 code[EV_ROWS];
    uint32_t byte[EV_ROWS];
    float sum[EV_ROWS];
    int src[EV_ROWS];
#pragma unroll
    for (int u = 0; u < EV_ROWS; ++u) {
      const int i = b0 + u * RPB + row;
      src[u] = i >= m ? -1 : i < EV_LIST ? list[i] : kept[i];
      byte[u] = 0;
      sum[u] = 0.f;
      code[u] = i32x4{0, 0, 0, 0};
      if (src[u] > i) {
        const int p = page(src[u]);
        const int64_t pg = good(p) ? p : 0;
        const int of = src[u] & (bs - 1);
        code[u] = *reinterpret_cast<const i32x4*>(cache + pg * sb + of * sn + 16 * (ch % CH));
        byte[u] = scale[pg * a.s.sb + of * SB + ch % CH];
        if (ch == 0) sum[u] = sum_at(src[u]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < EV_ROWS; ++u) {
      const int i = b0 + u * RPB + row;
      if (src[u] <= i) continue;
      const int p = page(i);
      if (ch == 0 && i < a.cols) w[i] = sum[u];
      if (!good(p)) continue;
      const int of = i & (bs - 1);
      *reinterpret_cast<i32x4*>(cache + (int64_t)p * sb + of * sn + 16 * (ch % CH)) = code[u];
      scale[(int64_t)p * a.s.sb + of * SB + ch % CH] = (uint8_t)byte[u];
    }
    __syncthreads();
  }
  for (int i = m + tid; i < min(n, a.cols); i += EV_THREADS) w[i] = 0.f;
}

// rows of `cols` elements, n0 x n1 of them at multiples of s0 and s1, of which no two share an element (any order of the two; a
// workgroup updates each in place)
bool rows_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t cols) {
  if (cols == 0) return true;
  if (n0 <= 1) return n1 <= 1 || s1 >= cols;
  if (n1 <= 1) return s0 >= cols;
  return s0 >= s1 ? s1 >= cols && s0 - cols >= (n1 - 1) * s1 : s0 >= cols && s1 - cols >= (n0 - 1) * s0;
}

}  // namespace

extern "C" {

int kvq_fp4_key_weights(const void* q, int64_t q_st, int64_t q_sh, const uint8_t* k_cache, int64_t k_sb, int64_t k_sn,
                        int64_t k_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_dim,
                        const uint8_t* k_scale, int64_t s_sb, int64_t s_sh, const float* lse, int64_t lse_st, float* weights,
                        int64_t w_sr, int64_t w_sh, int64_t w_cols, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                        const int32_t* block_table, int64_t bt_stride, int64_t num_seqs, int64_t num_q_heads,
                        double softmax_scale, int64_t max_query_len, int64_t qmax, void* stream) {
  const char* nm = "fp4_key_weights";
  if (num_seqs < 0 || num_seqs > INT32_MAX / 4 || max_query_len < 0 || qmax < 1 || w_cols < 0) return fail("%s: bad sizes", nm);
  if (num_seqs == 0 || w_cols == 0) { g_err.clear(); return KVQ_OK; }
  if (!(softmax_scale >= MIN_SOFTMAX_SCALE && softmax_scale <= MAX_SOFTMAX_SCALE))
    return fail("%s: softmax_scale must be positive and finite, from %g to %g", nm, MIN_SOFTMAX_SCALE, MAX_SOFTMAX_SCALE);
  if (const int rc = check_fp4(nm, num_blocks, block_size, num_kv_heads, head_dim, k_cache, k_sb, k_sn, k_sh, k_cache, k_sb,
                               k_sn, k_sh, k_scale, k_scale, s_sb, s_sh)) return rc;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads || num_q_heads > 65535)
    return fail("%s: bad head counts Hq=%lld Hkv=%lld", nm, (long long)num_q_heads, (long long)num_kv_heads);
  if (!q || !lse || !weights || !cu_seqlens_q || !seq_lens || !block_table) return fail("%s: null pointer", nm);
  if (!aligned16(q) || (q_st | q_sh) % 8) return fail("%s: rows must be 16-byte aligned (base pointers and strides)", nm);
  if (!rows_apart(num_seqs, w_sr, num_kv_heads, w_sh, w_cols)) return fail("%s: rows of weights overlap", nm);
  const int G = (int)(num_q_heads / num_kv_heads);
  const int64_t most = std::min<int64_t>(qmax, INT32_MAX / 4);
  if (G * most > INT32_MAX / 4) return fail("%s: too many rows for one kv head", nm);
  const int64_t rows = (int64_t)G * std::min<int64_t>(std::max<int64_t>(max_query_len, 1), most);
  const Tuning tune = read_tuning();
  KeyWeightArgs b;
  b.s = Fp4Scales{const_cast<uint8_t*>(k_scale), nullptr, s_sb, s_sh};
  b.lse = lse; b.w = weights; b.lse_st = lse_st; b.w_sr = w_sr; b.w_sh = w_sh;
  b.cols = (int)std::min<int64_t>(w_cols, INT32_MAX);
  AttnArgs& a = b.a;
  memset(&a, 0, sizeof(a));
  a.q = (const uint16_t*)q; a.kc = (const int8_t*)k_cache;
  a.cu_q = cu_seqlens_q; a.seq_lens = seq_lens; a.block_table = block_table;
  a.q_st = q_st; a.q_sh = q_sh; a.k_sb = k_sb; a.k_sn = k_sn; a.k_sh = k_sh; a.bt_stride = bt_stride;
  a.sm_log2 = (float)(softmax_scale * 1.4426950408889634);
  a.num_blocks = (int)num_blocks; a.lbs = log2i(block_size); a.G = G;
  a.g_inv = G > 1 && (G * most + 64) < (1ll << 32) / G ? (unsigned)(((1ll << 32) + G - 1) / G) : 0u;
  a.qmax = (int)most;
  a.num_seqs = (int)num_seqs; a.hkv = (int)num_kv_heads;
  a.max_splits = 1 << 20; a.cut_rows = INT32_MAX;   // (nothing is kept per piece: any number of them)
  a.rt = (int)((G * most + 15) / 16);               // all of a request's row tiles in one group
  a.ksplit = 1; a.waves = KW_WAVES; a.min_tiles = KW_WAVES; a.coop = 1;
  a.xcd_order = tune.xcd_order ? atoi(tune.xcd_order) : 1;
  a.plan_fast_max = tune.plan_fast_max ? (int)std::max(1ll, std::min(PLAN_FAST_MAX, atoll(tune.plan_fast_max)))
                                       : (int)PLAN_FAST_MAX;
  a.seg_cost = seg_cost_units(tune, 0);
  void (*kern)(KeyWeightArgs) = head_dim == 128
      ? (rows <= 16 ? key_weights_kernel<128, 1> : rows <= 32 ? key_weights_kernel<128, 2> : key_weights_kernel<128, 4>)
      : (rows <= 16 ? key_weights_kernel<64, 1> : rows <= 32 ? key_weights_kernel<64, 2> : key_weights_kernel<64, 4>);
  a.workers = (int)std::max<int64_t>(1, (int64_t)device_cus() * resident_waves((const void*)kern, WAVE * KW_WAVES, 0) / KW_WAVES);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(kern, dim3((unsigned)a.workers), dim3(WAVE * KW_WAVES), 0, st, b);
  return launched(nm);
}

int kvq_fp4_evict(uint8_t* k_cache, int64_t k_sb, int64_t k_sn, int64_t k_sh, uint8_t* v_cache, int64_t v_sb, int64_t v_sn,
                  int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim, uint8_t* k_scale,
                  uint8_t* v_scale, int64_t s_sb, int64_t s_sh, float* weights, int64_t w_sr, int64_t w_sh, int64_t w_cols,
                  const int32_t* seq_lens, const int32_t* keep, int64_t recent, const int32_t* block_table, int64_t bt_stride,
                  int64_t bt_cols, int64_t num_seqs, int32_t* kept, int64_t kp_sr, int64_t kp_sh, int64_t kept_cols,
                  int32_t* new_lens, void* stream) {
  const char* nm = "fp4_evict";
  if (num_seqs < 0 || w_cols < 0 || w_cols > INT32_MAX || bt_cols < 0 || bt_cols > INT32_MAX || kept_cols < 0 ||
      kept_cols > INT32_MAX || recent < 0)
    return fail("%s: bad sizes", nm);
  if (num_seqs == 0) { g_err.clear(); return KVQ_OK; }
  if (const int rc = check_fp4(nm, num_blocks, block_size, num_heads, head_dim, k_cache, k_sb, k_sn, k_sh, v_cache, v_sb, v_sn,
                               v_sh, k_scale, v_scale, s_sb, s_sh)) return rc;
  if (!seq_lens || !keep || !new_lens || (bt_cols && !block_table) || (w_cols && !weights) || (kept_cols && !kept))
    return fail("%s: null pointer", nm);
  if (bt_cols > (1 << 28) / block_size) return fail("%s: tables of more than 2^28 slots", nm);   // (32-bit byte offsets)
  if (num_seqs > INT32_MAX / num_heads) return fail("%s: too many requests and heads for one call", nm);
  if (!rows_apart(num_seqs, w_sr, num_heads, w_sh, w_cols)) return fail("%s: rows of weights overlap", nm);
  if (!rows_apart(num_seqs, kp_sr, num_heads, kp_sh, kept_cols)) return fail("%s: rows of kept overlap", nm);
  // (element r of new_lens follows from element r of the others alone)
  for (const int32_t* in : {seq_lens, keep})
    if (in != new_lens && (uintptr_t)in < (uintptr_t)(new_lens + num_seqs) && (uintptr_t)new_lens < (uintptr_t)(in + num_seqs))
      return fail("%s: new_lens may be seq_lens or keep, but not overlap them otherwise", nm);
  const bool in_place = new_lens == seq_lens || new_lens == keep;
  EvictArgs a;
  a.kc = k_cache; a.vc = v_cache; a.s = Fp4Scales{k_scale, v_scale, s_sb, s_sh}; a.w = weights;
  a.seq_lens = seq_lens; a.keep = keep; a.block_table = block_table; a.kept = kept;
  a.new_lens = in_place ? nullptr : new_lens;
  a.k_sb = k_sb; a.k_sn = k_sn; a.k_sh = k_sh; a.v_sb = v_sb; a.v_sn = v_sn; a.v_sh = v_sh; a.w_sr = w_sr; a.w_sh = w_sh;
  a.bt_stride = bt_stride; a.kp_sr = kp_sr; a.kp_sh = kp_sh;
  a.heads = (int)num_heads; a.num_blocks = (int)num_blocks; a.lbs = log2i(block_size); a.cols = (int)w_cols;
  a.bt_cols = (int)bt_cols; a.kept_cols = (int)kept_cols; a.recent = (int)std::min<int64_t>(recent, INT32_MAX);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(num_seqs * num_heads));
  if (head_dim == 128) hipLaunchKernelGGL(evict_kernel<128>, grid, dim3(EV_THREADS), 0, st, a);
  else hipLaunchKernelGGL(evict_kernel<64>, grid, dim3(EV_THREADS), 0, st, a);
  const int rc = launched(nm);
  if (rc != KVQ_OK || !in_place) return rc;
  hipLaunchKernelGGL(evict_lens_kernel, dim3((unsigned)((num_seqs + 255) / 256)), dim3(256), 0, st, a, new_lens, (int)num_seqs);
  return launched("fp4_evict: lengths");
}

}  // extern "C"
