// Attention of many query rows over a block-scaled INT8 cache: the tile loop that long queries (block_prefill_kernel) and
// verification (block_verify_kernel) share. Part of kvq_int8.hip, included by block_cache.h.
//
// NW wavefronts take 16 NW RB (token, q head) rows of one (request, kv head), RB blocks of 16 rows each, and walk 32-key
// tiles together. Per tile, in the log2 domain of block_attn_kernel:
//   QK  S^T[key][row]  = K . Q16^T   v_mfma_i32_16x16x64_i8, q in two int8 planes: the codes feed the MFMA as they are
//   e   = S sq scale k_scale,  P = 2^(e - m + log2(v_scale)),  l += P / v_scale
//   PV  O^T[chan][row] += V^T . P^T  v_mfma_f32_16x16x32_bf16, P rounded to bf16, V codes converted to bf16 (exactly)
// so that O stays in the accumulators from tile to tile (an int8 product needs 3 operations per channel and row to add
// its integers to O, which at 32 keys a tile costs more than the conversion of V by all the wavefronts). K in int8 also
// halves the LDS reads of the QK operands, of which every wavefront needs the whole tile.
//
// The tiles' codes and scales come by DMA into LDS rings of four slots, up to three tiles ahead; V is converted into one of
// two bf16 stages, a tile ahead of its use; one barrier a tile. The first tile sets each row's reference maximum, later
// tiles only accumulate, and a workgroup in which some row's scores then grew out of range is done again with rescaling
// (prefill_body's scheme).
namespace {

constexpr float Q16_MAX = 16256.f;   // 127 * 128: the hi plane of rint(q / sq) stays an int8

// Bytes e .. e + 3 (e = 4 w) of q as two int8 planes: v = rint(x * inv), v = 128 hi + lo
__device__ __forceinline__ void q_planes4(float x0, float x1, float x2, float x3, float inv, int& hi_out, int& lo_out) {
  const float x[4] = {x0, x1, x2, x3};
  uint32_t hi = 0u, lo = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int v = (int)__builtin_rintf(x[e] * inv), h = (v + 64) >> 7;
    hi |= (uint32_t)(h & 0xff) << (8 * e);
    lo |= (uint32_t)((v - 128 * h) & 0xff) << (8 * e);
  }
  hi_out = (int)hi;
  lo_out = (int)lo;
}

// What the tile loop reads of a call's arguments; kc / vc / ks / vs at the kv head, bt the request's row.
struct RowsView {
  const uint16_t* q;
  const int8_t* kc;
  const int8_t* vc;
  const int* bt;
  const float* ks;
  const float* vs;
  int64_t q_st, q_sh, k_sb, k_sn, v_sb, v_sn, s_sb, s_sg;
  float sm_log2;
  int G, num_blocks, lbs, lg;
};

// A group's rings: the codes and scales of four tiles, V as bf16 of the one computed and the next.
template <int D, int NW>
struct RowsLds {
  static constexpr int SLOTS = 4;
  uint8_t k8[SLOTS][PR_KEYS * D];
  uint8_t v8[SLOTS][PR_KEYS * D];
  uint8_t v16[2][PR_KEYS * 2 * D];
  float sc[SLOTS][NW][WAVE];   // [slot][wavefront]: K and V scale of the half tile that the wavefront's K or V rows lie in
};

// Rows row0 .. of request rows (tok, Q tokens, L keys) over tiles [c_lo, c_hi), whose last key is below kend. fin(rb, t,
// hq, valid, m, l, acc): row block rb's result in the lane of row n, channels 16 tt + 4 g + i in acc[tt][i].
// KW groups of NW wavefronts take the tiles in turn, each with rings of its own, and the first joins their results.
template <int D, int NW, int RB, int KW, typename Fin>
__device__ __forceinline__ void attend_rows(const RowsView& a, RowsLds<D, NW> (&lds_all)[KW], int tok, int Q, int L, int kvh, int row0,
                                            int c_lo, int c_hi, int kend, Fin&& fin) {
  constexpr int KS = D / 64;                // QK steps of 64 channels
  constexpr int VT = D / 16;                // PV channel tiles
  constexpr int CH = D / 8;                 // 16-byte chunks of a bf16 V row
  constexpr int ROWB = 2 * D, TILEB = PR_KEYS * ROWB;
  constexpr int CHR = D / 16;               // 16-byte chunks of an int8 row
  constexpr int TILE8B = PR_KEYS * D, PPM = TILE8B / 1024;   // DMA instructions per int8 matrix and tile
  constexpr int IPW = 2 * PPM / NW, VMT = IPW + 1;           // per wavefront and tile; with the scales
  constexpr int RPI = 1024 / D;             // int8 rows per DMA instruction
  const int lane = threadIdx.x & (WAVE - 1), wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int wave = wave_all % NW, kw = wave_all / NW;
  using Lds = RowsLds<D, NW>;
  Lds& lds = lds_all[kw];
  const int n = lane & 15, g = lane >> 4;
  const int G = a.G;
  const int steps = (c_hi - c_lo + KW - 1) / KW;     // every group's tiles: one past the last is not computed
  auto tile_of = [&](int i) { return c_lo + kw + i * KW; };
  const int wrow0 = row0 + wave * 16 * RB;
  const bool active = wrow0 < Q * G;        // else the wavefront only moves and converts tiles
  // the lane's row of block rb: its token of the request (found again where it is needed, not held through the tiles)
  auto row_of = [&](int rb) {
    int x = wrow0 + n;
    asm volatile("" : "+v"(x));
    return x + 16 * rb;
  };
  const int lim_lo = L - Q + 1 + wrow0 / G;

  // ---- q: two int8 planes per row, rs the factor of its integer scores ----
  i32x4 qop[RB][2][KS];
  float rs[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    u32x4 w[2 * KS];
    const int R = row_of(rb), t = R / G;
    const uint16_t* qp = a.q + (int64_t)(tok + t) * a.q_st + (int64_t)(kvh * G + R - t * G) * a.q_sh + 16 * g;
#pragma unroll
    for (int u = 0; u < 2 * KS; ++u) {
      w[u] = u32x4{0u, 0u, 0u, 0u};
      if (t < Q) w[u] = *reinterpret_cast<const u32x4*>(qp + 64 * (u / 2) + 8 * (u % 2));
    }
    float amax = 0.f;
#pragma unroll
    for (int u = 0; u < 2 * KS; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        amax = __builtin_fmaxf(amax, __builtin_fmaxf(__builtin_fabsf(bf16_lo(w[u][j])), __builtin_fabsf(bf16_hi(w[u][j]))));
    float odd = 0.f;   // 0, or NaN where the row holds a NaN or an infinity: then its output does too
#pragma unroll
    for (int u = 0; u < 2 * KS; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) odd = __builtin_fmaf(bf16_lo(w[u][j]), 0.f, __builtin_fmaf(bf16_hi(w[u][j]), 0.f, odd));
    amax = __builtin_fmaxf(group4_fmax(amax), 1e-30f);
    const float inv = Q16_MAX / amax;
    rs[rb] = amax / Q16_MAX * a.sm_log2 + group4_sum(odd);
#pragma unroll
    for (int u = 0; u < 2 * KS; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        int hi, lo;
        q_planes4(bf16_lo(w[u][2 * j]), bf16_hi(w[u][2 * j]), bf16_lo(w[u][2 * j + 1]), bf16_hi(w[u][2 * j + 1]), inv, hi, lo);
        qop[rb][0][u / 2][2 * (u % 2) + j] = hi;
        qop[rb][1][u / 2][2 * (u % 2) + j] = lo;
      }
  }

  // ---- DMA: wavefront w's instruction i is number j = w + NW i of the tile's 2 PPM: matrix j / PPM (K, V), key rows
  // RPI (j % PPM) .. + RPI - 1, lane l at byte 16 l. All of a wavefront's rows lie in one half tile (16 keys, one page, one
  // scale), of which it also brings the scales. K rows are swizzled (chunk c of row r at c ^ swz_k(r)) for the operand
  // reads below. Rows past the last key are rows of a valid page; the mask drops them. ----
  const int part = wave % PPM, half = RPI * part >= 16 ? 1 : 0;     // (the same for each i: NW is a multiple of PPM)
  static_assert(NW % PPM == 0 && IPW >= 1, "a wavefront's instructions share their rows");
  constexpr int HW1 = D == 128 ? 2 : 1;                             // a wavefront of half 1 (wavefront 0 is of half 0)
  uint32_t o8[IPW];
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const int mat = (wave + NW * i) / PPM, row = RPI * part + lane / CHR, ch = lane % CHR;
    o8[i] = mat ? (uint32_t)((row % 16) * a.v_sn + 16 * ch) : (uint32_t)((row % 16) * a.k_sn + 16 * (ch ^ swz_k<CHR>(row)));
  }
  const float* sbase = (lane & 1) ? a.vs : a.ks;
  const int bsm = (1 << a.lbs) - 1;
  // the id of the page that this wavefront's half of tile c lies in, read a tile before its use; half 1 past the last key
  // takes the last key's page
  auto key_of = [&](int c) { return half ? min(c * PR_KEYS + 16, kend - 1) : c * PR_KEYS; };
  auto page_id = [&](int i) {
    return ((const __attribute__((address_space(4))) int*)a.bt)[key_of(min(tile_of(i), c_hi - 1)) >> a.lbs];
  };
  auto issue = [&](int i, int id) {
    const int c = min(tile_of(i), c_hi - 1);   // past the end: the last tile again
    int p = __builtin_amdgcn_readfirstlane(id);
    p = p >= 0 && p < a.num_blocks ? p : 0;
    const int slot = i & (Lds::SLOTS - 1), o = (c * PR_KEYS + 16 * half) & bsm;
    const float* sp = sbase + ((int64_t)p * a.s_sb + (int64_t)((key_of(c) & bsm) >> a.lg) * a.s_sg);
    __builtin_amdgcn_global_load_lds((const void*)sp, (__attribute__((address_space(3))) void*)(&lds.sc[slot][wave][0]), 4, 0, 0);
#pragma unroll
    for (int k = 0; k < IPW; ++k) {
      const int mat = (wave + NW * k) / PPM;   // uniform
      const int8_t* b = mat ? a.vc + ((int64_t)p * a.v_sb + (int64_t)o * a.v_sn) : a.kc + ((int64_t)p * a.k_sb + (int64_t)o * a.k_sn);
      uint8_t* dst = (mat ? lds.v8[slot] : lds.k8[slot]) + 1024 * part;
      asm volatile("" : "+s"(b));
      asm volatile("" : "+v"(o8[k]));
      __builtin_amdgcn_global_load_lds((const void*)(b + (uint64_t)o8[k]), (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
    }
  };

  // ---- LDS addresses (slot / stage 0) ----
  auto vswz = [](int row) { return (2 * row) % CH; };
  const uint32_t k0 = (uint32_t)(uintptr_t)(&lds.k8[0][0]), s0 = (uint32_t)(uintptr_t)(&lds.sc[0][0][0]);
  const uint32_t v0 = (uint32_t)(uintptr_t)(&lds.v16[0][0]);
  uint32_t kadr[KS], vadr[VT];
#pragma unroll
  for (int s = 0; s < KS; ++s) kadr[s] = k0 + n * D + 16 * ((4 * s + g) ^ swz_k<CHR>(n));   // (row 16 + n: the same swizzle)
  const int vr0 = 4 * g + n / 4;
#pragma unroll
  for (int tt = 0; tt < VT; ++tt) vadr[tt] = v0 + vr0 * ROWB + 16 * ((2 * tt + ((n % 4) >> 1)) ^ vswz(vr0)) + 8 * (n & 1);

  // ---- V codes of tile c -> bf16 stage sb: thread x takes the 8-channel chunk x % CH of rows x / CH + CR i ----
  constexpr int CR = NW * WAVE / CH, NPT = PR_KEYS / CR;
  static_assert((CR % CH == 0 || NPT == 1) && NPT * CR == PR_KEYS && (NPT == 1 || NPT == 2), "conversion share");
  const int cx = wave * WAVE + lane, cc = cx % CH, crow = cx / CH;
  const uint32_t cra = (uint32_t)(uintptr_t)(&lds.v8[0][0]) + crow * D + 8 * cc, cwv = v0 + crow * ROWB + 16 * (cc ^ vswz(crow));
  auto vofs = [](auto st_t) -> uint32_t {
    if constexpr (std::is_same_v<decltype(st_t), int>) return (uint32_t)(st_t * TILEB);
    else return 0u;
  };
  auto iofs = [](auto st_t) -> int {
    if constexpr (std::is_same_v<decltype(st_t), int>) return 0;
    else return decltype(st_t)::value * TILEB;
  };
  u32x2 w[NPT];   // V codes to convert, read with a tile's K operands
  auto convert = [&](auto sb_t) {
    const uint32_t wv = cwv + vofs(sb_t);
    const int WO = iofs(sb_t);
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const u32x4 b = cv8(w[i].x, w[i].y);
      asm volatile("ds_write_b128 %0, %1 offset:%c2" : : "v"(wv), "v"(b), "i"(WO + i * CR * ROWB) : "memory");
    }
  };
  auto read_codes = [&](int i) {
    const uint32_t ra = cra + (i & (Lds::SLOTS - 1)) * TILE8B;
    if constexpr (NPT == 2)
      asm volatile("ds_read_b64 %0, %2\n\tds_read_b64 %1, %2 offset:%c3\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(w[0]), "=&v"(w[NPT - 1]) : "v"(ra), "i"(CR * D) : "memory");
    else
      asm volatile("ds_read_b64 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(w[0]) : "v"(ra) : "memory");
  };

  float m[RB], l[RB];
  f32x4 acc[RB][VT];
  auto clear = [&] {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -1e30f;
      l[rb] = 0.f;
#pragma unroll
      for (int tt = 0; tt < VT; ++tt) acc[rb][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  clear();

  // ---- scores of the group's tile i and what turns them into P: factor f (by row), addend lv = log2(V scale), iv = 1 / V
  // scale. The LDS reads -- the V codes of tile i + 1 with them -- stand in assembly that waits for them alone (as plain
  // loads they would wait for every DMA). ----
  float sc[RB][2][4], f[RB][2], lv[2], iv[2];
  auto scores = [&](int i, auto mask_t) {
    pr_prio<1>();
    const int slot = i & (Lds::SLOTS - 1), n0 = tile_of(i) * PR_KEYS;
    const uint32_t ko = slot * TILE8B, so = s0 + slot * (NW * WAVE * 4);
    const uint32_t ra = cra + ((i + 1) & (Lds::SLOTS - 1)) * TILE8B;
    i32x4 kop[2][KS];
    u32x2 s2[2];
    if constexpr (KS == 2 && NPT == 2)
      asm volatile(
          "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %8 offset:%c12\n\tds_read_b128 %3, %9 offset:%c12\n\t"
          "ds_read_b64 %4, %10\n\tds_read_b64 %5, %10 offset:%c13\n\tds_read_b64 %6, %11\n\tds_read_b64 %7, %11 offset:%c14\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(kop[0][0]), "=&v"(kop[0][KS - 1]), "=&v"(kop[1][0]), "=&v"(kop[1][KS - 1]), "=&v"(s2[0]), "=&v"(s2[1]),
            "=&v"(w[0]), "=&v"(w[NPT - 1])
          : "v"(kadr[0] + ko), "v"(kadr[KS - 1] + ko), "v"(so), "v"(ra), "i"(16 * D), "i"(HW1 * WAVE * 4), "i"(CR * D)
          : "memory");
    else if constexpr (KS == 2)
      asm volatile(
          "ds_read_b128 %0, %7\n\tds_read_b128 %1, %8\n\tds_read_b128 %2, %7 offset:%c11\n\tds_read_b128 %3, %8 offset:%c11\n\t"
          "ds_read_b64 %4, %9\n\tds_read_b64 %5, %9 offset:%c12\n\tds_read_b64 %6, %10\n\ts_waitcnt lgkmcnt(0)"
          : "=&v"(kop[0][0]), "=&v"(kop[0][KS - 1]), "=&v"(kop[1][0]), "=&v"(kop[1][KS - 1]), "=&v"(s2[0]), "=&v"(s2[1]),
            "=&v"(w[0])
          : "v"(kadr[0] + ko), "v"(kadr[KS - 1] + ko), "v"(so), "v"(ra), "i"(16 * D), "i"(HW1 * WAVE * 4)
          : "memory");
    else
      asm volatile(   // (NPT == 1)
          "ds_read_b128 %0, %5\n\tds_read_b128 %1, %5 offset:%c8\n\tds_read_b64 %2, %6\n\tds_read_b64 %3, %6 offset:%c9\n\t"
          "ds_read_b64 %4, %7\n\ts_waitcnt lgkmcnt(0)"
          : "=&v"(kop[0][0]), "=&v"(kop[1][0]), "=&v"(s2[0]), "=&v"(s2[1]), "=&v"(w[0])
          : "v"(kadr[0] + ko), "v"(so), "v"(ra), "i"(16 * D), "i"(HW1 * WAVE * 4)
          : "memory");
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        i32x4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(kop[b][s], qop[rb][0][s], hi, 0, 0, 0);
          lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(kop[b][s], qop[rb][1][s], lo, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[rb][b][i] = (float)((hi[i] << 7) + lo[i]);
      }
    pr_prio<0>();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      auto uniform = [](float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); };
      const float k = uniform(__builtin_fmaxf(__uint_as_float(s2[b].x), MIN_BLOCK_SCALE));
      const float v = __builtin_fmaxf(__uint_as_float(s2[b].y), MIN_V_SCALE);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) f[rb][b] = rs[rb] * k;
      lv[b] = uniform(__builtin_amdgcn_logf(v));
      iv[b] = uniform(__builtin_amdgcn_rcpf(v));
    }
    if (decltype(mask_t)::value && n0 + PR_KEYS > lim_lo) {  // a tile on the causal edge of some row
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int lim = L - Q + 1 + row_of(rb) / G;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          f[rb][b] = f[rb][b] < 1e-37f ? 1e-37f : f[rb][b];   // (a product that underflowed times -inf is no number)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n0 + 16 * b + 4 * g + i >= lim) sc[rb][b][i] = -INFINITY;
        }
      }
    }
  };
  // the reference of the row's largest score in the tile (the 4 lanes of a row agree)
  auto row_top = [&](int rb) {
    float h[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
      h[b] = __builtin_fmaxf(__builtin_fmaxf(sc[rb][b][0], sc[rb][b][1]), __builtin_fmaxf(sc[rb][b][2], sc[rb][b][3])) * f[rb][b];
    return group4_fmax(__builtin_fmaxf(h[0], h[1])) + BLOCK_REF;
  };
  auto softmax_pv = [&](auto st_t) {
    const uint32_t so = vofs(st_t);
    const int SOI = iofs(st_t);
    bf16x8 pop[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float p[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float e0 = lv[b] - m[rb];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rb][b][i], f[rb][b], e0));
      }
      u32x4 pw;
      pw.x = pack_bf16x2_rne(p[0][0], p[0][1]);
      pw.y = pack_bf16x2_rne(p[0][2], p[0][3]);
      pw.z = pack_bf16x2_rne(p[1][0], p[1][1]);
      pw.w = pack_bf16x2_rne(p[1][2], p[1][3]);
      pop[rb] = *reinterpret_cast<bf16x8*>(&pw);
    }
    typedef unsigned long long u64;
#pragma unroll
    for (int t0 = 0; t0 < VT; t0 += 4) {
      u64 lo[4], hi[4];
      asm volatile(
          "ds_read_b64_tr_b16 %0, %8 offset:%c12\n"
          "ds_read_b64_tr_b16 %1, %8 offset:%c13\n"
          "ds_read_b64_tr_b16 %2, %9 offset:%c12\n"
          "ds_read_b64_tr_b16 %3, %9 offset:%c13\n"
          "ds_read_b64_tr_b16 %4, %10 offset:%c12\n"
          "ds_read_b64_tr_b16 %5, %10 offset:%c13\n"
          "ds_read_b64_tr_b16 %6, %11 offset:%c12\n"
          "ds_read_b64_tr_b16 %7, %11 offset:%c13\n"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
          : "v"(vadr[t0] + so), "v"(vadr[t0 + 1] + so), "v"(vadr[t0 + 2] + so), "v"(vadr[t0 + 3] + so), "i"(SOI),
            "i"(SOI + 16 * ROWB)
          : "memory");
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        u32x4 vw = {(uint32_t)lo[u], (uint32_t)(lo[u] >> 32), (uint32_t)hi[u], (uint32_t)(hi[u] >> 32)};
        const bf16x8 vop = *reinterpret_cast<bf16x8*>(&vw);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          acc[rb][t0 + u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, pop[rb], acc[rb][t0 + u], 0, 0, 0);
      }
    }
    // the denominators come from the matrix cores too: row b of this operand picks the keys of half b, so that the sums of
    // the rounded P by half stand in the lanes of group 0
    u32x4 pw = {n == 0 ? 0x3f803f80u : 0u, 0u, n == 1 ? 0x3f803f80u : 0u, 0u};
    pw.y = pw.x;
    pw.w = pw.z;
    const bf16x8 pick = *reinterpret_cast<bf16x8*>(&pw);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const f32x4 sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pick, pop[rb], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      l[rb] = __builtin_fmaf(sum[0], iv[0], __builtin_fmaf(sum[1], iv[1], l[rb]));
    }
  };

  if (c_hi > c_lo) {   // (uniform across the workgroup)
    int ahead = 0;     // page id of the next tile to request
    auto prologue = [&] {
      int id[3];
#pragma unroll
      for (int j = 0; j < 3; ++j) id[j] = page_id(j);
      ahead = page_id(3);
#pragma unroll
      for (int j = 0; j < 3; ++j) issue(j, id[j]);
      wait_vm<VMT * 2>();
      lds_barrier();
      read_codes(0);
      convert(std::integral_constant<int, 0>{});
    };
    // tile i may be computed after this: its codes, scales and bf16 V are there for every wavefront, and so are tile i + 1's
    // codes (converted at the end of the tile); tile i + 3 is requested into the slots of tile i - 1
    auto next_tile = [&](int i) {
      wait_vm<VMT>();
      lds_barrier();
      issue(i + 3, ahead);
      ahead = page_id(i + 4);
    };
    auto mine = [&](int i) { return active && (KW == 1 || tile_of(i) < c_hi); };
    auto tile = [&](int i, auto st_t, auto nx_t, auto mask_t) {   // bf16 stage of tile i, and of tile i + 1
      next_tile(i);
      if (mine(i)) {
        scores(i, mask_t);
        softmax_pv(st_t);
      } else {
        read_codes(i + 1);
      }
      convert(nx_t);   // (past the last tile: old codes, not used)
      __builtin_amdgcn_sched_barrier(0);
    };
    // the group's tiles below J have no key past any row's limit
    const int J = min(steps, (min(c_hi, max(lim_lo, 0) / PR_KEYS) - c_lo - kw + KW - 1) / KW);
    prologue();
    next_tile(0);
    if (mine(0)) {
      scores(0, std::true_type{});
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) m[rb] = __builtin_fmaxf(row_top(rb), -1e30f);
      softmax_pv(std::integral_constant<int, 0>{});
    } else {
      read_codes(1);
    }
    convert(std::integral_constant<int, 1>{});
    int i = 1;
    const std::integral_constant<int, 0> st0;
    const std::integral_constant<int, 1> st1;
    // (J and `active` are the wavefront's own; every wavefront runs each step's barrier and conversion once)
    for (; i + 2 <= J; i += 2) {
      tile(i, st1, st0, std::false_type{});
      tile(i + 1, st0, st1, std::false_type{});
    }
    for (; i < steps; ++i) tile(i, i & 1, (i + 1) & 1, std::true_type{});
    wait_vm<0>();
    bool jump = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      // weights stay in range while a lane's denominator does; times large V scales they may overflow the accumulators
      jump |= !(l[rb] <= PR_FAST_PSUM_MAX);
      float z = 0.f;
#pragma unroll
      for (int tt = 0; tt < VT; ++tt)
#pragma unroll
        for (int e = 0; e < 4; ++e) z = __builtin_fmaf(acc[rb][tt][e], 0.f, z);
      jump |= z != 0.f;
    }
    if (__syncthreads_or(jump)) {
      clear();
      prologue();
      for (i = 0; i < steps; ++i) {
        next_tile(i);
        if (mine(i)) {
          scores(i, std::true_type{});
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const float top = row_top(rb);
            const float mnew = top > m[rb] + PR_SLACK ? top : m[rb];
            const float alpha = __builtin_amdgcn_exp2f(m[rb] - mnew);
            m[rb] = mnew;
            l[rb] *= alpha;
#pragma unroll
            for (int tt = 0; tt < VT; ++tt) acc[rb][tt] *= alpha;
          }
          softmax_pv(i & 1);
        } else {
          read_codes(i + 1);
        }
        convert((i + 1) & 1);
      }
      wait_vm<0>();
      __syncthreads();   // (the rings may be written again)
    }
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) l[rb] = group4_sum(l[rb]);
  if constexpr (KW > 1) {
    // the groups' results, through the rings of the later ones: [field][wavefront][lane]
    static_assert(KW == 2 && sizeof(Lds) >= (4 * VT + 2) * RB * NW * WAVE * sizeof(float), "merge fits the rings");
    float* sl = reinterpret_cast<float*>(&lds_all[1]) + wave * WAVE + lane;
    constexpr int F = NW * WAVE;
    if (kw == 1) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float* x = sl + rb * (4 * VT + 2) * F;
        x[0] = m[rb];
        x[F] = l[rb];
#pragma unroll
        for (int tt = 0; tt < VT; ++tt)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[(2 + 4 * tt + e) * F] = acc[rb][tt][e];
      }
    }
    __syncthreads();
    if (kw == 0) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float* x = sl + rb * (4 * VT + 2) * F;
        const float m1 = x[0], M = __builtin_fmaxf(m[rb], m1);
        const float w0 = __builtin_amdgcn_exp2f(m[rb] - M), w1 = __builtin_amdgcn_exp2f(m1 - M);
        m[rb] = M;
        l[rb] = __builtin_fmaf(w1, x[F], l[rb] * w0);
#pragma unroll
        for (int tt = 0; tt < VT; ++tt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[rb][tt][e] = __builtin_fmaf(w1, x[(2 + 4 * tt + e) * F], acc[rb][tt][e] * w0);
      }
    }
    __syncthreads();   // (the rings may be written again)
    if (kw) return;
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int R = row_of(rb), t = R / G;
    if (L - Q + 1 + t <= 0) {   // a row that sees no key, zero whatever its q holds
      l[rb] = 0.f;
#pragma unroll
      for (int tt = 0; tt < VT; ++tt) acc[rb][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    fin(rb, t, kvh * G + R - t * G, t < Q, m[rb], l[rb], acc[rb]);
  }
}

}  // namespace
