// The ragged attention kernel for wide latents, D = 512 and 576 (ragged.hip includes this inside its
// namespace, after the units).
//
// One workgroup = one unit: 4 waves, one per SIMD with the whole register file (512 VGPRs per lane),
// over tiles of 32 entries held as bf16 in LDS.
//   S^T  wave (eh, hh): entries 16 eh .. + 15 of the tile x rows 32 hh .. + 31 over all channels
//        (v_mfma_f32_16x16x32_bf16, two row groups per K operand read), so a score is whole in the
//        lane that has it;
//   P^T  goes to LDS in bf16 (4 KB a tile, two of them), what the matrix instructions take beside V^T: each
//        weight is off by up to 2^-8 of itself, while the row sums take the unrounded ones in 32 bits.  Against 64
//        bits a result is off by 0.0017 to 0.0022 of its norm, by 0.0017 with unrounded weights (its own bf16);
//        weights as two bf16 terms would double the work of O^T;
//   O^T  wave w: the 16-channel blocks w, w + 4, .. for all 64 rows, one V^T operand read for four
//        row groups.
// One barrier per tile: in iteration u the workgroup runs S(u+1) and PV(u), whose matrix work covers
// the softmax of u+1, while tile u+2 (8-bit entries, dequantized from registers) or u+3 (bf16
// entries, loaded straight into LDS) arrives.
//
// RG: the unit's row groups of 16, 4, or for one new token of up to 16 or 32 heads 1 or 2 (1: the waves of
// hh = 1 repeat the scores of hh = 0).  The matrix work falls with them, and the device's clock need not: 32
// sequences of up to 32k, 8-bit entries, 154 -> 120 us with 16 heads, 158 -> 128 with 32.
//
// What bounds it: the matrix units, shared with one wave's issue of everything else.  8192 tokens x 128 heads of 576
// channels, causal, take 8.3 to 9.2 ms (1190 to 1080 TFLOP/s, by the clock the device holds); 32 sequences of up
// to 32768 x 128 heads, 8-bit, 248 us with the join's 12 (820 TFLOP/s; shares of unequal length, a start of 15
// us), and the launch alone 263 to 305 in twenty calls on end under a kernel trace, presumably by the clock too; one of
// 4096 21 us, a chain: unit 3, q and tables 5, tiles 5, results 4.  Behind a window of 128, 16 heads,
// 23.7 K tokens take 420 us: q 4, tiles 6, results 3 of a unit's 18 us, one after the other.  Pages also cost a
// pause every CT tiles, where the next codes are laid out with no tile in flight.
//
// A tile in LDS is D / 64 columns of 32 rows of 128 bytes: a wave's load instruction (8 rows x 128
// bytes, a lane 16 of them) fills 1 KB of one column, in lane order as the hardware wants it, from
// one address per lane and tile.  The 16-byte piece x of row r sits at slot x ^ wide_swz(r).
//
// Softmax: the exponent's reference of a row is its maximum over the first tile (0 where it sees
// none of that): softmax is exact for any reference as long as nothing overflows or underflows.  A
// weight may then reach 2^(rise of the scores above it): up to kRoomHigh the product with a value
// is within the range of a rescaled softmax; above, the accumulators are looked at after the
// pass.  Where the sum would overflow, or a row that began at 0 stayed far below, the pass is made
// again from the true maxima of a pass over the scores alone.  So no tile waits for the other
// waves' maxima, and O^T is never rescaled.
//
// Entries hidden from a row have weight 0, which does not hide a value that is not finite: a unit of
// several tokens whose result is not finite is computed again one token at a time, each over what it
// sees itself.

// Rows 2 j and 2 j + 1 share a line of banks; rows 16 apart the same slots.  With the bits of j =
// row / 2 reversed, the 16 rows of a K operand's phase lie on 16 distinct bank quads, and so do the
// four rows x 32 bytes of a phase of the transposing reads of V^T.
__device__ __forceinline__ int wide_swz(int row) { return ((row >> 1 & 1) << 2) | ((row >> 2 & 1) << 1) | (row >> 3 & 1); }

template <int FMT, int D>
struct WideLds {
  static constexpr bool kDirect = FMT == kFmtBf16;
  static constexpr int TILE = 64 * D;
  static constexpr int BUFS = kDirect ? 4 : 3;
  static constexpr int PB = BUFS * TILE;           // P^T: 2 x [4 row groups][64 lanes] x 16 bytes
  static constexpr int CT = kDirect ? 40 : 64;     // tiles whose entry codes are laid out at a time (at most 64)
  static constexpr int TAB = PB + 2 * 4096;        // codes; fetched up to 4 tiles past the last
  static constexpr int TABN = (CT + 4) * kTile;
  static constexpr int MASK = TAB + 4 * TABN;      // entries that are there, of each tile
  static constexpr int PMAX = MASK + 4 * 72;       // [2 eh][64]
  static constexpr int LSUM = PMAX + 512;          // [2 eh][64]
  static constexpr int SINK = LSUM + 512;          // [64]
  static constexpr int RED = SINK + 256;
  static constexpr int LDS = RED + 32;
  static_assert(LDS <= 160 * 1024 && sizeof(PlanLds) <= PB, "LDS");
};

// 16 bytes per lane from `at` + 128 J to LDS, column J of a tile: lane l's to byte lds + 4096 J + 16 l.  The
// wave's base is in m0, and the instruction's offset counts for both addresses.
template <int J>
__device__ __forceinline__ void load_column(gptr_t at, uint32_t lds) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2"
               : : "s"(lds), "v"(at), "n"(128 * J), "n"((4096 - 128) * J) : "memory", "scc");
}
template <int J, int N>
__device__ __forceinline__ void load_columns(gptr_t at, uint32_t lds) {
  load_column<J>(at, lds);
  if constexpr (J + 1 < N) load_columns<J + 1, N>(at, lds);
}

// 8-bit entries in flight: one thread's pieces of entry tid / 8.
struct WideRaw {
  u32x4 v[5];
  u32x4 s;  // the entry's four block scales
};

template <int FMT, int D, int NOPE, int RG>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
ragged_wide_kernel(const RaggedParams p) {
  using M = WideLds<FMT, D>;
  constexpr bool kDirect = M::kDirect;
  constexpr int NT = 256, KS = D / 32, NI = D / 64, COL = 4096;
  constexpr int SB = RG == 4 ? 2 : 1, ROWS = 16 * RG;  // row groups of a wave's scores; rows
  constexpr int EB = Layout<FMT, D, NOPE>::kEntryBytes;
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* const tab = reinterpret_cast<uint32_t*>(smem + M::TAB);
  uint32_t* const masks = reinterpret_cast<uint32_t*>(smem + M::MASK);
  float* const pmax = reinterpret_cast<float*>(smem + M::PMAX);
  float* const lsum = reinterpret_cast<float*>(smem + M::LSUM);
  float* const sinks = reinterpret_cast<float*>(smem + M::SINK);
  int* const redo = reinterpret_cast<int*>(smem + M::RED);
  int* const high = redo + 1;
  int* const odd = redo + 2;
  uint8_t* const pbuf = smem + M::PB;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int eh = wave & 1, hh = RG == 1 ? 0 : wave >> 1;
  const int g = lane >> 4, e16 = lane & 15;

  Unit u;
  zero_rows(p, tid);
  if (!find_unit(p, u, smem, tid)) return;  // uniform

  // q: the B operand of S^T (rows 32 hh + 16 b + e16, channels 32 st + 8 g ..) through LDS, from
  // whole lines
  const int rows = u.r1 - u.r0;
  constexpr int QROW = D / 8, QP = (ROWS * QROW + NT - 1) / NT;
  u32x4 qraw[QP];
  if (RG == 4 && p.G == 1 && rows == 64) {  // one run of rows
    const u32x4* const qb = reinterpret_cast<const u32x4*>(p.q + (static_cast<int64_t>(u.t0) * p.H + u.r0) * D);
#pragma unroll
    for (int k = 0; k < QP; ++k) qraw[k] = (qb + NT * k)[tid];
  } else {
#pragma unroll
    for (int k = 0; k < QP; ++k) {
      const int at = tid + NT * k;
      const int r = at / QROW;  // (beyond the unit's rows: its first)
      int head;
      qraw[k] = *reinterpret_cast<const u32x4*>(
          p.q + static_cast<int64_t>(row_at(p, u, u.r0 + (r < rows ? r : 0), head)) * D + 8 * (at - r * QROW));
    }
  }
  const int tok0 = p.by_heads(u.r0), tok1 = p.by_heads(u.r1 - 1) + 1;
  const int shift = u.len - u.n;
  int share_lo, share_hi;
  unit_range(p, u, tok0, tok1, share_lo, share_hi);
  int tok_b[SB];  // the tokens of this lane's rows
#pragma unroll
  for (int b = 0; b < SB; ++b) {
    const int r = u.r0 + 16 * (SB * hh + b) + e16;
    tok_b[b] = p.by_heads(r < u.r1 ? r : u.r0);
  }
  float sink = -__builtin_huge_valf();  // of row tid, kept in LDS for the end
  if (p.sinks && tid < 64) {
    int head;
    row_at(p, u, tid < rows ? u.r0 + tid : u.r0, head);
    sink = p.sinks[head];
  }

  // ---- addresses -------------------------------------------------------------------------
  const int te = tid >> 3, tj = tid & 7;
  const uint32_t k_even = static_cast<uint32_t>((16 * eh + e16) * 128 + 16 * (g ^ wide_swz(e16)));
  const uint32_t k_odd = k_even ^ 64u;
  const int vrow = 4 * g + (e16 >> 2);
  const uint32_t v_at = static_cast<uint32_t>(vrow * 128 + 16 * ((2 * wave + ((e16 >> 1) & 1)) ^ wide_swz(vrow)) + 8 * (e16 & 1));
  // 8-bit entries: this thread's code pieces are pairs of bf16 pieces of columns tj / 4 + 2 k
  const uint32_t st_at = static_cast<uint32_t>(COL * (tj >> 2) + te * 128 + 16 * ((2 * (tj & 3)) ^ wide_swz(te)));
  const uint32_t rope_at = static_cast<uint32_t>(COL * 8 + te * 128 + 16 * (tj ^ wide_swz(te)));
  const uint64_t pool_piece = reinterpret_cast<uint64_t>(p.entries) +
                              (p.tables ? 0 : static_cast<uint64_t>(u.t0) * p.entry_stride + static_cast<uint64_t>(u.g) * EB) +
                              16u * (kDirect ? tj ^ wide_swz(te) : tj);
  const uint32_t entry_stride = static_cast<uint32_t>(p.entry_stride);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)smem)) + 1024u * wave;
  const bool paged = p.tables != nullptr;

  auto entry_at = [&](uint32_t code) __attribute__((always_inline)) -> gptr_t {
    return (gptr_t)(pool_piece + static_cast<uint64_t>(code) * entry_stride);
  };
  auto fetch_part = [&](gptr_t e, WideRaw& r, int k) __attribute__((always_inline)) {
    if (k < 4) r.v[k] = gload<u32x4>(e + 128 * k);
    if (k == 4) r.v[4] = gload<u32x4>(e + NOPE + 16);
    if (k == 5) r.s = gload<u32x4>(e - 16 * tj + NOPE);
  };
  // part k (of 9) of a fetched tile into LDS: parts 2 q, 2 q + 1 are the halves of code piece q (16
  // codes: two bf16 pieces), part 8 the rope slice
  auto store_part = [&](uint8_t* t, const WideRaw& r, int k) __attribute__((always_inline)) {
    if (k < 8) {
      const int q = k >> 1;
      const uint2 codes = k & 1 ? uint2{r.v[q].z, r.v[q].w} : uint2{r.v[q].x, r.v[q].y};
      *reinterpret_cast<uint4*>(t + ((k & 1 ? st_at ^ 16u : st_at) + 2 * COL * q)) = dequant_fp8x8_bf16(codes, __uint_as_float(r.s[q]));
    } else {
      *reinterpret_cast<uint4*>(t + rope_at) = uint4{r.v[4].x, r.v[4].y, r.v[4].z, r.v[4].w};
    }
  };
  auto k_frag = [&](const uint8_t* t, int st) __attribute__((always_inline)) -> v8bf {
    return __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(t + (st & 1 ? k_odd : k_even) + COL * (st >> 1)));
  };
  auto tile_at = [&](int i) __attribute__((always_inline)) -> uint32_t { return static_cast<uint32_t>(i) * M::TILE; };

  float m4[RG], m_own[SB], l_own[SB], m_seen[SB];
  v4f acc[NI][RG];
  v8bf qf[KS][SB];
  v4f s_acc[SB];
  WideRaw raw[2];

  int lo = 0, hi = 0;       // the pass's entries: positions lo .. hi - 1
  int c0 = 0, nt = 0;       // the chunk at hand: its first entry (from lo), its tiles
  int row_lo[SB], row_span[SB];  // of this lane's rows, entries seen, from lo
  int full_lo = 0, full_hi = 0;  // tiles (from lo) of which every row sees every entry
  // the entry that a lane fetches for tile t of the chunk: past the end of the range its last one
  auto code_of = [&](int t) __attribute__((always_inline)) -> uint32_t {
    if (paged) return tab[t * kTile + te];
    const int v = c0 + t * kTile + te;
    return static_cast<uint32_t>(lo + (v < hi - lo ? v : hi - lo - 1));
  };
  auto direct = [&](gptr_t e, uint32_t buf) __attribute__((always_inline)) {
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds0 + buf);
    load_columns<0, NI>(e, at);
  };
  // a whole tile into a buffer, waited for by nobody yet
  auto bring = [&](int t, uint32_t buf) __attribute__((always_inline)) {
    const gptr_t e = entry_at(code_of(t));
    if constexpr (kDirect) {
      direct(e, buf);
    } else {
#pragma unroll
      for (int k = 0; k < 6; ++k) fetch_part(e, raw[0], k);
#pragma unroll
      for (int k = 0; k < 9; ++k) store_part(smem + buf, raw[0], k);
    }
  };
  auto landed = [&]() __attribute__((always_inline)) {
    if constexpr (kDirect) asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    lds_barrier();
  };

  // The entry codes of the chunk's tiles and which entries are there; false: none is.  An empty slot
  // is fetched as another entry that is there (its weight is 0).
  int first = 0, last = 0;  // the chunk's first and last tile that hold an entry
  auto lay_out = [&]() __attribute__((always_inline)) -> bool {
    const int left = hi - lo - c0;
    nt = (left < M::CT * kTile ? left + kTile - 1 : M::CT * kTile) / kTile;
    if (!paged) {
      nt = (left + kTile - 1) / kTile;
      first = 0;
      last = nt - 1;
      return left > 0;
    }
    constexpr uint32_t kEmpty = 0xffffffffu;
    const int n_tab = (nt + 4) * kTile;
    for (int e0 = 0; e0 < n_tab; e0 += NT) {
      const int e = e0 + tid;
      uint32_t code = kEmpty;
      if (e < nt * kTile && e < left) {
        code = static_cast<uint32_t>(pool_entry(p, u, lo + c0 + e));  // -1: kEmpty
      }
      const uint64_t bal = __ballot(code != kEmpty);
      if (e < n_tab) {
        tab[e] = code;
        if ((lane & 31) == 0) masks[e / kTile] = static_cast<uint32_t>(lane ? bal >> 32 : bal);
      }
    }
    lds_barrier();
    const uint64_t some = __ballot(lane < nt && masks[lane < nt ? lane : 0] != 0u);
    if (some == 0) {
      lds_barrier();  // the next chunk's codes come here
      return false;
    }
    first = __builtin_ctzll(some);
    last = 63 - __builtin_clzll(some);
    const uint32_t any = tab[first * kTile + __builtin_ctz(masks[first])];
    for (int e = tid; e < n_tab; e += NT)
      if (tab[e] == kEmpty) tab[e] = any;
    lds_barrier();
    return true;
  };

  // whether tile t of the chunk is seen whole by every row
  auto whole = [&](int t) __attribute__((always_inline)) -> bool {
    const int at = c0 / kTile + t;
    return at >= full_lo && at < full_hi && (!paged || __builtin_amdgcn_readfirstlane(masks[t]) == 0xffffffffu);
  };
  // entry r (of 4) of this lane in tile t, for row group b
  auto sees = [&](int t, uint32_t bits, int b, int r) __attribute__((always_inline)) -> bool {
    const int v = c0 + t * kTile + 16 * eh + 4 * g + r;
    return ((bits >> (16 * eh + 4 * g + r)) & 1u) != 0u && static_cast<uint32_t>(v - row_lo[b]) < static_cast<uint32_t>(row_span[b]);
  };
  auto scores = [&](int t, float (&v)[SB][4]) __attribute__((always_inline)) {
    const uint32_t bits = paged ? masks[t] : 0xffffffffu;
#pragma unroll
    for (int b = 0; b < SB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[b][r] = sees(t, bits, b, r) ? s_acc[b][r] * p.scale_log2 : -__builtin_huge_valf();
  };
  auto s_tile = [&](const uint8_t* kt) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < SB; ++b) s_acc[b] = v4f{};
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const v8bf kf = k_frag(kt, st);
#pragma unroll
      for (int b = 0; b < SB; ++b) s_acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[st][b], s_acc[b], 0, 0, 0);
    }
  };
  auto max4 = [](const float (&v)[4]) __attribute__((always_inline)) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); };
  auto row_max = [](float x) __attribute__((always_inline)) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
  };
  // the rows' maxima over both entry halves into m4 / m_own (one barrier); 0 for a row without one
  auto agree_max = [&](float (&t)[SB]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < SB; ++b) {
      t[b] = row_max(t[b]);
      if (g == 0) pmax[eh * 64 + 16 * (SB * hh + b) + e16] = t[b];
    }
    lds_barrier();
    auto known = [](float a, float b) { const float m = fmaxf(a, b); return m == -__builtin_huge_valf() ? 0.0f : m; };
#pragma unroll
    for (int hg = 0; hg < RG; ++hg) m4[hg] = known(pmax[16 * hg + e16], pmax[64 + 16 * hg + e16]);
#pragma unroll
    for (int b = 0; b < SB; ++b) m_own[b] = known(pmax[16 * (SB * hh + b) + e16], pmax[64 + 16 * (SB * hh + b) + e16]);
  };
  auto put_p = [&](int t, int b, uint2 w) __attribute__((always_inline)) {
    *reinterpret_cast<uint2*>(pbuf + (t & 1) * 4096 + 1024 * (SB * hh + b) + 16 * lane + 8 * eh) = w;
  };
  auto read_v = [&](const uint8_t* vt, int i, v4s (&va)[2]) __attribute__((always_inline)) {
    const uint8_t* tp = vt + v_at + COL * i;
    va[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_v4s(tp));
    va[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_v4s(tp + 2048));
  };

  // the chunk's first two tiles requested
  auto ask = [&]() __attribute__((always_inline)) {
    const gptr_t a = entry_at(code_of(first)), b = entry_at(code_of(first < last ? first + 1 : first));
    if constexpr (kDirect) {
      direct(a, tile_at(0));
      direct(b, tile_at(1));
    } else {
#pragma unroll
      for (int k = 0; k < 6; ++k) fetch_part(a, raw[0], k);
#pragma unroll
      for (int k = 0; k < 6; ++k) fetch_part(b, raw[1], k);
    }
  };

  // ---- one chunk of the pass: tiles `first` .. `last`, the first two asked for ------------------------------------------
  // begin: the rows' references come from its first tile
  auto chunk = [&](bool begin) __attribute__((always_inline)) {
    const int t0 = first, n = last + 1;
    if constexpr (kDirect) {
      direct(entry_at(code_of(t0 + 2 < n ? t0 + 2 : t0)), tile_at(2));
      if constexpr (NI > 8) asm volatile("s_waitcnt vmcnt(18)" : : : "memory");
      else asm volatile("s_waitcnt vmcnt(16)" : : : "memory");
    } else {
#pragma unroll
      for (int k = 0; k < 9; ++k) store_part(smem, raw[0], k);
      if (n - t0 > 1) {
#pragma unroll
        for (int k = 0; k < 9; ++k) store_part(smem + M::TILE, raw[1], k);
        const int second = (n - 1 - t0) & 1;  // set 1 is stored first then
#pragma unroll
        for (int k = 0; k < 6; ++k) fetch_part(entry_at(code_of(t0 + 2 + second)), raw[0], k);
#pragma unroll
        for (int k = 0; k < 6; ++k) fetch_part(entry_at(code_of(t0 + 3 - second)), raw[1], k);
      }
    }
    lds_barrier();
    s_tile(smem);
    {
      float v[SB][4];
      scores(t0, v);
      if (begin) {
        float top[SB];
#pragma unroll
        for (int b = 0; b < SB; ++b) top[b] = max4(v[b]);
        agree_max(top);
      }
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = __builtin_amdgcn_exp2f(v[b][r] - m_own[b]);
        l_own[b] = l_own[b] + ((w[0] + w[1]) + (w[2] + w[3]));
        put_p(t0, b, uint2{pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])});
        if (!begin) m_seen[b] = fmaxf(m_seen[b], max4(v[b]) / p.scale_log2);  // (this tile's s_acc has the hidden entries too)
      }
    }
    uint32_t at_v = 0, at_k = tile_at(1), at_n = tile_at(2), at_w = tile_at(kDirect ? 3 : 2);
    // One wave per SIMD issues in order, so the iteration is laid out by hand: every LDS operand
    // is requested several matrix instructions before its use (K six steps, V^T four blocks),
    // the softmax, the stores and the loads are spread one slice after each matrix instruction,
    // whose 16 cycles they fill, and the last two blocks of PV(u-1), whose operands are in
    // registers by then, follow the barrier and cover the first reads of K.
    constexpr int AH = 6, VH = 4, LATE = 2;
    v4s va[VH + 1][2];
    v8bf pf[RG];
    auto pv_block = [&](int i, auto&& fill) __attribute__((always_inline)) {
      const v4s a = va[i % (VH + 1)][0], b = va[i % (VH + 1)][1];
      const v8bf vf = __builtin_bit_cast(v8bf, v8s{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
#pragma unroll
      for (int hg = 0; hg < 4; ++hg) {
        if (hg < RG) acc[i][hg < RG ? hg : 0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[hg < RG ? hg : 0], acc[i][hg < RG ? hg : 0], 0, 0, 0);
        fill(hg);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto read_p = [&](int t, int hg) __attribute__((always_inline)) {
      pf[hg] = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(pbuf + (t & 1) * 4096 + 1024 * hg + 16 * lane));
    };
#pragma unroll
    for (int i = 0; i <= VH; ++i) va[i][0] = va[i][1] = v4s{0, 0, 0, 0};
#pragma unroll
    for (int hg = 0; hg < RG; ++hg) pf[hg] = __builtin_bit_cast(v8bf, v4i{0, 0, 0, 0});
    if constexpr (kDirect) {  // tile t0 + 1
      if constexpr (NI > 8) asm volatile("s_waitcnt vmcnt(9)" : : : "memory");
      else asm volatile("s_waitcnt vmcnt(8)" : : : "memory");
    }
    lds_barrier();  // P(t0) complete
    auto step = [&](int t, WideRaw& r) __attribute__((always_inline)) {
      // the barrier before: P(t) and tile t+1 complete; tile t-1 is read no more
      const uint8_t* vt = smem + at_v;
      const uint8_t* kt = smem + at_k;
      uint8_t* const wt = smem + at_w;
      v8bf kf[AH];
#pragma unroll
      for (int i = 0; i < AH; ++i) kf[i] = k_frag(kt, i);
      uint32_t code;
      if constexpr (kDirect) code = code_of(t + 3 < n ? t + 3 : n - 1);
      else code = tab[(t + 4) * kTile + te];
      // hidden entries start from kHidden instead of 0, so that no score needs a test
      v4f init[SB];
#pragma unroll
      for (int b = 0; b < SB; ++b) init[b] = v4f{};
      if (!whole(t + 1)) {
        const uint32_t bits = paged ? masks[t + 1] : 0xffffffffu;
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
          for (int k = 0; k < 4; ++k) init[b][k] = sees(t + 1, bits, b, k) ? 0.0f : kHidden;
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = NI - LATE; i < NI; ++i) pv_block(i, [](int) {});
      uint64_t next = 0;
      uint32_t to = 0;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const v8bf cur = kf[st % AH];
        s_acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cur, qf[st][0], st == 0 ? init[0] : s_acc[0], 0, 0, 0);
        if (st + AH < KS) kf[st % AH] = k_frag(kt, st + AH);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (SB > 1) s_acc[SB - 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cur, qf[st][SB - 1], st == 0 ? init[SB - 1] : s_acc[SB - 1], 0, 0, 0);
        if (st == 2) next = pool_piece + static_cast<uint64_t>(code) * entry_stride;
        if (st >= 8 && st < 8 + RG) read_p(t, st - 8);
        if (st >= KS - VH - 2 && st < KS - 2) read_v(vt, st - (KS - VH - 2), va[st - (KS - VH - 2)]);
        if constexpr (!kDirect) {
          if (st >= KS - 2) store_part(wt, r, 7 + st - (KS - 2));
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kDirect) {  // one of tile t + 3's loads
          if (st == 2) to = __builtin_amdgcn_readfirstlane(lds0 + at_w);
          if (st >= 3 && st < 3 + NI) {
            const gptr_t e = (gptr_t)next;
            if (st == 3) load_column<0>(e, to);
            if (st == 4) load_column<1>(e, to);
            if (st == 5) load_column<2>(e, to);
            if (st == 6) load_column<3>(e, to);
            if (st == 7) load_column<4>(e, to);
            if (st == 8) load_column<5>(e, to);
            if (st == 9) load_column<6>(e, to);
            if (st == 10) load_column<7>(e, to);
            if (NI > 8 && st == 11) load_column<(NI > 8 ? 8 : 0)>(e, to);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      const gptr_t from = (gptr_t)next;
      float v[SB][4], pr[SB][4];
      // slice k of what fills the matrix instructions of PV
      auto slice = [&](int k) __attribute__((always_inline)) {
        if (k >= 2 && k < 10) {
          const int b = (k - 2) >> 2, j = (k - 2) & 3;
          if (b >= SB) return;
          v[b][j] = s_acc[b][j];
          pr[b][j] = __builtin_fmaf(v[b][j], p.scale_log2, -m_own[b]);
        } else if (k >= 10 && k < 18) {  // v_exp_f32 directly: results below 2^-126 may flush to 0
          const int b = (k - 10) >> 2, j = (k - 10) & 3;
          if (b >= SB) return;
          pr[b][j] = __builtin_amdgcn_exp2f(pr[b][j]);
        } else if (k == 18 || k == 19) {
          const int b = k - 18;
          if (b >= SB) return;
          put_p(t + 1, b, uint2{pack_bf16x2(pr[b][0], pr[b][1]), pack_bf16x2(pr[b][2], pr[b][3])});
        } else if (k >= 20 && k < 22) {
          const int b = k - 20;
          if (b >= SB) return;
          l_own[b] = l_own[b] + ((pr[b][0] + pr[b][1]) + (pr[b][2] + pr[b][3]));
        } else if (k >= 22 && k < 24) {
          const int b = k - 22;
          if (b >= SB) return;
          m_seen[b] = fmaxf(fmaxf(m_seen[b], v[b][0]), fmaxf(v[b][1], fmaxf(v[b][2], v[b][3])));
        }
      };
#pragma unroll
      for (int i = 0; i < NI - LATE; ++i)
        pv_block(i, [&](int hg) __attribute__((always_inline)) {
          if (hg == 0 && i + VH < NI) read_v(vt, i + VH, va[(i + VH) % (VH + 1)]);
          slice(4 * i + hg);
          if constexpr (!kDirect) {
            if (hg == 1) store_part(wt, r, i);
            // a piece is requested again, for tile t + 4, once all of it is stored
            if (hg == 3 && (i & 1)) fetch_part(from, r, i >> 1);
            if (hg >= 2 && i == 6) fetch_part(from, r, hg == 2 ? 3 : 5);
            if (hg == 3 && i == 0) fetch_part(from, r, 4);
          }
        });
      if constexpr (kDirect) {  // tile t + 2; the loads of t + 3 stay in flight
        if constexpr (NI > 8) asm volatile("s_waitcnt vmcnt(9)" : : : "memory");
        else asm volatile("s_waitcnt vmcnt(8)" : : : "memory");
      }
      lds_barrier();
      const uint32_t done = at_v;
      at_v = at_k;
      if constexpr (kDirect) {
        at_k = at_n;
        at_n = at_w;
      } else {
        at_k = at_w;
      }
      at_w = done;
    };
    int t = t0;
    if constexpr (kDirect) {
#pragma unroll 1
      for (; t + 1 < n; ++t) step(t, raw[0]);
    } else {
      // an odd number of steps takes one first: the loop is two steps long (two sets of loads in
      // flight) with a single exit, or every accumulator would be copied between its ends
      if ((n - 1 - t0) & 1) step(t++, raw[1]);
#pragma unroll 1
      for (; t + 1 < n; t += 2) {
        step(t, raw[0]);
        step(t + 1, raw[1]);
      }
    }
    {  // the rest of the last but one, and the last tile
      const uint8_t* vt = smem + at_v;
#pragma unroll
      for (int i = NI - LATE; i < NI; ++i) pv_block(i, [](int) {});
#pragma unroll
      for (int hg = 0; hg < RG; ++hg) read_p(n - 1, hg);
#pragma unroll
      for (int i = 0; i < VH; ++i) read_v(vt, i, va[i]);
#pragma unroll
      for (int i = 0; i < NI; ++i)
        pv_block(i, [&](int hg) __attribute__((always_inline)) {
          if (hg == 0 && i + VH < NI) read_v(vt, i + VH, va[(i + VH) % (VH + 1)]);
        });
    }
    landed();  // the LDS is free again
  };

  // the entries that tokens sub0 .. sub1 - 1 see of this unit's share, and what the rows see of them
  int sub0 = tok0, sub1 = tok1;
  auto set_range = [&]() __attribute__((always_inline)) {
    token_range(p, u, sub0, sub1, lo, hi);
    lo = lo > share_lo ? lo : share_lo;
    hi = hi < share_hi ? hi : share_hi;
    if (hi < lo) hi = lo;
    int most_lo = lo, least_hi = hi;
    if (!p.idx) {
      most_lo = clamp32(shift + sub1 - p.window, lo, 0x7fffffff - kTile);
      least_hi = shift + sub0 + 1 < hi ? shift + sub0 + 1 : hi;
    }
    full_lo = (most_lo - lo + kTile - 1) / kTile;
    full_hi = least_hi > lo ? (least_hi - lo) / kTile : 0;
#pragma unroll
    for (int b = 0; b < SB; ++b) {
      int a = lo, z = hi;
      if (!p.idx) {
        const int pos = shift + tok_b[b];
        if (pos - p.window + 1 > a) a = pos - p.window + 1;
        if (pos + 1 < z) z = pos + 1;
      }
      row_lo[b] = a - lo;
      row_span[b] = z > a ? z - a : 0;
    }
  };

  // The first chunk is laid out and its first tiles requested while q arrives; then q goes into its
  // operand's layout through the LDS behind those tiles.  (One after the other this took 17 us of a
  // split call over 4096 entries.)
  set_range();
  const bool none = !(lo < hi && lay_out());  // uniform
  if (!none) ask();
  {
    constexpr int QPITCH = 2 * D + 16;  // the pad spreads 16 rows' pieces over the banks
    constexpr int QB = M::PB + 2 * 4096 - ROWS * QPITCH;
    static_assert(QB >= (kDirect ? 2 * M::TILE : 0), "q behind the first tiles");
#pragma unroll
    for (int k = 0; k < QP; ++k) {
      const int at = tid + NT * k;
      const int r = at / QROW;
      if (ROWS * QROW % NT == 0 || at < ROWS * QROW)
        *reinterpret_cast<u32x4*>(smem + QB + r * QPITCH + 16 * (at - r * QROW)) = qraw[k];
    }
    if (tid < 64) sinks[tid] = sink;
    lds_barrier();
#pragma unroll
    for (int b = 0; b < SB; ++b)
#pragma unroll
      for (int st = 0; st < KS; ++st)
        qf[st][b] = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(smem + QB + (16 * (SB * hh + b) + e16) * QPITCH + 64 * st + 16 * g));
    lds_barrier();
    // the first query fragments live in accumulation registers beside O^T, which the matrix
    // instructions read directly; left to itself the compiler spills
#pragma unroll
    for (int st = 0; st < KS - 6; ++st)
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        v4i x = __builtin_bit_cast(v4i, qf[st][b]);
        asm volatile("" : "+a"(x));
        qf[st][b] = __builtin_bit_cast(v8bf, x);
      }
  }

  // ---- the passes --------------------------------------------------------------------------
  // The q rows of the unit that this compute unit is likely to be given next (blocks go down the rows,
  // 256 compute units ahead) are asked into the L2, a word of each line, while the result leaves.  In units
  // of few tiles only: 9 prompts of 16 heads behind a window of 128 take 449 us without, 424 with; one
  // of 8192 tokens x 128 heads, whose units are long, gains nothing.
  constexpr int LINES = (64 * D * 2 / 128 + NT - 1) / NT;
  uint32_t hint[LINES];
#pragma unroll
  for (int k = 0; k < LINES; ++k) hint[k] = 0;
  auto look_ahead = [&]() __attribute__((always_inline)) {
    const int64_t row = static_cast<int64_t>(u.t0) * p.H + u.r0 - 256 * 64;
    if (RG < 4 || !p.cu || p.slots || p.G != 1 || row < 0 || hi - lo > 32 * kTile) return;
    int line = tid;
    asm volatile("" : "+v"(line));
    const uint8_t* const at = reinterpret_cast<const uint8_t*>(p.q + row * D);
#pragma unroll
    for (int k = 0; k < LINES; ++k)
      if (64 * D * 2 / 128 % NT == 0 || line + NT * k < 64 * D * 2 / 128)
        hint[k] = *reinterpret_cast<const uint32_t*>(at + 128 * (line + NT * k));
  };
  bool strict = false, at_start = true;
  while (true) {
    if (!at_start) set_range();
    float l4[RG];
    int e4[RG];
    for (bool given = false;; given = true) {
      if (tid == 0) *redo = *high = *odd = 0;
      bool begun = false;
      if (given) {  // the true maxima of every row: scores only
        float top[SB];
#pragma unroll
        for (int b = 0; b < SB; ++b) top[b] = -__builtin_huge_valf();
        for (c0 = 0; c0 < hi - lo; c0 += nt * kTile) {
          if (!lay_out()) continue;
#pragma unroll 1
          for (int t = first; t <= last; ++t) {
            bring(t, 0);
            landed();
            s_tile(smem);
            float v[SB][4];
            scores(t, v);
#pragma unroll
            for (int b = 0; b < SB; ++b) top[b] = fmaxf(top[b], max4(v[b]));
            lds_barrier();
          }
        }
        agree_max(top);
        lds_barrier();
        begun = true;
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int hg = 0; hg < RG; ++hg) acc[i][hg] = v4f{};
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        l_own[b] = 0.0f;
        m_seen[b] = -__builtin_huge_valf();
        if (!begun) m_own[b] = 0.0f;
      }
      if (!begun) {
#pragma unroll
        for (int hg = 0; hg < RG; ++hg) m4[hg] = 0.0f;
      }
      for (c0 = 0; c0 < hi - lo; c0 += nt * kTile) {
        const bool ready = at_start && c0 == 0;
        if (ready ? none : !lay_out()) continue;
        if (!ready) ask();
        chunk(!begun);
        begun = true;
      }
      if (at_start) look_ahead();
      at_start = false;
      // each row's sum: its four lanes, then the two entry halves
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        l_own[b] = l_own[b] + __shfl_xor(l_own[b], 16, 64);
        l_own[b] = l_own[b] + __shfl_xor(l_own[b], 32, 64);
        if (g == 0) lsum[eh * 64 + 16 * (SB * hh + b) + e16] = l_own[b];
      }
      if (!given) {  // (zero before the barriers of the pass; without an entry nothing is set)
#pragma unroll
        for (int b = 0; b < SB; ++b) {
          const float top = m_seen[b] * p.scale_log2, rise = top - m_own[b];
          if (rise > kRoomHigh) *high = 1;
          if (rise > kRoomAbove || (rise < kRoomBelow && m_own[b] == 0.0f && m_seen[b] > 0.5f * kHidden)) *redo = 1;
        }
      }
      lds_barrier();
#pragma unroll
      for (int hg = 0; hg < RG; ++hg) l4[hg] = lsum[16 * hg + e16] + lsum[64 + 16 * hg + e16];
      if (__builtin_expect(!given && *high != 0, 0)) {  // uniform
        // O^T through the tiles' place, half of it at a time, each lane its own: a few stores and a
        // short loop
        float any_bad = 0.0f;  // NaN if an accumulator is not finite
        v4f* const slot = reinterpret_cast<v4f*>(smem) + tid;
        static_assert(2 * NI * NT * 16 <= M::PB, "half of O^T in the tiles' place");
#pragma unroll
        for (int h0 = 0; h0 < RG; h0 += 2) {
          constexpr int W = RG < 2 ? RG : 2;  // row groups at a time
#pragma unroll
          for (int k = 0; k < W * NI; ++k) slot[k * NT] = acc[k / W][h0 + k % W];
#pragma unroll 1
          for (int k = 0; k < W * NI; ++k) {
            const v4f x = slot[k * NT];
#pragma unroll
            for (int r = 0; r < 4; ++r) any_bad = __builtin_fmaf(x[r], 0.0f, any_bad);
          }
        }
        if (any_bad != 0.0f) *redo = 1;
        lds_barrier();
      }
      if (given || *redo == 0) break;  // uniform: set before the barrier above
      lds_barrier();
    }
    // (m, l) with l in [1, 2): the reference is not the maximum, so l may be far from 1
#pragma unroll
    for (int hg = 0; hg < RG; ++hg) {
      e4[hg] = l4[hg] > 0.0f && l4[hg] < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(l4[hg]) - 1 : 0;
      l4[hg] = __builtin_amdgcn_ldexpf(l4[hg], -e4[hg]);
      m4[hg] = l4[hg] == 0.0f ? -__builtin_huge_valf() : m4[hg] + static_cast<float>(e4[hg]);
    }
    // (an address that depends on nothing in the passes would be computed before them, and kept in memory)
    int col = e16;
    asm volatile("" : "+v"(col));
    // ---- the result: acc[i][hg][r] is row 16 hg + e16, channel 16 (wave + 4 i) + 4 g + r ------------
    // A unit of several tokens whose result is not finite is looked at again, token by token: its rows
    // are written here and once more then.
    float bad = 0.0f;  // NaN if a result is not finite
    const int keep0 = (sub0 * p.HG > u.r0 ? sub0 * p.HG : u.r0) - u.r0;
    const int keep1 = (sub1 * p.HG < u.r1 ? sub1 * p.HG : u.r1) - u.r0;
    if (u.shares > 1) {
#pragma unroll
      for (int hg = 0; hg < RG; ++hg) {
        const int r = 16 * hg + col;
        if (r >= keep0 && r < keep1) {
          const float inv = l4[hg] > 0.0f || l4[hg] != l4[hg] ? __builtin_amdgcn_ldexpf(1.0f / l4[hg], -e4[hg]) : 0.0f;
          float* o = p.part_o + static_cast<int64_t>(u.slot) * 64 * D + 1024 * wave + 16 * r + 4 * g;
#pragma unroll
          for (int i = 0; i < NI; ++i, o += 4096) {
            const v4f x = acc[i][hg] * inv;
#pragma unroll
            for (int c = 0; c < 4; ++c) bad = __builtin_fmaf(x[c], 0.0f, bad);
            *reinterpret_cast<v4f*>(o) = x;
          }
          if (wave == hg && g == 0)
            *reinterpret_cast<float2*>(p.part_ml + 2 * (static_cast<int64_t>(u.slot) * 64 + r)) = float2{m4[hg], l4[hg]};
        }
      }
      if (bad != 0.0f) *odd = 1;
      lds_barrier();
    } else {
      // through LDS, so that the rows leave in whole lines
      constexpr int OPITCH = 2 * D + 16;
#pragma unroll
      for (int hg = 0; hg < RG; ++hg) {
        const int r = 16 * hg + col;
        if (r >= keep0 && r < keep1) {
          int head;
          const int at = row_at(p, u, u.r0 + r, head);
          float lse;
          const float scale = __builtin_amdgcn_ldexpf(finish_row(m4[hg], l4[hg], sinks[r], lse), -e4[hg]);
          uint8_t* const orow = smem + r * OPITCH + 32 * wave + 8 * g;
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const v4f x = acc[i][hg] * scale;
#pragma unroll
            for (int c = 0; c < 4; ++c) bad = __builtin_fmaf(x[c], 0.0f, bad);
            *reinterpret_cast<uint2*>(orow + 128 * i) = uint2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
          }
          if (wave == hg && g == 0) p.lse[at] = lse;
        }
      }
      if (bad != 0.0f) *odd = 1;
#pragma unroll
      for (int k = 0; k < LINES; ++k) asm volatile("" : : "v"(hint[k]));
      lds_barrier();
      if (RG == 4 && p.G == 1 && keep0 == 0 && keep1 == 64) {  // one run of rows
        u32x4* const ob = reinterpret_cast<u32x4*>(p.out + (static_cast<int64_t>(u.t0) * p.H + u.r0) * D);
        int mine = tid;
        asm volatile("" : "+v"(mine));
#pragma unroll
        for (int k = 0; k < QP; ++k) {
          const int at = mine + NT * k;
          (ob + NT * k)[mine] = *reinterpret_cast<const u32x4*>(smem + 16 * at + (OPITCH - 2 * D) * (at / QROW));
        }
      } else {
#pragma unroll 1
        for (int at = tid; at < ROWS * QROW; at += NT) {
          const int r = at / QROW;
          int head;
          if (r >= keep0 && r < keep1)
            *reinterpret_cast<u32x4*>(p.out + static_cast<int64_t>(row_at(p, u, u.r0 + r, head)) * D + 8 * (at - r * QROW)) =
                *reinterpret_cast<const u32x4*>(smem + r * OPITCH + 16 * (at - r * QROW));
        }
      }
    }
    if (!strict && tok1 - tok0 > 1 && *odd != 0) {  // uniform: set before the barrier above
      strict = true;
      sub0 = tok0;
      sub1 = tok0 + 1;
      lds_barrier();
      continue;
    }
    if (!strict || sub1 >= tok1) break;
    ++sub0;
    ++sub1;
    lds_barrier();
  }
}
