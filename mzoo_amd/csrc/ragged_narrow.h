// The ragged attention kernel for latents of up to 256 channels (ragged.hip includes this inside its
// namespace, after the units).
//
// One workgroup = one unit: 4 waves over tiles of 64 entries held as bf16 in LDS, two tiles (one at work,
// one arriving).  Per tile:
//   S^T  wave w: entries 16 w .. + 15 x all 64 rows (v_mfma_f32_16x16x32_bf16, q in registers, one
//        K operand read for four row groups), so a lane has 4 entries of each of its 4 rows;
//   P^T  to LDS in bf16 (8 KB; the row sums take the unrounded weights: see ragged_wide.h);
//   O^T  wave w: the 16-channel blocks w, w + 4, .. x 64 rows, one V^T operand read for four row groups.
// Two barriers a tile.  A tile is some 200 cycles of matrix work at D = 160 and its softmax as many of
// vector work, so what carries it is two workgroups on a compute unit, each in the other's waits (256
// registers, at most 80 KB).  bf16 entries are loaded straight into LDS, D / 32 instructions a wave and tile; 8-bit
// ones pass through registers.
//
// What bounds it: latency and vector work.  17 prompts of up to 700 tokens x 8 heads of 160 channels take 35
// us (8 at the memory's rate, 6 at the matrix units'), 24 sequences of up to 9000 with four new tokens of 16 heads
// 26 us and 8 for the join (9 at the memory's rate), 32 of up to 20000 x 16 heads 43 us in all (26).  Pages also
// cost a pause every CT tiles, where the next codes are laid out with no tile in flight.
//
// A tile in LDS is D / 32 columns of 64 rows of 64 bytes: a wave's load instruction (16 rows x 64 bytes, a
// lane 16 of them) fills 1 KB of one column from one address per lane and tile, and an MFMA step of S^T
// reads one column.  The 16-byte piece x of row r sits at slot x ^ narrow_swz(r) of its 64 bytes.
//
// Softmax and hidden entries as in ragged_wide.h: a fixed reference from the first tile, a second pass
// from the true maxima where that does not hold, and token by token where a result is not finite.

constexpr int kTile64 = 64;

// Four rows are a line of banks, so the rows of a phase that meet in one are told apart: 16 rows of a K
// operand's piece, four rows x 32 bytes of V^T.
__device__ __forceinline__ int narrow_swz(int row) { return row >> 2 & 3; }

// 16 bytes per lane from `at` + 64 J to LDS, column J of a tile (see load_column in ragged_wide.h)
template <int J, int N>
__device__ __forceinline__ void load_narrow(gptr_t at, uint32_t lds) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2"
               : : "s"(lds), "v"(at), "n"(64 * J), "n"((4096 - 64) * J) : "memory", "scc");
  if constexpr (J + 1 < N) load_narrow<J + 1, N>(at, lds);
}

template <int FMT, int D>
struct NarrowLds {
  static constexpr bool kDirect = FMT == kFmtBf16;
  static constexpr int TILE = kTile64 * 2 * D;
  static constexpr int PB = 2 * TILE;              // P^T: [2 K-steps][4 row groups][64 lanes] x 16 bytes
  static constexpr int CT = 8;                     // tiles whose entry codes are laid out at a time
  static constexpr int TAB = PB + 8192;
  static constexpr int MASK = TAB + 4 * CT * kTile64;  // [CT][2] words
  static constexpr int PMAX = MASK + 8 * CT;       // [4 waves][64]
  static constexpr int LSUM = PMAX + 1024;         // [4 waves][64]
  static constexpr int RED = LSUM + 1024;
  static constexpr int END = RED + 32;
  static constexpr int LDS = END > static_cast<int>(sizeof(PlanLds)) ? END : static_cast<int>(sizeof(PlanLds));
  static_assert(LDS <= 80 * 1024, "two workgroups a compute unit");
};

template <int FMT, int D, int NOPE>
__global__ void __launch_bounds__(256, D > 160 ? 1 : 2) ragged_narrow_kernel(const RaggedParams p) {
  using M = NarrowLds<FMT, D>;
  using L = Layout<FMT, D, NOPE>;
  constexpr int NT = 256, KS = D / 32, NB = D / 16, NI = (NB + 3) / 4, COL = 4096;
  constexpr int PPT = (L::kPieces + 3) / 4;                 // 8-bit entries: pieces of a thread
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* const tab = reinterpret_cast<uint32_t*>(smem + M::TAB);
  uint32_t* const masks = reinterpret_cast<uint32_t*>(smem + M::MASK);
  float* const pmax = reinterpret_cast<float*>(smem + M::PMAX);
  float* const lsum = reinterpret_cast<float*>(smem + M::LSUM);
  int* const redo = reinterpret_cast<int*>(smem + M::RED);
  int* const high = redo + 1;
  int* const odd = redo + 2;
  uint8_t* const pbuf = smem + M::PB;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, e16 = lane & 15;

  Unit u;
  zero_rows(p, tid);
  if (!find_unit(p, u, smem, tid)) return;  // uniform

  const int tok0 = p.by_heads(u.r0), tok1 = p.by_heads(u.r1 - 1) + 1;
  const int shift = u.len - u.n;
  int share_lo, share_hi;
  unit_range(p, u, tok0, tok1, share_lo, share_hi);
  const bool paged = p.tables != nullptr;
  const uint64_t first_entry = reinterpret_cast<uint64_t>(p.entries) +
                               (paged ? 0 : static_cast<uint64_t>(u.t0) * p.entry_stride + static_cast<uint64_t>(u.g) * L::kEntryBytes);
  const uint32_t entry_stride = static_cast<uint32_t>(p.entry_stride);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)smem)) + 1024u * wave;

  // addresses within a tile
  const uint32_t k_at = static_cast<uint32_t>((16 * wave + e16) * 64 + 16 * (g ^ narrow_swz(e16)));
  const int vrow = 4 * g + (e16 >> 2);
  const uint32_t v_at = static_cast<uint32_t>(COL * (wave >> 1) + vrow * 64 + 16 * ((2 * (wave & 1) + ((e16 >> 1) & 1)) ^ narrow_swz(vrow)) +
                                              8 * (e16 & 1));
  const int ld_row = M::kDirect ? 16 * wave + (lane >> 2) : tid >> 2;  // the entry this lane fetches
  const uint64_t piece = first_entry + (M::kDirect ? 16u * ((lane & 3) ^ narrow_swz(ld_row)) : 0u);

  int lo = 0, hi = 0, c0 = 0, nt = 0;
  int sub0 = tok0, sub1 = tok1;
  int row_lo[4], row_span[4], tok_h[4];
  int full_lo = 0, full_hi = 0;
  auto set_range = [&]() __attribute__((always_inline)) {
    token_range(p, u, sub0, sub1, lo, hi);
    lo = lo > share_lo ? lo : share_lo;
    hi = hi < share_hi ? hi : share_hi;
    if (hi < lo) hi = lo;
    int most_lo = lo, least_hi = hi;
    if (!p.idx) {
      most_lo = clamp32(shift + sub1 - p.window, lo, 0x7fffffff - kTile64);
      least_hi = shift + sub0 + 1 < hi ? shift + sub0 + 1 : hi;
    }
    full_lo = (most_lo - lo + kTile64 - 1) / kTile64;
    full_hi = least_hi > lo ? (least_hi - lo) / kTile64 : 0;
  };
  auto set_rows = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      int a = lo, z = hi;
      if (!p.idx) {
        const int pos = shift + tok_h[hg];
        if (pos - p.window + 1 > a) a = pos - p.window + 1;
        if (pos + 1 < z) z = pos + 1;
      }
      row_lo[hg] = a - lo;
      row_span[hg] = z > a ? z - a : 0;
    }
  };

  // The codes of the chunk's entries and which are there; an empty slot is fetched as another entry that
  // is there (its weight is 0).  False: none is.
  auto lay_out = [&]() __attribute__((always_inline)) -> bool {
    const int left = hi - lo - c0;
    if (!paged) {
      nt = (left + kTile64 - 1) / kTile64;
      return left > 0;
    }
    constexpr uint32_t kEmpty = 0xffffffffu;
    nt = ((left < M::CT * kTile64 ? left : M::CT * kTile64) + kTile64 - 1) / kTile64;
    uint32_t any = kEmpty;
    for (int e0 = 0; e0 < nt * kTile64; e0 += NT) {
      const int e = e0 + tid;
      uint32_t code = kEmpty;
      if (e < nt * kTile64 && e < left) code = static_cast<uint32_t>(pool_entry(p, u, lo + c0 + e));  // -1: kEmpty
      const uint64_t bal = __ballot(code != kEmpty);
      if (e < nt * kTile64) {
        tab[e] = code;
        if (lane == 0) {
          masks[2 * (e / kTile64)] = static_cast<uint32_t>(bal);
          masks[2 * (e / kTile64) + 1] = static_cast<uint32_t>(bal >> 32);
        }
      }
    }
    lds_barrier();
    const int word = lane < 2 * nt ? static_cast<int>(masks[lane]) : 0;
    const uint64_t some = __ballot(word != 0);
    if (some == 0) {
      lds_barrier();  // the next chunk's codes come here
      return false;
    }
    const int at = __builtin_ctzll(some);
    any = tab[32 * at + __builtin_ctz(masks[at])];
    lds_barrier();
    for (int e = tid; e < nt * kTile64; e += NT)
      if (tab[e] == kEmpty) tab[e] = any;
    lds_barrier();
    return true;
  };
  auto code_of = [&](int t, int row) __attribute__((always_inline)) -> uint32_t {
    if (paged) return tab[t * kTile64 + row];
    const int v = c0 + t * kTile64 + row;
    return static_cast<uint32_t>(lo + (v < hi - lo ? v : hi - lo - 1));
  };
  Piece raw[M::kDirect ? 1 : PPT];
  // tile t requested: straight into its buffer, or into registers
  auto ask = [&](int t) __attribute__((always_inline)) {
    const gptr_t e = (gptr_t)(piece + static_cast<uint64_t>(code_of(t, ld_row)) * entry_stride);
    if constexpr (M::kDirect) {
      load_narrow<0, KS>(e, __builtin_amdgcn_readfirstlane(lds0 + (t & 1) * M::TILE));
    } else {
#pragma unroll
      for (int j = 0; j < PPT; ++j) {
        const int q = (tid & 3) + 4 * j;
        if (q < L::kPieces) raw[j] = fetch_piece<FMT, D, NOPE>(e, q);
      }
    }
  };
  // ... and there for this wave (all of it for everyone after the next barrier)
  auto arrive = [&](int t) __attribute__((always_inline)) {
    if constexpr (M::kDirect) {
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    } else {
      const int x = narrow_swz(ld_row);
      uint8_t* const at = smem + (t & 1) * M::TILE + ld_row * 64;
#pragma unroll
      for (int j = 0; j < PPT; ++j) {
        const int q = (tid & 3) + 4 * j;
        if (q < L::kCodePieces) {  // 16 codes: two bf16 pieces
          uint8_t* const c = at + COL * (q >> 1);
          *reinterpret_cast<uint4*>(c + 16 * ((2 * (q & 1)) ^ x)) = dequant_fp8x8_bf16(uint2{raw[j].v.x, raw[j].v.y}, raw[j].s);
          *reinterpret_cast<uint4*>(c + 16 * ((2 * (q & 1) + 1) ^ x)) = dequant_fp8x8_bf16(uint2{raw[j].v.z, raw[j].v.w}, raw[j].s);
        } else if (q < L::kPieces) {
          const int i = NOPE / 8 + q - L::kCodePieces;
          *reinterpret_cast<uint4*>(at + COL * (i >> 2) + 16 * ((i & 3) ^ x)) = uint4{raw[j].v.x, raw[j].v.y, raw[j].v.z, raw[j].v.w};
        }
      }
    }
  };
  v8bf qf[KS][4];
  // this lane's scaled scores of tile t, -inf where hidden
  auto scores = [&](int t, float (&v)[4][4]) __attribute__((always_inline)) {
    const uint8_t* const kt = smem + (t & 1) * M::TILE + k_at;
    v4f s[4] = {v4f{}, v4f{}, v4f{}, v4f{}};
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const v8bf kf = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(kt + COL * st));
#pragma unroll
      for (int hg = 0; hg < 4; ++hg) s[hg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[st][hg], s[hg], 0, 0, 0);
    }
#pragma unroll
    for (int hg = 0; hg < 4; ++hg)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[hg][r] = s[hg][r] * p.scale_log2;
    const int at = c0 / kTile64 + t;
    uint32_t bits = 0xffffu;
    bool whole = at >= full_lo && at < full_hi;
    if (paged) {
      const uint32_t m0 = masks[2 * t], m1 = masks[2 * t + 1];
      whole = whole && (m0 & m1) == 0xffffffffu;
      bits = (wave & 2 ? m1 : m0) >> (16 * (wave & 1));
    }
    if (!__builtin_amdgcn_readfirstlane(whole)) {  // uniform
      const int e0 = c0 + t * kTile64 + 16 * wave + 4 * g;
#pragma unroll
      for (int hg = 0; hg < 4; ++hg)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = ((bits >> (4 * g + r)) & 1u) != 0u && static_cast<uint32_t>(e0 + r - row_lo[hg]) < static_cast<uint32_t>(row_span[hg]);
          v[hg][r] = in ? v[hg][r] : -__builtin_huge_valf();
        }
    }
  };
  auto max4 = [](const float (&v)[4]) __attribute__((always_inline)) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); };
  float m4[4], l_own[4], m_seen[4];
  v4f acc[NI][4];
  // the rows' maxima over the four lanes and the four waves into m4; 0 for a row without one (one barrier)
  auto agree_max = [&](float (&t)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      t[hg] = fmaxf(t[hg], __shfl_xor(t[hg], 16, 64));
      t[hg] = fmaxf(t[hg], __shfl_xor(t[hg], 32, 64));
      if (g == 0) pmax[64 * wave + 16 * hg + e16] = t[hg];
    }
    lds_barrier();
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      const float* const at = pmax + 16 * hg + e16;
      const float m = fmaxf(fmaxf(at[0], at[64]), fmaxf(at[128], at[192]));
      m4[hg] = m == -__builtin_huge_valf() ? 0.0f : m;
    }
  };

  // The first tile is requested before q (the B operand of S^T: rows 16 hg + e16, channels 32 st + 8 g ..)
  // and what the rows see of it is worked out.
  set_range();
  const bool none = !(lo < hi && lay_out());  // uniform
  if (!none) ask(0);
  float sink4[4];
#pragma unroll
  for (int hg = 0; hg < 4; ++hg) {
    const int r = u.r0 + 16 * hg + e16;
    const int rc = r < u.r1 ? r : u.r0;
    int head;
    const uint16_t* const qr = p.q + static_cast<int64_t>(row_at(p, u, rc, head)) * D + 8 * g;
#pragma unroll
    for (int st = 0; st < KS; ++st) qf[st][hg] = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(qr + 32 * st));
    sink4[hg] = p.sinks ? p.sinks[head] : -__builtin_huge_valf();
    tok_h[hg] = p.by_heads(rc);
  }

  bool strict = false, at_start = true;
  while (true) {
    if (!at_start) set_range();
    set_rows();
    float l4[4];
    int e4[4];
    for (bool given = false;; given = true) {
      if (tid == 0) *redo = *high = *odd = 0;
      bool begun = false;
      if (given) {  // the true maxima of every row: scores only
        float top[4] = {-__builtin_huge_valf(), -__builtin_huge_valf(), -__builtin_huge_valf(), -__builtin_huge_valf()};
        for (c0 = 0; c0 < hi - lo; c0 += nt * kTile64) {
          if (!lay_out()) continue;
#pragma unroll 1
          for (int t = 0; t < nt; ++t) {
            ask(t);
            arrive(t);
            lds_barrier();
            float v[4][4];
            scores(t, v);
#pragma unroll
            for (int hg = 0; hg < 4; ++hg) top[hg] = fmaxf(top[hg], max4(v[hg]));
            lds_barrier();
          }
        }
        agree_max(top);
        lds_barrier();
        begun = true;
      }
#pragma unroll
      for (int hg = 0; hg < 4; ++hg) {
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i][hg] = v4f{};
        l_own[hg] = 0.0f;
        m_seen[hg] = -__builtin_huge_valf();
        if (!begun) m4[hg] = 0.0f;
      }
      for (c0 = 0; c0 < hi - lo; c0 += nt * kTile64) {
        const bool ready = at_start && c0 == 0;
        if (ready ? none : !lay_out()) continue;
        if (!ready) ask(0);
#pragma unroll 1
        for (int t = 0; t < nt; ++t) {
          arrive(t);
          lds_barrier();  // tile t is there; tile t - 1 and its weights are read no more
          if (t + 1 < nt) ask(t + 1);
          float v[4][4];
          scores(t, v);
          if (!begun) {
            float top[4];
#pragma unroll
            for (int hg = 0; hg < 4; ++hg) top[hg] = max4(v[hg]);
            agree_max(top);
            begun = true;
          }
#pragma unroll
          for (int hg = 0; hg < 4; ++hg) {
            m_seen[hg] = fmaxf(m_seen[hg], max4(v[hg]));
            // v_exp_f32 directly: results below 2^-126 may flush to 0
#pragma unroll
            for (int r = 0; r < 4; ++r) v[hg][r] = __builtin_amdgcn_exp2f(v[hg][r] - m4[hg]);
            l_own[hg] = l_own[hg] + ((v[hg][0] + v[hg][1]) + (v[hg][2] + v[hg][3]));
            *reinterpret_cast<uint2*>(pbuf + 4096 * (wave >> 1) + 1024 * hg + 16 * lane + 8 * (wave & 1)) =
                uint2{pack_bf16x2(v[hg][0], v[hg][1]), pack_bf16x2(v[hg][2], v[hg][3])};
          }
          lds_barrier();  // the weights of tile t are there
          const uint8_t* const vt = smem + (t & 1) * M::TILE + v_at;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            v8bf pf[4];
#pragma unroll
            for (int hg = 0; hg < 4; ++hg)
              pf[hg] = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(pbuf + 4096 * ks + 1024 * hg + 16 * lane));
#pragma unroll
            for (int i = 0; i < NI; ++i)
              if (wave + 4 * i < NB) {  // uniform
                const uint8_t* const tp = vt + 2 * COL * i + 2048 * ks;
                const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_v4s(tp));
                const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_v4s(tp + 1024));
                const v8bf vf = __builtin_bit_cast(v8bf, v8s{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
#pragma unroll
                for (int hg = 0; hg < 4; ++hg) acc[i][hg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[hg], acc[i][hg], 0, 0, 0);
              }
          }
        }
        lds_barrier();  // the LDS is free again
      }
      at_start = false;
      // each row's sum: its four lanes, then the four waves
#pragma unroll
      for (int hg = 0; hg < 4; ++hg) {
        l_own[hg] = l_own[hg] + __shfl_xor(l_own[hg], 16, 64);
        l_own[hg] = l_own[hg] + __shfl_xor(l_own[hg], 32, 64);
        if (g == 0) lsum[64 * wave + 16 * hg + e16] = l_own[hg];
      }
      if (!given) {  // (zero before the barriers of the pass; without an entry nothing is set)
#pragma unroll
        for (int hg = 0; hg < 4; ++hg) {
          const float rise = m_seen[hg] - m4[hg];
          if (rise > kRoomHigh) *high = 1;
          if (rise > kRoomAbove || (rise < kRoomBelow && m4[hg] == 0.0f && m_seen[hg] > -__builtin_huge_valf())) *redo = 1;
        }
      }
      lds_barrier();
#pragma unroll
      for (int hg = 0; hg < 4; ++hg) {
        const float* const at = lsum + 16 * hg + e16;
        l4[hg] = (at[0] + at[64]) + (at[128] + at[192]);
      }
      if (!given && *high != 0) {  // uniform
        float any_bad = 0.0f;      // NaN if an accumulator is not finite
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int hg = 0; hg < 4; ++hg)
#pragma unroll
            for (int r = 0; r < 4; ++r) any_bad = __builtin_fmaf(acc[i][hg][r], 0.0f, any_bad);
        if (any_bad != 0.0f) *redo = 1;
        lds_barrier();
      }
      if (given || *redo == 0) break;  // uniform: set before the barrier above
      lds_barrier();
    }
    // (m, l) with l in [1, 2): the reference is not the maximum, so l may be far from 1
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      e4[hg] = l4[hg] > 0.0f && l4[hg] < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(l4[hg]) - 1 : 0;
      l4[hg] = __builtin_amdgcn_ldexpf(l4[hg], -e4[hg]);
      m4[hg] = l4[hg] == 0.0f ? -__builtin_huge_valf() : m4[hg] + static_cast<float>(e4[hg]);
    }
    // the result: acc[i][hg][r] is row 16 hg + e16, channel 16 (wave + 4 i) + 4 g + r.  A unit of several
    // tokens whose result is not finite is looked at again, token by token: its rows are written here
    // and once more then.
    const int keep0 = (sub0 * p.HG > u.r0 ? sub0 * p.HG : u.r0) - u.r0;
    const int keep1 = (sub1 * p.HG < u.r1 ? sub1 * p.HG : u.r1) - u.r0;
    float bad = 0.0f;  // NaN if a result is not finite
    int col = e16;
    asm volatile("" : "+v"(col));  // (addresses formed here, not kept through the passes)
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      const int r = 16 * hg + col;
      if (r < keep0 || r >= keep1) continue;
      if (u.shares > 1) {
        const float inv = l4[hg] > 0.0f || l4[hg] != l4[hg] ? __builtin_amdgcn_ldexpf(1.0f / l4[hg], -e4[hg]) : 0.0f;
        float* const o = p.part_o + static_cast<int64_t>(u.slot) * 64 * D + 1024 * wave + 16 * r + 4 * g;
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (wave + 4 * i < NB) {
            const v4f x = acc[i][hg] * inv;
#pragma unroll
            for (int c = 0; c < 4; ++c) bad = __builtin_fmaf(x[c], 0.0f, bad);
            *reinterpret_cast<v4f*>(o + 4096 * i) = x;
          }
        if (wave == hg && g == 0)
          *reinterpret_cast<float2*>(p.part_ml + 2 * (static_cast<int64_t>(u.slot) * 64 + r)) = float2{m4[hg], l4[hg]};
      } else {
        int head;
        const int at = row_at(p, u, u.r0 + r, head);
        float lse;
        const float scale = __builtin_amdgcn_ldexpf(finish_row(m4[hg], l4[hg], sink4[hg], lse), -e4[hg]);
        uint16_t* const o = p.out + static_cast<int64_t>(at) * D + 16 * wave + 4 * g;
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (wave + 4 * i < NB) {
            const v4f x = acc[i][hg] * scale;
#pragma unroll
            for (int c = 0; c < 4; ++c) bad = __builtin_fmaf(x[c], 0.0f, bad);
            *reinterpret_cast<uint2*>(o + 64 * i) = uint2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
          }
        if (wave == hg && g == 0) p.lse[at] = lse;
      }
    }
    if (!strict && tok1 - tok0 > 1) {  // uniform
      if (bad != 0.0f) *odd = 1;
      lds_barrier();
      if (*odd == 0) break;
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
