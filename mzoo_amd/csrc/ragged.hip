// Shared-latent attention over sequences of different lengths: one new token or a few of each over its
// pages (paged_attend), or whole packed prompts, causal (packed_mqa).
//
//   o[t, h] = sum_j p_j e_j,  p = softmax over the entries j that token t sees of q[t, h] . e_j D^-1/2,
//   the head's sink one more term of the denominator; lse its logarithm.  K == V == e.
//   Token i of the n new ones of a sequence with len tokens is at position len - n + i and sees
//   positions 0 .. its own, the last `window` of them and the `first` of the sequence, or the
//   positions of its list.
//
// A unit of work is a block of 64 rows -- a row is a head of a token, the heads of one latent
// innermost, so 64 rows are 64 heads of a token or all heads of several -- over all of the
// sequence's entries, or, where the blocks alone would leave compute units idle, over a share of
// them; the shares' results are joined by a second launch (unit_slots, splits).
#include <type_traits>

#include "common.h"
#include "entries.h"

namespace mzk {
namespace {

constexpr int64_t kMaxInt = 0x7fffffff;
constexpr int kNoWindow = 1 << 30;  // packed prompts without a window: a call has fewer tokens

// Division of n < 2^31 by a constant of the call: floor(n m / 2^32) + n, shifted, with m = floor(2^32 (2^s -
// d) / d) + 1 and 2^s >= d.  Three instructions; what is executed once runs from a cold instruction
// cache, where a 64-bit division is half a microsecond.
struct FastDiv {
  uint32_t d, m;
  int s;
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), m) + static_cast<uint32_t>(n)) >> s);
  }
};
FastDiv fast_div(uint32_t d) {
  int s = 0;
  while ((1ull << s) < d) ++s;
  return FastDiv{d, static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

struct RaggedParams {
  const uint16_t* q;  // [T, H, D] bf16
  int64_t T;
  int H, G, HG;  // heads, latents, heads of a latent
  int D;
  const int64_t* cu;    // [B + 1], null: one token per sequence
  int64_t B;
  const int64_t* lens;  // [B] tokens in the pages, the new ones included; null: the new ones are all
  // entries: a pool of pages, or (tables null) one entry per packed token and latent
  const uint8_t* entries;
  int64_t entry_stride;  // bytes from entry to entry
  const int32_t* tables;
  int64_t table_stride, max_pages, pages;  // max_pages * page and pages * page below 2^31
  int page;
  const int32_t* idx;  // [B, topk] positions (one token per sequence), or null
  int64_t idx_stride;
  int topk;
  int window;
  int first;     // with a window: the sequence's first positions that every token behind them sees too
  int64_t past;  // lengths past a table's entries that are told apart: the window; without one -1
  const float* sinks;
  float scale_log2;
  FastDiv by_heads, by_page, by_blocks;  // HG, page, the row blocks of one token
  int unit_shift;      // log2 of a unit's rows: 32 for one head, else 64, so a unit spans at most 33 tokens
  int64_t blocks_max;  // row blocks at most
  // splitting: at most `slots` units (0: one unit per block, no joining), shares of at least
  // min_tiles tiles; a unit of a split sequence leaves its result in the slot of its number
  int slots, min_tiles;
  struct JoinRow* joins;  // [blocks], by each block's first share
  int32_t* blocks_out;    // the blocks, by the first workgroup
  float* part_o;       // [slots][D / 16][64][16]: O / l, a store instruction of the attention kernel 1 KB of it
  float* part_ml;      // [slots][64][2]: m in log2 units, l
  uint16_t* out;
  float* lse;          // [T, H]
  int zero_tail;       // rows of no sequence become 0 (else they are left as they are)
};

// What the joining launch knows of a row block.
struct JoinRow {
  int64_t row0;  // its first row of out and lse
  int32_t rows, shares, slot0, step;  // share s is in slot slot0 + s * step
};

// Where a unit's rows and entries are.
struct Unit {
  int b, t0;          // sequence, its first packed token
  int n, len;         // its new tokens, its tokens in all
  int room;           // those of them that its pages may hold: the table ends there
  int g;              // latent
  int r0, r1;         // rows of the sequence and latent: token r / HG, head g HG + r % HG
  int share, shares;  // of the tiles from the first to the last entry that a row sees
  int slot;
};

__device__ __forceinline__ int clamp32(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return static_cast<int64_t>(static_cast<uint32_t>(uniform(static_cast<int>(v)))) |
         static_cast<int64_t>(uniform(static_cast<int>(v >> 32))) << 32;
}

// Sums over a workgroup of 256 (lds: 4 words).
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& before, int64_t* lds, int tid) {
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(x, d, 64);
    if ((tid & 63) >= d) x += y;
  }
  if ((tid & 63) == 63) lds[tid >> 6] = x;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < (tid >> 6)) base += lds[w];
    total += lds[w];
  }
  __syncthreads();
  before = base + x - v;
  return total;
}

// Sequence i's packed tokens a .. z - 1, its row blocks of one latent and its tiles.
__device__ __forceinline__ int sequence(const RaggedParams& p, int i, int& a, int& z, int& tiles) {
  a = i;
  z = i + 1;
  if (p.cu) {
    a = static_cast<int>(clamp64(p.cu[i], 0, p.T));
    z = static_cast<int>(clamp64(p.cu[i + 1], a, p.T));
  }
  int seen = z - a;
  if (p.lens) seen = static_cast<int>(clamp64(p.lens[i], 0, p.max_pages * p.page));
  if (p.idx) seen = seen > 0 ? p.topk : 0;
  if (seen - (z - a) - p.first > p.window) seen = p.window + (z - a) + p.first;
  tiles = (seen + kTile - 1) / kTile;
  return ((z - a) * p.HG + (1 << p.unit_shift) - 1) >> p.unit_shift;
}

constexpr int kPlanRows = 1024;  // the most sequences that are split
constexpr int kMaxShares = 256;  // of one sequence
struct PlanLds {
  int64_t scan[8];
  int count[4][64];
  int blocks[kPlanRows], tiles[kPlanRows];
};

// ceil(t / c), at least 1, from an approximate quotient
__device__ __forceinline__ int shares_of(int t, int c, float rc) {
  int k = static_cast<int>(static_cast<float>(t) * rc);
  k += static_cast<int64_t>(k) * c < t;
  k -= k > 1 && static_cast<int64_t>(k - 1) * c >= t;
  return k > 1 ? k : 1;
}

// The tiles of a share lie between what an even division gives and what always fits: the sum of
// blocks * ceil(tiles / c) <= work / c + blocks <= slots for c >= work / (slots - blocks).
__device__ __forceinline__ void share_bounds(const RaggedParams& p, int blocks, float work, int most, int& lo, int& hi) {
  hi = static_cast<int>(work / static_cast<float>(p.slots - blocks) * 1.00001f) + 2;
  lo = static_cast<int>(work / static_cast<float>(p.slots));
  if (hi > most) hi = most;
  if (lo < p.min_tiles) lo = p.min_tiles;
  if (lo < (most + kMaxShares - 1) / kMaxShares) lo = (most + kMaxShares - 1) / kMaxShares;
  if (hi < lo) hi = lo;
}
__device__ __forceinline__ int share_candidate(int lo, int hi, int j) { return lo + static_cast<uint32_t>(hi - lo) * static_cast<uint32_t>(j) / 63u; }

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ int wave_most(int v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const int o = __shfl_xor(v, d, 64);
    v = o > v ? o : v;
  }
  return v;
}
// sum over the lanes before this one
__device__ __forceinline__ int wave_before(int v, int lane) {
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x - v;
}

// The tiles of a share: the least for which the units fit the slots, of 64 values between the bounds.
// Every workgroup finds the same.  (G == 1 where there are shares.)
__device__ int share_tiles(const RaggedParams& p, PlanLds& l, int tid) {
  int blocks = 0, most = 1;
  float work = 0.0f;
  for (int i = tid; i < p.B; i += 256) {
    int a, z, t;
    const int n = sequence(p, i, a, z, t);
    l.blocks[i] = n;
    l.tiles[i] = t;
    blocks += n;
    work += static_cast<float>(n) * static_cast<float>(t);
    most = t > most ? t : most;
  }
  blocks = wave_sum(blocks);
  work = wave_sum(work);
  most = wave_most(most);
  if ((tid & 63) == 0) {
    l.count[0][tid >> 6] = most;
    l.count[1][tid >> 6] = blocks;
    l.count[2][tid >> 6] = __float_as_int(work);
  }
  __syncthreads();
  blocks = 0;
  work = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    most = l.count[0][w] > most ? l.count[0][w] : most;
    blocks += l.count[1][w];
    work += __int_as_float(l.count[2][w]);
  }
  __syncthreads();
  int lo, hi;
  share_bounds(p, blocks, work, most, lo, hi);
  const int c = share_candidate(lo, hi, tid & 63);
  const float rc = 1.0f / static_cast<float>(c);
  int n = 0;
  for (int i = tid >> 6; i < p.B; i += 4) n += l.blocks[i] * shares_of(l.tiles[i], c, rc);
  l.count[tid >> 6][tid & 63] = n;
  __syncthreads();
  const int j = tid & 63;
  const bool fits = l.count[0][j] + l.count[1][j] + l.count[2][j] + l.count[3][j] <= p.slots || j == 63;
  const int first = __builtin_ctzll(__ballot(fits));
  __syncthreads();
  return share_candidate(lo, hi, first);
}

// This workgroup's unit; false: none.  Workgroups go to the 8 XCDs in turn: without shares, two
// neighbouring blocks (which read the same entries) follow each other on an XCD, and the last
// blocks, which see the most, come first; with shares, an XCD takes neighbouring units.
// Up to 64 sequences every wave finds it alone, a lane per sequence: through LDS and barriers, as for
// more, it took 5.4 of the 33 us of a split call's attention launch.
__device__ bool find_unit(const RaggedParams& p, Unit& u, uint8_t* smem, int tid) {
  PlanLds& l = *reinterpret_cast<PlanLds*>(smem);
  const int lane = tid & 63;
  const int w = static_cast<int>(blockIdx.x);
  int blk, blocks, k, ordinal = 0, a, z, t = 0;  // blocks: of one latent
  u.share = 0;
  u.shares = 1;
  const bool small = p.B <= 64;
  if (p.slots == 0) {
    k = ((w >> 4) * 8 + (w & 7)) * 2 + (w >> 3 & 1);
    if (p.cu == nullptr) {
      u.b = p.by_blocks(k);
      if (u.b >= p.B) return false;
      blk = k - u.b * static_cast<int>(p.by_blocks.d);
      blocks = (p.HG + 63) >> 6;
    } else if (small) {
      const int v = lane < p.B ? sequence(p, lane, a, z, t) * p.G : 0;  // in all below blocks_max
      const int before = wave_before(v, lane);
      const int total = __builtin_amdgcn_readlane(before + v, 63);
      if (k >= total) return false;
      k = total - 1 - k;
      const int at = __builtin_ctzll(__ballot(k >= before && k < before + v));
      u.b = at;
      blk = k - __builtin_amdgcn_readlane(before, at);
      blocks = __builtin_amdgcn_readlane(v, at) / p.G;
    } else {
      int64_t total = 0;
      for (int i = tid; i < p.B; i += 256) total += sequence(p, i, a, z, t) * p.G;
      int64_t before, base = 0;
      total = block_scan(total, before, l.scan, tid);
      if (k >= total) return false;
      k = static_cast<int>(total) - 1 - k;
      for (int i = 0;; i += 256) {  // ends: k < total
        const int64_t v = i + tid < p.B ? sequence(p, i + tid, a, z, t) * p.G : 0;
        const int64_t sum = block_scan(v, before, l.scan, tid);
        if (k >= base + before && k < base + before + v) {
          l.scan[4] = i + tid;
          l.scan[5] = k - base - before;
          l.scan[6] = v;
        }
        base += sum;
        if (k < base) break;
      }
      __syncthreads();
      u.b = static_cast<int>(l.scan[4]);
      blk = static_cast<int>(l.scan[5]);
      blocks = static_cast<int>(l.scan[6]) / p.G;
    }
  } else if (small) {
    int v = 0, lo, hi;
    if (lane < p.B) v = sequence(p, lane, a, z, t);
    const int most = wave_most(t);
    share_bounds(p, wave_sum(v), wave_sum(static_cast<float>(v) * static_cast<float>(t)), most > 1 ? most : 1, lo, hi);
    int c = lo;
    if (hi > lo) {
      c = share_candidate(lo, hi, lane);
      const float rc = 1.0f / static_cast<float>(c);
      int n = 0;
      for (int i = 0; i < p.B; ++i) n += __builtin_amdgcn_readlane(v, i) * shares_of(__builtin_amdgcn_readlane(t, i), c, rc);
      c = __builtin_amdgcn_readlane(c, __builtin_ctzll(__ballot(n <= p.slots || lane == 63)));
    }
    const int shares = shares_of(t, c, 1.0f / static_cast<float>(c));
    const int units = v * shares, before = wave_before(units, lane), blocks_before = wave_before(v, lane);
    const int total = __builtin_amdgcn_readlane(before + units, 63);
    const int in_all = __builtin_amdgcn_readlane(blocks_before + v, 63);
    const bool fits = total <= p.slots && in_all <= p.blocks_max;  // not where cu does not ascend
    const int per_xcd = (total + 7) / 8;
    k = (w & 7) * per_xcd + (w >> 3);
    if (w == 0 && tid == 63) *p.blocks_out = fits ? in_all : 0;
    if (!fits || (w >> 3) >= per_xcd || k >= total) return false;
    const int at = __builtin_ctzll(__ballot(k >= before && k < before + units));
    u.b = at;
    blocks = __builtin_amdgcn_readlane(v, at);
    u.shares = __builtin_amdgcn_readlane(shares, at);
    const int in = k - __builtin_amdgcn_readlane(before, at);
    u.share = in / blocks;
    blk = in - u.share * blocks;
    ordinal = __builtin_amdgcn_readlane(blocks_before, at) + blk;
  } else {
    const int c = share_tiles(p, l, tid);
    const float rc = 1.0f / static_cast<float>(c);
    int64_t total = 0, before, base = 0, blocks_base = 0;
    for (int i = tid; i < p.B; i += 256) total += l.blocks[i] * shares_of(l.tiles[i], c, rc);
    total = block_scan(total, before, l.scan, tid);
    const int per_xcd = static_cast<int>((total + 7) / 8);
    k = (w & 7) * per_xcd + (w >> 3);
    const bool mine = (w >> 3) < per_xcd && k < total && total <= p.slots;
    if (!mine && w != 0) return false;
    for (int i = 0; i < p.B; i += 256) {
      int shares = 1;
      int64_t n = 0, blocks_before;
      if (i + tid < p.B) {
        shares = shares_of(l.tiles[i + tid], c, rc);
        n = l.blocks[i + tid];
      }
      const int64_t sum = block_scan(n * shares, before, l.scan, tid);
      const int64_t blocks_sum = block_scan(n, blocks_before, l.scan, tid);
      if (mine && k >= base + before && k < base + before + n * shares) {
        l.scan[4] = i + tid;
        l.scan[5] = k - base - before;
        l.scan[6] = shares;
        l.scan[7] = blocks_base + blocks_before;
      }
      base += sum;
      blocks_base += blocks_sum;
    }
    const bool fits = total <= p.slots && blocks_base <= p.blocks_max;  // not where cu does not ascend
    if (w == 0 && tid == 0) *p.blocks_out = fits ? static_cast<int32_t>(blocks_base) : 0;
    __syncthreads();
    if (!mine || !fits) return false;
    u.b = static_cast<int>(l.scan[4]);
    blocks = l.blocks[u.b];
    u.shares = static_cast<int>(l.scan[6]);
    u.share = static_cast<int>(l.scan[5]) / blocks;
    blk = static_cast<int>(l.scan[5]) - u.share * blocks;
    ordinal = static_cast<int>(l.scan[7]) + blk;
  }
  u.b = uniform(u.b);
  sequence(p, u.b, a, z, t);
  u.t0 = uniform(a);
  u.n = uniform(z - a);
  u.g = p.G == 1 ? 0 : uniform(blk / blocks);
  u.r0 = uniform((blk - u.g * blocks) << p.unit_shift);
  u.r1 = u.r0 + (1 << p.unit_shift) < u.n * p.HG ? u.r0 + (1 << p.unit_shift) : u.n * p.HG;
  u.len = u.room = u.n;
  if (p.lens) {
    // A sequence may be longer than its table.  From `most` on its new tokens see what they see there:
    // nothing behind their window, or all that the table holds.
    const int64_t len = p.lens[u.b], room = p.max_pages * p.page;
    const int64_t most = room + u.n + p.past < kMaxInt - 64 ? room + u.n + p.past : kMaxInt - 64;
    u.room = uniform(static_cast<int>(clamp64(len, 0, room)));
    u.len = uniform(static_cast<int>(clamp64(len, 0, most)));
  }
  u.share = uniform(u.share);
  u.shares = uniform(u.shares);
  u.slot = uniform(k);
  if (p.slots && u.share == 0 && tid == 0)
    p.joins[ordinal] = JoinRow{static_cast<int64_t>(u.t0) * p.H + u.r0, u.r1 - u.r0, u.shares, u.slot, blocks};
  if (!small) __syncthreads();  // the plan's LDS is free
  return true;
}

// Rows behind the last sequence, shared out over the workgroups: 0, and a log-sum-exp of -inf.
__device__ __forceinline__ void zero_rows(const RaggedParams& p, int tid) {
  if (!p.zero_tail || !p.cu) return;
  const int64_t end = clamp64(p.cu[p.B], 0, p.T) * p.H;
  for (int64_t r = end + blockIdx.x; r < p.T * p.H; r += gridDim.x) {
    for (int i = tid; i < p.D / 2; i += 256) reinterpret_cast<uint32_t*>(p.out + r * p.D)[i] = 0;
    if (tid == 0) p.lse[r] = -__builtin_huge_valf();
  }
}

// Row r of the unit's sequence: its row of q, out and lse, and its head.
__device__ __forceinline__ int row_at(const RaggedParams& p, const Unit& u, int r, int& head) {
  const int tok = p.by_heads(r);
  head = u.g * p.HG + (r - tok * p.HG);
  return (u.t0 + tok) * p.H + head;
}

// The positions (or places of the list) that tokens tok0 .. tok1 - 1 of the sequence see.
__device__ __forceinline__ void token_range(const RaggedParams& p, const Unit& u, int tok0, int tok1, int& lo, int& hi) {
  const int shift = u.len - u.n;  // position of the first new token (negative: tokens that see nothing)
  lo = clamp32(shift + tok0 - p.window + 1, 0, u.room);
  hi = clamp32(shift + tok1, 0, u.room);
  if (p.idx) {
    lo = 0;
    hi = u.room > 0 ? p.topk : 0;
  }
}

// This unit's share of the tiles that its tokens tok0 .. tok1 - 1 see.  With first positions that stay visible
// (FIRST), `head` of them lie before the window's and are counted as if directly before it: no tile is there for them
// alone, and the tiles between them and the window are not passed at all.  128 heads of 576 channels, `window` + `first`
// entries beside a window of as many: one sequence, 1024 + 4 8-bit entries, 23.9 and 23.2 us; 32 sequences, 4096 + 64, 74.1
// and 72.9 (some 530 TFLOP/s, with the join's 11 us); prompts of 15.6 K tokens, 512 + 16 of bf16, 3198 and 3158 (680 TFLOP/s: of
// a unit's 17 tiles the first's loads, q before them and the results behind them overlap with nothing).
template <bool FIRST>
__device__ __forceinline__ void unit_range(const RaggedParams& p, const Unit& u, int tok0, int tok1, int& lo, int& hi) {
  token_range(p, u, tok0, tok1, lo, hi);
  if (FIRST) lo -= p.first < lo ? p.first : lo;
  if (u.shares > 1) {
    const int tiles = (hi - lo + kTile - 1) / kTile, per = (tiles + u.shares - 1) / u.shares;
    const int64_t from = lo + static_cast<int64_t>(u.share) * per * kTile;
    if (from + per * kTile < hi) hi = static_cast<int>(from) + per * kTile;
    lo = from < hi ? static_cast<int>(from) : hi;
  }
}

// The entries of a pass: places lo .. hi - 1, of which those from `body` on are positions, and those before it the
// positions `jump` away: the first of the sequence that stay visible.
struct Pass {
  int lo, hi;
  int body, jump;
};

// What the tokens sub0 .. sub1 - 1 of a unit of tokens tok0 .. see of its share share_lo .. share_hi - 1
// (places of the unit, of which the first positions are those before the unit's window).
template <bool FIRST>
__device__ __forceinline__ Pass pass_range(const RaggedParams& p, const Unit& u, int tok0, int sub0, int sub1, int share_lo, int share_hi) {
  Pass w;
  token_range(p, u, sub0, sub1, w.lo, w.hi);
  const int seen_lo = w.lo;
  w.lo = w.lo > share_lo ? w.lo : share_lo;
  w.hi = w.hi < share_hi ? w.hi : share_hi;
  if (w.hi < w.lo) w.hi = w.lo;
  w.body = w.lo;
  w.jump = 0;
  if (FIRST) {
    int unit_lo, unit_hi;  // the unit's window begins there
    token_range(p, u, tok0, tok0 + 1, unit_lo, unit_hi);
    // head: positions h0 .. h1 - 1, all before the window of every token of the pass
    int h0 = share_lo, h1 = share_hi;
    if (p.first < unit_lo) {
      h1 = h1 < unit_lo ? h1 : unit_lo;
      h0 -= unit_lo - p.first;
      h1 -= unit_lo - p.first;
    } else {
      h1 = h1 < p.first ? h1 : p.first;
      h1 = h1 < seen_lo ? h1 : seen_lo;
    }
    if (h1 > h0) {
      w.jump = h1 - w.body;
      w.lo = w.body - (h1 - h0);
    }
  }
  return w;
}

// The entry at position v of the unit's sequence (or of its list) in a pool; -1: none.
__device__ __forceinline__ int pool_entry(const RaggedParams& p, const Unit& u, int v) {
  if (p.idx) {
    v = p.idx[u.b * p.idx_stride + v];
    if (v < 0 || v >= u.room) return -1;
  }
  const int at = p.by_page(v);
  const int pid = p.tables[u.b * p.table_stride + at];
  if (pid < 0 || pid >= p.pages) return -1;
  return pid * p.page + (v - at * p.page);
}

// A row's result from its maximum, sum and sink (-inf: none): the factor of O^T and the log-sum-exp.
__device__ __forceinline__ float finish_row(float m, float l, float sink, float& lse) {
  const bool none = l == 0.0f && m == -__builtin_huge_valf();  // it sees nothing: lse is the sink itself
  float scale = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const float sk = sink * kLog2e, mm = fmaxf(m, sk);
  if (sk != -__builtin_huge_valf()) {
    const float a = m == -__builtin_huge_valf() ? 0.0f : exp2f(m - mm);
    l = l * a + exp2f(sk - mm);
    m = mm;
    scale = a / l;
  }
  lse = none ? sink : (m + __log2f(l)) * kLn2;
  return scale;
}

constexpr float kRoomHigh = 8.0f, kRoomAbove = 100.0f, kRoomBelow = -40.0f;  // log2 units from a row's reference
constexpr float kHidden = -3.0e38f;  // a hidden entry's score: weight 0

#include "ragged_wide.h"
#include "ragged_narrow.h"

// Joins the shares of 16 rows of a row block: o = sum_s w_s O_s / sum_s w_s with w_s = l_s 2^(m_s - m), and the
// sink.  A wave takes one 16-channel block, so that a load instruction covers 1 KB of a share; SPLIT: the
// four waves of a workgroup take a quarter of one's shares each.
// Bound by latency for a few rows (record, then maxima and sums, then the shares' rows, eight of them
// requested together; 6 us) and by the memory for many (64 blocks of four shares of 576 channels, 38 MB: 12 us).
template <int D, bool SPLIT>
__global__ void __launch_bounds__(256) join_kernel(const RaggedParams p) {
  constexpr int NB = D / 16;
  __shared__ float weight[16][kMaxShares + 1];
  const int tid = threadIdx.x;
  const int k = blockIdx.x >> 2, r0 = 16 * (blockIdx.x & 3);
  if (k >= *p.blocks_out) return;
  const JoinRow j = p.joins[k];
  if (j.shares <= 1 || r0 >= j.rows) return;
  {  // weights: 16 threads a row
    const int r = tid >> 4, row = r0 + r;
    const float* const ml = p.part_ml + 2 * (static_cast<int64_t>(j.slot0) * 64 + row);
    const int64_t step = 128ll * j.step;
    float m = -__builtin_huge_valf(), l = 0.0f;
    if (row < j.rows)
      for (int s = tid & 15; s < j.shares; s += 16) m = fmaxf(m, ml[step * s]);
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (row < j.rows)
      for (int s = tid & 15; s < j.shares; s += 16) {
        const float2 v = *reinterpret_cast<const float2*>(ml + step * s);
        // a share that saw nothing has l 0 and m -inf, one with a NaN has l NaN
        const float w = v.x == -__builtin_huge_valf() && v.y == 0.0f ? 0.0f : v.y * exp2f(v.x - m);
        weight[r][s] = w;
        l += w;
      }
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) l += __shfl_xor(l, d, 64);
    if (row < j.rows) {
      const int64_t at = j.row0 + row;
      float lse;
      const float scale = finish_row(m, l, p.sinks ? p.sinks[at % p.H] : -__builtin_huge_valf(), lse);
      if ((tid & 15) == 0 && blockIdx.y == 0) p.lse[at] = lse;
      for (int s = tid & 15; s < j.shares; s += 16) weight[r][s] *= scale;
    }
  }
  __syncthreads();
  const int wave = tid >> 6, r = (tid & 63) >> 2, c = 4 * (tid & 3), row = r0 + r;
  const int blk = SPLIT ? static_cast<int>(blockIdx.y) : 4 * static_cast<int>(blockIdx.y) + wave;
  if (!SPLIT && (row >= j.rows || blk >= NB)) return;
  const float* const o = p.part_o + (static_cast<int64_t>(j.slot0) * NB + blk) * 1024 + 16 * (row < j.rows ? row : r0) + c;
  const int64_t step = 64ll * D * j.step;
  v4f sum = v4f{};
  constexpr int AHEAD = 8;
  const int per = SPLIT ? (j.shares + 3) / 4 : j.shares;
  const int from = SPLIT ? per * wave : 0, to = from + per < j.shares ? from + per : j.shares;
  for (int s0 = from; s0 < to; s0 += AHEAD) {
    v4f v[AHEAD];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) v[s] = *reinterpret_cast<const v4f*>(o + step * (s0 + s < to ? s0 + s : s0));
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
      if (s0 + s < to) {
        const float w = weight[r][s0 + s];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(w, v[s][i], sum[i]);
      }
  }
  if constexpr (SPLIT) {
    __shared__ v4f part[3][64];
    if (wave > 0) part[wave - 1][tid & 63] = sum;
    __syncthreads();
    if (wave > 0 || row >= j.rows) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) sum = sum + part[w][tid];
  }
  *reinterpret_cast<uint2*>(p.out + (j.row0 + row) * D + 16 * blk + c) = uint2{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
}

template <int FMT, int D, int NOPE, bool FIRST>
int launch_ragged_as(const RaggedParams& p, hipStream_t s) {
  // (find_unit's order takes 16 workgroups at a time)
  const int64_t grid = p.slots ? p.slots : p.blocks_max / 16 * 16 + 16;
  using M = std::conditional_t<(D > 256), WideLds<FMT, D>, NarrowLds<FMT, D>>;
  void (*kern)(const RaggedParams);
  int which = 0;
  if constexpr (D > 256) {
    which = p.cu || p.H > 32 ? 0 : p.H > 16 ? 1 : 2;
    kern = which == 0   ? ragged_wide_kernel<FMT, D, NOPE, 4, FIRST>
           : which == 1 ? ragged_wide_kernel<FMT, D, NOPE, 2, FIRST>
                        : ragged_wide_kernel<FMT, D, NOPE, 1, FIRST>;
  } else {
    kern = ragged_narrow_kernel<FMT, D, NOPE, FIRST>;
  }
  // the dynamic-LDS limit is a per-device function attribute: set once per device
  static std::atomic<bool> attr_set[3][kMaxDevices] = {};  // setting it twice is harmless
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    set_last_error("ragged attention: no usable current device");
    return MZK_ELAUNCH;
  }
  if (!attr_set[which][dev].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, M::LDS) != hipSuccess) {
      set_last_error("ragged attention: cannot raise the kernel's LDS limit to %d bytes", M::LDS);
      return MZK_ELAUNCH;
    }
    attr_set[which][dev].store(true, std::memory_order_release);
  }
  kern<<<static_cast<unsigned>(grid), 256, M::LDS, s>>>(p);
  if (p.slots) {
    const unsigned x = static_cast<unsigned>(4 * p.blocks_max);
    // one sequence of up to 32768 x 128 heads, 2 blocks of 128 shares: 44 us, 50 with a wave per channel block; 200
    // blocks: 209 us, 179
    if (p.slots >= 16 * p.blocks_max) join_kernel<D, true><<<dim3(x, D / 16), 256, 0, s>>>(p);
    else join_kernel<D, false><<<dim3(x, (D / 16 + 3) / 4), 256, 0, s>>>(p);
  }
  MZK_LAUNCH_CHECK("ragged attention");
  return MZK_OK;
}

// (An instance of its own for `first`: with it alone, calls without take up to 8 % longer, of 8 heads x 160 channels
// 38.5 us for 35.6, of 16 heads x 576 behind a window 433 for 419.)
template <int FMT, int D, int NOPE>
int launch_ragged(const RaggedParams& p, hipStream_t s) {
  return p.first ? launch_ragged_as<FMT, D, NOPE, true>(p, s) : launch_ragged_as<FMT, D, NOPE, false>(p, s);
}

int dispatch_ragged(const char* name, int fmt, int nope, const RaggedParams& p, hipStream_t s) {
  if (fmt == kFmtFp8) {
    if (p.D == 576 && nope == 512) return launch_ragged<kFmtFp8, 576, 512>(p, s);
    if (p.D == 160 && nope == 128) return launch_ragged<kFmtFp8, 160, 128>(p, s);
    set_last_error("%s fp8: unsupported latent %d+%d (have 512+64, 128+32)", name, nope, p.D - nope);
    return MZK_EUNSUPPORTED;
  }
  switch (p.D) {
    case 64: return launch_ragged<kFmtBf16, 64, 64>(p, s);
    case 96: return launch_ragged<kFmtBf16, 96, 96>(p, s);
    case 128: return launch_ragged<kFmtBf16, 128, 128>(p, s);
    case 160: return launch_ragged<kFmtBf16, 160, 160>(p, s);
    case 256: return launch_ragged<kFmtBf16, 256, 256>(p, s);
    case 512: return launch_ragged<kFmtBf16, 512, 512>(p, s);
    case 576: return launch_ragged<kFmtBf16, 576, 576>(p, s);
    default:
      set_last_error("%s bf16: unsupported head dim %d (have 64, 96, 128, 160, 256, 512, 576)", name, p.D);
      return MZK_EUNSUPPORTED;
  }
}

// The divisions and the row blocks of a call: at most blocks_max, whatever the lengths are.
void set_units(RaggedParams& p) {
  p.unit_shift = p.HG == 1 ? 5 : 6;
  const int64_t per = (static_cast<int64_t>(p.HG) + (1 << p.unit_shift) - 1) >> p.unit_shift;
  p.blocks_max = p.cu == nullptr ? p.B * p.G * per : ((p.T * p.HG >> p.unit_shift) + (p.B < p.T ? p.B : p.T)) * p.G;
  p.by_heads = fast_div(static_cast<uint32_t>(p.HG));
  p.by_page = fast_div(static_cast<uint32_t>(p.page < 1 ? 1 : p.page));
  p.by_blocks = fast_div(static_cast<uint32_t>(p.G * per));
}

constexpr int64_t kMaxBlocks = (1 << 24) - 16;  // a launch has less than 2^32 threads
// Shares of at least 4 tiles (one sequence of 4096: 28 us).
constexpr int kMinTiles = 4;

// The most units a call is split into.  A unit fills a compute unit (two of them at D <= 160), so one
// round of them, or two where the blocks alone fill more than half a round (and any number of blocks
// past two rounds stays whole): 100 sequences of up to 20000 x 128 heads, 200 blocks, take 697 us whole,
// 457 as 512 units and 475 as 1024; 400 blocks of up to 16000 entries 977, 924 and 769.
int unit_slots(int64_t blocks, int64_t B, int D) {
  if (blocks > 512 || B > kPlanRows) return 0;
  if (blocks <= 128) return D <= 160 ? 512 : 256;
  return blocks <= 256 ? 512 : 1024;
}

// Whether a call is split in whose longest sequence a token may see so many tiles.  The joining launch
// and the second start of a compute unit cost some 7 and 15 us.  10 sequences x 128 heads over 8 tiles take
// 19.9 us whole and 23.2 split, 2 over 17 tiles 29.0 and 22.1; 140 blocks over 31 tiles 49 and 75, over 94
// tiles 115 and 102; 500 blocks over 125 tiles 290 and 317.  The host knows no lengths, so the table's room
// stands for them: short sequences in wide tables are split too (100 of 500 x 128 heads 34 us with a table of their
// width, 75 with one of 131072 entries).
bool splits(int64_t tiles, int64_t blocks) { return tiles > 12 && tiles > blocks / 2; }

int64_t align16_up(int64_t x) { return (x + 15) & ~static_cast<int64_t>(15); }

// The units that a call is split into (0: none is) by what a sequence can hold, or a token see: the room of its
// table, its window, first positions and new tokens, or its list (topk -1: none).
int call_slots(int64_t blocks, int64_t B, int64_t T, int D, int64_t room, int64_t window, int64_t first, int64_t topk) {
  int64_t most = room;
  if (window + first + T < most) most = window + first + T;
  if (topk >= 0) most = topk;
  return B && splits((most + kTile - 1) / kTile, blocks) ? unit_slots(blocks, B, D) : 0;
}

int64_t slot_bytes(int slots, int64_t blocks, int D) {
  return slots ? 16 + align16_up(static_cast<int64_t>(sizeof(JoinRow)) * blocks) + static_cast<int64_t>(slots) * 64 * 4 * (D + 2) : 0;
}

// A call's window: without one 2^31 - most_new, with which the position of no new token, as low as -most_new,
// overflows; it cuts no sequence, as the last of them is at most at room + most_new - 2 (attend's check).
bool has_window(int64_t window, int64_t most_new) { return window && window < (1ll << 31) - most_new; }
int64_t call_window(int64_t window, int64_t most_new) { return has_window(window, most_new) ? window : (1ll << 31) - most_new; }

}  // namespace
}  // namespace mzk

using namespace mzk;

extern "C" int mzk_paged_attend(const void* q, int64_t T, int H, int D, const int64_t* cu, int64_t B, int fmt, int nope,
                                const void* pool, int64_t pages, int page, const int32_t* tables, int64_t table_stride,
                                int64_t max_pages, const int64_t* lens, const int32_t* idx, int64_t idx_row_stride,
                                int topk, int64_t window, const float* sinks, void* workspace, int64_t workspace_bytes,
                                void* out, float* lse, int zero_tail, void* stream) {
  return mzk_paged_attend_first(q, T, H, D, cu, B, fmt, nope, pool, pages, page, tables, table_stride, max_pages, lens, idx,
                                idx_row_stride, topk, window, 0, sinks, workspace, workspace_bytes, out, lse, zero_tail, stream);
}

extern "C" int mzk_paged_attend_first(const void* q, int64_t T, int H, int D, const int64_t* cu, int64_t B, int fmt, int nope,
                                      const void* pool, int64_t pages, int page, const int32_t* tables, int64_t table_stride,
                                      int64_t max_pages, const int64_t* lens, const int32_t* idx, int64_t idx_row_stride,
                                      int topk, int64_t window, int64_t first, const float* sinks, void* workspace,
                                      int64_t workspace_bytes, void* out, float* lse, int zero_tail, void* stream) {
  MZK_CHECK_ARG(T >= 0 && B >= 0 && H >= 1 && D > 0, "paged_attend: bad sizes");
  MZK_CHECK_ARG(T < kNoWindow && B <= kMaxInt && H <= 65536 && pages >= 0 && pages <= kMaxInt && max_pages >= 0 &&
                    max_pages <= kMaxInt,
                "paged_attend: 2^30 tokens, or sizes of 2^31");
  MZK_CHECK_ARG(page >= 1, "paged_attend: pages of at least one entry");
  const int64_t most_new = cu ? T : 1;
  MZK_CHECK_ARG(max_pages * page <= kMaxInt - 64 - 2 * (T ? most_new - 1 : 0) && pages * page <= kMaxInt - 64 && topk <= kMaxInt - 64,
                "paged_attend: a sequence and a pool hold less than 2^31 entries, a sequence twice the new tokens less");
  MZK_CHECK_ARG(fmt == 0 || fmt == 1, "paged_attend: fmt must be 0 (bf16) or 1 (fp8-b128)");
  MZK_CHECK_ARG(window >= 0 && topk >= 0, "paged_attend: negative window or list");
  MZK_CHECK_ARG(first >= 0 && first < kNoWindow && (first == 0 || window > 0),
                "paged_attend: first positions, less than 2^30, go with a window");
  MZK_CHECK_ARG(cu || T == B, "paged_attend: without cu one token per sequence (%lld tokens, %lld sequences)",
                (long long)T, (long long)B);
  MZK_CHECK_ARG(!idx || (cu == nullptr && window == 0 && idx_row_stride >= topk),
                "paged_attend: a list of entries takes one token per sequence and no window, rows of at least topk");
  MZK_CHECK_ARG(table_stride >= max_pages, "paged_attend: table rows shorter than max_pages");
  if (T == 0) return MZK_OK;
  MZK_CHECK_ARG(q && out && lse && (B == 0 || (lens && (pool || pages == 0) && (tables || max_pages == 0))),
                "paged_attend: null pointer");
  MZK_CHECK_ARG(aligned16(q) && aligned16(pool) && aligned16(out) && aligned16(workspace),
                "paged_attend: q, pool, workspace and out must be 16-byte aligned");
  RaggedParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.T = T;
  p.H = p.HG = H;
  p.G = 1;
  p.D = D;
  p.cu = cu;
  p.B = B;
  p.lens = lens;
  p.entries = static_cast<const uint8_t*>(pool);
  p.entry_stride = fmt ? nope + nope / 32 + 2 * (D - nope) : 2 * D;
  // (null would mean packed entries; a table without columns is never read)
  p.tables = max_pages ? tables : reinterpret_cast<const int32_t*>(lens);
  p.table_stride = table_stride;
  p.max_pages = max_pages;
  p.pages = pages;
  p.page = page;
  p.idx = idx;
  p.idx_stride = idx_row_stride;
  p.topk = topk;
  p.window = static_cast<int>(call_window(window, most_new));
  p.past = has_window(window, most_new) ? p.window : -1;
  p.first = has_window(window, most_new) ? static_cast<int>(first) : 0;
  p.sinks = sinks;
  p.scale_log2 = (1.0f / __builtin_sqrtf(static_cast<float>(D))) * kLog2e;
  set_units(p);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.zero_tail = zero_tail;
  MZK_CHECK_ARG(p.blocks_max < kMaxBlocks && T * H <= kMaxInt - 64, "paged_attend: too many rows");
  p.min_tiles = kMinTiles;
  p.slots = call_slots(p.blocks_max, B, T, D, max_pages * page, p.window, p.first, idx ? topk : -1);
  const int64_t need = slot_bytes(p.slots, p.blocks_max, D);
  MZK_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "paged_attend: workspace needs %lld bytes",
                (long long)need);
  if (p.slots) {
    p.blocks_out = static_cast<int32_t*>(workspace);
    p.joins = reinterpret_cast<JoinRow*>(static_cast<uint8_t*>(workspace) + 16);
    p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 16 +
                                         align16_up(static_cast<int64_t>(sizeof(JoinRow)) * p.blocks_max));
    p.part_o = p.part_ml + static_cast<int64_t>(p.slots) * 64 * 2;
  }
  return dispatch_ragged("paged_attend", fmt, nope, p, as_stream(stream));
}

extern "C" int mzk_paged_attend_workspace_bytes(int64_t T, int H, int D, int packed, int64_t B, int64_t* bytes) {
  return mzk_paged_attend_call_workspace_bytes(T, H, D, packed, B, kMaxInt, 1, 0, -1, bytes);
}

extern "C" int mzk_paged_attend_call_workspace_bytes(int64_t T, int H, int D, int packed, int64_t B, int64_t max_pages,
                                                     int page, int64_t window, int topk, int64_t* bytes) {
  return mzk_paged_attend_first_workspace_bytes(T, H, D, packed, B, max_pages, page, window, 0, topk, bytes);
}

extern "C" int mzk_paged_attend_first_workspace_bytes(int64_t T, int H, int D, int packed, int64_t B, int64_t max_pages,
                                                      int page, int64_t window, int64_t first, int topk, int64_t* bytes) {
  MZK_CHECK_ARG(bytes != nullptr, "paged_attend_workspace_bytes: null output");
  MZK_CHECK_ARG(T >= 0 && B >= 0 && H >= 1 && D > 0 && max_pages >= 0 && max_pages <= kMaxInt && page >= 1 && window >= 0 &&
                    first >= 0 && first < kNoWindow && (first == 0 || window > 0),
                "paged_attend_workspace_bytes: bad sizes");
  MZK_CHECK_ARG(T <= kMaxInt && B <= kMaxInt && H <= 65536 && D <= 65536, "paged_attend_workspace_bytes: sizes of 2^31 or more");
  RaggedParams p{};
  p.T = T;
  p.HG = H;
  p.G = 1;
  p.B = B;
  const int64_t some = 0;
  p.cu = packed ? &some : nullptr;  // only whether there is one counts
  set_units(p);
  const int slots = call_slots(p.blocks_max, B, T, D, max_pages * page, call_window(window, packed ? T : 1),
                               has_window(window, packed ? T : 1) ? first : 0, topk);
  *bytes = slot_bytes(slots, p.blocks_max, D);
  return MZK_OK;
}

extern "C" int mzk_packed_mqa(const void* q, int64_t T, int H, int D, const int64_t* cu, int64_t B, const void* kv,
                              int64_t kv_row_stride, int G, int64_t window, const float* sinks, void* out, float* lse,
                              int zero_tail, void* stream) {
  return mzk_packed_mqa_first(q, T, H, D, cu, B, kv, kv_row_stride, G, window, 0, sinks, out, lse, zero_tail, stream);
}

extern "C" int mzk_packed_mqa_first(const void* q, int64_t T, int H, int D, const int64_t* cu, int64_t B, const void* kv,
                                    int64_t kv_row_stride, int G, int64_t window, int64_t first, const float* sinks, void* out,
                                    float* lse, int zero_tail, void* stream) {
  MZK_CHECK_ARG(T >= 0 && B >= 0 && H >= 1 && D > 0 && G >= 1, "packed_mqa: bad sizes");
  MZK_CHECK_ARG(T < kNoWindow && B <= kMaxInt && H <= 65536, "packed_mqa: 2^30 tokens, or sizes of 2^31");
  MZK_CHECK_ARG(H % G == 0, "packed_mqa: %d heads do not divide into %d latents", H, G);
  MZK_CHECK_ARG(window >= 0, "packed_mqa: negative window");
  MZK_CHECK_ARG(first >= 0 && first < kNoWindow && (first == 0 || window > 0),
                "packed_mqa: first positions, less than 2^30, go with a window");
  MZK_CHECK_ARG(kv_row_stride >= static_cast<int64_t>(G) * D && kv_row_stride % 8 == 0 && kv_row_stride < 1ll << 30,
                "packed_mqa: kv rows must be G * D apart or more, a multiple of 8 elements below 2^30");
  if (T == 0) return MZK_OK;
  MZK_CHECK_ARG(q && kv && cu && out && lse, "packed_mqa: null pointer");
  MZK_CHECK_ARG(aligned16(q) && aligned16(kv) && aligned16(out), "packed_mqa: q, kv and out must be 16-byte aligned");
  RaggedParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.T = T;
  p.H = H;
  p.G = G;
  p.HG = H / G;
  p.D = D;
  p.cu = cu;
  p.B = B;
  p.entries = static_cast<const uint8_t*>(kv);
  p.entry_stride = 2 * kv_row_stride;
  p.window = window && window < kNoWindow ? static_cast<int>(window) : kNoWindow;
  p.first = p.window < kNoWindow ? static_cast<int>(first) : 0;
  p.sinks = sinks;
  p.scale_log2 = (1.0f / __builtin_sqrtf(static_cast<float>(D))) * kLog2e;
  set_units(p);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.zero_tail = zero_tail;
  MZK_CHECK_ARG(p.blocks_max < kMaxBlocks && T * H <= kMaxInt - 64, "packed_mqa: too many rows");
  return dispatch_ragged("packed_mqa", kFmtBf16, D, p, as_stream(stream));
}
