// From logits to the next tokens: sampling behind temperature, top-k, top-p and min-p, verification of
// drafted tokens, and the step of a beam search.
//
// A row's tokens stand in the order of falling logits, equal ones by rising index.  With the weights
//   w_i = exp((l_i - max l) / T)
// top-k keeps the first k of the order, top-p the shortest prefix of those whose weights reach p of their
// sum, min-p those of at least min_p times the first one's weight: each keeps a prefix, so together the
// shortest.  The token drawn is the first whose running sum exceeds u times the kept sum W.  (T <= 0: the
// first of the order.)  NaN and -inf are no tokens; +inf counts as its type's largest finite number, -0 as 0.
//
// Tokens are whole numbers, so a token beside a border of the running sum has to come out right: weights are computed in 64 bits
// and summed as whole numbers, in any order the same.  A running sum's share of W is off by less than 2^-29:
//   bins      2^-44 of a weight for its second factor, and |t| 2^-52 ln 2 / 20 for its place t, at most 2^27 bins from
//             the origin: 2^-29.8, half of which can reach a share of W; half a unit of 1023 bins, 2^-33; what is too small to count,
//             2^20 tokens of 2^-51 each.  (Mostly t is below 2^10, and all of it some 2^-40.)
//   by value  2^-49 of a weight; half a unit of 2^-scale of each of at most 2^16 values, 2^-30 for rows of up to 2^17 tokens; each
//             doubling of a row's length doubles that, to 2^-27 for 2^20.
//
// No row is sorted.  What is to be found lies in few places of the order, and those are found from sums:
//   bins      weights are summed in bins of 1/20 octave, from the largest down, by atomic sums in LDS (survey);
//   by value  of bf16 logits the tokens of each of the 2^16 values are counted instead, and weights computed once a value.
// Running sums say in which bins (at which value) the cuts and the token are; the row is read once more to list its
// tokens there, and the token is selected among those.
// One workgroup does this for a row (row_kernel); where rows are fewer than compute units that way is bound by the 25 to
// 28 bytes a ns that one of them loads and by its arithmetic, and four launches share the work: bins of chunks of the
// row (survey_kernel), joined and searched (row_kernel), chunks listed (list_kernel), the selection (row_kernel).
//
// Measured: fp32, 1 row of 131072: 6.9 + 9.7 + 4.5 + 10.6 us in four launches, of which reading would be 0.1 us: bound
// by dependent steps, barriers and code that is executed once.  256 rows of 200019, with top-k, top-p and min-p by
// turns: 106 us a call: the first reading 58, at 3.5 TB/s near what memory gives (4.0), the second 23, from the caches.  bf16, 64
// rows of 131072: 43.5 us, of which the count 12.3 and the second reading 6.5; 160 drafted rows: 49.  fp16, 16 rows of 32000: 22 us.
#include "common.h"
#include "sampling_numbers.h"

namespace mzk {
namespace {

constexpr double kBelow = 1.0 - 0x1p-30, kAbove = 1.0 + 0x1p-30;  // slack of bounds
constexpr int kCap = 16384;  // listed tokens of a row
constexpr int64_t kMaxVocab = 1 << 20;
constexpr uint32_t kNone = 0xffffffffu;

enum Mode { kSample, kVerify, kBeams };

// What a survey finds besides its bins.
struct Surveyed {
  int top;    // the largest bin; kNoTop: no token
  float max;  // the largest logit
  float origin;
};

// What a row's bins say to the launches that list and finish it.
struct Plan {
  Surveyed r;
  int w0[4], w1[4];       // bins in which a cut or the token is (w1 < w0: none)
  float from[2], to[2];   // the logits to be listed
  double drafted_w;
};

// What a row leaves for the launches behind it.
struct Row {
  double kept;    // W, in units of 2^-scale
  uint64_t cut;   // key and index of the last token that top-k and top-p keep
  float max, origin;
  int32_t top, accepted, token;
};

struct Filter {
  const float* f;  // one for each row, or null: `all` for every row
  float all;
  __device__ float operator()(int row) const { return f ? f[row] : all; }
};

struct SamplingParams {
  const uint8_t* logits;
  int64_t stride;  // bytes from row to row
  int V, rows;
  int chunks, chunk_pieces;  // of a row's survey; 1: the row's workgroup surveys it
  int scale;                 // log2 of the whole number that stands for the weight at the largest bin: V of them stay below 2^63
  Mode mode;
  Filter temperature, top_p, min_p;
  const int32_t* top_k;
  int top_k_all;
  const float* u;  // [rows]
  // verify
  const int64_t* tokens;  // [rows]
  const int64_t* cu;      // [B + 1]
  int B;
  const float* draw;   // [B]
  const float* probs;  // [rows, V] or null
  int64_t probs_stride;
  int rest_chunks;
  // beams
  const float* scores;  // [rows]
  int width, keep;
  // workspace
  Surveyed* heads;   // [rows][chunks]
  uint64_t* hist;    // [rows][chunks][kBins] from the largest down
  uint32_t* counts;  // the same, tokens
  Plan* plans;       // [rows]
  uint64_t* sums;    // [rows][kBins] running sums of the joined bins
  uint32_t* sum_counts;
  uint32_t* listed;  // [rows]
  uint2* list;       // [rows][kCap] key; index, and the bin above bit 20
  Row* rowres;       // [rows]
  int32_t* refused;  // [B] the row of a refused token, or -1
  uint64_t* rest;    // [B][rest_chunks] sums of what the target has above the draft
  uint2* best;       // [rows][keep]
  uint32_t* nbest;   // [rows]
  // results
  int64_t* token;
  float* logprob;
  int64_t* accepted;
  int32_t* parents;
  float* out_scores;
};

// ---- numbers --------------------------------------------------------------------------------

// a b + c with c in scalar registers: left to itself the compiler copies c for the two-operand form.
__device__ __forceinline__ double fma_scalar(double a, double b, double c) {
  double d;
  asm volatile("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));  // (kept in this order)
  return d;
}

// 2^43 2^(r / 20) as a whole number for |r| <= 1/2, to about 2^-43.9: the power series to the sixth power, which is
// replaced by the lower ones that come nearest, but the constant one (its Chebyshev polynomial's), 2^-48; the last
// sum is with 2^52 more, which rounds it and leaves it in the low bits.
constexpr int kWhole = 43;
template <int N>
__device__ __forceinline__ void whole_exp2(const double (&r)[N], uint64_t (&w)[N]) {
  constexpr double c = kLn2D / kPerOctave, one = 8796093022208.0;
  // r^6 = (48 (r^4 / 4) - 18 (r^2 / 16)) / 32 nearly
  constexpr double c6 = one * c * c * c * c * c * c / 720.0;
  constexpr double by[6] = {one + 4503599627370496.0, one * c, one * c * c / 2.0 - c6 * 0.03515625, one * c * c * c / 6.0,
                            one * c * c * c * c / 24.0 + c6 * 0.375, one * c * c * c * c * c / 120.0};
  double e[N];
#pragma unroll
  for (int j = 0; j < N; ++j) e[j] = fma_scalar(r[j], by[5], by[4]);
#pragma unroll
  for (int i = 3; i >= 0; --i)
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = fma_scalar(e[j], r[j], by[i]);
#pragma unroll
  for (int j = 0; j < N; ++j) w[j] = static_cast<uint64_t>(__double_as_longlong(e[j])) & 0xfffffffffffffull;
}
__device__ __forceinline__ uint64_t whole_exp2(double r) {
  const double x[1] = {r};
  uint64_t w[1];
  whole_exp2(x, w);
  return w[0];
}

// log2 x for x >= 2^-190: the hardware's, a float32 of at most 128 and so off by some 2^-17, and what it leaves, 1 + d, by the series,
// whose first term left out is d^4 / 4 < 2^-68.
__device__ __forceinline__ double log2_of(double x) {
  const double y = static_cast<double>(__builtin_amdgcn_logf(static_cast<float>(x * 0x1p64))) - 64.0;
  const double d = x * exp2_of(-y) - 1.0;
  return y + (d - d * d * (0.5 - d * (1.0 / 3.0))) * kLog2eD;
}

// A random number as one of [0, 1): NaN as 0.
__device__ __forceinline__ double unit(float u) { return u > 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0; }

constexpr float kBig = 3.402823466e38f;
// A logit as it counts: NaN as -inf, +inf as its type's largest finite number, -0 as 0.
template <int DT>
__device__ __forceinline__ float logit_of(float x) {
  constexpr float big = DT == MZK_F32 ? kBig : DT == MZK_BF16 ? 0x1.fep127f : 65504.0f;
  return x != x ? -__builtin_huge_valf() : fminf(x + 0.0f, big);
}
// Keys rise as logits fall.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float logit_of_key(uint32_t ik) { return __uint_as_float(ik & 0x80000000u ? ik : ~ik & 0x7fffffffu); }

// ---- a row's settings -------------------------------------------------------------------------

struct Settings {
  double s;    // 20 log2 e / T: bins of a logit
  int k;       // 0: none
  double p;    // 1: none
  double f;    // 20 log2 min_p; -inf: none
  bool first;  // T <= 0: the first of the order
};
__device__ __forceinline__ Settings settings(const SamplingParams& q, int row) {
  Settings z;
  const bool beams = q.mode == kBeams;
  const float t = beams ? 1.0f : q.temperature(row);
  z.first = !(t > 0.0f);
  z.s = kPerOctave * kLog2eD / (z.first ? 1.0 : static_cast<double>(t));
  z.k = beams ? q.keep : q.top_k ? q.top_k[row] : q.top_k_all;
  if (!beams && (z.k < 0 || z.k >= q.V)) z.k = 0;
  const float p = beams ? 1.0f : q.top_p(row);
  z.p = z.first ? 0.0 : p < 1.0f ? (p > 0.0f ? static_cast<double>(p) : 0.0) : 1.0;
  const float f = beams ? 0.0f : q.min_p(row);
  z.f = f > 0.0f ? (f < 1.0f ? kPerOctave * log2_of(static_cast<double>(f)) : 0.0) : -__builtin_huge_val();
  if (z.first) z.k = 0, z.f = -__builtin_huge_val();
  return z;
}

// ---- loads ------------------------------------------------------------------------------------

// A row in pieces of 16 bytes of memory: the whole ones in order, then what of the row lies before them and behind
// them, filled up with -inf; those two are laid into LDS by `edges`, before a barrier of the caller.
template <int DT>
struct Pieces {
  static constexpr int SIZE = DT == MZK_F32 ? 4 : 2, N = 16 / SIZE;
  const uint8_t* row;
  int V, head, whole;  // elements before the first whole piece, whole pieces
  const uint4* edge;   // [2] in LDS
  __device__ Pieces(const uint8_t* r, int v, const uint4* e) : row(r), V(v), edge(e) {
    head = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(r) & 15u)) & 15u) / SIZE;
    if (head > V) head = V;
    whole = (V - head) / N;
  }
  __device__ void edges(int tid, uint4* e) const {
    if (tid >= 2 * N) return;
    const int i = tid < N ? tid : tid - N + head + whole * N;
    const uint32_t bits = i < (tid < N ? head : V) ? raw(i) : DT == MZK_F32 ? 0xff800000u : DT == MZK_BF16 ? 0xff80u : 0xfc00u;
    if constexpr (DT == MZK_F32) reinterpret_cast<uint32_t*>(e)[tid] = bits;
    else reinterpret_cast<uint16_t*>(e)[tid] = static_cast<uint16_t>(bits);
  }
  __device__ int count() const { return whole + 2; }
  __device__ int first(int piece) const { return piece < whole ? head + piece * N : piece == whole ? 0 : head + whole * N; }  // index of its first element
  __device__ uint32_t raw(int i) const {
    if constexpr (DT == MZK_F32) return reinterpret_cast<const uint32_t*>(row)[i];
    else return reinterpret_cast<const uint16_t*>(row)[i];
  }
  __device__ static float value(uint32_t bits) {
    return DT == MZK_F32 ? __uint_as_float(bits) : DT == MZK_BF16 ? bf16_to_f32(static_cast<uint16_t>(bits)) : f16_to_f32(static_cast<uint16_t>(bits));
  }
  __device__ float operator[](int i) const { return logit_of<DT>(value(raw(i))); }
  static constexpr float BIG = DT == MZK_F32 ? kBig : DT == MZK_BF16 ? 0x1.fep127f : 65504.0f;
  // a piece with its type's largest finite number in the place of +inf
  __device__ static uint4 finite(uint4 x) {
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      constexpr uint32_t inf = DT == MZK_F32 ? 0x7f800000u : DT == MZK_BF16 ? 0x7f80u : 0x7c00u;
      if (DT == MZK_F32) {
        w[j] -= w[j] == inf;
      } else {
        w[j] -= (w[j] & 0xffffu) == inf;
        w[j] -= (w[j] >> 16) == inf ? 0x10000u : 0u;
      }
    }
    return uint4{w[0], w[1], w[2], w[3]};
  }
  __device__ uint4 load(int piece, int end) const {  // from `end` on: -inf
    if (piece < whole && piece < end) return *reinterpret_cast<const uint4*>(row + (head + static_cast<int64_t>(piece) * N) * SIZE);
    if (piece >= end) return none();
    return edge[piece - whole];
  }
  __device__ static uint4 none() {
    constexpr uint32_t w = DT == MZK_F32 ? 0xff800000u : DT == MZK_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    return uint4{w, w, w, w};
  }
  // f(index, logit as it counts) for the thread's tokens, by a loop of little code with four pieces in flight.  (With
  // a load for each token, 2 fp32 rows of 131072 equal logits took 2080 us.)
  template <int NT, typename F>
  __device__ __forceinline__ void walk(int tid, F f) const {
    const int pieces = count();
    uint4 n0 = load(tid, pieces), n1 = load(tid + NT, pieces), n2 = load(tid + 2 * NT, pieces), n3 = load(tid + 3 * NT, pieces);
#pragma unroll 1
    for (int p = tid; p < pieces; p += NT) {
      uint32_t w0 = n0.x, w1 = n0.y, w2 = n0.z, w3 = n0.w;
      n0 = n1, n1 = n2, n2 = n3;
      n3 = load(p + 4 * NT, pieces);
      const int i0 = first(p);
#pragma unroll 1
      for (int e = 0; e < N; ++e) {
        const float l = logit_of<DT>(value(SIZE == 4 ? w0 : w0 & 0xffffu));
        if (l > -__builtin_huge_valf()) f(i0 + e, l);
        if (SIZE == 4) {
          w0 = w1, w1 = w2, w2 = w3;
        } else {
          w0 = w0 >> 16 | w1 << 16, w1 = w1 >> 16 | w2 << 16, w2 = w2 >> 16 | w3 << 16, w3 >>= 16;
        }
      }
    }
  }
  // element j (of N) of a loaded piece, not yet as it counts
  __device__ static float at(const uint4& x, int j) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    return DT == MZK_F32 ? value(w[j]) : value(w[j / 2] >> (16 * (j & 1)) & 0xffffu);
  }
};

// The sequence of a row of packed ones and the row behind its last; false: none.  The first that ends behind the row, by 64 of
// them at a time, evenly spaced: 2 dependent loads for 4096 sequences, 4 for 2^22.  (One after another, 65536 rows of as many
// sequences took 27.8 ms, of which reading and drawing is 3.8.)
__device__ __forceinline__ bool sequence_of(const SamplingParams& q, int row, int lane, int& b, int& end) {
  b = 0;
  for (int n = q.B; n > 0;) {  // among b .. b + n - 1
    const int step = (n + 63) / 64, last = (lane + 1) * step < n ? (lane + 1) * step - 1 : n - 1;
    const uint64_t in = __ballot(q.cu[b + last + 1] > row);
    if (in == 0) return false;
    const int before = __builtin_ctzll(in) * step;
    b += before;
    n = step < n - before ? step : n - before;
    if (step == 1) break;
  }
  if (q.B == 0) return false;
  const int64_t e = q.cu[b + 1];
  end = e < q.rows ? static_cast<int>(e) : q.rows;
  return q.cu[b] <= row;
}

// Across the wave with data-parallel moves: steps of 1, 2, 4, 8 within 16 lanes, then the sums of the lanes before.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, ROWS == 0xf));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  return static_cast<uint64_t>(moved<CTRL, ROWS>(static_cast<uint32_t>(v >> 32))) << 32 | moved<CTRL, ROWS>(static_cast<uint32_t>(v));
}
// The sums up to each lane.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)); }
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  return static_cast<uint64_t>(lane_of(static_cast<uint32_t>(v >> 32), lane)) << 32 | lane_of(static_cast<uint32_t>(v), lane);
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) { return lane_of(wave_scan(v), 63); }
// The largest of the wave (a NaN is none).
template <int CTRL, int ROWS>
__device__ __forceinline__ float larger(float v) {
  const int low = __float_as_int(-__builtin_huge_valf());
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(low, __float_as_int(v), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {
  v = larger<0x111, 0xf>(v);
  v = larger<0x112, 0xf>(v);
  v = larger<0x114, 0xf>(v);
  v = larger<0x118, 0xf>(v);
  v = larger<0x142, 0xa>(v);
  v = larger<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// ---- survey -------------------------------------------------------------------------------------

// Where a logit lies: t = (l - origin) s, in bins; its bin is the nearest whole number k, and its weight 2^(k / 20)
// times 2^((t - k) / 20).  A bin sums the second factors, as whole numbers of 2^43; the first is its own.
struct Grid {
  float origin;
  double s;
  __device__ double place(float l) const { return (static_cast<double>(l) - static_cast<double>(origin)) * s; }
};

// The origin: the largest of the row's first 1024 logits, the same for all its chunks.  With equal logits the
// second factors are 1, and sums of them exact.
template <int DT, int NT>
__device__ __forceinline__ float origin_of(const Pieces<DT>& x, int tid, float* lds) {
  float m = -__builtin_huge_valf();
  for (int i = tid; i < 1024 && i < x.V; i += NT) m = fmaxf(m, x[i]);
  m = wave_max(m);
  if ((tid & 63) == 0) lds[tid >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) m = fmaxf(m, lds[w]);
  __syncthreads();
  return m > -__builtin_huge_valf() ? m : 0.0f;
}

constexpr int kSurveyThreads = 1024, kSurveyElements = 16;  // of a chunk's workgroup; of its thread at once
constexpr int kAside = 64;     // places behind the bins for what is too small to count
constexpr int kFar = 1 << 28;  // bins from the origin that are told apart

// The bin of a maximum.
__device__ __forceinline__ int top_of(const Grid& g, float m) {
  return static_cast<int>(__builtin_rint(fmin(fmax(g.place(m), -static_cast<double>(kFar)), static_cast<double>(kFar))));
}

// Pieces from .. to - 1 of a row into the histogram (and, counting, the numbers of tokens): bin k in place k mod
// kBins, for the kBins - 1 bins from the largest on.  As that rises, places of bins that fall behind become its.
// Bound by memory where all compute units read, else by the arithmetic, some 20 instructions an element, 12 of them in 64
// bits (110 cycles a wave, of which they are 80; the atomic sums hide behind them: 56 us of 58 with narrower ones).
template <int DT, int NT, int AHEAD>
__device__ __forceinline__ Surveyed survey(const Pieces<DT>& x, const Grid& g, bool counting, int from, int to, int tid,
                                           unsigned long long* hist /* [kBins][kCopies], and kAside */, uint32_t* counts /* the same */,
                                           int* tops /* [2] */, float* lds /* [NT / 64] */) {
  using P = Pieces<DT>;
  constexpr int PER = AHEAD, ELEMENTS = PER * P::N;
  for (int i = tid; i < kCopies * kBins; i += NT) hist[i] = 0;
  if (counting)
    for (int i = tid; i < kCopies * kBins; i += NT) counts[i] = 0;
  if (tid < 2) tops[tid] = kNoTop;
  uint4 next[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) next[i] = x.load(from + i * NT + tid, to);
  float known = -__builtin_huge_valf();  // a maximum of this wave's that the others have heard of
  int top = kNoTop, turn = 0;
  // offsets in bytes: the copy's, and a place's that nobody reads
  const int copy = 8 * (tid & (kCopies - 1)), aside = 8 * (kCopies * kBins + (tid & 63));
  __syncthreads();
  for (int at = from; at < to; at += PER * NT) {
    uint4 now[PER];
    float m = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      now[i] = next[i];
#pragma unroll
      for (int j = 0; j < P::N; ++j) m = fmaxf(m, P::at(now[i], j));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int piece = at + (PER + i) * NT + tid;
      if (at + PER * NT < to) next[i] = x.load(piece, to);
    }
    if (__ballot(m > known)) {
      known = wave_max(m);
      if ((tid & 63) == 0) atomicMax(&tops[turn], top_of(g, logit_of<DT>(known)));
    }
    __syncthreads();
    const int risen = max(top, tops[turn]);
    turn ^= 1;
    if (risen > top) {  // uniform
      if (top > kNoTop) {
        const int n = risen - top < kBins ? risen - top : kBins;
        for (int i = tid; i < n * kCopies; i += NT) {
          const int j = ((risen - i / kCopies) & kRest) * kCopies + i % kCopies;
          hist[j] = 0;
          if (counting) counts[j] = 0;
        }
        __syncthreads();
      }
      top = risen;
    }
    if (__ballot(m > P::BIG)) {
#pragma unroll
      for (int i = 0; i < PER; ++i) now[i] = P::finite(now[i]);
    }
    const double bottom = bottom_of(top);
#pragma unroll
    for (int i = 0; i < ELEMENTS; i += 4) {  // (four at a time, so that the steps of one wait for nothing)
      double t[4];
      uint64_t w[4];
      int k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = g.place(P::at(now[(i + j) / P::N], (i + j) % P::N));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // the nearest whole number: the low bits of the sum with 3 2^51
        const double sum = t[j] + 0x1.8p52, n = sum - 0x1.8p52;
        k[j] = place_of(sum) | copy;
        k[j] = n > bottom ? k[j] : aside;  // (not of a NaN, nor of -inf)
        t[j] = t[j] - n;
      }
      whole_exp2(t, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) atomicAdd(reinterpret_cast<unsigned long long*>(reinterpret_cast<uint8_t*>(hist) + k[j]), static_cast<unsigned long long>(w[j]));
      if (counting) {
#pragma unroll
        for (int j = 0; j < 4; ++j) atomicAdd(&counts[k[j] >> 3], 1u);
      }
    }
  }
  float max_all = known;
  if ((tid & 63) == 0) lds[tid >> 6] = max_all;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) max_all = fmaxf(max_all, lds[w]);
  return Surveyed{top, logit_of<DT>(max_all), g.origin};
}

// Bin j from the largest down.
__device__ __forceinline__ void surveyed_bin(const Surveyed& r, int j, bool counting, const unsigned long long* hist, const uint32_t* counts,
                                             uint64_t& sum, uint32_t& num) {
  sum = 0;
  num = 0;
  if (j >= kRest) return;
  const int i = ((r.top - j) & kRest) * kCopies;
#pragma unroll
  for (int c = 0; c < kCopies; ++c) sum += hist[i + c];
  if (counting)
#pragma unroll
    for (int c = 0; c < kCopies; ++c) num += counts[i + c];
}

template <int DT>
__global__ void __launch_bounds__(kSurveyThreads) survey_kernel(const SamplingParams q) {
  __shared__ unsigned long long hist[kCopies * kBins + kAside];
  __shared__ uint32_t counts[kCopies * kBins + kAside];
  __shared__ float lds[kSurveyThreads / 64];
  __shared__ int tops[2];
  const int tid = threadIdx.x;
  // workgroups go to the 8 XCDs in turn: a row's chunks to the one that its own workgroup reads it from again
  const int of8 = blockIdx.x >> 3, row = of8 / q.chunks * 8 + (blockIdx.x & 7), chunk = of8 % q.chunks;
  if (row >= q.rows || (q.mode == kVerify && q.cu[q.B] <= row)) return;  // (a row of no sequence)
  __shared__ uint4 edge[2];
  const Pieces<DT> x(q.logits + row * q.stride, q.V, edge);
  x.edges(tid, edge);  // (barriers follow)
  const Settings z = settings(q, row);
  const bool counting = z.k > 0;
  const Grid g{origin_of<DT, kSurveyThreads>(x, tid, lds), z.s};
  const int from = chunk * q.chunk_pieces, all = x.count(), to = from + q.chunk_pieces < all ? from + q.chunk_pieces : all;
  const Surveyed r = survey<DT, kSurveyThreads, kSurveyElements / Pieces<DT>::N>(x, g, counting, from, to, tid, hist, counts, tops, lds);
  const int64_t at = static_cast<int64_t>(row) * q.chunks + chunk;
  if (tid == 0) q.heads[at] = r;
  if (r.top == kNoTop) return;  // uniform
  for (int j = tid; j < kBins; j += kSurveyThreads) {
    uint64_t sum;
    uint32_t num;
    surveyed_bin(r, j, counting, hist, counts, sum, num);
    q.hist[at * kBins + j] = sum;
    if (counting) q.counts[at * kBins + j] = num;
  }
}

// ---- list -----------------------------------------------------------------------------------------

// The tokens of a chunk with logits in the plan's ranges.
template <int DT>
__global__ void __launch_bounds__(kSurveyThreads) list_kernel(const SamplingParams q) {
  using P = Pieces<DT>;
  constexpr int NT = kSurveyThreads, NW = NT / 64, PER = kSurveyElements / P::N;
  __shared__ uint32_t part[NW], base;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int of8 = blockIdx.x >> 3, row = of8 / q.chunks * 8 + (blockIdx.x & 7), chunk = of8 % q.chunks;
  if (row >= q.rows || (q.mode == kVerify && q.cu[q.B] <= row)) return;
  __shared__ uint4 edge[2];
  const P x(q.logits + row * q.stride, q.V, edge);
  x.edges(tid, edge);
  __syncthreads();
  const int first = chunk * q.chunk_pieces, all = x.count(), end = first + q.chunk_pieces < all ? first + q.chunk_pieces : all;
  uint4 next[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) next[i] = x.load(first + i * NT + tid, end);
  const Plan p = q.plans[row];
  const Grid g{p.r.origin, settings(q, row).s};
  if (fmaxf(p.to[0], p.to[1]) == -__builtin_huge_valf()) return;  // uniform: no list
  for (int at = first; at < end; at += PER * NT) {
    uint4 now[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      now[i] = next[i];
      const int piece = at + (PER + i) * NT + tid;
      if (at + PER * NT < end) next[i] = x.load(piece, end);
    }
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kSurveyElements; ++i) {
      const float l = P::at(now[i / P::N], i % P::N);  // (a NaN is in no range)
      mine |= static_cast<uint32_t>((l >= p.from[0] && l <= p.to[0]) || (l >= p.from[1] && l <= p.to[1])) << i;
    }
    const uint32_t many = __popc(mine), s = wave_scan(many);
    if (lane == 63) part[wave] = s;
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < wave) before += part[w];
      total += part[w];
    }
    if (tid == 0 && total) base = atomicAdd(&q.listed[row], total);
    __syncthreads();
    uint32_t to = base + before + s - many;
#pragma unroll
    for (int i = 0; i < kSurveyElements; ++i) {
      if (mine >> i & 1u) {
        const float l = logit_of<DT>(P::at(now[i / P::N], i % P::N));
        const int j = static_cast<int>(fmin(static_cast<double>(p.r.top) - __builtin_rint(g.place(l)), static_cast<double>(kRest)));
        const int idx = x.first(at + i / P::N * NT + tid) + i % P::N;
        if (to < kCap) q.list[static_cast<int64_t>(row) * kCap + to] = uint2{key_of(l), static_cast<uint32_t>(idx) | static_cast<uint32_t>(j) << 20};
        ++to;
      }
    }
  }
}

// ---- a row --------------------------------------------------------------------------------------

constexpr int kRowThreads = kBins / 2;
constexpr int kMostChunks = 64;
constexpr int kDigits = 1024;  // of a selection's step
constexpr int kByValue = 16384;  // longer rows of bf16 logits are counted by value
// LDS of a row's workgroup: its own arrays, and behind them the list with the hot values' places, or a survey's bins.  The plan's
// launch asks for no more than any kernel has, the others for what a compute unit has.
constexpr int kRowStaticLds = 26 * 1024;
constexpr int kRowLds = kCap * static_cast<int>(sizeof(uint2)) + 4 * kRowThreads, kBinsLds = 12 * (kCopies * kBins + kAside);
static_assert(kBinsLds <= kRowLds && kBinsLds + kRowStaticLds <= 64 * 1024 && kRowLds + kRowStaticLds <= 160 * 1024, "LDS");

// A row in one launch, or, where its chunks are surveyed and listed by workgroups of their own, in two: up to the bins
// in which something is to be found, and from the list on.
enum Part { kWholeRow, kPlanPart, kFinishPart };

template <int DT, Part PART>
__global__ void __launch_bounds__(kRowThreads) row_kernel(const SamplingParams q) {
  constexpr int NT = kRowThreads, NW = NT / 64;
  constexpr int KS = DT == MZK_F32 ? 0 : DT == MZK_BF16 ? 16 : 13;  // low bits of a key that are all the same
  using P = Pieces<DT>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint2* const list = reinterpret_cast<uint2*>(smem);  // [kCap] key; index, and the bin above bit 20
  // (the survey's bins are there before the list is)
  unsigned long long* const bins = reinterpret_cast<unsigned long long*>(smem);
  uint32_t* const bin_counts = reinterpret_cast<uint32_t*>(smem + 8 * (kCopies * kBins + kAside));
  __shared__ unsigned long long hist[kDigits];
  __shared__ uint32_t counts[kDigits];
  __shared__ uint64_t cw[kBins];  // running sums of the bins' weights
  __shared__ uint32_t cn[kBins];  // and of their tokens
  __shared__ uint64_t part[NW], sel[4], last_ones[64][2];
  __shared__ uint32_t partn[NW], number[2];
  __shared__ int found[2][2][NW];
  __shared__ float lds[NW];
  __shared__ int tops[kMostChunks];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
  int b = 0, end = 0;
  if (q.mode == kVerify && !sequence_of(q, row, lane, b, end)) return;  // uniform
  __shared__ uint4 edge[2];
  const P x(q.logits + row * q.stride, q.V, edge);
  static_assert(sizeof(hist) + sizeof(counts) + sizeof(cw) + sizeof(cn) + sizeof(part) + sizeof(sel) + sizeof(last_ones) + sizeof(partn) +
                        sizeof(number) + sizeof(found) + sizeof(lds) + sizeof(tops) + sizeof(edge) <= kRowStaticLds, "row_kernel's static LDS");
  x.edges(tid, edge);
  __syncthreads();
  const Settings z = settings(q, row);
  const bool counting = z.k > 0;

  // ---- the row's histogram: bins 2 tid, 2 tid + 1, from the largest down, are this thread's ----
  Plan* const plan = q.plans + row;
  Grid g{PART == kWholeRow ? 0.0f : PART == kPlanPart ? q.heads[static_cast<int64_t>(row) * q.chunks].origin : plan->r.origin, z.s};
  uint64_t sum[2] = {0, 0};  // of the second factors
  uint32_t num[2] = {0, 0};
  Surveyed r{kNoTop, -__builtin_huge_valf(), 0.0f};
  bool by_value = false;  // bf16 logits: the counts of their values say where to look
  // ---- bf16 logits: how many tokens have each value ----
  // (64 rows, by value and with bins: of 8192 logits 25.4 and 23.5 us, 16384 26.2 and 27.2, 32768 30.6 and 34.2, 131072 45.5 and 63.2)
  // Two counters a word, the negative value's above the positive's, from the order's first 128 values (a block) on:
  // block j is thread j's.  A counter that passes 2^16 is found out by the sum of all.
  uint32_t* const tally = reinterpret_cast<uint32_t*>(smem);
  [[maybe_unused]] uint64_t reached = 0;  // the weights of the tokens that reach min-p
  // value o (of 2^16) of the order, 0 the largest of its sign's patterns
  auto pattern = [&](uint32_t o) -> uint32_t { return o < 0x8000u ? 0x7fffu - o : o; };
  auto value_of = [&](uint32_t o) -> float { return P::value(pattern(o)); };
  // the counters of values o, o + 1 (o even)
  auto tallied = [&](uint32_t o, uint32_t& c0, uint32_t& c1) __attribute__((always_inline)) {
    const uint2 w = *reinterpret_cast<const uint2*>(tally + (pattern(o) & 0x7ffeu));
    c0 = o < 0x8000u ? w.y & 0xffffu : w.x >> 16;
    c1 = o < 0x8000u ? w.x & 0xffffu : w.y >> 16;
  };
  auto weight = [&](float l) __attribute__((always_inline)) -> double { return weight_of(l, r.max, z.s, q.scale); };
  if (DT == MZK_BF16 && PART == kWholeRow && q.V > kByValue) {
    // blocks of numbers: before them NaN and +inf, behind them -inf and NaN
    constexpr int FIRST = 1, END = 511, INF = 0x7f80, AHEAD = 8;
    for (int i = tid; i < 8192; i += NT) reinterpret_cast<uint4*>(tally)[i] = uint4{0, 0, 0, 0};
    uint4 next[AHEAD];
    const int pieces = x.count();
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) next[a] = x.load(a * NT + tid, pieces);
    __syncthreads();
    uint32_t all = 0;
    // A value that many lanes have, as that of a masked vocabulary, would be summed one lane after the other: each wave has a
    // hot one, looked for in the first and the last of every 8 pieces, whose tokens each lane sums in a place of its own.
    // (80 rows of 131072, whole calls: 45 us, 44 without this; all but 5000 tokens masked at random 45, and 178.)
    uint8_t* const at = reinterpret_cast<uint8_t*>(tally);
    uint32_t* const own = tally + 32768 + tid;
    const uint32_t own_at = 4u * (32768u + tid);
    uint32_t hot = 0xffffu;  // (a NaN)
    *own = 0;
    auto flush = [&]() {  // (its lanes' own; the order of a wave's accesses is kept)
      const uint32_t n = *own;
      if (hot == 0xff80u) all -= n >> 16;  // -inf: no tokens
      else if (const uint32_t sum = wave_sum(n); lane == 0 && sum) atomicAdd(&tally[hot & 0x7fffu], sum);
      *own = 0;
    };
    for (int p0 = 0; p0 < pieces; p0 += AHEAD * NT) {
      {
        const bool full = p0 + AHEAD * NT <= pieces;  // (behind the row -inf is loaded)
        const uint32_t v0 = next[0].x & 0xffffu, v1 = (full ? next[AHEAD - 1].x : next[0].x) & 0xffffu;
        const uint32_t c0 = lane_of(v0, 0), c1 = lane_of(v1, 37);
        const int n0 = __popcll(__ballot(v0 == c0)), n1 = __popcll(__ballot(v1 == c1));
        const uint32_t c = n0 >= n1 ? c0 : c1;
        if (max(n0, n1) >= 6 && c != hot) {  // uniform
          flush();
          hot = c;
        }
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const uint32_t v[4] = {next[a].x, next[a].y, next[a].z, next[a].w};
        const int piece = p0 + (AHEAD + a) * NT + tid;
        if (p0 + AHEAD * NT < pieces) next[a] = x.load(piece, pieces);
        if (p0 + a * NT + tid >= pieces) continue;
        all += P::N;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t low = (v[i] & 0xffffu) == hot ? own_at : v[i] << 2 & 0x1fffcu, high = v[i] >> 16 == hot ? own_at : v[i] >> 14 & 0x1fffcu;
          atomicAdd(reinterpret_cast<uint32_t*>(at + low), 1u + (v[i] >> 15 & 1u) * 0xffffu);
          atomicAdd(reinterpret_cast<uint32_t*>(at + high), 1u + (v[i] >> 31) * 0xffffu);
        }
      }
    }
    flush();
    all = wave_sum(all);
    if (lane == 0) partn[wave] = all;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) all += partn[w];
    if (tid == 0) {  // -0 is 0, +inf the largest number
      const uint32_t zero = tally[0], most = tally[INF - 1];
      const uint32_t z2 = (zero & 0xffffu) + (zero >> 16), m2 = (most & 0xffffu) + (tally[INF] & 0xffffu);
      tally[0] = z2;
      tally[INF - 1] = (most & 0xffff0000u) | (m2 & 0xffffu);
      tally[INF] &= 0xffff0000u;
      number[0] = z2 > 0xffffu || m2 > 0xffffu;
    }
    __syncthreads();
    cw[tid] = 0;
    uint32_t mine = 0;  // tokens of block tid: 128 words, from another one on in every lane, so that no two meet
    {
      const uint32_t* const words = tally + (tid < 256 ? 255 - tid : tid - 256) * 128;
      const int sh = tid < 256 ? 0 : 16;
#pragma unroll 16
      for (int i = 0; i < 128; ++i) mine += words[(i + tid) & 127] >> sh & 0xffffu;
      cn[tid] = mine;
    }
    // the first block of numbers with a token, and the sum of all counters
    const uint64_t some = __ballot(mine != 0 && tid >= FIRST && tid < END);
    const uint32_t sums = wave_sum(mine);
    if (lane == 0) found[0][0][wave] = some ? 64 * wave + __builtin_ctzll(some) : END, partn[wave] = sums;
    __syncthreads();
    int first = END;
    uint32_t counted = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) first = min(first, found[0][0][w]), counted += partn[w];
    const bool exact = counted == all && number[0] == 0;
    by_value = true;
    if (first < END) {
      uint32_t c0, c1;
      tallied(128u * first + 2u * lane, c0, c1);
      const int at = __builtin_ctzll(__ballot((c0 | c1) != 0));
      r.max = value_of(128u * first + 2u * at + (lane_of(c0, at) ? 0u : 1u));
      r.top = 0;
      g.origin = r.max;
    }
    // blocks with weights that count
    const bool light = !(first < END) || tid < first || !(g.place(value_of(128u * tid)) > -static_cast<double>(kRest));
    const uint64_t heavy = __ballot(!light);
    __syncthreads();
    if (lane == 0) found[0][0][wave] = __popcll(heavy);
    __syncthreads();
    int end_heavy = first;
#pragma unroll
    for (int w = 0; w < NW; ++w) end_heavy += found[0][0][w];
    end_heavy = min(end_heavy, END);
    int end_count = END;
    if (__builtin_expect(!exact, 0)) {
      // Some counter has run over.  It may be one of those that do not count, as of a masked vocabulary: are the
      // others' tokens as many as there are?
      end_count = end_heavy;
      const float least = first < END ? value_of(128u * end_heavy - 1u) : -P::BIG;
      uint32_t are = 0;
      for (int p0 = tid; p0 < pieces; p0 += 8 * NT) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x.load(p0 + i * NT, pieces);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < P::N; ++e) are += P::at(v[i], e) >= least;
      }
      const uint32_t theirs = wave_sum(tid < end_count && tid >= FIRST ? mine : 0u), seen = wave_sum(are);
      if (lane == 0) partn[wave] = theirs - seen;
      __syncthreads();
      uint32_t differ = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) differ += partn[w];
      by_value = differ == 0 && number[0] == 0 && q.mode != kBeams;
      __syncthreads();
    }
    if (by_value && first < END) {
      // the blocks whose weights count, one after another
      const uint64_t live = __ballot(tid >= first && tid < end_heavy && mine != 0);
      if (lane == 0) found[1][0][wave] = __popcll(live);
      __syncthreads();
      int before_me = 0, lives = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w < wave) before_me += found[1][0][w];
        lives += found[1][0][w];
      }
      if (live >> lane & 1u) counts[before_me + __popcll(live & ((1ull << lane) - 1ull))] = static_cast<uint32_t>(tid);
      __syncthreads();
      uint64_t reach = 0;
      const double m = static_cast<double>(r.max);
      for (int i = 2 * wave; i < lives; i += 2 * NW) {
        float l[4];
        uint32_t c[4];
        int j[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          j[e] = static_cast<int>(counts[i + e < lives ? i + e : i]);
          const uint32_t o = 128u * j[e] + 2u * lane;
          tallied(o, c[2 * e], c[2 * e + 1]);
          l[2 * e] = value_of(o);
          l[2 * e + 1] = value_of(o + 1u);
        }
        uint64_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = static_cast<uint64_t>(static_cast<double>(c[e]) * weight(l[e]) + 0.5);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (i + e >= lives) continue;
          const uint64_t s = wave_sum(w[2 * e] + w[2 * e + 1]);
          if (lane == 0) cw[j[e]] = s;
          if (z.f > -__builtin_huge_val())
            reach += wave_sum(((static_cast<double>(l[2 * e]) - m) * z.s >= z.f ? w[2 * e] : 0) + ((static_cast<double>(l[2 * e + 1]) - m) * z.s >= z.f ? w[2 * e + 1] : 0));
        }
      }
      __syncthreads();
      if (tid < FIRST || tid >= end_count) mine = 0;
      uint64_t w = wave_scan(cw[tid]);
      uint32_t k = wave_scan(mine);
      if (lane == 63) part[wave] = w, partn[wave] = k;
      if (lane == 0) last_ones[wave][0] = reach;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        if (i < wave) w += part[i], k += partn[i];
        reached += last_ones[i][0];
      }
      cw[tid] = w;
      cn[tid] = k;
    }
    __syncthreads();
  }
  if (PART == kWholeRow && !by_value) g.origin = origin_of<DT, NT>(x, tid, lds);
  if (PART == kFinishPart) r = plan->r;
  for (bool whole_row = PART == kWholeRow; PART != kFinishPart && !by_value; whole_row = true) {
    if (whole_row) {
      // (8 pieces at a time are more code to fetch than they gain: 64 rows of 4096, bf16, 27.6 us and 24.7 with 4, 23.5 with 2;
      // 256 rows of 200019, fp32, 94.0, 93.5 and 99.1)
      r = survey<DT, NT, 4>(x, g, counting, 0, x.count(), tid, bins, bin_counts, tops, lds);
      if (r.top > kNoTop) {
        surveyed_bin(r, 2 * tid, counting, bins, bin_counts, sum[0], num[0]);
        surveyed_bin(r, 2 * tid + 1, counting, bins, bin_counts, sum[1], num[1]);
      }
    } else {
      const Surveyed h = lane < q.chunks ? q.heads[static_cast<int64_t>(row) * q.chunks + lane] : Surveyed{kNoTop, -__builtin_huge_valf(), 0.0f};
      r = h;
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) r.top = max(r.top, __shfl_xor(r.top, d, 64));
      r.max = wave_max(r.max);
      if (wave == 0) tops[lane] = h.top;
      __syncthreads();
      const uint64_t* const hs = q.hist + static_cast<int64_t>(row) * q.chunks * kBins;
      const uint32_t* const ns = q.counts + static_cast<int64_t>(row) * q.chunks * kBins;
      constexpr int AT_ONCE = 8;  // (unconditional loads: bins that a chunk lacks are fetched as its last)
      for (int c0 = 0; c0 < q.chunks; c0 += AT_ONCE) {
        uint64_t h8[AT_ONCE][2];
        uint32_t n8[AT_ONCE][2];
        bool some[AT_ONCE][2];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int c = min(c0 + i, q.chunks - 1), t = tops[c];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            some[i][e] = c0 + i < q.chunks && t > kNoTop && r.top - t <= 2 * tid + e;
            const int at = c * kBins + (some[i][e] ? 2 * tid + e - (r.top - t) : kRest);
            h8[i][e] = hs[at];
            n8[i][e] = counting ? ns[at] : 0;
          }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sum[e] += some[i][e] ? h8[i][e] : 0;
            num[e] += some[i][e] ? n8[i][e] : 0;
          }
      }
      if (tid == NT - 1) sum[1] = 0, num[1] = 0;  // kRest
    }
    if (whole_row && g.origin == r.max) break;
    // far from the origin bins are not told apart: once more, from the largest logit
    if (r.max == -__builtin_huge_valf() || (r.top < kFar / 2 && r.top > -kFar / 2)) break;
    g.origin = r.max;
    sum[0] = sum[1] = 0;
    num[0] = num[1] = 0;
    __syncthreads();
  }
  if (__builtin_expect(r.max == -__builtin_huge_valf(), 0)) {  // uniform: no token
    if (tid == 0) {
      if (PART == kPlanPart) plan->r = r, plan->to[0] = plan->to[1] = -__builtin_huge_valf(), q.listed[row] = 0;
      if (q.mode == kSample) q.token[row] = -1, q.logprob[row] = -__builtin_huge_valf();
      if (q.mode == kVerify) q.rowres[row] = Row{0.0, 0, r.max, 0.0f, 0, 0, -1};
      if (q.mode == kBeams) q.nbest[row] = 0;
    }
    return;
  }
  // ---- running sums, as whole numbers: a bin of nothing adds nothing ----
  // a unit of a bin's sum, in units of 2^-scale of the weight at the largest bin's middle
  auto unit_of = [&](int j) __attribute__((always_inline)) -> double {
    return exp2_of(static_cast<double>(-j) / kPerOctave) * __builtin_ldexp(1.0, q.scale - kWhole);
  };
  const double my_unit[2] = {by_value ? 0.0 : unit_of(2 * tid), by_value ? 0.0 : unit_of(2 * tid + 1)};
  const uint64_t my_w0 = static_cast<uint64_t>(static_cast<double>(sum[0]) * my_unit[0] + 0.5);
  const uint64_t my_w1 = static_cast<uint64_t>(static_cast<double>(sum[1]) * my_unit[1] + 0.5);
  double my_upto[2];
  uint32_t my_cn[2];
  {
    // (by value the sums are there)
    const int64_t at = static_cast<int64_t>(kBins) * row;
    uint64_t w = 0;
    uint32_t m = 0;
    if (PART != kFinishPart && !by_value) {
      w = wave_scan(my_w0 + my_w1);
      m = wave_scan(num[0] + num[1]);
      if (lane == 63) part[wave] = w, partn[wave] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (i < wave) w += part[i], m += partn[i];
      cw[2 * tid] = w - my_w1;
      cw[2 * tid + 1] = w;
      cn[2 * tid] = m - num[1];
      cn[2 * tid + 1] = m;
    }
    if (PART == kFinishPart) {
      cw[2 * tid] = q.sums[at + 2 * tid];
      cw[2 * tid + 1] = q.sums[at + 2 * tid + 1];
      cn[2 * tid] = q.sum_counts[at + 2 * tid];
      cn[2 * tid + 1] = q.sum_counts[at + 2 * tid + 1];
    }
    if (PART == kPlanPart) {
      q.sums[at + 2 * tid] = w - my_w1;
      q.sums[at + 2 * tid + 1] = w;
      q.sum_counts[at + 2 * tid] = m - num[1];
      q.sum_counts[at + 2 * tid + 1] = m;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // (each thread its own; by value it has one block)
      my_upto[e] = by_value ? static_cast<double>(cw[tid]) : static_cast<double>(cw[2 * tid + e]);
      my_cn[e] = by_value ? cn[tid] : cn[2 * tid + e];
    }
  }
  __syncthreads();
  const double total = static_cast<double>(cw[by_value ? 511 : kRest]);
  auto upto = [&](int j) -> double { return static_cast<double>(cw[j]); };
  auto before = [&](int j) -> double { return j > 0 ? static_cast<double>(cw[j - 1]) : 0.0; };
  int round = 0;
  // the numbers of bins of which a and c hold: the first of which they do not, if they hold for all before it
  auto find = [&](auto a, auto c, int& na, int& nc) __attribute__((always_inline)) {
    const int pa = __popcll(__ballot(a(0))) + __popcll(__ballot(a(1))), pc = __popcll(__ballot(c(0))) + __popcll(__ballot(c(1)));
    if (lane == 0) found[round][0][wave] = pa, found[round][1][wave] = pc;
    __syncthreads();
    na = nc = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) na += found[round][0][w], nc += found[round][1][w];
    na = __builtin_amdgcn_readfirstlane(na);
    nc = __builtin_amdgcn_readfirstlane(nc);
    round ^= 1;
  };
  auto in_bin = [&](float l) -> int {  // its bin from the largest down; kRest: too small to count
    const double n = __builtin_rint(g.place(l));
    return static_cast<int>(fmin(static_cast<double>(r.top) - n, static_cast<double>(kRest)));
  };
  auto reaches = [&](float l) -> bool { return (static_cast<double>(l) - static_cast<double>(r.max)) * z.s >= z.f; };
  // the logarithm of a sum of weights, of the largest token's
  auto log_of = [&](double w) -> double {
    return (log2_of(w * __builtin_ldexp(1.0, -q.scale)) + (static_cast<double>(r.top) - g.place(r.max)) / kPerOctave) * kLn2D;
  };
  auto second = [&](float l) -> uint64_t {
    const double t = g.place(l);
    return whole_exp2(t - __builtin_rint(t));
  };
  // a token's place in the order
  auto order_of = [&](uint32_t key, uint32_t idx) -> uint64_t { return static_cast<uint64_t>(key >> KS) << 20 | idx; };
  // the logits of bins b0 .. b1, a little more
  auto logits_of = [&](int b0, int b1, float& from, float& to) {
    const double top = static_cast<double>(r.top), o = static_cast<double>(g.origin);
    const float a = static_cast<float>(o + (top - b1 - 0.5) / z.s), c = static_cast<float>(o + (top - b0 + 0.5) / z.s);
    from = b1 >= kRest ? -kBig : fmaxf(a - fabsf(a) * 0x1p-20f - 1e-37f, -kBig);
    to = b0 == 0 ? __builtin_huge_valf() : fminf(c + fabsf(c) * 0x1p-20f + 1e-37f, kBig);
  };

  // ---- a drafted token that its row judges ----
  uint32_t drafted = kNone, drafted_key = 0;
  int drafted_bin = kBins;
  double drafted_w = 0.0;  // what it adds to the running sums, if it leaves the row once refused
  if (q.mode == kVerify && row + 1 < end) {
    const int64_t d = q.tokens[row + 1];
    if (d >= 0 && d < q.V) {
      const float l = x[static_cast<int>(d)];
      if (l > -__builtin_huge_valf()) {
        drafted = static_cast<uint32_t>(d);
        drafted_key = key_of(l);
        drafted_bin = in_bin(l);
      }
    }
  }
  const bool leaves = drafted_bin < kRest && !q.probs;
  if (PART == kFinishPart) {
    drafted_w = plan->drafted_w;
  } else if (leaves && !by_value) {  // uniform
    const int e = drafted_bin & 1;
    if (tid == drafted_bin >> 1)
      sel[0] = (e ? my_w1 : my_w0) - static_cast<uint64_t>(static_cast<double>(sum[e] - second(logit_of_key(drafted_key))) * my_unit[e] + 0.5);
    __syncthreads();
    drafted_w = static_cast<double>(sel[0]);
  }
  const double u = z.first || q.mode == kBeams ? 0.0 : unit(q.mode == kVerify ? q.draw[b] : q.u[row]);

  // ---- the bins in which something is to be found, before the cuts are known ----
  // windows: top-k's cut, top-p's, min-p's, the token
  int w0[4] = {1, 1, 1, 1}, w1[4] = {0, 0, 0, 0};
  if (PART != kFinishPart && !by_value) {
    int kb, last;
    find([&](int e) { return my_cn[e] < static_cast<uint32_t>(z.k); }, [&](int e) { return my_upto[e] < total; }, kb, last);
    double least = total, most = total;
    if (counting && kb < kRest) {
      w0[0] = w1[0] = kb;
      least = before(kb);
      most = upto(kb);
    }
    if (q.mode == kBeams) {
      // (with fewer tokens than wanted among the bins that count, all of the row's)
      w0[0] = 0;
      w1[0] = kb < kRest ? kb : kRest;
    } else {
      if (z.p < 1.0) {
        const double a = z.p * least * kBelow, c = z.p * most * kAbove;
        find([&](int e) { return my_upto[e] < a; }, [&](int e) { return my_upto[e] < c; }, w0[1], w1[1]);
        w1[1] = min(w1[1], last);
        w0[1] = min(w0[1], w1[1]);
        // a token of bin j weighs less than 2^((1 - j) / 20)
        const double one = exp2_of(static_cast<double>(1 - w0[1]) / kPerOctave) * __builtin_ldexp(1.0, q.scale);
        least = a;
        most = fmin(upto(w1[1]), c + one);
      }
      if (z.f > -__builtin_huge_val()) {
        // tokens whose place is not below this reach min-p
        const double y = g.place(r.max) + z.f, eps = 1e-6 + fabs(y) * 1e-13, top = static_cast<double>(r.top);
        w0[2] = static_cast<int>(fmin(fmax(top - __builtin_rint(y + eps), 0.0), static_cast<double>(kRest)));
        w1[2] = static_cast<int>(fmin(fmax(top - __builtin_rint(y - eps), 0.0), static_cast<double>(kRest - 1)));
        // the shortest prefix counts: of two cuts whose bins do not meet, the one before the other
        const int o0 = z.p < 1.0 ? w0[1] : w0[0], o1 = z.p < 1.0 ? w1[1] : w1[0];
        if (w0[2] >= kRest || (o1 >= o0 && w0[2] > o1)) {
          w0[2] = 1, w1[2] = 0;
        } else {
          if (o1 >= o0 && w1[2] < o0) w0[0] = w0[1] = 1, w1[0] = w1[1] = 0;
          least = fmin(least, before(w0[2]));
          most = fmin(most, upto(w1[2]));
        }
      }
      // with its bin before the cuts the drafted token is kept, behind them not, among them one or the other
      double gone = 0.0;
      bool sure = true;
      if (leaves) {
        int open = kBins, cut = kRest;
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (w1[i] >= w0[i]) open = min(open, w0[i]), cut = min(cut, w1[i]);
        gone = drafted_bin <= cut ? drafted_w : 0.0;
        sure = drafted_bin < open || drafted_bin > cut;
      }
      const double a = u * fmax(least - gone, 0.0) * kBelow, c = u * (sure ? most - gone : most) * kAbove;
      auto without = [&](int e) { return 2 * tid + e >= drafted_bin ? my_upto[e] - gone : my_upto[e]; };
      find([&](int e) { return (sure ? without(e) : my_upto[e]) <= a; }, [&](int e) { return without(e) <= c; }, w0[3], w1[3]);
      w1[3] = min(w1[3], kRest - 1);
      w0[3] = min(w0[3], w1[3]);
    }
  }

  // ---- the cuts and the token ----
  // the bins from the first cut's to the last's
  const int cuts0 = min(min(w1[0] < w0[0] ? kBins : w0[0], w1[1] < w0[1] ? kBins : w0[1]), w1[2] < w0[2] ? kBins : w0[2]);
  const int cuts1 = max(max(w1[0], w1[1]), w1[2]);
  // whether the tokens fit the list: a second factor is 1, nearly
  bool in_list = false, relist = by_value;
  if (PART == kFinishPart) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w0[i] = plan->w0[i], w1[i] = plan->w1[i];
  } else if (!by_value) {
    uint64_t many = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * tid + e;
      many += (j >= cuts0 && j <= cuts1) || (j >= w0[3] && j <= w1[3]) ? sum[e] >> kWhole : 0;
    }
    many = wave_sum(many);
    if (lane == 0) part[wave] = many;
    __syncthreads();
    many = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) many += part[w];
    relist = many > static_cast<uint64_t>(kCap - kCap / 16);
  }
  // two ranges of logits: the cuts' and the token's bins
  float from[2], to[2];
  if (!by_value) {
    logits_of(cuts0, cuts1, from[0], to[0]);
    logits_of(w0[3], w1[3], from[1], to[1]);
  }
  if (cuts1 < cuts0) from[0] = __builtin_huge_valf(), to[0] = -__builtin_huge_valf();
  if (w1[3] < w0[3]) from[1] = __builtin_huge_valf(), to[1] = -__builtin_huge_valf();
  if (PART == kPlanPart) {
    if (tid == 0) {
      Plan p{r, {}, {}, {}, {}, drafted_w};
      p.r.origin = g.origin;
#pragma unroll
      for (int i = 0; i < 4; ++i) p.w0[i] = w0[i], p.w1[i] = w1[i];
#pragma unroll
      for (int i = 0; i < 2; ++i) p.from[i] = from[i], p.to[i] = relist ? -__builtin_huge_valf() : to[i];
      *plan = p;
      q.listed[row] = relist ? static_cast<uint32_t>(kCap) + 1u : 0;
    }
    return;
  }
  // the windows that the listed tokens are from (by value: of one alone)
  const int windows = by_value ? 1 : (w1[0] >= w0[0]) + (w1[1] >= w0[1]) + (w1[2] >= w0[2]) + (w1[3] >= w0[3]);
  int n = 0;
  uint64_t cut = ~0ull;  // the last token that top-k and top-p keep
  double kept = total;
  uint32_t skip = kNone, token = kNone;
  bool accepted = false;
  float drawn = 0.0f;  // the token's logit
  // by value: how many of the equal ones at the cut are kept, and their logit
  uint64_t cut_need = ~0ull;
  bool beyond = false;  // a drafted token among them that is not
  float cut_value = 0.0f;
  const uint32_t my_total_n = by_value ? cn[511] : 0;
  auto order_index = [&](uint32_t key) -> uint32_t { return key >> 16; };  // of a value, from the key of its logit
#pragma unroll 1
  for (int step = -1; step < 5; ++step) {
    int b0 = w0[3], b1 = w1[3];
    if (step == 0) b0 = w0[0], b1 = w1[0];
    if (step == 1) b0 = w0[1], b1 = w1[1];
    if (step == 2) b0 = w0[2], b1 = w1[2];
    double target = 0.0, start = 0.0;  // what is looked for, what lies before the bin
    uint64_t need = 1;
    if (by_value) {
      if (step < 0 || (step == 0 && !counting) || (step == 1 && !(z.p < 1.0))) continue;  // uniform
      b0 = 0;
      b1 = kBins;
    }
    if (step >= 0) {
      if (b1 < b0 || (step == 4 && !by_value)) continue;  // uniform
      if (step == 1) target = by_value ? fmax(z.p * kept, 0.5) : z.p * kept;
      if (step == 3) {
        double left = kept;
        if (drafted != kNone) {
          const float l = logit_of_key(drafted_key);
          if (order_of(drafted_key, drafted) <= cut && !beyond && reaches(l)) {
            const double w = exp2_of((g.place(l) - static_cast<double>(r.top)) / kPerOctave) * __builtin_ldexp(1.0, q.scale);
            const double sure = q.probs ? static_cast<double>(q.probs[row * q.probs_stride + drafted]) : 1.0;
            accepted = static_cast<double>(q.u[row]) * sure * kept < w;
            // (what leaves less than 2^12 units is not refused: u is at most 1 - 2^-24)
            if (leaves && kept - w > 4096.0) {
              skip = drafted;
              left = kept - w;
            }
          }
        }
        target = u * left;
      }
      if (by_value) {
        if (step == 2) {
          if (z.f > -__builtin_huge_val()) kept = fmin(kept, static_cast<double>(reached));
          // a drafted token of the cut's value: kept if fewer equal ones than the cut keeps are before it
          if (__builtin_expect(drafted == kNone || order_of(drafted_key, 0xfffffu) != cut, 1)) continue;
          const float l = logit_of_key(drafted_key);
          uint32_t c0, c1;
          tallied(order_index(drafted_key) & ~1u, c0, c1);
          if ((order_index(drafted_key) & 1u ? c1 : c0) == 1u) continue;  // (it alone)
          uint32_t m = 0;
          const int upto = static_cast<int>(drafted) - x.head;  // behind the first edge, pieces up to the drafted token's
          const int last = upto < 0 ? 0 : min(upto / P::N + 1, x.whole), pieces = last + 2;
          auto counted = [&](const uint4& v, int first) {
#pragma unroll
            for (int i = 0; i < P::N; ++i) m += logit_of<DT>(P::at(v, i)) == l && first + i < static_cast<int>(drafted);
          };
          for (int p0 = tid; p0 < pieces; p0 += 8 * NT) {
            uint4 v[8];
#pragma unroll
            for (int a = 0; a < 8; ++a) {
              const int p = p0 + a * NT;
              v[a] = x.load(p < last ? p : x.whole + (p - last), x.count());
            }
#pragma unroll
            for (int a = 0; a < 8; ++a) {
              const int p = p0 + a * NT;
              if (p < pieces) counted(v[a], x.first(p < last ? p : x.whole + (p - last)));
            }
          }
          m = wave_sum(m);
          __syncthreads();
          if (lane == 0) partn[wave] = m;
          __syncthreads();
          m = 0;
#pragma unroll
          for (int i = 0; i < NW; ++i) m += partn[i];
          beyond = m >= cut_need;
          continue;
        } else if (step == 4) {
          // which of the equal ones at the cut are kept: wanted by the launches behind
          if (!q.probs || cut == ~0ull) continue;
          need = cut_need;
          from[0] = to[0] = cut_value;
          skip = kNone;
        } else if (step == 0 && my_total_n < static_cast<uint32_t>(z.k)) {
          if (q.mode != kBeams) continue;
          need = z.k;  // all of them
          from[0] = -P::BIG;
          to[0] = P::BIG;
        } else {
          // the block: the first whose running sum reaches the target, or for the token exceeds it
          double gone = 0.0;  // what the drafted token's value loses without it
          if (skip != kNone) {
            uint32_t c0, c1;
            tallied(order_index(drafted_key) & ~1u, c0, c1);
            const uint32_t c = order_index(drafted_key) & 1u ? c1 : c0;
            const double w = weight(logit_of_key(drafted_key));
            gone = static_cast<double>(static_cast<uint64_t>(c * w + 0.5) - static_cast<uint64_t>((c - 1) * w + 0.5));
          }
          const int gone_block = skip != kNone ? static_cast<int>(order_index(drafted_key) >> 7) : kBins;
          auto w = [&](int) { return tid >= gone_block ? my_upto[0] - gone : my_upto[0]; };
          int at, end_at;
          find([&](int e) { return e == 0 && (step == 0 ? my_cn[0] < static_cast<uint32_t>(z.k) : step == 3 ? w(0) <= target : w(0) < target); },
               [&](int e) { return e == 0 && (step == 0 ? my_cn[0] < my_total_n : w(0) < total - gone); }, at, end_at);
          at = min(at, end_at);
          // the value in it
          const uint32_t o = 128u * at + 2u * lane;
          uint32_t c0, c1;
          tallied(o, c0, c1);
          if (skip != kNone) c0 -= o == order_index(drafted_key), c1 -= o + 1u == order_index(drafted_key);
          const float l0 = value_of(o), l1 = value_of(o + 1u);
          const double one0 = weight(l0), one1 = weight(l1);
          const uint64_t a = static_cast<uint64_t>(c0 * one0 + 0.5), c = static_cast<uint64_t>(c1 * one1 + 0.5);
          const uint64_t sw = wave_scan(a + c);
          const uint32_t sn = wave_scan(c0 + c1);
          const double w0 = before(at) - (at > gone_block ? gone : 0.0), u1 = w0 + static_cast<double>(sw), u0 = w0 + static_cast<double>(sw - c);
          const uint32_t n0 = at > 0 ? cn[at - 1] : 0, k1 = n0 + sn, k0 = k1 - c1;
          const bool hit0 = c0 && (step == 0 ? k0 >= static_cast<uint32_t>(z.k) : step == 3 ? u0 > target : u0 >= target);
          const bool hit1 = c1 && (step == 0 ? k1 >= static_cast<uint32_t>(z.k) : step == 3 ? u1 > target : u1 >= target);
          const uint64_t hits = __ballot(hit0 || hit1), any = __ballot((c0 | c1) != 0);
          const int who = hits ? __builtin_ctzll(hits) : any ? 63 - __builtin_clzll(any) : 0;
          const bool second_one = !(hits ? hit0 : c1 == 0);
          const uint32_t odd = lane_of(static_cast<uint32_t>(second_one), who);
          const uint32_t many = lane_of(odd ? c1 : c0, who), k_before = lane_of(odd ? k0 : k0 - c0, who);
          const double w_before = w0 + static_cast<double>(lane_of(odd ? sw - c : sw - c - a, who));
          const float l = value_of(128u * at + 2u * who + odd);
          const double one = __longlong_as_double(static_cast<long long>(lane_of(static_cast<uint64_t>(__double_as_longlong(odd ? one1 : one0)), who)));
          // the token's place among the equal ones
          const double y = step == 0 ? static_cast<double>(z.k) - static_cast<double>(k_before) : fmax((target - w_before) / one, 0.0);
          need = static_cast<uint64_t>(fmin(step == 3 ? __builtin_floor(y) + 1.0 : fmax(__builtin_ceil(y), 1.0), static_cast<double>(many)));
          from[0] = to[0] = l;
          if (step < 2) {
            const uint64_t at_cut = order_of(key_of(l), 0xfffffu);
            kept = fmin(kept, w_before + static_cast<double>(need) * one);
            if (at_cut < cut || (at_cut == cut && need < cut_need)) cut = at_cut, cut_need = need, cut_value = l;
            if (q.mode != kBeams) continue;
            need = z.k;
            to[0] = P::BIG;
          }
        }
        if (to[0] == P::BIG) to[0] = __builtin_huge_valf();
      } else if (step == 1 || step == 3) {
        // the bin: the first whose running sum reaches the target, or for the token exceeds it
        const double gone = skip != kNone ? drafted_w : 0.0;
        auto w = [&](int e) { return 2 * tid + e >= drafted_bin ? my_upto[e] - gone : my_upto[e]; };
        int at, end_at;
        find([&](int e) { return step == 3 ? w(e) <= target : w(e) < target; }, [&](int e) { return w(e) < total - gone; }, at, end_at);
        at = min(at, end_at);
        b0 = b1 = min(max(at, b0), b1);
        start = before(b0) - (b0 > drafted_bin ? gone : 0.0);
      }
    }
    // ---- the tokens of the bins: all windows' at once, or, where those are too many, the bin's ----
    if (step < 0 && relist) continue;
    if (PART == kFinishPart && step < 0) {
      const uint32_t many = q.listed[row];
      in_list = many <= kCap;
      relist = !in_list;
      n = in_list ? static_cast<int>(many) : 0;
      const uint2* const theirs = q.list + static_cast<int64_t>(row) * kCap;
#pragma unroll 8
      for (int i = tid; i < n; i += NT) list[i] = theirs[i];  // (each thread comes back to its own)
      continue;
    }
    if (step < 0 || relist) {
      __syncthreads();
      if (tid == 0) number[0] = 0;
      __syncthreads();
      if (step >= 0) {
        if (!by_value) logits_of(b0, b1, from[0], to[0]);
        from[1] = __builtin_huge_valf();
        to[1] = -__builtin_huge_valf();
      }
      // bf16, one value: its pattern in both halves of a word (of 0 without the sign)
      const bool one_value = by_value && from[0] == to[0];
      const uint32_t sign = from[0] == 0.0f ? 0x7fff7fffu : 0xffffffffu, half = __float_as_uint(from[0]) >> 16, same = (half << 16 | half) & sign;
      const uint32_t same_key = key_of(from[0] + 0.0f);
      const int pieces = x.count();
      constexpr int AHEAD = 8, MASKS = AHEAD * P::N / 32;
      uint4 next[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) next[a] = x.load(a * NT + tid, pieces);
      for (int p0 = 0; p0 < pieces; p0 += AHEAD * NT) {
        uint32_t mine[MASKS];
        uint4 now[AHEAD];
#pragma unroll
        for (int k = 0; k < MASKS; ++k) mine[k] = 0;
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          now[a] = next[a];
          const int piece = p0 + (AHEAD + a) * NT + tid;
          if (p0 + AHEAD * NT < pieces) next[a] = x.load(piece, pieces);
        }
        if (DT == MZK_BF16 && one_value) {
          // halves of words equal to one pattern: of the exclusive or, those that are 0
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            const uint32_t v[4] = {now[a].x, now[a].y, now[a].z, now[a].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t d = (v[i] & sign) ^ same, other = ((d & 0x7fff7fffu) + 0x7fff7fffu) | d;  // bits 15, 31: not equal
              const uint32_t equal = ~other & 0x80008000u;
              mine[a * P::N / 32] |= (equal >> 15 & 1u) << (a * P::N % 32 + 2 * i) | (equal >> 31) << (a * P::N % 32 + 2 * i + 1);
            }
          }
        } else {
#pragma unroll
          for (int a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int i = 0; i < P::N; ++i) {
              const float l = P::at(now[a], i);  // (a NaN is in no range)
              const bool in = (l >= from[0] && l <= to[0]) || (l >= from[1] && l <= to[1]);
              mine[a * P::N / 32] |= static_cast<uint32_t>(in) << (a * P::N % 32 + i);
            }
        }
        uint32_t many = 0;
#pragma unroll
        for (int k = 0; k < MASKS; ++k) many += __popc(mine[k]);
        if (__ballot(many != 0) == 0) continue;
        const uint32_t s = wave_scan(many);
        uint32_t at = 0;
        if (lane == 63) at = atomicAdd(&number[0], s);
        at = lane_of(at, 63) + s - many;
#pragma unroll
        for (int k = 0; k < MASKS; ++k)
          while (mine[k]) {
            const int i = 32 * k + __builtin_ctz(mine[k]);
            mine[k] &= mine[k] - 1;
            if (at < kCap) list[at] = uint2{same_key, static_cast<uint32_t>(x.first(p0 + i / P::N * NT + tid) + i % P::N)};
            ++at;
          }
      }
      __syncthreads();
      in_list = number[0] <= kCap;
      n = in_list ? static_cast<int>(number[0]) : 0;
#pragma unroll 4
      for (int i = tid; i < n && !one_value; i += NT) {  // (each thread comes back to its own)
        const uint32_t idx = list[i].y;
        const float l = x[static_cast<int>(idx)];
        list[i] = uint2{key_of(l), idx | static_cast<uint32_t>(in_bin(l)) << 20};
      }
      if (step < 0) {
        relist = !in_list;
        continue;
      }
    }
    // f(place in the order, logit) for the tokens of bins b0 .. b1 between lo and hi, listed or of the whole row.  (What
    // few rows need is marked as unlikely, and so laid behind the steps that all take, whose code comes to the cache
    // first: 160 drafted rows 49.2 us for 50.8, 64 rows 44.3 for 45.5.)
    auto each = [&](uint64_t lo, uint64_t hi, auto f) __attribute__((always_inline)) {
      if (__builtin_expect(in_list, 1)) {
        for (int i = tid; i < n; i += NT) {
          const uint2 e = list[i];
          const int j = static_cast<int>(e.y >> 20);
          const uint32_t idx = e.y & 0xfffffu;
          const uint64_t me = order_of(e.x, idx);
          if (j >= b0 && j <= b1 && me >= lo && me <= hi && idx != skip) f(me, logit_of_key(e.x));
        }
      } else {
        x.template walk<NT>(tid, [&](int i, float l) __attribute__((always_inline)) {
          const uint64_t me = order_of(key_of(l), static_cast<uint32_t>(i));
          if (me < lo || me > hi || static_cast<uint32_t>(i) == skip) return;
          const int j = in_bin(l);
          if (j >= b0 && j <= b1) f(me, l);
        });
      }
    };
    const double u_bin = by_value ? 0.0 : unit_of(b0);
    if (step == 2 && !by_value) {
      // ---- the weights of those that reach min-p ----
      __syncthreads();
      if (tid == 0) sel[2] = 0;
      __syncthreads();
      uint64_t mine = 0;
      each(0, ~0ull, [&](uint64_t, float l) {
        if (!reaches(l)) return;
        const uint64_t w = second(l);
        const int j = in_bin(l);
        mine += j == b0 ? w : static_cast<uint64_t>(static_cast<double>(w) * exp2_of(static_cast<double>(b0 - j) / kPerOctave));
      });
      mine = wave_sum(mine);
      if (lane == 0 && mine) atomicAdd(reinterpret_cast<unsigned long long*>(&sel[2]), static_cast<unsigned long long>(mine));
      __syncthreads();
      kept = fmin(kept, before(b0) + static_cast<double>(sel[2]) * u_bin);
      continue;
    }
    // ---- the token at which the running sum, of ones or of weights, reaches `need` ----
    const bool by_count = step == 0 || by_value;
    uint64_t lo, hi;
    {
      float least = from[0], most = to[0];
      if (!by_value) logits_of(b0, b1, least, most);
      lo = order_of(key_of(fminf(most, kBig) + 0.0f), 0);
      hi = order_of(key_of(least + 0.0f), 0xfffffu);
      if (by_value) {
        // (known)
      } else if (by_count) {
        need = static_cast<uint64_t>(z.k) - (b0 > 0 ? cn[b0 - 1] : 0u);
      } else {
        const double y = fmax((target - start) / u_bin, 0.0);
        // (a border that is hit exactly, as with equal weights, is: y is off by some 2^-51 of itself, and a float32's share
        // of at most 2^20 equal ones that is on no border lies 2^-45 and more from it)
        need = step == 3 ? static_cast<uint64_t>(y * (1.0 + 0x1p-48)) + 1 : static_cast<uint64_t>(__builtin_ceil(y * (1.0 - 0x1p-48)));
      }
      if (need < 1) need = 1;
    }
    if (__builtin_expect(!in_list && !by_value, 0)) {  // uniform
      // the row's own keys in these bins, so that fewer steps of 10 bits are left (2 rows of 131072 equal logits, fp32:
      // with top-p 534 us, 1211 without this)
      uint32_t a = ~0u, c = 0;
      x.template walk<NT>(tid, [&](int, float l) __attribute__((always_inline)) {
        const uint32_t key = key_of(l);
        const uint64_t me = order_of(key, 0);
        if (me >= lo && me <= hi) a = min(a, key), c = max(c, key);
      });
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) a = min(a, static_cast<uint32_t>(__shfl_xor(a, d, 64))), c = max(c, static_cast<uint32_t>(__shfl_xor(c, d, 64)));
      __syncthreads();
      if (lane == 0) part[wave] = static_cast<uint64_t>(a) << 32 | c;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i) a = min(a, static_cast<uint32_t>(part[i] >> 32)), c = max(c, static_cast<uint32_t>(part[i]));
      if (a <= c) {
        lo = max(lo, order_of(a, 0));
        hi = min(hi, order_of(c, 0xfffffu));
      }
    }
    uint64_t passed = 0;  // weights and numbers before lo
    uint32_t passed_n = 0;
    // Of a short list the tokens are gathered at once, without a digit: mostly few of them are in these bins.  (fp32, whole
    // calls, top-k, top-p and min-p: 1 row of 131072 32.4 us for 34.3, 64 of 4096 20.4 for 22.8; the others +-1.)
    for (bool direct = in_list && n <= 64 * windows;; direct = false) {
      while (!direct) {
        const int bits = 64 - __builtin_clzll(hi - lo | 1), sh = bits > 10 ? bits - 10 : 0;
        __syncthreads();
        hist[tid] = hist[NT + tid] = 0;
        counts[tid] = counts[NT + tid] = 0;
        if (tid == 0) sel[0] = 0, sel[1] = passed, sel[2] = passed_n, number[1] = 0;
        __syncthreads();
        each(lo, hi, [&](uint64_t me, float l) {
          const uint32_t digit = static_cast<uint32_t>((me - lo) >> sh), bits = __float_as_uint(l);
          const uint64_t w = second(l);
          bool left = true;
          if (__builtin_expect(!in_list, 0)) {
            // the lanes with the same logit and digit, of which a row of few values has many, by one of them
  #pragma unroll 1
            for (uint64_t todo = __ballot(true); todo;) {
              const int leader = __builtin_ctzll(todo);
              const bool like = left && digit == lane_of(digit, leader) && bits == lane_of(bits, leader);
              const uint64_t same = __ballot(like);
              const uint32_t many = static_cast<uint32_t>(__popcll(same));
              if (many < 8) break;  // uniform
              if (lane == leader) {
                atomicAdd(&hist[digit], static_cast<unsigned long long>(many * w));
                atomicAdd(&counts[digit], many);
              }
              left = left && !like;
              todo &= ~same;
            }
          }
          if (left) {
            atomicAdd(&hist[digit], static_cast<unsigned long long>(w));
            atomicAdd(&counts[digit], 1u);
          }
        });
        __syncthreads();
        // digits 2 tid, 2 tid + 1
        const uint64_t v0 = hist[2 * tid], v1 = hist[2 * tid + 1];
        const uint32_t n0 = counts[2 * tid], n1 = counts[2 * tid + 1];
        const uint64_t s = wave_scan(v0 + v1);
        const uint32_t sn = wave_scan(n0 + n1);
        if (lane == 63) part[wave] = s, partn[wave] = sn;
        __syncthreads();
        uint64_t w = passed + s - v0 - v1, all = passed;
        uint32_t k = passed_n + sn - n0 - n1, all_n = passed_n;
  #pragma unroll
        for (int i = 0; i < NW; ++i) {
          if (i < wave) w += part[i], k += partn[i];
          all += part[i];
          all_n += partn[i];
        }
        const uint64_t most = by_count ? all_n : all;
        if (need > most) need = most;
        const uint64_t a = by_count ? k : w, c = a + (by_count ? n0 : v0), e = c + (by_count ? n1 : v1);
        if (a < need && need <= c) sel[0] = static_cast<uint64_t>(2 * tid) | static_cast<uint64_t>(n0) << 32, sel[1] = w, sel[2] = k;
        if (c < need && need <= e) sel[0] = static_cast<uint64_t>(2 * tid + 1) | static_cast<uint64_t>(n1) << 32, sel[1] = w + v0, sel[2] = k + n0;
        __syncthreads();
        const uint64_t got = sel[0];
        passed = sel[1];
        passed_n = static_cast<uint32_t>(sel[2]);
        lo = lo + ((got & 0xffffffffu) << sh);
        const uint64_t top = lo + ((1ull << sh) - 1ull);
        hi = top < hi ? top : hi;
        if ((got >> 32) <= 64 || sh == 0) break;  // uniform
      }
      if (direct) {  // uniform
        __syncthreads();
        if (tid == 0) number[1] = 0;
        __syncthreads();
      }
      // ---- at most 64: gathered, and every wave sums them in their order ----
      each(lo, hi, [&](uint64_t me, float l) {
        const uint32_t to = atomicAdd(&number[1], 1u);
        if (to < 64) {
          last_ones[to][0] = me;
          last_ones[to][1] = second(l);
        }
      });
      __syncthreads();
      if (!direct || number[1] <= 64) break;  // uniform
    }
    const int m = static_cast<int>(number[1]);
    const uint64_t me = lane < m ? last_ones[lane][0] : ~0ull, mine = lane < m ? last_ones[lane][1] : 0;
    uint64_t w = passed;
    uint32_t k = passed_n;
    uint64_t all = passed;
    for (int i = 0; i < m; ++i) {
      all += last_ones[i][1];
      if (last_ones[i][0] <= me) w += last_ones[i][1], ++k;
    }
    need = min(need, by_count ? passed_n + static_cast<uint64_t>(m) : all);
    const uint64_t measure = by_count ? k : w, one = by_count ? 1 : mine;
    const uint64_t hit = __ballot(lane < m && measure >= need && measure - one < need);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      const uint64_t found_at = __shfl(me, at, 64);
      if (step == 3) {
        token = static_cast<uint32_t>(found_at & 0xfffffu);
        drawn = x[static_cast<int>(token)];
      } else {
        cut = found_at < cut ? found_at : cut;
        if (!by_value) kept = fmin(kept, before(b0) + static_cast<double>(__shfl(w, at, 64)) * u_bin);
      }
    }
    if (q.mode == kBeams) break;  // uniform
  }
  // Beams keep the tokens up to the cut.  And top-k may end among tokens too light for the sums, without a cut: a drafted one of those is
  // accepted if fewer than k are before it.  (With a walk of its own among the steps above, 64 bf16 rows of 131072 that do not need it
  // took 0.8 us more, with this one 0.5.)
  if (q.mode == kBeams) {
    __syncthreads();
    if (tid == 0) number[1] = 0;
    __syncthreads();
    auto take = [&](uint32_t k, uint32_t i) {
      const uint32_t to = atomicAdd(&number[1], 1u);
      if (to < static_cast<uint32_t>(q.keep)) q.best[static_cast<int64_t>(row) * q.keep + to] = uint2{k, i};
    };
    if (in_list) {
      for (int i = tid; i < n; i += NT) {
        const uint32_t idx = list[i].y & 0xfffffu;
        if (order_of(list[i].x, idx) <= cut) take(list[i].x, idx);
      }
    } else {
      x.template walk<NT>(tid, [&](int i, float l) __attribute__((always_inline)) {
        const uint32_t k = key_of(l);
        if (order_of(k, static_cast<uint32_t>(i)) <= cut) take(k, static_cast<uint32_t>(i));
      });
    }
    __syncthreads();
    if (tid == 0) {
      q.nbest[row] = min(number[1], static_cast<uint32_t>(q.keep));
      q.rowres[row] = Row{log_of(total), 0, r.max, g.origin, r.top, 0, 0};
    }
    return;
  }
  // Top-k may end among tokens too light for the sums, without a cut: a drafted one of those is accepted if fewer than k are before it.  (Of
  // little code, here: with a walk in four pieces 64 bf16 rows of 131072 that do not need it take 0.5 us more, among the steps above 0.8.)
  if (__builtin_expect(accepted && counting && cut == ~0ull && drafted_bin == kRest, 0)) {  // uniform
    const uint64_t its = order_of(drafted_key, drafted);
    uint32_t m = 0;
#pragma unroll 4
    for (int i = tid; i < x.V; i += NT) {
      const float l = x[i];
      m += order_of(key_of(l), static_cast<uint32_t>(i)) < its;
    }
    __syncthreads();
    if (tid == 0) number[1] = 0;
    __syncthreads();
    atomicAdd(&number[1], m);
    __syncthreads();
    accepted = number[1] < static_cast<uint32_t>(z.k);
  }
  if (tid != 0) return;
  if (q.mode == kSample) {
    q.token[row] = token == kNone ? -1 : static_cast<int64_t>(token);
    // (a difference below what the sums tell apart is none)
    const double lp = (static_cast<double>(drawn) - static_cast<double>(r.max)) * z.s * (kLn2D / kPerOctave) - log_of(kept);
    q.logprob[row] = lp > -0x1p-40 ? 0.0f : static_cast<float>(lp);
  } else {
    q.rowres[row] = Row{kept, cut, r.max, g.origin, r.top, accepted ? 1 : 0, static_cast<int32_t>(token)};
  }
}

// ---- verify: the sequences ------------------------------------------------------------------------

// The rows of sequence b: the first whose drafted token is refused, or the last (by a whole wave; -1: no rows).
__device__ __forceinline__ int judged(const SamplingParams& q, int b, int lane, int& first, int& end, int& token) {
  auto clamp = [&](int64_t v, int lo) -> int { return v < lo ? lo : v > q.rows ? q.rows : static_cast<int>(v); };
  first = clamp(q.cu[b], 0);
  end = clamp(q.cu[b + 1], first);
  token = -1;
  for (int i0 = first; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    const Row* const r = q.rowres + (i < end ? i : end - 1);
    const int accepted = r->accepted, its = r->token;
    const uint64_t stop = __ballot(i < end && (i + 1 == end || !accepted));
    if (stop) {
      const int at = __builtin_ctzll(stop);
      token = __builtin_amdgcn_readlane(its, at);
      return i0 + at;
    }
  }
  return -1;
}

// The sequences, a wave each: without the draft's probabilities, and where no token is refused, the token of that row is
// the next.
__global__ void __launch_bounds__(256) verify_kernel(const SamplingParams q) {
  const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= q.B) return;
  int first, end, token;
  const int i = judged(q, b, lane, first, end, token);
  if (lane != 0) return;
  q.accepted[b] = i < 0 ? 0 : i - first;
  q.token[b] = token;
}

// What the target has above the draft at token i, 2^52 a probability of 1.  (Of tokens too light for the sums, a unit or two at most; nothing where
// top-k may end among them, whose place nobody knows.)
template <int DT>
__device__ __forceinline__ uint64_t above(const SamplingParams& q, const Settings& z, const Row& r, int row, float l, int i) {
  constexpr int KS = DT == MZK_F32 ? 0 : DT == MZK_BF16 ? 16 : 13;
  const uint64_t me = static_cast<uint64_t>(key_of(l) >> KS) << 20 | static_cast<uint32_t>(i);
  if (!(l > -__builtin_huge_valf()) || me > r.cut || (static_cast<double>(l) - static_cast<double>(r.max)) * z.s < z.f) return 0;
  const double place = Grid{r.origin, z.s}.place(l), t = place - static_cast<double>(r.top);
  if (r.cut == ~0ull && z.k > 0 && static_cast<double>(r.top) - __builtin_rint(place) >= static_cast<double>(kRest)) return 0;
  const double p = exp2_of(t / kPerOctave) * __builtin_ldexp(1.0, q.scale) / r.kept;
  const double d = p - static_cast<double>(fmaxf(q.probs[row * q.probs_stride + i], 0.0f));
  return d > 0.0 ? static_cast<uint64_t>(d * 0x1p52) : 0;
}

constexpr int kRestElements = 1024;  // of a chunk: 4 of a thread

// With the draft's probabilities: the sequences, and of refused tokens' rows the sums of what the target has above the draft.
template <int DT>
__global__ void __launch_bounds__(256) rest_kernel(const SamplingParams q) {
  __shared__ unsigned long long sums[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int b = blockIdx.x / q.rest_chunks, chunk = blockIdx.x - b * q.rest_chunks;
  int first, end, token;
  const int row = judged(q, b, lane, first, end, token);
  const bool refused = row >= 0 && row + 1 < end;  // uniform
  if (chunk == 0 && tid == 0) {
    q.accepted[b] = row < 0 ? 0 : row - first;
    q.token[b] = token;
    q.refused[b] = refused ? row : -1;
  }
  if (!refused) return;
  const Pieces<DT> x(q.logits + row * q.stride, q.V, nullptr);
  const Settings z = settings(q, row);
  const Row r = q.rowres[row];
  uint64_t s = 0;
#pragma unroll
  for (int k = 0; k < kRestElements / 256; ++k) {
    const int i = chunk * kRestElements + 256 * k + tid;
    if (i < q.V) s += above<DT>(q, z, r, row, x[i], i);
  }
  s = wave_sum(s);
  if (lane == 0) sums[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) q.rest[static_cast<int64_t>(b) * q.rest_chunks + chunk] = sums[0] + sums[1] + sums[2] + sums[3];
}

// The token of a refused row from what the target has above the draft, by rising index (where that is
// nothing it stays the one from the target itself).
template <int DT>
__global__ void __launch_bounds__(256) redraw_kernel(const SamplingParams q) {
  constexpr int PER = 4;  // chunks of a thread, at most 2^20 / kRestElements in all, and elements
  static_assert(kMaxVocab / kRestElements <= 256 * PER && kRestElements == 256 * PER, "redraw");
  __shared__ unsigned long long sums[4], part[4], at_before;
  __shared__ int at_chunk;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const int row = q.refused[b];
  if (row < 0) return;
  uint64_t mine[PER], upto = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = PER * tid + k;
    mine[k] = c < q.rest_chunks ? q.rest[static_cast<int64_t>(b) * q.rest_chunks + c] : 0;
    upto += mine[k];
  }
  const uint64_t of_me = upto;
  upto = wave_scan(upto);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  const uint64_t total = sums[0] + sums[1] + sums[2] + sums[3];
  if (total == 0) return;  // uniform
  uint64_t need = static_cast<uint64_t>(unit(q.draw[b]) * static_cast<double>(total)) + 1;
  if (need > total) need = total;
  uint64_t at = upto - of_me;
  for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (at < need && need <= at + mine[k]) at_chunk = PER * tid + k, at_before = at;
    at += mine[k];
  }
  __syncthreads();
  const Pieces<DT> x(q.logits + row * q.stride, q.V, nullptr);
  const Settings z = settings(q, row);
  const Row r = q.rowres[row];
  const int i0 = at_chunk * kRestElements + PER * tid;
  uint64_t s = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    mine[k] = i0 + k < q.V ? above<DT>(q, z, r, row, x[i0 + k], i0 + k) : 0;
    s += mine[k];
  }
  upto = wave_scan(s);
  if (lane == 63) part[wave] = upto;
  __syncthreads();
  at = at_before + upto - s;
  for (int w = 0; w < wave; ++w) at += part[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (at < need && need <= at + mine[k]) q.token[b] = i0 + k;
    at += mine[k];
  }
}

// ---- beams: the groups ----------------------------------------------------------------------------

constexpr int kMostBeams = 4096;  // width * keep

// The best of a group's rows' best, in order: values score + logit - log sum, ties by row and token.
__global__ void __launch_bounds__(1024) beams_kernel(const SamplingParams q, int size) {
  extern __shared__ __align__(16) uint8_t smem[];
  double* const val = reinterpret_cast<double*>(smem);
  uint64_t* const who = reinterpret_cast<uint64_t*>(smem + 8 * static_cast<size_t>(size));
  const int tid = threadIdx.x, g = blockIdx.x;
  for (int i = tid; i < size; i += blockDim.x) {
    double v = -__builtin_huge_val();
    uint64_t w = ~0ull;
    const int r = i / q.keep, j = i - r * q.keep;
    if (r < q.width) {
      const int row = g * q.width + r;
      const float score = q.scores[row];
      if (static_cast<uint32_t>(j) < q.nbest[row] && score > -__builtin_huge_valf()) {
        const uint2 x = q.best[static_cast<int64_t>(row) * q.keep + j];
        const Row& r = q.rowres[row];  // (kept: the logarithm of the sum)
        v = static_cast<double>(score) + ((static_cast<double>(logit_of_key(x.x)) - static_cast<double>(r.max)) - r.kept);
        w = static_cast<uint64_t>(row) << 32 | x.y;
      }
    }
    val[i] = v;
    who[i] = w;
  }
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = tid; i < size; i += blockDim.x) {
        const int o = i ^ j;
        if (o > i) {
          const double a = val[i], c = val[o];
          const uint64_t wa = who[i], wc = who[o];
          const bool after = a < c || (a == c && wa > wc);  // i belongs behind o
          if (after == ((i & k) == 0)) val[i] = c, val[o] = a, who[i] = wc, who[o] = wa;
        }
      }
      __syncthreads();
    }
  for (int i = tid; i < q.keep; i += blockDim.x) {
    const uint64_t w = who[i];
    const int64_t to = static_cast<int64_t>(g) * q.keep + i;
    q.parents[to] = w == ~0ull ? -1 : static_cast<int32_t>(w >> 32);
    q.token[to] = w == ~0ull ? -1 : static_cast<int64_t>(w & 0xffffffffu);
    q.out_scores[to] = static_cast<float>(val[i]);
  }
}

// ---- host -----------------------------------------------------------------------------------------

// Up to how many rows of V their chunks have workgroups of their own.  Four launches cost some 29 us and 2e-6 us an
// element of all rows; one launch some 20 us and 3.2e-4 us an element of a row, of bf16 by value 25 us and 1.45e-4 us.
// So the borders' two sides, split and whole: fp32, 131072: 59.3 and 63.8 us with 96 rows, 70.0 and 64.6 with 128; 65536: 32.9 and 42.1
// with 32, 42.6 and 41.9 with 96; 32768: 30.0 and 29.5 with 8; fp16, 131072: 50.8 and 60.2 with 96, 63.1 and 62.2 with 160;
// 65536: 39.2 and 41.3 with 64, 40.7 and 41.8 with 96, 50.2 and 42.1 with 128; bf16, 131072: 41.3 and 45.1 with 48, 48.7 and 45.2 with
// 64; 65536: 30.5 and 36.0 with 8, 38.7 and 35.7 with 64; 32768: 29.9 and 30.2 with 8, 31.5 and 30.6 with 64.
int64_t split_rows(int64_t V, int dtype) { return dtype == MZK_BF16 ? 72 - (3 << 20) / V : 144 - (5 << 20) / V; }

int64_t up(int64_t x) { return (x + 255) & ~static_cast<int64_t>(255); }

// The workspace's parts, in order; returns the bytes.
int64_t lay(SamplingParams& q, uint8_t* ws) {
  int64_t at = 0;
  auto take = [&](auto*& to, int64_t n) {
    to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(ws + at);
    at += up(n * static_cast<int64_t>(sizeof(*to)));
  };
  const int64_t r = q.rows, rc = q.chunks > 1 ? r * q.chunks : 0;
  take(q.heads, rc);
  take(q.hist, rc * kBins);
  take(q.counts, rc * kBins);
  const int64_t split = q.chunks > 1 ? r : 0;
  take(q.plans, split);
  take(q.sums, split * kBins);
  take(q.sum_counts, split * kBins);
  take(q.listed, split);
  take(q.list, split * kCap);
  if (q.mode != kSample) take(q.rowres, r);
  if (q.mode == kVerify && q.probs) {
    take(q.refused, q.B);
    take(q.rest, static_cast<int64_t>(q.B) * q.rest_chunks);
  }
  if (q.mode == kBeams) {
    take(q.best, r * q.keep);
    take(q.nbest, r);
  }
  return at;
}

// The dynamic-LDS limit is a per-device function attribute: set once per device.
template <typename K>
bool raise_lds(K kern, int bytes, std::atomic<bool> (&set)[kMaxDevices]) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    set_last_error("sampling: no usable current device");
    return false;
  }
  if (!set[dev].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
      set_last_error("sampling: cannot raise the kernel's LDS limit to %d bytes", bytes);
      return false;
    }
    set[dev].store(true, std::memory_order_release);
  }
  return true;
}

template <int DT>
int launch(const SamplingParams& q, hipStream_t s) {
  static std::atomic<bool> whole_set[kMaxDevices] = {}, finish_set[kMaxDevices] = {};
  const unsigned rows = static_cast<unsigned>(q.rows);
  if (q.chunks == 1) {
    if (!raise_lds(row_kernel<DT, kWholeRow>, kRowLds, whole_set)) return MZK_ELAUNCH;
    row_kernel<DT, kWholeRow><<<rows, kRowThreads, kRowLds, s>>>(q);
  } else {
    if (!raise_lds(row_kernel<DT, kFinishPart>, kRowLds, finish_set)) return MZK_ELAUNCH;
    const unsigned grid = (rows + 7) / 8 * 8 * static_cast<unsigned>(q.chunks);
    survey_kernel<DT><<<grid, kSurveyThreads, 0, s>>>(q);
    row_kernel<DT, kPlanPart><<<rows, kRowThreads, kBinsLds, s>>>(q);
    list_kernel<DT><<<grid, kSurveyThreads, 0, s>>>(q);
    row_kernel<DT, kFinishPart><<<rows, kRowThreads, kRowLds, s>>>(q);
  }
  if (q.mode == kVerify) {
    if (!q.probs) {
      verify_kernel<<<static_cast<unsigned>((q.B + 3) / 4), 256, 0, s>>>(q);
    } else {
      rest_kernel<DT><<<static_cast<unsigned>(q.B) * static_cast<unsigned>(q.rest_chunks), 256, 0, s>>>(q);
      redraw_kernel<DT><<<static_cast<unsigned>(q.B), 256, 0, s>>>(q);
    }
  }
  if (q.mode == kBeams) {
    int size = 2;
    while (size < q.width * q.keep) size <<= 1;
    beams_kernel<<<static_cast<unsigned>(q.rows / q.width), size < 1024 ? (size < 64 ? 64 : size) : 1024, static_cast<size_t>(size) * 16, s>>>(q, size);
  }
  MZK_LAUNCH_CHECK("sampling");
  return MZK_OK;
}

int size_of(int dtype) { return dtype == MZK_F32 ? 4 : 2; }

// What every call checks of its rows, and the parts of the parameters that follow from them.
int rows_of(SamplingParams& q, const char* name, int64_t rows, int64_t V, int dtype) {
  MZK_CHECK_ARG(dtype >= MZK_F32 && dtype <= MZK_F16, "%s: unsupported dtype %d", name, dtype);
  MZK_CHECK_ARG(rows >= 0 && V >= 1, "%s: bad sizes", name);
  MZK_CHECK_ARG(V <= kMaxVocab, "%s: at most %lld logits a row, got %lld", name, (long long)kMaxVocab, (long long)V);
  // a launch has less than 2^32 threads
  MZK_CHECK_ARG(rows < (1 << 22), "%s: too many rows: %lld", name, (long long)rows);
  q.V = static_cast<int>(V);
  q.scale = 62;
  while ((static_cast<int64_t>(1) << (62 - q.scale)) < V) --q.scale;
  // Chunks: of whole steps of a survey's workgroup, so that there are some 512 workgroups.
  const int64_t step = kSurveyThreads * kSurveyElements * size_of(dtype) / 16, pieces = V * size_of(dtype) / 16 + 2;
  const int64_t steps = (pieces + step - 1) / step;
  int64_t chunks = rows == 0 || rows > split_rows(V, dtype) ? 1 : 512 / rows;
  if (chunks > kMostChunks) chunks = kMostChunks;
  if (chunks > steps) chunks = steps;
  const int64_t per = (steps + chunks - 1) / chunks;
  q.chunk_pieces = static_cast<int>(per * step);
  q.chunks = static_cast<int>((steps + per - 1) / per);
  q.rest_chunks = static_cast<int>((V + kRestElements - 1) / kRestElements);
  q.rows = static_cast<int>(rows);
  return MZK_OK;
}

int run(SamplingParams& q, const char* name, const void* logits, int64_t stride, int dtype, void* workspace, int64_t workspace_bytes,
        void* stream) {
  MZK_CHECK_ARG(logits, "%s: null pointer", name);
  MZK_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % size_of(dtype) == 0 && aligned16(workspace), "%s: misaligned logits or workspace", name);
  MZK_CHECK_ARG(stride >= q.V || q.rows <= 1, "%s: rows of logits overlap", name);
  q.logits = static_cast<const uint8_t*>(logits);
  q.stride = stride * size_of(dtype);
  const int64_t need = lay(q, static_cast<uint8_t*>(workspace));
  MZK_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace needs %lld bytes", name, (long long)need);
  const hipStream_t s = as_stream(stream);
  return dtype == MZK_F32 ? launch<MZK_F32>(q, s) : dtype == MZK_BF16 ? launch<MZK_BF16>(q, s) : launch<MZK_F16>(q, s);
}

int bytes_of(SamplingParams& q, int64_t* bytes) {
  *bytes = q.rows ? lay(q, nullptr) : 0;
  return MZK_OK;
}

}  // namespace
}  // namespace mzk

using namespace mzk;

extern "C" int mzk_sample_workspace_bytes(int64_t rows, int64_t V, int dtype, int64_t* bytes) {
  MZK_CHECK_ARG(bytes != nullptr, "sample_workspace_bytes: null output");
  SamplingParams q{};
  q.mode = kSample;
  if (const int rc = rows_of(q, "sample_workspace_bytes", rows, V, dtype)) return rc;
  return bytes_of(q, bytes);
}

extern "C" int mzk_sample(const void* logits, int dtype, int64_t rows, int64_t V, int64_t row_stride, const float* u,
                          const float* temperature, float temperature_all, const int32_t* top_k, int top_k_all,
                          const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* tokens,
                          float* logprobs, void* workspace, int64_t workspace_bytes, void* stream) {
  SamplingParams q{};
  q.mode = kSample;
  if (const int rc = rows_of(q, "sample", rows, V, dtype)) return rc;
  if (rows == 0) return MZK_OK;
  MZK_CHECK_ARG(u && tokens && logprobs, "sample: null pointer");
  q.temperature = Filter{temperature, temperature_all};
  q.top_p = Filter{top_p, top_p_all};
  q.min_p = Filter{min_p, min_p_all};
  q.top_k = top_k;
  q.top_k_all = top_k_all;
  q.u = u;
  q.token = tokens;
  q.logprob = logprobs;
  return run(q, "sample", logits, row_stride, dtype, workspace, workspace_bytes, stream);
}

extern "C" int mzk_verify_workspace_bytes(int64_t T, int64_t B, int64_t V, int dtype, int probs, int64_t* bytes) {
  MZK_CHECK_ARG(bytes != nullptr, "verify_workspace_bytes: null output");
  MZK_CHECK_ARG(B >= 0 && B < 1 << 22, "verify_workspace_bytes: bad sizes");
  SamplingParams q{};
  q.mode = kVerify;
  if (const int rc = rows_of(q, "verify_workspace_bytes", T, V, dtype)) return rc;
  q.B = static_cast<int>(B);
  const float some = 0.0f;
  q.probs = probs ? &some : nullptr;  // only whether there are any counts
  *bytes = lay(q, nullptr);
  return MZK_OK;
}

extern "C" int mzk_verify(const void* logits, int dtype, int64_t T, int64_t V, int64_t row_stride, const int64_t* tokens,
                          const int64_t* cu, int64_t B, const float* u, const float* draw, const float* draft_probs,
                          int64_t draft_row_stride, const float* temperature, float temperature_all, const int32_t* top_k,
                          int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                          int64_t* accepted, int64_t* next, void* workspace, int64_t workspace_bytes, void* stream) {
  SamplingParams q{};
  q.mode = kVerify;
  if (const int rc = rows_of(q, "verify", T, V, dtype)) return rc;
  MZK_CHECK_ARG(B >= 0 && B < 1 << 22 && (!draft_probs || B * q.rest_chunks < 1 << 24), "verify: bad sizes");
  if (B == 0) return MZK_OK;
  MZK_CHECK_ARG(cu && accepted && next && draw && (T == 0 || (tokens && u)), "verify: null pointer");
  MZK_CHECK_ARG(!draft_probs || draft_row_stride >= V || T <= 1, "verify: rows of the draft's probabilities overlap");
  q.temperature = Filter{temperature, temperature_all};
  q.top_p = Filter{top_p, top_p_all};
  q.min_p = Filter{min_p, min_p_all};
  q.top_k = top_k;
  q.top_k_all = top_k_all;
  q.u = u;
  q.tokens = tokens;
  q.cu = cu;
  q.B = static_cast<int>(B);
  q.draw = draw;
  q.probs = draft_probs;
  q.probs_stride = draft_row_stride;
  q.accepted = accepted;
  q.token = next;
  if (T == 0) {  // no rows: sequences of nothing
    q.probs = nullptr;
    verify_kernel<<<static_cast<unsigned>((B + 3) / 4), 256, 0, as_stream(stream)>>>(q);
    MZK_LAUNCH_CHECK("verify");
    return MZK_OK;
  }
  return run(q, "verify", logits, row_stride, dtype, workspace, workspace_bytes, stream);
}

extern "C" int mzk_beams_workspace_bytes(int64_t rows, int64_t V, int dtype, int keep, int64_t* bytes) {
  MZK_CHECK_ARG(bytes != nullptr, "beams_workspace_bytes: null output");
  MZK_CHECK_ARG(keep >= 1 && keep <= kMostBeams, "beams_workspace_bytes: bad sizes");
  SamplingParams q{};
  q.mode = kBeams;
  if (const int rc = rows_of(q, "beams_workspace_bytes", rows, V, dtype)) return rc;
  q.keep = keep;
  return bytes_of(q, bytes);
}

extern "C" int mzk_beams(const void* logits, int dtype, int64_t rows, int64_t V, int64_t row_stride, const float* scores,
                         int width, int keep, int32_t* parents, int64_t* tokens, float* out_scores, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  SamplingParams q{};
  q.mode = kBeams;
  if (const int rc = rows_of(q, "beams", rows, V, dtype)) return rc;
  MZK_CHECK_ARG(width >= 1 && keep >= 1 && static_cast<int64_t>(width) * keep <= kMostBeams,
                "beams: width and keep of at least 1, width * keep of at most %d", kMostBeams);
  MZK_CHECK_ARG(rows % width == 0, "beams: %lld rows are no groups of %d", (long long)rows, width);
  if (rows == 0) return MZK_OK;
  MZK_CHECK_ARG(scores && parents && tokens && out_scores, "beams: null pointer");
  // (a group's workgroup reads its scores and then writes its new ones)
  const uintptr_t from = reinterpret_cast<uintptr_t>(scores), to = reinterpret_cast<uintptr_t>(out_scores);
  MZK_CHECK_ARG((from == to && keep == width) || to >= from + 4u * static_cast<uintptr_t>(rows) ||
                    from >= to + 4u * static_cast<uintptr_t>(rows / width * keep),
                "beams: the out scores are the scores themselves, as many, or overlap none of them");
  q.scores = scores;
  q.width = width;
  q.keep = keep;
  q.parents = parents;
  q.token = tokens;
  q.out_scores = out_scores;
  return run(q, "beams", logits, row_stride, dtype, workspace, workspace_bytes, stream);
}
