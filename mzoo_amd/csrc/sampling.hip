// From logits to the next tokens: sampling behind temperature, top-k, top-p and min-p, verification of
// drafted tokens, and the step of a beam search.
//
// A row's tokens stand in the order of falling logits, equal ones by rising index.  With the weights
//   w_i = exp((l_i - max l) / T)
// top-k keeps the first k of the order, top-p the shortest prefix of those whose weights reach p of their
// sum, min-p those of at least min_p times the first one's weight: each keeps a prefix, so together the
// shortest.  The token drawn is the first whose running sum exceeds u times the kept sum W.  (T <= 0: the
// first of the order.)  NaN and -inf are no tokens; +inf counts as the largest finite number, -0 as 0.
//
// Tokens are whole numbers, so a token beside a border of the running sum has to come out right: weights
// are computed in 64 bits to about 2^-50 of themselves, and summed as whole numbers, in any order the same.
//
// No row is sorted.  Three launches, none of which needs another's workgroups at the same time:
//   survey   chunks of a row: the chunk's maximum and a histogram of its weights over bins of 1/10 octave,
//            51 octaves down; what lies below them is 2^-50 of the largest weight and counts as 0
//   narrow   every chunk's workgroup joins the row's histograms, finds the few bins in which the cuts of
//            the filters and the drawn token lie, and lists its tokens of these bins
//   finish   a workgroup for each row finds the exact cuts and the token among the listed ones, by
//            weighted radix selection: a histogram over the bits that the open range of keys has left
#include "common.h"

namespace mzk {
namespace {

constexpr int kBins = 512, kRest = kBins - 1;  // the last bin takes what is too small to count
constexpr double kPerOctave = 10.0;
constexpr double kLog2eD = 1.4426950408889634074, kLn2D = 0.69314718055994530942;
constexpr int kCap = 16384;  // listed tokens of a row; where there are more, finish reads the row itself
constexpr int64_t kMaxVocab = 1 << 20;
constexpr uint32_t kNone = 0xffffffffu;

enum Mode { kSample, kVerify, kBeams };

// Bins b0 .. b1 in which something has to be found (none: b1 < b0), and the weights of the bins before them.
struct Window {
  int b0, b1;
  double before;
};

// What narrow leaves of a row for finish.
struct Plan {
  double total;       // all weights
  Window k, p, f, d;  // top-k's cut, top-p's, min-p's, the drawn token
  uint32_t count_before;  // tokens in the bins before k.b0
  float max;
};

// What finish leaves of a row for the launches behind it.
struct Row {
  double kept;             // W
  uint32_t ik, idx;        // the last token of the order that top-k and top-p keep: its key and index
  float max;
  int32_t accepted, token;
};

struct Filter {
  const float* f;  // one for each row, or null: `all` for every row
  float all;
  __device__ float operator()(int row) const { return f ? f[row] : all; }
};

struct SamplingParams {
  const uint8_t* logits;
  int64_t stride;  // bytes from row to row
  int V, rows, chunks;
  Mode mode;
  Filter temperature, top_p, min_p;
  const int32_t* top_k;
  int top_k_all;
  int count;  // whether tokens are counted: some row may have a top-k
  int scale;  // log2 of the whole number that stands for the largest weight: V of them stay below 2^63
  const float* u;  // [rows]
  // verify
  const int64_t* tokens;  // [rows]
  const int64_t* cu;      // [B + 1]
  int B;
  const float* draw;   // [B]
  const float* probs;  // [rows, V] or null
  int64_t probs_stride;
  // beams
  const float* scores;  // [rows]
  int width, keep;
  // workspace
  float* heads;      // [rows][chunks] maxima
  uint64_t* hist;    // [rows][chunks][kBins] weights, 2^50 the chunk's largest
  uint32_t* counts;  // the same, tokens
  Plan* plans;       // [rows]
  uint32_t* listed;  // [rows]
  uint2* list;       // [rows][kCap] key and index
  Row* rowres;       // [rows]
  int32_t* refused;  // [B] the row of a refused token, or -1
  uint64_t* rest;    // [B][chunks] sums of what the target has above the draft
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

// 2^t for t <= 0, to about 2^-51 of itself: the power series of exp(f ln 2) for |f| <= 1/2, whose
// first term left out is (ln 2 / 2)^13 / 13! = 1.7e-16.
__device__ __forceinline__ double exp2_neg(double t) {
  t = fmax(t, -1100.0);
  const double n = __builtin_rint(t);
  const double x = (t - n) * kLn2D;
  double e = 1.0 / 479001600.0;
  e = __builtin_fma(e, x, 1.0 / 39916800.0);
  e = __builtin_fma(e, x, 1.0 / 3628800.0);
  e = __builtin_fma(e, x, 1.0 / 362880.0);
  e = __builtin_fma(e, x, 1.0 / 40320.0);
  e = __builtin_fma(e, x, 1.0 / 5040.0);
  e = __builtin_fma(e, x, 1.0 / 720.0);
  e = __builtin_fma(e, x, 1.0 / 120.0);
  e = __builtin_fma(e, x, 1.0 / 24.0);
  e = __builtin_fma(e, x, 1.0 / 6.0);
  e = __builtin_fma(e, x, 0.5);
  e = __builtin_fma(e, x, 1.0);
  e = __builtin_fma(e, x, 1.0);
  return __builtin_ldexp(e, static_cast<int>(n));
}

// A number of 0 .. 2^51 to the nearest whole one: the low bits of its sum with 2^52.
__device__ __forceinline__ uint64_t whole(double x) {
  return static_cast<uint64_t>(__double_as_longlong(x + 4503599627370496.0)) & 0xfffffffffffffull;
}

// A random number as one of [0, 1): NaN as 0.
__device__ __forceinline__ double unit(float u) { return u > 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0; }

// A logit as it counts: NaN as -inf, +inf as the largest finite number, -0 as 0.
__device__ __forceinline__ float logit_of(float x) {
  x = x != x ? -__builtin_huge_valf() : x + 0.0f;
  return x > 3.402823466e38f ? 3.402823466e38f : x;
}
// Keys rise as logits fall.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float logit_of_key(uint32_t ik) { return __uint_as_float(ik & 0x80000000u ? ik : ~ik & 0x7fffffffu); }

// ---- a row's settings -------------------------------------------------------------------------

struct Settings {
  double s, s_bin;  // log2 e / T, and bins
  int k;            // 0: none
  double p;         // 1: none
  double f;         // log2 min_p; -inf: none
  bool first;       // T <= 0: the first of the order
};
__device__ __forceinline__ Settings settings(const SamplingParams& q, int row) {
  Settings z;
  const float t = q.mode == kBeams ? 1.0f : q.temperature(row);
  z.first = !(t > 0.0f);
  z.s = kLog2eD / (z.first ? 1.0 : static_cast<double>(t));
  z.s_bin = z.s * kPerOctave;
  z.k = q.mode == kBeams ? q.keep : q.top_k ? q.top_k[row] : q.top_k_all;
  if (q.mode != kBeams && (z.k < 0 || z.k >= q.V)) z.k = 0;
  const float p = q.mode == kBeams ? 1.0f : q.top_p(row);
  z.p = z.first ? 0.0 : p < 1.0f ? (p > 0.0f ? static_cast<double>(p) : 0.0) : 1.0;
  const float f = q.mode == kBeams ? 0.0f : q.min_p(row);
  z.f = f > 0.0f ? (f < 1.0f ? log2(static_cast<double>(f)) : 0.0) : -__builtin_huge_val();
  if (z.first) z.k = 0, z.f = -__builtin_huge_val();
  return z;
}

// The bin below a maximum whose place on the grid is `top`; kRest for what is too small.
__device__ __forceinline__ int bin_of(float l, double s_bin, double top) {
  return static_cast<int>(fmin(top - __builtin_floor(static_cast<double>(l) * s_bin), static_cast<double>(kRest)));
}

// ---- loads ------------------------------------------------------------------------------------

// A chunk: 256 threads, EPT elements each, in whole 16-byte pieces of memory as far as they lie inside the row.
template <int DT, int EPT>
struct Chunk {
  static constexpr int SIZE = DT == MZK_F32 ? 4 : 2, N = 16 / SIZE, PIECES = EPT / N;
  // elements of a row before the first whole piece are counted from the piece that they lie in
  __device__ static int mis(const uint8_t* row) { return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / SIZE); }
  __device__ static float value(const uint8_t* row, int i) { return logit_of(load_as_f32<DT>(row, i)); }
  // the index of element i (of EPT) of this thread
  __device__ static int index(int chunk, int tid, int i, int mis) { return (chunk * 256 * PIECES + (i / N) * 256 + tid) * N + i % N - mis; }
  __device__ static void load(const uint8_t* row, int V, int chunk, int tid, int mis, float (&v)[EPT]) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int e = index(chunk, tid, k * N, mis);
      if (e >= 0 && e + N <= V) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + static_cast<int64_t>(e) * SIZE);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (DT == MZK_F32) {
            v[k * N + j] = logit_of(__uint_as_float(w[j]));
          } else {
            const uint16_t h[2] = {static_cast<uint16_t>(w[j] & 0xffffu), static_cast<uint16_t>(w[j] >> 16)};
#pragma unroll
            for (int i = 0; i < 2; ++i) v[k * N + 2 * j + i] = logit_of(DT == MZK_BF16 ? bf16_to_f32(h[i]) : f16_to_f32(h[i]));
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[k * N + j] = e + j >= 0 && e + j < V ? value(row, e + j) : -__builtin_huge_valf();
      }
    }
  }
};

// The sequence of a row of packed ones and the row behind its last; false: none.
__device__ __forceinline__ bool sequence_of(const SamplingParams& q, int row, int lane, int& b, int& end) {
  for (int b0 = 0; b0 < q.B; b0 += 64) {
    const int64_t z = b0 + lane < q.B ? q.cu[b0 + lane + 1] : 0;
    const uint64_t in = __ballot(b0 + lane < q.B && z > row);
    if (in) {
      const int at = __builtin_ctzll(in);
      b = b0 + at;
      const int64_t e = q.cu[b + 1];
      end = e < q.rows ? static_cast<int>(e) : q.rows;
      return q.cu[b] <= row;
    }
  }
  return false;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

// ---- survey -------------------------------------------------------------------------------------

template <int DT, int EPT>
__global__ void __launch_bounds__(256) survey_kernel(const SamplingParams q) {
  using C = Chunk<DT, EPT>;
  __shared__ unsigned long long hist[kBins];
  __shared__ uint32_t counts[kBins];
  __shared__ float top[4];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / q.chunks, chunk = blockIdx.x - row * q.chunks;
  if (q.mode == kVerify && q.cu[q.B] <= row) return;  // a row of no sequence
  const uint8_t* const base = q.logits + row * q.stride;
  float v[EPT];
  C::load(base, q.V, chunk, tid, C::mis(base), v);
  const Settings z = settings(q, row);
  for (int i = tid; i < kBins; i += 256) {
    hist[i] = 0;
    counts[i] = 0;
  }
  float m = v[0];
#pragma unroll
  for (int i = 1; i < EPT; ++i) m = fmaxf(m, v[i]);
  m = wave_max(m);
  if ((tid & 63) == 0) top[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const int64_t at = static_cast<int64_t>(row) * q.chunks + chunk;
  if (tid == 0) {
    q.heads[at] = m;
    if (chunk == 0) q.listed[row] = 0;
  }
  if (m == -__builtin_huge_valf()) return;  // uniform
  const double grid = __builtin_floor(static_cast<double>(m) * z.s_bin);
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const int j = bin_of(v[i], z.s_bin, grid);
    if (j < kRest) {
      const double t = (static_cast<double>(v[i]) - static_cast<double>(m)) * z.s;
      atomicAdd(&hist[j], static_cast<unsigned long long>(whole(exp2_neg(t) * 0x1p50)));
      if (q.count) atomicAdd(&counts[j], 1u);
    }
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += 256) {
    q.hist[at * kBins + i] = hist[i];
    if (q.count) q.counts[at * kBins + i] = counts[i];
  }
}

// ---- narrow -------------------------------------------------------------------------------------

template <int DT, int EPT>
__global__ void __launch_bounds__(256) narrow_kernel(const SamplingParams q) {
  using C = Chunk<DT, EPT>;
  constexpr int kMost = 1024;  // chunks of a row
  __shared__ float heads[kMost];
  __shared__ double factor[kMost];
  __shared__ int shift[kMost];
  __shared__ uint64_t cw[kBins];  // running sums of the bins' weights
  __shared__ uint32_t cn[kBins];
  __shared__ uint64_t part_w[4];
  __shared__ uint32_t part_n[4];
  __shared__ float top[4];
  __shared__ int found[3][4][4];
  __shared__ uint32_t base_at;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / q.chunks, chunk = blockIdx.x - row * q.chunks;
  int b = 0, end = 0;
  if (q.mode == kVerify && !sequence_of(q, row, lane, b, end)) return;  // uniform
  const uint8_t* const base = q.logits + row * q.stride;
  const Settings z = settings(q, row);

  // the row's maximum, and where the chunks' bins lie among the row's
  float m = -__builtin_huge_valf();
  for (int c = tid; c < q.chunks; c += 256) {
    const float h = q.heads[static_cast<int64_t>(row) * q.chunks + c];
    heads[c] = h;
    m = fmaxf(m, h);
  }
  m = wave_max(m);
  if (lane == 0) top[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  Plan plan{};
  plan.max = m;
  plan.k = plan.p = plan.f = plan.d = Window{1, 0, 0.0};
  if (m == -__builtin_huge_valf()) {  // uniform: no token at all
    if (chunk == 0 && tid == 0) q.plans[row] = plan;
    return;
  }
  const double grid = __builtin_floor(static_cast<double>(m) * z.s_bin);
  for (int c = tid; c < q.chunks; c += 256) {
    const float h = heads[c];
    const bool some = h > -__builtin_huge_valf();
    shift[c] = some ? bin_of(h, z.s_bin, grid) : kBins;
    factor[c] = some ? exp2_neg((static_cast<double>(h) - static_cast<double>(m)) * z.s) * 0x1p-50 : 0.0;
  }
  __syncthreads();
  double w0 = 0.0, w1 = 0.0;  // bins 2 tid, 2 tid + 1 of the row
  uint32_t n0 = 0, n1 = 0;
  const int64_t at = static_cast<int64_t>(row) * q.chunks;
  for (int c = 0; c < q.chunks; ++c) {
    const int j = 2 * tid - shift[c];
    const double f = factor[c];
    const uint64_t* const h = q.hist + (at + c) * kBins;
    if (j >= 0) w0 = w0 + static_cast<double>(h[j]) * f;
    if (j + 1 >= 0 && j + 1 < kRest && 2 * tid + 1 < kRest) w1 = w1 + static_cast<double>(h[j + 1]) * f;
    if (q.count) {
      const uint32_t* const n = q.counts + (at + c) * kBins;
      if (j >= 0) n0 += n[j];
      if (j + 1 >= 0 && j + 1 < kRest && 2 * tid + 1 < kRest) n1 += n[j + 1];
    }
  }
  // As whole numbers from here: sums of them do not depend on their order, and a bin of nothing adds nothing.
  const double scale = __builtin_ldexp(1.0, q.scale), unscale = __builtin_ldexp(1.0, -q.scale);
  {
    const uint64_t i0 = static_cast<uint64_t>(w0 * scale + 0.5), i1 = static_cast<uint64_t>(w1 * scale + 0.5);
    const uint64_t s = wave_scan(i0 + i1, lane);
    const uint32_t n = wave_scan(n0 + n1, lane);
    if (lane == 63) part_w[wave] = s, part_n[wave] = n;
    __syncthreads();
    uint64_t before = s - (i0 + i1);
    uint32_t nbefore = n - (n0 + n1);
    for (int w = 0; w < wave; ++w) before += part_w[w], nbefore += part_n[w];
    cw[2 * tid] = before + i0;
    cw[2 * tid + 1] = before + i0 + i1;
    cn[2 * tid] = nbefore + n0;
    cn[2 * tid + 1] = nbefore + n0 + n1;
  }
  __syncthreads();
  auto upto = [&](int j) -> double { return static_cast<double>(cw[j]); };  // of `scale`
  auto before = [&](int j) -> double { return j > 0 ? static_cast<double>(cw[j - 1]) : 0.0; };
  const double total = upto(kRest);
  plan.total = total * unscale;
  // the first bin whose running sum is not below x
  int round = 0;
  auto find = [&](auto below_a, auto below_c, int& a, int& c) {
    const int na = __popcll(__ballot(below_a(2 * tid))) + __popcll(__ballot(below_a(2 * tid + 1)));
    const int nc = __popcll(__ballot(below_c(2 * tid))) + __popcll(__ballot(below_c(2 * tid + 1)));
    if (lane == 0) found[round][wave][0] = na, found[round][wave][1] = nc;
    __syncthreads();
    a = c = 0;
    for (int w = 0; w < 4; ++w) a += found[round][w][0], c += found[round][w][1];
    ++round;
  };
  int last, unused;
  // weights kept: between least and most
  double k_least = total, k_most = total;
  if (z.k) {
    int kb;
    find([&](int j) { return cn[j] < static_cast<uint32_t>(z.k); }, [&](int j) { return upto(j) < total; }, kb, last);
    if (kb < kRest) {
      plan.k = Window{kb, kb, before(kb) * unscale};
      plan.count_before = kb > 0 ? cn[kb - 1] : 0;
      k_least = before(kb);
      k_most = upto(kb);
    }
  } else {
    find([&](int j) { return upto(j) < total; }, [&](int) { return false; }, last, unused);
  }
  double least = k_least, most = k_most;
  if (z.p < 1.0) {
    int lo, hi;
    find([&](int j) { return upto(j) < z.p * k_least; }, [&](int j) { return upto(j) < z.p * k_most; }, lo, hi);
    if (hi > last) hi = last;
    if (lo > hi) lo = hi;
    plan.p = Window{lo, hi, before(lo) * unscale};
    // a token of bin j weighs 2^-((j - 1) / 10) at most
    const double over = z.p * k_most + exp2_neg(-(lo > 1 ? lo - 1 : 0) / kPerOctave) * scale;
    least = fmin(least, z.p * k_least);
    most = fmin(most, fmin(upto(hi), over));
  }
  if (z.f > -__builtin_huge_val()) {
    const double y = (static_cast<double>(m) * z.s + z.f) * kPerOctave, eps = 1e-6 + fabs(y) * 1e-13;
    const int lo = static_cast<int>(fmin(fmax(grid - __builtin_floor(y + eps), 0.0), static_cast<double>(kRest)));
    int hi = static_cast<int>(fmin(fmax(grid - __builtin_floor(y - eps), 0.0), static_cast<double>(kRest)));
    if (lo < kRest) {
      if (hi >= kRest) hi = kRest - 1;
      plan.f = Window{lo, hi, before(lo) * unscale};
      least = fmin(least, before(lo));
      most = fmin(most, upto(hi));
    }
  }
  if (q.mode == kBeams) {
    // with fewer tokens than wanted among the bins that count, all of the row's
    plan.k = Window{0, plan.k.b1 >= plan.k.b0 ? plan.k.b1 : kRest, 0.0};
    plan.count_before = 0;
    if (plan.k.b1 == kRest && chunk == 0 && tid == 0) atomicAdd(&q.listed[row], static_cast<uint32_t>(kCap) + 1u);
  } else {
    // The drawn token.  In verify a refused token that the draft was sure of leaves the row: with its bin
    // before the cuts it is kept, behind them not, among them one or the other.
    const double u = z.first ? 0.0 : unit(q.mode == kVerify ? q.draw[b] : q.u[row]);
    double wd = 0.0;
    int bd = kBins;
    bool sure = true;
    if (q.mode == kVerify && !q.probs && row + 1 < end) {
      const int64_t d = q.tokens[row + 1];
      if (d >= 0 && d < q.V) {
        const float l = C::value(base, static_cast<int>(d));
        if (l > -__builtin_huge_valf()) {
          bd = bin_of(l, z.s_bin, grid);
          int cut = kRest - 1, open = kBins;  // bins before `open` are kept, behind `cut` are not
          if (plan.k.b1 >= plan.k.b0) open = plan.k.b0, cut = plan.k.b1;
          if (plan.p.b1 >= plan.p.b0) open = min(open, plan.p.b0), cut = min(cut, plan.p.b1);
          if (plan.f.b1 >= plan.f.b0) open = min(open, plan.f.b0), cut = min(cut, plan.f.b1);
          if (bd <= cut) wd = exp2_neg((static_cast<double>(l) - static_cast<double>(m)) * z.s) * scale;
          sure = bd < open || bd > cut;
        }
      }
    }
    // (the slack covers the roundings of the bins' sums and of wd)
    const double slack = bd < kBins ? 2048.0 : 0.0;
    const double lo_x = u * fmax(least - wd, 0.0) - slack, hi_x = u * (sure ? most - wd : most) + slack;
    int lo, hi;
    find([&](int j) { return (sure && j >= bd ? upto(j) - wd : upto(j)) <= lo_x; },
         [&](int j) { return (j >= bd ? upto(j) - wd : upto(j)) <= hi_x; }, lo, hi);
    if (hi > last) hi = last;
    if (lo > hi) lo = hi;
    plan.d = Window{lo, hi, before(lo) * unscale};
  }
  if (chunk == 0 && tid == 0) q.plans[row] = plan;

  // this chunk's tokens of the windows
  const Window win[4] = {plan.k, plan.p, plan.f, plan.d};
  int hull0 = kBins, hull1 = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (win[i].b1 >= win[i].b0) {
      hull0 = min(hull0, win[i].b0);
      hull1 = max(hull1, win[i].b1);
    }
  if (shift[chunk] > hull1) return;  // uniform: all of it lies below
  const int mis = C::mis(base);
  float v[EPT];
  C::load(base, q.V, chunk, tid, mis, v);
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const int j = bin_of(v[i], z.s_bin, grid);
    if (j < kRest && j >= hull0 && j <= hull1) {
      bool in = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) in = in || (j >= win[w].b0 && j <= win[w].b1);
      mine |= static_cast<uint32_t>(in) << i;
    }
  }
  const uint32_t n = __popc(mine);
  const uint32_t incl = wave_scan(n, lane);
  __shared__ uint32_t sums[4];
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  if (tid == 0) {
    const uint32_t all = sums[0] + sums[1] + sums[2] + sums[3];
    base_at = all ? atomicAdd(&q.listed[row], all) : 0;
  }
  __syncthreads();
  uint32_t to = base_at + incl - n;
  for (int w = 0; w < wave; ++w) to += sums[w];
#pragma unroll
  for (int i = 0; i < EPT; ++i)
    if (mine >> i & 1u) {
      if (to < kCap) q.list[static_cast<int64_t>(row) * kCap + to] = uint2{key_of(v[i]), static_cast<uint32_t>(C::index(chunk, tid, i, mis))};
      ++to;
    }
}

// ---- finish -------------------------------------------------------------------------------------

constexpr int kFinish = 1024;  // threads

// A token of the order: weights up to and with it.
struct Found {
  uint32_t ik, idx;
  double upto, w;
};

template <int DT>
struct Finish {
  const SamplingParams& q;
  const Settings& z;
  const Plan& plan;
  const uint8_t* base;
  double grid;
  bool in_list;
  int n;
  int tid, lane, wave;
  // LDS
  uint2* own;                 // [kCap] the listed tokens
  unsigned long long* hist;   // [1024]
  unsigned long long* hist2;  // [1024]
  unsigned long long* sums;   // [2][16]
  unsigned long long* sel;    // [4]
  uint32_t* ext;              // [16]

  __device__ double weight(uint32_t k) const {
    return exp2_neg((static_cast<double>(logit_of_key(k)) - static_cast<double>(plan.max)) * z.s);
  }
  __device__ int bin(uint32_t k) const { return bin_of(logit_of_key(k), z.s_bin, grid); }

  __device__ void fetch(int row) {
    if (!in_list) return;
    const uint2* const from = q.list + static_cast<int64_t>(row) * kCap;
    for (int i = tid; i < n; i += kFinish) own[i] = from[i];  // (each thread reads its own only)
  }

  // f(key, index, weight) for the tokens with keys lo .. hi (weight only if WEIGHT)
  template <bool WEIGHT, typename F>
  __device__ void each(uint32_t lo, uint32_t hi, F f) const {
    if (in_list) {
      for (int i = tid; i < n; i += kFinish) {
        const uint2 x = own[i];
        if (x.x >= lo && x.x <= hi) f(x.x, x.y, WEIGHT ? weight(x.x) : 0.0);
      }
    } else {
      for (int e = tid; e < q.V; e += kFinish) {
        const float l = Chunk<DT, 8>::value(base, e);
        const uint32_t k = key_of(l);
        if (k >= lo && k <= hi && l > -__builtin_huge_valf()) f(k, static_cast<uint32_t>(e), WEIGHT ? weight(k) : 0.0);
      }
    }
  }

  __device__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total) const {
    const uint64_t s = wave_scan(v, lane);
    if (lane == 63) part[wave] = s;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kFinish / 64; ++i) {
      const uint64_t x = part[i];
      if (i < wave) before += x;
      total += x;
    }
    return before + s;
  }

  // The least and largest key of a window's tokens; false: it has none.
  __device__ bool range(const Window& win, uint32_t& lo, uint32_t& hi) {
    if (win.b1 < win.b0) return false;
    if (tid == 0) ext[0] = kNone, ext[1] = 0;
    __syncthreads();
    uint32_t a = kNone, c = 0;
    each<false>(0, kNone, [&](uint32_t k, uint32_t, double) {
      const int j = bin(k);
      if (j >= win.b0 && j <= win.b1) a = min(a, k), c = max(c, k);
    });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      a = min(a, static_cast<uint32_t>(__shfl_xor(static_cast<int>(a), d, 64)));
      c = max(c, static_cast<uint32_t>(__shfl_xor(static_cast<int>(c), d, 64)));
    }
    if (lane == 0 && a != kNone) {
      atomicMin(&ext[0], a);
      atomicMax(&ext[1], c);
    }
    __syncthreads();
    lo = ext[0];
    hi = ext[1];
    __syncthreads();
    return lo <= hi;
  }

  __device__ bool reaches(float l) const { return (static_cast<double>(l) - static_cast<double>(plan.max)) * z.s >= z.f; }

  // The weights of a window's tokens, of keys lo .. hi, that reach min-p.
  __device__ double reaching(uint32_t lo, uint32_t hi, const Window& win) {
    const int octave = static_cast<int>((win.b0 > 0 ? win.b0 - 1 : 0) / kPerOctave);
    const double scale = __builtin_ldexp(1.0, octave + 43), unscale = __builtin_ldexp(1.0, -(octave + 43));
    if (tid == 0) sel[0] = 0;
    __syncthreads();
    uint64_t sum = 0;
    each<true>(lo, hi, [&](uint32_t k, uint32_t, double wt) {
      if (reaches(logit_of_key(k))) sum += whole(wt * scale);
    });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0 && sum) atomicAdd(&sel[0], static_cast<unsigned long long>(sum));
    __syncthreads();
    const double w = static_cast<double>(sel[0]) * unscale;
    __syncthreads();
    return w;
  }

  // Of the tokens with keys lo .. hi, in the order, the first at which `before` + the running sum reaches x
  // (strict: exceeds it) -- of the weights, or, by_count, of ones (before and x: numbers of them); the last if none
  // does.  `skip` is left out.  Whole numbers: 2^43 the largest weight of bin b0.
  __device__ Found select(uint32_t lo, uint32_t hi, int b0, bool by_count, bool strict, double before, double x, uint32_t skip,
                          double weights_before) {
    const int octave = static_cast<int>((b0 > 0 ? b0 - 1 : 0) / kPerOctave);
    const double scale = __builtin_ldexp(1.0, octave + 43), unscale = __builtin_ldexp(1.0, -(octave + 43));
    uint64_t need;
    {
      const double y = fmin(fmax((x - before) * (by_count ? 1.0 : scale), 0.0), 0x1p63);
      need = strict ? static_cast<uint64_t>(y) + 1 : static_cast<uint64_t>(__builtin_ceil(y));
      if (need == 0) need = 1;
    }
    uint64_t sum = 0, sum2 = 0;  // of what lies before the open range: the measure, and by_count the weights
    bool begin = true;
    while (true) {
      const uint32_t span = hi - lo;
      const int bits = span ? 32 - __builtin_clz(span) : 0, sh = bits > 10 ? bits - 10 : 0;
      hist[tid] = 0;
      if (by_count) hist2[tid] = 0;
      __syncthreads();
      each<true>(lo, hi, [&](uint32_t k, uint32_t i, double wt) {
        if (i == skip) return;
        const uint32_t at = (k - lo) >> sh;
        const unsigned long long m = whole(wt * scale);
        atomicAdd(&hist[at], by_count ? 1ull : m);
        if (by_count) atomicAdd(&hist2[at], m);
      });
      __syncthreads();
      const uint64_t v = hist[tid];
      uint64_t total, total2;
      const uint64_t incl = sum + block_scan(v, reinterpret_cast<uint64_t*>(sums), total);
      uint64_t incl2 = 0, v2 = 0;
      if (by_count) {
        v2 = hist2[tid];
        incl2 = sum2 + block_scan(v2, reinterpret_cast<uint64_t*>(sums) + 16, total2);
      }
      if (begin && need > total) need = total ? total : 1;
      if (tid == 0) sel[0] = 0, sel[1] = sum, sel[2] = sum2;
      __syncthreads();
      if (incl - v < need && need <= incl) sel[0] = tid, sel[1] = incl - v, sel[2] = incl2 - v2;
      __syncthreads();
      const uint32_t digit = static_cast<uint32_t>(sel[0]);
      sum = sel[1];
      sum2 = sel[2];
      begin = false;
      lo = lo + (digit << sh);
      if (sh == 0) break;
      const uint32_t top = lo + ((1u << sh) - 1u);
      hi = top < hi ? top : hi;
    }
    // equal logits: the one in question by its place among them
    if (tid == 0) ext[0] = kNone, ext[1] = 0, ext[2] = 0;
    __syncthreads();
    each<false>(lo, lo, [&](uint32_t, uint32_t i, double) {
      if (i == skip) return;
      atomicMin(&ext[0], i);
      atomicMax(&ext[1], i);
      atomicAdd(&ext[2], 1u);
    });
    __syncthreads();
    Found r;
    r.ik = lo;
    r.w = weight(lo);
    const uint64_t m = whole(r.w * scale);
    uint32_t i0 = ext[0], i1 = ext[1];
    const uint32_t ties = ext[2];
    uint64_t place = by_count ? need - sum : m ? (need - sum + m - 1) / m : 1;
    if (place > ties) place = ties;
    if (place < 1) place = 1;
    r.upto = (by_count ? weights_before : before) + static_cast<double>((by_count ? sum2 : sum) + place * m) * unscale;
    uint32_t rank = static_cast<uint32_t>(place);
    __syncthreads();
    if (rank == 1) i1 = i0;
    if (rank == ties) i0 = i1;
    uint64_t seen = 0;
    while (i0 < i1) {
      const uint32_t span = i1 - i0;
      const int bits = 32 - __builtin_clz(span), sh = bits > 10 ? bits - 10 : 0;
      hist[tid] = 0;
      if (tid == 0) sel[0] = 0, sel[1] = seen;
      __syncthreads();
      each<false>(lo, lo, [&](uint32_t, uint32_t i, double) {
        if (i != skip && i >= i0 && i <= i1) atomicAdd(&hist[(i - i0) >> sh], 1ull);
      });
      __syncthreads();
      const uint64_t v = hist[tid];
      uint64_t total;
      const uint64_t incl = seen + block_scan(v, reinterpret_cast<uint64_t*>(sums), total);
      if (incl - v < rank && rank <= incl) sel[0] = tid, sel[1] = incl - v;
      __syncthreads();
      i0 = i0 + (static_cast<uint32_t>(sel[0]) << sh);
      seen = sel[1];
      const uint32_t top = i0 + ((1u << sh) - 1u);
      i1 = top < i1 ? top : i1;
      __syncthreads();
    }
    r.idx = i0;
    return r;
  }
};

template <int DT>
__global__ void __launch_bounds__(kFinish) finish_kernel(const SamplingParams q) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ unsigned long long hist[1024], hist2[1024], sums[32], sel[4];
  __shared__ uint32_t ext[16];
  const int tid = threadIdx.x, row = blockIdx.x;
  int b = 0, end = 0;
  if (q.mode == kVerify && !sequence_of(q, row, tid & 63, b, end)) return;  // uniform
  const Plan plan = q.plans[row];
  const Settings z = settings(q, row);
  const uint8_t* const base = q.logits + row * q.stride;
  if (plan.max == -__builtin_huge_valf()) {  // uniform: no token
    if (tid == 0) {
      if (q.mode == kSample) q.token[row] = -1, q.logprob[row] = -__builtin_huge_valf();
      if (q.mode == kVerify) q.rowres[row] = Row{0.0, 0, 0, plan.max, 0, -1};
      if (q.mode == kBeams) q.nbest[row] = 0;
    }
    return;
  }
  const uint32_t listed = q.listed[row];
  Finish<DT> f{q, z, plan, base, __builtin_floor(static_cast<double>(plan.max) * z.s_bin), listed <= kCap, static_cast<int>(listed),
               tid, tid & 63, tid >> 6, reinterpret_cast<uint2*>(smem), hist, hist2, sums, sel, ext};
  f.fetch(row);
  // the last token of the order that top-k and top-p keep, and the weights of what is kept
  uint32_t ik = kNone, idx = kNone;
  double kept = plan.total;
  auto cut = [&](uint32_t k, uint32_t i) {
    if (k < ik || (k == ik && i < idx)) ik = k, idx = i;
  };
  uint32_t skip = kNone, token = kNone;
  double logprob = 0.0;
  bool accepted = false;
  // top-k's cut, top-p's and min-p's, then the token (one loop: the code is fetched once)
#pragma unroll 1
  for (int step = 0; step < 4; ++step) {
    const Window win = step == 0 ? plan.k : step == 1 ? plan.p : step == 2 ? plan.f : plan.d;
    double before = win.before, x = 0.0;
    if (step == 0) before = static_cast<double>(plan.count_before), x = static_cast<double>(z.k);
    if (step == 1) x = z.p * kept;
    if (step == 3) {
      const double u = z.first ? 0.0 : unit(q.mode == kSample ? q.u[row] : q.mode == kVerify ? q.draw[b] : 0.0f);
      double left = kept;
      const int64_t d = q.mode == kVerify && row + 1 < end ? q.tokens[row + 1] : -1;
      if (d >= 0 && d < q.V) {
        const float l = Chunk<DT, 8>::value(base, static_cast<int>(d));
        const uint32_t k = key_of(l);
        const int j = bin_of(l, z.s_bin, f.grid);
        if (j < kRest && f.reaches(l) && (k < ik || (k == ik && static_cast<uint32_t>(d) <= idx))) {
          const double wd = f.weight(k);
          const double sure = q.probs ? static_cast<double>(q.probs[row * q.probs_stride + d]) : 1.0;
          accepted = static_cast<double>(q.u[row]) * sure * kept < wd;
          if (!q.probs && kept - wd > 0.0) {
            skip = static_cast<uint32_t>(d);
            left = kept - wd;
            if (j < plan.d.b0) before -= wd;
          }
        }
      }
      x = u * left;
    }
    uint32_t lo, hi;
    const bool some = f.range(win, lo, hi);  // uniform
    if (step == 2 && win.b1 >= win.b0) kept = fmin(kept, win.before + (some ? f.reaching(lo, hi, win) : 0.0));
    if (!some || step == 2) continue;
    const Found c = f.select(lo, hi, win.b0, step == 0, step == 3, before, x, skip, plan.k.before);
    if (step < 3) {
      cut(c.ik, c.idx);
      kept = fmin(kept, c.upto);
    } else {
      token = c.idx;
      logprob = (static_cast<double>(logit_of_key(c.ik)) - static_cast<double>(plan.max)) * (z.s * kLn2D) - log(kept);
    }
  }
  if (q.mode == kBeams) {
    if (tid == 0) ext[4] = 0;
    __syncthreads();
    f.template each<false>(0, ik, [&](uint32_t k, uint32_t i, double) {
      if (k == ik && i > idx) return;
      const uint32_t at = atomicAdd(&ext[4], 1u);
      if (at < static_cast<uint32_t>(q.keep)) q.best[static_cast<int64_t>(row) * q.keep + at] = uint2{k, i};
    });
    __syncthreads();
    if (tid == 0) q.nbest[row] = ext[4] < static_cast<uint32_t>(q.keep) ? ext[4] : static_cast<uint32_t>(q.keep);
    return;
  }
  if (tid != 0) return;
  if (q.mode == kSample) {
    q.token[row] = token == kNone ? -1 : static_cast<int64_t>(token);
    q.logprob[row] = static_cast<float>(logprob);
  } else {
    q.rowres[row] = Row{kept, ik, idx, plan.max, accepted ? 1 : 0, static_cast<int32_t>(token)};
  }
}

// ---- verify: the sequences ------------------------------------------------------------------------

// The first refused token of each sequence; without the draft's probabilities, and where none is refused, the
// token of that row is the next.
__global__ void __launch_bounds__(256) verify_kernel(const SamplingParams q) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= q.B) return;
  auto clamp = [&](int64_t v, int lo) -> int { return v < lo ? lo : v > q.rows ? q.rows : static_cast<int>(v); };
  const int a = clamp(q.cu[b], 0), z = clamp(q.cu[b + 1], a);
  int i = a;
  while (i + 1 < z && q.rowres[i].accepted) ++i;
  q.accepted[b] = i - a;
  q.token[b] = z > a ? q.rowres[i].token : -1;
  if (q.probs) q.refused[b] = i + 1 < z ? i : -1;
}

// What the target has above the draft at token i, 2^52 a probability of 1.
template <int DT>
__device__ __forceinline__ uint64_t above(const SamplingParams& q, const Settings& z, const Row& r, int row, float l, int i) {
  const uint32_t k = key_of(l);
  const double t = (static_cast<double>(l) - static_cast<double>(r.max)) * z.s;
  if (!(l > -__builtin_huge_valf()) || t < z.f || k > r.ik || (k == r.ik && static_cast<uint32_t>(i) > r.idx)) return 0;
  const double d = exp2_neg(t) / r.kept - static_cast<double>(fmaxf(q.probs[row * q.probs_stride + i], 0.0f));
  return d > 0.0 ? static_cast<uint64_t>(d * 0x1p52) : 0;
}

template <int DT, int EPT>
__global__ void __launch_bounds__(256) rest_kernel(const SamplingParams q) {
  using C = Chunk<DT, EPT>;
  __shared__ unsigned long long sums[4];
  const int tid = threadIdx.x;
  const int b = blockIdx.x / q.chunks, chunk = blockIdx.x - b * q.chunks;
  const int row = q.refused[b];
  if (row < 0) return;
  const uint8_t* const base = q.logits + row * q.stride;
  const Settings z = settings(q, row);
  const Row r = q.rowres[row];
  const int mis = C::mis(base);
  float v[EPT];
  C::load(base, q.V, chunk, tid, mis, v);
  uint64_t s = 0;
#pragma unroll
  for (int i = 0; i < EPT; ++i)
    if (v[i] > -__builtin_huge_valf()) s += above<DT>(q, z, r, row, v[i], C::index(chunk, tid, i, mis));
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
  if ((tid & 63) == 0) sums[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) q.rest[static_cast<int64_t>(b) * q.chunks + chunk] = sums[0] + sums[1] + sums[2] + sums[3];
}

// The token of a refused row from what the target has above the draft, by rising index (where that is
// nothing it stays the one from the target itself).
template <int DT, int EPT>
__global__ void __launch_bounds__(256) redraw_kernel(const SamplingParams q) {
  using C = Chunk<DT, EPT>;
  __shared__ unsigned long long sums[4];
  __shared__ unsigned long long at_before[2];
  __shared__ int at_chunk;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const int row = q.refused[b];
  if (row < 0) return;
  const uint64_t* const rest = q.rest + static_cast<int64_t>(b) * q.chunks;
  uint64_t total = 0;
  for (int c = tid; c < q.chunks; c += 256) total += rest[c];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor(total, d, 64);
  if (lane == 0) sums[wave] = total;
  __syncthreads();
  total = sums[0] + sums[1] + sums[2] + sums[3];
  if (total == 0) return;  // uniform
  uint64_t need = static_cast<uint64_t>(unit(q.draw[b]) * static_cast<double>(total)) + 1;
  if (need > total) need = total;
  if (tid == 0) {
    uint64_t s = 0;
    int c = 0;
    while (c < q.chunks - 1 && s + rest[c] < need) s += rest[c++];
    at_chunk = c;
    at_before[0] = s;
  }
  __syncthreads();
  const int chunk = at_chunk;
  uint64_t sum = at_before[0];
  const uint8_t* const base = q.logits + row * q.stride;
  const Settings z = settings(q, row);
  const Row r = q.rowres[row];
  const int mis = C::mis(base);
  const int first = C::index(chunk, 0, 0, mis);
  for (int e0 = 0; e0 < 256 * EPT; e0 += 256) {
    const int i = first + e0 + tid;
    const uint64_t v = i >= 0 && i < q.V ? above<DT>(q, z, r, row, C::value(base, i), i) : 0;
    const uint64_t s = wave_scan(v, lane);
    __syncthreads();
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    uint64_t before = sum;
    for (int w = 0; w < wave; ++w) before += sums[w];
    if (before + s - v < need && need <= before + s) q.token[b] = i;
    sum += sums[0] + sums[1] + sums[2] + sums[3];
    if (sum >= need) break;  // uniform
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
        const Plan& plan = q.plans[row];
        v = static_cast<double>(score) + ((static_cast<double>(logit_of_key(x.x)) - static_cast<double>(plan.max)) - log(plan.total));
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

// Elements of a chunk's thread: 32, or 8 where chunks of 8192 would leave compute units idle.
int chunk_elements(int64_t rows, int64_t V) { return rows * ((V + 8191) / 8192) < 512 ? 8 : 32; }

// Chunks of a row, whatever its alignment: up to 7 elements of the first piece belong to no row.
int chunk_count(int64_t V, int per) { return static_cast<int>((V + 7 + 256 * per - 1) / (256 * per)); }

int64_t up(int64_t x) { return (x + 255) & ~static_cast<int64_t>(255); }

// The workspace's parts, in order; returns the bytes.
int64_t lay(SamplingParams& q, uint8_t* ws) {
  int64_t at = 0;
  auto take = [&](auto*& to, int64_t n) {
    to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(ws + at);
    at += up(n * static_cast<int64_t>(sizeof(*to)));
  };
  const int64_t r = q.rows, rc = r * q.chunks;
  take(q.heads, rc);
  take(q.hist, rc * kBins);
  if (q.count) take(q.counts, rc * kBins);
  take(q.plans, r);
  take(q.listed, r);
  take(q.list, r * kCap);
  if (q.mode == kVerify) {
    take(q.rowres, r);
    if (q.probs) {
      take(q.refused, q.B);
      take(q.rest, static_cast<int64_t>(q.B) * q.chunks);
    }
  }
  if (q.mode == kBeams) {
    take(q.best, r * q.keep);
    take(q.nbest, r);
  }
  return at;
}

constexpr int kFinishLds = kCap * static_cast<int>(sizeof(uint2));

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

template <int DT, int EPT>
int launch_as(const SamplingParams& q, hipStream_t s) {
  static std::atomic<bool> finish_set[kMaxDevices] = {};
  if (!raise_lds(finish_kernel<DT>, kFinishLds, finish_set)) return MZK_ELAUNCH;
  const unsigned grid = static_cast<unsigned>(q.rows) * static_cast<unsigned>(q.chunks);
  survey_kernel<DT, EPT><<<grid, 256, 0, s>>>(q);
  narrow_kernel<DT, EPT><<<grid, 256, 0, s>>>(q);
  finish_kernel<DT><<<static_cast<unsigned>(q.rows), kFinish, kFinishLds, s>>>(q);
  if (q.mode == kVerify) {
    verify_kernel<<<static_cast<unsigned>((q.B + 255) / 256), 256, 0, s>>>(q);
    if (q.probs) {
      rest_kernel<DT, EPT><<<static_cast<unsigned>(q.B) * static_cast<unsigned>(q.chunks), 256, 0, s>>>(q);
      redraw_kernel<DT, EPT><<<static_cast<unsigned>(q.B), 256, 0, s>>>(q);
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

template <int DT>
int launch(const SamplingParams& q, hipStream_t s) {
  return chunk_elements(q.rows, q.V) == 8 ? launch_as<DT, 8>(q, s) : launch_as<DT, 32>(q, s);
}

int size_of(int dtype) { return dtype == MZK_F32 ? 4 : 2; }

// What every call checks of its rows, and the parts of the parameters that follow from them.
int rows_of(SamplingParams& q, const char* name, int64_t rows, int64_t V, int dtype) {
  MZK_CHECK_ARG(dtype >= MZK_F32 && dtype <= MZK_F16, "%s: unsupported dtype %d", name, dtype);
  MZK_CHECK_ARG(rows >= 0 && V >= 1, "%s: bad sizes", name);
  MZK_CHECK_ARG(V <= kMaxVocab, "%s: at most %lld logits a row, got %lld", name, (long long)kMaxVocab, (long long)V);
  const int per = chunk_elements(rows, V);
  q.V = static_cast<int>(V);
  q.chunks = chunk_count(V, per);
  q.scale = 62;
  while ((static_cast<int64_t>(1) << (62 - q.scale)) < V) --q.scale;
  // a launch has less than 2^32 threads
  MZK_CHECK_ARG(rows < (1 << 22) && rows * q.chunks < (1 << 24), "%s: too many rows: %lld of %lld logits", name, (long long)rows, (long long)V);
  q.rows = static_cast<int>(rows);
  return MZK_OK;
}

int run(SamplingParams& q, const char* name, const void* logits, int64_t stride, int dtype, void* workspace, int64_t workspace_bytes,
        void* stream) {
  MZK_CHECK_ARG(logits && workspace, "%s: null pointer", name);
  MZK_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % size_of(dtype) == 0 && aligned16(workspace), "%s: misaligned logits or workspace", name);
  MZK_CHECK_ARG(stride >= q.V || q.rows <= 1, "%s: rows of logits overlap", name);
  q.logits = static_cast<const uint8_t*>(logits);
  q.stride = stride * size_of(dtype);
  const int64_t need = lay(q, static_cast<uint8_t*>(workspace));
  MZK_CHECK_ARG(workspace_bytes >= need, "%s: workspace needs %lld bytes", name, (long long)need);
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
  q.count = 1;
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
  q.count = top_k || top_k_all > 0;
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
  q.count = 1;
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
  MZK_CHECK_ARG(B >= 0 && B < 1 << 22 && B * q.chunks < 1 << 24, "verify: bad sizes");
  if (B == 0) return MZK_OK;
  MZK_CHECK_ARG(cu && accepted && next && draw && (T == 0 || (tokens && u)), "verify: null pointer");
  MZK_CHECK_ARG(!draft_probs || draft_row_stride >= V || T <= 1, "verify: rows of the draft's probabilities overlap");
  q.temperature = Filter{temperature, temperature_all};
  q.top_p = Filter{top_p, top_p_all};
  q.min_p = Filter{min_p, min_p_all};
  q.top_k = top_k;
  q.top_k_all = top_k_all;
  q.count = top_k || top_k_all > 0;
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
    verify_kernel<<<static_cast<unsigned>((B + 255) / 256), 256, 0, as_stream(stream)>>>(q);
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
  q.count = 1;
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
  q.count = 1;
  q.scores = scores;
  q.width = width;
  q.keep = keep;
  q.parents = parents;
  q.token = tokens;
  q.out_scores = out_scores;
  return run(q, "beams", logits, row_stride, dtype, workspace, workspace_bytes, stream);
}
