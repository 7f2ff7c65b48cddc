// Shared-latent attention over sequences of different lengths: one new token or a few of each over its
// pages (paged_attend), or whole packed prompts, causal (packed_mqa).
//
//   o[t, h] = sum_j p_j e_j,  p = softmax over the entries j that token t sees of q[t, h] . e_j D^-1/2,
//   the head's sink one more term of the denominator; lse its logarithm.  K == V == e.
//   Token i of the n new ones of a sequence with len tokens is at position len - n + i and sees
//   positions 0 .. its own, the last `window` of them, or the positions of its list.
//
// A unit of work is a block of 64 rows -- a row is a head of a token, the heads of one latent
// innermost, so 64 rows are 64 heads of a token or all heads of several -- over a share of the
// sequence's entries.
#include "common.h"
#include "entries.h"

namespace mzk {
namespace {

constexpr int64_t kNoWindow = 1ll << 62;

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
  int64_t table_stride, max_pages, pages;
  int page;
  const int32_t* idx;  // [B, topk] positions (one token per sequence), or null
  int64_t idx_stride;
  int topk;
  int64_t window;
  const float* sinks;
  float scale_log2;
  int rows_per_unit;   // min(64, 32 HG): a unit spans at most 33 tokens
  int64_t blocks_max;  // units in the grid
  uint16_t* out;
  float* lse;          // [T, H]
  int zero_tail;       // rows of no sequence become 0 (else they are left as they are)
};

// Where a unit's rows are.
struct Unit {
  int64_t b, t0, n;     // sequence, its first packed token, its new tokens
  int64_t len;          // its tokens in the cache
  int g;                // latent
  int64_t r0, r1;       // rows of the sequence and latent: token r / HG, head g HG + r % HG
};

template <int FMT, int D, int NOPE>
struct RaggedLds {
  static constexpr int PITCH = 2 * D + 16;
  static constexpr int PB = kTile * PITCH;
  static constexpr int PMAX = PB + 4096;  // [2][64]
  static constexpr int LSUM = PMAX + 512;
  static constexpr int OKS = LSUM + 512;  // [32] words
  static constexpr int SCAN = OKS + 128;  // [8] int64
  static constexpr int LDS = SCAN + 128;
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// The sequence and row block of unit k, by a scan over the sequences' blocks; false: none.
__device__ bool find_unit(const RaggedParams& p, int64_t k, Unit& u, int64_t* scan, int tid) {
  int64_t blk, per;
  if (p.cu == nullptr) {
    per = (p.HG + p.rows_per_unit - 1) / p.rows_per_unit * static_cast<int64_t>(p.G);
    u.b = k / per;
    if (u.b >= p.B) return false;
    blk = k - u.b * per;
    u.t0 = u.b;
    u.n = 1;
  } else {
    int64_t base = 0;
    bool found = false;
    for (int64_t i = 0; i < p.B && !found; i += 256) {
      int64_t v = 0, a = 0, z = 0;
      if (i + tid < p.B) {
        a = clamp64(p.cu[i + tid], 0, p.T);
        z = clamp64(p.cu[i + tid + 1], a, p.T);
        v = ((z - a) * p.HG + p.rows_per_unit - 1) / p.rows_per_unit * p.G;
      }
      int64_t x = v;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(x, d, 64);
        if ((tid & 63) >= d) x += y;
      }
      if ((tid & 63) == 63) scan[tid >> 6] = x;
      __syncthreads();
      int64_t before = base + x - v, total = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (w < (tid >> 6)) before += scan[w];
        total += scan[w];
      }
      if (v > 0 && k >= before && k < before + v) {
        scan[4] = i + tid;
        scan[5] = k - before;
        scan[6] = a;
        scan[7] = z - a;
      }
      found = k < base + total;
      base += total;
      __syncthreads();
    }
    if (!found) return false;
    u.b = scan[4];
    blk = scan[5];
    u.t0 = scan[6];
    u.n = scan[7];
    per = (u.n * p.HG + p.rows_per_unit - 1) / p.rows_per_unit * p.G;
  }
  const int64_t per_latent = per / p.G;
  u.g = static_cast<int>(blk / per_latent);
  u.r0 = (blk - u.g * per_latent) * p.rows_per_unit;
  const int64_t rows = u.n * p.HG;
  u.r1 = u.r0 + p.rows_per_unit < rows ? u.r0 + p.rows_per_unit : rows;
  u.len = u.n;
  if (p.lens) u.len = clamp64(p.lens[u.b], 0, p.max_pages * p.page);
  return true;
}

// The address of the entry at position v of the unit's sequence (or of its list); null where there is none.
__device__ __forceinline__ const uint8_t* entry_of(const RaggedParams& p, const Unit& u, int64_t v, int entry_bytes) {
  if (p.tables == nullptr) return p.entries + (u.t0 + v) * p.entry_stride + static_cast<int64_t>(u.g) * entry_bytes;
  if (p.idx) {
    v = p.idx[u.b * p.idx_stride + v];
    if (v < 0 || v >= u.len) return nullptr;
  }
  const int64_t pid = p.tables[u.b * p.table_stride + v / p.page];
  if (pid < 0 || pid >= p.pages) return nullptr;
  return p.entries + (pid * p.page + v % p.page) * p.entry_stride;
}

// A tile of 32 entries at a time: bf16 rows in LDS, S^T by matrix instructions (each wave 16 entries x
// 32 rows), the softmax's running maximum, P^T through LDS, O^T by matrix instructions (each wave
// every fourth block of 16 channels x 64 rows).  Entries that are not there are rows of zeros.
template <int FMT, int D, int NOPE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
ragged_kernel(const RaggedParams p) {
  using M = RaggedLds<FMT, D, NOPE>;
  using L = Layout<FMT, D, NOPE>;
  constexpr int KS = D / 32, NB = D / 16, NI = (NB + 3) / 4;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* const pbuf = smem + M::PB;
  float* const pmax = reinterpret_cast<float*>(smem + M::PMAX);
  float* const lsum = reinterpret_cast<float*>(smem + M::LSUM);
  int* const oks = reinterpret_cast<int*>(smem + M::OKS);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int eh = wave & 1, hh = wave >> 1, g = lane >> 4, e16 = lane & 15;

  Unit u;
  if (!find_unit(p, blockIdx.x, u, reinterpret_cast<int64_t*>(smem + M::SCAN), tid)) return;  // uniform

  // the B operand of S^T: rows 32 hh + 16 b + e16, channels 32 st + 8 g ..
  v8bf qf[KS][2];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int64_t r = u.r0 + 32 * hh + 16 * b + e16;
    const int64_t rc = r < u.r1 ? r : u.r0;
    const uint16_t* qr = p.q + ((u.t0 + rc / p.HG) * p.H + u.g * p.HG + rc % p.HG) * D;
#pragma unroll
    for (int st = 0; st < KS; ++st)
      qf[st][b] = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(qr + 32 * st + 8 * g));
  }

  const int64_t tok0 = u.r0 / p.HG, tok1 = (u.r1 - 1) / p.HG + 1;
  const int64_t shift = u.len - u.n;  // position of the sequence's first new token (negative: tokens that see nothing)
  // one pass over all rows; if something in it is not finite, one pass for each token over what it sees
  // itself, since a weight of 0 times an entry hidden from a row would not be 0
  int64_t sub0 = tok0, sub1 = tok1;
  bool strict = false;
  while (true) {
    int64_t lo = clamp64(shift + sub0 - p.window + 1, 0, u.len), hi = clamp64(shift + sub1, 0, u.len);
    if (p.idx) { lo = 0; hi = u.len > 0 ? p.topk : 0; }
    int64_t row_lo[2], row_hi[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t r = u.r0 + 32 * hh + 16 * b + e16;
      const int64_t pos = shift + (r < u.r1 ? r : u.r0) / p.HG;
      row_lo[b] = p.idx ? 0 : pos - p.window + 1;
      row_hi[b] = p.idx ? hi : pos + 1;
    }
    float m_own[2] = {-__builtin_huge_valf(), -__builtin_huge_valf()}, l_own[2] = {0.0f, 0.0f};
    float m4[4];
    v4f acc[NI][4];
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      m4[hg] = -__builtin_huge_valf();
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i][hg] = v4f{};
    }
    const int te = tid >> 3, tj = tid & 7;
    for (int64_t v0 = lo; v0 < hi; v0 += kTile) {
      const uint8_t* const e = v0 + te < hi ? entry_of(p, u, v0 + te, L::kEntryBytes) : nullptr;
      for (int q = tj; q < L::kPieces; q += 8) {
        if (e) {
          store_piece<FMT, D, NOPE>(smem + te * M::PITCH, fetch_piece<FMT, D, NOPE>((gptr_t)e, q), q);
        } else {
          Piece z{};
          store_piece<FMT, D, NOPE>(smem + te * M::PITCH, z, q);
        }
      }
      if (tj == 0) oks[te] = e != nullptr;
      __syncthreads();
      v4f s[2] = {v4f{}, v4f{}};
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const v8bf kf = __builtin_bit_cast(
            v8bf, *reinterpret_cast<const v4i*>(smem + (16 * eh + e16) * M::PITCH + 64 * st + 16 * g));
        s[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[st][0], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[st][1], s[1], 0, 0, 0);
      }
      float v[2][4], t[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        t[b] = -__builtin_huge_valf();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = 16 * eh + 4 * g + r;
          const bool in = oks[at] != 0 && v0 + at >= row_lo[b] && v0 + at < row_hi[b];
          v[b][r] = in ? s[b][r] * p.scale_log2 : -__builtin_huge_valf();
          t[b] = fmaxf(t[b], v[b][r]);
        }
        t[b] = fmaxf(t[b], __shfl_xor(t[b], 16, 64));
        t[b] = fmaxf(t[b], __shfl_xor(t[b], 32, 64));
        if (g == 0) pmax[eh * 64 + 32 * hh + 16 * b + e16] = t[b];
      }
      __syncthreads();
#pragma unroll
      for (int hg = 0; hg < 4; ++hg) {
        const float mn = fmaxf(m4[hg], fmaxf(pmax[16 * hg + e16], pmax[64 + 16 * hg + e16]));
        const float a = m4[hg] == -__builtin_huge_valf() ? 0.0f : exp2f(m4[hg] - mn);
        m4[hg] = mn;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][hg][r] *= a;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int row = 32 * hh + 16 * b + e16;
        const float mn = fmaxf(m_own[b], fmaxf(pmax[row], pmax[64 + row]));
        const float a = m_own[b] == -__builtin_huge_valf() ? 0.0f : exp2f(m_own[b] - mn);
        m_own[b] = mn;
        const float ref = mn == -__builtin_huge_valf() ? 0.0f : mn;
        float w[4], sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[r] = exp2f(v[b][r] - ref);
          sum += w[r];
        }
        l_own[b] = l_own[b] * a + sum;
        *reinterpret_cast<uint2*>(pbuf + 2048 * hh + 1024 * b + 16 * lane + 8 * eh) =
            uint2{pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])};
      }
      __syncthreads();
#pragma unroll
      for (int hg = 0; hg < 4; ++hg) {
        const v8bf pf = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(pbuf + 1024 * hg + 16 * lane));
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          if (wave + 4 * i < NB) {
            const uint8_t* tp = smem + (4 * g + (e16 >> 2)) * M::PITCH + 32 * (wave + 4 * i) + 8 * (e16 & 3);
            const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_v4s(tp));
            const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_v4s(tp + 16 * M::PITCH));
            const v8bf vf = __builtin_bit_cast(v8bf, v8s{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
            acc[i][hg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, acc[i][hg], 0, 0, 0);
          }
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      l_own[b] += __shfl_xor(l_own[b], 16, 64);
      l_own[b] += __shfl_xor(l_own[b], 32, 64);
      if (g == 0) lsum[eh * 64 + 32 * hh + 16 * b + e16] = l_own[b];
    }
    if (tid == 0) oks[0] = 0;
    __syncthreads();
    float l4[4];
    float bad = 0.0f;
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      l4[hg] = lsum[16 * hg + e16] + lsum[64 + 16 * hg + e16];
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) bad = __builtin_fmaf(acc[i][hg][r], 0.0f, bad);
    }
    if (!strict && tok1 - tok0 > 1) {
      if (bad != 0.0f) oks[0] = 1;
      __syncthreads();
      if (oks[0]) {  // uniform
        strict = true;
        sub0 = tok0;
        sub1 = tok0 + 1;
        __syncthreads();
        continue;
      }
    }
#pragma unroll
    for (int hg = 0; hg < 4; ++hg) {
      const int64_t r = u.r0 + 16 * hg + e16;
      const int64_t tok = r / p.HG;
      if (r >= u.r1 || tok < sub0 || tok >= sub1) continue;
      const int head = u.g * p.HG + static_cast<int>(r - tok * p.HG);
      float m = m4[hg], l = l4[hg], scale = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      const bool none = l == 0.0f && m == -__builtin_huge_valf();  // it sees nothing: lse is the sink itself
      if (p.sinks) {
        const float sk = p.sinks[head] * kLog2e;
        const float mm = fmaxf(m, sk);
        if (mm > -__builtin_huge_valf()) {
          const float a = m == -__builtin_huge_valf() ? 0.0f : exp2f(m - mm);
          l = l * a + exp2f(sk - mm);
          m = mm;
          scale = a / l;
        }
      }
      uint16_t* const o = p.out + ((u.t0 + tok) * p.H + head) * D;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int c = 16 * (wave + 4 * i) + 4 * g;
        if (wave + 4 * i < NB)
          *reinterpret_cast<uint2*>(o + c) = uint2{pack_bf16x2(acc[i][hg][0] * scale, acc[i][hg][1] * scale),
                                                   pack_bf16x2(acc[i][hg][2] * scale, acc[i][hg][3] * scale)};
      }
      if (wave == hg && g == 0)
        p.lse[(u.t0 + tok) * p.H + head] = !none      ? (m + __log2f(l)) * kLn2
                                           : p.sinks ? p.sinks[head]
                                                     : -__builtin_huge_valf();
    }
    if (!strict || sub1 >= tok1) break;
    ++sub0;
    ++sub1;
    __syncthreads();
  }
}

// Rows behind the last sequence: 0, and a log-sum-exp of -inf.
__global__ void __launch_bounds__(256) ragged_tail_kernel(const RaggedParams p) {
  const int64_t end = clamp64(p.cu[p.B], 0, p.T);
  const int64_t rows = (p.T - end) * p.H;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  uint32_t* const o = reinterpret_cast<uint32_t*>(p.out + end * p.H * p.D);
  for (int64_t i = at; i < rows * (p.D / 2); i += step) o[i] = 0;
  for (int64_t i = at; i < rows; i += step) p.lse[end * p.H + i] = -__builtin_huge_valf();
}

template <int FMT, int D, int NOPE>
int launch_ragged(const RaggedParams& p, hipStream_t s) {
  using M = RaggedLds<FMT, D, NOPE>;
  ragged_kernel<FMT, D, NOPE><<<static_cast<unsigned>(p.blocks_max), 256, M::LDS, s>>>(p);
  if (p.zero_tail && p.cu) ragged_tail_kernel<<<256, 256, 0, s>>>(p);
  MZK_LAUNCH_CHECK("ragged attention");
  return MZK_OK;
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

// Units of rows_per_unit rows in the grid: at most this many, whatever the lengths are.
int64_t unit_bound(const RaggedParams& p) {
  const int64_t per = (static_cast<int64_t>(p.HG) + p.rows_per_unit - 1) / p.rows_per_unit;
  return p.cu == nullptr ? p.B * p.G * per : (p.T * p.HG / p.rows_per_unit + (p.B < p.T ? p.B : p.T)) * p.G;
}

constexpr int64_t kMaxInt = 0x7fffffff;

}  // namespace
}  // namespace mzk

using namespace mzk;

extern "C" int mzk_paged_attend(const void* q, int64_t T, int H, int D, const int64_t* cu, int64_t B, int fmt, int nope,
                                const void* pool, int64_t pages, int page, const int32_t* tables, int64_t table_stride,
                                int64_t max_pages, const int64_t* lens, const int32_t* idx, int64_t idx_row_stride,
                                int topk, int64_t window, const float* sinks, void* workspace, int64_t workspace_bytes,
                                void* out, float* lse, int zero_tail, void* stream) {
  MZK_CHECK_ARG(T >= 0 && B >= 0 && H >= 1 && D > 0, "paged_attend: bad sizes");
  MZK_CHECK_ARG(T <= kMaxInt && B <= kMaxInt && H <= 65536 && pages >= 0 && pages <= kMaxInt && max_pages >= 0 &&
                    max_pages <= kMaxInt,
                "paged_attend: sizes of 2^31 or more");
  MZK_CHECK_ARG(page >= 1, "paged_attend: pages of at least one entry");
  MZK_CHECK_ARG(fmt == 0 || fmt == 1, "paged_attend: fmt must be 0 (bf16) or 1 (fp8-b128)");
  MZK_CHECK_ARG(window >= 0 && topk >= 0, "paged_attend: negative window or list");
  MZK_CHECK_ARG(cu || T == B, "paged_attend: without cu one token per sequence (%lld tokens, %lld sequences)",
                (long long)T, (long long)B);
  MZK_CHECK_ARG(!idx || (cu == nullptr && window == 0 && idx_row_stride >= topk),
                "paged_attend: a list of entries takes one token per sequence and no window, rows of at least topk");
  MZK_CHECK_ARG(table_stride >= max_pages, "paged_attend: table rows shorter than max_pages");
  if (T == 0 || B == 0) return MZK_OK;
  MZK_CHECK_ARG(q && pool && tables && lens && out && lse, "paged_attend: null pointer");
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
  p.tables = tables;
  p.table_stride = table_stride;
  p.max_pages = max_pages;
  p.pages = pages;
  p.page = page;
  p.idx = idx;
  p.idx_stride = idx_row_stride;
  p.topk = topk;
  p.window = window ? window : kNoWindow;
  p.sinks = sinks;
  p.scale_log2 = (1.0f / __builtin_sqrtf(static_cast<float>(D))) * kLog2e;
  p.rows_per_unit = 32 * p.HG < 64 ? 32 * p.HG : 64;
  p.blocks_max = unit_bound(p);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.zero_tail = zero_tail;
  MZK_CHECK_ARG(p.blocks_max <= kMaxInt, "paged_attend: too many rows");
  return dispatch_ragged("paged_attend", fmt, nope, p, as_stream(stream));
}

extern "C" int mzk_paged_attend_workspace_bytes(int64_t T, int H, int D, int packed, int64_t B, int64_t* bytes) {
  MZK_CHECK_ARG(bytes != nullptr, "paged_attend_workspace_bytes: null output");
  MZK_CHECK_ARG(T >= 0 && B >= 0 && H >= 1 && D > 0, "paged_attend_workspace_bytes: bad sizes");
  (void)packed;
  *bytes = 0;
  return MZK_OK;
}

extern "C" int mzk_packed_mqa(const void* q, int64_t T, int H, int D, const int64_t* cu, int64_t B, const void* kv,
                              int64_t kv_row_stride, int G, int64_t window, const float* sinks, void* out, float* lse,
                              int zero_tail, void* stream) {
  MZK_CHECK_ARG(T >= 0 && B >= 0 && H >= 1 && D > 0 && G >= 1, "packed_mqa: bad sizes");
  MZK_CHECK_ARG(T <= kMaxInt && B <= kMaxInt && H <= 65536, "packed_mqa: sizes of 2^31 or more");
  MZK_CHECK_ARG(H % G == 0, "packed_mqa: %d heads do not divide into %d latents", H, G);
  MZK_CHECK_ARG(window >= 0, "packed_mqa: negative window");
  MZK_CHECK_ARG(kv_row_stride >= static_cast<int64_t>(G) * D && kv_row_stride % 8 == 0,
                "packed_mqa: kv rows must be G * D apart or more, a multiple of 8 elements");
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
  p.window = window ? window : kNoWindow;
  p.sinks = sinks;
  p.scale_log2 = (1.0f / __builtin_sqrtf(static_cast<float>(D))) * kLog2e;
  p.rows_per_unit = 32 * p.HG < 64 ? 32 * p.HG : 64;
  p.blocks_max = unit_bound(p);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.zero_tail = zero_tail;
  MZK_CHECK_ARG(p.blocks_max <= kMaxInt, "packed_mqa: too many rows");
  return dispatch_ragged("packed_mqa", kFmtBf16, D, p, as_stream(stream));
}
