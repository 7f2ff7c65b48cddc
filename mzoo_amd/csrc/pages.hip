// The paged latent cache: entries of new tokens into pages, and the pages themselves.
//
// A pool is [P, page, entry bytes]; a sequence's table row names its pages in order (-1: none), and
// its first `len` entries hold its tokens.  refs[p] counts the table entries that name page p (and
// whatever else holds it); a page of refs 0 is free.  All of it lives on the device, so a captured
// decode loop grows its sequences without the host.
//
//   append   token i of the n new ones of sequence b -> position len_b - n + i
//   grow     pages for n_b more tokens each: those that a row holds behind its tokens and nobody else
//            does, then the lowest free pages, in the order of the sequences; a partly filled last
//            page that others hold too is replaced by a copy; all or none
//   fork     sequence i goes on from the tokens of sequence parents[i]
//   compact  of U used pages, the k-th behind page U moves to the k-th free one before it
//
// Results do not depend on the order of workgroups: pages are ranked by prefix sums, and the only
// atomics add whole numbers.
#include "common.h"

namespace mzk {
namespace {

constexpr int kChunk = 4096;  // pages that one workgroup ranks, 16 a thread

__device__ __forceinline__ int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- append -------------------------------------------------------------------------------

struct AppendParams {
  const void* x;
  int64_t x_stride, T;
  const int64_t* cu;  // null: one token per sequence
  int64_t B;
  const int32_t* tables;
  int64_t table_stride, max_pages;
  const int64_t* lens;
  uint8_t* pool;
  int64_t P;
  int page, D, nope;  // nope 0: bf16 entries
};

// The sequence of packed token t (B: none), counted by the wave: lane l looks at boundaries l, l + 64, ..
__device__ __forceinline__ int64_t sequence_of(const int64_t* cu, int64_t B, int64_t t, int lane) {
  int64_t n = 0;
  for (int64_t i = 0; i <= B; i += 64) {
    const bool before = i + lane <= B && cu[i + lane] <= t;
    n += __builtin_popcountll(__ballot(before));
  }
  return n - 1;  // -1 or B: the token is in no sequence
}

typedef uint32_t u32x2a4 __attribute__((ext_vector_type(2), aligned(4)));  // entries of 128 + 32 channels are 196 bytes

// One wave per token.  fp8: a lane quantizes 8 neighbouring channels, 16 lanes share a block of 128.
// The row of x is requested before the chain boundaries -> length -> page that ends in its entry's
// address.  64 tokens, one each: 4.7 us, that chain.  12 prompts of 12097 tokens in all, bf16 to
// 8-bit: 11.2 us, 2.0 TB/s, a round and a half of it over the compute units.
template <int DT>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p, bool vec) {
  const int lane = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (t >= p.T) return;
  const int64_t x0 = t * p.x_stride;
  float v[8];
  auto load = [&](int c) {
    float h[4];
    load4_as_f32<DT>(p.x, x0 + c, vec, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = h[i];
    load4_as_f32<DT>(p.x, x0 + c + 4, vec, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 + i] = h[i];
  };
  if (8 * lane < p.D) load(8 * lane);
  int64_t b = t, pos;
  if (p.cu) {
    b = sequence_of(p.cu, p.B, t, lane);
    if (b < 0 || b >= p.B) return;
    pos = p.lens[b] - p.cu[b + 1] + t;
  } else {
    pos = p.lens[b] - 1;
  }
  if (pos < 0 || pos >= p.max_pages * p.page) return;
  const int64_t pid = p.tables[b * p.table_stride + pos / p.page];
  if (pid < 0 || pid >= p.P) return;
  const int eb = p.nope ? p.nope + p.nope / 32 + 2 * (p.D - p.nope) : 2 * p.D;
  uint8_t* const e = p.pool + (pid * p.page + pos % p.page) * eb;
  for (int c = 8 * lane; c < p.D; c += 512) {
    if (c >= 512) load(c);
    if (c < p.nope) {  // nope is a multiple of 128: 16 lanes are in or out together
      const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
      const float s = fp8_scale_from_amax(group_max(nn_max(abs_max4(lo), abs_max4(hi)), 16));
      const float inv = s <= 0x1p120f ? pow2_reciprocal(s) : 1.0f / s;  // as the block quantizer
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = clampf(v[i] * inv, 448.0f);
      int w[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k], v[4 * k + 1], 0, false);
        w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2], v[4 * k + 3], w[k], true);
      }
      *reinterpret_cast<u32x2a4*>(e + c) = u32x2a4{static_cast<uint32_t>(w[0]), static_cast<uint32_t>(w[1])};
      if ((c & 127) == 0) *reinterpret_cast<float*>(e + p.nope + c / 32) = s;
    } else {
      uint8_t* const at = e + (p.nope ? p.nope + p.nope / 32 : 0) + 2 * (c - p.nope);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        *reinterpret_cast<u32x2a4*>(at + 8 * k) =
            u32x2a4{f32_to_bf16(v[4 * k]) | static_cast<uint32_t>(f32_to_bf16(v[4 * k + 1])) << 16,
                    f32_to_bf16(v[4 * k + 2]) | static_cast<uint32_t>(f32_to_bf16(v[4 * k + 3])) << 16};
    }
  }
}

template <int DT>
void launch_append(const AppendParams& p, bool vec, hipStream_t s) {
  append_kernel<DT><<<static_cast<unsigned>((p.T + 3) / 4), 256, 0, s>>>(p, vec);
}

// ---- prefix sums over a workgroup of 256 ----------------------------------------------------

// Sum over the workgroup of every thread's v, and of those before this one.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& before, int64_t* lds4, int tid) {
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(x, d, 64);
    if ((tid & 63) >= d) x += y;
  }
  if ((tid & 63) == 63) lds4[tid >> 6] = x;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < (tid >> 6)) base += lds4[w];
    total += lds4[w];
  }
  __syncthreads();
  before = base + x - v;
  return total;
}

// This thread's 16 pages of a chunk: their counts (-1 past the last page: neither free nor used).
__device__ __forceinline__ void load_refs(const int32_t* refs, int64_t P, int64_t first, int32_t (&r)[16]) {
  if (first + 16 <= P && (reinterpret_cast<uintptr_t>(refs) & 15u) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int4 v = reinterpret_cast<const int4*>(refs + first)[i];
      r[4 * i] = v.x; r[4 * i + 1] = v.y; r[4 * i + 2] = v.z; r[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = first + i < P ? refs[first + i] : -1;
  }
}

__device__ __forceinline__ void store_refs(int32_t* refs, int64_t P, int64_t first, const int32_t (&r)[16]) {
  if (first + 16 <= P && (reinterpret_cast<uintptr_t>(refs) & 15u) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<int4*>(refs + first)[i] = int4{r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]};
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (first + i < P) refs[first + i] = r[i];
  }
}

// Bit i is set where page i of these is free (used).
__device__ __forceinline__ uint32_t page_bits(const int32_t (&r)[16], bool used) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m |= static_cast<uint32_t>(used ? r[i] > 0 : r[i] == 0) << i;
  return m;
}

// The sum of v[0 .. n - 1] by a workgroup, and of its first m.
template <typename T>
__device__ __forceinline__ int64_t sum_of(const T* v, int64_t step, int64_t n, int64_t m, int64_t& head, int64_t* lds, int tid) {
  int64_t all = 0, first = 0, unused;
  for (int64_t i = tid; i < n; i += 256) {
    const int64_t x = v[i * step];
    all += x;
    first += i < m ? x : 0;
  }
  head = block_scan(first, unused, lds, tid);
  return block_scan(all, unused, lds, tid);
}

// ---- grow ---------------------------------------------------------------------------------

struct GrowRow {
  int32_t first, end, want;  // want of the table entries first .. end - 1 get a fresh page
  int32_t src, fill;         // the page whose first `fill` entries the first fresh page begins with (-1: none)
  int32_t base;              // -1: all of them do; else they are told by kept[], whose first bit is entry `base`
};

struct GrowParams {
  const int32_t* tables;
  int32_t* tables_out;
  int64_t stride, stride_out, B, max_pages;
  const int64_t* lens;
  int64_t* lens_out;
  const int32_t* refs;
  int32_t* refs_out;
  int64_t P;
  const int64_t* tokens;
  int page;
  int64_t* missing;
  // workspace
  GrowRow* rows;    // [B]
  int64_t* old_len; // [B]
  int64_t* over;    // [B] pages past the table's width
  int64_t* free_in; // [chunks] free pages of the chunk
  int64_t* want;    // [1] the pages handed out, -1: none, some lack
  uint64_t* kept;   // [B][words] entries behind the row's tokens whose pages it alone holds: they stay
  uint64_t* given;  // [B][words] entries whose pages others hold too: they get fresh ones, and count one less
  int32_t* list;    // [P] the page of each rank
  int64_t chunks, words;
};

constexpr int64_t kMostOver = 1ll << 38;  // of a row's pages past its table: 2^24 rows stay below 2^63

// A count from the device, within what sums of two cannot overflow.
__device__ __forceinline__ int64_t row_count(int64_t n) { return n < 0 ? 0 : n < (1ll << 60) ? n : 1ll << 60; }

__global__ void __launch_bounds__(256) grow_count_kernel(const GrowParams p) {
  __shared__ int64_t lds[4];
  const int tid = threadIdx.x;
  const int64_t blk = blockIdx.x;
  if (blk < p.chunks) {
    int64_t before;
    int32_t r[16];
    load_refs(p.refs, p.P, blk * kChunk + 16 * tid, r);
    const int64_t total = block_scan(__builtin_popcount(page_bits(r, false)), before, lds, tid);
    if (tid == 0) p.free_in[blk] = total;
    return;
  }
  // A wave per row, a lane per entry.  After refused tokens a row names pages behind the ones that
  // its tokens fill; written over, they would be nobody's and never free again.
  const int64_t b = (blk - p.chunks) * 4 + (tid >> 6);
  const int lane = tid & 63;
  if (b >= p.B) return;
  const int64_t len = row_count(p.lens[b]), n = row_count(p.tokens[b]);
  const int64_t held = ceil_div64(len, p.page), end = ceil_div64(len + n, p.page);
  GrowRow r{0, 0, 0, -1, 0, -1};
  if (n > 0 && end <= p.max_pages) {
    const int64_t fill = len % p.page;
    const int64_t base = fill != 0 ? held - 1 : held;  // the partly filled last page, too
    int64_t first = base;
    int kept = 0;
    bool some = false;
    for (int64_t j0 = base; j0 < end; j0 += 64) {
      const int64_t j = j0 + lane;
      const int32_t pid = j < end ? p.tables[b * p.stride + j] : -1;
      const int32_t refs = pid >= 0 && pid < p.P ? p.refs[pid] : 0;
      const bool last = fill != 0 && j == base;
      const uint64_t keep = __ballot(last ? refs <= 1 : refs == 1), give = __ballot(!last && refs > 1);
      if (lane == 0) {
        const int64_t word = b * p.words + (j0 - base) / 64;
        p.kept[word] = keep;
        p.given[word] = give;
      }
      kept += __builtin_popcountll(keep);
      uint64_t behind = keep | give;
      if (fill != 0 && j0 == base) {
        if (keep & 1u) {
          first = held;
        } else {
          r.src = __builtin_amdgcn_readfirstlane(pid);
          r.fill = static_cast<int32_t>(fill);
        }
        behind &= ~1ull;
      }
      some |= behind != 0;
    }
    r.first = static_cast<int32_t>(first);
    r.end = static_cast<int32_t>(end);
    r.want = static_cast<int32_t>(end - base) - kept;
    if (some) r.base = static_cast<int32_t>(base);
  }
  if (lane != 0) return;
  const int64_t over = n > 0 && end > p.max_pages ? end - p.max_pages : 0;
  p.over[b] = over < kMostOver ? over : kMostOver;
  p.rows[b] = r;
  p.old_len[b] = len;
}

// grow is bound by its three launches in turn, each a chain of loads and scans: 128 sequences over 16384
// pages take 3.4 + 5.2 + 4.9 us, the copies of the shared last pages in the last.
//
// A chunk's free pages by rank, and its counts.  Every workgroup adds up the chunks' and the rows' numbers itself.
__global__ void __launch_bounds__(256) grow_assign_kernel(const GrowParams p) {
  __shared__ int64_t lds[4];
  const int tid = threadIdx.x;
  const int64_t blk = blockIdx.x;
  const int64_t first = blk * kChunk + 16 * tid;
  int32_t r[16];
  load_refs(p.refs, p.P, first, r);
  int64_t rank, unused, before;
  const int64_t free_pages = sum_of(p.free_in, 1, p.chunks, blk, rank, lds, tid);
  int64_t want = sum_of(&p.rows[0].want, sizeof(GrowRow) / 4, p.B, 0, unused, lds, tid);
  const int64_t over = sum_of(p.over, 1, p.B, 0, unused, lds, tid);
  const int64_t lack = over + (want > free_pages ? want - free_pages : 0);
  if (lack) want = -1;
  const uint32_t free_bits = page_bits(r, false);
  block_scan(__builtin_popcount(free_bits), before, lds, tid);
  rank += before;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (((free_bits >> i) & 1u) && rank < want) {
      p.list[rank] = static_cast<int32_t>(first + i);
      r[i] = 1;
    }
    rank += (free_bits >> i) & 1u;
  }
  store_refs(p.refs_out, p.P, first, r);
  if (blk == 0 && tid == 0) {
    *p.missing = lack;
    *p.want = want;
  }
}

constexpr int kPoolsPerLaunch = 32;
struct PoolList {
  uint8_t* base[kPoolsPerLaunch];
  int64_t entry[kPoolsPerLaunch];  // bytes of one entry, a multiple of 4
};

// bytes (a multiple of 4) from a to b by a workgroup
__device__ __forceinline__ void copy_bytes(const uint8_t* a, uint8_t* b, int64_t bytes, int64_t at, int64_t step) {
  if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) == 0) {
    const int64_t whole = bytes >> 4;
    for (int64_t i = at; i < whole; i += step) reinterpret_cast<uint4*>(b)[i] = reinterpret_cast<const uint4*>(a)[i];
    for (int64_t i = (whole << 2) + at; i < bytes >> 2; i += step)
      reinterpret_cast<uint32_t*>(b)[i] = reinterpret_cast<const uint32_t*>(a)[i];
  } else {
    for (int64_t i = at; i < bytes >> 2; i += step)
      reinterpret_cast<uint32_t*>(b)[i] = reinterpret_cast<const uint32_t*>(a)[i];
  }
}

// Row blockIdx.x: its table, length and count (the first workgroup), and its shared last page into its
// fresh one, a share of it per blockIdx.y; pool blockIdx.z.
__global__ void __launch_bounds__(256) grow_row_kernel(const GrowParams p, const PoolList pools, int npools, bool first) {
  __shared__ int64_t lds[4];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  const GrowRow r = p.rows[b];
  const int64_t want = *p.want;
  const bool lead = first && blockIdx.y == 0 && blockIdx.z == 0;
  const bool copies = want >= 0 && r.src >= 0;
  if (!lead && !copies) return;
  int64_t begin;
  sum_of(&p.rows[0].want, sizeof(GrowRow) / 4, b, b, begin, lds, tid);
  if (lead) {
    const int32_t* const from = p.tables + b * p.stride;
    int32_t* const to = p.tables_out + b * p.stride_out;
    for (int64_t j = tid; j < p.max_pages; j += 256) {
      int32_t page = from[j];
      if (want >= 0 && j >= r.first && j < r.end) {
        int64_t rank = j - r.first;
        bool fresh = true;
        if (r.base >= 0) {  // behind the entries that stay
          const uint64_t* const kept = p.kept + b * p.words;
          const int64_t at = j - r.base, word = at >> 6;
          const uint64_t bit = 1ull << (at & 63);
          rank = at - __builtin_popcountll(kept[word] & (bit - 1));
          for (int64_t w = 0; w < word; ++w) rank -= __builtin_popcountll(kept[w]);
          fresh = (kept[word] & bit) == 0;
          if (p.given[b * p.words + word] & bit) atomicSub(p.refs_out + page, 1);
        }
        if (fresh) page = p.list[begin + rank];
      }
      to[j] = page;
    }
    if (tid == 0) {
      p.lens_out[b] = want >= 0 ? p.old_len[b] + row_count(p.tokens[b]) : p.lens[b];
      if (copies) atomicSub(p.refs_out + r.src, 1);
    }
  }
  if (!copies || npools == 0) return;
  const int64_t dst = p.list[begin];
  const int64_t eb = pools.entry[blockIdx.z];
  uint8_t* const base = pools.base[blockIdx.z];
  copy_bytes(base + r.src * (p.page * eb), base + dst * (p.page * eb), r.fill * eb,
             static_cast<int64_t>(blockIdx.y) * 256 + tid, static_cast<int64_t>(gridDim.y) * 256);
}

// ---- fork ---------------------------------------------------------------------------------

struct ForkParams {
  const int32_t* tables;
  int64_t stride, B, max_pages;
  const int64_t* lens;
  const int32_t* refs;
  int32_t* refs_out;
  int64_t P;
  const int32_t* parents;
  int64_t R;
  int page;
  int32_t* tables_out;
  int64_t stride_out;
  int64_t* lens_out;
  // copies of tables [B, max_pages] and lens [B] for a call whose outputs are its inputs (null: none needed)
  int32_t* tables_copy;
  int64_t* lens_copy;
};

// Two launches, both bound by latency: 64 sequences of up to 512 of 32768 pages take 2.1 and 4.9 us.  Pages that
// a row keeps are not counted down and up again.
__global__ void __launch_bounds__(256) fork_copy_kernel(const ForkParams p) {
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  if (p.refs_out != p.refs)
    for (int64_t i = i0; i < p.P; i += step) p.refs_out[i] = p.refs[i];
  if (p.tables_copy) {
    for (int64_t i = i0; i < p.B * p.max_pages; i += step)
      p.tables_copy[i] = p.tables[i / p.max_pages * p.stride + i % p.max_pages];
    for (int64_t i = i0; i < p.B; i += step) p.lens_copy[i] = p.lens[i];
  }
}

__global__ void __launch_bounds__(256) fork_kernel(const ForkParams p) {
  const int64_t i = blockIdx.x;
  const int32_t* const t = p.tables_copy ? p.tables_copy : p.tables;
  const int64_t stride = p.tables_copy ? p.max_pages : p.stride;
  const int64_t* const lens = p.tables_copy ? p.lens_copy : p.lens;
  int64_t par = i < p.R ? p.parents[i] : -1;
  if (par >= p.B) par = -1;
  int64_t len = par >= 0 ? lens[par] : 0;
  if (len < 0) len = 0;
  const int64_t keep = ceil_div64(len, p.page);
  for (int64_t j = threadIdx.x; j < p.max_pages; j += 256) {
    const int64_t old = i < p.B ? t[i * stride + j] : -1;
    int64_t now = par >= 0 && j < keep ? t[par * stride + j] : -1;
    if (now < 0 || now >= p.P) now = -1;
    if (i < p.R) p.tables_out[i * p.stride_out + j] = static_cast<int32_t>(now);
    if (old != now) {
      if (old >= 0 && old < p.P) atomicSub(p.refs_out + old, 1);
      if (now >= 0) atomicAdd(p.refs_out + now, 1);
    }
  }
  if (i < p.R && threadIdx.x == 0) p.lens_out[i] = len;
}

// ---- compact ------------------------------------------------------------------------------

struct CompactParams {
  const int32_t* tables;
  int32_t* tables_out;
  int64_t stride, stride_out, B, max_pages;
  const int32_t* refs;
  int32_t* refs_out;
  int64_t P;
  int page;
  int32_t* moved;    // [P] where each page is now, or null
  // workspace
  int64_t* used_in;  // [chunks] used pages of the chunk
  int64_t* used;     // [2] U, and the moves M
  int32_t* from;     // [P] page of the k-th move
  int32_t* to;       // [P]
  int32_t* from_refs;  // [P]
  int32_t* rank;     // [P] the move of a page behind U
  int64_t chunks;
};

__global__ void __launch_bounds__(256) compact_count_kernel(const CompactParams p) {
  __shared__ int64_t lds[4];
  const int tid = threadIdx.x;
  int64_t before;
  int32_t r[16];
  load_refs(p.refs, p.P, blockIdx.x * static_cast<int64_t>(kChunk) + 16 * tid, r);
  const int64_t total = block_scan(__builtin_popcount(page_bits(r, true)), before, lds, tid);
  if (tid == 0) p.used_in[blockIdx.x] = total;
}

// The moves by rank, and the counts without what moves.  The outputs may be the inputs, so a workgroup
// reads no counts but its own: refs before page U come from the chunks' numbers and its own chunk.
__global__ void __launch_bounds__(256) compact_list_kernel(const CompactParams p) {
  __shared__ int64_t lds[4];
  const int tid = threadIdx.x;
  const int64_t blk = blockIdx.x;
  const int64_t first = blk * kChunk + 16 * tid;
  int32_t r[16];
  load_refs(p.refs, p.P, first, r);
  int64_t n, before;
  const int64_t U = sum_of(p.used_in, 1, p.chunks, blk, n, lds, tid);
  const uint32_t used_bits = page_bits(r, true);
  block_scan(__builtin_popcount(used_bits), before, lds, tid);
  n += before;  // used pages before this thread's
  // holes are ranked from the first page, moves from the last: the k-th move is the (M - 1 - k)-th from there
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t page = first + i;
    const bool used = (used_bits >> i) & 1u;
    if (page == U) p.used[1] = U - n;
    if (page < U) {
      if (!used) p.to[page - n] = static_cast<int32_t>(page);
    } else if (used) {
      const int64_t k = U - 1 - n;  // so many used pages come behind it
      p.from[k] = static_cast<int32_t>(page);
      p.from_refs[k] = r[i];
      p.rank[page] = static_cast<int32_t>(k);
      r[i] = 0;
    }
    n += used;
  }
  store_refs(p.refs_out, p.P, first, r);
  if (tid == 0 && blk == 0) {
    p.used[0] = U;
    if (U == p.chunks * kChunk) p.used[1] = 0;  // no page U in any chunk
  }
}

// Bound by the memory where pages move: of 4096 pages of 64 8-bit entries a third, 110 MB, take 18.7 us (5.9
// TB/s, part of it from the caches), beside 2.3 and 5.0 us for the ranks.
//
// blockIdx.y == 0: tables and counts; otherwise the moves of pool blockIdx.y - 1
__global__ void __launch_bounds__(256) compact_move_kernel(const CompactParams p, const PoolList pools, bool first) {
  const int64_t U = p.used[0], M = p.used[1];
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  if (blockIdx.y == 0) {
    if (!first) return;
    for (int64_t i = at; i < M; i += step) p.refs_out[p.to[i]] = p.from_refs[M - 1 - i];
    // rank[] is written for moved pages only: a page without references, whose word is whatever was
    // there, is no move's `from`, and a table that names it keeps it
    auto now = [&](int32_t v) -> int32_t {
      if (v < U || v >= p.P) return v;
      const int32_t k = p.rank[v];
      return k >= 0 && k < M && p.from[k] == v ? p.to[M - 1 - k] : v;
    };
    if (p.moved)
      for (int64_t i = at; i < p.P; i += step) p.moved[i] = now(static_cast<int32_t>(i));
    for (int64_t i = at; i < p.B * p.max_pages; i += step) {
      const int64_t b = i / p.max_pages, j = i - b * p.max_pages;
      const int32_t v = now(p.tables[b * p.stride + j]);
      p.tables_out[b * p.stride_out + j] = v;
    }
    return;
  }
  const int64_t eb = pools.entry[blockIdx.y - 1] * p.page;
  uint8_t* const base = pools.base[blockIdx.y - 1];
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x)
    copy_bytes(base + p.from[M - 1 - m] * eb, base + p.to[m] * eb, eb, threadIdx.x, 256);
}

int64_t align16_up(int64_t x) { return (x + 15) & ~static_cast<int64_t>(15); }

int64_t grow_bytes(int64_t B, int64_t max_pages, int64_t P) {
  const int64_t chunks = (P + kChunk - 1) / kChunk, words = (max_pages + 63) / 64;
  return align16_up(sizeof(GrowRow) * B) + 8 * (2 * B + chunks + 1 + 2 * B * words) + 4 * P + 16;
}
int64_t fork_bytes(int64_t B, int64_t max_pages) { return align16_up(4 * B * max_pages) + 8 * B; }
int64_t compact_bytes(int64_t P) { return 8 * ((P + kChunk - 1) / kChunk + 2) + 16 * P + 32; }

constexpr int64_t kMaxInt = 0x7fffffff;
constexpr int64_t kMaxRows = (1 << 24) - 1;  // a workgroup each: a launch has less than 2^32 threads

#define MZK_CHECK_PAGES(name, B, max_pages, P)                                                                     \
  MZK_CHECK_ARG((B) >= 0 && (B) <= kMaxRows && (max_pages) >= 0 && (max_pages) <= kMaxInt && (P) >= 0 && (P) <= kMaxInt, \
                name ": bad sizes")

int check_pools(const char* name, const void* const* pools, const int64_t* entry, int n) {
  MZK_CHECK_ARG(n >= 0 && (n == 0 || (pools && entry)), "%s: null pool list", name);
  for (int i = 0; i < n; ++i)
    MZK_CHECK_ARG(pools[i] && entry[i] > 0 && entry[i] % 4 == 0 && (reinterpret_cast<uintptr_t>(pools[i]) & 3u) == 0,
                  "%s: pool %d needs a 4-byte aligned base and entries of a multiple of 4 bytes", name, i);
  return MZK_OK;
}

}  // namespace
}  // namespace mzk

using namespace mzk;

extern "C" int mzk_paged_append(const void* x, int dtype, int64_t T, int64_t x_row_stride, const int64_t* cu, int64_t B,
                                const int32_t* tables, int64_t table_stride, int64_t max_pages, const int64_t* lens,
                                int fmt, int D, int nope, void* pool, int64_t pages, int page, void* stream) {
  MZK_CHECK_ARG(T >= 0 && B >= 0, "paged_append: bad sizes");
  MZK_CHECK_PAGES("paged_append", B, max_pages, pages);
  MZK_CHECK_ARG(page >= 1, "paged_append: pages of at least one entry");
  MZK_CHECK_ARG(fmt == 0 || fmt == 1, "paged_append: fmt must be 0 (bf16) or 1 (fp8-b128)");
  MZK_CHECK_ARG(D >= 8 && D % 8 == 0 && D <= 4096, "paged_append: D must be a multiple of 8 up to 4096, got %d", D);
  MZK_CHECK_ARG(fmt == 0 || (nope >= 128 && nope % 128 == 0 && nope <= D),
                "paged_append: fp8 entries need nope, a multiple of 128 up to D (got %d of %d)", nope, D);
  MZK_CHECK_ARG(x_row_stride >= D && table_stride >= max_pages, "paged_append: strides smaller than the row");
  MZK_CHECK_ARG(cu || T == B, "paged_append: without cu one token per sequence (%lld tokens, %lld sequences)",
                (long long)T, (long long)B);
  if (T == 0 || B == 0) return MZK_OK;
  MZK_CHECK_ARG(x && lens && (tables || max_pages == 0) && (pool || pages == 0), "paged_append: null pointer");
  MZK_CHECK_ARG(aligned16(pool), "paged_append: the pool must be 16-byte aligned");
  MZK_CHECK_ARG(T <= 4 * kMaxRows, "paged_append: too many tokens");
  if (max_pages == 0 || pages == 0) return MZK_OK;  // every position is on no page
  const AppendParams p{x, x_row_stride, T, cu, B, tables, table_stride, max_pages, lens, static_cast<uint8_t*>(pool),
                       pages, page, D, fmt ? nope : 0};
  const bool vec = aligned16(x) && x_row_stride % 8 == 0;
  MZK_DISPATCH_DT(dtype, launch_append, p, vec, as_stream(stream));
  MZK_LAUNCH_CHECK("paged_append");
  return MZK_OK;
}

extern "C" int mzk_paged_workspace_bytes(int64_t B, int64_t max_pages, int64_t pages, int64_t* bytes) {
  MZK_CHECK_ARG(bytes != nullptr, "paged_workspace_bytes: null output");
  MZK_CHECK_PAGES("paged_workspace_bytes", B, max_pages, pages);
  int64_t n = grow_bytes(B, max_pages, pages);
  if (fork_bytes(B, max_pages) > n) n = fork_bytes(B, max_pages);
  if (compact_bytes(pages) > n) n = compact_bytes(pages);
  *bytes = align16_up(n);
  return MZK_OK;
}

extern "C" int mzk_paged_grow(const int32_t* tables, int64_t table_stride, int64_t B, int64_t max_pages,
                              const int64_t* lens, const int32_t* refs, int64_t pages, const int64_t* tokens, int page,
                              void* const* pools, const int64_t* entry_bytes, int npools, int32_t* tables_out,
                              int64_t table_out_stride, int64_t* lens_out, int32_t* refs_out, int64_t* missing,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  MZK_CHECK_PAGES("paged_grow", B, max_pages, pages);
  MZK_CHECK_ARG(B >= 1 && pages >= 1 && page >= 1, "paged_grow: at least one sequence, and one page of one entry");
  MZK_CHECK_ARG(table_stride >= max_pages && table_out_stride >= max_pages, "paged_grow: strides smaller than the row");
  if (int rc = check_pools("paged_grow", pools, entry_bytes, npools)) return rc;
  MZK_CHECK_ARG(tables && lens && refs && tokens && tables_out && lens_out && refs_out && missing, "paged_grow: null pointer");
  MZK_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= grow_bytes(B, max_pages, pages),
                "paged_grow: a 16-byte aligned workspace of %lld bytes is needed", (long long)grow_bytes(B, max_pages, pages));
  GrowParams p{tables, tables_out, table_stride, table_out_stride, B, max_pages, lens, lens_out, refs, refs_out, pages,
               tokens, page, missing};
  p.chunks = (pages + kChunk - 1) / kChunk;
  p.words = (max_pages + 63) / 64;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  p.rows = reinterpret_cast<GrowRow*>(w);
  w += align16_up(sizeof(GrowRow) * B);
  p.old_len = reinterpret_cast<int64_t*>(w);
  p.over = p.old_len + B;
  p.free_in = p.over + B;
  p.want = p.free_in + p.chunks;
  p.kept = reinterpret_cast<uint64_t*>(p.want + 1);
  p.given = p.kept + B * p.words;
  p.list = reinterpret_cast<int32_t*>(p.given + B * p.words);
  hipStream_t s = as_stream(stream);
  grow_count_kernel<<<static_cast<unsigned>(p.chunks + (B + 3) / 4), 256, 0, s>>>(p);
  grow_assign_kernel<<<static_cast<unsigned>(p.chunks), 256, 0, s>>>(p);
  int done = 0;
  do {
    PoolList l{};
    const int n = npools - done < kPoolsPerLaunch ? npools - done : kPoolsPerLaunch;
    for (int i = 0; i < n; ++i) {
      l.base[i] = static_cast<uint8_t*>(pools[done + i]);
      l.entry[i] = entry_bytes[done + i];
    }
    grow_row_kernel<<<dim3(static_cast<unsigned>(B), n ? 4 : 1, n ? n : 1), 256, 0, s>>>(p, l, n, done == 0);
    done += n;
  } while (done < npools);
  MZK_LAUNCH_CHECK("paged_grow");
  return MZK_OK;
}

extern "C" int mzk_paged_fork(const int32_t* tables, int64_t table_stride, int64_t B, int64_t max_pages,
                              const int64_t* lens, const int32_t* refs, int64_t pages, const int32_t* parents,
                              int64_t rows_out, int page, int32_t* tables_out, int64_t table_out_stride,
                              int64_t* lens_out, int32_t* refs_out, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  MZK_CHECK_PAGES("paged_fork", B, max_pages, pages);
  MZK_CHECK_ARG(rows_out >= 0 && rows_out <= kMaxRows && page >= 1, "paged_fork: bad sizes");
  MZK_CHECK_ARG(table_stride >= max_pages && table_out_stride >= max_pages, "paged_fork: strides smaller than the row");
  MZK_CHECK_ARG(tables && lens && refs && parents && tables_out && lens_out && refs_out, "paged_fork: null pointer");
  ForkParams p{tables, table_stride, B, max_pages, lens, refs, refs_out, pages, parents, rows_out, page, tables_out,
               table_out_stride, lens_out, nullptr, nullptr};
  if (tables == tables_out || lens == lens_out) {
    MZK_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= fork_bytes(B, max_pages),
                  "paged_fork: in place, a 16-byte aligned workspace of %lld bytes is needed",
                  (long long)fork_bytes(B, max_pages));
    p.tables_copy = static_cast<int32_t*>(workspace);
    p.lens_copy = reinterpret_cast<int64_t*>(static_cast<uint8_t*>(workspace) + align16_up(4 * B * max_pages));
  }
  hipStream_t s = as_stream(stream);
  int64_t n = refs != refs_out ? pages : 0;
  if (p.tables_copy) {  // (the lengths, too, of tables without columns)
    const int64_t copied = max_pages ? B * max_pages : B;
    if (copied > n) n = copied;
  }
  if (n > 0) {
    const int64_t g = (n + 255) / 256;
    fork_copy_kernel<<<static_cast<unsigned>(g < 2048 ? g : 2048), 256, 0, s>>>(p);
  }
  const int64_t rows = B > rows_out ? B : rows_out;
  if (rows > 0) fork_kernel<<<static_cast<unsigned>(rows), 256, 0, s>>>(p);
  MZK_LAUNCH_CHECK("paged_fork");
  return MZK_OK;
}

extern "C" int mzk_paged_compact(const int32_t* tables, int64_t table_stride, int64_t B, int64_t max_pages,
                                 const int32_t* refs, int64_t pages, int page, void* const* pools,
                                 const int64_t* entry_bytes, int npools, int32_t* tables_out, int64_t table_out_stride,
                                 int32_t* refs_out, void* workspace, int64_t workspace_bytes, void* stream) {
  return mzk_paged_compact_map(tables, table_stride, B, max_pages, refs, pages, page, pools, entry_bytes, npools, tables_out,
                               table_out_stride, refs_out, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int mzk_paged_compact_map(const int32_t* tables, int64_t table_stride, int64_t B, int64_t max_pages,
                                     const int32_t* refs, int64_t pages, int page, void* const* pools,
                                     const int64_t* entry_bytes, int npools, int32_t* tables_out, int64_t table_out_stride,
                                     int32_t* refs_out, int32_t* moved, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  MZK_CHECK_PAGES("paged_compact", B, max_pages, pages);
  MZK_CHECK_ARG(page >= 1, "paged_compact: pages of at least one entry");
  MZK_CHECK_ARG(table_stride >= max_pages && table_out_stride >= max_pages, "paged_compact: strides smaller than the row");
  if (int rc = check_pools("paged_compact", pools, entry_bytes, npools)) return rc;
  MZK_CHECK_ARG(tables && refs && tables_out && refs_out, "paged_compact: null pointer");
  MZK_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= compact_bytes(pages),
                "paged_compact: a 16-byte aligned workspace of %lld bytes is needed", (long long)compact_bytes(pages));
  CompactParams p{tables, tables_out, table_stride, table_out_stride, B, max_pages, refs, refs_out, pages, page, moved};
  p.chunks = (pages + kChunk - 1) / kChunk;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  p.used_in = reinterpret_cast<int64_t*>(w);
  p.used = p.used_in + p.chunks;
  p.from = reinterpret_cast<int32_t*>(p.used + 2);
  p.to = p.from + pages;
  p.from_refs = p.to + pages;
  p.rank = p.from_refs + pages;
  hipStream_t s = as_stream(stream);
  if (pages == 0) return MZK_OK;
  compact_count_kernel<<<static_cast<unsigned>(p.chunks), 256, 0, s>>>(p);
  compact_list_kernel<<<static_cast<unsigned>(p.chunks), 256, 0, s>>>(p);
  int done = 0;
  do {
    PoolList l{};
    const int n = npools - done < kPoolsPerLaunch ? npools - done : kPoolsPerLaunch;
    for (int i = 0; i < n; ++i) {
      l.base[i] = static_cast<uint8_t*>(pools[done + i]);
      l.entry[i] = entry_bytes[done + i];
    }
    compact_move_kernel<<<dim3(1024, 1 + n), 256, 0, s>>>(p, l, done == 0);
    done += n;
  } while (done < npools);
  MZK_LAUNCH_CHECK("paged_compact");
  return MZK_OK;
}
