// What the attention kernels share: vector types, entry formats and the fetch of an entry's pieces
// into a tile of bf16 rows in LDS.
#pragma once

#include "common.h"

namespace mzk {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

enum { kFmtBf16 = 0, kFmtFp8 = 1 };

__device__ __forceinline__ __attribute__((address_space(3))) v4s* lds_v4s(const uint8_t* p) {
  return (__attribute__((address_space(3))) v4s*)(p);
}

constexpr int kTile = 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int FMT, int D, int NOPE>
struct Layout {
  static constexpr int kEntryBytes = FMT == kFmtFp8 ? NOPE + 4 * (NOPE / 128) + 2 * (D - NOPE) : 2 * D;
  // An entry is fetched as 16-byte pieces: fp8 = NOPE/16 code pieces (16 e4m3 codes each)
  // followed by (D-NOPE)/8 rope pieces (8 bf16 each); bf16 = D/8 pieces of 8 channels.
  static constexpr int kCodePieces = FMT == kFmtFp8 ? NOPE / 16 : 0;
  static constexpr int kPieces = FMT == kFmtFp8 ? NOPE / 16 + (D - NOPE) / 8 : D / 8;
};

typedef const uint8_t __attribute__((address_space(1)))* gptr_t;  // global (not flat) loads
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ T gload(gptr_t p) {
  return *(const __attribute__((address_space(1))) T*)(p);
}

// One fetched 16-byte piece of an entry (held in registers a tile ahead of use).
struct Piece {
  u32x4 v;  // fp8 code piece: 16 codes; rope / bf16 piece: 8 bf16
  float s;  // fp8 code piece: its 128-channel block scale
};

template <int FMT, int D, int NOPE>
__device__ __forceinline__ Piece fetch_piece(gptr_t e, int q) {
  using L = Layout<FMT, D, NOPE>;
  Piece r;
  r.s = 1.0f;
  if constexpr (FMT == kFmtFp8) {
    constexpr int NB = NOPE / 128;
    if (q < L::kCodePieces) {
      r.v = gload<u32x4>(e + 16 * q);
      r.s = gload<float>(e + NOPE + 4 * (q >> 3));
    } else {
      r.v = gload<u32x4>(e + NOPE + 4 * NB + 16 * (q - L::kCodePieces));
    }
  } else {
    r.v = gload<u32x4>(e + 16 * q);
  }
  return r;
}

// Writes piece q of an entry to its bf16 row in LDS: e4m3 codes times the pow2 block scale
// through the hardware conversion (exact in bf16); rope / bf16 pieces as they are.
template <int FMT, int D, int NOPE>
__device__ __forceinline__ void store_piece(uint8_t* krow, const Piece& r, int q) {
  using L = Layout<FMT, D, NOPE>;
  if constexpr (FMT == kFmtFp8) {
    if (q < L::kCodePieces) {
      *reinterpret_cast<uint4*>(krow + 32 * q) = dequant_fp8x8_bf16(uint2{r.v.x, r.v.y}, r.s);
      *reinterpret_cast<uint4*>(krow + 32 * q + 16) = dequant_fp8x8_bf16(uint2{r.v.z, r.v.w}, r.s);
    } else {
      *reinterpret_cast<uint4*>(krow + 2 * NOPE + 16 * (q - L::kCodePieces)) = uint4{r.v.x, r.v.y, r.v.z, r.v.w};
    }
  } else {
    *reinterpret_cast<uint4*>(krow + 16 * q) = uint4{r.v.x, r.v.y, r.v.z, r.v.w};
  }
}

}  // namespace
}  // namespace mzk
