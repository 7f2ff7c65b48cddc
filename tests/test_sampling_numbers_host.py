"""CPU: the numbers of ``csrc/sampling_numbers.h`` in a host build whose arithmetic is checked (overflowing conversions and sums
end it): what the GPU turns into 0 or a largest number by itself is undefined in C++, and no compiler has to keep it."""

import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "mzoo_amd" / "csrc"
CHECKS = ["-fsanitize=undefined,float-cast-overflow", "-fno-sanitize-recover=undefined,float-cast-overflow"]

HEAD = r"""
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#define __device__
#define __forceinline__ inline
#include "sampling_numbers.h"
using namespace mzk;
static float bf16(uint32_t bits) { bits <<= 16; float f; std::memcpy(&f, &bits, 4); return f; }
"""


def _run(tmp_path, body):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    src = tmp_path / "numbers.cpp"
    src.write_text(HEAD + "int main() {\n" + body + "\n  return 0;\n}\n")
    exe = tmp_path / "numbers"
    built = subprocess.run(["g++", "-O1", "-std=c++17", "-ffp-contract=off", *CHECKS, "-I", str(CSRC), str(src), "-o", str(exe)],
                           capture_output=True, text=True, timeout=120)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0, (ran.stdout + ran.stderr)[-2000:]
    return ran.stdout


def test_powers_of_two(tmp_path):
    """Below 2^-51 of itself, in units of 2^-53.  t - n is exact; x = (t - n) ln 2 is off by at most 0.52 (its rounding and ln 2's own, of
    |x| <= 0.347), the last two sums by at most half a step, 0.5 below 1 and 1 above, and 0.347 of that, those before
    by 0.1 in all, and the series by 1.55: at x = -0.347 0.5 + 0.17 + 0.1 + 0.37 + 1.55 of e = 0.707, 3.9; at 0.347
    1 + 0.35 + 0.1 + 0.74 + 1.55 of 1.414, 2.7.  At n the power is exact down to 2^-1022."""
    _run(tmp_path, r"""
  for (int i = -999000; i <= 999000; ++i) {
    const double t = i / 1000.0 + i * 1e-9;
    const long double want = exp2l(static_cast<long double>(t));
    if (fabsl(exp2_of(t) - want) > want * 0x1p-51L) { std::printf("%.17g: %.17g\n", t, exp2_of(t)); return 1; }
  }
  if (exp2_of(0.0) != 1.0 || exp2_of(-1e300) != 0.0 || exp2_of(-INFINITY) != 0.0 || exp2_of(NAN) != 0.0 || exp2_of(-700.0) != 0x1p-700) return 2;
""")


def test_weights_of_all_values_of_a_block(tmp_path):
    """Rows counted by value weigh every value of a block of 128, those above the row's largest among them, at any
    temperature: their number, 0, times their weight is 0."""
    _run(tmp_path, r"""
  const double temperatures[] = {1.401298464324817e-45, 1e-30, 1e-3, 0.01, 0.3, 1.0, 1e30, 3.4028234663852886e38, INFINITY};
  const uint32_t largest[] = {0x4220 /* 40 */, 0x0000, 0x3f80, 0x7f00, 0x7f7f, 0x0001, 0xbf80, 0xff7f, 0xff00, 0x807f};
  for (double T : temperatures)
    for (uint32_t m : largest) {
      const double s = kPerOctave * kLog2eD / T;
      for (uint32_t o = 128; o < 65408; ++o) {  // the order of falling values; without NaN and the infinities
        const uint32_t bits = o < 0x8000u ? 0x7fffu - o : o;
        const double w = weight_of(bf16(bits), bf16(m), s, 62);
        const double none = 0.0 * w + 0.5, all = 1.0 * w + 0.5;
        if (static_cast<uint64_t>(none) != 0) { std::printf("T %g, value %g of a largest %g: weight %g\n", T, bf16(bits), bf16(m), w); return 1; }
        if (bf16(bits) <= bf16(m) && static_cast<uint64_t>(all) > 1ull << 62) return 2;
        if (bf16(bits) == bf16(m) && w != 0x1p62) return 3;
      }
    }
  if (weight_of(-INFINITY, 1.0f, 0.0, 62) != 0.0) return 4;  // at an infinite temperature
""")


def test_the_bottom_of_no_token(tmp_path):
    """A row that begins masked has no largest bin yet: nothing is below what is kept, and -inf is not above it."""
    _run(tmp_path, r"""
  if (bottom_of(0) != -1023.0 || bottom_of(1 << 28) != 268434433.0) return 1;
  if (!(bottom_of(kNoTop) < -0x1p31) || -INFINITY > bottom_of(kNoTop)) return 2;
""")


def test_places_of_far_bins(tmp_path):
    """A masked token lies any number of bins below the largest; its place, which nobody reads, is one of the histogram's."""
    _run(tmp_path, r"""
  const double near[] = {0.0, 1.0, -1.0, 1023.0, 1024.0, -1024.0, 1e6, -1e6, 134217727.0, 134217728.0, 268435456.0, -268435456.0, -3e9, 1e12, -1e15};
  const double farther[] = {-1e30, -1e85, -INFINITY, NAN};
  for (double n : near) {
    const int at = place_of(n + 0x1.8p52), want = static_cast<int>(static_cast<long long>(n) & kRest) * 8 * kCopies;
    if (at != want) { std::printf("%g: %d\n", n, at); return 1; }
  }
  for (double far : farther) {
    const int at = place_of(far + 0x1.8p52);
    if (at < 0 || at > 8 * kCopies * kRest || at % (8 * kCopies)) return 2;
  }
""")
