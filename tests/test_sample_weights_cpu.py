"""The weights of sampling by row (csrc/qh_weights.h, which the kernels share), compiled for the CPU without any
contraction of products and sums, and held against exp."""
import os
import subprocess

from test_lds_reads_cpu import hipbuild

MAIN = r"""
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include "qh_weights.h"

int bad = 0;
void expect(bool good, const char* what, double heat, float top, float x, double v) {
  if (!good && ++bad < 10) std::printf("%s: temperature %g, largest %.9g, logit %.9g: %.17g\n", what, heat, top, x, v);
}

int main() {
  std::mt19937_64 rng(11);
  auto real = [&]() { return (double)(rng() >> 11) * 0x1p-53; };
  // the largest logit is in bin 0 of its own, also where neighbouring logits are many bins apart
  for (double heat : {1.0, 0.7, 1e-6, 1e-9, 1e-12, 3e-13, 1e-13, 1e-30})
    for (int i = 0; i < 200000; ++i) {
      const float top = (float)((real() - 0.5) * std::exp2(std::floor(12 * real())));
      const double c4 = 4.0 * 1.4426950408889634 / heat;
      const Scale s(c4, heat * 0.17328679513998632, top);
      int bin = -7;
      uint64_t fx = 0;
      expect(s.weigh(top, bin, fx) && bin == 0, "weigh", heat, top, top, bin);
      if (s.quick) {
        const double v = s.weigh_quick(top, bin);
        expect(bin == 0 && (uint64_t)(v - kWhole) == fx, "weigh_quick", heat, top, top, bin);
      }
      // and a logit below it weighs what it should: half a unit for the rounding to a whole number, 2^35 times the
      // polynomial's 1.1e-13 (0.004) and the 2^-48 of an exponent of 35 here (0.0001)
      const float x = top - (float)(30.0 * heat * real());
      if (heat < 0.5 || !s.weigh(x, bin, fx)) continue;
      const double want = std::exp2(std::log2((double)kOne) + std::fma((double)x, c4, bin - s.base) / 4.0);
      expect(std::fabs((double)fx - want) <= 0.5 + 0.005, "weight", heat, top, x, (double)fx - want);
    }
  std::printf("%d wrong\n", bad);
  return bad != 0;
}
"""


def run(tmp_path, header_dir):
    src, exe = tmp_path / "weights.cpp", tmp_path / "weights"
    src.write_text(MAIN)
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-ffp-contract=off", "-I", str(header_dir), str(src),
                    "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True)


def test_the_largest_is_in_bin_0_and_weights_are_what_they_are(tmp_path):
    r = run(tmp_path, hipbuild.CSRC)
    assert r.returncode == 0, r.stdout


def test_a_product_that_is_rounded_on_its_own_is_found(tmp_path):
    with open(os.path.join(hipbuild.CSRC, "qh_weights.h")) as f:
        text = f.read()
    line = "fma((double)top, c4, kRound) - kRound"
    assert text.count(line) == 1
    (tmp_path / "qh_weights.h").write_text(text.replace(line, "(t + kRound) - kRound"))
    r = run(tmp_path, tmp_path)
    assert r.returncode == 1 and "weigh" in r.stdout
