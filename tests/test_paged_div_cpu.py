"""The quotients of the paged cache's kernels (csrc/qh_paged_div.h, which the launches and the kernels
share), compiled for the CPU and held against divisions."""
import os
import subprocess

from test_lds_reads_cpu import hipbuild

MAIN = r"""
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <random>
#include "qh_paged_div.h"

int bad = 0;
void is(long long got, long long want, const char* what, long long x, long long d) {
  if (got != want && ++bad < 10) std::printf("%s: %lld / %lld gave %lld, is %lld\n", what, x, d, got, want);
}

int main() {
  std::mt19937_64 rng(3);
  auto below = [&](long long n) { return (long long)(rng() % (unsigned long long)n); };
  // page sizes: multiples of 8 up to the most positions of a table
  for (int i = 0; i < 4000; ++i) {
    const long long d = i < 75 ? 8 * (i + 1) : i == 75 ? 0x7FFF0000LL : 8 * (1 + below(1ll << (3 + i % 25)));
    if (d > 0x7FFFFFFF) continue;
    const QhDiv q = qh_div_by((uint32_t)d);
    auto at = [&](long long x) {
      if (x >= 0 && x <= 0x7FFFFFFF) is(qh_quotient((int)x, q.mul, q.shift), x / d, "page", x, d);
    };
    for (long long x : {0ll, 1ll, d - 1, d, d + 1, 0x7FFFFFFFll}) at(x);
    for (int k = 0; k < 200; ++k) {
      at(below(1ll << 31));
      const long long m = d * below((1ll << 31) / d + 1);
      at(m - 1);
      at(m);
    }
  }
  for (int group = 1; group <= 16; ++group)
    for (int i = 0; i < 1024; ++i) is(qh_group_quotient(i, qh_group_mul(group)), i / group, "group", i, group);
  // the kernel's reciprocal is off by an ulp at most, of b rounded to a float
  for (int k = 0; k < 2000000; ++k) {
    const int b = 1 + (int)below(1ll << (1 + k % 31)), most = 1 + (int)below(1ll << (1 + k % 20));
    const long long top = (long long)b * most + below(b);
    if (b < 1 || top > 0x7FFFFFFF) continue;
    const float r = 1.0f / (float)b;
    for (long long a : {top, (long long)b * most, (long long)b * most - 1, below(top + 1)})
      for (float e : {std::nextafterf(r, 0.0f), r, std::nextafterf(r, 2.0f)})
        is(qh_quotient_near((int)a, b, e), a / b, "near", a, b);
  }
  std::printf("%d wrong\n", bad);
  return bad != 0;
}
"""


def run(tmp_path, header_dir):
    src, exe = tmp_path / "div.cpp", tmp_path / "div"
    src.write_text(MAIN)
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-I", str(header_dir), str(src), "-o", str(exe)],
                   check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True)


def test_quotients(tmp_path):
    r = run(tmp_path, hipbuild.CSRC)
    assert r.returncode == 0, r.stdout


def test_a_wrong_multiplier_is_found(tmp_path):
    """One too small for pages and for groups, no correction of the near quotient (in a copy)."""
    text = open(os.path.join(hipbuild.CSRC, "qh_paged_div.h")).read()
    for was, now, what in (("/ d + 1)", "/ d)", "page"), ("+ group - 1) / group", ") / group", "group"),
                           ("rest < 0 ? q - 1 : rest >= b ? q + 1 : q", "q", "near")):
        assert text.count(was) == 1
        (tmp_path / "qh_paged_div.h").write_text(text.replace(was, now))
        r = run(tmp_path, tmp_path)
        assert r.returncode == 1 and what in r.stdout, was
