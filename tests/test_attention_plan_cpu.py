"""The attention call's plan (csrc/mer_attention_plan.hpp), compiled and run on
the CPU: a call that is no larger than another in any size reserves no more, so
it never moves a workspace that served the larger one, and every plan keeps
within what it was given."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import PKG_NAME, ROOT

CSRC = os.path.join(ROOT, PKG_NAME, "csrc")

MAIN = r"""
#include "mer_attention_plan.hpp"
#include <stdio.h>
using namespace mer;
static int bad = 0;
struct Sizes { size_t seqs, tokens; uint32_t group, heads, dim; size_t q, keys; };
#define CHECK(c) do { if (!(c) && bad++ < 20) printf("line %d: %s (seqs %zu tokens %zu group %u kv heads %u dim %u q %zu keys %zu window %u cus %d)\n", \
  __LINE__, #c, s.seqs, s.tokens, s.group, s.heads, s.dim, s.q, s.keys, window, cus); } while (0)
static size_t reserve(const Sizes &s, int cus) {
  return attn_reserve(s.seqs, s.tokens, s.group, s.heads, s.dim, s.q < s.tokens ? s.q : s.tokens, s.keys, cus);
}
int main() {
  const size_t seqs[] = {1, 2, 7, 64, 300}, tokens[] = {1, 2, 17, 128, 256, 300, 512, 1024, 2048, 4096, 8192};
  const size_t qs[] = {1, 2, 8, 100, 512, 4096, 8192}, keys[] = {0, 100, 256, 511, 4096, 32768, 131072};
  const uint32_t groups[] = {1, 3, 4, 8, 16, 20}, heads[] = {1, 3, 8, 64}, dims[] = {8, 64, 80, 128, 192, 256};
  const uint32_t windows[] = {0, 1, 1000};
  const unsigned n1 = 5, n2 = 11, n3 = 7, n4 = 7, n5 = 6, n6 = 4, n7 = 6;
  unsigned long plans = 0, split = 0, moved = 0;
  for (int cus : {256, 32, 304})
  for (unsigned a = 0; a < n1; ++a) for (unsigned b = 0; b < n2; ++b) for (unsigned c = 0; c < n3; ++c) for (unsigned d = 0; d < n4; ++d)
  for (unsigned e = 0; e < n5; ++e) for (unsigned f = 0; f < n6; ++f) for (unsigned g = 0; g < n7; ++g) {
    const Sizes s = {seqs[a], tokens[b], groups[e], heads[f], dims[g], qs[c], keys[d]};
    uint32_t window = 0;
    const size_t r = reserve(s, cus);
    auto up = [&](Sizes t) { CHECK(r <= reserve(t, cus)); };
    Sizes t;
    if (a + 1 < n1) { t = s; t.seqs = seqs[a + 1]; up(t); }
    if (b + 1 < n2) { t = s; t.tokens = tokens[b + 1]; up(t); }
    if (c + 1 < n3) { t = s; t.q = qs[c + 1]; up(t); }
    if (d + 1 < n4) { t = s; t.keys = keys[d + 1]; up(t); }
    if (e + 1 < n5) { t = s; t.group = groups[e + 1]; up(t); }
    if (f + 1 < n6) { t = s; t.heads = heads[f + 1]; up(t); }
    if (g + 1 < n7) { t = s; t.dim = dims[g + 1]; up(t); }
    CHECK(r <= kAttnRegionFloats || cus > 512);
    const size_t q = s.q < s.tokens ? s.q : s.tokens;
    for (uint32_t w : windows) for (size_t floats : {r, r / 3, (size_t)0}) {
      window = w;
      const AttnPlan p = attn_plan(s.seqs, s.tokens, s.group, s.heads, s.dim, q, s.keys, s.keys, w, cus, floats);
      ++plans; split += p.n_chunks > 1;
      const size_t need = p.part_o_floats + p.part_ml_floats;
      CHECK(need <= floats);
      CHECK(p.rows == 16 || p.rows == 32 || p.rows == 128);
      if (p.rows == 128) {
        const size_t base = (size_t)p.n_units * s.heads;
        CHECK(p.n_units >= (s.tokens * s.group + 127) / 128 + s.seqs && p.n_chunks >= 1 && p.n_wgs == base * p.n_chunks);
        CHECK(p.chunk >= 64 && p.chunk % 64 == 0 && (need == 0) == (p.n_chunks == 1));
        CHECK(w || (size_t)p.chunk * p.n_chunks >= s.keys);
        CHECK(p.n_chunks == 1 || need == base * p.n_chunks * 128 * (attn_padded_dim(s.dim) + 2));
      } else {
        CHECK(3 * (size_t)p.n_wgs <= attn_counters(cus) && need == 2 * (size_t)p.n_wgs * p.rows * (s.dim + 2));
        CHECK(p.rows == 16 || q * s.group > 16);
      }
      if (floats == r && b + 1 < n2 && cus == 256) {  // plans alone would move the buffer for a smaller call
        const size_t q2 = s.q < tokens[b + 1] ? s.q : tokens[b + 1];
        const AttnPlan l = attn_plan(s.seqs, tokens[b + 1], s.group, s.heads, s.dim, q2, s.keys, s.keys, w, cus, r);
        moved += l.part_o_floats + l.part_ml_floats < need;
      }
    }
  }
  printf("%lu plans, %lu with chunks, %lu that need more than a larger call's, %d failures\n", plans, split, moved, bad);
  return bad || !split || !moved;
}
"""


def test_reserve_grows_and_holds_every_plan(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not available")
    (tmp_path / "plan.cpp").write_text("#include <initializer_list>\n" + MAIN)
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", CSRC, str(tmp_path / "plan.cpp"),
                        "-o", str(tmp_path / "plan")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    out = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout
