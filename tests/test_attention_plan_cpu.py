"""The attention call's plan (csrc/mer_attention_plan.hpp), compiled and run on
the CPU: a call that is no larger than another in any size reserves no more, so
it never moves a workspace that served the larger one, and every plan keeps
within what it was given.  And the counters of the pieces that are joined, played
through: a launch counts right whatever an earlier one left in them."""
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
        CHECK(3 * (size_t)p.n_wgs + kAttnTickets * kAttnTicketWords <= attn_counters(cus) && p.n_wgs >= kAttnTickets && need == 2 * (size_t)p.n_wgs * p.rows * (s.dim + 2));
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


COUNTERS = r"""
#include "mer_attention_plan.hpp"
#include <algorithm>
#include <random>
#include <stdio.h>
#include <vector>
using namespace mer;
// Launches whose workgroups take their tickets, open a counter and count in it,
// each step in any order between workgroups.  Some launches leave counts behind:
// workgroups that stop after any of their steps, or count twice.
int main() {
  std::mt19937 rng(1);
  auto below = [&](uint32_t n) { return (uint32_t)(rng() % n); };
  std::vector<uint64_t> tickets(kAttnTickets, 0), counters(2048, 0);
  const uint32_t grids[] = {32, 33, 63, 64, 100, 256, 512, 1024, 2048};
  long units = 0, bad = 0, left = 0;
  for (int launch = 0; launch < 400; ++launch) {
    const uint32_t n = grids[below(9)];
    const bool broken = below(3) == 0;
    std::vector<uint32_t> first(n), pieces(n), step(n, 0), stop(n, 3), live(n), last_of(n, 0), counted(n, 0);
    std::vector<uint64_t> epoch(n);
    for (uint32_t w = 0; w < n;) {  // units of neighbouring workgroups
      const uint32_t k = std::min(n - w, 1 + below(40));
      for (uint32_t i = 0; i < k; ++i) first[w + i] = w, pieces[w + i] = k;
      w += k;
    }
    if (broken) for (uint32_t w = 0; w < n; ++w) if (below(4) == 0) stop[w] = 1 + below(2), left += 1;
    for (uint32_t w = 0; w < n; ++w) live[w] = w;
    while (!live.empty()) {
      const uint32_t at = below((uint32_t)live.size()), w = live[at];
      if (step[w] == 0) {
        uint64_t &t = tickets[w % kAttnTickets];
        epoch[w] = attn_epoch(t);
        t += attn_ticket(w, n);
      } else if (step[w] == 1) {
        counters[first[w]] = std::max(counters[first[w]], epoch[w]);
      } else {
        const int times = broken && below(8) == 0 ? 2 : 1;
        for (int i = 0; i < times; ++i) {
          const uint64_t before = counters[first[w]]++;
          ++counted[first[w]];
          if (attn_is_last(before, pieces[w])) {
            ++last_of[first[w]];
            if (!broken && counted[first[w]] != pieces[w]) ++bad;
          }
        }
      }
      if (++step[w] == stop[w]) live[at] = live.back(), live.pop_back();
    }
    for (uint32_t w = 0; w < n; ++w) if (epoch[w] != (uint64_t)launch * kAttnEpoch) ++bad;
    if (!broken) for (uint32_t w = 0; w < n; ++w) if (first[w] == w) ++units, bad += last_of[w] != 1;
  }
  printf("%ld units joined, %ld workgroups stopped before, %ld failures\n", units, left, bad);
  return bad || !units || !left;
}
"""


def test_counters_of_a_launch_that_others_left_theirs_to(tmp_path):
    build_and_run(tmp_path, COUNTERS)


def test_reserve_grows_and_holds_every_plan(tmp_path):
    build_and_run(tmp_path, "#include <initializer_list>\n" + MAIN)


def build_and_run(tmp_path, main):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not available")
    (tmp_path / "plan.cpp").write_text(main)
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", CSRC, str(tmp_path / "plan.cpp"),
                        "-o", str(tmp_path / "plan")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    out = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout
