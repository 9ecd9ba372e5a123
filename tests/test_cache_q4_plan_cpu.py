"""The plan of attention over a cache held in 4 bits (csrc/mer_attention_plan.hpp),
compiled and run on the CPU: it keeps within what every call reserves, in any
form that its kernels have, and falls back to one chunk without memory."""
from __future__ import annotations

from test_attention_plan_cpu import build_and_run

MAIN = r"""
#include <initializer_list>
#include "mer_attention_plan.hpp"
#include <stdio.h>
using namespace mer;
static int bad = 0;
#define CHECK(c) do { if (!(c) && bad++ < 20) printf("line %d: %s (seqs %zu tokens %zu group %u kv heads %u dim %u q %zu keys %zu window %u cus %d floats %zu)\n", \
  __LINE__, #c, seqs, tokens, group, heads, dim, q, keys, window, cus, floats); } while (0)
int main() {
  unsigned long plans = 0, wide = 0, narrow = 0, rows32 = 0, split = 0, far = 0;
  for (int cus : {256, 32, 304}) for (size_t seqs : {1, 2, 7, 24, 64, 300, 5000}) for (size_t tokens : {1, 2, 17, 128, 300, 1024, 8192})
  for (size_t longest : {1, 2, 5, 8, 100, 512, 8192}) for (size_t keys : {0, 100, 256, 511, 4096, 32768, 131072, 1 << 30})
  for (uint32_t group : {1, 3, 4, 8, 16, 20, 32, 33}) for (uint32_t heads : {1, 3, 8, 64}) for (uint32_t dim : {32, 64, 96, 128, 160, 256})
  for (uint32_t window : {0u, 1000u}) {
    const size_t q = longest < tokens ? longest : tokens;
    const size_t r = attn_reserve(seqs, tokens, group, heads, dim, q, keys, cus);
    for (size_t floats : {r, r / 3, (size_t)0}) {
      const AttnPlan p = attn_q4_plan(seqs, tokens, group, heads, dim, q, keys, keys, window, cus, floats);
      const size_t need = p.part_o_floats + p.part_ml_floats, rows = q * group;
      ++plans;
      CHECK(need <= floats);
      CHECK(p.rows == 16 || p.rows == 32 || p.rows == 128);
      if (p.rows == 128) {
        const size_t base = (size_t)p.n_units * heads;
        split += p.n_chunks > 1;
        CHECK(p.n_units >= (tokens * group + 127) / 128 + seqs && p.n_chunks >= 1 && p.n_wgs == base * p.n_chunks);
        CHECK(p.chunk >= 64 && p.chunk % 64 == 0 && (need == 0) == (p.n_chunks == 1));
        CHECK(window || (size_t)p.chunk * p.n_chunks >= keys);
        CHECK(p.n_chunks == 1 || need == base * p.n_chunks * 128 * (attn_padded_dim(dim) + 2));
        // small calls are taken by it where memory or 32 bits do not allow others
        if (rows <= 32 && floats == r) { ++far; CHECK((tokens * group / 16 + seqs) * heads * (keys / 128 + 2) >= (1ull << 31)); }
      } else {
        (p.rows == 32 ? rows32 : p.waves == 1 ? narrow : wide) += 1;
        CHECK(p.waves == 4 || (p.waves == 1 && p.rows == 16));  // what there are kernels for
        CHECK(p.rows == 16 || (dim <= 128 && rows > 16));
        CHECK(rows <= 32 && (p.rows == 32 || rows <= 16 || dim > 128 || (2 * seqs * heads <= (size_t)cus && seqs * heads * keys < 2048ull * cus)));
        CHECK((tokens * group / 16 + seqs) * heads * (keys / 128 + 2) < (1ull << 31));
        CHECK(p.n_wgs >= kAttnTickets && p.n_wgs < kAttnEpoch && 3 * (size_t)p.n_wgs + kAttnTickets * kAttnTicketWords <= attn_counters(cus));
        CHECK(need == 2 * (size_t)p.n_wgs * p.rows * (dim + 2) && p.min_granules == 1);
      }
    }
  }
  printf("%lu plans: %lu wide, %lu narrow, %lu of 32 rows, %lu with chunks, %lu past 32 bits, %d failures\n", plans, wide, narrow, rows32,
         split, far, bad);
  return bad || !wide || !narrow || !rows32 || !split || !far;
}
"""


def test_every_plan_keeps_within_what_is_reserved(tmp_path):
    build_and_run(tmp_path, MAIN)
