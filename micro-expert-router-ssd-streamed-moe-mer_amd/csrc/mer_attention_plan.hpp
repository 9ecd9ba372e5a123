// mer_attention_plan.hpp -- how an attention call is cut and what workspace it
// reserves (mer_hip_paged_attention, mer_attention.hip).  Host arithmetic on
// sizes only, without HIP, so that it can be compiled and checked anywhere.
#pragma once
#include <math.h>
#include <stddef.h>
#include <stdint.h>

namespace mer {

struct AttnPlan {
  uint32_t rows;             // rows of a tile
  uint32_t n_wgs, waves;     // workgroups, waves of each (tiles of 16 and 32 rows)
  uint32_t min_granules, n_units, chunk, n_chunks;
  size_t part_o_floats, part_ml_floats;  // partial sums
};

// Counters of the 16- and 32-row tiles, 64 bits each.  Of a launch, workgroups
// that have done a piece of a unit count themselves in (three counters for each
// of at most 8 workgroups a CU); the last one joins the pieces.  No launch
// relies on what an earlier one left there: a counter holds an epoch above its
// count, and whoever counts first raises it to its own launch's epoch.  Epochs
// come from tickets, each a sum to which the workgroups of a launch that share it
// (every kAttnTickets-th) add kAttnEpoch in all, so that all of them find the same
// multiple of it there, in whatever order they come.  32 tickets, a cache line
// each: one for all cost 1024 workgroups 10 us.
constexpr uint32_t kAttnTickets = 32, kAttnTicketWords = 16;
constexpr uint64_t kAttnEpoch = 1u << 16;
constexpr size_t attn_counters(int cus) { return kAttnTickets * kAttnTicketWords + 3 * 8 * (size_t)cus; }
// What workgroup `wg` of `n_wgs` adds to ticket wg % kAttnTickets.
constexpr uint64_t attn_ticket(uint32_t wg, uint32_t n_wgs) {
  return wg < kAttnTickets ? kAttnEpoch - (n_wgs - 1 - wg) / kAttnTickets : 1;
}
constexpr uint64_t attn_epoch(uint64_t ticket) { return ticket & ~(kAttnEpoch - 1); }
// Whether a counter that stood at `before` has its last piece now.
constexpr bool attn_is_last(uint64_t before, uint32_t n_pieces) { return (before & (kAttnEpoch - 1)) == n_pieces - 1; }

// Partial sums are given 256 MiB at most.
constexpr size_t kAttnRegionFloats = size_t(1) << 26;

// Elements of a head as the tiles hold it.
inline uint32_t attn_padded_dim(uint32_t head_dim) { return head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256); }

// Chunks that a row tile's keys are cut into at most: each at least four
// 64-key tiles.
inline size_t attn_most_chunks(size_t keys) {
  const size_t n = (keys + 63) / 64 / 4;
  return n < 1 ? 1 : (n > 64 ? 64 : n);
}

// Floats that a call reserves for partial sums.  A call that is no larger than
// an earlier one in any size must not make the workspace grow (a captured graph
// holds its address), while the number of chunks goes up and down with the
// sizes: so what is reserved grows with every size, and attn_plan keeps within
// it.  Sizes are the sequences, tokens, kv heads, query heads of each, head_dim
// and both lengths.  Up to 16 rows a sequence (decode): what the 16- and 32-row
// kernels' workgroups leave, at most two pieces each (attn_plan's n_wgs; 17 MB
// on 256 CUs).  Above: as many chunks as the keys allow, up to the region.
inline size_t attn_reserve(size_t n_seqs, size_t n_tokens, uint32_t group, uint32_t n_kv_heads, uint32_t head_dim,
                           size_t max_q_len, size_t max_kv_len, int cus) {
  const size_t small = 2 * 8 * 16 * (64 + 2) * (size_t)cus;  // of all their shapes
  if (max_q_len * group <= 16) return small;
  const size_t n = attn_most_chunks(max_kv_len);
  if (n == 1) return small;
  const size_t units = (n_tokens * group + 127) / 128 + n_seqs;
  const size_t most = units * n_kv_heads * n * 128 * (attn_padded_dim(head_dim) + 2);
  const size_t cap = most < kAttnRegionFloats ? most : kAttnRegionFloats;
  return cap < small ? small : cap;
}

// The plan of a call whose partial sums may take `floats`.  With none it is
// 128-row tiles in one chunk, which every call can be.
inline AttnPlan attn_plan(size_t n_seqs, size_t n_tokens, uint32_t group, uint32_t n_kv_heads, uint32_t head_dim,
                          size_t max_q_len, size_t max_kv_len, size_t table_keys, uint32_t window, int cus,
                          size_t floats) {
  AttnPlan a{};
  // Up to 16 rows a sequence: tiles of 16.  17 to 32 (a few tokens, or groups of
  // more than 16 heads): 128-row tiles where there are units enough to give the
  // CUs two workgroups (64 sequences of 8 x 4 rows, 500 - 2000 keys, 8 kv heads of
  // 128: 68 us, tiles of 32 95 us; 16 of 2000 - 6000: 73 and 60 us); two tiles of
  // 16 where there is little to read (1 of 4000: 17 us, 32 23 us; 8 of 4000 - 8000:
  // 66 and 52 us) and for heads of 256, whose 32 rows would not fit the registers
  // (8 of 4000 - 8000: 75 and 86 us).  Above, tiles of 128 (8 x 48 rows: 46 us, 32
  // 75 us).
  const uint64_t pairs = (uint64_t)n_seqs * n_kv_heads;
  a.rows = 128;
  if (max_q_len * group <= 16) a.rows = 16;
  else if (max_q_len * group <= 32 && pairs < (uint64_t)cus)
    a.rows = head_dim > 128 || pairs * max_kv_len < 1024ull * cus ? 16 : 32;
  // 16- and 32-row tiles count their granules of 128 keys in 32 bits.
  const uint64_t small_tiles = (n_tokens * group / 16 + n_seqs) * (uint64_t)n_kv_heads;
  if (small_tiles * (table_keys / 128 + 2) >= (1ull << 31)) a.rows = 128;
  if (a.rows <= 32) {
    // Long stretches of few units: the widest workgroups, as many as the CUs
    // hold at once.  Many short units: as many waves, each a workgroup of its
    // own, so that one's piece ends while the others' keys stream (512
    // sequences of 60 - 300 keys: 135 us wide, 98 us narrow; 8 of 1000: 11 us
    // wide, 16 us narrow).  Heads of 256 fill the LDS with two waves.
    const bool narrow = head_dim <= 128 && pairs >= 4ull * cus;
    a.waves = narrow ? 1 : (head_dim <= 128 ? 4 : 2);
    a.n_wgs = (uint32_t)cus * (narrow ? 4 : 1) * (head_dim <= 64 ? 2 : 1);
    a.min_granules = 1;
    a.part_o_floats = 2 * (size_t)a.n_wgs * a.rows * head_dim;
    a.part_ml_floats = 2 * (size_t)a.n_wgs * a.rows * 2;
    // (a launch takes every ticket and counts up to kAttnEpoch at most)
    if (a.part_o_floats + a.part_ml_floats <= floats && a.n_wgs >= kAttnTickets && a.n_wgs < kAttnEpoch / 2) return a;
    a = AttnPlan{};
    a.rows = 128;
  }
  a.n_units = (uint32_t)((n_tokens * group + a.rows - 1) / a.rows + n_seqs);
  // keys of a row tile, from a whole key tile's start on
  size_t max_keys = max_kv_len;
  const size_t reach = (size_t)window + (a.rows + group - 1) / group + 64;
  if (window && reach < max_keys) max_keys = reach;
  // How many chunks a row tile's keys are cut into, by the time of the busiest
  // CU in units of a 64-key tile at full rate.  A CU holds `resident`
  // workgroups; alone, one runs at 0.72 of the rate that they reach together
  // (two of 128-element heads; 1.02 against 0.74 PFLOP/s).  Rows of a prompt
  // see half its keys on average, longest first, which fills the rounds by
  // itself (`uneven`).  Only the longest sequence is known: of several, the
  // others are taken to be shorter (`ragged`) and to fill the rounds by half.
  // kStart, kSplit, kJoin: a workgroup's start, its partial sums, the join.
  // Measured, two sequences of 520 rows x 8 over 28000 keys: 1 chunk 794 us, 2 532
  // us, 3 642 us, 4 538 us, 5 599 us, 8 558 us, 16 606 us; 512 tokens over 8000 keys:
  // 1 193 us, 2 119 us, 4 83 us, 5 110 us, 8 94 us; three prompts of 500 - 900
  // tokens: 1 32 us, 2 46 us.
  const double resident = head_dim <= 64 ? 3 : (head_dim <= 128 ? 2 : 1), alone = resident > 1 ? 0.72 : 1.0;
  const double kStart = 1.0, kSplit = 1.5, kJoin = 9.0;
  const double ragged = n_seqs > 1 ? 0.9 : 1.0;
  const double units = ((double)(n_tokens * group) / a.rows + 0.5 * (double)(n_seqs - 1)) * n_kv_heads;
  const double longest = (double)(max_keys + 63) / 64, spread = (double)(max_q_len < max_keys ? max_q_len : max_keys) / 64;
  const double mean = window ? longest : longest - spread / 2, even = mean * units * ragged / cus;
  double uneven = longest > 0 ? 2 * (longest - mean) / longest : 0;
  uneven = n_seqs > 1 && uneven < 0.5 ? 0.5 : uneven;
  const size_t base = (size_t)a.n_units * n_kv_heads, row_floats = attn_padded_dim(head_dim) + 2;
  const size_t most = attn_most_chunks(max_keys);
  double best = 0;
  a.n_chunks = 1;
  for (size_t n = 1; n <= most && (n == 1 || (base * n <= 16 * resident * cus && base * n * a.rows * row_floats <= floats)); ++n) {
    const double per_cu = ceil(units) * n / cus, k = ceil(per_cu * ragged), len = mean / n;
    const double last = k - floor(k / resident) * resident;  // workgroups of the last round
    const double whole = (k - last + (last == 1 ? 1 / alone : last)) * len;
    // the longest workgroup beside as many as share its CU
    const double beside = fmin(fmax(per_cu, 1.0), resident), rate = alone + (1 - alone) * fmin(beside - 1, 1.0);
    const double smooth = fmax(longest / n * beside / rate, even);
    const double est = smooth + fmax(whole - smooth, 0.0) * (1 - uneven) + per_cu * kStart + (n > 1 ? per_cu * kSplit + kJoin : 0);
    if (n == 1 || est < best) {
      best = est;
      a.n_chunks = (uint32_t)n;
    }
  }
  a.chunk = (uint32_t)(((max_keys + a.n_chunks - 1) / a.n_chunks + 63) / 64 * 64);
  a.chunk = a.chunk ? a.chunk : 64;
  a.n_wgs = (uint32_t)(base * a.n_chunks < UINT32_MAX ? base * a.n_chunks : UINT32_MAX);
  if (a.n_chunks > 1) {
    const size_t rows = (size_t)a.n_wgs * a.rows;
    a.part_o_floats = rows * attn_padded_dim(head_dim);
    a.part_ml_floats = rows * 2;
  }
  return a;
}

}  // namespace mer
