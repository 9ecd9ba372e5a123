// mer_attention.hip -- attention of a chunk of new tokens over a paged cache.
//
// Row i of a sequence's n new tokens sits at position p = kv_len - n + i and
// sees the keys j <= p (and j > p - window):
//   o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) [+ exp(sink - m)]),
//   s_j = scale * q . k_j, m the running maximum.
// One pass over the keys: each tile's scores raise m, the sums so far are
// scaled by exp(m_old - m_new).
//
// The heads of a group share their kv head's keys, so a tile's rows are
// (token, head in group) pairs: row r = token r / group, head r % group.
//
// Products run on MFMA with the keys as the rows of the first one: S^T = K Q^T
// puts a q row into one lane column, so the softmax statistics are one value
// per lane, and the lane's own scores are, in an order of keys that V^T's
// operand repeats, what O^T = V^T P^T reads as its second operand: P never
// leaves the registers.  P is rounded to the cache's type for that product
// (half a step of a weight <= 1; its sum is kept from the f32 values).
#include "mer_attention_device.hpp"

#include <math.h>

namespace mer {
namespace {

// What a lane reads for a key outside the tile's range: rows of zeros.
__device__ u4 g_zero_row[kMaxHeadDim * 2 / 16];

// Geometry of a head row in LDS: DP elements (head_dim rounded up), in 16-byte
// pieces whose places are permuted by the row so that neither the row-wise
// reads of K nor the transposed reads of V pile up on a bank.
template <int DP>
struct RowLayout {
  static constexpr int kPieces = DP * 2 / 16;       // of a row
  static constexpr int kRowsPerLoad = 64 / kPieces; // rows of one asynchronous copy
  static constexpr int kKOffs = 16 / kRowsPerLoad;  // copies after which K's permutation repeats (V's: 8 rows)
  // K: 16 or 32 lanes read one piece of as many rows.
  static __device__ __forceinline__ uint32_t k_swizzle(uint32_t row) {
    return DP == 64 ? (row >> 1) & 7 : row & 15;
  }
  // V: a transposed read takes 32 bytes of each of four rows (x 4 groups).
  static __device__ __forceinline__ uint32_t v_swizzle(uint32_t row) {
    return DP == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
  }
};

// Asynchronous copies of a wave's share of a tile, SHARE keys from a multiple
// of 8 on: the pages of its 8-key groups are looked up a tile ahead, so that
// the lookups are off the copies' path.
// PAD: head_dim < DP.
template <int DP, int SHARE, bool PAD>
struct Share {
  typedef RowLayout<DP> L;
  static constexpr int kGroups = SHARE / 8;
  static constexpr int kLoads = SHARE / L::kRowsPerLoad;  // copies of K, and of V
  static constexpr int kPerGroup = 8 / L::kRowsPerLoad;   // copies of an 8-key group
  static constexpr int kOffs = L::kKOffs > kPerGroup ? L::kKOffs : kPerGroup;

  const uint8_t *k, *v;  // of this head in page 0
  uint32_t page_bytes, row_bytes, page_shift, n_pages;
  const int32_t *table;
  int32_t lo, hi;        // keys to copy; others, and those of unknown pages, read zeros
  int32_t key0, next_key;
  uint64_t off[kGroups]; // of a group's first row
  int32_t next_id[kGroups];
  uint32_t known;        // groups of pages that the cache has, a bit each
  bool whole;
  uint32_t koff[kOffs], voff[kPerGroup];  // a lane's piece, from its group's first row (kNone: beyond the head)

  __device__ __forceinline__ void init(const AttnParams &p, const int32_t *seq_table, uint32_t head, const Tile &t) {
    row_bytes = p.head_dim * 2;
    page_shift = p.page_shift;
    page_bytes = (p.n_kv_heads << page_shift) * row_bytes;
    n_pages = p.n_pages;
    k = (const uint8_t *)p.k + (uint64_t)(head << page_shift) * row_bytes;
    v = (const uint8_t *)p.v + (uint64_t)(head << page_shift) * row_bytes;
    table = seq_table;
    lo = t.lo;
    hi = t.hi;
    const uint32_t lane = lane_id(), sub = lane / L::kPieces, piece = lane % L::kPieces;
    // Pieces beyond the head dimension: K's are not copied and stay zero
    // (clear_pads), since they meet q's zeros in the score, where an infinity
    // would give a NaN; V's repeat the first one, and what they add up to is not
    // used.  (K's as copies of a row of zeros: 64 decoding sequences of 200 - 8000
    // keys, 8 kv heads of 192, 366 us instead of 332, prompts of 4096 401 instead
    // of 373.)
    auto at = [&](uint32_t row, uint32_t lg, uint32_t none) { return lg * 8 < p.head_dim ? row % 8 * row_bytes + lg * 16 : none; };
#pragma unroll
    for (uint32_t j = 0; j < kOffs; ++j) {
      const uint32_t row = j * L::kRowsPerLoad + sub;
      koff[j] = at(row, piece ^ L::k_swizzle(row), kNone);
    }
#pragma unroll
    for (uint32_t j = 0; j < kPerGroup; ++j) {
      const uint32_t row = j * L::kRowsPerLoad + sub;
      voff[j] = at(row, piece ^ L::v_swizzle(row), row % 8 * row_bytes);
    }
  }

  // Any key will do: page places are cut to those of [lo, hi), which is not empty.
  __device__ __forceinline__ void lookup(int32_t key) {
    next_key = key;
    const int32_t first = lo >> page_shift, last = (hi - 1) >> page_shift;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      int32_t pg = (key + g * 8) >> page_shift;
      pg = pg > last ? last : (pg < first ? first : pg);
      next_id[g] = sload(table, (uint32_t)pg);
    }
  }

  // On to the share last looked up, before its copies.
  __device__ __forceinline__ void advance(uint32_t *status) {
    key0 = next_key;
    const uint32_t mask = (1u << page_shift) - 1;
    known = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      off[g] = (uint64_t)(uint32_t)next_id[g] * page_bytes + ((uint32_t)(key0 + g * 8) & mask) * row_bytes;
      known |= (uint32_t)next_id[g] < n_pages ? 1u << g : 0u;
    }
    whole = key0 >= lo && key0 + SHARE <= hi && known == (1u << kGroups) - 1;
    if (known != (1u << kGroups) - 1 && lane_id() < kGroups) {
      const int32_t k0 = key0 + (int32_t)lane_id() * 8;
      if (!(known >> lane_id() & 1) && k0 < hi && k0 + 8 > lo) atomicCAS(status, 0u, 16u /* MER_ERR_RESIDENCY_MISS */);
    }
  }

  // Zeros where the copies of K to `lds` leave gaps.
  __device__ __forceinline__ void clear_pads(uint32_t lds) const {
    if (!PAD) return;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      if (koff[j % kOffs] == kNone)
        *(__attribute__((address_space(3))) u4 *)(uintptr_t)(lds + j * 1024u + lane_id() * 16) = u4{0, 0, 0, 0};
  }

  template <bool V>
  __device__ __forceinline__ void copy(uint32_t lds) const {
    const uint8_t *base = V ? v : k;
    if (whole && (V || !PAD)) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < kPerGroup; ++i) {
          const int j = g * kPerGroup + i;
          async_row16(base + off[g], V ? voff[i] : koff[j % kOffs], lds + j * 1024u);
        }
    } else if (whole) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < kPerGroup; ++i) {
          const int j = g * kPerGroup + i;
          async_row16_some(base + off[g], koff[j % kOffs], lds + j * 1024u);
        }
    } else {
      const uint32_t sub = lane_id() / L::kPieces;
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < kPerGroup; ++i) {
          const int j = g * kPerGroup + i;
          const int32_t key = key0 + j * L::kRowsPerLoad + (int32_t)sub;
          const bool in = (known >> g & 1) && key >= lo && key < hi;
          if (V || !PAD || koff[j % kOffs] != kNone)
            async_row16(in ? base + off[g] + (V ? voff[i] : koff[j % kOffs]) : (const uint8_t *)g_zero_row, lds + j * 1024u);
        }
    }
  }
};

// ---- values that are not finite ----
// An infinity or a NaN reaches the rows that see its key, whatever their weight
// of it, and no others; but in the products it meets weights of zero, of keys
// that a row does not see or that rounded to it, and makes a NaN.  So sums that
// are not finite are made once more with care: a tile's values are looked over,
// three products find the rows that see a NaN, +inf or -inf, which a mark notes
// for the end, and these values are cleared from the tile.  (Looking over the
// tiles that rows see in part, every time, cost prompts 1 - 2% and a window of
// 1024 with heads of 64 5%.)
// Marks are two bits an element: +inf, -inf, both for a NaN.
// Whether one of the values of [at, at + 64 * BYTES) of LDS is not finite.
template <class E, int BYTES>
__device__ __forceinline__ bool not_finite(uint32_t at) {
  constexpr uint32_t kMask = E::kExponent * 0x10001u, kCarry = (0x8000u - E::kExponent) * 0x10001u;
  uint32_t found = 0;
#pragma unroll 1
  for (int i = 0; i < BYTES / 16; ++i) {
    const u4 x = *(const __attribute__((address_space(3))) u4 *)(uintptr_t)(at + (i * 64 + lane_id()) * 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) found |= (x[k] & kMask) + kCarry;  // an exponent of ones carries into the sign's place
  }
  return __builtin_amdgcn_ballot_w64(found & 0x80008000u) != 0;
}
template <class E, int BYTES>
__device__ __forceinline__ void clear_not_finite(uint32_t at) {
#pragma unroll 1
  for (int i = 0; i < BYTES / 2; ++i) {
    __attribute__((address_space(3))) uint16_t *x =
        (__attribute__((address_space(3))) uint16_t *)(uintptr_t)(at + (i * 64 + lane_id()) * 2);
    if ((*x & E::kExponent) == E::kExponent) *x = 0;
  }
}
// Ones where there is a NaN, +inf or -inf (kind 0, 1, 2), else zeros.
template <class E>
__device__ __forceinline__ typename E::V8 where(typename E::V8 v, uint32_t kind) {
  u4 x = __builtin_bit_cast(u4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t word = 0;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      const uint32_t b = x[i] >> h & 0xffffu, a = b & 0x7fffu;
      const bool is = kind == 0 ? a > E::kExponent : b == (E::kExponent | (kind - 1) << 15);
      word |= (is ? E::kOne : 0u) << h;
    }
    x[i] = word;
  }
  return __builtin_bit_cast(typename E::V8, x);
}
// A lane's part of the weights, with one for each key that its row sees:
// element e's key is `first` + e / 4 * STEP + e % 4.
template <class E, int STEP>
__device__ __forceinline__ typename E::V8 ones(int32_t first, int32_t last, int32_t before) {
  u4 x;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const int32_t a = first + e / 4 * STEP + e % 4, b = a + 1;
    x[e / 2] = (a <= last && a > before ? E::kOne : 0u) | (b <= last && b > before ? E::kOne << 16 : 0u);
  }
  return __builtin_bit_cast(typename E::V8, x);
}
// The marks of N elements that x keys of that kind reach.
template <int N, class V>
__device__ __forceinline__ uint32_t mark(V x, uint32_t kind) {
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) bits |= x[e] > 0.0f ? 1u << 2 * e : 0u;
  return bits * (kind == 0 ? 3 : kind);
}
__device__ __forceinline__ float add_mark(float o, uint32_t bits) {
  o += bits & 1 ? __builtin_inff() : 0.0f;
  return o + (bits & 2 ? -__builtin_inff() : 0.0f);
}

// Sixteen rows: decode and short chunks.
//
// The work is cut into pieces of equal length whatever the sequences are: a
// granule is kGranule keys of one (row tile, kv head), the granules of all
// sequences stand in a row (sequence by sequence, unit by unit), and each
// workgroup takes an equal stretch of them.  A unit that a stretch's end cuts
// is joined from its pieces.  Nothing of this depends on the host's knowing
// the lengths.
//
// The waves of a workgroup take a piece's tiles of 32 keys in turn, each with
// a ring of LDS of its own (no barriers while the keys stream), and join
// their sums at the piece's end.
//
// Bound by the memory: every wave has two tiles of K and V on the way, 128 KiB
// a CU for heads of 128.  64 sequences of 200 - 8000 keys, 32 / 8 heads, bf16:
// 203 us (5.1 TB/s); one of 131,000 keys, f16: 97 us (5.5 TB/s; plain reads
// reach 5.9).  A single short one is bound by latency (700 keys: 11 us).
template <int DP, int WAVES, int NR>
struct Rows16 {
  static constexpr int kWaves = WAVES;
  static constexpr int kRows = 16 * NR;
  static constexpr int kKeys = 32;
  static constexpr int kGranule = 128;
  static constexpr int kTileBytes = kKeys * DP * 2;  // K or V of a tile
  static constexpr int kStages = 2;
  static constexpr int kLoads = Share<DP, kKeys, false>::kLoads;
  static constexpr int kLds = kWaves * kStages * 2 * kTileBytes;
};

template <class E, int DP, int WAVES, int NR, bool PAD>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(1, DP == 64 ? 2 : 1))) void attn_rows16_kernel(AttnParams p) {
  typedef Rows16<DP, WAVES, NR> C;
  typedef RowLayout<DP> L;
  typedef typename E::V8 V8;
  typedef typename E::T T;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = uni(tid / 64);
  const uint32_t col = lane % 16, quad = lane / 16;

  // where a lane reads its operands, from a tile's start
  uint32_t k_lane[DP / 32], v_lane[DP / 16];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) k_lane[d] = col * (DP * 2) + ((d * 4 + quad) ^ L::k_swizzle(col)) * 16;
  auto v_at = [&](uint32_t d) {
    const uint32_t r = quad * 4 + col / 4;
    return r * (DP * 2) + ((d * 2 + col % 4 / 2) ^ L::v_swizzle(r)) * 16 + col % 2 * 8;
  };
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) v_lane[d] = v_at(d);

  uint64_t epoch = 0;  // in thread 0
  if (tid == 0)
    epoch = attn_epoch(__hip_atomic_fetch_add(p.counters + blockIdx.x % kAttnTickets * kAttnTicketWords,
                                              attn_ticket(blockIdx.x, gridDim.x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));

  typedef Granules<32> G;
  G gr;
  gr.base = 0;
  gr.view<C::kGranule, C::kRows>(p, 0);
  uint32_t all = gr.total;
  if (p.n_seqs > 256) {
    for (uint32_t s = 256; s < p.n_seqs; s += 256) {
      gr.view<C::kGranule, C::kRows>(p, s);
      all += gr.total;
    }
    gr.view<C::kGranule, C::kRows>(p, 0);
  }
  uint32_t per = uni((all + gridDim.x - 1) / gridDim.x);
  per = per < p.min_granules ? p.min_granules : per;
  uint32_t x = blockIdx.x * per;
  const uint32_t x1 = all - (all < x ? all : x) < per ? all : x + per;
  bool first_piece = true;
  while (x < x1) {
    uint32_t seq, before;
    Span span;
    if (!gr.find<C::kGranule, C::kRows>(p, x, &seq, &before, &span)) return;
    int32_t start = 0;
    const uint32_t n_gran = uni(G::granules<C::kGranule>(p, span, &start));
    const uint32_t unit = uni((x - before) / n_gran), tile = uni(by_heads(p, unit)), head = unit - tile * p.n_kv_heads;
    const uint32_t unit0 = before + unit * n_gran, g0 = x - unit0;
    const uint32_t count = n_gran - g0 < x1 - x ? n_gran - g0 : x1 - x;
    // the unit's pieces: workgroups first_wg .. first_wg + n_pieces - 1
    const uint32_t first_wg = g0 == 0 ? blockIdx.x : (per == 1 ? unit0 : uni(unit0 / per));
    const uint32_t last_wg = g0 + count == n_gran ? blockIdx.x : (per == 1 ? unit0 + n_gran - 1 : uni((unit0 + n_gran - 1) / per));
    const uint32_t n_pieces = last_wg - first_wg + 1;
    const uint32_t first_slot = 2 * first_wg + (first_wg * per == unit0 ? 0 : 1);
    const uint32_t my_slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
    first_piece = false;
    x += count;
    Tile t;
    // (spans that overlap, past 2^32, or lengths that change under the kernel)
    if (!make_tile<C::kRows>(p, span, tile, &t) || head >= p.n_kv_heads || last_wg >= gridDim.x) return;
    start = (int32_t)uni((uint32_t)start);
    int32_t begin = start + (int32_t)(g0 * C::kGranule), end = begin + (int32_t)(count * C::kGranule);
    if (p.window && begin < (t.lo & ~31)) begin = t.lo & ~31;
    end = end < t.hi ? end : t.hi;

    // Q^T: lane column = a row of each group of 16, 8 consecutive dims per 32-dim slab
    const int32_t window = p.window ? (int32_t)p.window : 0x40000000;
    V8 q[NR][DP / 32];
    int32_t pos[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const uint32_t row = t.row0 + n * 16 + col, tok = by_group(p, row), hd = head * p.group + row - tok * p.group;
      pos[n] = t.pos0 + (int32_t)tok;
      const T *qp = (const T *)p.q + (uint64_t)(t.tok0 + tok) * p.q_stride + (uint64_t)hd * p.head_dim;
#pragma unroll
      for (int s = 0; s < DP / 32; ++s) {
        const uint32_t d = s * 32 + quad * 8;
        q[n][s] = V8{};
        if (row < t.n_rows && d < p.head_dim) q[n][s] = *(const V8 *)(qp + d);
      }
    }
    const uint32_t last = t.row0 + C::kRows - 1 < t.n_rows ? t.row0 + C::kRows - 1 : t.n_rows - 1;
    const int32_t pos_first = t.pos0 + (int32_t)by_group(p, t.row0), pos_last = t.pos0 + (int32_t)by_group(p, last);

    const int32_t n_tiles = end > begin ? (end - begin + C::kKeys - 1) / C::kKeys : 0;
    const int32_t mine = n_tiles > (int32_t)wave ? (n_tiles - (int32_t)wave + C::kWaves - 1) / C::kWaves : 0;
    const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem +
                          wave * (C::kStages * 2 * C::kTileBytes);
    auto key_of = [&](int32_t i) { return begin + (i * C::kWaves + (int32_t)wave) * C::kKeys; };
    auto slot_of = [&](int32_t i) { return ring + (uint32_t)(i & 1) * (2 * C::kTileBytes); };
    __syncthreads();  // the last piece is done with the LDS
    Share<DP, C::kKeys, PAD> sh;
    sh.init(p, p.table + (uint64_t)seq * p.table_stride, head, t);
    if (mine > 0) sh.lookup(key_of(0));
    for (int32_t i = 0; i < C::kStages; ++i) sh.clear_pads(slot_of(i));
    // q has to be there before the first copy goes out: a later wait for it,
    // which the compiler would put into the loop, would drain the copies.
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    float m[NR], l[NR];
    f4 o[NR][DP / 16];
    uint32_t marks[NR][DP / 64] = {};
    for (bool careful = false;; careful = true) {
      if (careful) sh.lookup(key_of(0));
      for (int32_t i = 0; i < C::kStages && i < mine; ++i) {
        sh.advance(p.status);
        sh.lookup(key_of(i + 1));
        sh.template copy<false>(slot_of(i));
        sh.template copy<true>(slot_of(i) + C::kTileBytes);
      }

#pragma unroll
      for (int n = 0; n < NR; ++n) {
        m[n] = -__builtin_inff();
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[n][d] = f4{0, 0, 0, 0};
      }
      for (int32_t i = 0; i < mine; ++i) {
        const int32_t left = mine - i;
        const int32_t key0 = key_of(i);
        const uint32_t kb = slot_of(i), vb = kb + C::kTileBytes;
        if (left == 1) wait_vm<C::kLoads>();
        else wait_vm<3 * C::kLoads>();
        f4 s[NR][2];
        V8 k[2][DP / 32];
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            k[b][d] = *(const __attribute__((address_space(3))) V8 *)(uintptr_t)(kb + k_lane[d] + b * 16 * (DP * 2));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          s[n][0] = s[n][1] = f4{0, 0, 0, 0};
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int b = 0; b < 2; ++b) s[n][b] = E::mfma16(k[b][d], q[n][d], s[n][b]);
        }
        wait_lds();
        if (left > C::kStages) {
          sh.advance(p.status);
          sh.lookup(key_of(i + C::kStages + 1));
          sh.template copy<false>(kb);
        }
        const int32_t key_end = key0 + C::kKeys;
        const bool partial = key_end > pos_first + 1 || key_end > t.hi || key0 <= pos_last - window;
        V8 pr[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          // scores in base 2; keys of lane: b * 16 + quad * 4 + e
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = s[n][e / 4][e % 4] * p.scale_log2;
          if (partial) {
            const int32_t last_key = pos[n] - key0 - (int32_t)quad * 4, before = last_key - window;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int32_t at = (e / 4) * 16 + e % 4;
              x[e] = at > last_key || at <= before ? -__builtin_inff() : x[e];
            }
          }
          float mx = x[0];
#pragma unroll
          for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
          mx = fmaxf(max_quad(mx), m[n]);
          const float mu = mx == -__builtin_inff() ? 0.0f : mx;
          const float a = __builtin_amdgcn_exp2f(m[n] - mu);
          f8 e8;
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            e8[e] = __builtin_amdgcn_exp2f(x[e] - (mu - E::kUp));
            sum += e8[e];
          }
          l[n] = l[n] * a + sum;
          if (__builtin_amdgcn_ballot_w64(mx != m[n])) {
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) o[n][d] *= a;
          }
          m[n] = mx;
          pr[n] = __builtin_convertvector(e8, V8);
        }
        if (left == 1) wait_vm<0>();
        else if (left == 2) wait_vm<2 * C::kLoads>();
        else wait_vm<3 * C::kLoads>();
        auto v_of = [&](uint32_t at) {
          s4 x[2];
#pragma unroll
          for (int b = 0; b < 2; ++b)
            x[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s4 *)(uintptr_t)(vb + at + b * 16 * (DP * 2)));
          return __builtin_bit_cast(V8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
        };
        if (careful && not_finite<E, C::kTileBytes / 64>(vb)) {
          // rolled up: few registers
#pragma unroll 1
          for (uint32_t i = 0; i < 3 * (DP / 16); ++i) {
            const uint32_t d = i / 3, kind = i % 3;
            const V8 v = where<E>(v_of(v_at(d)), kind);
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              const int32_t last_key = pos[n] - key0 - (int32_t)quad * 4;
              const V8 seen = ones<E, 16>(0, last_key, last_key - window);
              const uint32_t bits = mark<4>(E::mfma16(v, seen, f4{0, 0, 0, 0}), kind) << d % 4 * 8;
#pragma unroll
              for (uint32_t k = 0; k < DP / 64; ++k) marks[n][k] |= k == d / 4 ? bits : 0;
            }
          }
          wait_lds();
          clear_not_finite<E, C::kTileBytes / 64>(vb);
          wait_lds();
        }
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          const V8 v = v_of(v_lane[d]);
#pragma unroll
          for (int n = 0; n < NR; ++n) o[n][d] = E::mfma16(v, pr[n], o[n][d]);
        }
        wait_lds();
        if (left > C::kStages) sh.template copy<true>(vb);
      }
      if (careful) break;
      float z = 0.0f;
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) z += probe(o[n][d]);
      if (!not_a_number(z)) break;
    }
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        if (__builtin_amdgcn_ballot_w64(marks[n][d / 4])) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][d][e] = add_mark(o[n][d][e], marks[n][d / 4] >> (d % 4 * 8 + e * 2));
        }
    // join the waves: m, l and O of each in LDS
    __syncthreads();
    float *jo = (float *)smem;                      // [wave][row][DP]
    float *jm = jo + C::kWaves * C::kRows * DP;     // [wave][row][2]
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const uint32_t at = wave * C::kRows + n * 16 + col;
      l[n] = sum_quad(l[n]);
      if (quad == 0) *(f2 *)&jm[at * 2] = f2{m[n], l[n]};
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) *(f4 *)&jo[at * DP + d * 16 + quad * 4] = o[n][d];
    }
    __syncthreads();
    const Piece piece = {first_wg, n_pieces, first_slot, my_slot, epoch};
    join_waves<E, DP, C::kWaves, C::kRows>(p, t, head, piece, jo, jm);
    if (n_pieces > 1) finish_piece<E, DP, C::kWaves, C::kRows>(p, t, head, piece, jo, (uint32_t *)(jm + C::kWaves * C::kRows * 2));
  }
}

// 32 rows a wave: prompts and larger chunks.  The waves of a workgroup share
// tiles of 64 keys, two stages of K and V in LDS; each wave copies its share
// of the next tile while the present one is used.
//
// Bound by the matrix and the vector units, which overlap but in part: a wave's
// last products run beside its weights, its first ones only beside the other
// workgroup that a CU holds of 128-element heads.  They are busy 47% and 50% of
// the cycles over a prompt of 8192 tokens, 41% and 46% of 4096, heads of 64 42%
// and 74%, of 256 17% and 24%.  32 rows a wave read each operand from LDS half as often as 16 would;
// 64-key tiles leave 64 KiB for each of the two workgroups.  A 4096-token
// prompt, 32 / 8 heads of 128, bf16: 150 us (917 TFLOP/s); 16384 tokens: 1.0
// PFLOP/s; 4096 tokens of 64 heads of 64, where softmax outweighs the
// products: 175 us (784 TFLOP/s); 2048 of 16 heads of 256 (one workgroup a CU):
// 84 us (408 TFLOP/s).  Padded heads do the products of the size above them:
// 4096 tokens of 80 140 us, of 96 142, of 112 145.
template <int DP, int WAVES>
struct Rows32 {
  static constexpr int kWaves = WAVES;
  static constexpr int kRows = 32 * WAVES;
  static constexpr int kKeys = 64;
  static constexpr int kTileBytes = kKeys * DP * 2;  // K or V of a tile
  static constexpr int kShare = kKeys / WAVES;       // keys that a wave copies
  static constexpr int kLoads = Share<DP, kShare, false>::kLoads;
  static constexpr int kLds = 2 * 2 * kTileBytes + 2 * WAVES * 4;  // and flags
};

template <class E, int DP, int WAVES, bool PAD>
__global__ __launch_bounds__(64 * WAVES, DP == 256 ? 1 : (DP == 64 ? 3 : 2)) void attn_rows32_kernel(AttnParams p) {
  typedef Rows32<DP, WAVES> C;
  typedef RowLayout<DP> L;
  typedef typename E::V8 V8;
  typedef typename E::T T;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lane = lane_id(), wave = uni(threadIdx.x / 64);
  const uint32_t head = blockIdx.x % p.n_kv_heads;
  const uint32_t rest = blockIdx.x / p.n_kv_heads;
  // Chunk by chunk, so that neighbours are alike (workgroups go round the
  // shader engines in a fixed order); late rows, with more keys, first.
  const uint32_t c = rest / p.n_units, unit = p.n_units - 1 - rest % p.n_units;
  uint32_t seq, tile;
  find_unit<C::kRows>(p, unit, &seq, &tile);
  Tile t;
  const Span span = make_span(p, sload(p.q_start, seq), sload(p.q_start, seq + 1), sload(p.kv_len, seq));
  if (!make_tile<C::kRows>(p, span, tile, &t)) return;
  uint32_t chunk, n_chunks;
  chunks_of<C::kKeys>(p, t, &chunk, &n_chunks);
  const int32_t start = t.lo & ~(C::kKeys - 1);
  if (c >= n_chunks) return;
  const uint32_t col = lane % 32, half = lane / 32;
  const uint32_t row = t.row0 + wave * 32 + col;
  const bool row_ok = row < t.n_rows;
  const uint32_t tok = by_group(p, row), hd = head * p.group + row - tok * p.group;
  const int32_t pos = t.pos0 + (int32_t)tok, window = p.window ? (int32_t)p.window : 0x40000000;
  // the wave's positions; a wave without rows has none (first > last)
  const uint32_t wrow = t.row0 + wave * 32, wlast = wrow + 31 < t.n_rows ? wrow + 31 : t.n_rows - 1;
  const bool any = wrow < t.n_rows;
  const int32_t pos_first = t.pos0 + (int32_t)by_group(p, wrow), pos_last = t.pos0 + (int32_t)by_group(p, wlast);
  const float scale = fabsf(p.scale_log2);

  V8 q[DP / 16];
  const T *qp = (const T *)p.q + (uint64_t)(t.tok0 + tok) * p.q_stride + (uint64_t)hd * p.head_dim;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const uint32_t d = s * 16 + half * 8;
    q[s] = V8{};
    if (row_ok && d < p.head_dim) q[s] = *(const V8 *)(qp + d);
    if (p.scale_log2 < 0) q[s] = -q[s];
  }

  const int32_t begin = start + (int32_t)(c * chunk);
  int32_t end = begin + (int32_t)chunk;
  end = end < t.hi ? end : t.hi;
  const int32_t n_tiles = (end - begin + C::kKeys - 1) / C::kKeys;
  const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem;
  Share<DP, C::kShare, PAD> sh;
  sh.init(p, p.table + (uint64_t)seq * p.table_stride, head, t);
  const int32_t my_key = begin + (int32_t)wave * C::kShare;
  const uint32_t my_lds = wave * (C::kLoads * 1024u);
  auto stage = [&](int32_t i) { return ring + (uint32_t)(i & 1) * (2 * C::kTileBytes); };

  // a word for each stage and wave: its share of a tile has a value that is not
  // finite, and at the end one of its sums is not
  volatile uint32_t *flags = (volatile uint32_t *)(smem + 4 * C::kTileBytes);

  // Where a lane reads its operands, from a tile's start.  K: 32 keys x 16
  // dims a product.  V: 16 keys x 32 dims, 4 + 4 keys of a lane in the order
  // in which the scores lie in their lanes.
  uint32_t k_lane[DP / 16], v_lane[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) k_lane[d] = col * (DP * 2) + ((d * 2 + half) ^ L::k_swizzle(col)) * 16;
  auto v_at = [&](uint32_t d) {
    const uint32_t r = half * 4 + lane % 16 / 4;
    return r * (DP * 2) + ((d * 4 + lane / 16 % 2 * 2 + lane % 4 / 2) ^ L::v_swizzle(r)) * 16 + lane % 2 * 8;
  };
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) v_lane[d] = v_at(d);

  float m, l;
  uint32_t marks[DP / 32] = {};
  f16v o[DP / 32];
  auto all_tiles = [&](auto pass) {
    constexpr bool careful = decltype(pass)::careful;
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;

    if (n_tiles > 0) {
      sh.lookup(my_key);
      __builtin_amdgcn_s_waitcnt(kWaitVm0);  // q is there before the first copy goes out (as above)
      sh.advance(p.status);
      sh.lookup(my_key + C::kKeys);
      for (int32_t i = 0; i < 2; ++i) sh.clear_pads(stage(i) + my_lds);
      sh.template copy<false>(stage(0) + my_lds);
      sh.template copy<true>(stage(0) + C::kTileBytes + my_lds);
    }
    for (int32_t i = 0; i < n_tiles; ++i) {
      const int32_t key0 = begin + i * C::kKeys;
      const uint32_t kb = stage(i), vb = kb + C::kTileBytes;
      const bool more = i + 1 < n_tiles;
      if (careful) {
        wait_vm<0>();
        flags[(i & 1) * WAVES + wave] = not_finite<E, C::kTileBytes / WAVES / 64>(vb + my_lds);
      }
      // all waves' copies of this tile are there, and everyone is done with the
      // other stage, which the next tile's copies fill meanwhile
      wait_vm_barrier<0>();
      uint32_t flagged = 0;
      if (careful) {
#pragma unroll
        for (int w = 0; w < WAVES; ++w) flagged |= flags[(i & 1) * WAVES + w];
        flagged = uni(flagged);
      }
      if (more) {
        sh.advance(p.status);
        sh.lookup(my_key + (i + 2) * C::kKeys);
        sh.template copy<false>(stage(i + 1) + my_lds);
        sh.template copy<true>(stage(i + 1) + C::kTileBytes + my_lds);
      }
      auto v_of = [&](int ks, uint32_t at) {
        s4 x[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
          x[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s4 *)(uintptr_t)(vb + at + (ks * 16 + b * 8) * (DP * 2)));
        return __builtin_bit_cast(V8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
      };
      if (careful && flagged) {
#pragma unroll 1
        for (uint32_t i = 0; i < 3 * (DP / 32); ++i) {  // rolled up: few registers
          const uint32_t d = i / 3, kind = i % 3;
          const int32_t last = pos - key0 - (int32_t)half * 4, before = last - window;
          f16v x;
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll 1
          for (int ks = 0; ks < 4; ++ks) {
            const V8 seen = ones<E, 8>(ks * 16, last, before);
            x = E::mfma32(where<E>(v_of(ks, v_at(d)), kind), seen, x);
          }
          const uint32_t bits = mark<16>(x, kind);
#pragma unroll
          for (uint32_t k = 0; k < DP / 32; ++k) marks[k] |= k == d ? bits : 0;
        }
        __syncthreads();
        clear_not_finite<E, C::kTileBytes / WAVES / 64>(vb + my_lds);
        __syncthreads();
      }
      const bool live = any && key0 <= pos_last && key0 + C::kKeys > pos_first - window + 1;
      if (live) {
        f16v s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[b][e] = 0.0f;
        // operands are read a batch ahead of the products, so that the reads'
        // latency is paid once a batch and not once a product
        constexpr int kBatch = DP == 128 ? 8 : 4;
#pragma unroll
        for (int d0 = 0; d0 < DP / 16; d0 += kBatch) {
          V8 k[2][kBatch];
#pragma unroll
          for (int d = 0; d < kBatch; ++d)
#pragma unroll
            for (int b = 0; b < 2; ++b)
              k[b][d] = *(const __attribute__((address_space(3))) V8 *)(uintptr_t)(kb + k_lane[d0 + d] + b * 32 * (DP * 2));
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int d = 0; d < kBatch; ++d)
#pragma unroll
            for (int b = 0; b < 2; ++b) s[b] = E::mfma32(k[b][d], q[d0 + d], s[b]);
        }
        constexpr int kAhead = DP == 256 ? 1 : 2;
        V8 v[kAhead][DP / 32];
#pragma unroll
        for (int ks = 0; ks < kAhead; ++ks)
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) v[ks][d] = v_of(ks, v_lane[d]);
        __builtin_amdgcn_sched_barrier(0);
        // From here to the tile's end a wave goes before one that is at its scores,
        // whose products run beside it (4096-token prompt, against equal
        // priorities: 184 -> 158 us), and each quarter of the products beside the
        // next quarter's weights (173 -> 158 us).
        __builtin_amdgcn_s_setprio(1);
        if (key0 + C::kKeys > pos_first + 1 || key0 + C::kKeys > t.hi || key0 <= pos_last - window) {
          const int32_t last = pos - key0 - (int32_t)half * 4, before = last - window;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int32_t at = b * 32 + (e / 4) * 8 + e % 4;
              s[b][e] = at > last || at <= before ? -__builtin_inff() : s[b][e];
            }
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(fmaxf(mx, s[0][e]), s[1][e]);
        mx = fmaxf(mx, other_half(mx)) * scale;
        // The maximum in use may lag by up to 8 (weights up to 2^8): O and l
        // are scaled only when it would lag by more.
        if (__builtin_amdgcn_ballot_w64(mx > m + 8.0f)) {
          const float mn = fmaxf(m, mx);
          const float a = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= a;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) o[d] *= a;
        }
        const float mu = (m == -__builtin_inff() ? 0.0f : m) - E::kUp;
        V8 pr[4];
        float sums[2] = {0.0f, 0.0f};
        auto weights = [&](int ks) {
          f8 x;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks / 2][ks % 2 * 8 + e], scale, -mu));
            sums[e % 2] += x[e];
          }
          pr[ks] = __builtin_convertvector(x, V8);
        };
        weights(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          if (ks + 1 < 4) weights(ks + 1);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) {
            o[d] = E::mfma32(v[ks % kAhead][d], pr[ks], o[d]);
            if (ks + kAhead < 4) v[ks % kAhead][d] = v_of(ks + kAhead, v_lane[d]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        l += sums[0] + sums[1];
      }
    }
  };
  all_tiles(Pass<false>());
  float z = 0.0f;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) z += probe(o[d]);
  flags[wave] = not_a_number(z);
  __syncthreads();
  uint32_t again = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) again |= flags[w];
  __syncthreads();  // everyone has read them, and is done with the tiles
  if (uni(again)) all_tiles(Pass<true>());
  l += other_half(l);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
    if (__builtin_amdgcn_ballot_w64(marks[d])) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = add_mark(o[d][e], marks[d] >> 2 * e);
    }
  if (n_chunks == 1) {
    if (!row_ok) return;
    if (p.sinks) l += __builtin_amdgcn_exp2f(p.sinks[hd] * kLog2E - (m == -__builtin_inff() ? 0.0f : m) + E::kUp);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    T *op = (T *)p.out + (uint64_t)(t.tok0 + tok) * p.out_stride + (uint64_t)hd * p.head_dim;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t at = d * 32 + g * 8 + half * 4;
        typedef T T4 __attribute__((ext_vector_type(4)));
        const f4 x = {o[d][g * 4], o[d][g * 4 + 1], o[d][g * 4 + 2], o[d][g * 4 + 3]};
        if (at < p.head_dim) *(T4 *)(op + at) = __builtin_convertvector(weigh(x, inv, Pass<true>()), T4);
      }
  } else {
    // A partial sum lies as the accumulators do, so every store is a whole
    // kilobyte.
    const uint64_t slot = (uint64_t)(unit * p.n_kv_heads + head) * p.n_chunks + c;
    float *po = p.part_o + (slot * WAVES + wave) * (32 * DP) + lane * 4;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f4 *)(po + (d * 4 + g) * 256) = f4{o[d][g * 4], o[d][g * 4 + 1], o[d][g * 4 + 2], o[d][g * 4 + 3]};
    if (half == 0) *(f2 *)(p.part_ml + ((slot * WAVES + wave) * 32 + col) * 2) = f2{m, l};
  }
}

template <class E, int DP, int WAVES, int NR, bool PAD>
hipError_t launch16p(const AttnPlan &plan, const AttnParams &p, hipStream_t st) {
  typedef Rows16<DP, WAVES, NR> C;
  static std::atomic<uint64_t> devices{0};
  const hipError_t e = allow_lds((const void *)attn_rows16_kernel<E, DP, WAVES, NR, PAD>, C::kLds, &devices);
  if (e != hipSuccess) return e;
  attn_rows16_kernel<E, DP, WAVES, NR, PAD><<<plan.n_wgs, 64 * WAVES, C::kLds, st>>>(p);
  return hipGetLastError();
}
template <class E, int DP, int WAVES, int NR>
hipError_t launch16w(const AttnPlan &plan, const AttnParams &p, hipStream_t st) {
  return p.head_dim < DP ? launch16p<E, DP, WAVES, NR, true>(plan, p, st) : launch16p<E, DP, WAVES, NR, false>(plan, p, st);
}
template <class E, int DP>
hipError_t launch16(const AttnPlan &plan, const AttnParams &p, hipStream_t st) {
  constexpr int kWide = DP == 256 ? 2 : 4;
  const bool wide = plan.waves == kWide, narrow = plan.waves == 1 && DP < 256;
  if (plan.rows == 16 && wide) return launch16w<E, DP, kWide, 1>(plan, p, st);
  if constexpr (DP < 256) {
    if (plan.rows == 32 && wide) return launch16w<E, DP, kWide, 2>(plan, p, st);
    if (plan.rows == 16 && narrow) return launch16w<E, DP, 1, 1>(plan, p, st);
  }
  return hipErrorInvalidValue;
}

template <class E, int DP, bool PAD>
hipError_t launch32p(const AttnPlan &plan, const AttnParams &p, hipStream_t st) {
  typedef Rows32<DP, 4> C;
  static std::atomic<uint64_t> devices{0};
  const hipError_t e = allow_lds((const void *)attn_rows32_kernel<E, DP, 4, PAD>, C::kLds, &devices);
  if (e != hipSuccess) return e;
  attn_rows32_kernel<E, DP, 4, PAD><<<plan.n_wgs, 256, C::kLds, st>>>(p);
  if (plan.n_chunks > 1) attn_join_kernel<Rows32<DP, 4>, E, DP><<<plan.n_units * p.n_kv_heads * 4, 256, 0, st>>>(p);
  return hipGetLastError();
}

template <class E, int DP>
hipError_t launch32(const AttnPlan &plan, const AttnParams &p, hipStream_t st) {
  return p.head_dim < DP ? launch32p<E, DP, true>(plan, p, st) : launch32p<E, DP, false>(plan, p, st);
}

template <class E>
hipError_t launch_typed(const AttnPlan &plan, const AttnParams &p, hipStream_t st) {
  if (plan.rows == 128) {
    if (p.head_dim <= 64) return launch32<E, 64>(plan, p, st);
    if (p.head_dim <= 128) return launch32<E, 128>(plan, p, st);
    return launch32<E, 256>(plan, p, st);
  }
  if (p.head_dim <= 64) return launch16<E, 64>(plan, p, st);
  if (p.head_dim <= 128) return launch16<E, 128>(plan, p, st);
  return launch16<E, 256>(plan, p, st);
}

}  // namespace

void set_reciprocals(AttnParams *p) {
  auto set = [](uint32_t d, uint32_t *mul, uint32_t *shift) {
    uint32_t log2 = 0;
    while ((1u << log2) < d) ++log2;
    *shift = 26 + log2;
    *mul = (uint32_t)(((1ull << *shift) + d - 1) / d);
  };
  set(p->group, &p->group_mul, &p->group_shift);
  set(p->n_kv_heads, &p->heads_mul, &p->heads_shift);
}

hipError_t launch_attention(int type, const AttnPlan &plan, const AttnParams &p, hipStream_t st) {
  return type == kF16 ? launch_typed<F16>(plan, p, st) : launch_typed<BF16>(plan, p, st);
}

}  // namespace mer
