// mer_attention.hpp -- arguments of the attention-side kernels (q/k norm and
// rotation, paged append, paged attention) and their launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "mer_attention_plan.hpp"

namespace mer {

// Element types, by their UTH dtype ids.
enum FloatType : int { kF32 = 0, kF16 = 1, kBF16 = 6 };

constexpr uint32_t kMaxHeadDim = 256;

// One of q / k / v on its way through norm and rotation.
struct RopeTensor {
  const void *in;    // [n_tokens] rows of `heads` heads, in_stride elements apart
  void *out;         // the same, out_stride elements apart (norm_rope)
  const float *norm; // [head_dim] weights, or null
  uint64_t in_stride, out_stride;
  uint32_t heads;
};

struct NormRopeParams {
  RopeTensor t[2];           // q and k
  const int32_t *positions;  // [n_tokens], or null without rotation
  const float *inv_freq;     // [rot / 2]
  uint32_t n_tokens, head_dim, rot, interleaved;
  float eps, inv_dim;
  // append: where the rows go
  const int64_t *slots;      // [n_tokens]; negative = no row
  uint64_t n_slots;          // n_pages * page_size
  uint32_t page_shift;
  uint32_t heads_per_wave;   // consecutive heads that one wave walks
  uint32_t *status;
};

hipError_t launch_norm_rope(int in_type, int out_type, const NormRopeParams &p, int cus, hipStream_t st);
hipError_t launch_kv_append(int in_type, int cache_type, const NormRopeParams &p, int cus, hipStream_t st);

struct AttnParams {
  const void *k, *v;         // [n_pages][n_kv_heads][page_size][head_dim]
  const void *q;
  void *out;
  const int32_t *table;      // [n_seqs][table_stride]
  const int32_t *q_start;    // [n_seqs + 1]
  const int32_t *kv_len;     // [n_seqs]
  const float *sinks;        // [n_heads], or null
  uint64_t q_stride, out_stride;
  uint32_t table_stride, n_seqs, n_tokens;
  uint32_t n_pages, page_shift, n_kv_heads, head_dim, group;
  uint32_t group_mul, group_shift, heads_mul, heads_shift;  // reciprocals (set_reciprocals)
  uint32_t window;           // 0 = none
  float scale_log2;          // scale * log2(e)
  // decomposition (attn_plan)
  uint32_t min_granules;     // 16-row tiles: least granules of a workgroup
  uint32_t n_units;          // 128-row tiles of a kv head (an upper bound)
  uint32_t chunk, n_chunks;  // 128-row tiles: keys of one workgroup, workgroups of one row tile
  float *part_o;             // partial sums [slot][rows][head_dim]
  float *part_ml;            // their maxima and weights [slot][rows][2]
  uint64_t *counters;        // tickets, then finished pieces of a unit (mer_attention_plan.hpp)
  uint32_t *status;
};

// The cache held in 4 bits: k and v of AttnParams are codes
// [n_pages][n_kv_heads][page_size][head_dim / 2], their blocks' scales f16
// [n_pages][n_kv_heads][head_dim / 32][page_size].
constexpr uint32_t kQ4Block = 32;
struct AttnQ4Params : AttnParams {
  const void *k_scales, *v_scales;
};

// A cache's two planes of keys and of values.
struct CacheQ4 {
  uint8_t *codes[2];
  uint16_t *scales[2];
  uint64_t n_slots;          // n_pages * page_size
  uint32_t page_shift, heads, head_dim;
};
struct AppendQ4Params {
  CacheQ4 cache;
  const void *in[2];         // k and v: [n_tokens] rows of heads, in_stride elements apart
  uint64_t in_stride[2];
  const float *norm;         // [head_dim] of the keys, or null
  const int32_t *positions;  // [n_tokens], or null without rotation
  const float *inv_freq;     // [rot / 2]
  const int64_t *slots;      // [n_tokens]; negative = no row
  uint32_t n_tokens, rot, interleaved;
  uint32_t heads_per_wave;   // consecutive heads that one wave walks
  float eps;
  double inv_dim;
  uint32_t *status;
};
struct ReadQ4Params {
  CacheQ4 cache;
  const int64_t *slots;      // [n_rows]; negative = a row of zeros
  void *out[2];              // k and v, out_stride elements apart
  uint64_t out_stride[2];
  uint32_t n_rows;
  uint32_t *status;
};
hipError_t launch_append_q4(int in_type, const AppendQ4Params &p, int cus, hipStream_t st);
hipError_t launch_read_q4(int out_type, const ReadQ4Params &p, int cus, hipStream_t st);

void set_reciprocals(AttnParams *p);
hipError_t launch_attention(int type, const AttnPlan &plan, const AttnParams &p, hipStream_t st);
hipError_t launch_attention_q4(int type, const AttnPlan &plan, const AttnQ4Params &p, hipStream_t st);

}  // namespace mer
