// mer_rope.hip -- per-head norm and position rotation of queries and keys,
// and the append of keys and values to a paged cache with both on the way.
//
//   y = x / sqrt(mean(x^2) + eps) * w                    (with norm weights)
//   a = position * inv_freq[i], i < rot / 2
//   (u, v) -> (u cos a - v sin a, v cos a + u sin a)     on the pairs
//     (y[i], y[i + rot / 2]), or (y[2i], y[2i + 1]) interleaved
//
// Both kernels read each element once and write it once.  A lane holds eight
// elements of a head row as two groups of four, chosen so that it has both
// halves of its pairs: {4j.., rot/2 + 4j..} by halves, {8j.., 8j + 4..}
// interleaved and beyond the rotated part.  In each layout its pairs are those
// of the frequencies 4j .. 4j + 3, so a lane makes four cosines and sines for
// its token and turns every head with them.
//
// Angles: position * inv_freq / 2 pi in 64 bits, less its nearest whole
// number of turns, so far positions keep nearly the error of near ones (2^-26 of
// a turn from the last rounding; the product adds less up to positions of 10^8,
// and up to 2^-23 at the ends of 32 bits).
//
// Bound by the memory: q and k of 4096 tokens, 32 + 4 heads of 128, bf16, 14.3
// us for 75.5 MB (5.3 TB/s; a large copy reaches 5.5); 4096 tokens of 8 f32
// heads to a bf16 cache with the key's norm 10.9 us for 50.4 MB.  One token
// takes 2.6 us, which is the launch and two dependent loads.
#include "../../include/mer_hip.h"
#include "mer_attention.hpp"

namespace mer {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));

template <int TYPE> struct Elem;
template <> struct Elem<kF32> { typedef float T; typedef f4 V; };
template <> struct Elem<kF16> { typedef _Float16 T; typedef h4 V; };
template <> struct Elem<kBF16> { typedef __bf16 T; typedef b4 V; };

// 1 / sqrt(x) to two units in the last place; subnormal x, which the
// instruction takes for zero, are scaled up first.
__device__ __forceinline__ float inv_sqrt(float x) {
  const bool small = x < 0x1p-96f;
  const float r = __builtin_amdgcn_rsqf(small ? x * 0x1p96f : x);
  return small ? r * 0x1p48f : r;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
// Sum over groups of LANES lanes, in each of them.
template <int LANES>
__device__ __forceinline__ float sum_lanes(float x) {
  x += dpp<0xB1>(x);   // lane ^ 1
  x += dpp<0x4E>(x);   // lane ^ 2
  x += dpp<0x141>(x);  // the other four of eight
  if (LANES > 8) x += dpp<0x140>(x);  // the other eight of sixteen
  if (LANES > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// Passes of a wave: loads of all of them are in flight before the first is used.
constexpr uint32_t kPasses = 4;

// LANES: lanes of a head row, head_dim / 8 rounded up to a power of two.
template <int IN, int OUT, int LANES, bool APPEND>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeParams p) {
  typedef typename Elem<IN>::V VI;
  typedef typename Elem<OUT>::V VO;
  constexpr uint32_t kHeads = 64 / LANES;  // of a pass
  const uint32_t heads = p.t[0].heads + p.t[1].heads;
  const uint32_t per_token = (heads + p.heads_per_wave - 1) / p.heads_per_wave;
  const uint32_t wave = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t token = (uint32_t)__builtin_amdgcn_readfirstlane(wave / per_token);
  if (token >= p.n_tokens) return;
  const uint32_t head0 = (wave - token * per_token) * p.heads_per_wave;
  const uint32_t head1 = head0 + p.heads_per_wave < heads ? head0 + p.heads_per_wave : heads;
  const uint32_t lane = __lane_id(), j = lane % LANES, sub = lane / LANES;
  const bool in_row = j * 8 < p.head_dim;
  const bool split = !p.interleaved && j * 8 < p.rot;
  const uint32_t o0 = split ? 4 * j : 8 * j, o1 = split ? p.rot / 2 + 4 * j : 8 * j + 4;

  int64_t slot = 0;
  if (APPEND) {
    slot = p.slots[token];
    if (slot < 0) return;
    if ((uint64_t)slot >= p.n_slots) {
      if (lane == 0) atomicCAS(p.status, 0u, (uint32_t)MER_ERR_RESIDENCY_MISS);
      return;
    }
  }

  // What the angles and norms need is on its way before the rows.
  constexpr int kAngles = LANES > 16 ? 2 : 1;
  int32_t position = 0;
  float freq[kAngles];
  if (p.rot) {
    position = p.positions[token];
#pragma unroll
    for (int a = 0; a < kAngles; ++a) {
      const uint32_t f = a * 64 + lane;
      freq[a] = p.inv_freq[f < p.rot / 2 ? f : 0];
    }
  }
  const uint32_t tensor0 = head0 >= p.t[0].heads, tensor1 = head1 > p.t[0].heads;
  f4 w0[2], w1[2];
  if (in_row) {
    if (!tensor0 && p.t[0].norm) w0[0] = *(const f4 *)(p.t[0].norm + o0), w1[0] = *(const f4 *)(p.t[0].norm + o1);
    if (tensor1 && p.t[1].norm) w0[1] = *(const f4 *)(p.t[1].norm + o0), w1[1] = *(const f4 *)(p.t[1].norm + o1);
  }

  VI x0[kPasses], x1[kPasses];
#pragma unroll
  for (uint32_t k = 0; k < kPasses; ++k) {
    const uint32_t h = head0 + k * kHeads + sub;
    x0[k] = x1[k] = VI{};
    if (h < head1 && in_row) {
      const bool second = h >= p.t[0].heads;
      const RopeTensor &t = p.t[second];
      const typename Elem<IN>::T *row = (const typename Elem<IN>::T *)t.in + (uint64_t)token * t.in_stride +
                                        (uint64_t)(second ? h - p.t[0].heads : h) * p.head_dim;
      x0[k] = *(const VI *)(row + o0);
      x1[k] = *(const VI *)(row + o1);
    }
  }
  const bool turned = in_row && j * 8 < p.rot;
  f4 cs = {1, 1, 1, 1}, sn = {0, 0, 0, 0};
  if (p.rot) {
    // The wave's lanes make one angle each (two where there are more than 64)
    // and hand the cosine and sine to the lanes that turn by it.
    const double pos = (double)position;
    float c[kAngles], s[kAngles];
#pragma unroll
    for (int a = 0; a < kAngles; ++a) {
      const double t = pos * (double)freq[a] * 0.15915494309189535;  // 1 / (2 pi): turns
      sincospif((float)(2.0 * (t - rint(t))), &s[a], &c[a]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t f = 4 * j + i;
      const float c0 = __shfl(c[0], (int)(f % 64)), s0 = __shfl(s[0], (int)(f % 64));
      cs[i] = c0;
      sn[i] = s0;
      if (kAngles > 1) {
        const float c1 = __shfl(c[kAngles - 1], (int)(f % 64)), s1 = __shfl(s[kAngles - 1], (int)(f % 64));
        cs[i] = f < 64 ? c0 : c1;
        sn[i] = f < 64 ? s0 : s1;
      }
    }
  }
#pragma unroll
  for (uint32_t k = 0; k < kPasses; ++k) {
    const uint32_t h = head0 + k * kHeads + sub;
    if (head0 + k * kHeads >= head1) break;  // the whole wave
    const bool second = h >= p.t[0].heads;
    f4 a = __builtin_convertvector(x0[k], f4), b = __builtin_convertvector(x1[k], f4);
    const bool normed = (second ? p.t[1].norm : p.t[0].norm) != nullptr;
    if (p.t[0].norm || p.t[1].norm) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
      ss = sum_lanes<LANES>(ss);
      if (normed && in_row) {
        const float r = inv_sqrt(ss * p.inv_dim + p.eps);
        a = a * r * (second ? w0[1] : w0[0]);
        b = b * r * (second ? w1[1] : w1[0]);
      }
    }
    if (turned && !(APPEND && second)) {
      if (split) {
        const f4 u = a;
        a = u * cs - b * sn;
        b = b * cs + u * sn;
      } else {
        const f4 u = a, v = b;
        a = f4{u[0] * cs[0] - u[1] * sn[0], u[1] * cs[0] + u[0] * sn[0], u[2] * cs[1] - u[3] * sn[1],
               u[3] * cs[1] + u[2] * sn[1]};
        b = f4{v[0] * cs[2] - v[1] * sn[2], v[1] * cs[2] + v[0] * sn[2], v[2] * cs[3] - v[3] * sn[3],
               v[3] * cs[3] + v[2] * sn[3]};
      }
    }
    if (h < head1 && in_row) {
      const RopeTensor &t = p.t[second];
      const uint32_t hh = second ? h - p.t[0].heads : h;
      uint64_t at;
      if (APPEND) {
        const uint64_t page = (uint64_t)slot >> p.page_shift, off = (uint64_t)slot & ((1u << p.page_shift) - 1);
        at = (((page * t.heads + hh) << p.page_shift) + off) * p.head_dim;
      } else {
        at = (uint64_t)token * t.out_stride + (uint64_t)hh * p.head_dim;
      }
      typename Elem<OUT>::T *row = (typename Elem<OUT>::T *)t.out + at;
      // values of a cache's own type pass through unchanged
      *(VO *)(row + o0) = __builtin_convertvector(a, VO);
      *(VO *)(row + o1) = __builtin_convertvector(b, VO);
    }
  }
}

template <int IN, int OUT, bool APPEND>
hipError_t launch_lanes(NormRopeParams p, int cus, hipStream_t st) {
  const uint32_t lanes = p.head_dim <= 64 ? 8 : (p.head_dim <= 128 ? 16 : 32);
  const uint32_t heads = p.t[0].heads + p.t[1].heads, per_pass = 64 / lanes;
  // Heads of a wave: as many as its passes hold, fewer while that leaves the
  // chip with less than eight waves a CU.
  uint32_t passes = (heads + per_pass - 1) / per_pass;
  passes = passes > kPasses ? kPasses : passes;
  while (passes > 1 && (uint64_t)p.n_tokens * ((heads + passes * per_pass - 1) / (passes * per_pass)) < 8ull * cus) passes /= 2;
  // the same passes for every wave of a token
  const uint32_t all = (heads + per_pass - 1) / per_pass, per_token = (all + passes - 1) / passes;
  passes = (all + per_token - 1) / per_token;
  p.heads_per_wave = passes * per_pass;
  p.inv_dim = 1.0f / (float)p.head_dim;
  const uint64_t waves = (uint64_t)p.n_tokens * ((heads + p.heads_per_wave - 1) / p.heads_per_wave);
  const uint32_t grid = (uint32_t)((waves + 3) / 4);
  if (lanes == 8) norm_rope_kernel<IN, OUT, 8, APPEND><<<grid, 256, 0, st>>>(p);
  else if (lanes == 16) norm_rope_kernel<IN, OUT, 16, APPEND><<<grid, 256, 0, st>>>(p);
  else norm_rope_kernel<IN, OUT, 32, APPEND><<<grid, 256, 0, st>>>(p);
  return hipGetLastError();
}

template <int IN>
hipError_t launch_to(int out_type, const NormRopeParams &p, int cus, hipStream_t st) {
  switch (out_type) {
    case kF32: return launch_lanes<IN, kF32, false>(p, cus, st);
    case kF16: return launch_lanes<IN, kF16, false>(p, cus, st);
    default: return launch_lanes<IN, kBF16, false>(p, cus, st);
  }
}
template <int IN>
hipError_t append_to(int cache_type, const NormRopeParams &p, int cus, hipStream_t st) {
  return cache_type == kF16 ? launch_lanes<IN, kF16, true>(p, cus, st) : launch_lanes<IN, kBF16, true>(p, cus, st);
}

}  // namespace

hipError_t launch_norm_rope(int in_type, int out_type, const NormRopeParams &p, int cus, hipStream_t st) {
  switch (in_type) {
    case kF32: return launch_to<kF32>(out_type, p, cus, st);
    case kF16: return launch_to<kF16>(out_type, p, cus, st);
    default: return launch_to<kBF16>(out_type, p, cus, st);
  }
}

hipError_t launch_kv_append(int in_type, int cache_type, const NormRopeParams &p, int cus, hipStream_t st) {
  switch (in_type) {
    case kF32: return append_to<kF32>(cache_type, p, cus, st);
    case kF16: return append_to<kF16>(cache_type, p, cus, st);
    default: return append_to<kBF16>(cache_type, p, cus, st);
  }
}

}  // namespace mer
