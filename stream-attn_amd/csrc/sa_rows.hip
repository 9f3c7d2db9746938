// Rows of Q, K and V between a QKV projection and the attention: the norm of
// every head, the rotation by positions of one or several axes, and K and V
// rows into and out of the pages of a device-resident cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                (per head, where there is a weight)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t)  t = frequency[i] * position[axis of i]
//   INT8 pages: step = amax / 127, codes rint(y / step), scale fp16(step)
//
// Bytes bound: about ten operations per element that is read once and written
// once.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "sa_common.h"
#include "sa_types.h"

namespace sa {
namespace {

// Launches of 2^32 threads and more go in parts.
constexpr int64_t kTokensPerLaunch = 1 << 23;

struct PageRows {
  char* base;       // row of slot s: base + page * stride_p + row * stride_t + head * stride_h, in elements
  uint16_t* scale;  // fp16 scales, null for 16-bit pages
  int64_t sp, st, sh, ss_p, ss_t, ss_h;
};

struct RowsParams {
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_out;
  PageRows kp, vp;
  const int64_t* slots;
  const void* positions;
  const double* frequencies;
  const void *q_weight, *k_weight;
  int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h, sqo_t, sqo_h, sko_t, sko_h;
  int64_t pos_axis, pos_token, token0, tokens;
  float eps, inv_dim;
  uint32_t num_slots, page_tokens;
  int32_t q_heads, kv_heads, head_dim, pairs;
  int32_t end0, end1, end2;  // first pair past axis 0, 1, 2
  int32_t heads;             // rows of a token: Q's, K's and V's
  int32_t lane_log2;         // log2 of the lanes of a head
  int32_t beside;            // log2 of a token's waves in a workgroup
  int32_t pos64, qw32, kw32;
};

constexpr int kMostPairs = 128;  // of a head

// How a lane's W pairs lie in a row.  With halves, unit u holds pairs W u ..
// W u + W - 1: their first elements are W consecutive ones, their second
// elements W consecutive ones.  The elements past 2 * pairs go through as
// pairs of their own that are not turned.  The scalar form takes any number
// of pairs, element by element.
enum Form { kHalves, kAdjacent, kScalar };

template <Form F, int W>
struct Unit {
  int lo, hi;  // first elements of the two runs (halves), of the first pair (adjacent)
  int first;   // first pair
  int pairs, rest;

  __device__ Unit(int u, int pairs_, int head_dim) : first(u * W), pairs(pairs_), rest((head_dim - 2 * pairs_) / 2) {
    if (F == kAdjacent) {
      lo = 2 * first, hi = lo + 1;
    } else {
      const bool turned = first < pairs;
      lo = turned ? first : first + pairs;
      hi = lo + (turned ? pairs : rest);
    }
  }
  // Elements of pair i of the unit (scalar form).
  __device__ int at_lo(int i) const { return first + i < pairs ? first + i : first + i + pairs; }
  __device__ int at_hi(int i) const { return first + i < pairs ? first + i + pairs : first + i + pairs + rest; }
};

template <int N>
struct Words {
  uint32_t w[N];
};

// N dwords, aligned to 4 N bytes up to 16.  With kOnce past the caches (a
// launch over more than they hold reads and writes everything once).
template <int N, bool kOnce>
__device__ inline __attribute__((always_inline)) Words<N> load_words(const void* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const u32x4 t = kOnce ? __builtin_nontemporal_load(static_cast<const u32x4*>(p)) : *static_cast<const u32x4*>(p);
    for (int i = 0; i < 4; ++i) r.w[i] = t[i];
  } else if constexpr (N == 2) {
    const u32x2 t = kOnce ? __builtin_nontemporal_load(static_cast<const u32x2*>(p)) : *static_cast<const u32x2*>(p);
    r.w[0] = t[0], r.w[1] = t[1];
  } else {
    r.w[0] = *static_cast<const uint32_t*>(p);
  }
  return r;
}

template <int N, bool kOnce>
__device__ inline __attribute__((always_inline)) void store_words(void* p, const Words<N>& r) {
  if constexpr (N == 4) {
    const u32x4 t = {r.w[0], r.w[1], r.w[2], r.w[3]};
    if constexpr (kOnce)
      __builtin_nontemporal_store(t, static_cast<u32x4*>(p));
    else
      *static_cast<u32x4*>(p) = t;
  } else if constexpr (N == 2) {
    const u32x2 t = {r.w[0], r.w[1]};
    if constexpr (kOnce)
      __builtin_nontemporal_store(t, static_cast<u32x2*>(p));
    else
      *static_cast<u32x2*>(p) = t;
  } else {
    *static_cast<uint32_t*>(p) = r.w[0];
  }
}

// The 2 W elements of a unit as they lie in memory.
template <Form F, int W>
struct Raw {
  uint32_t w[W];  // kScalar: element pairs (lo, hi), halves and adjacent: the runs
};

template <Form F, int W, bool kOnce>
__device__ inline __attribute__((always_inline)) Raw<F, W> load_raw(const uint16_t* row, const Unit<F, W>& u) {
  Raw<F, W> r;
  if constexpr (F == kScalar) {
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = row[u.at_lo(i)] | (uint32_t)row[u.at_hi(i)] << 16;
  } else if constexpr (F == kAdjacent) {
#pragma unroll
    for (int n = 0; n < W; n += 4) {
      const Words<4> x = load_words<4, kOnce>(row + u.lo + 2 * n);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[n + i] = x.w[i];
    }
  } else {
    const Words<W / 2> x = load_words<W / 2, kOnce>(row + u.lo), y = load_words<W / 2, kOnce>(row + u.hi);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) r.w[i] = x.w[i], r.w[W / 2 + i] = y.w[i];
  }
  return r;
}

// Its W pairs as floats.
template <typename T, Form F, int W>
__device__ inline __attribute__((always_inline)) void pairs_of(const Raw<F, W>& r, float (&a)[W], float (&b)[W]) {
  if constexpr (F == kHalves) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      a[2 * i] = T::lo(r.w[i]), a[2 * i + 1] = T::hi(r.w[i]);
      b[2 * i] = T::lo(r.w[W / 2 + i]), b[2 * i + 1] = T::hi(r.w[W / 2 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) a[i] = T::lo(r.w[i]), b[i] = T::hi(r.w[i]);
  }
}

template <typename T, Form F, int W>
__device__ inline __attribute__((always_inline)) void load_weight(const void* weight, bool fp32, const Unit<F, W>& u,
                                                                  float (&a)[W], float (&b)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) a[i] = b[i] = 1.f;
  if (weight == nullptr) return;
  if (fp32) {
    const float* w = static_cast<const float*>(weight);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a[i] = w[F == kAdjacent ? u.lo + 2 * i : F == kHalves ? u.lo + i : u.at_lo(i)];
      b[i] = w[F == kAdjacent ? u.lo + 2 * i + 1 : F == kHalves ? u.hi + i : u.at_hi(i)];
    }
  } else {
    pairs_of<T, F, W>(load_raw<F, W, false>(static_cast<const uint16_t*>(weight), u), a, b);
  }
}

template <typename T, Form F, int W, bool kOnce>
__device__ inline void store_pairs(uint16_t* row, const Unit<F, W>& u, const float (&a)[W], const float (&b)[W]) {
  if constexpr (F == kScalar) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      row[u.at_lo(i)] = (uint16_t)T::pack(a[i], 0.f);
      row[u.at_hi(i)] = (uint16_t)T::pack(b[i], 0.f);
    }
  } else if constexpr (F == kAdjacent) {
#pragma unroll
    for (int n = 0; n < W; n += 4) {
      Words<4> x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.w[i] = T::pack(a[n + i], b[n + i]);
      store_words<4, kOnce>(row + u.lo + 2 * n, x);
    }
  } else {
    Words<W / 2> x, y;
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      x.w[i] = T::pack(a[2 * i], a[2 * i + 1]);
      y.w[i] = T::pack(b[2 * i], b[2 * i + 1]);
    }
    store_words<W / 2, kOnce>(row + u.lo, x);
    store_words<W / 2, kOnce>(row + u.hi, y);
  }
}

// The low bytes of four words.
__device__ inline uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

template <Form F, int W, bool kOnce>
__device__ inline void store_codes(char* row, const Unit<F, W>& u, const uint32_t (&a)[W],
                                   const uint32_t (&b)[W]) {
  if constexpr (F == kScalar) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      row[u.at_lo(i)] = (char)a[i];
      row[u.at_hi(i)] = (char)b[i];
    }
  } else if constexpr (F == kAdjacent) {
#pragma unroll
    for (int n = 0; n < W; n += 4)
      store_words<2, kOnce>(row + u.lo + 2 * n, Words<2>{{pack_codes(a[n], b[n], a[n + 1], b[n + 1]),
                                                          pack_codes(a[n + 2], b[n + 2], a[n + 3], b[n + 3])}});
  } else {
    Words<W / 4> x, y;
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      x.w[i] = pack_codes(a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]);
      y.w[i] = pack_codes(b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]);
    }
    store_words<W / 4, kOnce>(row + u.lo, x);
    store_words<W / 4, kOnce>(row + u.hi, y);
  }
}

// A sum or maximum over the 2^n lanes of a head, at most 32 (256 elements, 8 or
// more on a lane): exchanges within 4 lanes, then mirrored halves of 8 and 16
// (whose quarters hold one value by then).
template <int kControl>
__device__ inline float exchanged(float x) {
  const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kControl, 0xf, 0xf, true);
  return __builtin_bit_cast(float, y);
}
template <typename Join>
__device__ inline float over_lanes(float x, int lane_log2, Join join) {
  if (lane_log2 > 0) x = join(x, exchanged<0xb1>(x));
  if (lane_log2 > 1) x = join(x, exchanged<0x4e>(x));
  if (lane_log2 > 2) x = join(x, exchanged<0x141>(x));
  if (lane_log2 > 3) x = join(x, exchanged<0x140>(x));
  if (lane_log2 > 4) x = join(x, __shfl_xor(x, 16));
  return x;
}

// Without a branch or a memory operand, which a conditional expression over
// arrays can become.
__device__ inline float choose(uint32_t mask, float x, float y) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
  return __builtin_bit_cast(float, (a & mask) | (b & ~mask));
}
__device__ inline int64_t choose(uint32_t mask, int64_t x, int64_t y) {
  const int64_t m = (int64_t)(int32_t)mask;
  return (x & m) | (y & ~m);
}

// The bits of |x|, in the order of the magnitudes.
__device__ inline uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// The FP16 scale of an INT8 row: NaN for one that is not finite.
__device__ inline uint16_t scale_of(float amax, float step) {
  return (uint16_t)Fp16::pack(amax <= FLT_MAX ? step : NAN, 0.f);
}

// rint(x / step) in the low byte, with the quotient rounded as a division rounds
// it: only next to a half do the quotient and the product with the reciprocal (off
// by less than 127 * 2^-22) round apart.  Adding 1.5 * 2^23 rounds to an integer
// and leaves its two's complement in the low bits.  A finite row's are within 127
// (its largest magnitude is 127 steps); another's scale is NaN, and that of steps
// below float16's is 0, whatever the codes.
template <int N>
__device__ inline void codes(const float (&x)[N], float step, float reciprocal, uint32_t (&code)[N]) {
  constexpr float kRound = 12582912.f;
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = fmaf(x[i], reciprocal, kRound);
    code[i] = __builtin_bit_cast(uint32_t, y);
    off = fmaxf(off, fabsf(fmaf(x[i], reciprocal, kRound - y)));
  }
  if (__any(off > 0.5f - 1.f / 32768)) {
#pragma unroll
    for (int i = 0; i < N; ++i) code[i] = __builtin_bit_cast(uint32_t, x[i] / step + kRound);
  }
}

// A wave takes rows of one token (Q's heads, then K's, then V's), 64 >>
// lane_log2 at a time, and loads the next ones before it works on these.  The
// angles and weights are its own once per token, so with many tokens a wave
// has many rows of one; with few, the rows are dealt to gridDim.y times as many
// waves, which is less time on the way through one.
//
// Measured (a copy that streams 2 GiB reaches 6.4 TB/s): 61,312 tokens x 112 heads
// of 128, three axes, 585 us, 6.0 TB/s; 20,011 tokens of 32 + 8 + 8 heads into pages
// 84 us, 5.9 TB/s.  A launch of 48 tokens is 4.5 us, most of it latency: the
// positions, then the angles, then a row's sum.
template <typename T, Form F, int W, bool kInt8, bool kOnce>
__global__ __launch_bounds__(256) void rows_kernel(const RowsParams p) {
  // A token's waves: 2^beside in the workgroup, in gridDim.y workgroups.
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = p.token0 + (int64_t)blockIdx.x * (4 >> p.beside) + (wave >> p.beside);
  if (token >= p.tokens) return;
  const int unit_lane = lane & ((1 << p.lane_log2) - 1);
  const int per_step = 64 >> p.lane_log2;
  const bool live = unit_lane * 2 * W < p.head_dim;  // head_dim / 2W lanes of the 2^n hold a unit
  const Unit<F, W> u(live ? unit_lane : 0, p.pairs, p.head_dim);
  // Where the token's Q, K and V start, and their heads' strides.
  const int64_t in_q = (int64_t)(p.q + token * p.sq_t), in_k = (int64_t)(p.k + token * p.sk_t);
  const int64_t in_v = (int64_t)(p.v + token * p.sv_t);
  const int64_t sq_h = p.sq_h, sk_h = p.sk_h, sv_h = p.sv_h;
  const int v_row = p.q_heads + p.kv_heads;
  // Every lane loads something: what no row or unit needs is a repetition.
  const auto load = [&](int first) {
    const int row = min(first + (lane >> p.lane_log2), p.heads - 1);
    const uint32_t is_q = row < p.q_heads ? ~0u : 0u, is_v = row >= v_row ? ~0u : 0u;
    const int head = row - (~is_q & p.q_heads) - (is_v & p.kv_heads);
    const int64_t base = choose(is_q, in_q, choose(is_v, in_v, in_k));
    const int64_t stride = choose(is_q, sq_h, choose(is_v, sv_h, sk_h));
    return load_raw<F, W, kOnce>(reinterpret_cast<const uint16_t*>(base) + head * stride, u);
  };
  const int stride = (gridDim.y << p.beside) * per_step;
  int first = ((blockIdx.y << p.beside) + (wave & ((1 << p.beside) - 1))) * per_step;
  Raw<F, W> raw = load(first);

  bool stored = false;
  uint32_t page = 0, row_in_page = 0;
  if (p.slots != nullptr) {
    const int64_t slot = p.slots[token];
    stored = slot >= 0 && slot < (int64_t)p.num_slots;
    if (stored) page = (uint32_t)slot / p.page_tokens, row_in_page = (uint32_t)slot - page * p.page_tokens;
  }
  const int64_t at = page * p.kp.sp + row_in_page * p.kp.st;
  const int64_t k_base = (int64_t)p.kp.base, v_base = (int64_t)p.vp.base;
  const int64_t k_scales = (int64_t)p.kp.scale, v_scales = (int64_t)p.vp.scale;
  const int64_t scale_at = page * p.kp.ss_p + row_in_page * p.kp.ss_t;

  float cos_t[W], sin_t[W], wqa[W], wqb[W], wka[W], wkb[W];
  const bool normalizes = p.q_weight != nullptr || p.k_weight != nullptr;
  if (normalizes) {
    load_weight<T, F, W>(p.q_weight, p.qw32, u, wqa, wqb);
    load_weight<T, F, W>(p.k_weight, p.kw32, u, wka, wkb);
  }
  if (p.pairs > 0) {
    // A pair per lane, then every lane's own from LDS (the wave's part of it:
    // no barrier).
    __shared__ float angles[4][2][kMostPairs];
    for (int pair = lane; pair < p.pairs; pair += 64) {
      const int axis = (pair >= p.end0) + (pair >= p.end1) + (pair >= p.end2);
      const int64_t at = axis * p.pos_axis + token * p.pos_token;
      const double position = p.pos64 ? (double)static_cast<const int64_t*>(p.positions)[at]
                                      : (double)static_cast<const int32_t*>(p.positions)[at];
      // Turns in FP64 (far positions have their fraction there), its fraction
      // in FP32: the sine instruction takes turns.
      const double turns = position * (p.frequencies[pair] * 0.15915494309189533577);
      const float fraction = (float)(turns - rint(turns));
      angles[wave][0][pair] = __builtin_amdgcn_cosf(fraction);
      angles[wave][1][pair] = __builtin_amdgcn_sinf(fraction);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int pair = u.first + i;
      const float c = angles[wave][0][min(pair, p.pairs - 1)], s = angles[wave][1][min(pair, p.pairs - 1)];
      cos_t[i] = c, sin_t[i] = s;
    }
  }

  const int64_t out_q = (int64_t)(p.q_out + token * p.sqo_t), out_k = (int64_t)(p.k_out + token * p.sko_t);
  const int64_t sqo_h = p.sqo_h, sko_h = p.sko_h;
  const bool weight_q = p.q_weight != nullptr, weight_k = p.k_weight != nullptr;
  while (first < p.heads) {
    const int row = first + (lane >> p.lane_log2);
    const bool is_q = row < p.q_heads, is_v = row >= v_row;
    const uint32_t mask_q = is_q ? ~0u : 0u, mask_v = is_v ? ~0u : 0u;
    const int head = row - (~mask_q & p.q_heads) - (mask_v & p.kv_heads);
    const bool active = live && row < p.heads;
    float a[W], b[W];
    pairs_of<T, F, W>(raw, a, b);
    first += stride;
    if (first < p.heads) raw = load(first);
    if (normalizes) {
      float squares = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) squares += a[i] * a[i] + b[i] * b[i];
      squares = over_lanes(live ? squares : 0.f, p.lane_log2, [](float x, float y) { return x + y; });
      const bool weighted = is_q ? weight_q : !is_v && weight_k;
      const float r = weighted ? rsqrtf(squares * p.inv_dim + p.eps) : 1.f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        a[i] *= r * choose(mask_q, wqa[i], choose(mask_v, 1.f, wka[i]));
        b[i] *= r * choose(mask_q, wqb[i], choose(mask_v, 1.f, wkb[i]));
      }
    }
    // Elements past the pairs are passed over, not turned by an angle of zero:
    // an infinity or NaN there times that angle's sine is NaN in its neighbour.
    // Where a unit has both kinds, by the lanes that a pair's instructions run
    // on (the asm keeps the compiler from selections, two more per pair: 40,000
    // tokens of 32 heads of 80, half of each turned, 95 us, with them 101).
    const int turned = p.pairs - u.first;  // of the unit's pairs
    if (turned > 0 && !is_v) {
      const auto turn = [&](bool all) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          if (all || i < turned) {
            const float x = a[i] * cos_t[i] - b[i] * sin_t[i];
            b[i] = b[i] * cos_t[i] + a[i] * sin_t[i];
            a[i] = x;
            if (!all) asm volatile("" : "+v"(a[i]), "+v"(b[i]));
          }
        }
      };
      if (F == kHalves || p.pairs % W == 0)
        turn(true);
      else
        turn(false);
    }
    if (is_q || p.slots == nullptr) {
      uint16_t* out = reinterpret_cast<uint16_t*>(choose(mask_q, out_q, out_k)) + head * choose(mask_q, sqo_h, sko_h);
      if (active) store_pairs<T, F, W, kOnce>(out, u, a, b);
    }
    if (p.slots == nullptr) continue;
    char* pages = reinterpret_cast<char*>(choose(mask_v, v_base, k_base));
    if constexpr (kInt8) {
      // The largest magnitude; as integers infinities and NaN are larger still.
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < W; ++i)
        top = max(top, max(magnitude(a[i]), magnitude(b[i])));
      const float amax = over_lanes(__builtin_bit_cast(float, min(top, 0x7f800000u)), p.lane_log2,
                                    [](float x, float y) { return fmaxf(x, y); });
      if (active && !is_q && stored) {
        const float step = amax / 127.f > 0.f ? amax / 127.f : 1.f;
        const float reciprocal = 1.f / step;
        uint32_t code_a[W], code_b[W];
        codes(a, step, reciprocal, code_a);
        codes(b, step, reciprocal, code_b);
        store_codes<F, W, kOnce>(pages + at + head * p.kp.sh, u, code_a, code_b);
        if (unit_lane == 0)
          reinterpret_cast<uint16_t*>(choose(mask_v, v_scales, k_scales))[scale_at + head * p.kp.ss_h] =
              scale_of(amax, step);
      }
    } else if (active && !is_q && stored) {
      store_pairs<T, F, W, kOnce>(reinterpret_cast<uint16_t*>(pages) + at + head * p.kp.sh, u, a, b);
    }
  }
}

// log2 of the lanes of a head with `elements` on each, and the heads of a wave.
int32_t lanes_log2(int32_t head_dim, int32_t elements) {
  int32_t n = 0;
  while ((elements << n) < head_dim) ++n;
  return n;
}
int32_t rows_per_step(int32_t lane_log2) { return 64 >> lane_log2; }

struct StoreParams {
  const uint16_t *k, *v;
  PageRows kp, vp;
  const int64_t* slots;
  int64_t sk_t, sk_h, sv_t, sv_h, token0, tokens;
  uint32_t num_slots, page_tokens;
  int32_t kv_heads, head_dim, lane_log2;
  int32_t each;  // tokens of a workgroup
};

// K and V rows to their pages as they are, few per token: where a token's would
// leave lanes of a wave without one (rows_kernel), a workgroup has the rows of
// `each` tokens, four of a thread under way together.  A row's granules (8
// elements) are on 2^lane_log2 lanes.  60,000 rows of 128, with one K/V head
// 44 -> 30 us (INT8 66 -> 38), two 28 -> 24; four and more as fast in rows_kernel,
// 56 slower here (186 and 177).
template <typename T, bool kInt8>
__global__ __launch_bounds__(256) void store_kernel(const StoreParams p) {
  constexpr int kTogether = 4;
  const int64_t token0 = p.token0 + (int64_t)blockIdx.x * p.each;
  const int count = (int)std::min<int64_t>(p.each, p.tokens - token0), per_token = 2 * p.kv_heads;
  const int g = threadIdx.x & ((1 << p.lane_log2) - 1), d = 8 * g;
  const bool live = d < p.head_dim;
  const int groups = 256 >> p.lane_log2;
  for (int first = threadIdx.x >> p.lane_log2; first - (int)(threadIdx.x >> p.lane_log2) < count * per_token;
       first += kTogether * groups) {
    u32x4 x[kTogether];
    int64_t slot[kTogether];
    int head[kTogether];
    uint32_t is_v[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int row = first + i * groups;
      const bool has = live && row < count * per_token;
      const int t = has ? row / per_token : 0, h = has ? row - t * per_token : 0;
      is_v[i] = h >= p.kv_heads ? ~0u : 0u;
      head[i] = h - (is_v[i] & p.kv_heads);
      const int64_t base = choose(is_v[i], (int64_t)p.v, (int64_t)p.k);
      const int64_t at = (token0 + t) * choose(is_v[i], p.sv_t, p.sk_t) + head[i] * choose(is_v[i], p.sv_h, p.sk_h);
      x[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(base) + at + (live ? d : 0));
      slot[i] = p.slots[token0 + t];
      if (!has || slot[i] >= (int64_t)p.num_slots) slot[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const bool stored = slot[i] >= 0;
      const uint32_t page = stored ? (uint32_t)slot[i] / p.page_tokens : 0;
      const uint32_t row = stored ? (uint32_t)slot[i] - page * p.page_tokens : 0;
      const int64_t at = page * p.kp.sp + row * p.kp.st + head[i] * p.kp.sh + d;
      char* pages = reinterpret_cast<char*>(choose(is_v[i], (int64_t)p.vp.base, (int64_t)p.kp.base));
      if constexpr (kInt8) {
        float y[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[2 * e] = T::lo(x[i][e]), y[2 * e + 1] = T::hi(x[i][e]);
          top = max(top, max(magnitude(y[2 * e]), magnitude(y[2 * e + 1])));
        }
        const float amax = over_lanes(live ? __builtin_bit_cast(float, min(top, 0x7f800000u)) : 0.f, p.lane_log2,
                                      [](float a, float b) { return fmaxf(a, b); });
        const float step = amax / 127.f > 0.f ? amax / 127.f : 1.f;
        uint32_t code[8];
        codes(y, step, 1.f / step, code);
        if (!stored) continue;
        *reinterpret_cast<u32x2*>(pages + at) =
            u32x2{pack_codes(code[0], code[1], code[2], code[3]), pack_codes(code[4], code[5], code[6], code[7])};
        if (g == 0)
          reinterpret_cast<uint16_t*>(choose(is_v[i], (int64_t)p.vp.scale, (int64_t)p.kp.scale))
              [page * p.kp.ss_p + row * p.kp.ss_t + head[i] * p.kp.ss_h] = scale_of(amax, step);
      } else if (stored) {
        *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(pages) + at) = x[i];
      }
    }
  }
}

template <typename T>
int32_t launch_store(StoreParams p, bool int8, hipStream_t stream) {
  p.lane_log2 = lanes_log2(p.head_dim, 8);
  p.each = std::max(1, (1024 >> p.lane_log2) / (2 * p.kv_heads));
  const int64_t most = kTokensPerLaunch / p.each * p.each;
  for (p.token0 = 0; p.token0 < p.tokens; p.token0 += most) {
    const uint32_t grid = (uint32_t)((std::min(p.tokens - p.token0, most) + p.each - 1) / p.each);
    if (int8)
      store_kernel<T, true><<<grid, 256, 0, stream>>>(p);
    else
      store_kernel<T, false><<<grid, 256, 0, stream>>>(p);
    SA_HIP_RETURN(hipGetLastError());
  }
  return 0;
}

struct ReadParams {
  PageRows kp, vp;
  const int64_t* slots;
  uint16_t *k_out, *v_out;
  int64_t token0, tokens;
  uint32_t num_slots, page_tokens;
  int32_t kv_heads, head_dim, block_log2;
};

// Thread i of a workgroup moves granule (8 elements) i, i + 256, ... of K and
// V rows of kReadTokens tokens, whose loads are under way together.
constexpr int kReadTokens = 4;

template <typename T, PageKind kKind>
__global__ __launch_bounds__(256) void read_kernel(const ReadParams p) {
  const int64_t token = p.token0 + (int64_t)blockIdx.x * kReadTokens;
  int64_t at[kReadTokens], scale_at[kReadTokens];
  bool held[kReadTokens];
#pragma unroll
  for (int t = 0; t < kReadTokens; ++t) {
    const int64_t slot = token + t < p.tokens ? p.slots[token + t] : -1;
    held[t] = slot >= 0 && slot < (int64_t)p.num_slots;
    const uint32_t page = held[t] ? (uint32_t)slot / p.page_tokens : 0;
    const uint32_t row = held[t] ? (uint32_t)slot - page * p.page_tokens : 0;  // row 0 is there to be read
    at[t] = page * p.kp.sp + row * p.kp.st;
    scale_at[t] = page * p.kp.ss_p + (kKind == kE4m3Pages ? row >> p.block_log2 : row) * p.kp.ss_t;
  }
  const int granules = p.head_dim / 8, each = p.kv_heads * granules;
  for (int i = threadIdx.x; i < 2 * each; i += 256) {
    const bool is_v = i >= each;
    const int g = is_v ? i - each : i, head = g / granules, d = 8 * (g - head * granules);
    const char* base = is_v ? p.vp.base : p.kp.base;
    u32x4 w[kReadTokens];
    if constexpr (kKind == kE4m3Pages) {
      const uint8_t* scales = reinterpret_cast<const uint8_t*>(is_v ? p.vp.scale : p.kp.scale);
      u32x2 c[kReadTokens];
      uint8_t scale[kReadTokens];
#pragma unroll
      for (int t = 0; t < kReadTokens; ++t) {
        c[t] = *reinterpret_cast<const u32x2*>(base + at[t] + head * p.kp.sh + d);
        scale[t] = scales[scale_at[t] + head * p.kp.ss_h];
      }
#pragma unroll
      for (int t = 0; t < kReadTokens; ++t) {
        const float power = e8m0_value(scale[t]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x2 x = e4m3_floats<false>(c[t][j]), y = e4m3_floats<true>(c[t][j]);
          w[t][2 * j] = T::pack(x[0] * power, x[1] * power);
          w[t][2 * j + 1] = T::pack(y[0] * power, y[1] * power);
        }
      }
    } else if constexpr (kKind == kInt8Pages) {
      const uint16_t* scales = is_v ? p.vp.scale : p.kp.scale;
      u32x2 c[kReadTokens];
      uint16_t scale[kReadTokens];
#pragma unroll
      for (int t = 0; t < kReadTokens; ++t) {
        c[t] = *reinterpret_cast<const u32x2*>(base + at[t] + head * p.kp.sh + d);
        scale[t] = scales[scale_at[t] + head * p.kp.ss_h];
      }
#pragma unroll
      for (int t = 0; t < kReadTokens; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[t][j] = T::pack(byte_float(c[t][j / 2], 2 * (j & 1)) * Fp16::lo(scale[t]),
                            byte_float(c[t][j / 2], 2 * (j & 1) + 1) * Fp16::lo(scale[t]));
    } else {
#pragma unroll
      for (int t = 0; t < kReadTokens; ++t)
        w[t] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(base) + at[t] + head * p.kp.sh + d);
    }
#pragma unroll
    for (int t = 0; t < kReadTokens; ++t)
      if (token + t < p.tokens)
        *reinterpret_cast<u32x4*>((is_v ? p.v_out : p.k_out) + (token + t) * each * 8 + g * 8) =
            held[t] ? w[t] : u32x4{0, 0, 0, 0};
  }
}

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// scale_align: bytes of a scale.
template <typename Args>
bool page_rows(PageRows& r, const void* base, const void* scale, const Args* a, int64_t scale_align = 2) {
  const bool int8 = a->pages_int8;
  r = {static_cast<char*>(const_cast<void*>(base)), int8 ? static_cast<uint16_t*>(const_cast<void*>(scale)) : nullptr,
       a->stride_pp, a->stride_pt, a->stride_ph, a->stride_sp, a->stride_st, a->stride_sh};
  return base != nullptr && aligned(base, int8 ? 8 : 16) && r.sp % 8 == 0 && r.st % 8 == 0 && r.sh % 8 == 0 &&
         (!int8 || (scale != nullptr && aligned(scale, scale_align)));
}

int32_t invalid(const char* entry, const char* what) {
  set_error("%s: %s", entry, what);
  return SA_ERR_INVALID_ARGUMENT;
}

int32_t check_sizes(const char* entry, int32_t dtype, int32_t head_dim, int32_t heads, int64_t tokens) {
  if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_FP16) {
    set_error("%s: unsupported dtype code %d", entry, dtype);
    return SA_ERR_UNSUPPORTED_DTYPE;
  }
  if (head_dim < 16 || head_dim > 256 || head_dim % 8) {
    set_error("%s: head_dim must be a multiple of 8 in [16, 256], got %d", entry, head_dim);
    return SA_ERR_UNSUPPORTED_HEAD_DIM;
  }
  if (tokens < 0 || tokens > INT32_MAX || heads < 1 || heads > (1 << 20))
    return invalid(entry, "tokens or heads out of range");
  return 0;
}

int32_t check_pool(const char* entry, int64_t num_pages, int32_t page_tokens) {
  if (page_tokens < 1 || page_tokens > SA_MAX_PAGE_TOKENS || num_pages < 0 || num_pages > INT32_MAX / page_tokens)
    return invalid(entry, "page_tokens must be at most 2^20 and num_pages * page_tokens below 2^31");
  return 0;
}

// Waves that fill the chip: a token's rows are dealt to several waves where
// there are fewer tokens.  With 40 heads of 128: 4,099 tokens 18.3 us with 4,096,
// 23 with 16,384; 6,000 tokens 25.4 and 28.6.
constexpr int64_t kWavesToFill = 4096;
// Bytes read and written from which a launch passes the caches by, those that
// the Infinity Cache holds.  61,312 x 112 heads of 128 (3.5 GB) 677 -> 633 us,
// 20,011 tokens with the append (492 MB) 98 -> 92; 8,190 x 32 heads of 80 (84 MB),
// read again from the cache, 23 -> 26.
constexpr int64_t kCacheBytes = 256 << 20;
// A token's steps (64 >> lane_log2 rows each) from which two or four waves of
// a workgroup take them in turn, so that rows that lie together are read
// together.  Heads of 128, with one wave, two and four, us:
//   61,312 tokens of 5 steps 217, 220, 264; of 6 266, 252, 295; of 8 362, 335, 351;
//   of 11 512, 466, 456; of 12 562, 512, 492; of 14 683, 609, 586 (6.0 TB/s);
//   20,011 tokens of 5 steps 78, 78, 94; of 6 94, 89, 102; of 12 188, 177, 170;
//   20,011 tokens with the append, of 5 78, 77, 95; of 6 89, 87, 104; of 12 190, 175, 169.
constexpr int32_t kTwoBeside = 6, kFourBeside = 12;

template <typename T, bool kInt8, bool kOnce>
int32_t launch_rows(RowsParams p, bool adjacent, hipStream_t stream) {
  // Sixteen bytes per access wherever the pairs allow it, then 8, then single
  // elements.
  const int32_t rest = (p.head_dim - 2 * p.pairs) / 2;
  const auto fits = [&](int w) { return p.pairs % w == 0 && rest % w == 0; };
  const bool sixteen = p.head_dim % 16 == 0;  // elements of a lane
  const int form = p.pairs > 0 && !adjacent ? (fits(8) ? 1 : fits(4) ? 2 : 3) : sixteen ? 4 : 0;
  p.lane_log2 = lanes_log2(p.head_dim, form == 1 || form == 4 ? 16 : 8);
  const int32_t per_step = rows_per_step(p.lane_log2), steps = (p.heads + per_step - 1) / per_step;
  const int64_t waves = std::min<int64_t>(steps, (kWavesToFill + p.tokens - 1) / p.tokens);
  p.beside = steps >= kFourBeside ? 2 : steps >= kTwoBeside ? 1 : 0;
  for (p.token0 = 0; p.token0 < p.tokens; p.token0 += kTokensPerLaunch) {
    const int64_t count = std::min(p.tokens - p.token0, kTokensPerLaunch);
    const int64_t tokens = 4 >> p.beside;  // of a workgroup
    const dim3 grid((uint32_t)((count + tokens - 1) / tokens), (uint32_t)((waves + (1 << p.beside) - 1) >> p.beside));
    if (form == 0)
      rows_kernel<T, kAdjacent, 4, kInt8, kOnce><<<grid, 256, 0, stream>>>(p);
    else if (form == 4)
      rows_kernel<T, kAdjacent, 8, kInt8, kOnce><<<grid, 256, 0, stream>>>(p);
    else if (form == 1)
      rows_kernel<T, kHalves, 8, kInt8, kOnce><<<grid, 256, 0, stream>>>(p);
    else if (form == 2)
      rows_kernel<T, kHalves, 4, kInt8, kOnce><<<grid, 256, 0, stream>>>(p);
    else
      rows_kernel<T, kScalar, 4, kInt8, kOnce><<<grid, 256, 0, stream>>>(p);
    SA_HIP_RETURN(hipGetLastError());
  }
  return 0;
}

template <typename T>
int32_t launch_rows(const RowsParams& p, bool int8, bool adjacent, hipStream_t stream) {
  const bool once = p.tokens * p.heads * p.head_dim * 4 >= kCacheBytes;
  if (int8)
    return once ? launch_rows<T, true, true>(p, adjacent, stream) : launch_rows<T, true, false>(p, adjacent, stream);
  return once ? launch_rows<T, false, true>(p, adjacent, stream) : launch_rows<T, false, false>(p, adjacent, stream);
}

}  // namespace
}  // namespace sa

extern "C" {

int32_t sa_normalize_rotate_store(const sa_rows_args* a, int32_t device, void* stream) try {
  using namespace sa;
  const char* entry = "sa_normalize_rotate_store";
  clear_error();
  if (a == nullptr) return invalid(entry, "null arguments");
  const bool pages = a->k_pages != nullptr;
  int32_t rc = check_sizes(entry, a->dtype, a->head_dim, a->kv_heads, a->tokens);
  if (rc != 0) return rc;
  const bool has_q = a->q != nullptr;
  if (has_q && (a->q_heads < 1 || a->q_heads > (1 << 20))) return invalid(entry, "q_heads out of range");
  if (a->k == nullptr || has_q != (a->q_out != nullptr) || pages == (a->k_out != nullptr) ||
      pages != (a->v_pages != nullptr) || pages != (a->v != nullptr) || pages != (a->slots != nullptr))
    return invalid(entry, "q with q_out; k with k_out, or k and v with k_pages, v_pages and slots");
  const int64_t strides[] = {a->stride_qt, a->stride_qh, a->stride_kt, a->stride_kh, a->stride_vt, a->stride_vh,
                             a->stride_qot, a->stride_qoh, a->stride_kot, a->stride_koh};
  for (int64_t s : strides)
    if (s % 8) return invalid(entry, "strides must be multiples of 8 elements");
  for (const void* x : {a->q, a->k, a->v, (const void*)a->q_out, (const void*)a->k_out, a->q_weight, a->k_weight})
    if (!aligned(x, 16)) return invalid(entry, "rows and weights must be 16-byte aligned");
  if (a->pairs < 0 || 2 * (int64_t)a->pairs > a->head_dim) return invalid(entry, "at most head_dim / 2 pairs");
  int32_t ends[SA_MAX_ROTARY_AXES] = {};
  if (a->pairs > 0) {
    if (a->positions == nullptr || a->frequencies == nullptr || !aligned(a->positions, a->positions_int64 ? 8 : 4) ||
        !aligned(a->frequencies, 8))
      return invalid(entry, "a rotation needs positions and frequencies");
    if (a->axes < 1 || a->axes > SA_MAX_ROTARY_AXES) return invalid(entry, "1 to 4 axes");
    int32_t end = 0;
    for (int32_t x = 0; x < a->axes; ++x) {
      if (a->sections[x] < 1 || a->sections[x] > a->pairs - end)
        return invalid(entry, "the sections must add up to the pairs");
      ends[x] = end += a->sections[x];
    }
    if (end != a->pairs) return invalid(entry, "the sections must add up to the pairs");
    for (int32_t x = a->axes; x < SA_MAX_ROTARY_AXES; ++x) ends[x] = end;
  }
  RowsParams p{};
  if (pages) {
    rc = check_pool(entry, a->num_pages, a->page_tokens);
    if (rc != 0) return rc;
    if (a->pages_int8 == SA_PAGES_E4M3) return invalid(entry, "rows go into e4m3 pages by sa_append_kv_blocks");
    if (!page_rows(p.kp, a->k_pages, a->k_scales, a) || !page_rows(p.vp, a->v_pages, a->v_scales, a) ||
        !aligned(a->slots, 8))
      return invalid(entry, "pages, scales or slots are missing or not aligned");
    p.num_slots = (uint32_t)(a->num_pages * a->page_tokens);
    p.page_tokens = (uint32_t)a->page_tokens;
    p.slots = a->slots;
  }
  if (a->tokens == 0) return 0;
  p.q = static_cast<const uint16_t*>(a->q), p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.q_out = static_cast<uint16_t*>(a->q_out), p.k_out = static_cast<uint16_t*>(a->k_out);
  p.positions = a->positions, p.frequencies = a->frequencies;
  p.q_weight = a->q_weight, p.k_weight = a->k_weight;
  p.sq_t = a->stride_qt, p.sq_h = a->stride_qh, p.sk_t = a->stride_kt, p.sk_h = a->stride_kh;
  p.sv_t = a->stride_vt, p.sv_h = a->stride_vh;
  p.sqo_t = a->stride_qot, p.sqo_h = a->stride_qoh, p.sko_t = a->stride_kot, p.sko_h = a->stride_koh;
  p.pos_axis = a->stride_pos_axis, p.pos_token = a->stride_pos_token;
  p.eps = (float)a->eps, p.inv_dim = 1.f / (float)a->head_dim;
  p.q_heads = has_q ? a->q_heads : 0, p.kv_heads = a->kv_heads, p.head_dim = a->head_dim;
  p.heads = p.q_heads + p.kv_heads * (pages ? 2 : 1);
  p.pairs = a->pairs;
  p.end0 = ends[0], p.end1 = ends[1], p.end2 = ends[2];
  p.pos64 = a->positions_int64, p.qw32 = a->q_weight_fp32, p.kw32 = a->k_weight_fp32;
  DeviceGuard guard(device);
  SA_HIP_RETURN(guard.status());
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const bool bf16 = a->dtype == SA_DTYPE_BF16;
  p.tokens = a->tokens;
  const bool int8 = pages && a->pages_int8;
  if (!has_q && pages && p.pairs == 0 && p.k_weight == nullptr &&
      p.heads <= rows_per_step(lanes_log2(p.head_dim, 16))) {
    StoreParams s{};
    s.k = p.k, s.v = p.v, s.kp = p.kp, s.vp = p.vp, s.slots = p.slots;
    s.sk_t = p.sk_t, s.sk_h = p.sk_h, s.sv_t = p.sv_t, s.sv_h = p.sv_h, s.tokens = p.tokens;
    s.num_slots = p.num_slots, s.page_tokens = p.page_tokens, s.kv_heads = p.kv_heads, s.head_dim = p.head_dim;
    return bf16 ? launch_store<Bf16>(s, int8, hs) : launch_store<Fp16>(s, int8, hs);
  }
  return bf16 ? launch_rows<Bf16>(p, int8, a->adjacent, hs) : launch_rows<Fp16>(p, int8, a->adjacent, hs);
} catch (const std::exception& error) {
  return sa::exception_status("sa_normalize_rotate_store", error);
}

int32_t sa_read_kv(const sa_read_args* a, int32_t device, void* stream) try {
  using namespace sa;
  const char* entry = "sa_read_kv";
  clear_error();
  if (a == nullptr) return invalid(entry, "null arguments");
  int32_t rc = check_sizes(entry, a->dtype, a->head_dim, a->kv_heads, a->tokens);
  if (rc == 0) rc = check_pool(entry, a->num_pages, a->page_tokens);
  if (rc != 0) return rc;
  ReadParams p{};
  const bool e4m3 = a->pages_int8 == SA_PAGES_E4M3;
  const int64_t scale_align = e4m3 ? 1 : 2;
  if (!page_rows(p.kp, a->k_pages, a->k_scales, a, scale_align) || !page_rows(p.vp, a->v_pages, a->v_scales, a, scale_align))
    return invalid(entry, "pages or scales are missing or not aligned");
  if (e4m3 && (p.block_log2 = block_log2(a->block_tokens, a->page_tokens)) < 0)
    return invalid(entry, "block_tokens must be a power of two from 16 on that divides page_tokens");
  if (a->slots == nullptr || !aligned(a->slots, 8) || a->k_out == nullptr || a->v_out == nullptr ||
      !aligned(a->k_out, 16) || !aligned(a->v_out, 16))
    return invalid(entry, "slots or outputs are missing or not aligned");
  if (a->tokens == 0) return 0;
  if (a->num_pages < 1) return invalid(entry, "the pool must have at least one page");  // row 0 is read for bad slots
  p.k_out = static_cast<uint16_t*>(a->k_out), p.v_out = static_cast<uint16_t*>(a->v_out);
  p.slots = a->slots, p.tokens = a->tokens;
  p.num_slots = (uint32_t)(a->num_pages * a->page_tokens), p.page_tokens = (uint32_t)a->page_tokens;
  p.kv_heads = a->kv_heads, p.head_dim = a->head_dim;
  DeviceGuard guard(device);
  SA_HIP_RETURN(guard.status());
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const bool bf16 = a->dtype == SA_DTYPE_BF16;
  for (p.token0 = 0; p.token0 < a->tokens; p.token0 += kTokensPerLaunch) {
    const dim3 grid((uint32_t)((std::min(a->tokens - p.token0, kTokensPerLaunch) + kReadTokens - 1) / kReadTokens));
    if (e4m3)
      bf16 ? read_kernel<Bf16, kE4m3Pages><<<grid, 256, 0, hs>>>(p) : read_kernel<Fp16, kE4m3Pages><<<grid, 256, 0, hs>>>(p);
    else if (a->pages_int8)
      bf16 ? read_kernel<Bf16, kInt8Pages><<<grid, 256, 0, hs>>>(p) : read_kernel<Fp16, kInt8Pages><<<grid, 256, 0, hs>>>(p);
    else
      bf16 ? read_kernel<Bf16, kRowPages><<<grid, 256, 0, hs>>>(p) : read_kernel<Fp16, kRowPages><<<grid, 256, 0, hs>>>(p);
    SA_HIP_RETURN(hipGetLastError());
  }
  return 0;
} catch (const std::exception& error) {
  return sa::exception_status("sa_read_kv", error);
}

}  // extern "C"
