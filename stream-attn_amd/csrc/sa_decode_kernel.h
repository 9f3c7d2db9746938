// Device code of the decoding attention (see sa_decode.h); included by the
// sources that compile one head size.
//
//   s_j = scale * q . k_j,  out = sum_j e^(s_j) v_j / sum_j e^(s_j),  lse = log sum_j e^(s_j)
//
// Bytes bound: K and V are read once, 4 flop per element and query head.  So
// the kernel is made to keep loads in flight, and the products go where they
// need least else: a wave takes 32 keys per step, all of one K/V head's query
// heads at once in 16x16x32 MFMAs, while the next step's 16 loads are under
// way in registers.
//
// Lane l of a wave is (j = l / 16, g = l % 16).  In step loads t = 0 .. 7 it
// reads the elements of granule g of key 4t + j (16 consecutive lanes read a
// row), for K and for V.
//
// S^T = K Q^T.  K goes through the wave's own LDS (no barrier) to become the A
// operand: row r of 16-key block b is key 16b + 4(r % 4) + r / 4, so that the
// result's element e of block b on lane (j, column) is key 4(4b + e) + j: the
// key of that lane's own load t = 4b + e.
//
// O^T = V^T P^T.  The A operand, V^T, comes from the lane's own loads: row g of
// product i is element i of granule g, its k slots 8j + t the keys 4t + j, which
// are one register half each of the eight loads.  P^T, the B operand, has the
// same keys on the lane as S^T.
//
// Columns 0 - 7 are query heads, columns 8 - 15 the same heads again: their
// logits are the same, and each weight p is split over the two as 16-bit high
// and low part, so P keeps 16 (bfloat16) or 22 (float16) bits at the cost of
// columns that a group of up to 8 heads leaves unused anyway.
#pragma once

#include <cmath>

#include "sa_common.h"
#include "sa_decode.h"

namespace sa {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;

template <typename T>
constexpr float kBias = 0.f;
// float16 weights up to 2^7 of the running maximum's: keys far below it stay
// clear of the type's smallest steps (2^-24).
template <>
constexpr float kBias<Fp16> = 7.f;
// The maximum moves when a logit exceeds it by more than this (log2 units).
constexpr float kSlack = 8.f;

template <int DP>
struct Shape {
  static constexpr int EL = DP == 64 ? 4 : 8;      // elements of a granule
  static constexpr int NP = DP / (16 * EL);        // granules of a lane's row
  static constexpr int NI = NP * EL;               // products of O^T
  static constexpr int NC = DP / 32;               // 32-element chunks of q . k
};

// Orders a wave's own LDS accesses: they execute in program order, the
// compiler must keep them in it.
__device__ inline void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int N>
struct Dwords {
  uint32_t w[N];
};

template <int N>
__device__ inline Dwords<N> load_dwords(const char* base, uint32_t offset) {
  Dwords<N> r;
  const char* p = base + offset;
  if constexpr (N == 4) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(p);
    r.w[0] = x[0], r.w[1] = x[1], r.w[2] = x[2], r.w[3] = x[3];
  } else if constexpr (N == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    r.w[0] = x[0], r.w[1] = x[1];
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return r;
}

__device__ inline int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// The value on the lane whose column is 8 further, of the same 16.
__device__ inline float other_half(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
}

// 2^x of a running maximum's change: 0 from -inf, 1 where nothing changes.
__device__ inline float ratio(float from, float to) { return from == to ? 1.f : __builtin_amdgcn_exp2f(from - to); }

// A wave's loads of one step, in flight while the step before is computed.
template <bool kInt8, int DP, bool kAnyPage>
struct Step {
  static constexpr int EL = Shape<DP>::EL, NP = Shape<DP>::NP;
  static constexpr int RW = kInt8 ? EL / 4 : EL / 2;  // dwords of a granule
  static constexpr int ES = kInt8 ? 1 : 2;            // bytes of an element
  Dwords<RW> k[8][NP], v[8][NP];
  uint32_t scale;  // INT8: lane g's of K (g < 8) or V, key 4 (g % 8) + j
  uint32_t seen;   // bit t: key 4t + j has weight
  bool full;       // all 32 keys have

  // Keys key0 .. key0 + 31 of a sequence with `length` keys.  key0 is in row
  // `row` of page number `page` of the sequence.
  __device__ __attribute__((always_inline)) void load(const DecodeParams& p, const int32_t* table, int head, int32_t key0,
                                                      int32_t length, int32_t page, int32_t row, int j, int g) {
    uint32_t at[NP];
#pragma unroll
    for (int c = 0; c < NP; ++c) at[c] = (128 * c + EL * g < p.head_dim ? 128 * c + EL * g : 0) * ES;
    const bool second = g >= 8;
    if constexpr (!kAnyPage) {
      // Two runs of 16 keys, each in one page.
      bool held = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int32_t n = page, r = row + 16 * h;
        if (r >= p.page_tokens) ++n, r -= p.page_tokens;
        int32_t id = n < p.max_pages ? uniform(table[n]) : -1;
        const bool ok = id >= 0 && id < p.num_pages;
        if (!ok) id = 0;  // rows of a page that exists, read and not used
        held = held && ok;
        const char* kb = p.k + (id * p.kp + r * p.kt + head * p.kh) * ES;
        const char* vb = p.v + (id * p.vp + r * p.vt + head * p.vh) * ES;
        const uint32_t kr = j * (uint32_t)p.kt * ES, vr = j * (uint32_t)p.vt * ES;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < NP; ++c) k[4 * h + u][c] = load_dwords<RW>(kb + 4 * u * p.kt * ES, kr + at[c]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < NP; ++c) v[4 * h + u][c] = load_dwords<RW>(vb + 4 * u * p.vt * ES, vr + at[c]);
        if constexpr (kInt8) {
          const uint16_t* s = second ? p.vs + id * p.vsp + r * p.vst + head * p.vsh : p.ks + id * p.ksp + r * p.kst + head * p.ksh;
          if ((g >> 2 & 1) == h) scale = s[(4 * (g & 3) + j) * (second ? p.vst : p.kst)];
        }
        const uint32_t mask = ok ? 15u : 0u;
        seen = h == 0 ? mask : seen | mask << 4;
      }
      full = held && key0 + kDecodeTile <= length;
    } else {
      seen = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int32_t key = key0 + 4 * t + j;
        const int32_t n = (int32_t)((uint64_t)(uint32_t)key * p.page_magic >> p.page_shift);
        const int32_t r = key - n * p.page_tokens;
        int32_t id = n < p.max_pages ? table[n] : -1;
        const bool ok = id >= 0 && id < p.num_pages;
        if (!ok) id = 0;
        seen |= (uint32_t)ok << t;
        const char* kb = p.k + (id * p.kp + r * p.kt + head * p.kh) * ES;
        const char* vb = p.v + (id * p.vp + r * p.vt + head * p.vh) * ES;
#pragma unroll
        for (int c = 0; c < NP; ++c) k[t][c] = load_dwords<RW>(kb, at[c]), v[t][c] = load_dwords<RW>(vb, at[c]);
        if constexpr (kInt8)
          if ((g & 7) == t) scale = second ? p.vs[id * p.vsp + r * p.vst + head * p.vsh] : p.ks[id * p.ksp + r * p.kst + head * p.ksh];
      }
      full = __all(seen == 255u) && key0 + kDecodeTile <= length;
    }
    if (key0 + kDecodeTile > length) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (key0 + 4 * t + j >= length) seen &= ~(1u << t);
    }
  }
};

// Part of a sequence's keys, for one item: maximum, sum and O^T per query head.
template <typename T, bool kInt8, int DP, int NB, bool kAnyPage>
__global__ __launch_bounds__(64 * kDecodeWaves, DP == 256 ? 1 : 2) void decode_kernel(const DecodeParams p) {
  using S = Shape<DP>;
  using PT = std::conditional_t<kInt8, Bf16, T>;  // INT8: weights times V's scales, beyond float16's range
  constexpr int EL = S::EL, NP = S::NP, NI = S::NI, NC = S::NC;
  constexpr float bias = kBias<PT>;
  constexpr int kRow = 2 * DP;  // bytes of a key in LDS
  __shared__ __attribute__((aligned(16))) char lds[kDecodeWaves][kDecodeTile * kRow + (kInt8 ? 256 : 0)];
  __shared__ float stats[kDecodeWaves][8 * NB][2];
  __shared__ int64_t found[3];

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int j = lane >> 4, g = lane & 15;
  const int items = p.kv_heads * p.blocks;
  const int w = blockIdx.x, workgroups = gridDim.x;
  const auto length_of = [&](int s) {
    const int32_t n = p.lengths[s];
    return n < p.room ? n : p.room;
  };
  const auto tiles_of = [&](int s) {
    const int32_t n = length_of(s);
    return n > 0 ? (n + kDecodeTile - 1) / kDecodeTile : 0;
  };

  // Tiles before every thread's run of sequences; the workgroup's range.
  int64_t* sums = reinterpret_cast<int64_t*>(&lds[0][0]);
  const int run = (p.sequences + 64 * kDecodeWaves - 1) / (64 * kDecodeWaves);
  const int s_first = tid * run, s_last = s_first + run < p.sequences ? s_first + run : p.sequences;
  int64_t own = 0;
  for (int s = s_first; s < s_last; ++s) own += tiles_of(s);
  int64_t upto = own;  // inclusive
  for (int i = 1; i < 64; i <<= 1) {
    const int64_t x = __shfl_up(upto, i);
    if (lane >= i) upto += x;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int64_t total = 0;
  for (int i = 0; i < kDecodeWaves; ++i) {
    if (i < wave) upto += sums[i];
    total += sums[i];
  }
  total *= items;
  // At least a tile for each of its waves.
  int64_t share = (total + workgroups - 1) / workgroups;
  if (share < kDecodeWaves) share = kDecodeWaves;
  const int64_t begin = w * share, end = begin + share < total ? begin + share : total;
  if (begin < end && (upto - own) * items <= begin && begin < upto * items) {
    int64_t before = upto - own;
    int s = s_first;
    for (; s < s_last; ++s) {
      const int64_t n = tiles_of(s);
      if (begin < (before + n) * items) break;
      before += n;
    }
    found[0] = s, found[1] = before * items;
  }
  // Sequences without keys have no tiles.
  for (int s = w; s < p.sequences; s += workgroups) {
    if (length_of(s) > 0) continue;
    for (int i = tid; i < p.kv_heads * p.group * (p.head_dim / 8); i += 64 * kDecodeWaves) {
      const int h = i / (p.head_dim / 8), d = 8 * (i - h * (p.head_dim / 8));
      *reinterpret_cast<u32x4*>(p.out + s * p.so_t + h * p.so_h + d) = u32x4{0, 0, 0, 0};
      if (d == 0 && p.lse != nullptr) p.lse[h * p.lse_h + s] = -INFINITY;
    }
  }
  __syncthreads();
  if (tid == 0) p.owned[4 * w] = -1;
  if (begin >= end) return;

  char* mine = &lds[wave][0];
  float* scales = reinterpret_cast<float*>(mine + kDecodeTile * kRow);
  int s = uniform((int)found[0]);
  int64_t at = begin;        // the next tile
  int64_t s_start = found[1];  // the sequence's first
  while (at < end) {
    int32_t tiles = uniform(tiles_of(s));
    while (at >= s_start + (int64_t)tiles * items) {
      s_start += (int64_t)tiles * items;
      tiles = uniform(tiles_of(++s));
    }
    const int32_t length = uniform(length_of(s));
    const int item = uniform((int)((at - s_start) / tiles));
    const int64_t item_start = s_start + (int64_t)item * tiles, item_end = item_start + tiles;
    const int32_t first = uniform((int32_t)(at - item_start));
    const int32_t last = uniform((int32_t)((item_end < end ? item_end : end) - item_start));
    const int kv_head = item / p.blocks;
    const int h0 = (item - kv_head * p.blocks) * 8 * NB;                  // of the group
    const int heads = p.group - h0 < 8 * NB ? p.group - h0 : 8 * NB;
    const int32_t* table = p.table + s * p.s_table;

    // Q^T: chunk c of column g's head, elements 32c + 8j .. + 7.
    u32x4 q[NB][NC];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int h = 8 * n + (g & 7);
      const uint16_t* row = p.q + s * p.sq_t + (kv_head * p.group + h0 + (h < heads ? h : 0)) * p.sq_h;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = 32 * c + 8 * j;
        q[n][c] = h < heads && d < p.head_dim ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0, 0, 0, 0};
      }
    }
    // K's elements past head_dim are zeros that no step writes.
    if (p.head_dim < DP) {
      for (int i = lane; i < kDecodeTile * kRow / 16; i += 64) reinterpret_cast<u32x4*>(mine)[i] = u32x4{0, 0, 0, 0};
      wave_lds_order();
    }

    f32x4 acc[NB][NI];
    float m[NB], l[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    Step<kInt8, DP, kAnyPage> step;
    int32_t tile = first + wave;
    int32_t page = uniform((int32_t)((uint64_t)(uint32_t)(tile * kDecodeTile) * p.page_magic >> p.page_shift));
    int32_t row = tile * kDecodeTile - page * p.page_tokens;
    if (tile < last) step.load(p, table, kv_head, tile * kDecodeTile, length, page, row, j, g);
    while (tile < last) {
      // K to LDS, 16-byte granules of row r exchanged by r so that the reads
      // below meet every bank once.
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int r = 4 * t + j;
        const int turn = DP == 64 ? r >> 1 & 7 : r & 15;
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          if (128 * c + EL * g >= p.head_dim) continue;
          uint32_t x[EL / 2];
          if constexpr (kInt8) {
#pragma unroll
            for (int i = 0; i < EL / 2; ++i)
              x[i] = T::pack(byte_float(step.k[t][c].w[i / 2], 2 * (i & 1)), byte_float(step.k[t][c].w[i / 2], 2 * (i & 1) + 1));
          } else {
#pragma unroll
            for (int i = 0; i < EL / 2; ++i) x[i] = step.k[t][c].w[i];
          }
          if constexpr (EL == 8)
            *reinterpret_cast<u32x4*>(mine + r * kRow + 16 * ((16 * c + g) ^ turn)) = u32x4{x[0], x[1], x[2], x[3]};
          else
            *reinterpret_cast<u32x2*>(mine + r * kRow + 16 * ((g >> 1) ^ turn) + 8 * (g & 1)) = u32x2{x[0], x[1]};
        }
      }
      if constexpr (kInt8) scales[16 * j + g] = Fp16::lo(step.scale);
      const bool full = step.full;
      const uint32_t seen = step.seen;
      // Rows without weight may hold anything: 0 * NaN is not 0.
      if (!full) {
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (!(seen >> t & 1)) {
#pragma unroll
            for (int c = 0; c < NP; ++c)
#pragma unroll
              for (int i = 0; i < step.RW; ++i) step.v[t][c].w[i] = 0;
          }
      }
      // V^T: product i's keys, a pair of loads per dword.
      u32x4 vt[NI];
#pragma unroll
      for (int c = 0; c < NP; ++c)
#pragma unroll
        for (int i = 0; i < EL; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if constexpr (kInt8)
              vt[EL * c + i][u] = PT::pack(byte_float(step.v[2 * u][c].w[i / 4], i & 3), byte_float(step.v[2 * u + 1][c].w[i / 4], i & 3));
            else
              vt[EL * c + i][u] = __builtin_amdgcn_perm(step.v[2 * u + 1][c].w[i / 2], step.v[2 * u][c].w[i / 2],
                                                        i & 1 ? 0x07060302u : 0x05040100u);
          }
      tile += kDecodeWaves;
      if (tile < last) {
        page += p.step_pages, row += p.step_rows;
        if (row >= p.page_tokens) ++page, row -= p.page_tokens;
        step.load(p, table, kv_head, tile * kDecodeTile, length, page, row, j, g);
      }
      wave_lds_order();

      f32x4 st[NB][2];
#pragma unroll
      for (int n = 0; n < NB; ++n) st[n][0] = st[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int r = 16 * b + 4 * (g & 3) + (g >> 2);
          const int turn = DP == 64 ? r >> 1 & 7 : r & 15;
          const u32x4 a = *reinterpret_cast<const u32x4*>(mine + r * kRow + 16 * ((4 * c + j) ^ turn));
#pragma unroll
          for (int n = 0; n < NB; ++n) st[n][b] = T::mma(a, q[n][c], st[n][b]);
        }
      float ks[8], vs[8];
      if constexpr (kInt8) {
#pragma unroll
        for (int t = 0; t < 8; t += 4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(scales + 16 * j + t), y = *reinterpret_cast<const f32x4*>(scales + 16 * j + 8 + t);
#pragma unroll
          for (int i = 0; i < 4; ++i) ks[t + i] = x[i], vs[t + i] = seen >> (t + i) & 1 ? y[i] : 0.f;
        }
      }
      wave_lds_order();
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float y[8], top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          y[t] = st[n][t / 4][t & 3] * p.scale_log2;
          if constexpr (kInt8) y[t] *= ks[t];
          if (!full && !(seen >> t & 1)) y[t] = -INFINITY;
          top = fmaxf(top, y[t]);
        }
        if (__any(top > m[n] + (bias + kSlack))) {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32)) - bias;
          const float next = fmaxf(m[n], top), keep = ratio(m[n], next);
          m[n] = next;
          l[n] *= keep;
#pragma unroll
          for (int i = 0; i < NI; ++i) acc[n][i] *= keep;
        }
        const float base = m[n] == -INFINITY ? 0.f : m[n];
        const float low = g >= 8 ? 1.f : 0.f;
        u32x4 weights;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float a = __builtin_amdgcn_exp2f(y[2 * u] - base), b = __builtin_amdgcn_exp2f(y[2 * u + 1] - base);
          l[n] += a + b;
          if constexpr (kInt8) a *= vs[2 * u], b *= vs[2 * u + 1];
          const uint32_t high = PT::pack(a, b);
          weights[u] = PT::pack(a - low * PT::lo(high), b - low * PT::hi(high));
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[n][i] = PT::mma(vt[i], weights, acc[n][i]);
      }
    }

    // The waves' parts: maxima and sums first, then O^T at the common maximum.
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      l[n] += __shfl_xor(l[n], 16);
      l[n] += __shfl_xor(l[n], 32);
      if (lane < 8) stats[wave][8 * n + lane][0] = m[n], stats[wave][8 * n + lane][1] = l[n];
    }
    __syncthreads();
    float* part = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float top = -INFINITY;
      for (int i = 0; i < kDecodeWaves; ++i) top = fmaxf(top, stats[i][8 * n + (g & 7)][0]);
      const float f = ratio(m[n], top);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = acc[n][i][e] * f;
          acc[n][i][e] = x + other_half(x);
        }
      if (g < 8) {
#pragma unroll
        for (int c = 0; c < NP; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < EL; i += 4)
              *reinterpret_cast<f32x4*>(part + (8 * n + g) * DP + 128 * c + EL * (4 * j + e) + i) =
                  f32x4{acc[n][EL * c + i][e], acc[n][EL * c + i + 1][e], acc[n][EL * c + i + 2][e], acc[n][EL * c + i + 3][e]};
      }
    }
    __syncthreads();
    const bool starts = first == 0, ends = last == tiles;
    float* slot = p.parts + ((int64_t)w * 2 + (starts ? 1 : 0)) * (8 * NB * (DP + 2));
    for (int i = tid; i < heads * (DP / 4); i += 64 * kDecodeWaves) {
      const int h = i / (DP / 4), d = 4 * (i % (DP / 4));
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float top = -INFINITY, weight = 0.f;
#pragma unroll
      for (int x = 0; x < kDecodeWaves; ++x) {
        sum += *reinterpret_cast<const f32x4*>(&lds[x][0] + (h * DP + d) * 4);
        top = fmaxf(top, stats[x][h][0]);
      }
#pragma unroll
      for (int x = 0; x < kDecodeWaves; ++x) weight += stats[x][h][1] * ratio(stats[x][h][0], top);
      if (starts && ends) {
        const int head = kv_head * p.group + h0 + h;
        const float inv = weight == 0.f ? 0.f : 1.f / weight;
        if (d < p.head_dim) {
          const u32x2 o = {T::pack(sum[0] * inv, sum[1] * inv), T::pack(sum[2] * inv, sum[3] * inv)};
          *reinterpret_cast<u32x2*>(p.out + s * p.so_t + head * p.so_h + d) = o;
        }
        if (d == 0 && p.lse != nullptr) p.lse[head * p.lse_h + s] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * kLn2;
      } else {
        *reinterpret_cast<f32x4*>(slot + h * DP + d) = sum;
        if (d == 0) slot[8 * NB * DP + 2 * h] = top, slot[8 * NB * DP + 2 * h + 1] = weight;
      }
    }
    if (starts && !ends && tid == 0) {
      p.owned[4 * w] = s, p.owned[4 * w + 1] = item;
      p.owned[4 * w + 2] = (int32_t)((item_end - 1) / share);
    }
    __syncthreads();
    at = item_start + last;
  }
}

// An item split over workgroups w .. last: its parts joined, one workgroup per
// query head, a lane per four elements, the parts dealt to groups of lanes.
template <typename T, int DP, int NB>
__global__ __launch_bounds__(128) void join_kernel(const DecodeParams p) {
  constexpr int kLanes = DP / 4, kGroups = 128 / kLanes, kSlot = 8 * NB * (DP + 2);
  __shared__ f32x4 sums[kGroups][kLanes];
  __shared__ float stats[kGroups][2];
  const int w = blockIdx.x, h = blockIdx.y;
  const int s = p.owned[4 * w];
  if (s < 0) return;
  const int item = p.owned[4 * w + 1], last = p.owned[4 * w + 2];
  const int kv_head = item / p.blocks, h0 = (item - kv_head * p.blocks) * 8 * NB;
  if (h0 + h >= p.group) return;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const auto slot = [&](int i) { return p.parts + ((int64_t)i * 2 + (i == w ? 1 : 0)) * kSlot; };
  float top = -INFINITY, weight = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = w + group; i <= last; i += kGroups) top = fmaxf(top, slot(i)[8 * NB * DP + 2 * h]);
  for (int i = w + group; i <= last; i += kGroups) {
    const float* part = slot(i);
    const float f = ratio(part[8 * NB * DP + 2 * h], top);
    weight += part[8 * NB * DP + 2 * h + 1] * f;
    sum += *reinterpret_cast<const f32x4*>(part + h * DP + 4 * lane) * f;
  }
  sums[group][lane] = sum;
  if (lane == 0) stats[group][0] = top, stats[group][1] = weight;
  __syncthreads();
  if (group != 0) return;
  for (int i = 1; i < kGroups; ++i) top = fmaxf(top, stats[i][0]);
  sum = f32x4{0.f, 0.f, 0.f, 0.f}, weight = 0.f;
  for (int i = 0; i < kGroups; ++i) {
    const float f = ratio(stats[i][0], top);
    weight += stats[i][1] * f;
    sum += sums[i][lane] * f;
  }
  const int head = kv_head * p.group + h0 + h, d = 4 * lane;
  const float inv = weight == 0.f ? 0.f : 1.f / weight;
  if (d < p.head_dim)
    *reinterpret_cast<u32x2*>(p.out + s * p.so_t + head * p.so_h + d) =
        u32x2{T::pack(sum[0] * inv, sum[1] * inv), T::pack(sum[2] * inv, sum[3] * inv)};
  if (lane == 0 && p.lse != nullptr) p.lse[head * p.lse_h + s] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * kLn2;
}

template <typename T, bool kInt8, int DP, int NB>
void launch_decode(const DecodeLaunch& l) {
  if (l.any_page)
    decode_kernel<T, kInt8, DP, NB, true><<<l.workgroups, 64 * kDecodeWaves, 0, l.stream>>>(l.p);
  else
    decode_kernel<T, kInt8, DP, NB, false><<<l.workgroups, 64 * kDecodeWaves, 0, l.stream>>>(l.p);
  const int heads = l.p.group < 8 * NB ? l.p.group : 8 * NB;
  join_kernel<T, DP, NB><<<dim3(l.workgroups, heads), 128, 0, l.stream>>>(l.p);
}

template <typename T, int DP>
void launch_decode(const DecodeLaunch& l) {
  if (l.int8)
    l.wide ? launch_decode<T, true, DP, 2>(l) : launch_decode<T, true, DP, 1>(l);
  else
    l.wide ? launch_decode<T, false, DP, 2>(l) : launch_decode<T, false, DP, 1>(l);
}

}  // namespace
}  // namespace sa
