// Device code of a prompt's attention over the paged cache; included by the
// sources that compile one head size.
//
//   s_ij = scale * q_i . k_j over the keys j <= p_i with p_i - j < window or j < sinks
//   out_i = sum_j e^(s_ij) v_j / sum_j e^(s_ij),  lse_i = log sum_j e^(s_ij)
//
// One pass over a row's keys with the running maximum and sum.
//
// Matrix bound for long prompts: 4 * head_dim flop per visible (row, key), bytes only
// once per block of 128 to 384 rows.  A row is a (token, query head) pair of one K/V
// head, so that a K/V tile of 64 keys in LDS serves all heads of the group.  Eight waves
// have 16 to 48 rows each: S^T = K Q^T leaves the weights on the lanes where O^T =
// V^T P^T takes them, the layouts are the update kernel's.  Tiles come by asynchronous
// loads, one to three ahead; 8-bit ones through a raw buffer, converted by the first wave
// of a SIMD before its products and by the second one after them.
//
// Measured (a library product reaches 1,620 TFLOP/s): 61,312 tokens, 56/8 heads of 128,
// window 4,096, 5.9 ms, 1,181 TFLOP/s; 2,000 tokens behind 129,072 e4m3 keys, 40/8 heads,
// 5.0 ms, 1,056 TFLOP/s; 20,011 tokens of 7 sequences 0.56 ms, 1,024 TFLOP/s (a card whose
// clock falls lower under load: 1,067, 1,031 and 955).  A tile of
// 384 rows takes 2.4 us (1,300 TFLOP/s), matrix and vector units half busy each and meeting
// only in part with two waves per SIMD; an item 13 us to start and end.
#pragma once

#include <cmath>
#include <type_traits>

#include "sa_prefill.h"
#include "sa_update_kernel.h"

namespace sa {
namespace {

template <typename T>
__device__ inline __attribute__((always_inline)) T uniform(T x) {
  if constexpr (sizeof(T) == 8) {
    const uint64_t v = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return __builtin_bit_cast(T, (uint64_t)lo | (uint64_t)hi << 32);
  } else {
    return __builtin_amdgcn_readfirstlane(x);
  }
}

// 2^x of a running maximum's change: 0 from -inf, 1 where nothing changes.
__device__ inline float prefill_ratio(float from, float to) { return from == to ? 1.f : __builtin_amdgcn_exp2f(from - to); }

// A weight is held at most 2^kWeightTop; a new maximum's is 2^kWeightShift.  float16
// weights lie high in their range, so that those of 2^-32 of the largest still count.
template <typename W>
constexpr int kWeightTop = std::is_same_v<W, Fp16> ? 15 : 8;
template <typename W>
constexpr int kWeightShift = std::is_same_v<W, Fp16> ? 7 : 0;

// Bits 15 and 31: the halves of a dword that are infinite or NaN (all ones in the
// exponent, which one more carries over).
template <typename T>
__device__ inline uint32_t not_finite(uint32_t w) {
  constexpr bool bf16 = std::is_same_v<T, Bf16>;
  return ((w & (bf16 ? 0x7f807f80u : 0x7c007c00u)) + (bf16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
// The larger magnitudes of the halves, as bits.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ inline u16x2 larger(u16x2 top, uint32_t w) {
  return __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w & 0x7fff7fffu));
}
// Bits 0 .. n - 1.
__device__ inline uint32_t below(int n) { return n > 0 ? ~0u >> (32 - (n < 32 ? n : 32)) : 0u; }
// Bits 15 and 31: bits n and n + 1.
__device__ inline uint32_t two_bits(uint32_t bits, int n) { return (bits >> n & 1) << 15 | (bits >> n & 2) << 30; }
// Halves of ones where those bits are.
__device__ inline uint32_t halves(uint32_t m) { return (m - (m >> 15)) | m; }

// The kernel's arguments, read again where they are used: what only a piece's ends
// and masked steps need would otherwise sit in scalar registers, and those that do
// not fit in lanes of vector registers, all through the loop over the tiles.
typedef const PrefillParams SA_CONSTANT* PrefillArguments;
__device__ inline PrefillArguments prefill_arguments() {
  PrefillArguments a = (PrefillArguments)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}

template <typename T, int DP, int QB, PageKind kKind, int STAGES>
__global__ __launch_bounds__(kPrefillThreads, 2 * prefill_occupancy(DP, 128 * QB, kKind)) void prefill_kernel(const PrefillParams p) {
  using Geo = Geometry<DP>;
  constexpr bool QUANT = kKind != kRowPages;
  // What weights and V enter their product as, each rounded once.  A second 16-bit part of
  // the weights, which single tokens have, would double this product, half of the matrix
  // work: so outputs in bfloat16 are 0.0020 to 0.0023 of their norm off, 0.0016 of it by
  // their own rounding, as the update kernel's are; in float16 0.00026 and 0.0002.  INT8
  // times a float16 scale has three bits more in float16 than in bfloat16: 0.0017.
  using W = std::conditional_t<kKind == kInt8Pages, Fp16, T>;
  constexpr int CK = Geo::CK, DB = Geo::DB;
  constexpr int KB = DP == 256 ? (QB == 1 ? 4 : 2) : CK;
  constexpr int VB = DP == 256 ? (QB == 1 ? 8 : 4) : DP == 128 && QB > 1 ? 8 : 4;
  constexpr int BLOCK_M = Geo::WAVES * 16 * QB;
  constexpr int STAGE_BYTES = 2 * Geo::TILE_BYTES;
  constexpr int RAW_BYTES = Geo::I8_TILE_BYTES;  // of K or V of a raw tile
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * STAGE_BYTES];
  __shared__ __attribute__((aligned(1024))) uint8_t raw[QUANT ? 4 * RAW_BYTES : 16];
  // Of the tiles in flight: which keys are in a page of the pool; by key what a logit's
  // FMA multiplies it by, and what K's and V's values are converted with.
  __shared__ __attribute__((aligned(8))) uint16_t seen_lds[4][4];
  __shared__ __attribute__((aligned(16))) float scale_lds[QUANT ? 4 : 1][3][kTileKeys];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r16 = lane & 15, j = lane >> 4;
  const bool issues = wave < 4;

  // The run of tiles of this workgroup; neighbouring runs are on one XCD.
  const int run = (blockIdx.x & 7) * (p.runs >> 3) + (blockIdx.x >> 3);
  const int64_t tiles = uniform(p.plan->tiles);
  const int blocks = uniform(p.plan->blocks);
  const int64_t total = tiles * p.kv_heads, share = (total + p.runs - 1) / p.runs;
  const int64_t begin = run * share, end = begin + share < total ? begin + share : total;
  if (tid == 0) p.splits[run].block = -1;
  const bool whole_items = uniform(p.plan->whole);
  if (total == 0 || (!whole_items && begin >= end)) return;

  // Elements of K past head_dim are zeros that no tile writes.
  if (p.head_dim < DP) {
    for (int i = tid; i < STAGES * STAGE_BYTES / 16; i += kPrefillThreads)
      reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
  }

  // The block that the run starts in: 64 of them looked at at once.
  int head = 0, block = 0;
  if (!whole_items) {
    head = (int)(begin / tiles);
    const int64_t into = begin - head * tiles;
    for (int left = blocks; left > 1;) {
      const int step = (left + 63) >> 6, at = lane * step;
      const bool before = at < left && p.blocks[block + (at < left ? at : 0)].before <= into;
      const int skipped = (__popcll(__ballot(before)) - 1) * step;
      block += skipped;
      left = min(step, left - skipped);
    }
  }

  // Whole items: the next of this XCD's.
  __shared__ int32_t next_lds;
  constexpr int kFetcher = kPrefillThreads - 64;  // a wave that issues no loads
  const int xcd = blockIdx.x & 7;
  int fetched = 0;
  if (whole_items && tid == kFetcher) next_lds = atomicAdd(&p.plan->next[xcd], 1);

  // What a wave wrote to LDS, and loaded and stored, is through before the others go on: the
  // compiler leaves this wait out here, and which keys are in a page came too late for some.
  const auto barrier = []() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
  };
  const float cf = scale_factor(p.scale_log2);
  for (int64_t at = begin; whole_items || at < end;) {
    barrier();  // the stages are free (and, at first, cleared)
    if (whole_items) {
      const int item = 8 * uniform(next_lds) + xcd;
      if (item >= blocks * p.kv_heads) break;
      block = uniform(p.order[item / p.kv_heads]), head = item % p.kv_heads;
      if (tid == kFetcher) fetched = atomicAdd(&p.plan->next[xcd], 1);
    }
    // ---- a piece: tiles first .. last - 1 of an item ----
    const int64_t before = uniform(p.blocks[block].before) + head * tiles;
    const int s = uniform(p.blocks[block].sequence), row0 = uniform(p.blocks[block].row);
    PrefillSequence seq = prefill_sequence(p, s);
    seq.from = uniform(seq.from), seq.count = uniform(seq.count), seq.base = uniform(seq.base);
    const int rows = min(seq.count * p.group, row0 + BLOCK_M);  // end of the block's rows
    PrefillTiles span = prefill_tiles(p, seq, row0, rows);
    span.count = uniform(span.count), span.sinks = uniform(span.sinks), span.skip = uniform(span.skip);
    const int first = whole_items ? 0 : (int)(at - before);
    const int last = whole_items ? span.count : (int)min((int64_t)span.count, end - before);
    const int ntiles = last - first;
    const int32_t* table = p.table + s * p.s_table;

    // Rows of this wave, and the bounds of what they see: no key at or past
    // wave_end, every (window's) key before wave_first; no key below low_first but
    // the sinks, every key (before wave_first) from low_last on.
    const int qw0 = row0 + wave * 16 * QB;
    const bool has_rows = qw0 < rows;
    const int pos_first = uniform(seq.base + prefill_query(p, min(qw0, rows - 1)));
    const int pos_last = uniform(seq.base + prefill_query(p, min(qw0 + 16 * QB, rows) - 1));
    const int wave_end = has_rows ? pos_last + 1 : 0, wave_first = pos_first + 1;
    const int low_first = (int)max((int64_t)pos_first - p.window + 1, (int64_t)0);
    const int low_last = (int)max((int64_t)pos_last - p.window + 1, (int64_t)0);

    // ---- loads ----
    // Issuing wave w has keys 16 w .. + 15 of every tile, in one page where pages are
    // multiples of 16.  Where those of tiles held_first .. + 63 are (-1: in no page), and
    // their scales (INT8: where they are), it then looks up at once and keeps in LDS: in
    // registers read across lanes they did not outlive what the compiler does with
    // registers where only some lanes are on.
    constexpr int ES = QUANT ? 1 : 2;
    const char* k_head = p.k + head * p.sh * ES;
    const char* v_head = p.v + head * p.sh * ES;
    int held_first = first - 64;
    __shared__ int64_t held_lds[4][64];
    __shared__ int64_t held_scales_at[kKind == kInt8Pages ? 4 : 1][64];
    __shared__ float held_scales[kKind == kE4m3Pages ? 4 : 1][2][64];
    const auto page_of = [](const auto& a, int key, int& row) {
      const int number = (int)((uint64_t)(uint32_t)key * a.page_magic >> a.page_shift);
      row = key - number * a.page_tokens;
      return number;
    };
    // The page and row of a key; a row that exists, read and not used, where there is no page.
    const auto find = [&](const auto& a, int key, int& row, bool& ok) {
      const int number = page_of(a, key, row);
      int id = number < a.max_pages ? table[number] : -1;
      ok = (uint32_t)id < (uint32_t)a.num_pages;
      if (!ok) id = row = 0;
      return id;
    };
    const auto hold = [&](int tile) {
      const auto& a = *prefill_arguments();
      held_first = tile;
      int row;
      bool ok;
      const int id = find(a, span.key_of(min(tile + lane, last - 1)) + 16 * wave, row, ok);
      const int64_t at = id * a.sp + row * a.st;
      held_lds[wave][lane] = ok ? at * ES : -1;
      if constexpr (kKind == kE4m3Pages) {
        const int64_t scale = id * a.ssp + (row >> a.block_log2) * a.sst + head * a.ssh;
        held_scales[wave][0][lane] = e8m0_value(static_cast<const uint8_t*>(a.ks)[scale]);
        held_scales[wave][1][lane] = e8m0_value(static_cast<const uint8_t*>(a.vs)[scale]);
      }
      if constexpr (kKind == kInt8Pages) {
        held_scales_at[wave][lane] = id * a.ssp + row * a.sst + head * a.ssh;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    // A wave-uniform address plus 32 bits per lane.
    auto dma = [](const char* base, uint32_t offset, uint8_t* dst) __attribute__((always_inline)) {
      asm volatile("" : "+s"(base));
      __builtin_amdgcn_global_load_lds((const SA_GLOBAL void*)(base + offset), (SA_LDS void*)dst, 16, 0, 0);
    };
    // INT8 scales of the raw tile in flight: lane l's of key l % 16, K's (l < 16) or V's.
    uint16_t scale_next = 0;
    // K's scales go into the logits, their sign (and NaN) into the values; a factor of at
    // least the smallest normal keeps a masked logit at -inf.
    const auto put = [&](int tile, float scale) __attribute__((always_inline)) {
      if (lane >= 32) return;
      float(&to)[3][kTileKeys] = scale_lds[QUANT ? tile & 3 : 0];
      const int key = 16 * wave + r16;
      if (j == 0) {
        to[0][key] = scale == scale ? fmaxf(fabsf(scale) * cf, 1.17549435e-38f) : cf;
        to[1][key] = scale == scale ? (scale < 0.f ? -1.f : 1.f) : NAN;
      } else {
        to[2][key] = scale;
      }
    };
    // Tile `tile`: its 16-bit rows to the stage, or its bytes to the raw buffer.
    auto issue_tile = [&](int tile, uint8_t* to) __attribute__((always_inline)) {
      if (!issues) return;
      int l = lane;
      if constexpr (QB > 1 && DP >= 128) asm volatile("" : "+v"(l));  // lane offsets anew: registers are short
      const int key = QUANT ? l * 16 / DP : l >> 2;  // a lane's of a wave-wide load's
      constexpr int KEYS = QUANT ? 1024 / DP : 16;
      uint32_t seen;
      if (__builtin_expect(!p.any_page, 1)) {
        if (tile - held_first >= 64) hold(tile);
        const int x = tile - held_first;
        const int64_t held = uniform(held_lds[wave][x]), at = held < 0 ? 0 : held;
        seen = held < 0 ? 0u : 0xffffu;
        // Without a page every lane reads row 0 of one that exists.
        const uint32_t step = seen ? (uint32_t)p.st * ES : 0u;
        if constexpr (QUANT) {
          const int d = l * 16 % DP;
          const uint32_t offset = key * step + (d < p.head_dim ? d : 0);
#pragma unroll
          for (int i = 0; i < 16 / KEYS; ++i) {
            dma(k_head + at + (int64_t)i * KEYS * step, offset, to + wave * 16 * DP + i * 1024);
            dma(v_head + at + (int64_t)i * KEYS * step, offset, to + RAW_BYTES + wave * 16 * DP + i * 1024);
          }
          if constexpr (kKind == kE4m3Pages)
            put(tile, held_scales[wave][j & 1][x]);
        } else {
          const int kd = 8 * Geo::k_granule((l & 3) ^ (l >> 4)), vd = 8 * ((l & 3) ^ (2 * ((l >> 4) & 1)));
          const uint32_t k_offset = key * step + kd * ES, v_offset = key * step + vd * ES;
          if (__builtin_expect(p.head_dim == DP, 1)) {
#pragma unroll
            for (int c = 0; c < CK; ++c) {
              dma(k_head + at + 32 * c * ES, k_offset, to + (CK * wave + c) * 1024);
              dma(v_head + at + 32 * c * ES, v_offset, to + Geo::TILE_BYTES + (4 * c + wave) * 1024);
            }
          } else {
            for (int c = 0; c < CK; ++c) {
              if (32 * c + kd < p.head_dim) dma(k_head + at + 32 * c * ES, k_offset, to + (CK * wave + c) * 1024);
              if (32 * c + vd < p.head_dim)
                dma(v_head + at + 32 * c * ES, v_offset, to + Geo::TILE_BYTES + (4 * c + wave) * 1024);
            }
          }
        }
      } else {
        // Pages that end anywhere: every lane looks for its key.
        const auto& a = *prefill_arguments();
        seen = 0;
        for (int i = 0; i < 16 / KEYS; ++i) {
          int row;
          bool ok;
          const int id = find(a, span.key_of(tile) + 16 * wave + i * KEYS + key, row, ok);
          const char *k_row = k_head + (id * a.sp + row * a.st) * ES, *v_row = v_head + (id * a.sp + row * a.st) * ES;
          const uint64_t held = __ballot(ok);
          const auto dma_lane = [](const char* at, uint8_t* dst) {
            __builtin_amdgcn_global_load_lds((const SA_GLOBAL void*)at, (SA_LDS void*)dst, 16, 0, 0);
          };
          for (int k = 0; k < KEYS; ++k) seen |= (uint32_t)(held >> (k * (64 / KEYS)) & 1) << (i * KEYS + k);
          if constexpr (QUANT) {
            const int d = l * 16 % DP < a.head_dim ? l * 16 % DP : 0;
            dma_lane(k_row + d, to + wave * 16 * DP + i * 1024);
            dma_lane(v_row + d, to + RAW_BYTES + wave * 16 * DP + i * 1024);
          } else {
            const int kd = 8 * Geo::k_granule((l & 3) ^ (l >> 4)), vd = 8 * ((l & 3) ^ (2 * ((l >> 4) & 1)));
            for (int c = 0; c < CK; ++c) {
              if (32 * c + kd < a.head_dim) dma_lane(k_row + (32 * c + kd) * ES, to + (CK * wave + c) * 1024);
              if (32 * c + vd < a.head_dim) dma_lane(v_row + (32 * c + vd) * ES, to + Geo::TILE_BYTES + (4 * c + wave) * 1024);
            }
          }
        }
      }
      if constexpr (kKind == kInt8Pages) {
        const uint16_t* from = static_cast<const uint16_t*>(j & 1 ? p.vs : p.ks);
        if (__builtin_expect(!p.any_page, 1)) {
          const int x = tile - held_first;
          from += held_scales_at[wave][x] + (seen ? r16 * p.sst : 0);
        } else {
          const auto& a = *prefill_arguments();
          int row;
          bool ok;
          const int id = find(a, span.key_of(tile) + 16 * wave + r16, row, ok);
          from += id * a.ssp + row * a.sst + head * a.ssh;
        }
        scale_next = *from;
      }
      if (lane == 0) seen_lds[tile & 3][wave] = (uint16_t)seen;
      __builtin_amdgcn_sched_barrier(0);
    };
    // The INT8 scales that came with raw tile `tile`, by the waves that loaded them.
    auto put_scales = [&](int tile) __attribute__((always_inline)) {
      if constexpr (kKind == kInt8Pages) {
        if (issues) put(tile, Fp16::lo(scale_next));
      }
    };
    // A raw tile to 16 bits.  K's values as they are, exact: their scales are in the
    // logits.  V's times their scale: INT8 rounded once, to float16 (to bfloat16 it was
    // 0.0028 of the output's norm instead of 0.0018), e4m3 times a power of two, exact in
    // bfloat16 (float16 has steps of its own below 2^-14).  In float16 at most the type's
    // largest value, which the product of a row's largest can pass by a rounding.  (Weights
    // times V's INT8 scales instead: registers short, 950 instead of 1,000 TFLOP/s at
    // head_dim 128 and an eighth at 256.  So are they with a path of their own for scales
    // past 512: a third of the rate.)
    auto dequant = [&](int tile, const uint8_t* from, uint8_t* stage) __attribute__((always_inline)) {
      constexpr int GR = Geo::I8_GR;
#pragma unroll
      for (int x = 0; x < (Geo::I8_GRANULES + kPrefillThreads - 1) / kPrefillThreads; ++x) {
        const int i = tid + x * kPrefillThreads;
        if (i >= Geo::I8_GRANULES) break;
        const int row = i / GR, gr = i % GR;
        if (16 * gr >= p.head_dim) continue;
#pragma unroll
        for (int tensor = 0; tensor < 2; ++tensor) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(from + tensor * RAW_BYTES + row * DP + gr * 16);
          const float scale = scale_lds[tile & 3][1 + tensor][row];
          u32x4 o[2];
          if constexpr (kKind == kInt8Pages) {
            if (tensor == 0) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                o[e / 4][e % 4] = T::pack(byte_float(w[e / 2], 2 * (e & 1)) * scale, byte_float(w[e / 2], 2 * (e & 1) + 1) * scale);
            } else {
              // The bytes plus 128 behind the exponent of 1024, less 1152.
              const _Float16 h = (_Float16)scale;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t bytes = __builtin_amdgcn_perm(w[e / 2] ^ 0x80808080u, 0x64646464u, e & 1 ? 0x00070006u : 0x00050004u);
                const f16x2 x = (__builtin_bit_cast(f16x2, bytes) - f16x2{1152, 1152}) * f16x2{h, h};
                o[e / 4][e % 4] = __builtin_bit_cast(uint32_t, x);
              }
              if (__builtin_expect(!(fabsf(scale) < 512.f), 0)) {
                // NaN bounds leave NaN.
                const _Float16 m = fabsf(scale) < INFINITY ? (_Float16)65504.f : (_Float16)NAN;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const uint32_t bits = o[e / 4][e % 4];  // (a cast of the element itself takes the vector's first)
                  const f16x2 x = __builtin_elementwise_min(__builtin_bit_cast(f16x2, bits), f16x2{m, m});
                  o[e / 4][e % 4] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, f16x2{-m, -m}));
                }
              }
            }
          } else {
            const float power = scale;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[e / 2][2 * (e & 1)] = T::template e4m3_pair<false>(w[e], power);
              o[e / 2][2 * (e & 1) + 1] = T::template e4m3_pair<true>(w[e], power);
            }
            if (std::is_same_v<T, Fp16> && tensor == 1 && !(power < 256.f)) {
              // Values past float16's largest become that.
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const f32x2 y = e & 1 ? e4m3_floats<true>(w[e / 2]) : e4m3_floats<false>(w[e / 2]);
                const float a = y[0] * power, b = y[1] * power;
                o[e / 4][e % 4] = T::pack(a == a ? __builtin_amdgcn_fmed3f(a, -65504.f, 65504.f) : a,
                                          b == b ? __builtin_amdgcn_fmed3f(b, -65504.f, 65504.f) : b);
              }
            }
          }
          uint8_t* to = stage + tensor * Geo::TILE_BYTES;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (16 * gr + 8 * h >= p.head_dim) continue;
            *reinterpret_cast<u32x4*>(to + (tensor == 0 ? Geo::k_offset(row, 2 * gr + h) : Geo::v_offset(row, 2 * gr + h))) = o[h];
          }
        }
      }
    };

    if constexpr (!QUANT) {
      for (int t = 0; t < min(ntiles, STAGES - 1); ++t) issue_tile(first + t, lds + t * STAGE_BYTES);
    } else {
      issue_tile(first, raw);
    }

    // Q fragments: row qw0 + 16 qb + r16, d = 32 c + 8 j .. + 7.
    u32x4 qf[QB][CK];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int row = min(qw0 + 16 * qb + r16, rows - 1), query = prefill_query(p, row);
      const uint16_t* from = p.q + (int64_t)(seq.from + query) * p.sq_t + (int64_t)(head * p.group + row - query * p.group) * p.sq_h;
#pragma unroll
      for (int c = 0; c < CK; ++c) {
        const int d = 32 * c + 8 * j;
        qf[qb][c] = *reinterpret_cast<const u32x4*>(from + (d < p.head_dim ? d : 0));
      }
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int c = 0; c < CK; ++c)
        qf[qb][c] = qw0 + 16 * qb + r16 < rows && 32 * c + 8 * j < p.head_dim ? qf[qb][c] ^ q_sign(p.scale_log2) : u32x4{0, 0, 0, 0};

    float m_run[QB], l_part[QB];
    f32x4 acc[DB][QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      m_run[qb] = -INFINITY, l_part[qb] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int k_lane = 64 * r16 + ((Geo::k_slot(j) ^ (r16 >> 2)) << 4);
    const int v_lane = 256 * j + 64 * (r16 >> 2) + 32 * (j & 1) + 8 * (r16 & 3);

    // ---- a tile's products ----
    auto compute = [&](int tile, const uint8_t* stage) __attribute__((always_inline)) {
      const int kt = span.key_of(tile);
      const uint32_t base = (uint32_t)(uintptr_t)(const SA_LDS uint8_t*)(stage);
      const uint64_t seen = uniform(*reinterpret_cast<const uint64_t*>(seen_lds[tile & 3]));
#pragma unroll
      for (int sub = 0; sub < kTileKeys / kSubKeys; ++sub) {
        const int rb = sub * kSubKeys, key0 = kt + rb;
        if (key0 >= wave_end) break;
        if (key0 + kSubKeys <= low_first && key0 >= p.sinks) continue;
        const uint32_t held = (uint32_t)(seen >> rb);
        const bool masked = key0 + kSubKeys > wave_first || (key0 < low_last && key0 + kSubKeys > p.sinks) || held != ~0u;
        f32x4 st[2][QB];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) st[kb][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c0 = 0; c0 < CK; c0 += KB) {
          u32x4 kf[2 * KB];
          read_k(kf, base + k_lane, (rb / 16 * CK + c0) * 1024, CK * 1024);
#pragma unroll
          for (int c = 0; c < KB; ++c)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int i = 0; i < QB; ++i) {
                const int qb = kb == 0 ? i : QB - 1 - i;
                st[kb][qb] = T::mma(kf[kb * KB + c], qf[qb][c0 + c], st[kb][qb]);
              }
        }
        // By what a logit's FMA multiplies it: of all keys, e4m3's of 16 keys, INT8's of each.
        constexpr bool BY_KEY = kKind == kInt8Pages;
        f32x4 factor[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const float* at = &scale_lds[QUANT ? tile & 3 : 0][0][rb + 16 * kb];
          const float f = QUANT ? at[0] : cf;
          factor[kb] = BY_KEY ? *reinterpret_cast<const f32x4*>(at + 4 * j) : f32x4{f, f, f, f};
        }
        // Bit k: row r16 of the query block sees the lane's key 4 j + k of the step (k 0 - 3
        // and 16 - 19 are its own).
        uint32_t sees[QB];
        if (__builtin_expect(masked, 0)) {
          const auto& a = *prefill_arguments();
          int l = r16;
          asm volatile("" : "+v"(l));
          const uint32_t here = held >> (4 * j);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) {
            const int behind = seq.base + prefill_query(a, min(qw0 + 16 * qb + l, rows - 1)) - key0 - 4 * j;
            sees[qb] = below(behind + 1) & here;
            uint32_t near = ~below((int)max((int64_t)behind - a.window + 1, (int64_t)0));
            if (key0 < a.sinks) near |= below(a.sinks - key0 - 4 * j);
            sees[qb] &= near;
          }
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
#pragma unroll
              for (int i = 0; i < 4; ++i) st[kb][qb][i] = sees[qb] >> (16 * kb + i) & 1 ? st[kb][qb][i] : -INFINITY;
        }
        auto exps = [&](int qb, float neg_m, u32x4& pq) -> float {
          float sum = 0.f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float p0 = __builtin_amdgcn_exp2f(fmaf(st[kb][qb][2 * e], factor[kb][2 * e], neg_m));
              const float p1 = __builtin_amdgcn_exp2f(fmaf(st[kb][qb][2 * e + 1], factor[kb][2 * e + 1], neg_m));
              sum = (kb == 0 && e == 0) ? p0 + p1 : sum + (p0 + p1);
              pq[2 * kb + e] = W::pack(p0, p1);
            }
          return sum;
        };
        u32x4 pf[QB];
        float psum[QB];
        bool grow[QB], any = false;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          // Every p is at most that wherever the lane's sum is; against m = -inf the sum is
          // inf or NaN.
          psum[qb] = exps(qb, -m_run[qb], pf[qb]);
          grow[qb] = !(psum[qb] <= (float)(1 << kWeightTop<W>));
          any = any || grow[qb];
        }
        if (__builtin_expect(__ballot(any) != 0, 0)) {
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) {
            const uint64_t bal = __ballot(grow[qb]);
            uint32_t fold = (uint32_t)bal | (uint32_t)(bal >> 32);
            fold |= fold >> 16;
            const bool mine = (fold >> r16) & 1u;
            float full = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              if constexpr (BY_KEY)
#pragma unroll
                for (int i = 0; i < 4; ++i) full = fmaxf(full, st[kb][qb][i] * factor[kb][i]);
              else
                full = fmaxf(full, fmaxf(fmaxf(st[kb][qb][0], st[kb][qb][1]), fmaxf(st[kb][qb][2], st[kb][qb][3])) * factor[kb][0]);
            }
            full = fmaxf(full, __shfl_xor(full, 16));
            full = fmaxf(full, __shfl_xor(full, 32));
            const float m_new = mine && full > m_run[qb] + kWeightTop<W> ? full - kWeightShift<W> : m_run[qb];
            const bool none = m_new == -INFINITY;
            if (m_new != m_run[qb] || none) {
              const float alpha = none ? 1.f : __builtin_amdgcn_exp2f(m_run[qb] - m_new);
              l_part[qb] *= alpha;
#pragma unroll
              for (int db = 0; db < DB; ++db) acc[db][qb] *= alpha;
              m_run[qb] = m_new;
              psum[qb] = exps(qb, none ? 0.f : -m_new, pf[qb]);
            }
          }
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) l_part[qb] += psum[qb];

        const uint32_t v_addr = base + Geo::TILE_BYTES + v_lane, v_odd = base + Geo::TILE_BYTES + (v_lane ^ 32);
#pragma unroll
        for (int d0 = 0; d0 < DB; d0 += VB) {
          u32x4 vf[VB];
          read_v(vf, v_addr, v_odd, d0 / 2 * 4096 + rb * 64);
          // A key that not every row sees: 0 * NaN is not 0, so what is not finite stays
          // out of the products.
          bool odd = false;
          if (__builtin_expect(masked, 0)) {
            u16x2 top = {0, 0};
#pragma unroll
            for (int dd = 0; dd < VB; ++dd)
#pragma unroll
              for (int i = 0; i < 4; ++i) top = larger(top, vf[dd][i]);
            odd = __any(top[0] >= W::kInfinity || top[1] >= W::kInfinity);
            if (__builtin_expect(odd, 0)) {
#pragma unroll
              for (int dd = 0; dd < VB; ++dd)
#pragma unroll
                for (int i = 0; i < 4; ++i) vf[dd][i] &= ~halves(not_finite<W>(vf[dd][i]));
            }
          }
#pragma unroll
          for (int dd = 0; dd < VB; ++dd)
#pragma unroll
            for (int i = 0; i < QB; ++i) {
              const int qb = dd % 2 == 0 ? i : QB - 1 - i;
              acc[d0 + dd][qb] = W::mma(vf[dd], pf[qb], acc[d0 + dd][qb]);
            }
          if (__builtin_expect(odd, 0)) {
            // The elements of the rows that see one: their number, as a product of ones.
            constexpr uint32_t kOnes = std::is_same_v<W, Bf16> ? 0x3f803f80u : 0x3c003c00u;
            read_v(vf, v_addr, v_odd, d0 / 2 * 4096 + rb * 64);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
              u32x4 seers;
#pragma unroll
              for (int x = 0; x < 4; ++x) seers[x] = kOnes & halves(two_bits(sees[qb], x / 2 * 16 + 2 * (x & 1)));
#pragma unroll
              for (int dd = 0; dd < VB; ++dd) {
                u32x4 ones;
#pragma unroll
                for (int i = 0; i < 4; ++i) ones[i] = halves(not_finite<W>(vf[dd][i])) & kOnes;
                const f32x4 count = W::mma(ones, seers, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (count[e] > 0.f) acc[d0 + dd][qb][e] = NAN;
              }
            }
          }
        }
      }
    };

    // ---- the tiles ----
    if constexpr (!QUANT) {
      // Tile t is computed while the next STAGES - 1 are in flight; an issuing wave's
      // loads complete in order.
      // Tile t is there once no more than the later tiles' loads are outstanding; with
      // a padded head_dim they are fewer than that.
      constexpr int PER_TILE = 2 * CK;
      for (int t = 0; t < ntiles; ++t) {
        const int later = p.head_dim < DP ? 0 : min(ntiles - 1 - t, STAGES - 2);
        if (later >= 2)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER_TILE) : "memory");
        else if (later == 1)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER_TILE) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (t + STAGES - 1 < ntiles)
          issue_tile(first + t + STAGES - 1, lds + (t + STAGES - 1) % STAGES * STAGE_BYTES);
        compute(first + t, lds + t % STAGES * STAGE_BYTES);
      }
    } else if constexpr (STAGES == 1) {
      // LDS holds one converted tile (head_dim 256).
      for (int t = 0; t < ntiles; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        put_scales(first + t);
        barrier();
        dequant(first + t, raw + t % 2 * 2 * RAW_BYTES, lds);
        if (t + 1 < ntiles) issue_tile(first + t + 1, raw + (t + 1) % 2 * 2 * RAW_BYTES);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile under way stays so
        __syncthreads();
        compute(first + t, lds);
      }
    } else {
      static_assert(STAGES == 2, "stages of converted tiles");
      // At tile t: its 16-bit form is in its stage, raw tile t + 1 has arrived.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      put_scales(first);
      barrier();
      dequant(first, raw, lds);
      if (ntiles > 1) issue_tile(first + 1, raw + 2 * RAW_BYTES);
      for (int t = 0; t < ntiles; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (t + 1 < ntiles) put_scales(first + t + 1);
        barrier();
        // The first wave of a SIMD converts before its products and the second one
        // after them, so that each one's vector work meets the other's matrix work.
        auto next = [&]() __attribute__((always_inline)) {
          if (t + 1 < ntiles) dequant(first + t + 1, raw + (t + 1) % 2 * 2 * RAW_BYTES, lds + (t + 1) % 2 * STAGE_BYTES);
        };
        if (issues) {
          next();
          if (t + 2 < ntiles) issue_tile(first + t + 2, raw + t % 2 * 2 * RAW_BYTES);
        }
        compute(first + t, lds + t % 2 * STAGE_BYTES);
        if (!issues) next();
      }
    }

    // ---- the piece's end ----
    const auto& a = *prefill_arguments();
    const bool whole = first == 0 && last == span.count;
    float* part = a.parts + ((int64_t)run * 2 + (first == 0)) * prefill_part_floats(BLOCK_M, DP);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float l = l_part[qb] + __shfl_xor(l_part[qb], 16);
      l += __shfl_xor(l, 32);
      const int row = qw0 + 16 * qb + r16;
      if (whole) {
        // One rounding more than a division, in FP32.
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int at_row = min(row, rows - 1);  // lanes past the rows take part in the exchange
        const int query = prefill_query(a, at_row), q_head = head * a.group + at_row - query * a.group;
        // Two blocks of 16 elements: lanes of odd j hand their four of the first to j - 1 and
        // take those of the second, so that a lane stores eight.
        uint16_t* to = a.out + (int64_t)(seq.from + query) * a.so_t + (int64_t)q_head * a.so_h + 16 * (j & 1) + 8 * (j >> 1);
#pragma unroll
        for (int db = 0; db < DB; db += 2) {
          const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
          const f32x4 o = l == 0.f ? zero : acc[db][qb] * inv, next = l == 0.f ? zero : acc[db + 1][qb] * inv;
          const auto x = __builtin_amdgcn_permlane16_swap(T::pack(o[0], o[1]), T::pack(next[0], next[1]), false, false);
          const auto y = __builtin_amdgcn_permlane16_swap(T::pack(o[2], o[3]), T::pack(next[2], next[3]), false, false);
          if (row < rows && 16 * (db + (j & 1)) + 8 * (j >> 1) < a.head_dim)
            *reinterpret_cast<u32x4*>(to + 16 * db) = u32x4{x[0], y[0], x[1], y[1]};
        }
        if (a.lse != nullptr && j == 0 && row < rows)
          a.lse[q_head * a.lse_h + seq.from + query] = l == 0.f ? -INFINITY : (m_run[qb] + log2f(l)) * 0.69314718055994530942f;
      } else if (has_rows) {
        // In the order of the lanes.
#pragma unroll
        for (int db = 0; db < DB; ++db)
          *reinterpret_cast<f32x4*>(part + ((wave * QB + qb) * DB + db) * 256 + 4 * lane) = acc[db][qb];
        if (j == 0) {
          float* stats = part + BLOCK_M * DP + 2 * (row - row0);
          stats[0] = m_run[qb], stats[1] = l;
        }
      }
    }
    if (!whole && first == 0 && tid == 0) a.splits[run] = {block, head, (int32_t)((before + span.count - 1) / share), 0};
    if (whole_items && tid == kFetcher) next_lds = fetched;
    at = before + last;
    if (++block == blocks) block = 0, ++head;
  }
}

// The parts of a split item joined: a thread has four elements of a row.  With many
// parts (few rows over long keys) a workgroup's waves share them, four by four: 16
// tokens behind 40,000 keys, 64 parts an item, 17 us instead of 30.
constexpr int kPrefillJoinThreads = 256, kPrefillJoiners = 16, kPrefillSharedParts = 8, kPrefillSharedChunks = 4096;

struct PrefillJoin {
  float top, weight;
  f32x4 sum;
  __device__ inline void rescale(float to) {
    const float keep = prefill_ratio(top, to);
    weight *= keep, sum *= keep, top = to;
  }
};

template <typename T, int DP>
__global__ __launch_bounds__(kPrefillJoinThreads) void prefill_join_kernel(const PrefillParams p) {
  constexpr int DB = DP / 16, kWaves = kPrefillJoinThreads / 64;
  __shared__ PrefillJoin joins[kWaves][64];
  const int run = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const PrefillSplit split = p.splits[run];
  if (split.block < 0) return;
  const PrefillBlock b = p.blocks[split.block];
  const PrefillSequence seq = prefill_sequence(p, b.sequence);
  const int64_t size = prefill_part_floats(p.rows, DP);
  const auto part = [&](int i) { return p.parts + ((int64_t)i * 2 + (i == run)) * size; };
  const int rows = min(seq.count * p.group - b.row, p.rows), chunks = (rows + 15) / 16 * 4 * DP;
  const bool shared = split.last - run >= kPrefillSharedParts && chunks <= kPrefillSharedChunks;
  const int mine = shared ? wave : 0, step = shared ? kWaves : 1;         // parts run + mine, + step, ...
  const int width = shared ? 64 : kPrefillJoinThreads, at = shared ? tid & 63 : tid;
  // In the parts' order: 16 rows of the block after the other.
  for (int first_chunk = blockIdx.y * width; first_chunk < chunks; first_chunk += kPrefillJoiners * width) {
    const int chunk = first_chunk + at;
    const int lane = chunk & 63, d = 16 * ((chunk >> 6) % DB) + 4 * (lane >> 4);
    const int local = (chunk >> 6) / DB * 16 + (lane & 15);
    const bool live = chunk < chunks && local < rows && d < p.head_dim;
    PrefillJoin x{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
    if (live) {
      // Four parts' loads under way together.
      for (int first = run + mine; first <= split.last; first += 4 * step) {
        float m[4], l[4];
        f32x4 y[4];
        float to = x.top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float* from = part(min(first + i * step, split.last));
          m[i] = from[p.rows * DP + 2 * local], l[i] = from[p.rows * DP + 2 * local + 1];
          y[i] = *reinterpret_cast<const f32x4*>(from + 4 * chunk);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) to = fmaxf(to, first + i * step <= split.last ? m[i] : -INFINITY);
        x.rescale(to);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (first + i * step > split.last) continue;
          const float f = prefill_ratio(m[i], to);
          x.weight += l[i] * f, x.sum += y[i] * f;
        }
      }
    }
    if (shared) {
      __syncthreads();  // the joins of the chunks before are read
      joins[wave][at] = x;
      __syncthreads();
      if (wave > 0) continue;
      for (int w = 1; w < kWaves; ++w) {
        const PrefillJoin y = joins[w][at];
        const float to = fmaxf(x.top, y.top), f = prefill_ratio(y.top, to);
        x.rescale(to);
        x.weight += y.weight * f, x.sum += y.sum * f;
      }
    }
    if (!live) continue;
    const int row = b.row + local, query = prefill_query(p, row), q_head = split.head * p.group + row - query * p.group;
    const f32x4 o = x.weight == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : x.sum * (1.f / x.weight);
    *reinterpret_cast<u32x2*>(p.out + (int64_t)(seq.from + query) * p.so_t + (int64_t)q_head * p.so_h + d) =
        u32x2{T::pack(o[0], o[1]), T::pack(o[2], o[3])};
    if (p.lse != nullptr && d == 0)
      p.lse[q_head * p.lse_h + seq.from + query] = x.weight == 0.f ? -INFINITY : (x.top + log2f(x.weight)) * 0.69314718055994530942f;
  }
}

template <typename T, int DP, int QB, PageKind kKind>
hipError_t launch_prefill(const PrefillLaunch& l) {
  constexpr int stages = kKind == kRowPages ? (QB == 1 && DP <= 64 ? 4 : 2) : DP == 256 ? 1 : 2;
  prefill_kernel<T, DP, QB, kKind, stages><<<l.p.runs, kPrefillThreads, 0, l.stream>>>(l.p);
  const hipError_t status = hipGetLastError();
  if (status != hipSuccess) return status;
  prefill_join_kernel<T, DP><<<dim3(l.p.runs, kPrefillJoiners), kPrefillJoinThreads, 0, l.stream>>>(l.p);
  return hipGetLastError();
}

template <typename T, int DP, int QB>
hipError_t launch_prefill(const PrefillLaunch& l) {
  return l.kind == kE4m3Pages ? launch_prefill<T, DP, QB, kE4m3Pages>(l)
         : l.kind == kInt8Pages ? launch_prefill<T, DP, QB, kInt8Pages>(l)
                                : launch_prefill<T, DP, QB, kRowPages>(l);
}

template <int DP>
hipError_t launch_prefill(const PrefillLaunch& l) {
  constexpr int many = prefill_rows(DP, true) / 128;
  if (l.p.rows == 128) return l.bf16 ? launch_prefill<Bf16, DP, 1>(l) : launch_prefill<Fp16, DP, 1>(l);
  return l.bf16 ? launch_prefill<Bf16, DP, many>(l) : launch_prefill<Fp16, DP, many>(l);
}

}  // namespace
}  // namespace sa
