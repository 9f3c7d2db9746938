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
// columns that a group of up to 8 heads leaves unused anyway.  In one part the
// weights' own rounding would be as large as the output's.
//
// Measured (a kernel that only reads reaches 7.0 TB/s): 64 sequences of 16,384
// keys, 32/8 heads of 128, 633 us, 6.8 TB/s; one of 524,288 keys 325 us, 6.6 TB/s; 96
// over 1,048,576 INT8 keys, 40/8 heads, 370 us, 5.9 TB/s: there two waves per SIMD
// wait for each other's conversions (vector units half busy), and a third has no
// registers.  200 short sequences, 60,013 keys of 4 heads of 96, 24 us and 4 for
// the join: 13 us of bytes, the rest the scan of the lengths, the first loads
// and the joins.
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

// Past the caches: K and V are read once per step, and the caches hold other
// things.  64 sequences of 16,384 keys 738 -> 669 us, 57,330 keys of head_dim 256
// 167 -> 154; keys that the caches hold from the step before are read as fast
// (32,000 keys, 131 MB: 31.0 and 30.5; 64,000 keys, 262 MB: 49 and 53).
template <int N>
__device__ inline Dwords<N> load_dwords(const char* base, uint32_t offset) {
  Dwords<N> r;
  const char* p = base + offset;
  if constexpr (N == 4) {
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    r.w[0] = x[0], r.w[1] = x[1], r.w[2] = x[2], r.w[3] = x[3];
  } else if constexpr (N == 2) {
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.w[0] = x[0], r.w[1] = x[1];
  } else {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}

__device__ inline __attribute__((always_inline)) int32_t uniform(int32_t x) {
  return __builtin_amdgcn_readfirstlane(x);
}

// The value on the lane whose column is 8 further, of the same 16.
__device__ inline float other_half(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
}

// 2^x of a running maximum's change: 0 from -inf, 1 where nothing changes.
__device__ inline float ratio(float from, float to) { return from == to ? 1.f : __builtin_amdgcn_exp2f(from - to); }

// A wave's share of one item: tiles first .. last - 1 of the item's `tiles`.
struct Piece {
  int64_t start;  // the launch's tile that is the item's first
  const int32_t* table;
  int32_t s, length, tiles, first, last;
  int32_t kv_head, block;  // query heads 8 NB block .. of the K/V head's group

  __device__ inline void bound(int64_t end) {  // as far as a run up to `end` goes
    const int64_t left = end - start;
    last = left < tiles ? (int32_t)left : tiles;
  }
};

// The kernel's arguments, read again where they are used: what only a piece's
// ends need would otherwise sit in scalar registers, and those that do not fit
// in lanes of vector registers, all through the loop over the keys.
typedef const DecodeParams __attribute__((address_space(4)))* Arguments;
__device__ inline Arguments arguments() {
  Arguments a = (Arguments)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}

__device__ inline int32_t length_of(Arguments a, int s) {
  const int32_t n = a->lengths[s];
  return n < a->room ? n : a->room;
}
__device__ inline int32_t tiles_of(int32_t length) { return length > 0 ? (length - 1) / kDecodeTile + 1 : 0; }

// Where a wave's next load is: a tile of a piece, in row `row` of the
// sequence's page number `page`.
struct Reader {
  Piece x;
  int32_t tile, page, row;
  int32_t ids, first_id;  // page numbers first_id + lane of the sequence

  // Has pages n .. upto in `ids` (n never falls, upto - n < 64).
  __device__ inline void hold(const DecodeParams& p, int32_t n, int32_t upto, int lane) {
    if (upto - first_id >= 64) {
      first_id = n;
      ids = n + lane < p.max_pages ? x.table[n + lane] : -1;
    }
  }
  __device__ inline int32_t id_of(const DecodeParams& p, int32_t n, int lane) {
    hold(p, n, n, lane);
    return __builtin_amdgcn_readlane(ids, n - first_id);
  }

  __device__ inline void enter(const DecodeParams& p) {  // at the piece's first tile
    tile = x.first;
    page = uniform((int32_t)((uint64_t)(uint32_t)(tile * kDecodeTile) * p.page_magic >> p.page_shift));
    row = tile * kDecodeTile - page * p.page_tokens;
    first_id = page - 64;
  }

  // To the next tile of a run up to tile `end` of the launch, which has one.
  __device__ inline void advance(const DecodeParams& p, int64_t end) {
    if (++tile < x.last) {
      page += p.step_pages, row += p.step_rows;
      if (row >= p.page_tokens) ++page, row -= p.page_tokens;
      return;
    }
    // The next item: the sequence's next, or the first of the next sequence
    // that has keys.
    const Arguments a = arguments();
    x.start += x.tiles, x.first = 0;
    if (++x.block == a->blocks) x.block = 0, ++x.kv_head;
    if (x.kv_head == a->kv_heads) {
      x.kv_head = 0;
      do x.length = uniform(length_of(a, ++x.s));
      while (x.length <= 0);
      x.tiles = tiles_of(x.length);
      x.table = a->table + x.s * a->s_table;
    }
    x.bound(end);
    enter(p);
  }
};

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
  Piece x;       // whose keys they are
  int32_t tile;  // 32 tile .. of the sequence

  __device__ __attribute__((always_inline)) void load(const DecodeParams& p, Reader& from, int lane) {
    x = from.x, tile = from.tile;
    const int j = lane >> 4, g = lane & 15;
    const int32_t key0 = tile * kDecodeTile;
    int32_t page = from.page, row = from.row;
    const char *kh = p.k + x.kv_head * p.sh * ES, *vh = p.v + x.kv_head * p.sh * ES;
    uint32_t at[NP];
#pragma unroll
    for (int c = 0; c < NP; ++c) at[c] = (128 * c + EL * g < p.head_dim ? 128 * c + EL * g : 0) * ES;
    const bool second = g >= 8;
    if constexpr (!kAnyPage) {
      // Two runs of 16 keys, each in one page.
      full = x.length - key0 >= kDecodeTile;
      const uint32_t rows = j * (uint32_t)p.st * ES;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && (row += 16) >= p.page_tokens) ++page, row -= p.page_tokens;
        int32_t id = from.id_of(p, page, lane);
        const bool ok = (uint32_t)id < (uint32_t)p.num_pages;
        if (!ok) id = 0;  // rows of a page that exists, read and not used
        full = full && ok;
        const int64_t base = (id * p.sp + row * p.st) * ES;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < NP; ++c) k[4 * h + u][c] = load_dwords<RW>(kh + base + 4 * u * p.st * ES, rows + at[c]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < NP; ++c) v[4 * h + u][c] = load_dwords<RW>(vh + base + 4 * u * p.st * ES, rows + at[c]);
        if constexpr (kInt8) {
          const uint16_t* s = (second ? p.vs : p.ks) + id * p.ssp + row * p.sst + x.kv_head * p.ssh;
          if ((g >> 2 & 1) == h) scale = s[(4 * (g & 3) + j) * p.sst];
        }
        const uint32_t mask = ok ? 15u : 0u;
        seen = h == 0 ? mask : seen | mask << 4;
      }
    } else {
      seen = 0;
      const uint64_t rows_on = (uint32_t)(row + kDecodeTile - 1);  // the last key's, from the first's page
      from.hold(p, page, page + uniform((int32_t)(rows_on * p.page_magic >> p.page_shift)), lane);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        int32_t r = row + 4 * t + j;
        const int32_t past = (int32_t)((uint64_t)(uint32_t)r * p.page_magic >> p.page_shift);
        r -= past * p.page_tokens;
        int32_t id = __shfl(from.ids, page + past - from.first_id);
        const bool ok = (uint32_t)id < (uint32_t)p.num_pages;
        if (!ok) id = 0;
        seen |= (uint32_t)ok << t;
        const int64_t base = (id * p.sp + r * p.st) * ES;
#pragma unroll
        for (int c = 0; c < NP; ++c)
          k[t][c] = load_dwords<RW>(kh + base, at[c]), v[t][c] = load_dwords<RW>(vh + base, at[c]);
        if constexpr (kInt8)
          if ((g & 7) == t) scale = (second ? p.vs : p.ks)[id * p.ssp + r * p.sst + x.kv_head * p.ssh];
      }
      full = __all(seen == 255u) && x.length - key0 >= kDecodeTile;
    }
    if (x.length - key0 < kDecodeTile) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (key0 + 4 * t + j >= x.length) seen &= ~(1u << t);
    }
  }
};

// What a wave leaves of an item that it does not have whole: the item's head
// (it started in an earlier range) or tail (it ends in a later one).
struct PartInfo {
  int64_t end;  // the launch's tile behind the item
  int32_t s, kv_head, block;
  int32_t state;  // 0: none, 1: goes on in the next wave, 2: ends here
};

// Every wave has an equal run of the launch's tiles.  Items that lie whole in
// it are done there; the others' parts meet in LDS, and those of items that
// leave the workgroup's run in the workspace.
template <typename T, bool kInt8, int DP, int NB, bool kAnyPage>
__global__ __launch_bounds__(64 * kDecodeWaves, decode_occupancy(DP, NB, kInt8)) void decode_kernel(
    const DecodeParams p) {
  using S = Shape<DP>;
  using PT = std::conditional_t<kInt8, Bf16, T>;  // INT8: weights times V's scales, beyond float16's range
  constexpr int EL = S::EL, NP = S::NP, NI = S::NI, NC = S::NC;
  constexpr float bias = kBias<PT>;
  constexpr int kRow = 2 * DP;  // bytes of a key in LDS
  constexpr int kPart = 8 * NB * DP;  // floats of a part
  // K and its INT8 scales, then the tail.
  __shared__ __attribute__((aligned(16))) char lds[kDecodeWaves][kDecodeTile * kRow + (kInt8 ? 256 : 0)];
  __shared__ __attribute__((aligned(16))) float heads_lds[kDecodeWaves][kPart];
  __shared__ float stats[kDecodeWaves][2][8 * NB][2];  // maximum and sum of the head's, the tail's rows
  __shared__ PartInfo info[kDecodeWaves][2];
  __shared__ int64_t found[kDecodeWaves][2];
  static_assert(kPart * 4 <= kDecodeTile * kRow, "the tail's place");

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int j = lane >> 4, g = lane & 15;
  int64_t share, total;  // tiles of a wave's run
  int64_t begin, end;
  {
    const Arguments a = arguments();
    const int items = a->kv_heads * a->blocks, w = blockIdx.x, workgroups = gridDim.x;
    // Tiles before every thread's run of sequences.
    int64_t* sums = reinterpret_cast<int64_t*>(&lds[0][0]);
    const int run = (a->sequences + 64 * kDecodeWaves - 1) / (64 * kDecodeWaves);
    const int s_first = tid * run, s_last = s_first + run < a->sequences ? s_first + run : a->sequences;
    int64_t own = 0;
    for (int s = s_first; s < s_last; ++s) own += tiles_of(length_of(a, s));
    int64_t upto = own;  // inclusive
    for (int i = 1; i < 64; i <<= 1) {
      const int64_t x = __shfl_up(upto, i);
      if (lane >= i) upto += x;
    }
    if (lane == 63) sums[wave] = upto;
    if (tid < 2 * kDecodeWaves) info[tid >> 1][tid & 1].state = 0;
    __syncthreads();
    total = 0;
    for (int i = 0; i < kDecodeWaves; ++i) {
      if (i < wave) upto += sums[i];
      total += sums[i];
    }
    total *= items;
    const int64_t waves = (int64_t)workgroups * kDecodeWaves;
    share = (total + waves - 1) / waves;
    for (int i = 0; i < kDecodeWaves; ++i) {
      const int64_t at = (w * kDecodeWaves + i) * share;
      if (at >= total || at < (upto - own) * items || at >= upto * items) continue;
      int64_t before = upto - own;
      int s = s_first;
      for (; s < s_last; ++s) {
        const int64_t n = tiles_of(length_of(a, s));
        if (at < (before + n) * items) break;
        before += n;
      }
      found[i][0] = s, found[i][1] = before * items;
    }
    // Sequences without keys have no tiles.
    for (int s = w; s < a->sequences; s += workgroups) {
      if (length_of(a, s) > 0) continue;
      const int granules = a->head_dim / 8;
      for (int i = tid; i < a->kv_heads * a->group * granules; i += 64 * kDecodeWaves) {
        const int h = i / granules, d = 8 * (i - h * granules);
        *reinterpret_cast<u32x4*>(a->out + s * a->so_t + h * a->so_h + d) = u32x4{0, 0, 0, 0};
        if (d == 0 && a->lse != nullptr) a->lse[h * a->lse_h + s] = -INFINITY;
      }
      for (int i = tid; a->by_item && i < items; i += 64 * kDecodeWaves) a->owned[4 * (s * items + i)] = -1;
    }
    if (tid == 0 && !a->by_item) a->owned[4 * w] = -1;
    __syncthreads();
    begin = (w * kDecodeWaves + wave) * share, end = begin + share < total ? begin + share : total;
  }
  if ((int64_t)blockIdx.x * kDecodeWaves * share >= total) return;

  char* mine = &lds[wave][0];
  float* scales = reinterpret_cast<float*>(mine + kDecodeTile * kRow);
  if (begin < end) {
    Reader reader;
    Step<kInt8, DP, kAnyPage> step;
    {
      const Arguments a = arguments();
      Piece& x = reader.x;
      x.s = uniform((int)found[wave][0]);
      x.length = uniform(length_of(a, x.s));
      x.tiles = tiles_of(x.length);
      const int64_t into = begin - found[wave][1];
      const int item = uniform((int)(into / x.tiles));
      x.start = found[wave][1] + (int64_t)item * x.tiles;
      x.first = uniform((int32_t)(begin - x.start));
      x.kv_head = item / a->blocks, x.block = item - x.kv_head * a->blocks;
      x.table = a->table + x.s * a->s_table;
      x.bound(end);
      reader.enter(p);
    }
    step.load(p, reader, lane);

    u32x4 q[NB][NC];
    f32x4 acc[NB][NI];
    float m[NB], l[NB];
    const auto start_piece = [&](const Piece& cur) __attribute__((always_inline)) {
      // Q^T: chunk c of column g's head, elements 32c + 8j .. + 7.
      {
        const Arguments a = arguments();
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int h = 8 * (NB * cur.block + n) + (g & 7);  // of the group
          const uint16_t* at = a->q + cur.s * a->sq_t + (cur.kv_head * a->group + (h < a->group ? h : 0)) * a->sq_h;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const int d = 32 * c + 8 * j;
            q[n][c] = h < a->group && d < a->head_dim ? *reinterpret_cast<const u32x4*>(at + d) : u32x4{0, 0, 0, 0};
          }
        }
      }
      // K's elements past head_dim are zeros that no step writes.
      if (p.head_dim < DP) {
        for (int i = lane; i < kDecodeTile * kRow / 16; i += 64) reinterpret_cast<u32x4*>(mine)[i] = u32x4{0, 0, 0, 0};
        wave_lds_order();
      }

#pragma unroll
      for (int n = 0; n < NB; ++n) {
        m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    };
    // A tile's products; its step takes the next load.
    const auto work = [&](bool more) __attribute__((always_inline)) {
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
              x[i] = T::pack(byte_float(step.k[t][c].w[i / 2], 2 * (i & 1)),
                             byte_float(step.k[t][c].w[i / 2], 2 * (i & 1) + 1));
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
      // K's scales with the softmax's.
      if constexpr (kInt8) scales[16 * j + g] = Fp16::lo(step.scale) * (g < 8 ? p.scale_log2 : 1.f);
      const bool full = step.full;
      const uint32_t seen = step.seen;
      // Rows without weight may hold anything: 0 * NaN is not 0.
      if (!full) {
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int c = 0; c < NP; ++c)
#pragma unroll
            for (int i = 0; i < step.RW; ++i) step.v[t][c].w[i] = seen >> t & 1 ? step.v[t][c].w[i] : 0;
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
              vt[EL * c + i][u] = PT::pack(byte_float(step.v[2 * u][c].w[i / 4], i & 3),
                                           byte_float(step.v[2 * u + 1][c].w[i / 4], i & 3));
            else
              vt[EL * c + i][u] = __builtin_amdgcn_perm(step.v[2 * u + 1][c].w[i / 2], step.v[2 * u][c].w[i / 2],
                                                        i & 1 ? 0x07060302u : 0x05040100u);
          }
      if (more) {
        reader.advance(p, end);
        step.load(p, reader, lane);
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
          const u32x4 x = *reinterpret_cast<const u32x4*>(mine + r * kRow + 16 * ((4 * c + j) ^ turn));
#pragma unroll
          for (int n = 0; n < NB; ++n) st[n][b] = T::mma(x, q[n][c], st[n][b]);
        }
      f32x4 factors[2] = {f32x4{p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2}, factors[0]};
      if constexpr (kInt8) {
        factors[0] = *reinterpret_cast<const f32x4*>(scales + 16 * j);
        factors[1] = *reinterpret_cast<const f32x4*>(scales + 16 * j + 4);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float y[8], top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          y[t] = st[n][t / 4][t & 3] * factors[t / 4][t & 3];
        }
        if (!full) {
#pragma unroll
          for (int t = 0; t < 8; ++t) y[t] = seen >> t & 1 ? y[t] : -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) top = fmaxf(top, y[t]);
        if (__any(top > m[n] + (bias + kSlack))) {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32)) - bias;
          const float to = fmaxf(m[n], top), keep = ratio(m[n], to);
          m[n] = to;
          l[n] *= keep;
#pragma unroll
          for (int i = 0; i < NI; ++i) acc[n][i] *= keep;
        }
        f32x4 vs[2];
        if constexpr (kInt8) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            vs[b] = *reinterpret_cast<const f32x4*>(scales + 16 * j + 8 + 4 * b);
            if (!full)
#pragma unroll
              for (int e = 0; e < 4; ++e) vs[b][e] = seen >> (4 * b + e) & 1 ? vs[b][e] : 0.f;
          }
        }
        const float base = m[n] == -INFINITY ? 0.f : m[n];
        const float low = g >= 8 ? 1.f : 0.f;
        u32x4 weights;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float a = __builtin_amdgcn_exp2f(y[2 * u] - base), b = __builtin_amdgcn_exp2f(y[2 * u + 1] - base);
          l[n] += a + b;
          if constexpr (kInt8) a *= vs[u / 2][2 * (u & 1)], b *= vs[u / 2][2 * (u & 1) + 1];
          const uint32_t high = PT::pack(a, b);
          weights[u] = PT::pack(a - low * PT::lo(high), b - low * PT::hi(high));
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[n][i] = PT::mma(vt[i], weights, acc[n][i]);
      }
      wave_lds_order();
    };
    // A piece's end: high and low parts together, the lanes' sums together.
    const auto end_piece = [&](const Piece& cur) __attribute__((always_inline)) {
      const Arguments a = arguments();
      const bool starts = cur.first == 0, ends = cur.last == cur.tiles;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][i][e] += other_half(acc[n][i][e]);
        const int h = 8 * (NB * cur.block + n) + (g & 7);
        if (g >= 8 || h >= a->group) continue;
        if (starts && ends) {
          const int head = cur.kv_head * a->group + h;
          const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];
          uint16_t* out = a->out + cur.s * a->so_t + head * a->so_h;
#pragma unroll
          for (int c = 0; c < NP; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = 128 * c + EL * (4 * j + e);
              uint32_t o[EL / 2];
#pragma unroll
              for (int i = 0; i < EL; i += 2)
                o[i / 2] = T::pack(acc[n][EL * c + i][e] * inv, acc[n][EL * c + i + 1][e] * inv);
              if (d >= a->head_dim) continue;
              if constexpr (EL == 8)
                *reinterpret_cast<u32x4*>(out + d) = u32x4{o[0], o[1], o[2], o[3]};
              else
                *reinterpret_cast<u32x2*>(out + d) = u32x2{o[0], o[1]};
            }
          if (j == 0 && a->lse != nullptr)
            a->lse[head * a->lse_h + cur.s] = l[n] == 0.f ? -INFINITY : (m[n] + log2f(l[n])) * kLn2;
        } else {
          float* part = starts ? reinterpret_cast<float*>(mine) : heads_lds[wave];
#pragma unroll
          for (int c = 0; c < NP; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < EL; i += 4)
                *reinterpret_cast<f32x4*>(part + (8 * n + g) * DP + 128 * c + EL * (4 * j + e) + i) =
                    f32x4{acc[n][EL * c + i][e], acc[n][EL * c + i + 1][e], acc[n][EL * c + i + 2][e],
                          acc[n][EL * c + i + 3][e]};
          if (j == 0) stats[wave][starts][8 * n + g][0] = m[n], stats[wave][starts][8 * n + g][1] = l[n];
        }
      }
      if (lane == 0) {
        if (starts && ends) {
          if (a->by_item) a->owned[4 * ((cur.s * a->kv_heads + cur.kv_head) * a->blocks + cur.block)] = -1;
        } else {
          info[wave][starts] = {cur.start + cur.tiles, cur.s, cur.kv_head, cur.block, ends ? 2 : 1};
        }
      }
    };
    for (int64_t left = end - begin; left > 0; --left) {
      const Piece cur = step.x;
      const int32_t tile = step.tile;
      if (tile == cur.first) start_piece(cur);
      work(left > 1);
      if (tile + 1 == cur.last) end_piece(cur);
    }
  }

  // The parts: wave 0's head, and the tails, each with the heads that go on from
  // it in the waves behind.
  __syncthreads();
  const Arguments a = arguments();
  const int w = blockIdx.x;
  for (int from = -1; from < kDecodeWaves; ++from) {
    const PartInfo part = info[from < 0 ? 0 : from][from < 0 ? 0 : 1];
    if (part.state == 0) continue;
    // Parts: (from, tail) or (0, head), then the heads of waves after .. upto - 1.
    const int after = from < 0 ? 1 : from + 1;
    int upto = after, state = part.state;
    while (state == 1 && upto < kDecodeWaves && info[upto][0].state != 0) state = info[upto++][0].state;
    const bool whole = from >= 0 && state == 2;
    float* slot = a->parts + ((int64_t)w * 2 + (from < 0 ? 0 : 1)) * (8 * NB * (DP + 2));
    const int h0 = 8 * NB * part.block, heads = a->group - h0 < 8 * NB ? a->group - h0 : 8 * NB;
    for (int i = tid; i < heads * (DP / 4); i += 64 * kDecodeWaves) {
      const int h = i / (DP / 4), d = 4 * (i % (DP / 4));
      const float* x = from < 0 ? heads_lds[0] : reinterpret_cast<const float*>(&lds[from][0]);
      const float* x_stats = stats[from < 0 ? 0 : from][from < 0 ? 0 : 1][h];
      float top = x_stats[0];
      for (int y = after; y < upto; ++y) top = fmaxf(top, stats[y][0][h][0]);
      const float f = ratio(x_stats[0], top);
      float weight = x_stats[1] * f;
      f32x4 sum = *reinterpret_cast<const f32x4*>(x + h * DP + d) * f;
      for (int y = after; y < upto; ++y) {
        const float r = ratio(stats[y][0][h][0], top);
        weight += stats[y][0][h][1] * r;
        sum += *reinterpret_cast<const f32x4*>(heads_lds[y] + h * DP + d) * r;
      }
      if (whole) {
        const int head = part.kv_head * a->group + h0 + h;
        const float inv = weight == 0.f ? 0.f : 1.f / weight;
        if (d < a->head_dim)
          *reinterpret_cast<u32x2*>(a->out + part.s * a->so_t + head * a->so_h + d) =
              u32x2{T::pack(sum[0] * inv, sum[1] * inv), T::pack(sum[2] * inv, sum[3] * inv)};
        if (d == 0 && a->lse != nullptr)
          a->lse[head * a->lse_h + part.s] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * kLn2;
      } else {
        *reinterpret_cast<f32x4*>(slot + h * DP + d) = sum;
        if (d == 0) slot[8 * NB * DP + 2 * h] = top, slot[8 * NB * DP + 2 * h + 1] = weight;
      }
    }
    if (tid == 0 && from >= 0 && (a->by_item || !whole)) {
      const int item = part.kv_head * a->blocks + part.block;
      int32_t* entry = a->owned + 4 * (a->by_item ? part.s * a->kv_heads * a->blocks + item : w);
      entry[0] = whole ? -1 : part.s, entry[1] = item, entry[2] = w;
      entry[3] = (int32_t)((part.end - 1) / (kDecodeWaves * share));
    }
  }
}

// The parts of a split item joined: a workgroup per query head, a lane per four
// elements, the parts dealt to groups of lanes.  A launch of its own, 4 - 5 us:
// joined by the workgroup that comes last instead, every wave's release writes
// its XCD's L2 back, 24 sequences with 192,007 keys 218 us against 135.
constexpr int kJoinThreads = 256;

template <typename T, int DP, int NB>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const DecodeParams p) {
  constexpr int kLanes = DP / 4, kGroups = kJoinThreads / kLanes, kSlot = 8 * NB * (DP + 2);
  __shared__ f32x4 sums[kGroups][kLanes];
  __shared__ float factors[kMaxWorkgroups], wave_stats[2][kJoinThreads / 64];
  const int32_t* entry = p.owned + 4 * blockIdx.x;
  const int s = entry[0], h = blockIdx.y, tid = threadIdx.x;
  if (s < 0) return;
  const int item = entry[1], w = entry[2], count = entry[3] - w + 1;
  const int kv_head = item / p.blocks, h0 = (item - kv_head * p.blocks) * 8 * NB;
  if (h0 + h >= p.group) return;
  const float* parts = p.parts + (int64_t)w * 2 * kSlot;
  const auto part = [&](int i) { return parts + (i == 0 ? kSlot : (int64_t)i * 2 * kSlot); };

  // At most kMaxWorkgroups parts, kEach per thread.
  constexpr int kEach = kMaxWorkgroups / kJoinThreads;
  float m[kEach], l[kEach], top = -INFINITY, weight = 0.f;
#pragma unroll
  for (int x = 0; x < kEach; ++x) {
    const int i = tid + x * kJoinThreads;
    m[x] = i < count ? part(i)[8 * NB * DP + 2 * h] : -INFINITY;
    l[x] = i < count ? part(i)[8 * NB * DP + 2 * h + 1] : 0.f;
    top = fmaxf(top, m[x]);
  }
  for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
  if ((tid & 63) == 0) wave_stats[0][tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / 64; ++i) top = fmaxf(top, wave_stats[0][i]);
#pragma unroll
  for (int x = 0; x < kEach; ++x) {
    const int i = tid + x * kJoinThreads;
    const float f = ratio(m[x], top);
    weight += l[x] * f;
    if (i < count) factors[i] = f;
  }
  for (int i = 1; i < 64; i <<= 1) weight += __shfl_xor(weight, i);
  if ((tid & 63) == 0) wave_stats[1][tid >> 6] = weight;
  __syncthreads();
  weight = 0.f;
#pragma unroll
  for (int i = 0; i < kJoinThreads / 64; ++i) weight += wave_stats[1][i];

  const int lane = tid % kLanes, group = tid / kLanes;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = group; i < count; i += kGroups)
    sum += *reinterpret_cast<const f32x4*>(part(i) + h * DP + 4 * lane) * factors[i];
  sums[group][lane] = sum;
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) sum += sums[i][lane];
  const int head = kv_head * p.group + h0 + h, d = 4 * lane;
  const float inv = weight == 0.f ? 0.f : 1.f / weight;
  if (d < p.head_dim)
    *reinterpret_cast<u32x2*>(p.out + s * p.so_t + head * p.so_h + d) =
        u32x2{T::pack(sum[0] * inv, sum[1] * inv), T::pack(sum[2] * inv, sum[3] * inv)};
  if (lane == 0 && p.lse != nullptr)
    p.lse[head * p.lse_h + s] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * kLn2;
}

template <typename T, bool kInt8, int DP, int NB>
void launch_decode(const DecodeLaunch& l) {
  if (l.any_page)
    decode_kernel<T, kInt8, DP, NB, true><<<l.workgroups, 64 * kDecodeWaves, 0, l.stream>>>(l.p);
  else
    decode_kernel<T, kInt8, DP, NB, false><<<l.workgroups, 64 * kDecodeWaves, 0, l.stream>>>(l.p);
  const int heads = l.p.group < 8 * NB ? l.p.group : 8 * NB;
  const int entries = l.p.by_item ? l.p.sequences * l.p.kv_heads * l.p.blocks : l.workgroups;
  join_kernel<T, DP, NB><<<dim3(entries, heads), kJoinThreads, 0, l.stream>>>(l.p);
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
