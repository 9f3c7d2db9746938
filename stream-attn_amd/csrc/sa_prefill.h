// The launch of a prompt's attention over the paged cache, shared by the sources
// that compile one head size's kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sa_types.h"

namespace sa {

constexpr int kPrefillTile = 64;     // keys of a workgroup's step
constexpr int kPrefillThreads = 512; // 8 waves
constexpr int kPrefillCUs = 256;
// Bytes of a float per element and of a row's maximum and sum.
constexpr int64_t prefill_part_floats(int rows, int padded_dim) { return (int64_t)rows * (padded_dim + 2); }

// A sequence's new tokens times the query heads of one K/V head are its rows, one
// (token, head) each, token by token.  A block is a workgroup's rows of one
// sequence; every K/V head has the same blocks.
struct PrefillBlock {
  int64_t before;  // tiles of the blocks before it
  int32_t sequence, row;
};
struct PrefillPlan {
  int64_t tiles;  // of all blocks
  int32_t blocks;
  int32_t whole;    // items are not split, each XCD's workgroups take its items in turn
  int32_t next[8];  // of every XCD
};
// An item (a K/V head's block) that is split over runs first .. last.
struct PrefillSplit {
  int32_t block, head;  // block -1: none
  int32_t last, pad;
};

struct PrefillParams {
  const uint16_t* q;
  const char *k, *v;
  const void *ks, *vs;
  const int32_t *table, *lengths, *cu;
  uint16_t* out;
  float* lse;
  PrefillPlan* plan;
  PrefillBlock* blocks;
  int32_t* first_block;  // of every sequence, the plan's
  int32_t* order;        // whole items: the blocks, long ones first
  PrefillSplit* splits;  // by the run that an item starts in
  float* parts;          // two per run
  int64_t sq_t, sq_h, so_t, so_h, sp, st, sh, ssp, sst, ssh, s_table, lse_h, tokens;
  float scale_log2;
  int32_t sequences, num_pages, max_pages, head_dim, page_tokens, room, kv_heads, group;
  int32_t window, sinks;  // every key: window INT32_MAX
  int32_t block_log2, max_blocks, any_page, runs, rows;
  uint32_t page_magic, page_shift, group_magic, group_shift;  // x / page_tokens = x * magic >> shift
};

struct PrefillLaunch {
  PrefillParams p;
  bool bf16;
  PageKind kind;
  hipStream_t stream;
};

// Rows of a workgroup: 128 or, with many rows, what the registers hold.
constexpr int prefill_rows(int padded_dim, bool many) { return !many ? 128 : padded_dim == 128 ? 384 : 256; }

// Workgroups of a CU: two where registers and LDS hold them.  One sequence, 32/8 heads of
// 128, narrow, two of two stages against one of four, us: 2,048 tokens with a window of 512
// 53 and 57, 512 behind 20,000 keys with one of 1,024 43 and 47, 2,048 tokens of 16/16
// heads 58 and 63, with a window of 512 (fewer items than CUs) 43 and 40.
//
// Not all registers are there: scratch of a lane, bytes, by rows of a workgroup (16-bit
// pages; 8-bit ones): head_dim 64, 256 rows 24; 36 to 76; 128, 128 rows 56; none, 384 rows
// none; 20 to 32; 256, 256 rows 148; 236 to 252; 128 rows of 64 and 256 none.  All times
// here and at rows_of() are with it.
constexpr int prefill_occupancy(int padded_dim, int rows, PageKind kind) {
  return padded_dim == 64 || (padded_dim == 128 && rows == 128 && kind == kRowPages) ? 2 : 1;
}

// One padded head_dim each.
hipError_t launch_prefill_d64(const PrefillLaunch& l);
hipError_t launch_prefill_d128(const PrefillLaunch& l);
hipError_t launch_prefill_d256(const PrefillLaunch& l);

#ifdef __HIPCC__
namespace {

// A sequence's new tokens: rows `from` .. of q, the first at position `base`.
struct PrefillSequence {
  int32_t from, count, base;
};
template <typename Params>
__device__ inline PrefillSequence prefill_sequence(const Params& p, int32_t s) {
  int64_t from = p.cu[s], to = p.cu[s + 1];
  from = from < 0 ? 0 : from > p.tokens ? p.tokens : from;
  to = to < from ? from : to > p.tokens ? p.tokens : to;
  int32_t length = p.lengths[s];
  length = length < 0 ? 0 : length > p.room ? p.room : length;
  return {(int32_t)from, (int32_t)(to - from), length - (int32_t)(to - from)};
}

template <typename Params>
__device__ inline int32_t prefill_query(const Params& p, int32_t row) {
  return (int32_t)((uint64_t)(uint32_t)row * p.group_magic >> p.group_shift);
}

// The tiles that hold a key that one of the rows row .. end - 1 sees: all up to the
// last row's position, or those up to the sinks' last and those from the first
// row's window on, `skip` tiles later.  One, of which no key is seen, where there
// are none: the rows are written all the same.
struct PrefillTiles {
  int32_t count, sinks, skip;
  __device__ inline int32_t key_of(int32_t tile) const { return (tile + (tile < sinks ? 0 : skip)) * kPrefillTile; }
};
template <typename Params>
__device__ inline PrefillTiles prefill_tiles(const Params& p, const PrefillSequence& s, int32_t row, int32_t end) {
  const int32_t last = s.base + prefill_query(p, end - 1);
  if (last < 0) return {1, 1, 0};
  const int32_t all = last / kPrefillTile + 1;
  const int64_t low64 = (int64_t)s.base + prefill_query(p, row) - p.window + 1;
  if (low64 <= 0) return {all, all, 0};
  const int32_t low = (int32_t)low64, first = p.sinks < low ? p.sinks : low;
  const int32_t sinks = first > 0 ? (first - 1) / kPrefillTile + 1 : 0, between = low / kPrefillTile - sinks;
  return between > 0 ? PrefillTiles{all - between, sinks, between} : PrefillTiles{all, all, 0};
}

}  // namespace
#endif

}  // namespace sa
