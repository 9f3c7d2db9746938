// The decoding attention's launch, shared by the sources that compile one head
// size's kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sa_types.h"

namespace sa {

constexpr int kDecodeWaves = 4;  // wavefronts of a workgroup
constexpr int kDecodeTile = 32;  // keys of a wave's step
// Workgroups of a CU, by the registers that a wave takes (512 of a SIMD lane).
// INT8 pages are half the bytes for more vector work per key, so that more
// waves pay: head_dim 64, 1.5 M keys of 8 heads 453 us with two, 292 with four;
// head_dim 128 with 16 query heads per K/V head, 700,000 keys of 8 heads 435 with
// one, 383 with two, also though two leave it 3 to 5 registers short (16 to 24
// bytes of scratch); with 9 query heads 433 and 369.  16-bit pages there, with more
// to spill, 443 and 522.
constexpr int decode_occupancy(int padded_dim, int blocks, PageKind kind) {
  if (padded_dim == 256 || (padded_dim == 128 && blocks == 2 && kind == kRowPages)) return 1;
  return kind != kRowPages && padded_dim == 64 && blocks == 1 ? 4 : 2;
}
constexpr int kDecodeCUs = 256;
constexpr int kMaxWorkgroups = 4 * kDecodeCUs;

// A sequence's keys of one K/V head, for up to 8 NB of its query heads, are an
// item.  The tiles of all items, sequence by sequence and head by head, are
// dealt to the waves in equal contiguous runs, so an item is in one wave's run
// or split over neighbouring ones.
struct DecodeParams {
  const uint16_t* q;
  const char *k, *v;
  const uint16_t *ks, *vs;
  const int32_t *table, *lengths;
  uint16_t* out;
  float* lse;
  float* parts;    // two per workgroup: 8 NB rows of head_dim padded, then maximum and sum of each row
  // The items that are split: (sequence or -1, item of the sequence, first and
  // last workgroup).  By item where there are no more items than workgroups
  // (by_item), else by the first workgroup, whose run ends in it.
  int32_t* owned;
  int64_t sq_t, sq_h, so_t, so_h, s_table, lse_h;
  int64_t sp, st, sh, ssp, sst, ssh;  // of the pages and their scales
  float scale_log2;
  int32_t sequences, num_pages, max_pages, head_dim, page_tokens, room;  // room: keys of a table row
  int32_t by_item;
  int32_t kv_heads, group, blocks;  // blocks: items of a K/V head
  int32_t window, sinks;            // every key: window INT32_MAX
  int32_t block_log2;               // e4m3: rows of a block
  int32_t step_pages, step_rows;    // a tile in pages and rows
  uint32_t page_magic, page_shift;  // key / page_tokens = key * magic >> shift
};

struct DecodeLaunch {
  DecodeParams p;
  int32_t workgroups;
  bool bf16;
  PageKind kind;
  bool wide;      // 16 query heads per item instead of 8
  bool any_page;  // pages that end inside 16 keys
  hipStream_t stream;
};

// One padded head_dim each.
void launch_decode_d64(const DecodeLaunch& l);
void launch_decode_d128(const DecodeLaunch& l);
void launch_decode_d256(const DecodeLaunch& l);

}  // namespace sa
