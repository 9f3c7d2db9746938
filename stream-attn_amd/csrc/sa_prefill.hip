// Entry points of a prompt's attention over the paged cache and the plan of its
// launch (sa_prefill.h, sa_prefill_kernel.h).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sa_common.h"
#include "sa_prefill.h"

namespace sa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanSequences = 4096;  // whose first blocks LDS holds
constexpr int kClasses = 8;           // of blocks, by their tiles
// What splitting items costs a workgroup, in tiles: writing and joining the parts.  With
// 0, this and 20, us: one sequence of 32/8 heads of 128, 2,048 tokens with a window of 512
// 70, 53, 54; 9,000 with one of 1,024 221, 192, 192; 4,000 without 197, 197, 215; 16/16 of
// 256, 3,000 tokens 148, 160, 160 (5 tiles 148); 12/4 of 64, four sequences, 9,000 tokens with a window of
// 2,048 87, 88, 93; nine, 2,700 behind 36,000 INT8 keys 70, 70, 99.
constexpr int kSplitTiles = 10;

// Inclusive sum over a workgroup's threads; `sums` has a place per wave and one more.
__device__ inline int64_t scan(int64_t x, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = 1; i < 64; i <<= 1) {
    const int64_t y = __shfl_up(x, i);
    if (lane >= i) x += y;
  }
  __syncthreads();  // the sums of an earlier call are read
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  total = 0;
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i < wave) x += sums[i];
    total += sums[i];
  }
  return x;
}

// The blocks of all sequences and the tiles before each: one workgroup, a thread
// per block after one pass over the sequences.
__global__ __launch_bounds__(kPlanThreads) void prefill_plan_kernel(const PrefillParams p) {
  __shared__ int64_t sums[kPlanThreads / 64];
  __shared__ int32_t first_lds[kPlanSequences];
  __shared__ int32_t most, of_class[kClasses], done[kClasses], of_wave[kPlanThreads / 64][kClasses];
  const int tid = threadIdx.x;
  const bool in_lds = p.sequences <= kPlanSequences;
  const int run = (p.sequences + kPlanThreads - 1) / kPlanThreads;
  const int s_first = min(tid * run, p.sequences), s_last = min(s_first + run, p.sequences);
  const auto blocks_of = [&](int s) -> int64_t {
    return ((int64_t)prefill_sequence(p, s).count * p.group + p.rows - 1) / p.rows;
  };
  int64_t own = 0, all;
  for (int s = s_first; s < s_last; ++s) own += blocks_of(s);
  int64_t before = scan(own, sums, all) - own;
  for (int s = s_first; s < s_last; ++s) {
    const int32_t first = (int32_t)min(before, (int64_t)p.max_blocks);
    if (in_lds)
      first_lds[s] = first;
    else
      p.first_block[s] = first;
    before += blocks_of(s);
  }
  if (tid < kClasses) of_class[tid] = 0;
  if (tid == 0) most = 1;
  __syncthreads();
  const int blocks = (int)min(all, (int64_t)p.max_blocks);  // more only if the starts are in disorder
  int64_t tiles = 0;
  int count = 0;  // of the thread's last block
  for (int base = 0; base < blocks; base += kPlanThreads) {
    const int i = base + tid;
    int s = 0, row = 0;
    count = 0;
    if (i < blocks) {
      // The last sequence whose first block is not past i.
      for (int left = p.sequences; left > 1;) {
        const int half = left >> 1, first = in_lds ? first_lds[s + half] : p.first_block[s + half];
        if (first <= i) s += half, left -= half;
        else left = half;
      }
      row = (i - (in_lds ? first_lds[s] : p.first_block[s])) * p.rows;
      const PrefillSequence seq = prefill_sequence(p, s);
      count = prefill_tiles(p, seq, row, min(seq.count * p.group, row + p.rows)).count;
    }
    int64_t of_all;
    const int64_t upto = scan(count, sums, of_all);
    if (i < blocks) p.blocks[i] = {tiles + upto - count, s, row}, atomicMax(&most, count);
    tiles += of_all;
  }
  __syncthreads();
  // Whole items, long ones first, where their longest workgroup has hardly more than an
  // equal share and splitting costs more.  A block's class: 0 has the longest.
  const float class_tiles = (float)kClasses / (float)most;
  const auto class_of = [&](int i) {
    int tiles_of = count;
    if (blocks > kPlanThreads) tiles_of = (int)((i + 1 < blocks ? p.blocks[i + 1].before : tiles) - p.blocks[i].before);
    return max(0, kClasses - 1 - (int)((float)(tiles_of - 1) * class_tiles));
  };
  for (int i = tid; i < blocks; i += kPlanThreads) atomicAdd(&of_class[class_of(i)], 1);
  __syncthreads();
  float items = 0.f, longest = 0.f;
  for (int c = 0; c < kClasses; ++c) {
    items += (float)of_class[c] * (float)p.kv_heads;
    longest = fmaxf(longest, ceilf(items / (float)p.runs) * ((float)(kClasses - c) - 0.5f) / class_tiles);
  }
  const bool whole = longest <= (float)tiles * (float)p.kv_heads / (float)p.runs + kSplitTiles;
  if (whole) {
    // The last blocks first, stable, so that neighbours stay together.
    const int lane = tid & 63, wave = tid >> 6;
    for (int chunk = 0; chunk < blocks; chunk += kPlanThreads) {
      const int base = (blocks - 1 - chunk) / kPlanThreads * kPlanThreads, i = base + tid;  // whole chunks from the last on
      const int mine = i < blocks ? class_of(i) : -1;
      int behind = 0;  // of the class, on later lanes
      for (int c = 0; c < kClasses; ++c) {
        const uint64_t same = __ballot(mine == c);
        if (mine == c) behind = __popcll(same >> 1 >> lane);
        if (lane == 0) of_wave[wave][c] = __popcll(same);
      }
      __syncthreads();
      if (mine >= 0) {
        int at = behind;
        for (int c = 0; c < mine; ++c) at += of_class[c];
        for (int w = wave + 1; w < kPlanThreads / 64; ++w) at += of_wave[w][mine];
        p.order[at + (chunk > 0 ? done[mine] : 0)] = i;
      }
      __syncthreads();
      if (tid < kClasses) {
        int sum = chunk > 0 ? done[tid] : 0;
        for (int w = 0; w < kPlanThreads / 64; ++w) sum += of_wave[w][tid];
        done[tid] = sum;
      }
      __syncthreads();
    }
  }
  if (tid == 0) *p.plan = {tiles, blocks, whole, {}};
}

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int32_t invalid(const char* what) {
  set_error("sa_paged_prefill: %s", what);
  return SA_ERR_INVALID_ARGUMENT;
}

int32_t check(const sa_prefill_args* a) {
  if (a->dtype != SA_DTYPE_BF16 && a->dtype != SA_DTYPE_FP16) {
    set_error("sa_paged_prefill: unsupported dtype code %d", a->dtype);
    return SA_ERR_UNSUPPORTED_DTYPE;
  }
  const int32_t kind = a->pages_kind;
  if (kind < kRowPages || kind > kE4m3Pages) return invalid("unknown kind of pages");
  const int32_t step = kind == kRowPages ? 8 : 16;
  if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % step) {
    set_error("sa_paged_prefill: head_dim must be a multiple of %d in [16, 256], got %d", step, a->head_dim);
    return SA_ERR_UNSUPPORTED_HEAD_DIM;
  }
  if (a->kv_heads < 1 || a->q_heads < 1 || a->q_heads > (1 << 16) || a->q_heads % a->kv_heads)
    return invalid("q_heads must be a multiple of kv_heads");
  if (a->sequences < 0 || a->sequences > (1 << 30) || a->tokens < 0 ||
      a->tokens > (INT32_MAX - 4096) / (a->q_heads / a->kv_heads))
    return invalid("at most 2^30 sequences, and tokens times query heads per K/V head below 2^31 - 4096");
  if (a->max_pages < 0 || a->page_tokens < 1 || a->page_tokens > SA_MAX_PAGE_TOKENS || a->num_pages < 0 ||
      a->num_pages > INT32_MAX / a->page_tokens || a->max_pages > INT32_MAX / a->page_tokens)
    return invalid("page_tokens must be at most 2^20 and pages * page_tokens below 2^31");
  if (a->window < 0 || a->sinks < 0 || (a->window == 0 && a->sinks > 0))
    return invalid("window and sinks must not be negative, and sinks need a window");
  if (kind == kE4m3Pages && block_log2(a->block_tokens, a->page_tokens) < 0)
    return invalid("block_tokens must be a power of two from 16 on that divides page_tokens");
  return 0;
}

int padded(int32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Where the parts of the workspace start.
struct Workspace {
  int32_t rows, runs;
  int64_t max_blocks, blocks, order, first_block, splits, parts, bytes;
};

// Rows of a workgroup.  Wide ones take less time per row and tile (head_dim 128 2.0, 256
// 1.4, 64 1.2 times less) and more to start, end, split and even out, so they need many
// tiles for every workgroup, and sequences that fill them.  The tiles are guessed: of a
// window, else of all keys that the table has room for before a middle token.  (Lengths are
// not known here: in a table with far more room a short prompt gets wide ones.)
// One sequence, wide and narrow in us, guessed tiles:
//   head_dim 128, 32/8 heads: 2,048 tokens 104, 97 (11); 6,000 with a window of 512 102, 131
//   (18); 128 behind 20,000 keys 108, 90 (13); 256 128, 141 (26); 2,048 587, 887;
//   256, 16/16 heads: 6,000 tokens 425, 382 (70); with a window of 1,024 239, 170 (27);
//   2,048 behind 20,000 keys 615, 755 (156); 512 250, 232 (39);
//   64, 12/4 heads: 6,000 tokens 116, 128 (26); 512 behind 20,000 keys 68, 77 (15); 256 59,
//   52 (7); 512 with a window of 1,024 44, 35 (1).
int32_t rows_of(const sa_prefill_args* a, int dim, int64_t rows, int32_t runs) {
  const int many = prefill_rows(dim, true);
  if (rows < (int64_t)a->sequences * many * 2) return 128;
  double keys = (double)a->max_pages * a->page_tokens - 0.5 * (double)a->tokens / a->sequences;
  if (a->window > 0) keys = std::min(keys, (double)a->window + a->sinks);
  const double tiles = (double)rows / many * a->kv_heads / runs * (keys / kPrefillTile + 1);
  return tiles >= (dim == 128 ? 16 : dim == 256 ? 80 : 9) ? many : 128;
}

Workspace workspace(const sa_prefill_args* a) {
  Workspace w;
  const int dim = padded(a->head_dim);
  const int64_t rows = a->tokens * (a->q_heads / a->kv_heads);
  w.rows = rows_of(a, dim, rows, kPrefillCUs * (dim == 64 ? 2 : 1));
  w.runs = kPrefillCUs * prefill_occupancy(dim, w.rows, (PageKind)a->pages_kind);
  w.max_blocks = std::min(rows, rows / w.rows + a->sequences);
  const auto next = [](int64_t at) { return (at + 255) & ~(int64_t)255; };
  w.blocks = next(sizeof(PrefillPlan));
  w.order = next(w.blocks + w.max_blocks * (int64_t)sizeof(PrefillBlock));
  w.first_block = next(w.order + w.max_blocks * 4);
  w.splits = next(w.first_block + (a->sequences > kPlanSequences ? a->sequences * (int64_t)4 : 0));
  w.parts = next(w.splits + w.runs * (int64_t)sizeof(PrefillSplit));
  w.bytes = w.parts + w.runs * 2 * prefill_part_floats(w.rows, dim) * 4;
  return w;
}

// x / by = x * magic >> shift for x below 2^31: magic = floor(2^(31 + n) / by) + 1
// with 2^n >= by is off by less than 2^-31 per unit of x.
void divider(uint32_t by, uint32_t& magic, uint32_t& shift) {
  uint32_t n = 0;
  while ((1u << n) < by) ++n;
  shift = 31 + n;
  magic = (uint32_t)(((uint64_t)1 << shift) / by + 1);
}

}  // namespace
}  // namespace sa

extern "C" {

int32_t sa_paged_prefill_workspace_bytes(const sa_prefill_args* a, int32_t device, int64_t* bytes) {
  (void)device;
  sa::clear_error();
  if (a == nullptr || bytes == nullptr) return sa::invalid("null arguments");
  const int32_t rc = sa::check(a);
  *bytes = rc == 0 && a->tokens > 0 && a->sequences > 0 ? sa::workspace(a).bytes : 0;
  return rc;
}

int32_t sa_paged_prefill(const sa_prefill_args* a, int32_t device, void* stream) try {
  using namespace sa;
  clear_error();
  if (a == nullptr) return invalid("null arguments");
  const int32_t rc = check(a);
  if (rc != 0) return rc;
  if (a->tokens == 0 || a->sequences == 0) return 0;
  if (a->num_pages < 1) return invalid("the pool must have at least one page");  // the kernel reads page 0 for bad pages
  const PageKind kind = (PageKind)a->pages_kind;
  const int64_t page_step = kind == kRowPages ? 8 : 16;  // elements
  for (int64_t s : {a->stride_qt, a->stride_qh, a->stride_ot, a->stride_oh})
    if (s % 8) return invalid("strides must be multiples of 8 elements");
  for (int64_t s : {a->stride_pp, a->stride_pt, a->stride_ph})
    if (s % page_step) return invalid("the pages' strides must be multiples of 16 bytes");
  // An offset within 16 rows of a page has 32 bits.
  if (a->stride_pt < 0 || a->stride_pt >= (1 << 26)) return invalid("the pages' token stride must be below 2^26 elements");
  if (a->q == nullptr || a->out == nullptr || a->k_pages == nullptr || a->v_pages == nullptr || a->lengths == nullptr ||
      a->cu_tokens == nullptr || (a->page_table == nullptr && a->max_pages > 0) ||
      (kind != kRowPages && (a->k_scales == nullptr || a->v_scales == nullptr)) || !aligned(a->q, 16) ||
      !aligned(a->out, 16) || !aligned(a->k_pages, 16) || !aligned(a->v_pages, 16) || !aligned(a->page_table, 4) ||
      !aligned(a->lengths, 4) || !aligned(a->cu_tokens, 4) || !aligned(a->lse, 4) ||
      (kind == kInt8Pages && (!aligned(a->k_scales, 2) || !aligned(a->v_scales, 2))))
    return invalid("an operand is missing or not aligned");
  const Workspace w = workspace(a);
  if (a->workspace == nullptr || !aligned(a->workspace, 16) || a->workspace_bytes < w.bytes)
    return invalid("the workspace is missing, too small or not aligned");
  if (w.max_blocks > INT32_MAX / a->kv_heads) return invalid("too many tokens and sequences");
  PrefillLaunch launch{};
  PrefillParams& p = launch.p;
  p.q = static_cast<const uint16_t*>(a->q), p.out = static_cast<uint16_t*>(a->out), p.lse = a->lse;
  p.k = static_cast<const char*>(a->k_pages), p.v = static_cast<const char*>(a->v_pages);
  p.ks = a->k_scales, p.vs = a->v_scales;
  p.table = a->page_table, p.lengths = a->lengths, p.cu = a->cu_tokens;
  char* base = static_cast<char*>(a->workspace);
  p.plan = reinterpret_cast<PrefillPlan*>(base);
  p.blocks = reinterpret_cast<PrefillBlock*>(base + w.blocks);
  p.order = reinterpret_cast<int32_t*>(base + w.order);
  p.first_block = reinterpret_cast<int32_t*>(base + w.first_block);
  p.splits = reinterpret_cast<PrefillSplit*>(base + w.splits);
  p.parts = reinterpret_cast<float*>(base + w.parts);
  p.sq_t = a->stride_qt, p.sq_h = a->stride_qh, p.so_t = a->stride_ot, p.so_h = a->stride_oh;
  p.sp = a->stride_pp, p.st = a->stride_pt, p.sh = a->stride_ph;
  p.ssp = a->stride_sp, p.sst = a->stride_st, p.ssh = a->stride_sh;
  p.s_table = a->stride_table, p.lse_h = a->lse_stride_h, p.tokens = a->tokens;
  p.scale_log2 = (float)(a->softmax_scale * 1.4426950408889634074);
  p.sequences = a->sequences, p.num_pages = (int32_t)a->num_pages, p.max_pages = a->max_pages;
  p.head_dim = a->head_dim, p.page_tokens = a->page_tokens, p.room = a->max_pages * a->page_tokens;
  p.kv_heads = a->kv_heads, p.group = a->q_heads / a->kv_heads;
  p.window = a->window > 0 ? a->window : INT32_MAX, p.sinks = a->sinks;
  p.block_log2 = kind == kE4m3Pages ? block_log2(a->block_tokens, a->page_tokens) : 0;
  p.max_blocks = (int32_t)w.max_blocks, p.any_page = a->page_tokens % 16 != 0, p.runs = w.runs, p.rows = w.rows;
  divider((uint32_t)p.page_tokens, p.page_magic, p.page_shift);
  divider((uint32_t)p.group, p.group_magic, p.group_shift);
  launch.bf16 = a->dtype == SA_DTYPE_BF16, launch.kind = kind, launch.stream = static_cast<hipStream_t>(stream);
  DeviceGuard guard(device);
  SA_HIP_RETURN(guard.status());
  prefill_plan_kernel<<<1, kPlanThreads, 0, launch.stream>>>(p);
  SA_HIP_RETURN(hipGetLastError());
  const int width = padded(a->head_dim);
  SA_HIP_RETURN((width == 64 ? launch_prefill_d64 : width == 128 ? launch_prefill_d128 : launch_prefill_d256)(launch));
  return 0;
} catch (const std::exception& error) {
  return sa::exception_status("sa_paged_prefill", error);
}

}  // extern "C"
