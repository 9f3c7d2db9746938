// Entry points of the decoding attention (sa_decode.h, sa_decode_kernel.h).

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "sa_common.h"
#include "sa_decode.h"

namespace sa {
namespace {

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int32_t invalid(const char* what) {
  set_error("sa_paged_decode: %s", what);
  return SA_ERR_INVALID_ARGUMENT;
}

int32_t check(const sa_decode_args* a) {
  if (a->dtype != SA_DTYPE_BF16 && a->dtype != SA_DTYPE_FP16) {
    set_error("sa_paged_decode: unsupported dtype code %d", a->dtype);
    return SA_ERR_UNSUPPORTED_DTYPE;
  }
  if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 8) {
    set_error("sa_paged_decode: head_dim must be a multiple of 8 in [16, 256], got %d", a->head_dim);
    return SA_ERR_UNSUPPORTED_HEAD_DIM;
  }
  if (a->kv_heads < 1 || a->q_heads < 1 || a->q_heads > (1 << 16) || a->q_heads % a->kv_heads)
    return invalid("q_heads must be a multiple of kv_heads");
  if (a->sequences > (1 << 30)) return invalid("at most 2^30 sequences");
  if (a->sequences < 0 || a->max_pages < 0 || a->page_tokens < 1 || a->page_tokens > SA_MAX_PAGE_TOKENS ||
      a->num_pages < 0 || a->num_pages > INT32_MAX / a->page_tokens || a->max_pages > INT32_MAX / a->page_tokens)
    return invalid("page_tokens must be at most 2^20 and pages * page_tokens below 2^31");
  return 0;
}

int padded(int32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Workgroups of a launch: what the chip holds at once.  A launch over fewer
// tiles leaves some without work.
bool wide(const sa_decode_args* a) { return a->q_heads / a->kv_heads > 8; }
PageKind kind_of(const sa_decode_args* a) {
  return a->pages_int8 == SA_PAGES_E4M3 ? kE4m3Pages : a->pages_int8 ? kInt8Pages : kRowPages;
}
int workgroups(const sa_decode_args* a, PageKind kind) {
  return kDecodeCUs * decode_occupancy(padded(a->head_dim), wide(a) ? 2 : 1, kind);
}

// owned, then parts.
int64_t owned_bytes(const sa_decode_args* a, PageKind kind) { return (int64_t)workgroups(a, kind) * 16; }
int64_t workspace_bytes(const sa_decode_args* a, PageKind kind) {
  return owned_bytes(a, kind) + (int64_t)workgroups(a, kind) * 2 * (wide(a) ? 16 : 8) * (padded(a->head_dim) + 2) * 4;
}

}  // namespace
}  // namespace sa

extern "C" {

int32_t sa_paged_decode_workspace_bytes(const sa_decode_args* a, int32_t device, int64_t* bytes) {
  (void)device;
  sa::clear_error();
  if (a == nullptr || bytes == nullptr) return sa::invalid("null arguments");
  const int32_t rc = sa::check(a);
  *bytes = rc == 0 && a->sequences > 0 ? sa::workspace_bytes(a, sa::kind_of(a)) : 0;
  return rc;
}

}  // extern "C"

namespace sa {
namespace {

// window INT32_MAX: every key.
int32_t run(const sa_decode_args* a, PageKind kind, int32_t window, int32_t sinks, int32_t block_tokens, int32_t device,
            void* stream) {
  const int32_t rc = check(a);
  if (rc != 0) return rc;
  const int32_t log2 = kind == kE4m3Pages ? block_log2(block_tokens, a->page_tokens) : 0;
  if (log2 < 0) return invalid("block_tokens must be a power of two from 16 on that divides page_tokens");
  if (a->sequences == 0) return 0;
  if (a->num_pages < 1) return invalid("the pool must have at least one page");  // the kernel reads page 0 for bad pages
  const int64_t strides[] = {a->stride_qt, a->stride_qh, a->stride_ot, a->stride_oh, a->stride_pp, a->stride_pt,
                             a->stride_ph};
  for (int64_t s : strides)
    if (s % 8) return invalid("strides must be multiples of 8 elements");
  const int64_t page_align = kind != kRowPages ? 8 : 16;
  if (a->q == nullptr || a->out == nullptr || a->k_pages == nullptr || a->v_pages == nullptr || a->lengths == nullptr ||
      (a->page_table == nullptr && a->max_pages > 0) ||
      (kind != kRowPages && (a->k_scales == nullptr || a->v_scales == nullptr)) || !aligned(a->q, 16) ||
      !aligned(a->out, 16) || !aligned(a->k_pages, page_align) || !aligned(a->v_pages, page_align) ||
      !aligned(a->page_table, 4) || !aligned(a->lengths, 4) || !aligned(a->lse, 4) ||
      (kind != kE4m3Pages && (!aligned(a->k_scales, 2) || !aligned(a->v_scales, 2))))
    return invalid("an operand is missing or not aligned");
  if (a->workspace == nullptr || !aligned(a->workspace, 16) || a->workspace_bytes < workspace_bytes(a, kind))
    return invalid("the workspace is missing, too small or not aligned");
  if (a->stride_pt < 0 || a->stride_pt >= (1 << 26))
    return invalid("the pages' token stride must be below 2^26 elements");
  DecodeLaunch launch{};
  DecodeParams& p = launch.p;
  p.q = static_cast<const uint16_t*>(a->q), p.out = static_cast<uint16_t*>(a->out), p.lse = a->lse;
  p.k = static_cast<const char*>(a->k_pages), p.v = static_cast<const char*>(a->v_pages);
  p.ks = static_cast<const uint16_t*>(a->k_scales), p.vs = static_cast<const uint16_t*>(a->v_scales);
  p.table = a->page_table, p.lengths = a->lengths;
  p.sq_t = a->stride_qt, p.sq_h = a->stride_qh, p.so_t = a->stride_ot, p.so_h = a->stride_oh;
  p.sp = a->stride_pp, p.st = a->stride_pt, p.sh = a->stride_ph;
  p.ssp = a->stride_sp, p.sst = a->stride_st, p.ssh = a->stride_sh;
  p.s_table = a->stride_table, p.lse_h = a->lse_stride_h;
  p.scale_log2 = (float)(a->softmax_scale * 1.4426950408889634074);
  p.sequences = a->sequences, p.num_pages = (int32_t)a->num_pages, p.max_pages = a->max_pages;
  p.head_dim = a->head_dim, p.page_tokens = a->page_tokens, p.room = a->max_pages * a->page_tokens;
  launch.wide = wide(a);
  p.kv_heads = a->kv_heads, p.group = a->q_heads / a->kv_heads;
  const int32_t item_heads = launch.wide ? 16 : 8;
  p.blocks = (p.group + item_heads - 1) / item_heads;
  p.step_pages = kDecodeTile / p.page_tokens, p.step_rows = kDecodeTile % p.page_tokens;
  // Exact for keys below 2^31: magic = floor(2^(31 + n) / page_tokens) + 1 with
  // 2^n >= page_tokens is off by less than 2^-31 of a page per key.
  uint32_t n = 0;
  while ((1u << n) < (uint32_t)p.page_tokens) ++n;
  p.page_shift = 31 + n;
  p.page_magic = (uint32_t)(((uint64_t)1 << p.page_shift) / (uint32_t)p.page_tokens + 1);
  p.owned = static_cast<int32_t*>(a->workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + owned_bytes(a, kind));
  launch.workgroups = workgroups(a, kind);
  p.by_item = (int64_t)a->sequences * p.kv_heads * p.blocks <= launch.workgroups;
  p.window = window, p.sinks = sinks, p.block_log2 = log2;
  launch.bf16 = a->dtype == SA_DTYPE_BF16, launch.kind = kind;
  launch.any_page = a->page_tokens % 16 != 0;
  launch.stream = static_cast<hipStream_t>(stream);
  DeviceGuard guard(device);
  SA_HIP_RETURN(guard.status());
  const int width = padded(a->head_dim);
  (width == 64 ? launch_decode_d64 : width == 128 ? launch_decode_d128 : launch_decode_d256)(launch);
  SA_HIP_RETURN(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace sa

extern "C" {

int32_t sa_paged_decode(const sa_decode_args* a, int32_t device, void* stream) try {
  sa::clear_error();
  if (a == nullptr) return sa::invalid("null arguments");
  if (a->pages_int8 == SA_PAGES_E4M3) return sa::invalid("e4m3 pages are read by sa_paged_window_decode");
  return sa::run(a, a->pages_int8 ? sa::kInt8Pages : sa::kRowPages, INT32_MAX, 0, 0, device, stream);
} catch (const std::exception& error) {
  return sa::exception_status("sa_paged_decode", error);
}

int32_t sa_paged_window_decode(const sa_window_decode_args* a, int32_t device, void* stream) try {
  sa::clear_error();
  if (a == nullptr) return sa::invalid("null arguments");
  const int32_t kind = a->base.pages_int8;
  if (kind < sa::kRowPages || kind > sa::kE4m3Pages) return sa::invalid("unknown kind of pages");
  if (a->window < 0 || a->sinks < 0 || (a->window == 0 && a->sinks > 0))
    return sa::invalid("window and sinks must not be negative, and sinks need a window");
  return sa::run(&a->base, (sa::PageKind)kind, a->window > 0 ? a->window : INT32_MAX, a->sinks, a->block_tokens, device,
                 stream);
} catch (const std::exception& error) {
  return sa::exception_status("sa_paged_window_decode", error);
}

}  // extern "C"
