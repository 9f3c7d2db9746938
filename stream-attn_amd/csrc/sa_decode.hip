// Attention of one new token per sequence over a paged K/V cache.
//
//   s_j = scale * q . k_j,  out = sum_j e^(s_j) v_j / sum_j e^(s_j),  lse = log sum_j e^(s_j)
//
// The plainest form: a wave per (sequence, query head), one key at a time.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "sa_common.h"
#include "sa_types.h"

namespace sa {
namespace {

struct DecodeParams {
  const uint16_t* q;
  const char *k, *v;
  const uint16_t *ks, *vs;
  const int32_t *table, *lengths;
  uint16_t* out;
  float* lse;
  int64_t sq_t, sq_h, so_t, so_h, kp, kt, kh, vp, vt, vh, ksp, kst, ksh, vsp, vst, vsh, s_table, lse_h;
  float scale_log2;
  int32_t num_pages, max_pages, group, head_dim, page_tokens;
};

template <typename T, bool kInt8>
__device__ inline float element(const char* base, int64_t at) {
  if constexpr (kInt8) return (float)base[at];
  return T::lo(reinterpret_cast<const uint16_t*>(base)[at]);
}

template <typename T, bool kInt8>
__global__ __launch_bounds__(64) void decode_kernel(const DecodeParams p) {
  const int s = blockIdx.x, h = blockIdx.y, kvh = h / p.group, lane = threadIdx.x;
  const int64_t room = (int64_t)p.max_pages * p.page_tokens;
  const int64_t len = p.lengths[s] < room ? p.lengths[s] : room;
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    q[i] = d < p.head_dim ? T::lo(p.q[s * p.sq_t + h * p.sq_h + d]) : 0.f;
  }
  for (int64_t j = 0; j < len; ++j) {
    const int32_t page = p.table[s * p.s_table + j / p.page_tokens];
    const int64_t row = j % p.page_tokens;
    if (page < 0 || page >= p.num_pages) continue;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < p.head_dim) dot += q[i] * element<T, kInt8>(p.k, page * p.kp + row * p.kt + kvh * p.kh + d);
    }
    for (int i = 1; i < 64; i <<= 1) dot += __shfl_xor(dot, i);
    if (kInt8) dot *= Fp16::lo(p.ks[page * p.ksp + row * p.kst + kvh * p.ksh]);
    if (dot * p.scale_log2 == -INFINITY) continue;
    const float x = dot * p.scale_log2, top = fmaxf(m, x);
    const float keep = exp2f(m - top), w = exp2f(x - top);
    m = top;
    l = l * keep + w;
    const float vw = kInt8 ? w * Fp16::lo(p.vs[page * p.vsp + row * p.vst + kvh * p.vsh]) : w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < p.head_dim) acc[i] = acc[i] * keep + vw * element<T, kInt8>(p.v, page * p.vp + row * p.vt + kvh * p.vh + d);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < p.head_dim) p.out[s * p.so_t + h * p.so_h + d] = (uint16_t)T::pack(l == 0.f ? 0.f : acc[i] / l, 0.f);
  }
  if (p.lse != nullptr && lane == 0) p.lse[h * p.lse_h + s] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
}

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
  if (a->sequences < 0 || a->max_pages < 0 || a->page_tokens < 1 || a->num_pages < 0 ||
      a->num_pages > INT32_MAX / a->page_tokens || a->max_pages > INT32_MAX / a->page_tokens)
    return invalid("pages * page_tokens must be below 2^31");
  return 0;
}

}  // namespace
}  // namespace sa

extern "C" {

int32_t sa_paged_decode_workspace_bytes(const sa_decode_args* a, int32_t device, int64_t* bytes) {
  (void)device;
  sa::clear_error();
  if (a == nullptr || bytes == nullptr) return sa::invalid("null arguments");
  const int32_t rc = sa::check(a);
  *bytes = 0;
  return rc;
}

int32_t sa_paged_decode(const sa_decode_args* a, int32_t device, void* stream) try {
  using namespace sa;
  clear_error();
  if (a == nullptr) return invalid("null arguments");
  const int32_t rc = check(a);
  if (rc != 0) return rc;
  if (a->sequences == 0) return 0;
  const int64_t strides[] = {a->stride_qt, a->stride_qh, a->stride_ot, a->stride_oh, a->stride_kpp, a->stride_kpt,
                             a->stride_kph, a->stride_vpp, a->stride_vpt, a->stride_vph};
  for (int64_t s : strides)
    if (s % 8) return invalid("strides must be multiples of 8 elements");
  const int64_t page_align = a->pages_int8 ? 8 : 16;
  if (a->q == nullptr || a->out == nullptr || a->k_pages == nullptr || a->v_pages == nullptr || a->lengths == nullptr ||
      (a->page_table == nullptr && a->max_pages > 0) || (a->pages_int8 && (a->k_scales == nullptr || a->v_scales == nullptr)) ||
      !aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->k_pages, page_align) || !aligned(a->v_pages, page_align) ||
      !aligned(a->page_table, 4) || !aligned(a->lengths, 4))
    return invalid("an operand is missing or not aligned");
  DecodeParams p{};
  p.q = static_cast<const uint16_t*>(a->q), p.out = static_cast<uint16_t*>(a->out), p.lse = a->lse;
  p.k = static_cast<const char*>(a->k_pages), p.v = static_cast<const char*>(a->v_pages);
  p.ks = static_cast<const uint16_t*>(a->k_scales), p.vs = static_cast<const uint16_t*>(a->v_scales);
  p.table = a->page_table, p.lengths = a->lengths;
  p.sq_t = a->stride_qt, p.sq_h = a->stride_qh, p.so_t = a->stride_ot, p.so_h = a->stride_oh;
  p.kp = a->stride_kpp, p.kt = a->stride_kpt, p.kh = a->stride_kph, p.vp = a->stride_vpp, p.vt = a->stride_vpt, p.vh = a->stride_vph;
  p.ksp = a->stride_ksp, p.kst = a->stride_kst, p.ksh = a->stride_ksh, p.vsp = a->stride_vsp, p.vst = a->stride_vst, p.vsh = a->stride_vsh;
  p.s_table = a->stride_table, p.lse_h = a->lse_stride_h;
  p.scale_log2 = (float)(a->softmax_scale * 1.4426950408889634074);
  p.num_pages = (int32_t)a->num_pages, p.max_pages = a->max_pages;
  p.group = a->q_heads / a->kv_heads, p.head_dim = a->head_dim, p.page_tokens = a->page_tokens;
  DeviceGuard guard(device);
  SA_HIP_RETURN(guard.status());
  const dim3 grid(a->sequences, a->q_heads);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const bool bf16 = a->dtype == SA_DTYPE_BF16;
  if (a->pages_int8)
    bf16 ? decode_kernel<Bf16, true><<<grid, 64, 0, hs>>>(p) : decode_kernel<Fp16, true><<<grid, 64, 0, hs>>>(p);
  else
    bf16 ? decode_kernel<Bf16, false><<<grid, 64, 0, hs>>>(p) : decode_kernel<Fp16, false><<<grid, 64, 0, hs>>>(p);
  SA_HIP_RETURN(hipGetLastError());
  return 0;
} catch (const std::exception& error) {
  return sa::exception_status("sa_paged_decode", error);
}

}  // extern "C"
