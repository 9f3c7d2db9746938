// K and V rows quantised into e4m3 pages with one power-of-two scale per block of
// rows and K/V head.
//
//   scale of a block: the smallest 2^e, e >= -126, with |x| <= 448 2^e for the finite
//   elements written; code = e4m3(x 2^-e)
//
// A power of two costs e4m3 no precision (its values have an exponent of their
// own), and a scale that grows moves the codes of rows already there by whole
// binades: those are exact again unless they fall below 2^-6 of the scale, where
// e4m3's steps end.  So a block can take its rows one call at a time.
//
// Bytes bound: 16-bit rows read once, a byte per element written.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "sa_common.h"
#include "sa_types.h"

namespace sa {
namespace {

constexpr int kAppendWaves = 4;
// Workgroups over the blocks of a launch; every one looks at all sequences.
constexpr int64_t kMaxBlockGroups = 4096;
// Loads of a wave (a granule of a row per lane each) that it holds between the
// block's largest magnitude and its codes, the others it reads again; a block is on
// as many waves as make it no more, up to a workgroup's.  Time goes into the way
// from the lengths over the table to the rows and codes, so that waves count: 20,011
// tokens of 8 heads of 128 with a block per wave 34.5 us, on four waves 29.0, with six
// waves a SIMD instead of four 27.6, four loads held instead of eight 25.4; four heads
// of 256, then half of a block read again, 24.4 and 26.2.
constexpr int kHeldLoads = 4;

struct AppendParams {
  const uint16_t *k, *v;
  uint8_t *kp, *vp, *ks, *vs;
  const int32_t *table, *lengths, *cu;
  int64_t sk_t, sk_h, sv_t, sv_h, sp, st, sh, ssp, ssb, ssh, s_table, tokens;
  int32_t sequences, num_pages, room, kv_heads, head_dim, page_tokens, block_log2, lane_log2;
  int32_t unit_log2;  // log2 of the waves of a block, K/V head and one of K and V
};

// The new rows of a sequence: positions start .. end - 1, rows row0 .. of k and v.
struct NewRows {
  int64_t row0;
  int32_t start, end;
  __device__ inline int32_t blocks(int32_t log2) const { return end > start ? ((end - 1) >> log2) - (start >> log2) + 1 : 0; }
};

__device__ inline NewRows new_rows(const AppendParams& p, int32_t s) {
  int64_t from = s, to = s + 1;
  if (p.cu != nullptr) {
    from = p.cu[s], to = p.cu[s + 1];
    from = from < 0 ? 0 : from > p.tokens ? p.tokens : from;
    to = to < from ? from : to > p.tokens ? p.tokens : to;
  } else if (to > p.tokens) {
    to = from = p.tokens;
  }
  const int64_t length = p.lengths[s], first = length - (to - from);
  NewRows n;
  n.start = (int32_t)(first < 0 ? 0 : first > p.room ? p.room : first);
  n.end = (int32_t)(length < n.start ? n.start : length > p.room ? p.room : length);
  n.row0 = from + (n.start - first);
  return n;
}

// The E8M0 byte of the smallest scale of at least 2^-126 of which 448 reach x.
__device__ inline int32_t scale_byte(float x) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, x);
  const int32_t byte = (int32_t)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);  // 448 = 1.75 * 2^8
  return byte < 1 ? 1 : byte;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The halves of a dword that are infinite or NaN, as halves of ones.
template <typename T>
__device__ inline uint32_t not_finite(uint32_t w) {
  return ((w & T::kInfinity) == T::kInfinity ? 0xffffu : 0u) |
         ((w >> 16 & T::kInfinity) == T::kInfinity ? 0xffff0000u : 0u);
}

// A lane's largest magnitudes, as the bits of 16-bit floats (which are in their
// order); with kFinite of the finite ones.
template <bool kFinite, typename T>
__device__ inline u16x2 largest(u32x4 x, u16x2 top) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = x[i] & 0x7fff7fffu;
    if (kFinite) w &= ~not_finite<T>(w);
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w));
  }
  return top;
}

__device__ inline uint32_t over_wave(u16x2 x) {
  uint32_t top = x[0] > x[1] ? x[0] : x[1];
  for (int i = 1; i < 64; i <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, i));
  return top;
}

// Row `first` + step * i of this lane, or the last row (one of the same block, so
// that the largest magnitude is the same): a load under a condition would wait for
// the one before.
struct RowReader {
  const uint16_t* base;
  int64_t stride;
  int32_t first, step, count;
  __device__ inline u32x4 operator()(int i) const {
    return *reinterpret_cast<const u32x4*>(base + min(first + step * i, count - 1) * stride);
  }
};

// A unit is the rows of one block, one K/V head and one of K and V, on 2^unit_log2
// waves; a granule (8 elements) of a row is on each of 2^lane_log2 lanes.
//
// Measured (a copy that streams 2 GiB reaches 6.4 TB/s): 20,011 tokens of 8 heads of 128,
// K and V, 25 us, 4.8 TB/s; 56 heads 170 us, 5.1 TB/s; one token of each of 24
// sequences 3.8 us, all of it latency.
template <typename T>
__global__ __launch_bounds__(64 * kAppendWaves, 6) void append_blocks_kernel(const AppendParams p) {
  __shared__ int64_t sums[kAppendWaves];
  __shared__ int64_t found[2];
  __shared__ uint32_t tops[2][2 * kAppendWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Items are blocks that take rows, numbered sequence by sequence; with one row
  // each, sequences.
  int64_t begin, end, before;
  int s;
  if (p.cu == nullptr) {
    const int64_t share = (p.sequences + gridDim.y - 1) / gridDim.y;
    begin = before = blockIdx.y * share, end = min(begin + share, (int64_t)p.sequences);
    s = (int)begin;
    if (begin >= end) return;
  } else {
    const int run = (p.sequences + 64 * kAppendWaves - 1) / (64 * kAppendWaves);
    const int s_first = min(tid * run, p.sequences), s_last = min(s_first + run, p.sequences);
    int64_t own = 0;
    for (int x = s_first; x < s_last; ++x) own += new_rows(p, x).blocks(p.block_log2);
    int64_t upto = own;  // inclusive
    for (int i = 1; i < 64; i <<= 1) {
      const int64_t x = __shfl_up(upto, i);
      if (lane >= i) upto += x;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int64_t total = 0;
    for (int i = 0; i < kAppendWaves; ++i) {
      if (i < wave) upto += sums[i];
      total += sums[i];
    }
    const int64_t share = (total + gridDim.y - 1) / gridDim.y;
    begin = blockIdx.y * share, end = min(begin + share, total);
    if (begin >= upto - own && begin < upto) {
      int64_t ahead = upto - own;
      int x = s_first;
      for (; x < s_last; ++x) {
        const int64_t n = new_rows(p, x).blocks(p.block_log2);
        if (begin < ahead + n) break;
        ahead += n;
      }
      found[0] = x, found[1] = ahead;
    }
    __syncthreads();
    if (begin >= end) return;
    s = __builtin_amdgcn_readfirstlane((int)found[0]);
    before = found[1];
  }
  // Waves past the last unit take it along: the workgroup's waves meet at barriers.
  const int waves = 1 << p.unit_log2, part = wave & (waves - 1);
  const int wanted = blockIdx.x * (kAppendWaves >> p.unit_log2) + (wave >> p.unit_log2);
  const bool writes = wanted < 2 * p.kv_heads;
  const int unit = min(wanted, 2 * p.kv_heads - 1);
  const bool is_v = unit >= p.kv_heads;
  const int head = is_v ? unit - p.kv_heads : unit;
  const int g = lane & ((1 << p.lane_log2) - 1), per_load = 64 >> p.lane_log2;
  const int r = part * per_load + (lane >> p.lane_log2), step = waves * per_load;
  const bool live = 8 * g < p.head_dim;
  const uint16_t* rows = is_v ? p.v + head * p.sv_h : p.k + head * p.sk_h;
  const int64_t stride = is_v ? p.sv_t : p.sk_t;
  uint8_t* pages = (is_v ? p.vp : p.kp) + head * p.sh;
  uint8_t* scales = (is_v ? p.vs : p.ks) + head * p.ssh;
  NewRows n = new_rows(p, s);
  int turn = 0;
  for (int64_t at = begin; at < end; ++at) {
    if (p.cu == nullptr) {
      n = new_rows(p, (int)at), s = (int)at, before = at;
      if (n.end <= n.start) continue;
    } else {
      while (at >= before + n.blocks(p.block_log2)) before += n.blocks(p.block_log2), n = new_rows(p, ++s);
    }
    const int32_t block = (n.start >> p.block_log2) + (int32_t)(at - before), low = block << p.block_log2;
    const int32_t first = max(n.start, low), last = min(n.end, low + (1 << p.block_log2));
    const int32_t page = low / p.page_tokens, in_page = low - page * p.page_tokens;
    const int32_t id = p.table[s * p.s_table + page];
    const RowReader read{rows + (n.row0 + (first - n.start)) * stride + (live ? 8 * g : 0), stride, r, step, last - first};
    const int32_t loads = (last - first + step - 1) / step;

    u32x4 held[kHeldLoads];
#pragma unroll
    for (int i = 0; i < kHeldLoads; i += 4) {
      if (i < loads) {
#pragma unroll
        for (int x = i; x < i + 4; ++x) held[x] = read(x);
      } else {
#pragma unroll
        for (int x = i; x < i + 4; ++x) held[x] = u32x4{0, 0, 0, 0};
      }
    }
    if ((uint32_t)id >= (uint32_t)p.num_pages) continue;  // of all waves alike
    uint8_t* scale = scales + id * p.ssp + (in_page >> p.block_log2) * p.ssb;
    const int32_t old = *scale;
    // What is not finite is rare: only where it comes up is it left out.
    const auto top_of = [&](auto finite) {
      u16x2 x = {0, 0};
#pragma unroll
      for (int i = 0; i < kHeldLoads; ++i) x = largest<decltype(finite)::value, T>(held[i], x);
      for (int i = kHeldLoads; i < loads; ++i) x = largest<decltype(finite)::value, T>(read(i), x);
      return over_wave(x);
    };
    uint32_t any = top_of(std::false_type()), top = any;
    if (any >= T::kInfinity) top = top_of(std::true_type());
    if (waves > 1) {
      // A place is written again two barriers later.
      if (lane == 0) tops[turn][2 * wave] = any, tops[turn][2 * wave + 1] = top;
      __syncthreads();
      for (int i = wave - part; i < wave - part + waves; ++i)
        any = max(any, tops[turn][2 * i]), top = max(top, tops[turn][2 * i + 1]);
      turn ^= 1;
    }
    int32_t byte = scale_byte(T::lo(top));
    if (first > low) byte = max(byte, old);
    const float power = e8m0_value(byte);

    uint8_t* to = pages + id * p.sp + in_page * p.st + 8 * g;
    if (first > low && byte != old && live && writes) {
      // Rows of earlier calls, in the scale that is theirs now.
      const int32_t shift = old - byte;
      for (int32_t x = r; x < first - low; x += step) {
        u32x2* row = reinterpret_cast<u32x2*>(to + x * p.st);
        u32x2 c = *row;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x2 a = e4m3_floats<false>(c[i]), b = e4m3_floats<true>(c[i]);
          c[i] = e4m3_pack(__builtin_ldexpf(a[0], shift), __builtin_ldexpf(a[1], shift), __builtin_ldexpf(b[0], shift),
                           __builtin_ldexpf(b[1], shift));
        }
        *row = c;
      }
    }
    to += (first - low + r) * p.st;
    const auto store = [&](int i, u32x4 x) __attribute__((always_inline)) {
      u32x2 codes = {T::to_e4m3(x[0], x[1], power), T::to_e4m3(x[2], x[3], power)};
      if (any >= T::kInfinity) {
        // Infinities are NaN too.
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t off = not_finite<T>(x[w]), bytes = (off & 0x7f) | (off >> 16 & 0x7f) << 8;
          codes[w / 2] |= bytes << (16 * (w & 1));
        }
      }
      if (live && writes && r + step * i < last - first) *reinterpret_cast<u32x2*>(to + step * i * p.st) = codes;
    };
#pragma unroll
    for (int i = 0; i < kHeldLoads; ++i)
      if (i < loads) store(i, held[i]);
    for (int i = kHeldLoads; i < loads; ++i) store(i, read(i));
    if (lane == 0 && part == 0 && writes) *scale = (uint8_t)byte;
  }
}

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int32_t invalid(const char* what) {
  set_error("sa_append_kv_blocks: %s", what);
  return SA_ERR_INVALID_ARGUMENT;
}

}  // namespace
}  // namespace sa

extern "C" int32_t sa_append_kv_blocks(const sa_append_blocks_args* a, int32_t device, void* stream) try {
  using namespace sa;
  clear_error();
  if (a == nullptr) return invalid("null arguments");
  if (a->dtype != SA_DTYPE_BF16 && a->dtype != SA_DTYPE_FP16) {
    set_error("sa_append_kv_blocks: unsupported dtype code %d", a->dtype);
    return SA_ERR_UNSUPPORTED_DTYPE;
  }
  if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 8) {
    set_error("sa_append_kv_blocks: head_dim must be a multiple of 8 in [16, 256], got %d", a->head_dim);
    return SA_ERR_UNSUPPORTED_HEAD_DIM;
  }
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->kv_heads < 1 || a->kv_heads > (1 << 16) || a->sequences < 0 ||
      a->sequences > (1 << 30))
    return invalid("tokens, heads or sequences out of range");
  if (a->page_tokens < 1 || a->page_tokens > SA_MAX_PAGE_TOKENS || a->num_pages < 0 || a->max_pages < 0 ||
      a->num_pages > INT32_MAX / a->page_tokens || a->max_pages > INT32_MAX / a->page_tokens)
    return invalid("page_tokens must be at most 2^20 and pages * page_tokens below 2^31");
  AppendParams p{};
  p.block_log2 = block_log2(a->block_tokens, a->page_tokens);
  if (p.block_log2 < 0) return invalid("block_tokens must be a power of two from 16 on that divides page_tokens");
  if (a->cu_tokens == nullptr && a->tokens != a->sequences) return invalid("one row per sequence without cu_tokens");
  if (a->tokens == 0 || a->sequences == 0 || a->max_pages == 0) return 0;
  const int64_t strides[] = {a->stride_kt, a->stride_kh, a->stride_vt, a->stride_vh, a->stride_pp, a->stride_pt, a->stride_ph};
  for (int64_t s : strides)
    if (s % 8) return invalid("strides must be multiples of 8 elements");
  if (a->k == nullptr || a->v == nullptr || a->k_pages == nullptr || a->v_pages == nullptr || a->k_scales == nullptr ||
      a->v_scales == nullptr || a->page_table == nullptr || a->lengths == nullptr || !aligned(a->k, 16) ||
      !aligned(a->v, 16) || !aligned(a->k_pages, 8) || !aligned(a->v_pages, 8) || !aligned(a->page_table, 4) ||
      !aligned(a->lengths, 4) || !aligned(a->cu_tokens, 4))
    return invalid("an operand is missing or not aligned");
  p.k = static_cast<const uint16_t*>(a->k), p.v = static_cast<const uint16_t*>(a->v);
  p.kp = static_cast<uint8_t*>(a->k_pages), p.vp = static_cast<uint8_t*>(a->v_pages);
  p.ks = static_cast<uint8_t*>(a->k_scales), p.vs = static_cast<uint8_t*>(a->v_scales);
  p.table = a->page_table, p.lengths = a->lengths, p.cu = a->cu_tokens;
  p.sk_t = a->stride_kt, p.sk_h = a->stride_kh, p.sv_t = a->stride_vt, p.sv_h = a->stride_vh;
  p.sp = a->stride_pp, p.st = a->stride_pt, p.sh = a->stride_ph;
  p.ssp = a->stride_sp, p.ssb = a->stride_sb, p.ssh = a->stride_sh;
  p.s_table = a->stride_table, p.tokens = a->tokens;
  p.sequences = a->sequences, p.num_pages = (int32_t)a->num_pages, p.room = a->max_pages * a->page_tokens;
  p.kv_heads = a->kv_heads, p.head_dim = a->head_dim, p.page_tokens = a->page_tokens;
  while ((8 << p.lane_log2) < p.head_dim) ++p.lane_log2;
  DeviceGuard guard(device);
  SA_HIP_RETURN(guard.status());
  // A sequence's rows are in at most two blocks more than they fill, and in no
  // more than there are rows.
  const int64_t blocks = std::min(a->tokens, (a->tokens >> p.block_log2) + 2 * (int64_t)a->sequences);
  const int64_t block_loads = (((int64_t)1 << p.block_log2) << p.lane_log2) / 64;  // of a wave alone
  while ((1 << p.unit_log2) < kAppendWaves && (kHeldLoads << p.unit_log2) < block_loads && a->cu_tokens != nullptr) ++p.unit_log2;
  const int64_t units = kAppendWaves >> p.unit_log2;  // of a workgroup
  // Neighbouring workgroups have the heads of the same rows.
  const dim3 grid((uint32_t)((2 * a->kv_heads + units - 1) / units), (uint32_t)std::min(blocks, kMaxBlockGroups));
  hipStream_t hs = static_cast<hipStream_t>(stream);
  if (a->dtype == SA_DTYPE_BF16)
    append_blocks_kernel<Bf16><<<grid, 64 * kAppendWaves, 0, hs>>>(p);
  else
    append_blocks_kernel<Fp16><<<grid, 64 * kAppendWaves, 0, hs>>>(p);
  SA_HIP_RETURN(hipGetLastError());
  return 0;
} catch (const std::exception& error) {
  return sa::exception_status("sa_append_kv_blocks", error);
}
