// The paged key/value cache as its kernels see it: the order of its elements, its 8-bit code and the
// rows of a call. Shared by the append, the read and the attention.
//
// A page holds `page` tokens of `heads` heads in units of 16 tokens x 64 dimensions, a unit being what
// one step of v_mfma_f32_16x16x32 takes as its A operand: lane l of a wavefront reads 16 consecutive
// bytes at 16 l and has its operand registers, for keys (rows = tokens, K = dimensions) and for values
// (rows = dimensions, K = tokens) alike. With n = token % 16, e = dimension % 64, per unit:
//   e4m3 keys    byte  (e / 16) * 256 + n * 16 + e % 16
//   e4m3 values  byte  (n / 4) * 256 + (e / 4) * 16 + (e % 4) * 4 + n % 4
//   16-bit keys   elem  (e / 8 % 2) * 512 + (e / 16) * 128 + n * 8 + e % 8
//   16-bit values elem  (e / 2 % 2) * 512 + (n / 4) * 128 + (e / 4) * 8 + (e % 2) * 4 + n % 4
#pragma once

#include "tile.h"

namespace plm {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct KvCache {
  char* k;
  char* v;
  float* k_scale;  // [pages, heads], powers of two; null for 16-bit caches
  float* v_scale;
  int64_t pages;
  int heads, page, page_shift, dim, chunks;  // chunks of 64 dimensions
};

// Rows of one call: sequence b has rows [starts[b], starts[b + 1]) of the packed row tensors (every
// sequence `max_rows` of them where starts is null) after a context of lengths[b] tokens.
struct KvRows {
  const int32_t* table;  // [seqs, width], stride table_stride
  const int64_t* lengths;
  const int64_t* starts;
  int64_t table_stride;
  int total, seqs, max_rows, width;
};

// What a call's numbers on the device say about one sequence, held to what its buffers hold: numbers
// out of range shorten a sequence, they never move an access out of a buffer.
struct KvSeq {
  int start, rows, context;
};

__device__ __forceinline__ KvSeq kv_seq(const KvRows& r, int b, int page_shift) {
  KvSeq s;
  int64_t first = static_cast<int64_t>(b) * r.max_rows, rows = r.max_rows;
  if (r.starts != nullptr) {
    first = r.starts[b];
    rows = r.starts[b + 1] - first;
  }
  const int64_t most = static_cast<int64_t>(r.width) << page_shift;
  const int64_t length = r.lengths[b];
  s.start = static_cast<int>(min(max(first, int64_t{0}), static_cast<int64_t>(r.total)));
  s.rows = static_cast<int>(min(max(rows, int64_t{0}), static_cast<int64_t>(min(r.max_rows, r.total - s.start))));
  s.context = static_cast<int>(min(max(length, int64_t{0}), most));
  return s;
}

// Rows [first, end) between sequence b's and the next one's (b = -1: before the first; `seq`: kv_seq of b), which no sequence
// holds: gaps of row_starts, rows past max_rows, rows past the last start. Results have zeros there.
struct KvGap {
  int first, end;
};

__device__ __forceinline__ KvGap kv_gap(const KvRows& r, int b, const KvSeq& seq) {
  if (r.starts == nullptr) return {0, 0};
  const int64_t next = b + 1 < r.seqs ? min(max(r.starts[b + 1], int64_t{0}), static_cast<int64_t>(r.total)) : r.total;
  return {b < 0 ? 0 : seq.start + seq.rows, static_cast<int>(next)};
}

// Zeros in all gaps' rows of `out` ([total, 8 row8] of 16 bits): workgroup `index` of the `count` that a launch has for it.
__device__ __forceinline__ void kv_clear(const KvRows& r, int page_shift, uint16_t* out, int64_t row8, int index, int count) {
  const int lane = threadIdx.x & 63;
  for (int base = -1; base < r.seqs; base += 64) {
    const int b = base + lane;
    KvGap gap = {0, 0};
    if (b < r.seqs) gap = kv_gap(r, b, b < 0 ? KvSeq{0, 0, 0} : kv_seq(r, b, page_shift));
    for (uint64_t some = __ballot(gap.end > gap.first); some != 0; some &= some - 1) {
      const int at = __builtin_ctzll(some);
      const int64_t end = __builtin_amdgcn_readlane(gap.end, at) * row8;
      for (int64_t x = __builtin_amdgcn_readlane(gap.first, at) * row8 + static_cast<int64_t>(index) * blockDim.x + threadIdx.x; x < end;
           x += static_cast<int64_t>(count) * blockDim.x)
        reinterpret_cast<u32x4*>(out)[x] = u32x4{0u, 0u, 0u, 0u};
    }
  }
}

// How many workgroups that is: none without row_starts, whose rows have no gaps, else one per 64 KiB of `out` up to 64. What
// the others do is not held up by it. (Done by the workgroups that turn out to have no work it cost every call 4 us of 242 for
// 4096 rows after 4096 tokens, by the kernel's registers.)
inline int64_t kv_clear_groups(const KvRows& r, int64_t row8) {
  const int64_t pieces = r.total * row8 / 4096;
  return r.starts == nullptr ? 0 : pieces < 1 ? 1 : pieces > 64 ? 64 : pieces;
}

// Two e4m3 codes of a word as the model's type, times the power of two `scale` (exact, but for fp16
// results below 2^-14, which keep fp16's absolute step).
template <int DT>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t word, float scale, bool high) {
  if constexpr (DT == DT_BF16) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false));
  } else {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, false));
  }
}

template <int DT>
__device__ __forceinline__ u32x4 fp8_eight(uint32_t lo, uint32_t hi, float scale) {
  return u32x4{fp8_pair<DT>(lo, scale, false), fp8_pair<DT>(lo, scale, true), fp8_pair<DT>(hi, scale, false),
               fp8_pair<DT>(hi, scale, true)};
}

// e4m3 code of x, rounded to nearest even; |x| <= 448 but for what is not finite, which becomes NaN.
__device__ __forceinline__ uint32_t fp8_word(float a, float b, float c, float d) {
  constexpr float top = 448.0f;
  const float nan = __builtin_nanf("");
  a = fabsf(a) <= top ? a : nan;
  b = fabsf(b) <= top ? b : nan;
  c = fabsf(c) <= top ? c : nan;
  d = fabsf(d) <= top ? d : nan;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return static_cast<uint32_t>(w);
}

__device__ __forceinline__ float fp8_value(uint32_t word, int byte) {
  switch (byte) {
    case 0: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 0);
    case 1: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 1);
    case 2: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 2);
    default: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 3);
  }
}

// The least power of two s with amax <= 448 s, at least 2^-64: with amax = m 2^e, m in [1, 2),
// 448 = 1.75 * 2^8 puts it at 2^(e - 8) up to m = 1.75 and at 2^(e - 7) above.
__device__ __forceinline__ float fp8_scale_of(float amax) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  int e = static_cast<int>(bits >> 23) - 127 - 8;
  if ((bits & 0x7fffffu) > 0x600000u) e += 1;
  e = max(e, -64);
  return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23);
}

// The kernels' view of a cache; false where the handle is not one.
inline bool kv_cache_of(const plm_kv_cache* h, KvCache& c) {
  if (h == nullptr || h->k == nullptr || h->v == nullptr || h->pages < 1 || h->pages >= (int64_t{1} << 31)) return false;
  if (h->kv_heads < 1 || h->kv_heads > 1024 || h->head_dim < 8 || h->head_dim > 256 || h->head_dim % 8 != 0) return false;
  if (h->page != 16 && h->page != 32 && h->page != 64 && h->page != 128) return false;
  if (h->type != PLM_CACHE_BF16 && h->type != PLM_CACHE_F16 && h->type != PLM_CACHE_E4M3) return false;
  if (h->type == PLM_CACHE_E4M3 && (h->k_scale == nullptr || h->v_scale == nullptr)) return false;
  c.k = static_cast<char*>(h->k);
  c.v = static_cast<char*>(h->v);
  c.k_scale = h->k_scale;
  c.v_scale = h->v_scale;
  c.pages = h->pages;
  c.heads = h->kv_heads;
  c.page = h->page;
  c.page_shift = __builtin_ctz(static_cast<unsigned>(h->page));
  c.dim = h->head_dim;
  c.chunks = (h->head_dim + 63) / 64;
  return true;
}

inline bool kv_type_fits(const plm_kv_cache* h, int64_t dtype) {
  if (dtype != PLM_BF16 && dtype != PLM_F16) return false;
  return h->type == PLM_CACHE_E4M3 || h->type == (dtype == PLM_BF16 ? PLM_CACHE_BF16 : PLM_CACHE_F16);
}

// A call's rows; false where its numbers do not go together.
inline bool kv_rows_of(const KvCache& c, const plm_kv_rows& h, KvRows& r) {
  if (h.total < 1 || h.total >= (1 << 28) || h.seqs < 1 || h.seqs > (1 << 20) || h.max_rows < 1 || h.max_rows > h.total)
    return false;
  if (h.row_starts == nullptr && h.seqs * h.max_rows != h.total) return false;
  if (h.table == nullptr || h.lengths == nullptr) return false;
  if (h.table_width < 1 || h.table_width > ((int64_t{1} << 29) >> c.page_shift) || h.table_stride < h.table_width) return false;
  r = {h.table, h.lengths, h.row_starts, h.table_stride, static_cast<int>(h.total), static_cast<int>(h.seqs),
       static_cast<int>(h.max_rows), static_cast<int>(h.table_width)};
  return true;
}

}  // namespace plm
