// The paged cache's append (with the position rotation of keys and queries) and its read, declared in
// include/plm_amd.h.
//
// Rotation: dimensions (a, b) of a pair become (a cos - b sin, b cos + a sin); a pair is (i, i + rotary / 2), or (2 i,
// 2 i + 1) side by side. What becomes the model's type is computed in fp32 and rounded from there, off by half a step and
// 2^-16 of one at most. An 8-bit code has 2^20 fp32 values to a step, so of a million keys' values about one would come out
// on the other side of a border: what is that close is computed in fp64 and rounded once.
//
// 8-bit pages: codes times one power of two per (page, head). Appending rows needs their largest
// magnitude first: a workgroup owns one (page, head) of the keys or of the values, keeps its new rows
// in registers while it finds it, and rounds the rows that stay again only where the scale grows.
#include <hip/hip_runtime.h>

#include "kv_cache.h"
#include "plm_amd.h"

namespace plm {

struct AppendArgs {
  KvCache cache;
  KvRows rows;
  const uint16_t* q;
  const uint16_t* new_k;
  const uint16_t* new_v;
  uint16_t* q_out;  // contiguous [total, heads, dim]
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  const int64_t* positions;
  const float* rope;  // [rope_rows, rotary]: cosines, then sines
  int64_t rope_rows;
  int heads, rotary, side_by_side, page_slots, parts, kv_blocks, q_blocks;
};

// a c + b s in fp32. `close` gets the bit where that is within its error, 2^-23 of the larger term at most, of a place where
// 8-bit codes may part: at most four bits of mantissa, so 19 zeros at the end. `near` is twice that error, kNear, or less than
// nothing for a cosine of 1 and a sine of 0, which are exact and leave about one value in eight on a border. Zeros are too.
constexpr float kNear = 0x1p-22f;
__device__ __forceinline__ float turn_one(float a, float c, float b, float s, float near, int bit, uint32_t& close) {
  const float part = b * s, sum = fmaf(a, c, part);
  const float border = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, sum) + 0x40000u) & 0xfff80000u);
  close |= fabsf(sum - border) < near * fmaxf(fabsf(part), fabsf(sum)) ? 1u << bit : 0u;
  return sum;
}

// `near` of a group of pairs: of all of them at once, which the positions that turn nothing have alike.
template <int N>
__device__ __forceinline__ float near_of(const float (&c)[N], const float (&s)[N]) {
  float turned = fabsf(s[0]), least = c[0], most = c[0];
#pragma unroll
  for (int k = 1; k < N; ++k) {
    turned = fmaxf(turned, fabsf(s[k]));
    least = fminf(least, c[k]);
    most = fmaxf(most, c[k]);
  }
  return turned == 0.0f && least == 1.0f && most == 1.0f ? -1.0f : kNear;
}

// Dimension e of a row, turned in fp64, which holds the products exactly, to the fp32 value on either side whose last bit
// is set, if it is not one itself: rounded again to fewer bits that is as if rounded once.
template <int DT>
__device__ __forceinline__ float turned_exact(const uint16_t* x, int e, const float* turn, int rotary, bool side_by_side) {
  const int half = rotary >> 1;
  const bool low = side_by_side ? (e & 1) == 0 : e < half;
  const int at = side_by_side ? e >> 1 : low ? e : e - half;
  const double own = from_bits16<DT>(x[e]), other = from_bits16<DT>(x[side_by_side ? e ^ 1 : low ? e + half : e - half]);
  const double part = other * static_cast<double>(turn[half + at]);
  const double sum = fma(own, static_cast<double>(turn[at]), low ? -part : part);
  const float near = static_cast<float>(sum);
  const double off = sum - static_cast<double>(near);
  uint32_t bits = __builtin_bit_cast(uint32_t, near);
  if (fabs(off) > 0.0 && fabs(off) < __builtin_inf() && (bits & 1u) == 0u)
    bits += (off < 0.0) == ((bits >> 31) != 0u) ? 1u : ~0u;
  return __builtin_bit_cast(float, bits);
}

// Dimensions [e0, e0 + 8) of a row, as fp32, turned. `turn` is the position's row of the rotation table,
// null where the table does not hold the position: what it would have turned is NaN.
template <int DT>
__device__ __forceinline__ void rotated8(const uint16_t* x, int e0, const float* turn, int rotary, bool side_by_side,
                                         uint32_t& close, float (&out)[8]) {
  const u32x4 own = *reinterpret_cast<const u32x4*>(x + e0);
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = from_bits16<DT>(static_cast<uint16_t>(own[i / 2] >> (16 * (i & 1))));
  if (e0 >= rotary) return;
  const int half = rotary >> 1;
  if (turn == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e0 + i < rotary) out[i] = __builtin_nanf("");
  } else if (side_by_side && (half & 3) == 0 && e0 + 8 <= rotary) {
    float c[4], s[4];
    *reinterpret_cast<f32x4*>(c) = *reinterpret_cast<const f32x4*>(turn + (e0 >> 1));
    *reinterpret_cast<f32x4*>(s) = *reinterpret_cast<const f32x4*>(turn + half + (e0 >> 1));
    const float near = near_of(c, s);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = out[i], b = out[i + 1];
      out[i] = turn_one(a, c[i / 2], -b, s[i / 2], near, i, close);
      out[i + 1] = turn_one(b, c[i / 2], a, s[i / 2], near, i + 1, close);
    }
  } else if (side_by_side) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (e0 + i < rotary) {
        const float c[1] = {turn[(e0 + i) >> 1]}, s[1] = {turn[half + ((e0 + i) >> 1)]}, near = near_of(c, s);
        const float a = out[i], b = out[i + 1];
        out[i] = turn_one(a, c[0], -b, s[0], near, i, close);
        out[i + 1] = turn_one(b, c[0], a, s[0], near, i + 1, close);
      }
    }
  } else if ((half & 7) == 0) {
    // The partners are eight consecutive dimensions too.
    const bool low = e0 < half;
    const u32x4 other = *reinterpret_cast<const u32x4*>(x + (low ? e0 + half : e0 - half));
    const float* at = turn + (low ? e0 : e0 - half);
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<f32x4*>(c + i) = *reinterpret_cast<const f32x4*>(at + i);
      *reinterpret_cast<f32x4*>(s + i) = *reinterpret_cast<const f32x4*>(at + half + i);
    }
    const float near = near_of(c, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = from_bits16<DT>(static_cast<uint16_t>(other[i / 2] >> (16 * (i & 1))));
      out[i] = turn_one(out[i], c[i], low ? -o : o, s[i], near, i, close);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = e0 + i;
      if (e < rotary) {
        const bool low = e < half;
        const float o = from_bits16<DT>(x[low ? e + half : e - half]);
        const int at = low ? e : e - half;
        const float c[1] = {turn[at]}, s[1] = {turn[half + at]};
        out[i] = turn_one(out[i], c[0], low ? -o : o, s[0], near_of(c, s), i, close);
      }
    }
  }
}

__device__ __forceinline__ const float* turn_of(const AppendArgs& a, int row, int slot, bool& none) {
  none = a.rope == nullptr;
  if (none) return nullptr;
  const int64_t at = a.positions != nullptr ? a.positions[row] : slot;
  return at >= 0 && at < a.rope_rows ? a.rope + at * a.rotary : nullptr;
}

template <int DT>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = to_bits16<DT>(x[2 * i]) | (static_cast<uint32_t>(to_bits16<DT>(x[2 * i + 1])) << 16);
  return o;
}

// Eight pairs, partners in `lo` and `hi`, turned.
template <int DT>
__device__ __forceinline__ void turned8(u32x4 lo, u32x4 hi, const float (&c)[8], const float (&s)[8], uint32_t& close, float* x,
                                        float* y) {
  const float near = near_of(c, s);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float p = from_bits16<DT>(static_cast<uint16_t>(lo[k / 2] >> (16 * (k & 1))));
    const float q = from_bits16<DT>(static_cast<uint16_t>(hi[k / 2] >> (16 * (k & 1))));
    x[k] = turn_one(p, c[k], -q, s[k], near, k, close);
    y[k] = turn_one(q, c[k], p, s[k], near, 8 + k, close);
  }
}

// Queries: a thread has one place of a row and head, both partners' eight dimensions where a half is whole groups of 8.
// (Four heads per thread, which read the cosines and sines once, measured the same over four prompts of up to 2048 rows
// of 16 heads of 128, 22 us with the pages read back, and slower over three of 333 rows of 32 heads of 80, 20 against 19:
// they come from L2.)
template <int DT>
__device__ __forceinline__ void append_queries(const AppendArgs& a, int block) {
  const int b = block / a.q_blocks;
  const KvSeq seq = kv_seq(a.rows, b, a.cache.page_shift);
  const int dim = a.cache.dim, rotary = a.rope != nullptr ? a.rotary : 0, half = rotary >> 1;
  const bool paired = rotary > 0 && !a.side_by_side && (half & 7) == 0;
  const int places = paired ? (dim - half) >> 3 : dim >> 3, per_row = places * a.heads;
  const int at = (block - b * a.q_blocks) * 256 + static_cast<int>(threadIdx.x), i = at / per_row;
  if (i >= seq.rows) return;
  const int rest = at - i * per_row, head = rest / places, place = rest - head * places;
  const int64_t row = seq.start + i;
  bool none;
  const float* turn = turn_of(a, static_cast<int>(row), seq.context + i, none);
  const uint16_t* from = a.q + row * a.q_row + head * a.q_head;
  uint16_t* to = a.q_out + (row * a.heads + head) * dim;
  const bool both = paired && place < (half >> 3);
  uint32_t close = 0;  // of no account: queries are rounded to the model's type
  if (both && turn != nullptr) {
    const int e = place << 3;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(from + e), hi = *reinterpret_cast<const u32x4*>(from + e + half);
    float c[8], s[8], x[8], y[8];
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      *reinterpret_cast<f32x4*>(c + k) = *reinterpret_cast<const f32x4*>(turn + e + k);
      *reinterpret_cast<f32x4*>(s + k) = *reinterpret_cast<const f32x4*>(turn + half + e + k);
    }
    turned8<DT>(lo, hi, c, s, close, x, y);
    *reinterpret_cast<u32x4*>(to + e) = pack8<DT>(x);
    *reinterpret_cast<u32x4*>(to + e + half) = pack8<DT>(y);
    return;
  }
  // Everything else eight dimensions at a time: pairs side by side, halves of other sizes, what is not turned, both
  // partners of a position that the table does not hold.
#pragma unroll 1
  for (int k = 0; k < (both ? 2 : 1); ++k) {
    const int e = paired && !both ? (place << 3) + half : (place << 3) + k * half;
    float x[8];
    rotated8<DT>(from, e, turn, rotary, a.side_by_side != 0, close, x);
    *reinterpret_cast<u32x4*>(to + e) = pack8<DT>(x);
  }
}

// A thread's 16 values of the workgroup's page. Values: 4 dimensions (i / 4, from e[0]) of 4 tokens (i % 4), one 16-byte
// word in 8 bits and two, 1 KiB apart, in 16. Keys: dimensions [e[0], e[0] + 8) and [e[1], e[1] + 8) of one token, the
// second maybe past the head's end; where halves are whole groups of 8 the two are partners, so that each is read once
// and the cosines and sines serve both.
struct PageUnit {
  int token;     // the first token, in the page
  int e[2];
  int64_t at[2]; // bytes from the (page, head)'s start
};

__device__ __forceinline__ bool paired_halves(const AppendArgs& a) {
  return a.rope != nullptr && !a.side_by_side && (a.rotary & 15) == 0;
}

template <bool VALUES, bool E8>
__device__ __forceinline__ PageUnit page_unit(const AppendArgs& a, int x) {
  const KvCache& c = a.cache;
  PageUnit p;
  constexpr int bytes = E8 ? 1024 : 2048;  // of a unit of 16 tokens x 64 dimensions
  if constexpr (VALUES) {
    const int per = c.dim >> 2;
    p.token = x / per;
    p.e[0] = p.e[1] = (x - p.token * per) << 2;
    p.token <<= 2;
    p.at[0] = p.at[1] = ((p.token >> 4) * c.chunks + (p.e[0] >> 6)) * bytes + ((p.token & 15) >> 2) * 256 + ((p.e[0] & 63) >> 2) * 16;
  } else {
    const int per = (c.dim + 15) >> 4;
    p.token = x / per;
    const int place = x - p.token * per, pairs = paired_halves(a) ? a.rotary >> 4 : 0;
    p.e[0] = place < pairs ? place << 3 : place << 4;
    p.e[1] = place < pairs ? p.e[0] + (a.rotary >> 1) : p.e[0] + 8;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = p.e[k];
      p.at[k] = ((p.token >> 4) * c.chunks + (e >> 6)) * bytes + ((e & 63) >> 4) * 256 + (p.token & 15) * 16 +
                (E8 ? e & 8 : (e & 8) * 128);
    }
  }
  return p;
}

// The unit's new values in fp32, zero where a token is not new. Bit i of `close`: see turn_one.
template <int DT, bool VALUES>
__device__ __forceinline__ void new_values(const AppendArgs& a, const KvSeq& seq, const PageUnit& p, int base, int head,
                                           float (&x)[16], uint32_t& close) {
  const int end = seq.context + seq.rows;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.0f;
  if constexpr (VALUES) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int slot = base + p.token + n;
      if (slot >= seq.context && slot < end) {
        const int64_t row = seq.start + (slot - seq.context);
        const u32x2 w = *reinterpret_cast<const u32x2*>(a.new_v + row * a.v_row + head * a.v_head + p.e[0]);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * j + n] = from_bits16<DT>(static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1))));
      }
    }
  } else {
    const int slot = base + p.token;
    if (slot < seq.context || slot >= end) return;
    const int row = seq.start + (slot - seq.context);
    bool none;
    const float* turn = turn_of(a, row, slot, none);
    const uint16_t* from = a.new_k + static_cast<int64_t>(row) * a.k_row + head * a.k_head;
    const int rotary = none ? 0 : a.rotary;
    if (turn != nullptr && paired_halves(a) && p.e[0] < (rotary >> 1)) {
      const u32x4 lo = *reinterpret_cast<const u32x4*>(from + p.e[0]), hi = *reinterpret_cast<const u32x4*>(from + p.e[1]);
      float c[8], s[8];
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        *reinterpret_cast<f32x4*>(c + k) = *reinterpret_cast<const f32x4*>(turn + p.e[0] + k);
        *reinterpret_cast<f32x4*>(s + k) = *reinterpret_cast<const f32x4*>(turn + p.e[1] + k);
      }
      turned8<DT>(lo, hi, c, s, close, x, x + 8);
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (p.e[k] < a.cache.dim) {
          float half[8];
          uint32_t of_half = 0;
          rotated8<DT>(from, p.e[k], turn, rotary, a.side_by_side != 0, of_half, half);
          close |= of_half << (8 * k);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[8 * k + i] = half[i];
        }
    }
  }
}

// Element i of the unit's new keys, one that turns, exactly (turned_exact).
template <int DT>
__device__ __forceinline__ float exact_value(const AppendArgs& a, const KvSeq& seq, const PageUnit& p, int base, int head, int i) {
  const int slot = base + p.token, row = seq.start + (slot - seq.context);
  bool none;
  const float* turn = turn_of(a, row, slot, none);
  const uint16_t* from = a.new_k + static_cast<int64_t>(row) * a.k_row + head * a.k_head;
  return turned_exact<DT>(from, (i < 8 ? p.e[0] : p.e[1]) + (i & 7), turn, a.rotary, a.side_by_side != 0);
}

// Rows of one page of one head into an 8-bit cache. UPT units of 16 values per thread.
template <int DT, bool VALUES, int UPT>
__device__ __forceinline__ void append_page_fp8(const AppendArgs& a, const KvSeq& seq, int64_t id, int base, int head,
                                                float* red) {
  const KvCache& c = a.cache;
  const int count = VALUES ? (c.page >> 2) * (c.dim >> 2) : c.page * ((c.dim + 15) >> 4);
  const int end = seq.context + seq.rows;
  float* held = (VALUES ? c.v_scale : c.k_scale) + id * c.heads + head;
  const bool stays = base < seq.context;  // the page holds rows from before
  const float before = stays ? *held : 0.0f;
  float x[UPT][16];
  PageUnit p[UPT];
  uint64_t close[2] = {0, 0};
  float amax = 0.0f;
#pragma unroll
  for (int u = 0; u < UPT; ++u) {
    p[u] = page_unit<VALUES, true>(a, min(static_cast<int>(threadIdx.x) + u * 256, count - 1));
    uint32_t bits = 0;
    new_values<DT, VALUES>(a, seq, p[u], base, head, x[u], bits);
    close[u / 4] |= static_cast<uint64_t>(bits) << (16 * (u % 4));
  }
  // About one turned value in 2^16 is that close: one at a time, from memory. (All keys in fp64 from the start: prompts 25.3
  // us for 22.9, single tokens 9.8 for 9.5; without any of it 22.1 and 8.9. 2048 rows of 4 heads of 256 in pages of 128 take
  // 18 us, and 17 if they are zeros or do not turn; with those taken for close 221 and 71.)
  if constexpr (!VALUES) {
    while ((close[0] | close[1]) != 0) {
      const int word = close[0] != 0 ? 0 : 1, i = 64 * word + __builtin_ctzll(word == 0 ? close[0] : close[1]);
      if (word == 0) close[0] &= close[0] - 1;
      else close[1] &= close[1] - 1;
      const PageUnit of = page_unit<false, true>(a, min(static_cast<int>(threadIdx.x) + (i >> 4) * 256, count - 1));
      const float y = exact_value<DT>(a, seq, of, base, head, i & 15);
#pragma unroll
      for (int u = 0; u < UPT; ++u)
#pragma unroll
        for (int k = 0; k < 16; ++k) x[u][k] = 16 * u + k == i ? y : x[u][k];
    }
  }
#pragma unroll
  for (int u = 0; u < UPT; ++u) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float m = fabsf(x[u][i]);
      amax = m < __builtin_inff() ? fmaxf(amax, m) : amax;  // what is not finite has no part in the scale
    }
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float wanted = fp8_scale_of(amax);
  const float scale = stays ? fmaxf(before, wanted) : wanted;
  const float inverse = 1.0f / scale;
  const bool again = stays && scale > before;
  const float ratio = before * inverse;  // a power of two, at most 1
  char* page = (VALUES ? c.v : c.k) + (id * c.heads + head) * (static_cast<int64_t>(c.page) * c.chunks * 64);
#pragma unroll
  for (int u = 0; u < UPT; ++u) {
    if (static_cast<int>(threadIdx.x) + u * 256 >= count) continue;
    const int first = base + p[u].token, last = first + (VALUES ? 4 : 1);  // slots [first, last)
    const bool any_new = last > seq.context && first < end, any_old = first < seq.context;
    if (!any_new && !(again && any_old)) continue;
    if constexpr (VALUES) {
      u32x4* to = reinterpret_cast<u32x4*>(page + p[u].at[0]);
      const u32x4 old = any_old ? *to : u32x4{0u, 0u, 0u, 0u};
      u32x4 word;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          y[n] = first + n < seq.context ? fp8_value(old[j], n) * ratio : x[u][4 * j + n] * inverse;
        word[j] = fp8_word(y[0], y[1], y[2], y[3]);
      }
      *to = word;
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // The last 16 dimensions' second 8 may be padding: written, as zeros.
        u32x2* to = reinterpret_cast<u32x2*>(page + p[u].at[k]);
        const u32x2 old = any_old ? *to : u32x2{0u, 0u};
        u32x2 word;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float y[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) y[n] = any_old ? fp8_value(old[j], n) * ratio : x[u][8 * k + 4 * j + n] * inverse;
          word[j] = fp8_word(y[0], y[1], y[2], y[3]);
        }
        *to = word;
      }
    }
  }
  if (threadIdx.x == 0) *held = scale;
}

template <int DT, bool VALUES>
__device__ __forceinline__ void append_page_16(const AppendArgs& a, const KvSeq& seq, int64_t id, int base, int head,
                                               int part) {
  const KvCache& c = a.cache;
  const int count = VALUES ? (c.page >> 2) * (c.dim >> 2) : c.page * ((c.dim + 15) >> 4);
  const int end = seq.context + seq.rows;
  char* page = (VALUES ? c.v : c.k) + (id * c.heads + head) * (static_cast<int64_t>(c.page) * c.chunks * 128);
  const int at = part * 256 + static_cast<int>(threadIdx.x);
  if (at >= count) return;
  const PageUnit p = page_unit<VALUES, false>(a, at);
  const int first = base + p.token, last = first + (VALUES ? 4 : 1);
  if (last <= seq.context || first >= end) return;
  float x[16];
  uint32_t close = 0;  // of no account: rounded to the model's type
  new_values<DT, VALUES>(a, seq, p, base, head, x, close);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32x4* to = reinterpret_cast<u32x4*>(page + p.at[h] + (VALUES ? h * 1024 : 0));
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[8 * h + i];
    u32x4 word = pack8<DT>(y);
    if constexpr (VALUES) {
      if (first < seq.context) {  // tokens from before share the word: lanes n of both dimensions
        const u32x4 old = *to;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (first + n < seq.context) {
            const uint32_t keep = 0xffffu << (16 * (n & 1));
            word[n / 2] = (word[n / 2] & ~keep) | (old[n / 2] & keep);
            word[2 + n / 2] = (word[2 + n / 2] & ~keep) | (old[2 + n / 2] & keep);
          }
      }
    } else if (p.e[h] >= c.dim) {
      continue;
    }
    *to = word;
  }
}

// A workgroup has a page of one head's keys or values (8 bits), 256 units of it (16 bits), 256 places of queries or a share of
// the rows that no sequence holds, all in one launch: what is bound by latency then waits once. Every row is read once, every code written once, in pieces of 8
// or 16 bytes that lie side by side over the lanes as the units' order has them. Bound by memory and the vector units (busy for
// 69 % of the cycles) where rows are many: 5327 rows of prompts, 16 heads of 128 over 4 in 8 bits, 15.6 us for 63 MB, 4.0
// TB/s; 650 rows of 32 heads of 80 over 32 in 16 bits 9.6 us for 20 MB, 2.1 TB/s, a beginning of 4 us to it; 32 single tokens
// 5.6 us, all latency.
template <int DT, bool E8, int UPT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  __shared__ float red[4];
  int block = blockIdx.x;
  if (block >= a.kv_blocks) {
    const int clears = a.kv_blocks + a.q_blocks * a.rows.seqs;
    if (block < clears) append_queries<DT>(a, block - a.kv_blocks);
    else kv_clear(a.rows, a.cache.page_shift, a.q_out, static_cast<int64_t>(a.heads) * (a.cache.dim >> 3), block - clears, gridDim.x - clears);
    return;
  }
  const bool values = block & 1;
  block >>= 1;
  int part = 0;
  if constexpr (!E8) {
    part = block % a.parts;
    block /= a.parts;
  }
  const int head = block % a.cache.heads;
  block /= a.cache.heads;
  const int b = block / a.page_slots;
  const KvSeq seq = kv_seq(a.rows, b, a.cache.page_shift);
  const int number = (seq.context >> a.cache.page_shift) + block - b * a.page_slots;
  const int base = number << a.cache.page_shift;
  if (seq.rows == 0 || number >= a.rows.width || base >= seq.context + seq.rows) return;
  const int64_t id = a.rows.table[b * a.rows.table_stride + number];
  if (id < 0 || id >= a.cache.pages) return;
  if constexpr (E8) {
    if (values) append_page_fp8<DT, true, UPT>(a, seq, id, base, head, red);
    else append_page_fp8<DT, false, UPT>(a, seq, id, base, head, red);
  } else {
    if (values) append_page_16<DT, true>(a, seq, id, base, head, part);
    else append_page_16<DT, false>(a, seq, id, base, head, part);
  }
}

struct ReadArgs {
  KvCache cache;
  const int32_t* table;
  const int64_t* first;
  const int64_t* ends;
  uint16_t* k;  // [seqs, most, heads, dim]
  uint16_t* v;
  int64_t table_stride;
  int width, seqs, most, key_blocks, value_blocks;
};

// Pages back as rows. Thread: keys, 8 dimensions of one token; values, 8 dimensions of the 4 tokens that share their
// words. Bound by latency and, where tokens are many, by the vector units, which find the addresses (about 100 instructions per
// 16 bytes written, four divisions by sizes known at run time among them; busy for 62 % of the cycles): 1007 tokens of 32
// sequences, 4 heads of 128 in 8 bits, 4.9 us; 5459 tokens of four 8.4 us for 17 MB, 23 with the zeros behind them; 895 tokens
// of 32 heads of 80 in 16 bits 7.5 us for 18 MB.
template <int DT, bool E8>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const KvCache& c = a.cache;
  const bool values = static_cast<int>(blockIdx.x) >= a.key_blocks;
  const int blocks = values ? a.value_blocks : a.key_blocks, block = static_cast<int>(blockIdx.x) - (values ? a.key_blocks : 0);
  const int each = blocks / a.seqs, b = block / each;
  const int64_t most_tokens = static_cast<int64_t>(a.width) << c.page_shift;
  const int64_t first = a.first[b], end = min(a.ends[b], most_tokens);
  const int x = (block - b * each) * 256 + static_cast<int>(threadIdx.x);
  constexpr int bytes = E8 ? 1024 : 2048;
  const int64_t head_bytes = static_cast<int64_t>(c.page >> 4) * c.chunks * bytes;
  const int per_head = c.dim >> 3, per = per_head * c.heads;
  // Item: a token (keys) or the quad of tokens from the one that holds `first` (values). Keys go by blocks of 8 tokens x 8
  // places, whose 16-byte pieces lie side by side both in the cache (over tokens) and in the result (over places).
  int item, rest;
  if (values) {
    item = x / per;
    rest = x - item * per;
  } else {
    const int wide = (per + 7) >> 3, block8 = x >> 6, tokens8 = block8 / wide;
    item = (tokens8 << 3) + ((x >> 3) & 7);
    rest = ((block8 - tokens8 * wide) << 3) + (x & 7);
    if (rest >= per) return;
  }
  const int head = rest / per_head, e = (rest - head * per_head) << 3;
  const int64_t row = static_cast<int64_t>(c.heads) * c.dim;  // elements from a token to the next
  const int64_t out0 = static_cast<int64_t>(b) * a.most * row + head * c.dim + e;
  if (!values) {
    if (item >= a.most) return;
    const int64_t t = first + item;
    u32x4 out = u32x4{0u, 0u, 0u, 0u};
    if (t >= 0 && t < end) {
      const int64_t id = a.table[b * a.table_stride + (t >> c.page_shift)];
      if (id >= 0 && id < c.pages) {
        const int n = static_cast<int>(t & (c.page - 1));
        const char* from = c.k + (id * c.heads + head) * head_bytes + ((n >> 4) * c.chunks + (e >> 6)) * bytes +
                           ((e & 63) >> 4) * 256 + (n & 15) * 16;
        if constexpr (E8) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(from + (e & 8));
          const float scale = c.k_scale[id * c.heads + head];
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = fp8_value(w[j / 4], j & 3) * scale;
          out = pack8<DT>(y);
        } else {
          out = *reinterpret_cast<const u32x4*>(from + (e & 8) * 128);
        }
      }
    }
    *reinterpret_cast<u32x4*>(a.k + out0 + item * row) = out;
    return;
  }
  const int64_t t0 = ((first >> 2) + item) << 2;
  if (t0 - first >= a.most) return;
  u32x4 w[2][E8 ? 1 : 2];  // of dimensions e .. e + 3 and e + 4 .. e + 7
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int h = 0; h < (E8 ? 1 : 2); ++h) w[q][h] = u32x4{0u, 0u, 0u, 0u};
  float scale = 1.0f;
  if (t0 >= 0 && t0 < end) {
    const int64_t id = a.table[b * a.table_stride + (t0 >> c.page_shift)];
    if (id >= 0 && id < c.pages) {
      const int n = static_cast<int>(t0 & (c.page - 1));
      const char* from = c.v + (id * c.heads + head) * head_bytes + ((n >> 4) * c.chunks + (e >> 6)) * bytes +
                         ((n & 15) >> 2) * 256 + ((e & 63) >> 2) * 16;
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int h = 0; h < (E8 ? 1 : 2); ++h) w[q][h] = *reinterpret_cast<const u32x4*>(from + q * 16 + h * 1024);
      if constexpr (E8) scale = c.v_scale[id * c.heads + head];
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int64_t i = t0 + n - first;
    if (i < 0 || i >= a.most) continue;
    u32x4 out = u32x4{0u, 0u, 0u, 0u};
    if (t0 + n < end) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = j & 3;
        uint32_t half;
        if constexpr (E8) half = to_bits16<DT>(fp8_value(w[j / 4][0][k], n) * scale);
        else half = (w[j / 4][k / 2][2 * (k & 1) + n / 2] >> (16 * (n & 1))) & 0xffffu;
        out[j / 2] |= half << (16 * (j & 1));
      }
    }
    *reinterpret_cast<u32x4*>(a.v + out0 + i * row) = out;
  }
}

namespace {

template <int DT, bool E8>
void append_go(const AppendArgs& a, unsigned grid, hipStream_t s) {
  if constexpr (!E8) {
    append_kernel<DT, false, 1><<<grid, 256, 0, s>>>(a);
  } else {
    // Units of 16 values per thread, as many as keep a page's rows in registers.
    const int units = a.cache.page * ((a.cache.dim + 15) / 16);
    if (units <= 256) append_kernel<DT, true, 1><<<grid, 256, 0, s>>>(a);
    else if (units <= 512) append_kernel<DT, true, 2><<<grid, 256, 0, s>>>(a);
    else if (units <= 1024) append_kernel<DT, true, 4><<<grid, 256, 0, s>>>(a);
    else append_kernel<DT, true, 8><<<grid, 256, 0, s>>>(a);
  }
}

}  // namespace
}  // namespace plm

extern "C" {

int plm_kv_append(const plm_append_call* call, void* stream) {
  if (call == nullptr) return PLM_ERR_ARGUMENT;
  const plm_append_call& h = *call;
  plm::AppendArgs a{};
  if (!plm::kv_cache_of(h.cache, a.cache) || !plm::kv_type_fits(h.cache, h.dtype)) return PLM_ERR_ARGUMENT;
  if (!plm::kv_rows_of(a.cache, h.rows, a.rows)) return PLM_ERR_ARGUMENT;
  if (h.k == nullptr || h.v == nullptr) return PLM_ERR_ARGUMENT;
  if (h.q != nullptr && (h.heads < 1 || h.heads > 4096 || h.q_out == nullptr)) return PLM_ERR_ARGUMENT;
  if (h.rope != nullptr && (h.rotary < 2 || h.rotary > a.cache.dim || h.rotary % 2 != 0 || h.rope_rows < 1))
    return PLM_ERR_ARGUMENT;
  if ((h.q_row | h.q_head | h.k_row | h.k_head | h.v_row | h.v_head) % 8 != 0) return PLM_ERR_ALIGNMENT;
  for (const void* p : {h.q, static_cast<const void*>(h.q_out), h.k, h.v, static_cast<const void*>(a.cache.k),
                        static_cast<const void*>(a.cache.v), static_cast<const void*>(h.rope)})
    if (!plm::aligned16_ptr(p)) return PLM_ERR_ALIGNMENT;
  a.q = static_cast<const uint16_t*>(h.q);
  a.q_out = static_cast<uint16_t*>(h.q_out);
  a.new_k = static_cast<const uint16_t*>(h.k);
  a.new_v = static_cast<const uint16_t*>(h.v);
  a.q_row = h.q_row, a.q_head = h.q_head, a.k_row = h.k_row, a.k_head = h.k_head, a.v_row = h.v_row, a.v_head = h.v_head;
  a.positions = h.positions;
  a.rope = h.rope;
  a.rope_rows = h.rope_rows;
  a.heads = static_cast<int>(h.heads);
  a.rotary = static_cast<int>(h.rotary);
  a.side_by_side = h.side_by_side != 0;
  const int64_t page = a.cache.page, seqs = h.rows.seqs, max_rows = h.rows.max_rows;
  a.page_slots = static_cast<int>((page - 1 + max_rows + page - 1) / page);
  const bool e8 = h.cache->type == PLM_CACHE_E4M3;
  a.parts = e8 ? 1 : (a.cache.page * ((a.cache.dim + 15) / 16) + 255) / 256;
  const int64_t kv_blocks = seqs * a.page_slots * a.cache.heads * a.parts * 2;
  const int half = h.rope != nullptr ? a.rotary / 2 : 0;
  const int64_t places = half > 0 && !a.side_by_side && half % 8 == 0 ? (a.cache.dim - half) / 8 : a.cache.dim / 8;
  const int64_t q_items = h.q == nullptr ? 0 : max_rows * places * h.heads;
  const int64_t q_blocks = (q_items + 255) / 256;
  const int64_t clears = h.q == nullptr ? 0 : plm::kv_clear_groups(a.rows, h.heads * (a.cache.dim / 8));
  if (kv_blocks + q_blocks * seqs + clears >= (int64_t{1} << 31) || q_items >= (int64_t{1} << 31)) return PLM_ERR_ARGUMENT;
  a.kv_blocks = static_cast<int>(kv_blocks);
  a.q_blocks = static_cast<int>(q_blocks);
  const unsigned grid = static_cast<unsigned>(kv_blocks + q_blocks * seqs + clears);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (h.dtype == PLM_BF16) e8 ? plm::append_go<plm::DT_BF16, true>(a, grid, s) : plm::append_go<plm::DT_BF16, false>(a, grid, s);
  else e8 ? plm::append_go<plm::DT_F16, true>(a, grid, s) : plm::append_go<plm::DT_F16, false>(a, grid, s);
  return hipGetLastError() == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

int plm_kv_read(const plm_read_call* call, void* stream) {
  if (call == nullptr) return PLM_ERR_ARGUMENT;
  const plm_read_call& h = *call;
  plm::ReadArgs a{};
  if (!plm::kv_cache_of(h.cache, a.cache) || !plm::kv_type_fits(h.cache, h.dtype)) return PLM_ERR_ARGUMENT;
  if (h.seqs < 1 || h.seqs > (1 << 20) || h.most < 1 || h.most >= (1 << 30) || h.table == nullptr || h.first == nullptr ||
      h.ends == nullptr || h.k == nullptr || h.v == nullptr)
    return PLM_ERR_ARGUMENT;
  if (h.table_width < 1 || h.table_width > ((int64_t{1} << 29) >> a.cache.page_shift) || h.table_stride < h.table_width)
    return PLM_ERR_ARGUMENT;
  for (const void* p : {static_cast<const void*>(h.k), static_cast<const void*>(h.v), static_cast<const void*>(a.cache.k),
                        static_cast<const void*>(a.cache.v)})
    if (!plm::aligned16_ptr(p)) return PLM_ERR_ALIGNMENT;
  a.table = h.table;
  a.first = h.first;
  a.ends = h.ends;
  a.k = static_cast<uint16_t*>(h.k);
  a.v = static_cast<uint16_t*>(h.v);
  a.table_stride = h.table_stride;
  a.width = static_cast<int>(h.table_width);
  a.seqs = static_cast<int>(h.seqs);
  a.most = static_cast<int>(h.most);
  // Keys: an item per token and 8 dimensions; values: per quad of tokens (one more where `first` is inside a quad).
  const int64_t per = static_cast<int64_t>(a.cache.heads) * (a.cache.dim / 8);
  const int64_t keys = ((h.most + 7) / 8 * ((per + 7) / 8) * 64 + 255) / 256, quads = (((h.most + 3) / 4 + 1) * per + 255) / 256;
  if (keys >= (int64_t{1} << 23) || (keys + quads) * h.seqs >= (int64_t{1} << 31)) return PLM_ERR_ARGUMENT;
  a.key_blocks = static_cast<int>(keys * h.seqs);
  a.value_blocks = static_cast<int>(quads * h.seqs);
  const unsigned grid = static_cast<unsigned>((keys + quads) * h.seqs);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool e8 = h.cache->type == PLM_CACHE_E4M3;
  if (h.dtype == PLM_BF16) {
    if (e8) plm::read_kernel<plm::DT_BF16, true><<<grid, 256, 0, s>>>(a);
    else plm::read_kernel<plm::DT_BF16, false><<<grid, 256, 0, s>>>(a);
  } else {
    if (e8) plm::read_kernel<plm::DT_F16, true><<<grid, 256, 0, s>>>(a);
    else plm::read_kernel<plm::DT_F16, false><<<grid, 256, 0, s>>>(a);
  }
  return hipGetLastError() == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

}  // extern "C"
