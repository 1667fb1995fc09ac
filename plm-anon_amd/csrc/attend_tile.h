// Attention of many columns (prompts, rounds) over the paged cache: the products of attend.h with the keys and
// values of 64 tokens staged in LDS for all four wavefronts of a workgroup, each of which has 16 NC columns of its
// own. What a column costs is then the matrix cores and the exponentials, not the loads, and 8-bit codes are turned
// into the model's type once per workgroup instead of once per wavefront.
//
// LDS holds operands: 1 KiB each, lane l's registers at 16 l, so every access is 16 consecutive bytes per lane.
// Keys: [unit][chunk][half]; values: [pair of units][chunk][j], a lane's eight tokens from both units of the pair.
// Two sets of 64 tokens: the next one's loads are in flight in registers while the current is multiplied, and are
// stored behind it; one barrier per 64 tokens.
#pragma once

#include "attend.h"

namespace plm {

constexpr int kTile = 64;  // tokens staged at once
constexpr int attend_set_bytes(int chunks) { return 16 * chunks * 1024; }

template <int DT, bool E8, int C, int NC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attend_tile_kernel(AttendArgs a) {
  constexpr int COLS = 64 * NC;
  constexpr int kUnitBytes = E8 ? 1024 : 2048, kLoads = E8 ? 1 : 2;
  constexpr int kKeys = 8 * C * 1024, kSet = attend_set_bytes(C);  // bytes of a set: keys, then values
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const AttendItem it = attend_item<COLS, false>(a, blockIdx.x, lane);
  if (it.ranges == 0) return;
  KvSeq seq = kv_seq(a.rows, it.b, a.cache.page_shift);
  seq.start = __builtin_amdgcn_readfirstlane(seq.start);
  seq.rows = __builtin_amdgcn_readfirstlane(seq.rows);
  seq.context = __builtin_amdgcn_readfirstlane(seq.context);
  const int columns = seq.rows * a.group;
  const int end = seq.context + seq.rows;
  const int last_page = (end + a.cache.page - 1) >> a.cache.page_shift;

  AttendColumns<NC> cols;
  const int first_col = wave * 16 * NC;
  cols.set(a, seq, it, it.tile * COLS + first_col, columns, col);
  u32x4 q[NC][C][2];
  cols.template queries<DT, C>(a, seq, g, q);
  f32x4 o[NC][C][4];
  float m[NC], l[NC];
  // The walk is the workgroup's: bounds over all four wavefronts' windows.
  AttendWalk<kTile> walk;
  int lo_least, lo_most;
  window_bounds(a, cols, lo_least, lo_most);
  int* bounds = reinterpret_cast<int*>(lds);
  if (lane == 0) {
    bounds[2 * wave] = lo_least;
    bounds[2 * wave + 1] = lo_most;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo_least = min(lo_least, bounds[2 * i]);
    lo_most = max(lo_most, bounds[2 * i + 1]);
  }
  lo_least = __builtin_amdgcn_readfirstlane(lo_least);
  walk.lo_most = __builtin_amdgcn_readfirstlane(lo_most);
  walk.set(a, seq, it, COLS, columns, cols, lo_least);
  __syncthreads();

  // Pages: lane i has number page_first + i of the sequence. fp16 values are staged in units of the largest scale
  // of their pages so far (`ref`), which keeps codes times scale inside fp16; bf16 takes any scale.
  int page_id = -1, page_first = -64;
  float page_ks = 0.0f, page_vs = 0.0f, ref = DT == DT_F16 ? 0.0f : 1.0f, next_ref = ref;
  auto pages = [&](int number) {
    page_first = number;
    const int at = number + lane;
    int id = -1;
    if (at < last_page && at < a.rows.width) id = a.rows.table[it.b * a.rows.table_stride + at];
    const bool good = id >= 0 && id < a.cache.pages;
    page_id = good ? id : -1;
    if constexpr (E8) {
      page_ks = good ? fmaxf(a.cache.k_scale[static_cast<int64_t>(id) * a.cache.heads + it.head], kLeastScale) : kLeastScale;
      page_vs = good ? a.cache.v_scale[static_cast<int64_t>(id) * a.cache.heads + it.head] : 0.0f;
      if constexpr (DT == DT_F16) {
        float most = page_vs;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor(most, x));
        next_ref = fmaxf(next_ref, __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, most))));
      }
    }
  };

  // A wavefront stages C jobs of 4 C: keys or values of a pair of units of one chunk.
  u32x4 stage[C][2][kLoads];
  float unit_ks[4], unit_vs[4];
  uint32_t unit_held = 0;  // bit u: unit u's page is there
  auto fetch = [&](int t0) {
    int64_t base[4];
    // A page of one head is at most 128 KiB, a page of all heads 128 MiB.
    const uint32_t page_bytes = static_cast<uint32_t>(a.cache.page >> 4) * (C * kUnitBytes);
    unit_held = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + 16 * u;
      const int number = t >> a.cache.page_shift;
      if (number < page_first || number >= page_first + 64) pages(number);
      const int id = __builtin_amdgcn_readlane(page_id, number - page_first);
      unit_held |= static_cast<uint32_t>(id >= 0) << u;
      if constexpr (E8) {
        unit_ks[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, page_ks), number - page_first));
        unit_vs[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, page_vs), number - page_first));
      }
      base[u] = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(max(id, 0))) * (page_bytes * a.cache.heads) +
                                     page_bytes * static_cast<uint32_t>(it.head) +
                                     static_cast<uint32_t>((t & (a.cache.page - 1)) >> 4) * (C * kUnitBytes));
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int job = wave + 4 * i;
      const bool values = job >= 2 * C;
      const int x = values ? job - 2 * C : job, pair = x / C, c = x - pair * C;
      const bool inside = (values ? 4 * col : 16 * g) < a.cache.dim - 64 * c;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const __amdgpu_buffer_rsrc_t rs =
            unit_rsrc(values ? a.cache.v : a.cache.k, pair ? base[2 + u] : base[u], C * kUnitBytes);
#pragma unroll
        for (int h = 0; h < kLoads; ++h)
          stage[i][u][h] = buffer_load16(rs, inside ? static_cast<uint32_t>(c * kUnitBytes + h * 1024 + lane * 16) : kOutOfRange);
      }
    }
  };
  bool odd = false;  // staged a value that is not finite for columns that may not all look (see attend_kernel)
  auto store = [&](int t0, char* set) {
    const bool edge = walk.edge(t0) || unit_held != 15u;
    const bool cut = t0 + kTile > end || unit_held != 15u;  // tokens that are no one's: values there are zero
    const float less = DT == DT_F16 ? (ref > 0.0f ? 1.0f / ref : 0.0f) : 1.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int job = wave + 4 * i;
      const bool values = job >= 2 * C;
      const int x = values ? job - 2 * C : job, pair = x / C, c = x - pair * C;
      if (!values) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          char* to = set + ((2 * pair + u) * C + c) * 2048 + lane * 16;
          if constexpr (E8) {
            *reinterpret_cast<u32x4*>(to) = fp8_eight<DT>(stage[i][u][0][0], stage[i][u][0][1], 1.0f);
            *reinterpret_cast<u32x4*>(to + 1024) = fp8_eight<DT>(stage[i][u][0][2], stage[i][u][0][3], 1.0f);
          } else {
            *reinterpret_cast<u32x4*>(to) = stage[i][u][0];
            *reinterpret_cast<u32x4*>(to + 1024) = stage[i][u][1];
          }
        }
      } else {
        char* to = set + kKeys + (pair * C + c) * 4096 + lane * 16;
        const float r0 = (pair ? unit_vs[2] : unit_vs[0]) * less, r1 = (pair ? unit_vs[3] : unit_vs[1]) * less;
        u32x4 keep = {~0u, ~0u, ~0u, ~0u};
        if (cut) {
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            const int u = 2 * pair + i2 / 2, t = t0 + 16 * u + 4 * g + 2 * (i2 & 1);
            const bool held = ((unit_held >> u) & 1u) != 0;
            keep[i2] = (held && t < end ? 0xffffu : 0u) | (held && t + 1 < end ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u32x4 v;
          if constexpr (E8) {
            v = u32x4{fp8_pair<DT>(stage[i][0][0][j], r0, false), fp8_pair<DT>(stage[i][0][0][j], r0, true),
                      fp8_pair<DT>(stage[i][1][0][j], r1, false), fp8_pair<DT>(stage[i][1][0][j], r1, true)};
          } else {
            v = u32x4{stage[i][0][j / 2][2 * (j & 1)], stage[i][0][j / 2][2 * (j & 1) + 1], stage[i][1][j / 2][2 * (j & 1)],
                      stage[i][1][j / 2][2 * (j & 1) + 1]};
          }
          v &= keep;
          *reinterpret_cast<u32x4*>(to + j * 1024) = v;
          if (edge) {
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) odd = odd || pair_not_finite<DT>(v[i2]);
          }
        }
      }
    }
  };

  auto compute = [&](auto careful, const char* set, int t0, const float (&ks)[4], uint32_t held) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const bool edge = walk.edge(t0) || held != 15u;
    const char* keys = set + lane * 16;
    const char* values = keys + kKeys;
    f32x4 s[NC][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int n = 0; n < NC; ++n) s[n][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 k = *reinterpret_cast<const u32x4*>(keys + ((u * C + c) * 2 + h) * 1024);
#pragma unroll
          for (int n = 0; n < NC; ++n) s[n][u] = mfma_16x16x32<DT>(k, q[n][c][h], s[n][u]);
        }
    }
    uint32_t seen[NC];
    if (edge) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        seen[n] = cols.template seen_bits<4>(a, seq, n, t0, g, held);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[n][u][r] = (seen[n] >> (4 * u + r)) & 1u ? s[n][u][r] : kMinusInf;
      }
    }
    float mult[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) mult[u] = E8 ? a.scale * ks[u] : a.scale;
    u32x4 p[NC][2];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      // The scale is positive: maxima are found before it is multiplied in, which then costs no instruction.
      float top = kMinusInf;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        top = larger_of(top, larger_of(larger_of(larger_of(s[n][u][0], s[n][u][1]), s[n][u][2]), s[n][u][3]) * mult[u]);
      top = column_max(top);
      if (__any(top > m[n] + kSlack)) {
        const float next = larger_of(m[n], top);
        const float less = m[n] == next ? 1.0f : __builtin_amdgcn_exp2f(m[n] - next);
        m[n] = next;
        l[n] *= less;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][c][j] *= less;
      }
      const float base = m[n] == kMinusInf ? 0.0f : m[n] - kShift<DT>;
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = __builtin_amdgcn_exp2f(fmaf(s[n][u][r], mult[u], -base));
          sum += e[r];
        }
        p[n][u / 2][2 * (u & 1)] = pack2<DT>(e[0], e[1]);
        p[n][u / 2][2 * (u & 1) + 1] = pack2<DT>(e[2], e[3]);
      }
      l[n] += sum;
    }
    if (!CAREFUL || !edge) {
#pragma unroll
      for (int pair = 0; pair < 2; ++pair)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(values + ((pair * C + c) * 4 + j) * 1024);
#pragma unroll
            for (int n = 0; n < NC; ++n) o[n][c][j] = mfma_16x16x32<DT>(v, p[n][pair], o[n][c][j]);
          }
      return;
    }
    // One token at a time, as in attend_kernel.
#pragma unroll
    for (int pair = 0; pair < 2; ++pair)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(values + ((pair * C + c) * 4 + j) * 1024);
#pragma unroll 1
          for (int x = 0; x < 32; ++x) {
            const TokenOf t(x, g);
#pragma unroll
            for (int n = 0; n < NC; ++n)
              take_token<DT>(v & t.only, p[n][pair] & t.only, t.seen(seen[n], pair, col), o[n][c][j]);
          }
        }
  };

  // The accumulators follow `ref` when the set that was staged with the new one is up.
  auto follow = [&]() {
    if constexpr (E8 && DT == DT_F16) {
      if (next_ref > ref) {
        const float less = ref / next_ref;
        ref = next_ref;
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][c][j] *= less;
      }
    }
  };
  auto begin = [&]() {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][c][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      m[n] = kMinusInf;
      l[n] = 0.0f;
    }
    page_first = -64;
    ref = next_ref = DT == DT_F16 ? 0.0f : 1.0f;
  };

  begin();
  if (walk.from < walk.to) {
    int t0 = walk.token_of(walk.from);
    fetch(t0);
    follow();
    store(t0, lds);
    __syncthreads();
    int set = 0;
    for (int s = walk.from; s < walk.to; ++s) {
      const float ks[4] = {unit_ks[0], unit_ks[1], unit_ks[2], unit_ks[3]};
      const uint32_t held = unit_held;
      const int now = t0;
      const bool more = s + 1 < walk.to;
      if (more) {
        t0 = walk.token_of(s + 1);
        fetch(t0);
      }
      compute(std::false_type{}, lds + set * kSet, now, ks, held);
      set ^= 1;
      if (more) {
        follow();
        store(t0, lds + set * kSet);
      }
      __syncthreads();
    }
    if (__syncthreads_or(odd)) {
      begin();
#pragma unroll 1
      for (int s = walk.from; s < walk.to; ++s) {
        t0 = walk.token_of(s);
        fetch(t0);
        follow();
        store(t0, lds);
        __syncthreads();
        compute(std::true_type{}, lds, t0, unit_ks, unit_held);
        __syncthreads();
      }
    }
  }

#pragma unroll
  for (int n = 0; n < NC; ++n) {
    l[n] = column_sum(l[n]);
    if constexpr (E8 && DT == DT_F16) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][c][j] *= ref;
    }
  }
  if (it.ranges == 1) {
    cols.template store<DT, C>(a, seq, g, o, l);
    return;
  }
  attend_publish<NC, C>(a, it, COLS, first_col, g, col, cols, o, m, l);
}

}  // namespace plm
