// Attention of many columns (prompts, rounds) over the paged cache: the products of attend.h with the keys and
// values of 64 tokens staged in LDS for all four wavefronts of a workgroup, each of which has 16 NC columns of its
// own. What a column costs is then the matrix cores and the exponentials, not the loads, and 8-bit codes are turned
// into the model's type once per workgroup instead of once per wavefront.
//
// LDS holds operands: 1 KiB each, lane l's registers at 16 l, so every access is 16 consecutive bytes per lane.
// Keys: [unit][chunk][half]; values: [pair of units][chunk][j], a lane's eight tokens from both units of the pair.
// Two sets of 64 tokens: the next one's loads are in flight in registers while the current is multiplied, and are
// stored behind it; one barrier per 64 tokens.
//
// Bound by three things in turn, which the two wavefronts that a SIMD holds overlap in part: the vector units (per score
// a scaling, an exponential, a sum, half a maximum and half a rounding), the matrix cores, and LDS, from which every
// wavefront reads every operand for its 32 columns. 4096 rows after 4096 tokens, 16 heads of 128 over 4 in 8 bits: 242 us
// or 853 TFLOP/s of visible pairs (a product of 8192^3 reaches 1122), the vector units busy for 56 % of the cycles, the
// matrix cores for 40 %, LDS for about 58 %. At heads of 64 there are half the products to a score: 3381 rows through
// windows of 512, 32 heads over 8, 38.5 us or 316 TFLOP/s, 62 % and 17 %, 12 vector instructions to each of 60 million walked
// scores (48 million are visible), one of them the exponential. Measured without gain: loads two steps ahead, the
// sums of exponentials by a product with ones, raised priority around the products, no maxima but where a sum shows that
// one has grown (248 us for 242).
#pragma once

#include "attend.h"

namespace plm {

constexpr int kTile = 64;  // tokens staged at once
constexpr int kNoLds = 0x1e;  // __builtin_amdgcn_sched_barrier: all but LDS accesses may move across
constexpr int attend_set_bytes(int chunks) { return 16 * chunks * 1024; }
// Of longer heads one set: two workgroups fit a CU then, which is worth more than the barrier that it costs (prompts of
// heads of 256: 365 us with two sets, 240 with one).
constexpr int attend_sets(int chunks) { return chunks > 2 ? 1 : 2; }

template <int DT, bool E8, int C, int NC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attend_tile_kernel(AttendArgs a) {
  constexpr int COLS = 64 * NC;
  constexpr int kUnitBytes = E8 ? 1024 : 2048, kLoads = E8 ? 1 : 2;
  constexpr int kKeys = 8 * C * 1024, kSet = attend_set_bytes(C);  // bytes of a set: keys, then values
  constexpr int kSets = attend_sets(C);
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  if (static_cast<int>(blockIdx.x) >= a.walkers) return attend_clear(a);
  const AttendItem it = attend_item<COLS, false>(a, blockIdx.x, lane);
  if (it.ranges == 0) return;
  const KvSeq& seq = it.seq;
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

  // Pages: lane i has number page_first + i of the sequence: the byte where its head begins (bit 0: it is not there,
  // and page 0 is read) and its scales. fp16 values are staged in the accumulators' unit `ref` (kUnits): one for all 64
  // pages where their scales allow it (`calm`), looked for at every set of tokens only where not (at every set throughout:
  // 2048 rows of 32 heads of 64 60 us for 56).
  const uint32_t page_bytes = static_cast<uint32_t>(a.cache.page >> 4) * (C * kUnitBytes);  // of a head, 128 KiB at most
  uint32_t page_lo = 1, page_hi = 0;
  int page_first = -64;
  float page_ks = kLeastScale, page_vs = 0.0f, ref = 1.0f, next_ref = 1.0f;
  bool calm = true;
  auto first_lane = [](float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); };
  auto pages = [&](int number) {
    page_first = number;
    const int at = number + lane;
    int64_t id = -1;
    if (at < last_page && at < a.rows.width) id = a.rows.table[it.b * a.rows.table_stride + at];
    const bool good = id >= 0 && id < a.cache.pages;
    const uint64_t byte = good ? static_cast<uint64_t>(id) * (page_bytes * static_cast<uint64_t>(a.cache.heads)) + page_bytes * static_cast<uint32_t>(it.head) : 1;
    page_lo = static_cast<uint32_t>(byte);
    page_hi = static_cast<uint32_t>(byte >> 32);
    if constexpr (E8) {
      const int64_t of = good ? id * a.cache.heads + it.head : 0;
      page_ks = good ? fmaxf(a.cache.k_scale[of], kLeastScale) : kLeastScale;
      page_vs = good ? a.cache.v_scale[of] : 0.0f;
      if constexpr (kUnits<DT, E8>) {
        float most = page_vs >= kSilent ? page_vs : 0.0f, least = page_vs >= kSilent ? page_vs : __builtin_inff();
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) {
          most = fmaxf(most, __shfl_xor(most, x));
          least = fminf(least, __shfl_xor(least, x));
        }
        const float of_all[2] = {first_lane(most), first_lane(fminf(least, most))};
        next_ref = ref;
        calm = unit_for(of_all, next_ref);
      }
    }
  };
  auto lane_float = [](float v, int at) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), at));
  };

  // A wavefront stages keys (wavefronts 0 and 1) or values (2 and 3) of one pair of the four units.
  const int pair = wave & 1;
  const bool values_role = wave >= 2;
  const bool inside = (values_role ? 4 * col : 16 * g) < a.cache.dim - 64 * (C - 1);  // of the last chunk
  const char* const role_base = values_role ? a.cache.v : a.cache.k;
  struct Stage {
    u32x4 x[2][C][kLoads];
    float ks[4], vs[2];
    uint32_t held;  // bit u: unit u's page is there
    int t0;
  };
  Stage st;
  auto fetch = [&](int t0) {
    const int shift = a.cache.page_shift, number = t0 >> shift;
    if (number < page_first || ((t0 + 48) >> shift) >= page_first + 64) pages(number);
    st.t0 = t0;
    st.held = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = ((t0 + 16 * u) >> shift) - page_first;
      st.held |= (~static_cast<uint32_t>(__builtin_amdgcn_readlane(page_lo, at)) & 1u) << u;
      if constexpr (E8) st.ks[u] = lane_float(page_ks, at);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = t0 + 32 * pair + 16 * u, at = (t >> shift) - page_first;
      if constexpr (E8) st.vs[u] = lane_float(page_vs, at);
      const uint64_t byte = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(page_hi, at))) << 32 |
                            (static_cast<uint32_t>(__builtin_amdgcn_readlane(page_lo, at)) & ~1u);
      load_unit<E8, C, false>(role_base, static_cast<int64_t>(byte + static_cast<uint32_t>((t & (a.cache.page - 1)) >> 4) * (C * kUnitBytes)),
                       lane, inside, st.x[u]);
    }
  };
  bool odd = false;  // staged a value that is not finite for columns that may not all look, or `apart` (see attend_kernel)
  bool apart = false;  // the staged tokens' pages have no unit in common: their values are the codes themselves (0 of silent ones)
  auto store = [&](char* set) {
    if (!values_role) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          char* to = set + ((2 * pair + u) * C + c) * 2048 + lane * 16;
          if constexpr (E8) {
            const u32x4 x = st.x[u][c][0];
            *reinterpret_cast<u32x4*>(to) = fp8_eight<DT>(x[0], x[1], 1.0f);
            *reinterpret_cast<u32x4*>(to + 1024) = fp8_eight<DT>(x[2], x[3], 1.0f);
          } else {
            *reinterpret_cast<u32x4*>(to) = st.x[u][c][0];
            *reinterpret_cast<u32x4*>(to + 1024) = st.x[u][c][1];
          }
        }
      return;
    }
    const float less = kUnits<DT, E8> ? (ref > 0.0f ? 1.0f / ref : 0.0f) : 1.0f;
    auto ratio = [&](float vs) { return !apart ? vs * less : vs < kSilent ? 0.0f : 1.0f; };
    const float r0 = ratio(st.vs[0]), r1 = ratio(st.vs[1]);
    const bool edge = walk.edge(st.t0) || st.held != 15u;
    // Tokens that are no one's, past the end or of a page that is not there, have values of zero.
    u32x4 keep = {~0u, ~0u, ~0u, ~0u};
    if (st.t0 + kTile > end || st.held != 15u) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool held = ((st.held >> (2 * pair + u)) & 1u) != 0;
        const int live = held ? end - (st.t0 + 32 * pair + 16 * u + 4 * g) : 0;  // of the lane's four tokens
        keep[2 * u] = live >= 2 ? ~0u : live == 1 ? 0xffffu : 0u;
        keep[2 * u + 1] = live >= 4 ? ~0u : live == 3 ? 0xffffu : 0u;
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 v;
        if constexpr (E8) {
          v = u32x4{fp8_pair<DT>(st.x[0][c][0][j], r0, false), fp8_pair<DT>(st.x[0][c][0][j], r0, true),
                    fp8_pair<DT>(st.x[1][c][0][j], r1, false), fp8_pair<DT>(st.x[1][c][0][j], r1, true)};
        } else {
          v = u32x4{st.x[0][c][j / 2][2 * (j & 1)], st.x[0][c][j / 2][2 * (j & 1) + 1], st.x[1][c][j / 2][2 * (j & 1)],
                    st.x[1][c][j / 2][2 * (j & 1) + 1]};
        }
        v &= keep;
        *reinterpret_cast<u32x4*>(set + kKeys + ((pair * C + c) * 4 + j) * 1024 + lane * 16) = v;
        if (edge) {
#pragma unroll
          for (int i = 0; i < 4; ++i) odd = odd || pair_not_finite<DT>(v[i]);
        }
      }
  };

  auto value_scale = [&](int t0, int u) { return lane_float(page_vs, ((t0 + 16 * u) >> a.cache.page_shift) - page_first); };
  auto move = [&](float to) {
    if (to == ref) return;
    const float by = unit_ratio(ref, to);
    ref = to;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][c][j] *= by;
  };
  auto compute = [&](auto careful, const char* set, int t0, const float (&ks)[4], uint32_t held) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const bool edge = walk.edge(t0) || held != 15u;
    const char* keys = set + lane * 16;
    const char* values = keys + kKeys;
    // Operands come from LDS four at a time, the next four ahead of the products with the current: the products of
    // one (chunk, half) with all four units are independent of each other and take longer than a read.
    u32x4 x[2][4];
    auto read_keys = [&](int ch, u32x4 (&to)[4]) {
#pragma unroll
      for (int u = 0; u < 4; ++u) to[u] = *reinterpret_cast<const u32x4*>(keys + (u * 2 * C + ch) * 1024);
    };
    auto read_values = [&](int pc, u32x4 (&to)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j] = *reinterpret_cast<const u32x4*>(values + (pc * 4 + j) * 1024);
    };
    f32x4 s[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int u = 0; u < 4; ++u) s[n][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    read_keys(0, x[0]);
#pragma unroll
    for (int ch = 0; ch < 2 * C; ++ch) {
      if (ch + 1 < 2 * C) read_keys(ch + 1, x[(ch + 1) & 1]);
      else read_values(0, x[(ch + 1) & 1]);
      __builtin_amdgcn_sched_barrier(kNoLds);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][u] = mfma_16x16x32<DT>(x[ch & 1][u], q[n][ch / 2][ch & 1], s[n][u]);
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
        // Rounded once to the model's type. (In two parts, as attend_kernel has them: 324 us for 242 at 4096 rows after 4096
        // tokens, 42 for 37.5 through a window, since here the matrix cores and vector units are what bounds; over 8-bit pages
        // in fp16, whose products cost the same, 3 to 8 % more for the values' units. Of outputs that are rounded themselves
        // the error against 64 bits is 1.3 times the output's rounding alone, 0.0023 for 0.0017 in bf16.)
        p[n][u / 2][2 * (u & 1)] = pack2<DT>(e[0], e[1]);
        p[n][u / 2][2 * (u & 1) + 1] = pack2<DT>(e[2], e[3]);
      }
      l[n] += sum;
    }
    if (!CAREFUL || !(edge || apart)) {
#pragma unroll
      for (int pc = 0; pc < 2 * C; ++pc) {
        if (pc + 1 < 2 * C) read_values(pc + 1, x[(pc + 1) & 1]);
        __builtin_amdgcn_sched_barrier(kNoLds);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int n = 0; n < NC; ++n) o[n][pc % C][j] = mfma_16x16x32<DT>(x[pc & 1][j], p[n][pc / C], o[n][pc % C][j]);
      }
      return;
    }
    // One token at a time, as in attend_kernel.
    if (!edge) {
#pragma unroll
      for (int n = 0; n < NC; ++n) seen[n] = ~0u;
    }
#pragma unroll
    for (int pair = 0; pair < 2; ++pair) {
#pragma unroll 1
      for (int u = 0; u < (apart ? 2 : 1); ++u) {
        if (apart) {
          const float to = value_scale(t0, 2 * pair + u);
          if (to >= kSilent) move(to);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(values + ((pair * C + c) * 4 + j) * 1024);
#pragma unroll 1
            for (int x = 16 * u; x < (apart ? 16 * u + 16 : 32); ++x) {
              const TokenOf t(x, g);
#pragma unroll
              for (int n = 0; n < NC; ++n)
                take_token<DT>(v & t.only, p[n][pair] & t.only, t.seen(seen[n], pair, col), o[n][c][j]);
            }
          }
      }
    }
  };

  // The accumulators take the unit of the tokens to be staged once those before are multiplied.
  auto follow = [&]() {
    if constexpr (kUnits<DT, E8>) {
      float to = next_ref;
      if (!calm) {
        const float vs[4] = {value_scale(st.t0, 0), value_scale(st.t0, 1), value_scale(st.t0, 2), value_scale(st.t0, 3)};
        to = ref;
        apart = !unit_for(vs, to);
        odd = odd || apart;
      } else {
        apart = false;
      }
      move(to);
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
    ref = next_ref = kUnits<DT, E8> ? 0.0f : 1.0f;
  };

  begin();
  if (walk.from < walk.to) {
    // The first turn only fetches: one copy of the code, which short walks wait for too.
#pragma unroll 1
    for (int s = walk.from - 1; s < walk.to; ++s) {
      const int t0 = st.t0, set = kSets == 2 ? (s - walk.from) & 1 : 0;
      const float ks[4] = {st.ks[0], st.ks[1], st.ks[2], st.ks[3]};
      const uint32_t held = st.held;
      if (s + 1 < walk.to) fetch(walk.token_of(s + 1));
      if (s >= walk.from) compute(std::false_type{}, lds + set * kSet, t0, ks, held);
      if (s + 1 < walk.to) {
        follow();
        if constexpr (kSets == 1) __syncthreads();
        store(lds + (kSets == 2 ? set ^ 1 : 0) * kSet);
      }
      __syncthreads();
    }
    if (__syncthreads_or(odd)) {
      begin();
#pragma unroll 1
      for (int s = walk.from; s < walk.to; ++s) {
        fetch(walk.token_of(s));
        follow();
        store(lds);
        __syncthreads();
        compute(std::true_type{}, lds, st.t0, st.ks, st.held);
        __syncthreads();
      }
    }
  }

#pragma unroll
  for (int n = 0; n < NC; ++n) {
    l[n] = column_sum(l[n]);
    if constexpr (kUnits<DT, E8>) {
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
