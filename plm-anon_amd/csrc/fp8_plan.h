// How a product over e4m3 rows is cut into workgroups: by what each way takes, estimated from what a CU pulls and what comes from
// memory.
//
// Measured at 2048 x 2048 to 50257 x 2048, 8192 x 8192, 2560 x 10240 and two gate/up weights, 16-bit and fp32 results, over 1 to
// 2048 rows, each way by itself: of 210 choices all but two are the fastest way or within a tenth of it, gate/up of 28672 x 2048
// over 30 rows (16.0 us for 13.8) and of 11264 x 2048 over 512 in fp32 (33.1 for 29.6).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace plm {

constexpr int kFp8Cus = 256;

// How long `groups` workgroups take against one: CUs left over in the last turn find their neighbours' work half done.
inline double fp8_turns(int64_t groups) {
  const int64_t whole = (groups + kFp8Cus - 1) / kFp8Cus;
  return whole == 1 ? 1.0 : 0.5 * (static_cast<double>(groups) / kFp8Cus + static_cast<double>(whole));
}

// us that a weight takes from memory, at a copy's rate; and with `work` us on the CUs, which hides the shorter of the two in part.
inline double fp8_memory(int64_t w_frags, int64_t blocks) { return static_cast<double>(w_frags * blocks) * 2048 / 5.1e6; }
inline double fp8_beside(double work, double memory, double shown) {
  return 2.2 + std::max(work, memory) + shown * std::min(work, memory);
}

// Few rows: a workgroup has `rows` fragments of X and `width` of the weight and `waves` wavefronts, and K is cut into `ranges`,
// whose sums a second launch joins.
struct Fp8Narrow {
  int rows, width, waves, ranges;
  double us;
};

// `in16`: rows of 16 bits, which every workgroup rounds.
inline Fp8Narrow narrow_plan(int64_t x_frags, int64_t w_frags, int64_t blocks, bool act, bool in16) {
  const int64_t down = (x_frags + 3) / 4;
  const double memory = fp8_memory(w_frags, blocks);
  Fp8Narrow best{static_cast<int>((x_frags + down - 1) / down), 2, 8, 1, 1e30};
  // Above 256 fragments of the weight two at a time: 6144 x 2048 at 56 rows 6.3 us for 7.6; at 128 fragments one: 4.2 for 4.7.
  for (int width = act || w_frags > 256 ? 2 : 1; width <= 2; ++width) {
    const int64_t across = (w_frags + width - 1) / width * down;
    // One range, or as many as there are CUs for, of eight blocks at least. 2048 x 8192 at 64 rows: 14.2 us whole, 10.8 in four
    // ranges, at 16 rows 8.3 and 8.7; 2560 x 10240 at 42 rows 15.2 whole, 12.5 in three.
    const int64_t most = std::min(std::max<int64_t>(kFp8Cus / across, 1), (blocks + 7) / 8);
    for (int64_t ranges = 1; ranges <= most; ranges = ranges < most ? most : most + 1) {
      // Of a fragment, in thousands of bytes; a CU reads 24 to 28 GB/s of weights and 94 to 110 of X.
      const double kib = 2.048 * static_cast<double>((blocks + ranges - 1) / ranges);
      const double each = width == 1 ? kib / 24 + kib * best.rows / 94 : kib * 2 / 28 + kib * best.rows / 110;
      const double us = fp8_beside(each * fp8_turns(across * ranges), memory, 0.35) + (ranges > 1 ? 4.5 : 0.0);
      if (us < best.us) best = {best.rows, width, 8, static_cast<int>(ranges), us};
    }
  }
  // What every workgroup rounds for itself is better shared by fewer wavefronts where there are many workgroups: the LM head
  // of 50257 x 2048 over one token 21.2 us for 25.7, gate/up of 11264 x 2048 7.8 for 8.6, 6144 x 2048 5.4 for 5.0.
  if (in16 && w_frags > 512) best.waves = 4;
  return best;
}

// Many rows, or a weight of so many that X is read too often otherwise: tiles of the weight's rows x rows of X. 50257 x 2048 over
// 56 rows 26.7 us for 32.8 the way of few rows, 28672 x 2048 gate/up over 64 15.2 for 19.7, 11264 x 2048 over 56 10.1 for 10.6.
// Below 33 rows they are not tried; of what was measured there only these weights would gain (24.6 for 26.2, 13.8 for 16.0 over 30).
constexpr int kFp8TileFrags = 3;
enum Fp8TileKind { kTile64x64, kTile128x64, kTile128x128, kTile128x256, kTile256x256 };

struct Fp8TilePlan {
  Fp8TileKind kind;
  double us;
};

// `exact`: results in fp32, from products in bf16; tiles of 128 x 64 and 128 x 128.
inline Fp8TilePlan tile_plan(int64_t x_frags, int64_t w_frags, int64_t blocks, bool exact) {
  struct Size {
    int n, m;             // fragments
    double step, end;     // us a block of K, and a tile's stores
    double exact;         // a block of K in fp32, 0 for none
  };
  constexpr Size sizes[] = {{4, 4, 0.27, 0.0, 0.0}, {8, 4, 0.40, 0.0, 0.6}, {8, 8, 0.53, 0.0, 1.02}, {8, 16, 0.80, 3.0, 0.0}, {16, 16, 1.07, 5.6, 0.0}};
  const double steps = static_cast<double>((blocks + 3) / 4 * 4), memory = fp8_memory(w_frags, blocks);
  Fp8TilePlan best{kTile64x64, 1e30};
  for (int k = kTile64x64; k <= kTile256x256; ++k) {
    const Size& z = sizes[k];
    if (exact && z.exact == 0.0) continue;
    const int64_t tiles = ((w_frags + z.n - 1) / z.n) * ((x_frags + z.m - 1) / z.m);
    // The largest are bound by the matrix cores, whose clock falls as more of them work.
    const double step = exact ? z.exact : k == kTile256x256 ? z.step + 0.3 * std::min(1.0, static_cast<double>(tiles) / kFp8Cus) : z.step;
    const double work = fp8_turns(tiles) * (steps * step + z.end);
    const double us = k == kTile256x256 ? 2.2 + work : fp8_beside(work, memory, 0.5);
    if (us < best.us) best = {static_cast<Fp8TileKind>(k), us};
  }
  return best;
}

}  // namespace plm
