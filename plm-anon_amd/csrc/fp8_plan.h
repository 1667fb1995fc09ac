// How a product over e4m3 rows is cut into workgroups: by what each way takes, estimated from what a CU pulls.
//
// Measured at 2048 x 2048 to 50257 x 2048 and 2560 x 10240 over 1 to 2048 rows, weights from memory: the way with the least
// estimate is the fastest measured one, or within a tenth of it. What bounds nearly all of them is a CU's reads, 55 to 65 GB/s
// of both operands where several wavefronts share them, 24 of weights and 94 of X where each reads its own.
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

// Few rows: a workgroup has `rows` fragments of X and `width` of the weight and `waves` wavefronts, and K is cut into `ranges`,
// whose sums a second launch joins.
struct Fp8Narrow {
  int rows, width, waves, ranges;
  double us;
};

// `in16`: rows of 16 bits, which every workgroup rounds.
inline Fp8Narrow narrow_plan(int64_t x_frags, int64_t w_frags, int64_t blocks, bool act, bool in16) {
  const int64_t down = (x_frags + 3) / 4;
  Fp8Narrow best{static_cast<int>((x_frags + down - 1) / down), 2, 8, 1, 1e30};
  // Above 256 fragments of the weight two at a time: 6144 x 2048 at 56 rows 6.3 us for 7.6; at 128 fragments one: 4.2 for 4.7.
  for (int width = act || w_frags > 256 ? 2 : 1; width <= 2; ++width) {
    const int64_t across = (w_frags + width - 1) / width * down;
    // One range, or as many as there are CUs for, of eight blocks at least. 2048 x 8192 at 64 rows: 14.2 us whole, 10.8 in four
    // ranges, at 16 rows 8.3 and 8.7; 2560 x 10240 at 42 rows 15.2 whole, 12.5 in three.
    const int64_t most = std::min(std::max<int64_t>(kFp8Cus / across, 1), (blocks + 7) / 8);
    for (int64_t ranges = 1; ranges <= most; ranges = ranges < most ? most : most + 1) {
      const double kib = 2.048 * static_cast<double>((blocks + ranges - 1) / ranges);   // of a fragment, in thousands of bytes
      const double each = width == 1 ? kib / 24 + kib * best.rows / 94 : kib * 2 / 28 + kib * best.rows / 110;
      const double us = 2.2 + each * fp8_turns(across * ranges) + (ranges > 1 ? 4.5 : 0.0);
      if (us < best.us) best = {best.rows, width, 8, static_cast<int>(ranges), us};
    }
  }
  // What every workgroup rounds for itself is better shared by fewer wavefronts where there are many workgroups: the LM head
  // of 50257 x 2048 over one token 21.2 us for 25.7, gate/up of 11264 x 2048 7.8 for 8.6, 6144 x 2048 5.4 for 5.0.
  if (in16 && w_frags > 512) best.waves = 4;
  return best;
}

// More than 64 rows: tiles of the weight's rows x rows of X. (Fewer fill no tile: gate/up of 11264 x 2048 at 42 rows 13.5 us for 9.9.)
enum Fp8TileKind { kTile64x64, kTile128x64, kTile128x128, kTile256x256 };

struct Fp8TilePlan {
  Fp8TileKind kind;
  double us;
};

// `exact`: results in fp32, from products in bf16; tiles of 128 x 64 and 128 x 128.
inline Fp8TilePlan tile_plan(int64_t x_frags, int64_t w_frags, int64_t blocks, bool exact) {
  struct Size {
    int n, m;             // fragments
    double step, end;     // us a block of K, and a tile's beginning and end
    double exact;         // a block's step in fp32, 0 for none
  };
  constexpr Size sizes[] = {{4, 4, 0.27, 1.0, 0.0}, {8, 4, 0.40, 1.5, 0.6}, {8, 8, 0.53, 2.0, 1.02}, {16, 16, 1.07, 5.6, 0.0}};
  const double steps = static_cast<double>((blocks + 3) / 4 * 4);
  Fp8TilePlan best{kTile64x64, 1e30};
  for (int k = kTile64x64; k <= kTile256x256; ++k) {
    const Size& z = sizes[k];
    if (exact && z.exact == 0.0) continue;
    const int64_t tiles = ((w_frags + z.n - 1) / z.n) * ((x_frags + z.m - 1) / z.m);
    // The largest are bound by the matrix cores, whose clock falls as more of them work.
    const double step = exact ? z.exact : k == kTile256x256 ? z.step + 0.3 * std::min(1.0, static_cast<double>(tiles) / kFp8Cus) : z.step;
    const double us = k == kTile256x256 ? 2.2 + fp8_turns(tiles) * (steps * step + z.end) : 2.2 + z.end + fp8_turns(tiles) * steps * step;
    if (us < best.us) best = {static_cast<Fp8TileKind>(k), us};
  }
  return best;
}

}  // namespace plm
