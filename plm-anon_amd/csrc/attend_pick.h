// Which kernel a launch of plm_attend takes (a translation unit per type of rows and cache includes it).
#pragma once

#include <atomic>

#include "attend.h"
#include "attend_tile.h"

namespace plm {

// Lets `kern` have more than 64 KiB of LDS, once per device (`done`: a bit each).
inline hipError_t allow_lds(const void* kern, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  const hipError_t err = hipGetDevice(&dev);
  if (err != hipSuccess) return err;
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  const hipError_t raised = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (raised == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return raised;
}

template <int DT, bool E8, int C, int NC, bool ONCE, int W>
hipError_t attend_stream_go(const AttendArgs& a, unsigned grid, hipStream_t s) {
  constexpr size_t waves = static_cast<size_t>(W) * NC * (C * 16 + 2) * 64 * 4;
  auto* kern = &attend_kernel<DT, E8, C, NC, ONCE, W>;
  if constexpr (waves > 64 * 1024) {
    static std::atomic<uint64_t> done{0};
    const hipError_t raised = allow_lds(reinterpret_cast<const void*>(kern), waves, done);
    if (raised != hipSuccess) return raised;
  }
  kern<<<grid, 64 * W, waves, s>>>(a);
  return hipGetLastError();
}

// Where a tile holds all of a sequence's columns its keys and values are read by no other tile of the sequence and need not
// stay in the caches: from memory 64 tokens over 288352, 16 heads of 128 over 4 in 8 bits, take 62 to 64 us so and 70 to 72
// otherwise, 32 windows of 1024 in 16 bits 51.4 and 58.5; what the Infinity Cache holds takes the same. Rounds of 42 rows,
// three tiles of which read the same, are slower so: 16.6 against 15.6 us. So are sequences that share most of their pages,
// which sizes do not tell: 64 tokens after 4600 of which 4096 are the same 38.3 against 37.1 us (57.5 and 65.4 where nothing
// is), 256 after 2100, 2048 the same, 58 against 54, 32 after 2300 in 16 bits and 16 key heads, 2048 the same, 46 against 39.
template <int DT, bool E8, int C, int NC>
hipError_t attend_stream(const AttendArgs& a, unsigned grid, hipStream_t s) {
  const bool once = static_cast<int64_t>(a.rows.max_rows) * a.group <= 16 * NC;
  constexpr int wide = NC == 1 ? attend_wide(E8, C) : kWaves;
  if constexpr (wide > kWaves) {
    if (a.wide && once) return attend_stream_go<DT, E8, C, NC, true, wide>(a, grid, s);
    if (a.wide) return attend_stream_go<DT, E8, C, NC, false, wide>(a, grid, s);
  }
  return once ? attend_stream_go<DT, E8, C, NC, true, kWaves>(a, grid, s) : attend_stream_go<DT, E8, C, NC, false, kWaves>(a, grid, s);
}

template <int DT, bool E8, int C, int NC>
hipError_t attend_tiled(const AttendArgs& a, unsigned grid, hipStream_t s) {
  constexpr size_t sets = static_cast<size_t>(attend_sets(C)) * attend_set_bytes(C);
  auto* kern = &attend_tile_kernel<DT, E8, C, NC>;
  if constexpr (sets >= 64 * 1024) {  // with what the kernel has besides
    static std::atomic<uint64_t> done{0};
    const hipError_t raised = allow_lds(reinterpret_cast<const void*>(kern), sets, done);
    if (raised != hipSuccess) return raised;
  }
  kern<<<grid, 64 * kWaves, sets, s>>>(a);
  return hipGetLastError();
}

template <int DT, bool E8, int C>
hipError_t attend_columns(const AttendArgs& a, int columns, unsigned grid, hipStream_t s) {
  if (columns == 16) return attend_stream<DT, E8, C, 1>(a, grid, s);
  if (columns == 64) return attend_tiled<DT, E8, C, 1>(a, grid, s);
  if constexpr (C <= 2) {  // of longer heads so many columns' sums do not fit the registers
    if (columns == 32) return attend_stream<DT, E8, C, 2>(a, grid, s);
    if (columns == 128) return attend_tiled<DT, E8, C, 2>(a, grid, s);
  }
  return hipErrorInvalidValue;
}

template <int DT, bool E8>
hipError_t attend_pick(const AttendArgs& a, int columns, unsigned grid, hipStream_t s) {
  switch (a.cache.chunks) {
    case 1: return attend_columns<DT, E8, 1>(a, columns, grid, s);
    case 2: return attend_columns<DT, E8, 2>(a, columns, grid, s);
    case 3: return attend_columns<DT, E8, 3>(a, columns, grid, s);
    case 4: return attend_columns<DT, E8, 4>(a, columns, grid, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace plm
