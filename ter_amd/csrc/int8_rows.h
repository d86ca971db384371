// int8_rows.h -- where the products' buffer loads of rows in 8 bits are, for the
// device and (tests) the host: integer arithmetic only.
//
// One resource covers the rows at hand, from the first value of the first to the
// last of the last.  The hardware checks a load's vector and immediate offsets
// against its size, not the scalar one.  So a load's whole way into the rows is in
// its vector offset: where that is at or behind the size, as of units behind K,
// the load gives zeros and reads nothing.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define TER_I8_HD __host__ __device__ __forceinline__
#else
#define TER_I8_HD inline
#endif

namespace terhip {

constexpr int kI8Unit = 128;  // K is padded to this

// Bytes from the first value of `rows` rows of Kx, ldx apart, to the last.
TER_I8_HD unsigned i8_rows_size(int rows, int ldx, int Kx) { return (unsigned)((rows - 1) * ldx + Kx); }

// 16 bytes of a row's unit u, 64-byte half t of it, for a lane whose 16 bytes of
// unit 0 and half 0 are at `lane_at`.
TER_I8_HD unsigned i8_rows_at(unsigned lane_at, int u, int t) { return lane_at + (unsigned)(u * kI8Unit + t * 64); }

// Few rows: row m, chunk g of a half.  Rows behind the last: the last one's loads,
// whose sums nobody stores.
TER_I8_HD unsigned i8_stream_lane(int m, int g, int rows, int ldx) {
    return (unsigned)((m < rows ? m : rows - 1) * ldx + g * 16);
}

// Tiles: row `row` of a tile, 128 bytes of which 8 lanes load, each the chunk of 16
// that belongs at its place in LDS.
TER_I8_HD int i8_swizzle(int row) { return (row & 7) ^ (row >> 3 & 1); }
TER_I8_HD unsigned i8_tile_lane(int row, int lane, int ldx) {
    return (unsigned)(row * ldx + ((lane & 7) ^ i8_swizzle(row)) * 16);
}

}  // namespace terhip
