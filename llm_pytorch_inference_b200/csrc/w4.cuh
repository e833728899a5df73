// Layout of 4-bit weights, shared by their makers, their reader and the products with them.
//
// A weight of row n, column k stands for scale (code - zero): code and zero in 0 .. 15, scale in bf16, one scale and
// zero per row and group of 32, 64 or 128 columns.  A record holds 16 rows by 128 columns: 64 bytes of codes
// a row, then for each row a 32-bit word per group, the scale's bits below the bf16 number 128 + zero.
//
// Column k of a record is nibble kNibble(k % 8) of the row's word (k / 32, t = k / 8 % 4), which is word k / 32 of the
// row's 16 bytes at place t ^ (row / 2 % 4).
//   * A word covers 8 consecutive columns, the 4 words of one i a row's 32: what lane t of a quad holds for one step of
//     the matrix instruction, so that groups of 32 columns are whole steps, and the rows' operand is 16 or 8
//     consecutive bytes of a row of activations.
//   * (word >> 4 j) & 0x000f000f is columns 2 j and 2 j + 1, in the places of a pair of 16-bit numbers, and
//     | 0x43004300 makes the pair 128 + code in bf16.
//   * The places are swapped by the row, so that 8 threads that read the same 16 bytes of 8 rows touch all banks.
// Records of 128 rows stand together: for each 128 columns the 8 of those rows (behind the last whole 128 rows those
// that are left), one contiguous copy of up to 8 records.  Everything behind the last row or column is zero.
#pragma once

#include <cstdint>

namespace mvb {

constexpr int kW4Rows = 16;
constexpr int kW4Cols = 128;
constexpr int kW4CodeBytes = kW4Rows * kW4Cols / 2;

__host__ __device__ constexpr int w4_record_bytes(int group) { return kW4CodeBytes + kW4Rows * (kW4Cols / group) * 4; }

// Where the record of the 16 rows `tile`, columns 128 block .. + 127 begins, in records.
__host__ __device__ inline int64_t w4_record(int tile, int block, int tiles, int blocks) {
  const int first = tile & ~7;
  const int together = tiles - first < 8 ? tiles - first : 8;
  return static_cast<int64_t>(first) * blocks + static_cast<int64_t>(block) * together + (tile - first);
}

__host__ __device__ constexpr int w4_place(int t, int row) { return t ^ (row >> 1 & 3); }

// The 8 codes of a word in the order of the columns, from nibbles in the order of the word, and back.
__host__ __device__ constexpr int w4_nibble(int column) { return (column & 1) * 4 + (column >> 1); }

}  // namespace mvb
