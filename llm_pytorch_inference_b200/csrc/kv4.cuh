// Layout of the 4-bit paged KV pool, shared by its writer, its reader and the attention over it.
//
// The pool is uint8 [L, num_blocks, Hkv, block_size / 16, 18 D]: one record of 18 D contiguous bytes
// per 16 tokens of a KV head,
//   K codes [16][D / 2] | V codes [16][D / 2] | K pairs [16][D / 64] | V pairs [16][D / 64].
// A group of 64 channels of a token shares one pair (scale, min) of bf16; a code u in 0..15 stands
// for min + scale * u.  bf16 pairs have the range of the bf16 K and V that they come from, so no
// group overflows; their rounding is part of the definition (codes are chosen against the rounded
// pair), which leaves it at half a step of the code.
//
// One record is one contiguous copy (2,304 bytes at D = 128), whatever the block size.  Within a
// row the 32-bit words of the groups are interleaved: word NG * w + g holds channels
// 64 g + 8 w .. + 7, the lowest nibble first, so 16 consecutive bytes hold an equal share of
// every group and a lane of the attention reads its share of all groups with one vector load.
#pragma once

#include <cstdint>

namespace mvb {

constexpr int kKv4Tokens = 16;  // tokens of a record
constexpr int kKv4Group = 64;   // channels that share a pair

template <int D>
struct Kv4 {
  static constexpr int NG = D / kKv4Group;           // groups of a row
  static constexpr int ROW = D / 2;                  // bytes of a row of codes
  static constexpr int PAIRS = NG * 4;               // bytes of a row of pairs
  static constexpr int V_CODES = kKv4Tokens * ROW;   // byte offsets in the record
  static constexpr int K_PAIRS = 2 * kKv4Tokens * ROW;
  static constexpr int V_PAIRS = K_PAIRS + kKv4Tokens * PAIRS;
  static constexpr int RECORD = K_PAIRS + 2 * kKv4Tokens * PAIRS;
};

// Two fp32 numbers to an instruction, each rounded as by its own.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

}  // namespace mvb
