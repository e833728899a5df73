// Products of few rows with 4-bit weights: y[m, n] = sum_g scale[n, g] sum_{k in g} (code[n, k] - zero[n, g]) x[m, k].
//
// x in bf16, or in 8 bits with a scale a[m] per row (q8_rows.cu), which multiplies the result.
//
// Bound by the weights' bytes (0.53 a weight in groups of 128): at the memory's rate an SM gets 44 weights a cycle and
// has 128 lanes to unpack them.  So the products run in whole numbers, where a mask unpacks four codes at once (six
// operations for the sixteen codes that a lane gives to a step of the matrix instruction; as bf16 numbers they took 22):
// mma.sync with 16 weight rows by 32 columns, 8 columns of rows of x, 32-bit sums, exact.  The zeros go out of the
// group's sum: sum (code - zero) q = sum code q - zero sum q.
//
// A bf16 row is taken apart into four rows of 8 bits, by group: with 2^E the size of the group's largest element and
// U = 2^(E - 21), x = U (2^16 q0 + 2^8 q1 + q2 + 2^-7 q3) + r, the first three the digits of -128 .. 127 of the nearest
// whole number.  That is exact for elements from 2^(E - 21) on.  What it leaves of those below, r (bf16 holds it), is added
// element by element (left_out): so how far a result is off depends on what its products are, not on a large element that
// meets a zero weight.  In ordinary rows some two groups in ten thousand leave an r.  A row's digits lie in one lane (of an odd
// tile's rows, in two); its sums 2^8 q0 + q1 and 2^7 q2 + q3 are whole numbers, which are scaled and added in 32 bits.  A group
// with an infinity or a NaN gives NaN.
//
// A block works on pairs of 16 weight rows.  Its warps split the columns; each is a worker with a ring of its own,
// into which one bulk copy brings the records of both tiles for 128 columns.  x lies in shared memory in the order of
// the lanes.  The warps' sums of a pair meet in shared memory and are added in the order of the warps.  A cluster of
// up to 8 blocks splits the columns further, where few weight rows would leave SMs idle or x would not fit; its sums
// meet in distributed shared memory, in the order of the blocks.  So every result is the same on every call.
//
// Measured, groups of 128: one bf16 row by 151936 x 4096 55.3 us (49.4 at the rate of a copy), 24576 x 4096 14.2 (8.0), 4096 x
// 4096 6.4, 2048 x 1024 4.4; 8 rows by 24576 x 4096 22.7, 4096 x 4096 9.7.  The long ones stream; 24576 x 4096 gives an SM 5 or 6
// pairs and issues in half of the slots on average, start and end included; the short ones are their launch, x and a chain of
// latencies.  Beside a column of 1e4 times the others' size 24576 x 4096 takes 14.2 us with 1 row and 25.8 with 8, beside one of 1e6
// 17.5 and 46.3.
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "host.h"
#include "w4.cuh"
#include "w4_linear.h"
#include "w4_ring.h"

namespace mvb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kRound = 16;  // pairs after which the blocks of a cluster add up
constexpr int kMaxCluster = 8;
constexpr int kMaxStages = 8;
// What a pair's end (sums through shared memory, one barrier, the results) takes, in items of 128 columns.  Against 1.5:
// 24576 x 4096 14.3 us and 15.1, 151936 x 4096 55.9 and 54.6, one row.
constexpr double kPairEnd = 3.0;
constexpr size_t kMostSmem = 227 * 1024;

struct LinearArgs {
  __nv_bfloat16* y;
  int64_t ldy;
  const void* x;
  int64_t ldx;
  const float* a;  // scales of the rows of x
  const uint8_t* records;
  int rows, n, k;
  int tiles, blocks, pairs;  // 16-row tiles, 128-column blocks, pairs of tiles
  int cluster, split;        // blocks of a cluster; warps that share a pair's columns
  int stages;                // items of a warp's ring
  unsigned* err;
};

__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared memory, from its start: flags; barriers [warp][stages]; the rings [warp][stages][2 records]; x; what the
// groups of x need; what its digits leave out; the warps' sums; the cluster's sums.
// Digits D: 1 for rows of 8 bits, 4 for bf16.
template <int GROUP, int D, int NT>
struct Layout {
  static constexpr int PER = kW4Cols / GROUP;
  static constexpr int REC = w4_record_bytes(GROUP);
  static constexpr int ROWS = 8 * NT / D;                      // the most rows of x
  static constexpr int WHOLE = D == 1 ? ROWS : NT / 2 * 4;     // of them those with one column of sums; others have two
  static constexpr int COLS = 2 * ROWS - WHOLE;                // columns of a warp's sums of a pair
  static constexpr int PER_LANE = COLS / 4;                    // of them a lane has so many, for 4 weight rows
  static constexpr int PITCH = D == 1 ? 36 : 40;               // floats between columns: 4 of them by 8 rows touch all banks
  static constexpr int SUMS = COLS * PITCH;
  static constexpr int X_BLOCK = NT * 1024;                    // bytes of x per 128 columns
  static constexpr int INFO_BLOCK = PER * ROWS * (D == 1 ? 4 : 16);
  static constexpr int LEFT_ROWS = (ROWS + 3) / 4 * 4;         // in whole 16 bytes
  static constexpr int LEFT_BLOCK = D == 1 ? 0 : LEFT_ROWS * 4;
  static constexpr int AHEAD = D == 1 ? 4 : 1;                 // pieces of 8 columns of x that a thread asks for at a time
  static constexpr int FIXED = 128 + kWarps * kMaxStages * 8;
  static_assert(FIXED % 16 == 0 && REC % 16 == 0 && X_BLOCK % 16 == 0 && INFO_BLOCK % 16 == 0 && LEFT_BLOCK % 16 == 0 &&
                    SUMS % 4 == 0 && PITCH % 4 == 0 && COLS % 4 == 0,
                "what is read by 16 bytes");
  // Column i of a lane, t = lane % 4.
  __device__ static int column(int t, int i) { return D == 1 ? (i >> 1) * 8 + 2 * t + (i & 1) : t + 4 * i; }
  // The first column of a row's sums, and the row of a column.
  __device__ static int column_of(int m) { return m < WHOLE ? m : 2 * m - WHOLE; }
  __device__ static int row_of(int column) { return column < WHOLE ? column : (column + WHOLE) >> 1; }
  // Column of the product that has digit z of row m: columns 2 t and 2 t + 1 of a tile are two digits of a row.
  __device__ static int place(int m, int z) {
    if (D == 1) return m;
    if (m >= WHOLE) return (NT - 1) * 8 + 4 * (m - WHOLE) + z;
    return (2 * (m >> 2) + (z >> 1)) * 8 + 2 * (m & 3) + (z & 1);
  }
  int most;  // 128-column blocks of a block
  int stages;
  bool cluster;
  __host__ __device__ constexpr size_t ring() const { return FIXED; }
  __host__ __device__ constexpr size_t x() const { return ring() + static_cast<size_t>(kWarps) * stages * 2 * REC; }
  __host__ __device__ constexpr size_t info() const { return x() + static_cast<size_t>(most) * X_BLOCK; }
  __host__ __device__ constexpr size_t left() const { return info() + static_cast<size_t>(most) * INFO_BLOCK; }
  __host__ __device__ constexpr size_t red() const { return left() + static_cast<size_t>(most) * LEFT_BLOCK; }
  __host__ __device__ constexpr size_t part() const { return red() + 2 * kWarps * SUMS * 4; }
  __host__ __device__ constexpr size_t bytes() const { return part() + (cluster ? kRound * ROWS * PITCH * 4 : 0); }
};

// What a group of a row of x needs beside its codes.  Rows of 8 bits: their sum, an int.  Digits:
struct Info {
  int high, low;  // the sums of 2^8 q0 + q1 and of 2^7 q2 + q3
  float scale;    // 2^8 U, what the first are times; the second are times 2^-15 of that
  int pad;
};

// The columns' order of a word's bytes: 0 4 1 5, then 2 6 3 7.
__device__ __forceinline__ uint2 ordered(uint32_t lo, uint32_t hi) {
  return make_uint2(__byte_perm(lo, hi, 0x5140), __byte_perm(lo, hi, 0x7362));
}
// Byte `at` of each of four words.
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int at) {
  return __byte_perm(__byte_perm(a, b, at | (at + 4) << 4), __byte_perm(c, d, at | (at + 4) << 4), 0x5410);
}

// Two elements of bf16: the nearest whole numbers of U as the low bits of f, of U / 128 what that leaves as those of g, and
// what is left.  A multiply-add rounds, and another is exact, whatever the elements' sizes.
__device__ __forceinline__ void digits_of(uint32_t two, float unit, float inv, float2& f, float2& g, float2& left) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23; whole numbers are below 2^22
  const float2 magic = make_float2(kMagic, kMagic), less = make_float2(-kMagic, -kMagic);
  const float2 x = make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
  const float u = 0.0078125f * unit, i = 128.0f * inv;
  f = __ffma2_rn(x, make_float2(inv, inv), magic);
  left = __ffma2_rn(__fadd2_rn(f, less), make_float2(-unit, -unit), x);
  g = __ffma2_rn(left, make_float2(i, i), magic);
  left = __ffma2_rn(__fadd2_rn(g, less), make_float2(-u, -u), left);
}
__device__ __forceinline__ bool is_some(float left) { return (__float_as_uint(left) & 0x7fffffffu) != 0; }

// What a row's 128 columns leave out: 0 where nothing; where one element leaves something, that in bf16 above its
// column; else a bit for each piece of 8 columns that does.
__device__ __forceinline__ bool is_one(uint32_t left) { return left >> 16 != 0; }

// x of this block's columns into shared memory: for each 128 columns, tile of 8 columns of the product, pair of steps of 32 columns
// and lane 16 bytes, 8 a step.  The lane's column of the product is lane / 4, its columns of x 8 (lane % 4) .. + 7 of
// the step's.  Returns whether this thread has noted elements that the digits do not hold.
template <int GROUP, int D, int NT>
__device__ __forceinline__ bool stage_x(uint8_t* sx, uint8_t* info, uint32_t* left, const LinearArgs& a, int block0,
                                        int blocks) {
  using L = Layout<GROUP, D, NT>;
  constexpr int LANES = GROUP / 8;
  const int chunks = blocks * 16, n = a.rows * chunks;
  const int lane = threadIdx.x & 31;
  bool noted = false;
  if (D > 1)  // rows that are not there leave nothing
    for (int i = threadIdx.x; i < blocks * L::LEFT_ROWS; i += kThreads)
      if (i % L::LEFT_ROWS >= a.rows) left[i] = 0;
  // 8-bit rows: four chunks a thread are asked for at a time (16 by 4096 x 4096 11.8 us for one, 10.5 for four).  Taking a
  // bf16 row apart is longer than its wait, and four were the same.
  using Raw = std::conditional_t<D == 1, uint2, uint4>;
  constexpr int AHEAD = L::AHEAD;
  Raw raw[AHEAD];
#pragma unroll 1
  for (int first = threadIdx.x & ~31; first < n; first += AHEAD * kThreads) {  // whole warps, for the exchanges
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = first + u * kThreads + lane, m = i / chunks, c = i - m * chunks;
      const int col = block0 * kW4Cols + 8 * c;
      raw[u] = Raw{};
      if (i < n && col < a.k)
        raw[u] = *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(a.x) + (m * a.ldx + col) * (D == 1 ? 1 : 2));
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i0 = first + u * kThreads;
      if (i0 >= n) break;
      const int i = i0 + lane, m = i / chunks, c = i - m * chunks;
      uint32_t q[D][2];
      float scale = 0.0f;
      if constexpr (D == 1) {
        const uint2 o = ordered(raw[u].x, raw[u].y);
        q[0][0] = o.x, q[0][1] = o.y;
      } else {
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(w[e] << 16 & 0x7fff0000u, w[e] & 0x7fff0000u));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool fine = top < 0x7f800000u;
        const uint32_t exponent = max(top >> 23, 29u);  // of 2^E; U / 128 and 128 / U are normal numbers
        const float unit = __uint_as_float((exponent - 21) << 23), inv = __uint_as_float((275 - exponent) << 23);
        scale = fine ? 256.0f * unit : __uint_as_float(0x7fc00000u);
        uint32_t b[8], last[8], some = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float2 f, g, rest;
          digits_of(fine ? w[e] : 0u, unit, inv, f, g, rest);
          // the digits' bytes, 128 above them each: the number is 0x400000 above itself
          b[2 * e] = __float_as_uint(f.x) + 0x408080u, b[2 * e + 1] = __float_as_uint(f.y) + 0x408080u;
          last[2 * e] = __float_as_uint(g.x), last[2 * e + 1] = __float_as_uint(g.y);
          some |= __float_as_uint(rest.x) | __float_as_uint(rest.y);
        }
#pragma unroll
        for (int z = 0; z < 3; ++z) {
          q[z][0] = bytes_of(b[0], b[4], b[1], b[5], 2 - z) ^ 0x80808080u;
          q[z][1] = bytes_of(b[2], b[6], b[3], b[7], 2 - z) ^ 0x80808080u;
        }
        q[3][0] = bytes_of(last[0], last[4], last[1], last[5], 0);
        q[3][1] = bytes_of(last[2], last[6], last[3], last[7], 0);
        const uint32_t pieces = __ballot_sync(0xffffffffu, (some & 0x7fffffffu) != 0) >> (lane & 16) & 0xffffu;
        uint32_t entry = pieces;
        if (some & 0x7fffffffu) {
          noted = true;
          int count = 0;
          uint32_t one = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float2 f, g, rest;
            digits_of(w[e], unit, inv, f, g, rest);
            if (is_some(rest.x)) ++count, one = (__float_as_uint(rest.x) & 0xffff0000u) | (8 * (c & 15) + 2 * e);
            if (is_some(rest.y)) ++count, one = (__float_as_uint(rest.y) & 0xffff0000u) | (8 * (c & 15) + 2 * e + 1);
          }
          if (count == 1 && (pieces & (pieces - 1)) == 0) entry = one;
        }
        // written by the first piece that leaves something
        if (i < n && (lane & 15) == (pieces ? __ffs(pieces) - 1 : 0)) left[(c >> 4) * L::LEFT_ROWS + m] = entry;
      }
      int sum[D];
#pragma unroll
      for (int z = 0; z < D; ++z)
        sum[z] = __dp4a(static_cast<int>(q[z][0]), 0x01010101, __dp4a(static_cast<int>(q[z][1]), 0x01010101, 0));
      int high = sum[0], low = 0;
      if (D > 1) high = 256 * sum[0] + sum[1 % D], low = 128 * sum[2 % D] + sum[3 % D];
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) {
        high += __shfl_xor_sync(0xffffffffu, high, o);
        if (D > 1) low += __shfl_xor_sync(0xffffffffu, low, o);
      }
      if (i < n) {
#pragma unroll
        for (int z = 0; z < D; ++z) {
          const int v = L::place(m, z), nt = v >> 3, b = c >> 4, step = c >> 2 & 3;
          *reinterpret_cast<uint2*>(sx + (((b * NT + nt) * 2 + (step >> 1)) * 32 + (v & 7) * 4 + (c & 3)) * 16 + (step & 1) * 8) =
              make_uint2(q[z][0], q[z][1]);
        }
        if (c % LANES == 0) {
          const int at = c / LANES * L::ROWS + m;
          if (D == 1) reinterpret_cast<int*>(info)[at] = high;
          else reinterpret_cast<Info*>(info)[at] = {high, low, scale, 0};
        }
      }
    }
  }
  return noted;
}

// One item: the records of both tiles at `rec`, 128 columns of x.  acc[s][h][i]: tile s, weight row lane / 4 + 8 h, column i
// of the lane.
template <int GROUP, int D, int NT>
__device__ __forceinline__ void compute(const uint8_t* rec, const uint8_t* sx, const uint8_t* info, int block, int lane,
                                        float (&acc)[2][2][Layout<GROUP, D, NT>::PER_LANE]) {
  using L = Layout<GROUP, D, NT>;
  constexpr int PER = L::PER, STEPS = 4 / PER;  // steps of 32 columns in a group
  const int g = lane >> 2, t = lane & 3;
  uint32_t words[2][2][4], pairs[2][2][PER];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* row = rec + s * L::REC + (g + 8 * h) * 64 + w4_place(t, g) * 16;
      const uint4 v = *reinterpret_cast<const uint4*>(row);
      words[s][h][0] = v.x, words[s][h][1] = v.y, words[s][h][2] = v.z, words[s][h][3] = v.w;
      const uint8_t* p = rec + s * L::REC + kW4CodeBytes + (g + 8 * h) * PER * 4;
#pragma unroll
      for (int i = 0; i < PER; ++i) pairs[s][h][i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
  const uint4* xb = reinterpret_cast<const uint4*>(sx) + block * NT * 64 + lane;
  const uint8_t* ib = info + block * L::INFO_BLOCK;
#pragma unroll
  for (int grp = 0; grp < PER; ++grp) {
    int d[2][NT][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q) d[s][nt][q] = 0;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int i = grp * STEPS + st;
      uint32_t a[2][4];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        a[s][0] = words[s][0][i] & 0x0f0f0f0fu;
        a[s][1] = words[s][1][i] & 0x0f0f0f0fu;
        a[s][2] = words[s][0][i] >> 4 & 0x0f0f0f0fu;
        a[s][3] = words[s][1][i] >> 4 & 0x0f0f0f0fu;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint2 b = reinterpret_cast<const uint2*>(xb + (nt * 2 + (i >> 1)) * 32)[i & 1];
#pragma unroll
        for (int s = 0; s < 2; ++s) mma_u8s8(d[s][nt], a[s][0], a[s][1], a[s][2], a[s][3], b.x, b.y);
      }
    }
    auto zero_of = [&](int s, int h) { return static_cast<int>(pairs[s][h][grp] >> 16 & 15u); };
    auto scale_of = [&](int s, int h) { return __uint_as_float(pairs[s][h][grp] << 16); };
    if constexpr (D == 1) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int2 f = *reinterpret_cast<const int2*>(ib + (grp * L::ROWS + nt * 8 + 2 * t) * 4);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int v = d[s][nt][q] - zero_of(s, q >> 1) * (q & 1 ? f.y : f.x);
            float& sum = acc[s][q >> 1][nt * 2 + (q & 1)];
            sum = fmaf(scale_of(s, q >> 1), static_cast<float>(v), sum);
          }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NT / 2; ++i) {
        const Info f = reinterpret_cast<const Info*>(ib)[grp * L::ROWS + t + 4 * i];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int zero = zero_of(s, h);
            const int high = d[s][2 * i][2 * h] * 256 + d[s][2 * i][2 * h + 1] - zero * f.high;
            const int low = d[s][2 * i + 1][2 * h] * 128 + d[s][2 * i + 1][2 * h + 1] - zero * f.low;
            const float v = fmaf(static_cast<float>(low), 0x1p-15f, static_cast<float>(high));
            acc[s][h][i] = fmaf(scale_of(s, h) * f.scale, v, acc[s][h][i]);
          }
      }
      if constexpr (NT & 1) {  // two lanes of a quad have the first and the last two digits of a row
        constexpr int LAST = NT - 1;
        const Info f = reinterpret_cast<const Info*>(ib)[grp * L::ROWS + L::WHOLE + (t >> 1)];
        const bool low = t & 1;
        const int by = low ? 128 : 256, of = low ? f.low : f.high;
        const float unit = low ? 0x1p-15f * f.scale : f.scale;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int v = d[s][LAST][2 * h] * by + d[s][LAST][2 * h + 1] - zero_of(s, h) * of;
            float& sum = acc[s][h][L::PER_LANE - 1];
            sum = fmaf(scale_of(s, h) * unit, static_cast<float>(v), sum);
          }
      }
    }
  }
}

// What a row's digits leave out, `left`, adds to a pair's sums: in lane i to those of its weight row i.  x: the row's 128
// columns.  Code less zero, times the scale, is exact in 32 bits.
template <int GROUP, int ROWS>
__device__ __forceinline__ float left_sum(const uint8_t* rec, uint32_t left, const __nv_bfloat16* x, const Info* info) {
  constexpr int PER = kW4Cols / GROUP, REC = w4_record_bytes(GROUP);
  const int lane = threadIdx.x & 31, row = lane & 15;
  const uint8_t* tile = rec + (lane >> 4) * REC;
  auto word_of = [&](int piece) {
    return *reinterpret_cast<const uint32_t*>(tile + row * 64 + w4_place(piece & 3, row) * 16 + (piece >> 2) * 4);
  };
  auto pair_of = [&](int piece) {
    return *reinterpret_cast<const uint32_t*>(tile + kW4CodeBytes + (row * PER + piece / (GROUP / 8)) * 4);
  };
  auto weight_of = [&](uint32_t word, int column, uint32_t pair) {
    const int code = word >> (4 * w4_nibble(column)) & 15u, zero = pair >> 16 & 15u;
    return __uint_as_float(pair << 16) * static_cast<float>(code - zero);
  };
  if (is_one(left)) {
    const int piece = left >> 3 & 15u;
    return weight_of(word_of(piece), left & 7u, pair_of(piece)) * __uint_as_float(left & 0xffff0000u);
  }
  float2 rest[4];  // of piece `lane`
#pragma unroll
  for (int e = 0; e < 4; ++e) rest[e] = make_float2(0.0f, 0.0f);
  if (left >> lane & 1u) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + 8 * lane);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const uint32_t exponent = (__float_as_uint(info[lane / (GROUP / 8) * ROWS].scale) >> 23) - 8;  // the unit's
    const float unit = __uint_as_float(exponent << 23), inv = __uint_as_float((254 - exponent) << 23);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 f, g;
      digits_of(w[e], unit, inv, f, g, rest[e]);
    }
  }
  float sum = 0.0f;
#pragma unroll 1
  for (; left; left &= left - 1) {
    const int piece = __ffs(left) - 1;
    const uint32_t word = word_of(piece), pair = pair_of(piece);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float r = __shfl_sync(0xffffffffu, e & 1 ? rest[e >> 1].y : rest[e >> 1].x, piece);
      if (is_some(r)) sum = fmaf(weight_of(word, e, pair), r, sum);
    }
  }
  return sum;
}

// What an item's rows leave out, added up in shared memory where a warp's sums of the pair will be; `had`: the rows that have
// left something in this pair.  x: the first row, at the item's columns.
template <int GROUP, int D, int NT>
__device__ __forceinline__ void left_out(const uint8_t* rec, const uint32_t* left, const __nv_bfloat16* x, int64_t ldx,
                                         const Info* info, float* out, int lane, uint32_t& had) {
  using L = Layout<GROUP, D, NT>;
  uint32_t rows = 0;
#pragma unroll
  for (int i = 0; i < L::LEFT_ROWS / 4; ++i) {
    const uint4 l = reinterpret_cast<const uint4*>(left)[i];
    rows |= ((l.x ? 1u : 0u) | (l.y ? 2u : 0u) | (l.z ? 4u : 0u) | (l.w ? 8u : 0u)) << 4 * i;
  }
#pragma unroll 1
  for (; rows; rows &= rows - 1) {  // the same in all lanes
    const int m = __ffs(rows) - 1;
    const float sum = left_sum<GROUP, L::ROWS>(rec, left[m], x + m * ldx, info + m);
    float* to = out + L::column_of(m) * L::PITCH + lane;
    *to = had >> m & 1u ? *to + sum : sum;
    had |= 1u << m;
  }
}

__device__ __forceinline__ void group_bar(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <int GROUP, int D, int NT>
__global__ void __launch_bounds__(kThreads, 1) w4_linear_kernel(const LinearArgs a) {
  using L = Layout<GROUP, D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int c = a.cluster, rank = static_cast<int>(blockIdx.x) % c, unit = static_cast<int>(blockIdx.x) / c;
  const int units = static_cast<int>(gridDim.x) / c;
  const int block0 = static_cast<int>(static_cast<int64_t>(rank) * a.blocks / c);
  const int blocks = static_cast<int>(static_cast<int64_t>(rank + 1) * a.blocks / c) - block0;
  const L at = {(a.blocks + c - 1) / c, a.stages, c > 1};
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem);
  int* lost = reinterpret_cast<int*>(smem) + 16 + wid;  // this warp's place whose wait gave up
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 128) + wid * kMaxStages;
  uint8_t* places = smem + at.ring() + static_cast<size_t>(wid) * a.stages * 2 * L::REC;
  uint8_t* sx = smem + at.x();
  uint8_t* info = smem + at.info();
  uint32_t* left = reinterpret_cast<uint32_t*>(smem + at.left());  // [blocks][LEFT_ROWS]
  float* red = reinterpret_cast<float*>(smem + at.red());    // [2][warp][SUMS]
  float* part = reinterpret_cast<float*>(smem + at.part());  // [kRound][ROWS][PITCH]

  // Pairs unit, unit + units, ..; of those this warp's team takes every teams-th, and of a pair's columns this
  // warp blocks kw, kw + split, ..
  const int split = a.split, teams = kWarps / split, team = wid / split, kw = wid % split;
  const int mine = unit < a.pairs ? (a.pairs - unit + units - 1) / units : 0;  // pairs of this block

  // The copies of this warp's items, lane 0's: the next one to ask for.
  W4Ring ring(team);
  int load_b = kw;
  uint64_t policy = 0;
  auto ask = [&]() {
    if (load_b >= blocks || ring.pair >= mine) return;  // (a warp without columns asks for none)
    const int tile = 2 * (unit + ring.pair * units);
    const int64_t r = w4_record(tile, block0 + load_b, a.tiles, a.blocks);
    // the last pair may lack its second tile: what its place holds then is computed with and not written
    const uint32_t bytes = (tile + 1 < a.tiles ? 2 : 1) * L::REC;
    mbar_arrive_expect_tx(&bars[ring.fill], bytes);
    copy_bulk(places + ring.fill * 2 * L::REC, a.records + r * L::REC, bytes, &bars[ring.fill], policy);
    ring.asked(a.stages);
    load_b += split;
    if (load_b >= blocks) load_b = kw, ring.pair += teams;
  };
  if (tid == 0) *abort_flag = 0;
  if (lane == 0) {
    for (int s = 0; s < a.stages; ++s) mbar_init(&bars[s], 1);
    fence_barrier_init();
    policy = l2_policy_evict_first();
    // weights are constant: their copies need not wait for the kernel before
    for (int s = 0; s < a.stages; ++s) ask();
  }
  pdl_launch_dependents();
  pdl_wait();
  // Whether the digits of all this block's rows hold them, which is usual: the loop without left_out then runs (with the branch
  // in it 4 by 24576 x 4096 took 20.2 us for 18.3).
  bool some_left = stage_x<GROUP, D, NT>(sx, info, left, a, block0, blocks);
  if (D > 1) some_left = __syncthreads_or(some_left) != 0;
  else __syncthreads();

  const int rounds = c > 1 ? (mine + kRound - 1) / kRound : 1;  // the same in every block of a cluster
  for (int round = 0; round < rounds; ++round) {
    const int j0 = c > 1 ? round * kRound : 0, j1 = c > 1 ? min(mine, j0 + kRound) : mine;
    int buf = 0;
    // kRound is a multiple of the teams, so a team's pairs of a round begin at j0 + team
    for (int j = j0 + team; j < j1; j += teams) {
      float acc[2][2][L::PER_LANE];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < L::PER_LANE; ++i) acc[s][h][i] = 0.0f;
      float* out = red + (buf * kWarps + wid) * L::SUMS;  // two pairs ago everybody had read it
      float* own = out + lane / 4;                        // of this lane's weight rows
      auto items = [&](auto with_left) {
        uint32_t had = 0;
        for (int b = kw; b < blocks; b += split) {
          // where it gives up the item is computed all the same, and the rest, so that all barriers are met
          if (!mbar_wait(&bars[ring.read], ring.phase, abort_flag, a.err) && lane == 0) ring.stop(*lost);
          const uint8_t* rec = places + ring.read * 2 * L::REC;
          compute<GROUP, D, NT>(rec, sx, info, b, lane, acc);
          if constexpr (decltype(with_left)::value)
            left_out<GROUP, D, NT>(rec, left + b * L::LEFT_ROWS,
                                   static_cast<const __nv_bfloat16*>(a.x) + (block0 + b) * kW4Cols, a.ldx,
                                   reinterpret_cast<const Info*>(info + b * L::INFO_BLOCK), out, lane, had);
          __syncwarp();  // every lane has read: the next copy may come
          if (lane == 0) ask();
          ring.next(a.stages);
        }
        if constexpr (decltype(with_left)::value) {
#pragma unroll
          for (int i = 0; i < L::PER_LANE; ++i) {
            const int col = L::column(lane & 3, i);
            const int m = L::row_of(col);
            if (col == L::column_of(m) && (had >> m & 1u))
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[r >> 1][r & 1][i] += own[col * L::PITCH + r * 8];
          }
          __syncwarp();  // all have read
        }
      };
      if (D > 1 && some_left) items(std::bool_constant<(D > 1)>());
      else items(std::false_type());
#pragma unroll
      for (int i = 0; i < L::PER_LANE; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) own[L::column(lane & 3, i) * L::PITCH + r * 8] = acc[r >> 1][r & 1][i];
      if (split > 1) group_bar(1 + team, 32 * split);
      else __syncwarp();
      const float* in = red + (buf * kWarps + team * split) * L::SUMS;
      const int pair = unit + j * units;
      for (int i = kw * 32 + lane; i < 32 * a.rows; i += 32 * split) {
        const int m = i >> 5, r = i & 31;
        float v = 0.0f;
        const float* of_row = in + L::column_of(m) * L::PITCH + r;
        const bool two = L::WHOLE < L::ROWS && m >= L::WHOLE;
        for (int w = 0; w < split; ++w) {
          v += of_row[w * L::SUMS];
          if (two) v += of_row[w * L::SUMS + L::PITCH];
        }
        if (c > 1) {
          part[((j - j0) * L::ROWS + m) * L::PITCH + r] = v;
        } else {
          const int col = pair * 32 + r;
          if (col < a.n) {
            if (D == 1) v *= a.a[m];
            a.y[m * a.ldy + col] = __float2bfloat16_rn(v);
          }
        }
      }
      buf ^= 1;
    }
    if (c > 1) {
      cluster_sync();
      const int n = (j1 - j0) * a.rows * 8;
      for (int i = rank * kThreads + tid; i < n; i += c * kThreads) {
        const int r = 4 * (i & 7), m = (i >> 3) % a.rows, j = (i >> 3) / a.rows;
        const int col = (unit + (j0 + j) * units) * 32 + r;
        const float4 v = dsmem_sum4(part + (j * L::ROWS + m) * L::PITCH + r, c);
        const float scale = D == 1 ? a.a[m] : 1.0f, y4[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col + k < a.n) a.y[m * a.ldy + col + k] = __float2bfloat16_rn(y4[k]);
      }
      cluster_sync();  // everybody has read: the sums may change, or their block end
    }
  }
  // Every copy has been waited for, unless a wait gave up: then those under way are, before the block ends.
  if (lane == 0 && ring.stopped()) {
    ring.back(*lost);
    do mbar_wait(&bars[ring.read], ring.phase, nullptr, a.err);
    while (ring.more(a.stages));
  }
}

template <int GROUP, int D, int NT>
int run(const char* name, LinearArgs a, cudaStream_t stream) {
  using L = Layout<GROUP, D, NT>;
  const int sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "%s: no device", name);
  auto kernel = w4_linear_kernel<GROUP, D, NT>;
  static std::atomic<uint64_t> done{0};
  MVB_TRY(set_smem_once(done, kernel, kMostSmem, name));
  // The warps that share a pair's columns: what a warp computes and what a pair's end takes, in items.
  auto split_of = [](int mine, int blocks, double& fewest) {
    int best = 0;
    for (int split = kWarps; split >= 1; split /= 2) {
      const int teams = kWarps / split;
      const double items = ((mine + teams - 1) / teams) * ((blocks + split - 1) / split + kPairEnd);
      if (best == 0 || items < fewest) fewest = items, best = split;
    }
    return best;
  };
  // The cluster, by what takes a block's time: its items and one for each pair's end, what its busiest warp does (5 each), x (8
  // for what its threads ask for at once, and 0.05 for 128 columns of a row) and a cluster's meeting (20).  Of 1, 2, 4 and 8 blocks
  // measured at 80 sizes that picks what is 0.4 % above the best on average, 5 % at most: 8 rows by 4096 x 4096, bf16, 12.9, 10.9,
  // 9.5 and 10.5 us, by 24576 x 4096 28.0, 22.7, 25.5 and 35.1; 1 row by 4096 x 4096 6.0, 6.6, 6.7 and 7.4.
  static PerDevice clusters[kMaxCluster + 1];
  auto units_of = [&](int c) {
    return c == 1 ? sms : clusters_at_once(clusters[c], kernel, c, kThreads, kMostSmem);
  };
  int best = 0;
  double least = 0;
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    const int units = units_of(c), blocks = (a.blocks + c - 1) / c, mine = (a.pairs + units - 1) / units;
    if (L{blocks, 1, c > 1}.bytes() > kMostSmem || c > a.blocks) continue;
    double warp = 0;
    const int split = split_of(mine, blocks, warp);
    const int of_x = a.rows * blocks, at_once = kThreads * L::AHEAD / 16;
    const double cost = double(mine) * (blocks + 1) + 5 * warp + (c > 1 ? 20 : 0) + 8 * ((of_x + at_once - 1) / at_once) +
                        0.05 * of_x;
    if (best == 0 || cost < least) best = c, least = cost, a.split = split;
  }
  MVB_REQUIRE(best > 0, "%s: %d columns", name, a.k);
  a.cluster = best;
  const int units = a.pairs < units_of(best) ? a.pairs : units_of(best);
  L at = {(a.blocks + best - 1) / best, kMaxStages, best > 1};
  while (at.bytes() > kMostSmem) --at.stages;
  a.stages = at.stages;
  const dim3 grid(static_cast<unsigned>(units * best));
  if (best == 1) return launch(name, kernel, grid, dim3(kThreads), at.bytes(), stream, a);
  return launch_cluster(name, kernel, grid, dim3(kThreads), static_cast<unsigned>(best), at.bytes(), stream, a);
}

// Whether shared memory holds x of these columns, a cluster's blocks sharing them.
template <int GROUP, int D, int NT>
constexpr bool fits(int blocks, int cluster) {
  return Layout<GROUP, D, NT>{(blocks + cluster - 1) / cluster, 1, true}.bytes() <= kMostSmem;
}

// As many columns of the product as the rows need; other calls go to tcgen05, `few` false.  A kernel here reads the records
// once.
//   8 rows of bf16, here and on tcgen05, where a cluster of 4 holds x: 24576 x 4096 22.8 us and 26.4, 4096 x 12288 18.8 and 19.8, in
//   groups of 32 21.4 and 23.0, 16384 x 8192 36.8 and 34.7.  A cluster of 8 leaves SMs idle, which few weight rows do not need:
//   4096 x 20480 26.8 and 26.0, in groups of 32 39.6 and 31.3; but 1024 x 20480 13.7 and 17.1, in groups of 32 16.6 and 21.3.
//   Up to 6 rows fit at any k: 4096 x 24576 26.8 and 28.6, in groups of 32 33.1 and 34.7, at worst (32768) 45.9 and 43.0.
//   16 rows of 8 bits: 24576 x 4096 20.2 and 24.8, 4096 x 12288 14.8 and 18.9, in groups of 32 18.0 and 26.4, at worst (4096 x
//   32768) 35.0 and 33.3; 20 by 24576 x 4096 36.0 and 24.8, 24 by 4096 x 4096 18.6 and 13.4.
template <int GROUP, bool Q8>
int run_few(const char* name, const LinearArgs& a, cudaStream_t stream, bool& few) {
  constexpr int MOST = 32768 / kW4Cols;
  few = true;
  if constexpr (Q8) {
    static_assert(fits<GROUP, 1, 2>(MOST, kMaxCluster), "16 rows");
    if (a.rows <= 8) return run<GROUP, 1, 1>(name, a, stream);
    if (a.rows <= 16) return run<GROUP, 1, 2>(name, a, stream);
  } else {
    static_assert(fits<GROUP, 4, 3>(MOST, kMaxCluster), "6 rows");
    if (a.rows <= 2) return run<GROUP, 4, 1>(name, a, stream);
    if (a.rows <= 4) return run<GROUP, 4, 2>(name, a, stream);
    if (a.rows <= 6) return run<GROUP, 4, 3>(name, a, stream);
    if (a.rows <= 8 && fits<GROUP, 4, 4>(a.blocks, a.pairs <= 64 ? kMaxCluster : 4)) return run<GROUP, 4, 4>(name, a, stream);
  }
  few = false;
  return MVB_OK;
}

template <bool Q8>
int run_group(const char* name, const LinearArgs& a, int64_t group, cudaStream_t stream, bool& few) {
  if (group == 32) return run_few<32, Q8>(name, a, stream, few);
  if (group == 64) return run_few<64, Q8>(name, a, stream, few);
  return run_few<128, Q8>(name, a, stream, few);
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_linear_w4(void* y, int64_t ldy, const void* x, int64_t ldx, const float* row_scales,
                             const void* records, int64_t rows, int64_t n, int64_t k, int64_t group,
                             mvb_stream_t stream) {
  const char* name = "mvb_linear_w4";
  MVB_REQUIRE(rows >= 0 && rows <= (1 << 18), "%s: %lld rows", name, (long long)rows);
  MVB_REQUIRE(n >= 0 && n <= (1 << 24), "%s: %lld weight rows", name, (long long)n);
  MVB_REQUIRE(k > 0 && k <= 32768 && k % 32 == 0, "%s: %lld columns (a multiple of 32, at most 32768)", name,
              (long long)k);
  MVB_REQUIRE(group == 32 || group == 64 || group == 128, "%s: groups of %lld columns (32, 64 or 128)", name,
              (long long)group);
  if (rows == 0 || n == 0) return MVB_OK;
  MVB_REQUIRE(y && x && records, "%s: null pointer", name);
  const int64_t e = row_scales != nullptr ? 1 : 2;
  MVB_REQUIRE(aligned(records, 16) && aligned(x, 16) && (rows == 1 || ldx * e % 16 == 0) && (rows == 1 || ldx >= k) &&
                  (rows == 1 || ldy >= n),
              "%s: records and rows of x on 16 bytes, rows %lld and %lld apart", name, (long long)ldx, (long long)ldy);
  LinearArgs a = {};
  a.y = static_cast<__nv_bfloat16*>(y);
  a.ldy = ldy;
  a.x = x;
  a.ldx = ldx;
  a.a = row_scales;
  a.records = static_cast<const uint8_t*>(records);
  a.rows = static_cast<int>(rows);
  a.n = static_cast<int>(n);
  a.k = static_cast<int>(k);
  a.tiles = (a.n + kW4Rows - 1) / kW4Rows;
  a.blocks = (a.k + kW4Cols - 1) / kW4Cols;
  a.pairs = (a.tiles + 1) / 2;
  a.err = device_status_ptr();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  bool few = false;
  MVB_TRY(row_scales != nullptr ? run_group<true>(name, a, group, st, few) : run_group<false>(name, a, group, st, few));
  if (few) return MVB_OK;
  const W4LinearCall call = {a.y, ldy, x, ldx, row_scales, a.records, a.rows, a.n, a.k, static_cast<int>(group)};
  return w4_gemm(name, call, st);
}
