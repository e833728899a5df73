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
// A bf16 row is taken apart into three rows of 8 bits, by group: with 2^E the size of the group's largest element,
// x = 2^(E - 5) (q0 + 2^-7 q1 + 2^-14 q2), each the nearest whole number to what is left.  That is exact but for elements
// below 2^(E - 12), which are off by at most 2^(E - 20): as much as rounding a sum of the size of the group's largest
// product to 32 bits a few times.  A group's three sums are scaled and added in 32 bits; a group with an infinity or a NaN
// gives NaN.
//
// A block works on pairs of 16 weight rows.  Its warps split the columns; each is a worker with a ring of its own,
// into which one bulk copy brings the records of both tiles for 128 columns.  x lies in shared memory in the order of
// the lanes.  The warps' sums of a pair meet in shared memory and are added in the order of the warps.  A cluster of
// up to 8 blocks splits the columns further, where few weight rows would leave SMs idle or x would not fit; its sums
// meet in distributed shared memory, in the order of the blocks.  So every result is the same on every call.
//
// Measured, one row, groups of 128: 151936 x 4096 bf16 55.8 us (49.4 at the rate of a copy), 24576 x 4096 14.4 (8.0),
// 4096 x 4096 6.35, 2048 x 1024 4.6.  The long ones stream; 24576 x 4096 gives an SM 5 or 6 pairs and issues in 48 % of
// the slots on average, start and end included; the short ones are their launch, x and a chain of latencies.
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "host.h"
#include "w4.cuh"
#include "w4_linear.h"

namespace mvb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPitch = 36;  // floats between columns of a pair's 32 sums: 4 columns by 8 rows touch all banks
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

__device__ __forceinline__ void copy_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// Shared memory, from its start: barriers [warp][stages]; the rings [warp][stages][2 records]; x; what the
// groups of x need; the warps' sums; the cluster's sums.
template <int GROUP, int P, int NT>
struct Layout {
  static constexpr int PER = kW4Cols / GROUP;
  static constexpr int REC = w4_record_bytes(GROUP);
  static constexpr int ROWS = 8 * NT / P;        // rows of x of a block
  static constexpr int SUMS = 8 * NT * kPitch;   // floats of a warp's sums of a pair
  static constexpr int X_BLOCK = NT * 1024;      // bytes of x per 128 columns
  static constexpr int INFO_BLOCK = PER * 8 * NT * 8;
  static constexpr int FIXED = 128 + kWarps * kMaxStages * 8;
  int most;  // 128-column blocks of a block
  int stages;
  bool cluster;
  __host__ __device__ size_t ring() const { return FIXED; }
  __host__ __device__ size_t x() const { return ring() + static_cast<size_t>(kWarps) * stages * 2 * REC; }
  __host__ __device__ size_t info() const { return x() + static_cast<size_t>(most) * X_BLOCK; }
  __host__ __device__ size_t red() const { return info() + static_cast<size_t>(most) * INFO_BLOCK; }
  __host__ __device__ size_t part() const { return red() + 2 * kWarps * SUMS * 4; }
  __host__ __device__ size_t bytes() const { return part() + (cluster ? kRound * ROWS * kPitch * 4 : 0); }
};

// What a group of a row of x needs beside its codes: their sum, and what they are times.
struct Info {
  int sum;
  float scale;
};

// The columns' order of a word's bytes: 0 4 1 5, then 2 6 3 7.
__device__ __forceinline__ uint2 ordered(uint32_t lo, uint32_t hi) {
  return make_uint2(__byte_perm(lo, hi, 0x5140), __byte_perm(lo, hi, 0x7362));
}
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                     __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}

// x of this block's columns into shared memory: for each 128 columns, tile of 8 columns of the product, pair of steps of 32 columns
// and lane 16 bytes, 8 a step.  The lane's column of the product is lane / 4, its columns of x 8 (lane % 4) .. + 7 of
// the step's.  P: 8-bit rows that a row is taken apart into.
template <int GROUP, int P, int NT>
__device__ __forceinline__ void stage_x(uint8_t* sx, Info* info, const LinearArgs& a, int row0, int block0, int blocks) {
  using L = Layout<GROUP, P, NT>;
  constexpr int LANES = GROUP / 8;
  const int chunks = blocks * 16, rows = min(L::ROWS, a.rows - row0), n = rows * chunks;
  const int lane = threadIdx.x & 31;
  // 8-bit rows: four chunks a thread are asked for at a time (16 by 4096 x 4096 11.8 us for one, 10.5 for four).  Taking a
  // bf16 row apart is longer than its wait, and four were the same.
  using Raw = std::conditional_t<P == 1, uint2, uint4>;
  constexpr int AHEAD = P == 1 ? 4 : 1;
  Raw raw[AHEAD];
#pragma unroll 1
  for (int first = threadIdx.x & ~31; first < n; first += AHEAD * kThreads) {  // whole warps, for the exchanges
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = first + u * kThreads + lane, m = i / chunks, c = i - m * chunks;
      const int col = block0 * kW4Cols + 8 * c;
      raw[u] = Raw{};
      if (i < n && col < a.k)
        raw[u] = *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(a.x) + ((row0 + m) * a.ldx + col) * (P == 1 ? 1 : 2));
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i0 = first + u * kThreads;
      if (i0 >= n) break;
      const int i = i0 + lane, m = i / chunks, c = i - m * chunks;
      uint32_t q[P][2];
      float scale = 1.0f;
      if constexpr (P == 1) {
        q[0][0] = raw[u].x, q[0][1] = raw[u].y;
      } else {
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(w[e] << 16 & 0x7fff0000u, w[e] & 0x7fff0000u));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // 2^(E - 5), and its reciprocal; below 2^-105 nothing is told apart
        const uint32_t exponent = max(top >> 23, 22u);
        scale = top == 0 ? 0.0f : __uint_as_float((exponent - 5) << 23);
        const float inv = __uint_as_float((259 - exponent) << 23);
        const bool fine = top < 0x7f800000u;
        if (!fine) scale = __uint_as_float(0x7fc00000u);
        constexpr float kMagic = 12582912.0f;
        float p[3][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = fine ? __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16) * inv : 0.0f;
          p[0][e] = y + kMagic;
          const float r = (y - (p[0][e] - kMagic)) * 128.0f;
          p[1][e] = r + kMagic;
          p[2][e] = (r - (p[1][e] - kMagic)) * 128.0f + kMagic;
        }
#pragma unroll
        for (int z = 0; z < P; ++z) {
          q[z][0] = low_bytes(p[z % 3][0], p[z % 3][1], p[z % 3][2], p[z % 3][3]);
          q[z][1] = low_bytes(p[z % 3][4], p[z % 3][5], p[z % 3][6], p[z % 3][7]);
        }
      }
#pragma unroll
      for (int z = 0; z < P; ++z) {
        int sum = __dp4a(static_cast<int>(q[z][0]), 0x01010101, __dp4a(static_cast<int>(q[z][1]), 0x01010101, 0));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (i < n) {
          const int v = m * P + z, nt = v >> 3, b = c >> 4, step = c >> 2 & 3;
          *reinterpret_cast<uint2*>(sx + (((b * NT + nt) * 2 + (step >> 1)) * 32 + (v & 7) * 4 + (c & 3)) * 16 + (step & 1) * 8) =
              ordered(q[z][0], q[z][1]);
          if (c % LANES == 0)
            info[(c / LANES) * 8 * NT + v] = {sum, z == 0 ? scale : z == 1 ? scale * 0.0078125f : scale * 6.1035156e-5f};
        }
      }
    }
  }
}

// One item: the records of both tiles at `rec`, 128 columns of x.
template <int GROUP, int P, int NT>
__device__ __forceinline__ void compute(const uint8_t* rec, const uint8_t* sx, const Info* info, int block, int lane,
                                        float (&acc)[2][NT][4]) {
  using L = Layout<GROUP, P, NT>;
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
  const Info* ib = info + block * PER * 8 * NT + 2 * t;
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
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int4 f = *reinterpret_cast<const int4*>(ib + (grp * NT + nt) * 8);  // of columns 2 t and 2 t + 1
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t pair = pairs[s][q >> 1][grp];
          const int v = d[s][nt][q] - static_cast<int>(pair >> 16 & 15u) * (q & 1 ? f.z : f.x);
          float scale = __uint_as_float(pair << 16);
          if (P > 1) scale *= __int_as_float(q & 1 ? f.w : f.y);
          acc[s][nt][q] = fmaf(scale, static_cast<float>(v), acc[s][nt][q]);
        }
    }
  }
}

__device__ __forceinline__ void group_bar(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <int GROUP, int P, int NT>
__global__ void __launch_bounds__(kThreads, 1) w4_linear_kernel(const LinearArgs a) {
  using L = Layout<GROUP, P, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int c = a.cluster, rank = static_cast<int>(blockIdx.x) % c, unit = static_cast<int>(blockIdx.x) / c;
  const int units = static_cast<int>(gridDim.x) / c;
  const int row0 = blockIdx.y * L::ROWS;
  const int block0 = static_cast<int>(static_cast<int64_t>(rank) * a.blocks / c);
  const int blocks = static_cast<int>(static_cast<int64_t>(rank + 1) * a.blocks / c) - block0;
  const L at = {(a.blocks + c - 1) / c, a.stages, c > 1};
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 128) + wid * kMaxStages;
  uint8_t* ring = smem + at.ring() + static_cast<size_t>(wid) * a.stages * 2 * L::REC;
  uint8_t* sx = smem + at.x();
  Info* info = reinterpret_cast<Info*>(smem + at.info());
  float* red = reinterpret_cast<float*>(smem + at.red());    // [2][warp][SUMS]
  float* part = reinterpret_cast<float*>(smem + at.part());  // [kRound][ROWS][kPitch]

  // Pairs unit, unit + units, ..; of those this warp's team takes every teams-th, and of a pair's columns this
  // warp blocks kw, kw + split, ..
  const int split = a.split, teams = kWarps / split, team = wid / split, kw = wid % split;
  const int mine = unit < a.pairs ? (a.pairs - unit + units - 1) / units : 0;  // pairs of this block

  // The copies of this warp's items, lane 0's: the next one to ask for.
  int load_j = team, load_b = kw, load_at = 0;
  uint64_t policy = 0;
  auto ask = [&]() {
    if (load_b >= blocks || load_j >= mine) return;  // (a warp without columns asks for none)
    const int tile = 2 * (unit + load_j * units);
    const int64_t r = w4_record(tile, block0 + load_b, a.tiles, a.blocks);
    // the last pair may lack its second tile: what its place holds then is computed with and not written
    const uint32_t bytes = (tile + 1 < a.tiles ? 2 : 1) * L::REC;
    mbar_arrive_expect_tx(&bars[load_at], bytes);
    copy_bulk(ring + load_at * 2 * L::REC, a.records + r * L::REC, bytes, &bars[load_at], policy);
    load_at = load_at + 1 == a.stages ? 0 : load_at + 1;
    load_b += split;
    if (load_b >= blocks) load_b = kw, load_j += teams;
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
  stage_x<GROUP, P, NT>(sx, info, a, row0, block0, blocks);
  __syncthreads();

  int stage = 0;
  uint32_t phase = 0;
  const int rounds = c > 1 ? (mine + kRound - 1) / kRound : 1;  // the same in every block of a cluster
  for (int round = 0; round < rounds; ++round) {
    const int j0 = c > 1 ? round * kRound : 0, j1 = c > 1 ? min(mine, j0 + kRound) : mine;
    int buf = 0;
    // kRound is a multiple of the teams, so a team's pairs of a round begin at j0 + team
    for (int j = j0 + team; j < j1; j += teams) {
      float acc[2][NT][4];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[s][nt][q] = 0.0f;
      for (int b = kw; b < blocks; b += split) {
        mbar_wait(&bars[stage], phase, abort_flag, a.err);
        compute<GROUP, P, NT>(ring + stage * 2 * L::REC, sx, info, b, lane, acc);
        __syncwarp();  // every lane has read: the next copy may come
        if (lane == 0) ask();
        if (++stage == a.stages) stage = 0, phase ^= 1;
      }
      float* out = red + (buf * kWarps + wid) * L::SUMS;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            out[(nt * 8 + 2 * (lane & 3) + (q & 1)) * kPitch + s * 16 + (q >> 1) * 8 + (lane >> 2)] = acc[s][nt][q];
      if (split > 1) group_bar(1 + team, 32 * split);
      else __syncwarp();
      const float* in = red + (buf * kWarps + team * split) * L::SUMS;
      const int pair = unit + j * units;
      const int rows = min(L::ROWS, a.rows - row0);
      for (int i = kw * 32 + lane; i < 32 * rows; i += 32 * split) {
        const int m = i >> 5, r = i & 31;
        float v = 0.0f;
        for (int w = 0; w < split; ++w)
#pragma unroll
          for (int z = 0; z < P; ++z) v += in[w * L::SUMS + (m * P + z) * kPitch + r];
        if (c > 1) {
          part[((j - j0) * L::ROWS + m) * kPitch + r] = v;
        } else {
          const int row = row0 + m, col = pair * 32 + r;
          if (col < a.n) {
            if (P == 1) v *= a.a[row];
            a.y[row * a.ldy + col] = __float2bfloat16_rn(v);
          }
        }
      }
      buf ^= 1;
    }
    if (c > 1) {
      cluster_sync();
      const int rows = min(L::ROWS, a.rows - row0), n = (j1 - j0) * rows * 8;
      for (int i = rank * kThreads + tid; i < n; i += c * kThreads) {
        const int r = 4 * (i & 7), m = (i >> 3) % rows, j = (i >> 3) / rows;
        const int row = row0 + m, col = (unit + (j0 + j) * units) * 32 + r;
        const float4 v = dsmem_sum4(part + (j * L::ROWS + m) * kPitch + r, c);
        const float scale = P == 1 ? a.a[row] : 1.0f, y4[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col + k < a.n) a.y[row * a.ldy + col + k] = __float2bfloat16_rn(y4[k]);
      }
      cluster_sync();  // everybody has read: the sums may change, or their block end
    }
  }
  // Every copy has been waited for, unless a wait gave up: then those under way are, before the block ends.
  if (*abort_flag && lane == 0)
    for (int s = 0; s < a.stages; ++s) mbar_wait(&bars[s], phase ^ (s < stage ? 0 : 1), nullptr, a.err);
}

template <int GROUP, int P, int NT>
int run(const char* name, LinearArgs a, cudaStream_t stream) {
  using L = Layout<GROUP, P, NT>;
  const int sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "%s: no device", name);
  auto kernel = w4_linear_kernel<GROUP, P, NT>;
  static std::atomic<uint64_t> done{0};
  MVB_TRY(set_smem_once(done, kernel, kMostSmem, name));
  // The cluster: what its blocks' work takes, in records of a pair of tiles, and what a cluster's meeting costs (two cluster
  // barriers and remote reads, some 1.2 us, take as long as 24 records).
  static std::atomic<int> clusters[kMaxCluster + 1] = {};
  auto units_of = [&](int c) {
    return c == 1 ? sms : clusters_at_once(clusters[c], kernel, c, kThreads, kMostSmem);
  };
  int best = 0;
  double least = 0;
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    if (L{(a.blocks + c - 1) / c, 2, c > 1}.bytes() > kMostSmem || c > a.blocks) continue;
    const int units = units_of(c);
    const double cost = double((a.pairs + units - 1) / units) * ((a.blocks + c - 1) / c) + (c > 1 ? 24 : 0);
    if (best == 0 || cost < least) best = c, least = cost;
  }
  MVB_REQUIRE(best > 0, "%s: %d columns", name, a.k);
  a.cluster = best;
  const int units = a.pairs < units_of(best) ? a.pairs : units_of(best);
  // The warps that share a pair's columns: in items, what they compute and what a pair's end takes.
  const int blocks = (a.blocks + best - 1) / best, mine = (a.pairs + units - 1) / units;
  double fewest = 0;
  a.split = 0;
  for (int split = kWarps; split >= 1; split /= 2) {
    const int teams = kWarps / split;
    const double items = ((mine + teams - 1) / teams) * ((blocks + split - 1) / split + kPairEnd);
    if (a.split == 0 || items < fewest) fewest = items, a.split = split;
  }
  L at = {(a.blocks + best - 1) / best, kMaxStages, best > 1};
  while (at.bytes() > kMostSmem) --at.stages;
  a.stages = at.stages;
  const dim3 grid(static_cast<unsigned>(units * best), static_cast<unsigned>((a.rows + L::ROWS - 1) / L::ROWS));
  if (best == 1) return launch(name, kernel, grid, dim3(kThreads), at.bytes(), stream, a);
  return launch_cluster(name, kernel, grid, dim3(kThreads), static_cast<unsigned>(best), at.bytes(), stream, a);
}

template <int GROUP, int P, int NT>
bool fits(const LinearArgs& a) {
  return Layout<GROUP, P, NT>{(a.blocks + kMaxCluster - 1) / kMaxCluster, 2, true}.bytes() <= kMostSmem;
}

template <int GROUP, int P>
int run_rows(const char* name, const LinearArgs& a, cudaStream_t stream) {
  // as many columns of the product as the rows need, where x then fits into a cluster's shared memory
  const int need = (a.rows * P + 7) / 8;
  if constexpr (P == 3)
    if (need > 2 && fits<GROUP, P, 3>(a)) return run<GROUP, P, 3>(name, a, stream);
  if (need > 1 && fits<GROUP, P, 2>(a)) return run<GROUP, P, 2>(name, a, stream);
  return run<GROUP, P, 1>(name, a, stream);
}

template <int P>
int run_group(const char* name, const LinearArgs& a, int64_t group, cudaStream_t stream) {
  if (group == 32) return run_rows<32, P>(name, a, stream);
  if (group == 64) return run_rows<64, P>(name, a, stream);
  return run_rows<128, P>(name, a, stream);
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
  // Few rows here, more on tcgen05.  A bf16 row is three columns of the product here.  8 bf16 rows, here and on tcgen05:
  // 24576 x 4096 25.9 us and 26.2, 12288 x 4096 15.5 and 19.8, 4096 x 8192 15.1 and 16.8; but 4096 x 12288 24.7 and 19.6, 3584 x
  // 14336 29.6 and 19.0, because the columns of 6 rows and more leave too little shared memory there for a block by itself (5
  // rows: 13.8 and 19.5, 17.1 and 18.6).  16 rows of 8 bits: 24576 x 4096 20.4 and 24.8, 4096 x 12288 17.4 and 19.1, 2048 x 1024
  // 5.5 and 9.1; 20 by 24576 x 4096 36.0 and 24.8, 24 by 4096 x 4096 18.6 and 13.4.
  if (rows > (row_scales != nullptr ? 16 : k > 8192 ? 5 : 8)) {
    const W4LinearCall call = {a.y, ldy, x, ldx, row_scales, a.records, a.rows, a.n, a.k, static_cast<int>(group)};
    return w4_gemm(name, call, reinterpret_cast<cudaStream_t>(stream));
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return row_scales != nullptr ? run_group<1>(name, a, group, st) : run_group<3>(name, a, group, st);
}
