// Products of few rows with 4-bit weights: y[m, n] = sum_g scale[n, g] sum_{k in g} (code[n, k] - zero[n, g]) x[m, k].
//
// x in bf16, or in 8 bits with a scale a[m] per row (q8_rows.cu), which multiplies the result.  Codes less zeros are
// whole numbers of -15 .. 15, exact in bf16 and in 8 bits: a group's sum runs through the matrix instruction as they
// are (32-bit sums; for 8-bit rows whole numbers, exact), and only the sum is scaled, in 32 bits.  No product is rounded.
//
// Bound by the weights' bytes (0.53 a weight in groups of 128).  At the memory's rate an SM gets 44 weights a cycle
// and has 128 lanes to unpack them: three operations for two codes in bf16 (shift, mask and bias in one, subtract), seven
// for eight in 8 bits.  mma.sync takes 1024 (bf16) or 2048 (8 bits) products a cycle, so up to some 20 rows cost nothing.
// The weights are its 16-row operand and the rows of x its 8 columns.
//
// A block works on pairs of 16 weight rows.  Its warps split the columns, each with a record of both 16-row tiles under
// way in registers while it computes the one before; x lies in shared memory in the order of the lanes.  The warps' sums
// of a pair meet in shared memory and are added in the order of the warps.  A cluster of up to 8 blocks splits
// the columns further, where few weight rows would leave SMs idle or x would not fit; its sums meet in distributed
// shared memory, in the order of the blocks.  So every result is the same on every call.
#include <climits>

#include "common.cuh"
#include "host.h"
#include "mma_sync.cuh"
#include "w4.cuh"

namespace mvb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPitch = 36;     // floats between columns of a pair's 32 sums: 4 columns by 8 rows touch all banks
constexpr int kRound = 16;     // pairs after which the blocks of a cluster add up
constexpr int kMaxCluster = 8;

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
};

__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// (w >> 4 j) of a word, less the zero: two bf16 numbers code - zero (z2: 128 + zero twice)
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w, uint32_t z2) {
  uint32_t v = (w & 0x000f000fu) | 0x43004300u, d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(z2));
  return d;
}
// The low nibbles of four bytes, less the zero (z4: four times): with the top bit set no byte borrows from the next.
__device__ __forceinline__ uint32_t codes_s8(uint32_t w, uint32_t z4) {
  return (((w & 0x0f0f0f0fu) | 0x80808080u) - z4) ^ 0x80808080u;
}

__device__ __forceinline__ uint4 load_codes(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// What a lane holds of a record of each of a pair's tiles: rows lane / 4 and lane / 4 + 8, its place's 16 bytes and all pairs.
template <int PER>
struct Item {
  uint4 codes[2][2];
  uint32_t pairs[2][2][PER];
};

template <int PER>
__device__ __forceinline__ void load_item(Item<PER>& it, const uint8_t* first, const uint8_t* second, int lane) {
  const int g = lane >> 2;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint8_t* rec = s == 0 ? first : second;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      it.codes[s][h] = load_codes(rec + (g + 8 * h) * 64 + (lane & 3) * 16);
      const uint8_t* p = rec + kW4CodeBytes + (g + 8 * h) * PER * 4;
      if (PER == 1) {
        it.pairs[s][h][0] = __ldg(reinterpret_cast<const uint32_t*>(p));
      } else if (PER == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        it.pairs[s][h][0] = v.x, it.pairs[s][h][1 % PER] = v.y;
      } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        it.pairs[s][h][0] = v.x, it.pairs[s][h][1 % PER] = v.y, it.pairs[s][h][2 % PER] = v.z, it.pairs[s][h][3 % PER] = v.w;
      }
    }
  }
}

// x of this block's columns in the order of the lanes: 16 bytes (8 bf16) or 8 bytes (8 codes) for each 32 columns, tile
// of 8 rows and lane; the lane's row is lane / 4, its columns 8 (lane % 4) .. + 7 of the 32.  Which
// columns: the lane's place of a record's row r holds t = place ^ (r / 2 % 4), the same for rows r and r + 8 but not for
// the 8 rows of a step, so a lane takes its codes from place t ^ (r / 2 % 4) and keeps t = lane % 4.
template <bool Q8, int NT>
__device__ __forceinline__ void stage_x(uint8_t* sx, const LinearArgs& a, int row0, int block0, int blocks) {
  const int n = blocks * 4 * NT * 32;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int lane = i & 31, nt = (i >> 5) % NT, step = (i >> 5) / NT;  // step: 32 columns
    const int row = row0 + nt * 8 + (lane >> 2), col = block0 * kW4Cols + step * 32 + (lane & 3) * 8;
    const bool some = row < a.rows && col < a.k;
    if (Q8) {
      uint2 v = make_uint2(0, 0);
      if (some) v = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.x) + row * a.ldx + col);
      // the columns' order of a word's bytes: 0 4 1 5, then 2 6 3 7
      const uint2 o = make_uint2(__byte_perm(v.x, v.y, 0x5140), __byte_perm(v.x, v.y, 0x7362));
      *reinterpret_cast<uint2*>(sx + ((((step >> 1) * NT + nt) * 32 + lane) * 2 + (step & 1)) * 8) = o;
    } else {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (some) v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.x) + row * a.ldx + col);
      *reinterpret_cast<uint4*>(sx + ((step * NT + nt) * 32 + lane) * 16) = v;
    }
  }
}

template <bool Q8, int PER, int NT>
__device__ __forceinline__ void compute(const Item<PER>& it, const uint8_t* sx, int block, int lane, float (&acc)[2][NT][4]) {
  constexpr int STEPS = 4 / PER;  // steps of 32 columns in a group
#pragma unroll
  for (int grp = 0; grp < PER; ++grp) {
    int di[2][NT][4];
    float df[2][NT][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q) di[s][nt][q] = 0, df[s][nt][q] = 0.0f;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int i = grp * STEPS + st;
      uint4 b[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (Q8) {
          const uint2 v = *reinterpret_cast<const uint2*>(sx + ((((block * 2 + (i >> 1)) * NT + nt) * 32 + lane) * 2 + (i & 1)) * 8);
          b[nt] = make_uint4(v.x, v.y, 0, 0);
        } else {
          b[nt] = *reinterpret_cast<const uint4*>(sx + (((block * 4 + i) * NT + nt) * 32 + lane) * 16);
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t w0 = i == 0 ? it.codes[s][0].x : i == 1 ? it.codes[s][0].y : i == 2 ? it.codes[s][0].z : it.codes[s][0].w;
        const uint32_t w1 = i == 0 ? it.codes[s][1].x : i == 1 ? it.codes[s][1].y : i == 2 ? it.codes[s][1].z : it.codes[s][1].w;
        if (Q8) {
          const uint32_t z0 = __byte_perm(it.pairs[s][0][grp], 0, 0x2222) & 0x0f0f0f0fu;
          const uint32_t z1 = __byte_perm(it.pairs[s][1][grp], 0, 0x2222) & 0x0f0f0f0fu;
          const uint32_t a0 = codes_s8(w0, z0), a2 = codes_s8(w0 >> 4, z0);
          const uint32_t a1 = codes_s8(w1, z1), a3 = codes_s8(w1 >> 4, z1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_s8_16832(di[s][nt], a0, a1, a2, a3, b[nt].x, b[nt].y);
        } else {
          const uint32_t z0 = __byte_perm(it.pairs[s][0][grp], 0, 0x3232), z1 = __byte_perm(it.pairs[s][1][grp], 0, 0x3232);
          uint32_t p0[4], p1[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p0[j] = codes_bf16(w0 >> (4 * j), z0), p1[j] = codes_bf16(w1 >> (4 * j), z1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16_16816(df[s][nt], p0[0], p1[0], p0[1], p1[1], b[nt].x, b[nt].y);
            mma_bf16_16816(df[s][nt], p0[2], p1[2], p0[3], p1[3], b[nt].z, b[nt].w);
          }
        }
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const float c0 = __uint_as_float(it.pairs[s][0][grp] << 16), c1 = __uint_as_float(it.pairs[s][1][grp] << 16);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float d = Q8 ? static_cast<float>(di[s][nt][q]) : df[s][nt][q];
          acc[s][nt][q] = fmaf(q < 2 ? c0 : c1, d, acc[s][nt][q]);
        }
    }
  }
}

__device__ __forceinline__ void group_bar(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <bool Q8, int GROUP, int NT>
__global__ void __launch_bounds__(kThreads, 1) w4_linear_kernel(const LinearArgs a) {
  constexpr int PER = kW4Cols / GROUP;
  constexpr int REC = w4_record_bytes(GROUP);
  constexpr int SUMS = 8 * NT * kPitch;  // floats of a pair's sums
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int c = a.cluster, rank = static_cast<int>(blockIdx.x) % c, unit = static_cast<int>(blockIdx.x) / c;
  const int units = static_cast<int>(gridDim.x) / c;
  const int row0 = blockIdx.y * 8 * NT;
  const int block0 = static_cast<int>(static_cast<int64_t>(rank) * a.blocks / c);
  const int blocks = static_cast<int>(static_cast<int64_t>(rank + 1) * a.blocks / c) - block0;
  const int most = (a.blocks + c - 1) / c;
  uint8_t* sx = smem;
  float* red = reinterpret_cast<float*>(smem + static_cast<int64_t>(most) * 4 * NT * (Q8 ? 256 : 512));  // [2][warp][SUMS]
  float* part = red + 2 * kWarps * SUMS;  // [kRound][SUMS], where the cluster adds up

  // Pairs unit, unit + units, ..; of those this warp's group takes every teams-th, and of a pair's columns this
  // warp blocks kw, kw + split, ..
  const int split = a.split, teams = kWarps / split, team = wid / split, kw = wid % split;
  const int mine = unit < a.pairs ? (a.pairs - unit + units - 1) / units : 0;  // pairs of this block
  auto at = [&](int j, int b, int s) {  // record of tile s of the block's j-th pair
    const int tile = 2 * (unit + j * units) + s;
    // the last pair may lack its second tile: its first is read again and what comes of it is not written
    return a.records + w4_record(tile < a.tiles ? tile : tile - 1, block0 + b, a.tiles, a.blocks) * REC;
  };

  const int src = (lane & ~3) | w4_place(lane & 3, lane >> 2);  // the lane's place
  Item<PER> next;
  int nj = team, nb = kw;  // the next item to load: pair and block
  bool more = nj < mine && nb < blocks;
  // weights are constant: their loads need not wait for the kernel before
  if (more) load_item<PER>(next, at(nj, nb, 0), at(nj, nb, 1), src);
  pdl_launch_dependents();
  pdl_wait();
  stage_x<Q8, NT>(sx, a, row0, block0, blocks);
  __syncthreads();

  const int rounds = (mine + kRound - 1) / kRound;
  // every block of a cluster has the same pairs, so the same rounds
  for (int round = 0; round < (c > 1 ? rounds : 1); ++round) {
    const int j1 = c > 1 ? min(mine, (round + 1) * kRound) : mine;
    const int j0 = c > 1 ? round * kRound : 0;
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
        const Item<PER> item = next;
        nb += split;
        if (nb >= blocks) nb = kw, nj += teams;
        if (nj < mine) load_item<PER>(next, at(nj, nb, 0), at(nj, nb, 1), src);
        compute<Q8, PER, NT>(item, sx, b, lane, acc);
      }
      float* out = red + (buf * kWarps + wid) * SUMS;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            out[(nt * 8 + 2 * (lane & 3) + (q & 1)) * kPitch + s * 16 + (q >> 1) * 8 + (lane >> 2)] = acc[s][nt][q];
      if (split > 1) group_bar(1 + team, 32 * split);
      else __syncwarp();
      const float* in = red + (buf * kWarps + team * split) * SUMS;
      const int pair = unit + j * units;
      for (int i = kw * 32 + lane; i < 256 * NT; i += 32 * split) {
        const int m = i >> 5, r = i & 31;
        float v = 0.0f;
        for (int w = 0; w < split; ++w) v += in[w * SUMS + m * kPitch + r];
        if (c > 1) {
          part[(j - j0) * SUMS + m * kPitch + r] = v;
        } else {
          const int row = row0 + m, col = pair * 32 + r;
          if (row < a.rows && col < a.n) {
            if (Q8) v *= a.a[row];
            a.y[row * a.ldy + col] = __float2bfloat16_rn(v);
          }
        }
      }
      buf ^= 1;
    }
    if (c > 1) {
      cluster_sync();
      for (int i = rank * kThreads + tid; i < (j1 - j0) * 256 * NT; i += c * kThreads) {
        const int j = i / (256 * NT), m = i / 32 % (8 * NT), r = i & 31;
        const int row = row0 + m, col = (unit + (j0 + j) * units) * 32 + r;
        if (row >= a.rows || col >= a.n) continue;
        float v = 0.0f;
        for (int q = 0; q < c; ++q) v += dsmem_ld_f32(part + j * SUMS + m * kPitch + r, q);
        if (Q8) v *= a.a[row];
        a.y[row * a.ldy + col] = __float2bfloat16_rn(v);
      }
      cluster_sync();  // everybody has read: the sums may change, or their block end
    }
  }
}

constexpr size_t kMostSmem = 227 * 1024;

template <bool Q8, int NT>
size_t smem_of(int blocks, int cluster) {
  const int most = (blocks + cluster - 1) / cluster;
  return static_cast<size_t>(most) * 4 * NT * (Q8 ? 256 : 512) + (2 * kWarps + (cluster > 1 ? kRound : 0)) * 8 * NT * kPitch * 4;
}

template <bool Q8, int GROUP, int NT>
int run(const char* name, LinearArgs a, cudaStream_t stream) {
  const int sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "%s: no device", name);
  auto kernel = w4_linear_kernel<Q8, GROUP, NT>;
  static std::atomic<uint64_t> done{0};
  MVB_TRY(set_smem_once(done, kernel, kMostSmem, name));
  // The cluster: what its blocks' work takes, in records of a pair of tiles, and what a cluster's meeting costs.
  int best = 0;
  double least = 0;
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    if (smem_of<Q8, NT>(a.blocks, c) > kMostSmem || (c > 1 && a.blocks < c)) continue;
    const int units = c == 1 ? sms : sms / c;
    const double cost = double((a.pairs + units - 1) / units) * ((a.blocks + c - 1) / c) + (c > 1 ? 24 : 0);
    if (best == 0 || cost < least) best = c, least = cost;
  }
  MVB_REQUIRE(best > 0, "%s: %d columns", name, a.k);
  a.cluster = best;
  const int units = a.pairs < sms / best ? a.pairs : sms / best;
  const int blocks = a.blocks / best;
  a.split = 1;
  while (a.split < kWarps && a.split < blocks) a.split *= 2;
  const size_t smem = smem_of<Q8, NT>(a.blocks, best);
  const dim3 grid(static_cast<unsigned>(units * best), static_cast<unsigned>((a.rows + 8 * NT - 1) / (8 * NT)));
  if (best == 1) return launch(name, kernel, grid, dim3(kThreads), smem, stream, a);
  return launch_cluster(name, kernel, grid, dim3(kThreads), static_cast<unsigned>(best), smem, stream, a);
}

template <bool Q8, int GROUP>
int run_rows(const char* name, const LinearArgs& a, cudaStream_t stream) {
  // 16 rows of more columns than this do not fit into a cluster's shared memory: 8 at a time
  if (a.rows <= 8 || smem_of<Q8, 2>(a.blocks, kMaxCluster) > kMostSmem) return run<Q8, GROUP, 1>(name, a, stream);
  return run<Q8, GROUP, 2>(name, a, stream);
}

template <bool Q8>
int run_group(const char* name, const LinearArgs& a, int64_t group, cudaStream_t stream) {
  if (group == 32) return run_rows<Q8, 32>(name, a, stream);
  if (group == 64) return run_rows<Q8, 64>(name, a, stream);
  return run_rows<Q8, 128>(name, a, stream);
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return row_scales != nullptr ? run_group<true>(name, a, group, st) : run_group<false>(name, a, group, st);
}
