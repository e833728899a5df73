// Products of many rows with 4-bit weights, on tcgen05 (few rows: w4_linear.cu, with the formula).
//
// Codes less zeros are whole numbers of -15 .. 15, exact in bf16 and in 8 bits.  They are unpacked from shared memory into
// TMEM, where they are the 128-row operand of tcgen05.mma; rows of x are its columns, from shared memory as TMA brings
// them: bf16 products with fp32 sums, or 8-bit ones with whole sums.  A group's sum is scaled as it leaves TMEM and added
// up in registers, in 32 bits: no weight and no product is rounded.  In bf16 the whole numbers are taken times 2^-11, and the
// results times 2^11: so a group's sum, 128 times 15 times 2^-11 of its largest element at most, never leaves fp32's range
// (and at the other end 12 bits of product times bf16's least number, 2^-144, is still a number of fp32).
//
// A block takes up to 256 weight rows, as two halves of 128 lanes, by BN rows of x (32 or 64); or (SPLIT) up to 128 weight
// rows by 32, 64 or 128, the columns of a step shared by the two sets of warps that unpack, and the rows of x by the two
// that take sums out.  Roles:
//   warp 0        for 128 columns the records, a bulk copy per run that lies together, and TMA boxes of x, into a ring
//   warp 1        the products of a group, into one of two accumulators a half
//   warps 2 and 3 wait for what has no thread behind it (copies, products) and tell those who unpack, and take sums out
//   warps 4 - 11  unpack, a weight row (or half of its columns) a thread, into one of two operands a half in TMEM
//   warps 12 - 19 accumulator out of TMEM, times the row's scale, onto the sums; the results' rows
// Weight rows are given out in tiles of 16, so that few of them leave no SM idle; a cluster of up to 8 blocks splits the
// columns where there are fewer, and its sums meet in distributed shared memory in the order of the blocks.
//
// Bound by the chain of a step of 128 columns (words read, unpacked and stored to TMEM, products, sums read and scaled),
// whose parts meet at barriers: 0.4 to 0.7 us in groups of 128 whatever the tiles, at 40 to 60 % of the issue slots, 15 to 30 % of
// the tensor pipe and 20 % of the memory's rate for 64 rows.  Measured, 24576 x 4096 in groups of 128: 64 rows 29.6 us bf16, 28.7
// 8-bit (groups of 64: 32.8, 40.2; of 32: 44.4, 69.6); 2048 rows 365 and 440 (1.13 and 0.94 PFLOP/s).  More warps with fewer registers each, warps
// that both unpack and sum, words read a step ahead, two blocks an SM with a half each, zeros taken out of the sums instead of
// the codes: all the same or slower (38, 36, 33, 32 and 40 us for some 31).
#include <climits>

#include "common.cuh"
#include "host.h"
#include "w4.cuh"
#include "w4_linear.h"

namespace mvb {
namespace {

constexpr int kThreads = 640;
constexpr int kMaxStages = 8;
constexpr int kMaxCluster = 8;
constexpr size_t kMostSmem = 227 * 1024;

struct GemmW4Args {
  __nv_bfloat16* y;
  int64_t ldy;
  const float* a;  // scales of the rows of x
  const uint8_t* records;
  int rows, n;
  int tiles, blocks;  // 16-row tiles, 128-column blocks
  int chunk, chunks;  // tiles of an item; items down the weight rows
  int columns;        // items across the rows of x
  int cluster, stages;
  unsigned* err;
};

// D[tmem] (+)= A[tmem] * B[smem]^T: bf16 with fp32 sums, or 8 bits with whole ones.
template <bool Q8>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (Q8)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor of kind::i8: D = s32, A = B = s8, both K-major.
__host__ __device__ constexpr uint32_t umma_idesc_s8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// (a & b) | c as one instruction: of two constants the compiler makes two.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// The low nibbles of two halves as 2^-4 + 2^-11 code in bf16.
__device__ __forceinline__ uint32_t nibbles_bf16(uint32_t w) { return and_or(w, 0x000f000fu, 0x3d803d80u); }
constexpr float kUnit = 2048.0f;
// (w >> 4 j) of a word, less the zero: two bf16 numbers 2^-11 (code - zero) (z2: the zero's twice)
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w, uint32_t z2) {
  uint32_t v = nibbles_bf16(w), d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(z2));
  return d;
}
// The low nibbles of four bytes, less the zero (z4: four times): with the top bit set no byte borrows from the next.
__device__ __forceinline__ uint32_t codes_s8(uint32_t w, uint32_t z4) {
  return (and_or(w, 0x0f0f0f0fu, 0x80808080u) - z4) ^ 0x80808080u;
}

// Sums out of TMEM, two at a time.  Whole sums are below 2^18 in size: added to the bits of 1.5 * 2^23 they are its low
// bits, where the conversion instruction would take a quarter of the rate.
template <bool Q8>
__device__ __forceinline__ float2 sums_of(uint32_t a, uint32_t b) {
  if (!Q8) return make_float2(__uint_as_float(a), __uint_as_float(b));
  return __fadd2_rn(make_float2(__uint_as_float(a + 0x4b400000u), __uint_as_float(b + 0x4b400000u)),
                    make_float2(-12582912.0f, -12582912.0f));
}

__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// The block's barriers of the instruction `bar`, by whole warps: `threads` take part, those who sync also wait.  Sixteen warps
// that poll an mbarrier each keep the unit that shared memory is read through busy (4 cycles a poll); where one warp polls
// and tells the others so, 64 rows by 24576 x 4096 in groups of 64 take 32.8 us for 34.7, 200 by 4096 x 4096 21.8 for 23.3.
// No wait here has a limit, and none needs one: the order below makes every arrival that a wait is for follow from arrivals
// before it, whether the polls of warps 2 and 3 end well or give up, and no barrier gets arrivals of its next use before
// this one is over:
//   kUnpack    warp 2 -> who unpacks: records and x of a step there, its operand free
//   kProducts  who unpacks (groups of 128: and takes sums out, two steps later) -> warp 1: operand written (sums read)
//   kToUnpack  warp 1 -> warp 2: products of a step begun; waited for before kUnpack two steps later
//   kToSums    warp 1 -> warp 3: products of a group issued
//   kSums      warp 3 -> who takes sums out: a group's sums there
//   kRead      who takes sums out -> warp 1 (groups of 32 and 64): sums read, two groups later
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
enum Bar { kUnpack = 1, kProducts = 3, kSums = 5, kRead = 7, kToUnpack = 9, kToSums = 11 };  // two of each
// A whole warp's wait for the phase of parity `parity` (its low bit), bounded like mbar_wait; the clock is first read at
// the 64th poll.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned* err) {
  unsigned long long t0 = 0;
  bool ok = false;
  for (unsigned n = 1; n < kWaitMaxPolls; ++n) {
    ok = mbar_try_wait(bar, parity & 1u);
    if (ok) break;
    if ((n & 63u) == 0) {
      if (*abort_flag) break;
      const unsigned long long now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > kWaitLimitNs) {
        report(err, kDevWaitTimeout);
        *abort_flag = 1;
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok) != 0;
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&v)[N], const uint8_t* p) {
  if (N == 1) {
    v[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else if (N == 2) {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
    v[0] = x.x, v[1 % N] = x.y;
  } else {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    v[0] = x.x, v[1 % N] = x.y, v[2 % N] = x.z, v[3 % N] = x.w;
  }
}

// Shared memory: barriers; the ring of x boxes; the ring of records; the cluster's sums.
template <bool Q8, int GROUP, int BN, bool SPLIT>
struct Layout {
  static constexpr int PER = kW4Cols / GROUP;
  static constexpr int REC = w4_record_bytes(GROUP);
  // 16-row tiles of a block: up to 8, or above that
  static constexpr int LEAST = SPLIT ? 1 : 9, MOST = SPLIT ? 8 : 16;
  // What a step of 128 columns takes, in us, measured with a wave of blocks and 16 and 48 steps.
  static constexpr double step_us() {
    constexpr double bf16[3][5] = {{0.58, 0.69, 0.41, 0.39, 0.45}, {0.60, 0.77, 0.40, 0.41, 0.55}, {0.87, 1.26, 0.60, 0.64, 0.96}};
    constexpr double q8[3][5] = {{0.54, 0.66, 0.37, 0.40, 0.53}, {0.62, 1.07, 0.42, 0.54, 0.89}, {1.05, 2.01, 0.67, 0.96, 1.69}};
    return (Q8 ? q8 : bf16)[PER >> 1][(SPLIT ? 2 : 0) + (BN >> 6)];
  }
  static constexpr int BOX = BN * 128;              // bytes of a box of x: 128 of each row
  static constexpr int X_STAGE = BOX * (Q8 ? 1 : 2);
  static constexpr int FIXED = 1024;
  int chunk, stages;
  bool cluster;
  __host__ __device__ int w_stage() const { return chunk * REC; }
  __host__ __device__ int x() const { return FIXED; }
  __host__ __device__ int w() const { return x() + stages * X_STAGE; }
  __host__ __device__ int part() const { return w() + stages * w_stage(); }
  // 1023 more: the boxes begin on 1024 bytes
  __host__ __device__ size_t bytes() const { return 1023 + part() + (cluster ? BN * chunk * kW4Rows * 4 : 0); }
};

struct Item {
  int tile, count, column;  // first tile and number of tiles; first row of x / BN
  __device__ __forceinline__ Item(const GemmW4Args& a, int i) {
    const int r = i / a.columns;
    column = i - r * a.columns;
    tile = r * a.chunk;
    count = min(a.chunk, a.tiles - tile);
  }
};

template <bool Q8, int GROUP, int BN, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    w4_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ GemmW4Args a) {
  using L = Layout<Q8, GROUP, BN, SPLIT>;
  constexpr int PER = L::PER;
  constexpr int KSTEPS = Q8 ? 4 : 8;           // steps of 32 bytes of x in 128 columns
  constexpr int A_COLS = Q8 ? 32 : 64;         // TMEM columns of an operand
  constexpr uint32_t IDESC = Q8 ? umma_idesc_s8(128, BN) : umma_idesc_bf16(128, BN);
  constexpr int HALVES = SPLIT ? 1 : 2;         // of 128 weight rows
  constexpr int WORDS = SPLIT ? 2 : 4;          // words of each 16 bytes of a row that a thread unpacks
  constexpr int CN = SPLIT ? BN / 2 : BN;       // rows of x whose sums a thread takes
  constexpr uint32_t TMEM_COLS = 512;          // a power of two above two operands and two accumulators a half
  static_assert(2 * HALVES * (A_COLS + BN) <= 512, "TMEM");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // an offset: a cast address would be read as a generic one
  uint64_t* full_at = reinterpret_cast<uint64_t*>(smem);  // [stages] a ring's place filled
  uint64_t* drain = full_at + 2 * kMaxStages + 4;
  const uint32_t full = smem_u32(smem), empty = full + 8 * kMaxStages;  // [stages] and read
  const uint32_t a_empty = empty + 8 * kMaxStages;  // [2] operands used (groups of 128: d_full says so)
  const uint32_t d_full = a_empty + 16;             // [2] a group's sums made
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = a.cluster, rank = static_cast<int>(blockIdx.x) % c, unit = static_cast<int>(blockIdx.x) / c;
  const int units = static_cast<int>(gridDim.x) / c;
  const L at = {a.chunk, a.stages, c > 1};
  uint8_t* sx = smem + at.x();
  uint8_t* sw = smem + at.w();
  float* part = reinterpret_cast<float*>(smem + at.part());  // [BN][16 chunk]
  const int S = a.stages;
  const int items = a.chunks * a.columns;
  const int mine = unit < items ? (items - unit + units - 1) / units : 0;
  const int block0 = static_cast<int>(static_cast<int64_t>(rank) * a.blocks / c);
  const int nk = static_cast<int>(static_cast<int64_t>(rank + 1) * a.blocks / c) - block0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(full_at + i, 1);
      mbar_init(full_at + kMaxStages + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(full_at + 2 * kMaxStages + i, 1);
      mbar_init(full_at + 2 * kMaxStages + 2 + i, 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (threadIdx.x == 0) pdl_launch_dependents();
  if (warp != 0) pdl_wait();  // warp 0 asks for weights first, which are constant

  bool ok = true;
  int it = 0;      // 128-column steps so far, over all items; their place in the ring and its parity
  int s = 0;
  uint32_t ph = 0;
  auto step = [&]() {
    ++it;
    if (++s == S) s = 0, ph ^= 1;
  };
  const int steps = mine * nk;
  constexpr int team = 256;  // threads that unpack, and that take sums out
  constexpr int products = 32 + team + (PER > 1 ? 0 : team);
  auto wait = [&](uint32_t bar, uint32_t parity) { return warp_wait(bar, parity, abort_flag, a.err); };
  if (warp == 0) {
    // Lanes 0 - 2 each ask for a run of records that lie together (up to three), lanes 3 and 4 for a box of x.
    const uint64_t policy = lane < 3 ? l2_policy_evict_first() : l2_policy_evict_last();
    for (int n = 0; n < mine; ++n) {
      const Item item(a, unit + n * units);
      const int first = 8 - (item.tile & 7);  // tiles of the first run
      const int from = lane == 0 ? 0 : first + 8 * (lane - 1), to = min(item.count, first + 8 * lane);
      const int run = (lane < 3 ? max(to - from, 0) : 0) * L::REC;
      const int tile = item.tile + from;
      const uint8_t* src = a.records;
      int64_t apart = 0;  // bytes between the run's records of consecutive 128 columns
      if (run > 0) {
        src += w4_record(tile, block0, a.tiles, a.blocks) * L::REC;
        apart = static_cast<int64_t>(min(8, a.tiles - (tile & ~7))) * L::REC;
      }
      const bool box = lane == 3 || (!Q8 && lane == 4);
      const int row = item.column * BN;
      int col = block0 * kW4Cols + (lane == 4 ? 64 : 0);
      auto ask_w = [&](int at_stage) {
        if (lane == 0) mbar_arrive_expect_tx(&full_at[at_stage], item.count * L::REC + L::X_STAGE);
        if (run > 0) copy_bulk(sw + at_stage * at.w_stage() + from * L::REC, src, run, &full_at[at_stage], policy);
        src += apart;
      };
      auto ask_x = [&](int at_stage) {
        if (box)
          tma_load_2d(sx + at_stage * L::X_STAGE + (lane == 4 ? L::BOX : 0), &tmX, &full_at[at_stage], col, row, policy);
        col += kW4Cols;
      };
      int kb = 0;
      if (n == 0) {
        // weights are constant: their copies need not wait for the kernel before
        const int pro = min(S, nk);
        for (int i = 0; i < pro; ++i) ask_w(i);
        pdl_wait();
        for (; kb < pro; ++kb, step()) ask_x(kb);
      }
      for (; kb < nk && ok; ++kb, step()) {
        ok = wait(empty + 8 * s, ph ^ 1);
        if (!ok) break;
        ask_w(s);
        ask_x(s);
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // The whole warp runs the loops, so that addresses and descriptors stay in uniform registers; one thread issues.
    const bool leader = elect_one();
    for (int n = 0; n < mine; ++n) {
      for (int kb = 0; kb < nk; ++kb, step()) {
        const uint64_t bd = umma_desc_sw128(smem_u32(sx + s * L::X_STAGE));
        const uint32_t ta = tmem + (it & 1) * HALVES * A_COLS;
#pragma unroll
        for (int g = 0; g < PER; ++g) {
          const int e = it * PER + g;
          if (g == 0) {
            bar_sync(kProducts + (it & 1), products);  // x has come too: who unpacked has been told
            bar_arrive(kToUnpack + (it & 1), 64);
          }
          if (PER > 1 && e > 1) bar_sync(kRead + (e & 1), 32 + team);
          tc_fence_after();
          if (leader) {
            const uint32_t td = tmem + HALVES * (2 * A_COLS + (e & 1) * BN);
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
              for (int k = g * KSTEPS / PER; k < (g + 1) * KSTEPS / PER; ++k)
                umma_ts<Q8>(td + h * BN, ta + h * A_COLS + 8 * k, bd + (k & 3) * 2 + (k >> 2) * (L::BOX >> 4), IDESC,
                            k > g * KSTEPS / PER ? 1u : 0u);
            commit(d_full + 8 * (e & 1));
            if (PER > 1 && g == PER - 1) commit(a_empty + 8 * (it & 1));
            if (g == PER - 1) commit(empty + 8 * s);
          }
          __syncwarp();
          bar_arrive(kToSums + (e & 1), 64);
        }
      }
    }
  } else if (warp == 2) {
    for (; it < steps; step()) {
      if (it > 1) bar_sync(kToUnpack + (it & 1), 64);
      // The operand's last use: the products of two steps ago.  Groups of 128 columns show it by their sums.
      ok = ok && wait(full + 8 * s, ph) && wait((PER > 1 ? a_empty : d_full) + 8 * (it & 1), (it >> 1) ^ 1);
      tc_fence_after();
      tc_fence_before();
      bar_sync(kUnpack + (it & 1), 32 + team);
    }
    for (int i = steps; i < steps + 2; ++i)
      if (i > 1) bar_sync(kToUnpack + (i & 1), 64);
  } else if (warp == 3) {
    for (int e = 0; e < steps * PER; ++e) {
      bar_sync(kToSums + (e & 1), 64);
      ok = ok && wait(d_full + 8 * (e & 1), e >> 1);
      tc_fence_after();
      tc_fence_before();
      bar_sync(kSums + (e & 1), 32 + team);
    }
  } else if (warp >= 4 && warp < 12) {
    const int h = (warp - 4) >> 2, q = warp & 3, tile = (SPLIT ? 0 : h * 8) + q * 2;  // a warp's two tiles
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    for (int n = 0; n < mine; ++n) {
      const Item item(a, unit + n * units);
      const int offset = min(tile + (lane >> 4), item.count - 1) * L::REC + (lane & 15) * 64;
      for (int kb = 0; kb < nk; ++kb, step()) {
        bar_sync(kUnpack + (it & 1), 32 + team);
        if (tile < item.count) {
          const uint8_t* row = sw + s * at.w_stage() + offset;
          constexpr int PAIRS = PER * WORDS > 4 ? PER * WORDS / 4 : 1;
          uint32_t w[WORDS][4], pair[PAIRS];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if (SPLIT) {
              const uint2 v = *reinterpret_cast<const uint2*>(row + w4_place(t, lane) * 16 + h * 8);
              w[0][t] = v.x, w[1][t] = v.y;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(row + w4_place(t, lane) * 16);
              w[0][t] = v.x, w[1][t] = v.y, w[2 % WORDS][t] = v.z, w[3 % WORDS][t] = v.w;
            }
          }
          const uint32_t* pairs = reinterpret_cast<const uint32_t*>(row - (lane & 15) * (64 - PER * 4) + kW4CodeBytes);
#pragma unroll
          for (int g = 0; g < PAIRS; ++g) pair[g] = pairs[g + (SPLIT ? h * PER / 2 : 0)];
          tc_fence_after();
          const uint32_t ta = tmem + lanes + (SPLIT ? (it & 1) * A_COLS + h * (A_COLS / 2) : ((it & 1) * 2 + h) * A_COLS);
          if (Q8) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 2) {
              uint32_t o[16];
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const uint32_t z4 = __byte_perm(pair[(i + z) * PER / 4], 0, 0x2222) & 0x0f0f0f0fu;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                  const uint32_t lo = codes_s8(w[i + z][t], z4), hi = codes_s8(w[i + z][t] >> 4, z4);
                  o[z * 8 + t * 2] = __byte_perm(lo, hi, 0x6420);
                  o[z * 8 + t * 2 + 1] = __byte_perm(lo, hi, 0x7531);
                }
              }
              tmem_st_x16(ta + i * 8, o);
            }
          } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
              const uint32_t z2 = nibbles_bf16(__byte_perm(pair[i * PER / 4], 0, 0x3232));
              uint32_t o[16];
#pragma unroll
              for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t * 4 + e] = codes_bf16(w[i][t] >> (4 * e), z2);
              tmem_st_x16(ta + i * 16, o);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        bar_arrive(kProducts + (it & 1), products);
      }
    }
  } else {
    const int h = (warp - 12) >> 2, q = warp & 3;
    const int tile = (SPLIT ? 0 : h * 8) + q * 2 + (lane >> 4);  // of the item
    const int first = SPLIT ? h * CN : 0;                        // row of x of the item
    const uint32_t td = tmem + (static_cast<uint32_t>(q * 32) << 16) + HALVES * 2 * A_COLS + (SPLIT ? first : h * BN);
    if (PER == 1) {  // nothing to read yet
      if (steps > 0) bar_arrive(kProducts, products);
      if (steps > 1) bar_arrive(kProducts + 1, products);
    }
    for (int n = 0; n < mine; ++n) {
      const Item item(a, unit + n * units);
      const bool some = (SPLIT ? 0 : h * 8) + q * 2 < item.count;
      // The rows' scales come straight from memory, a step ahead: no wait for the ring.
      const int at_tile = item.tile + min(tile, item.count - 1);
      const uint8_t* src = a.records + w4_record(at_tile, block0, a.tiles, a.blocks) * L::REC + kW4CodeBytes + (lane & 15) * PER * 4;
      const int64_t apart = static_cast<int64_t>(min(8, a.tiles - (at_tile & ~7))) * L::REC;
      float2 acc[CN / 2];
#pragma unroll
      for (int i = 0; i < CN / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
      uint32_t pair[PER], next[PER];
      load_words<PER>(next, src);
      for (int kb = 0; kb < nk; ++kb, step()) {
#pragma unroll
        for (int g = 0; g < PER; ++g) pair[g] = next[g];
        src += apart;
        if (kb + 1 < nk) load_words<PER>(next, src);
#pragma unroll
        for (int g = 0; g < PER; ++g) {
          const int e = it * PER + g;
          bar_sync(kSums + (e & 1), 32 + team);
          tc_fence_after();
          if (some) {
            const float scale = __uint_as_float(pair[g] << 16);
            const float2 s2 = make_float2(scale, scale);
#pragma unroll
            for (int c0 = 0; c0 < CN; c0 += 16) {
              uint32_t d[16];
              tmem_ld_x16(td + (e & 1) * HALVES * BN + c0, d);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; i += 2)
                acc[(c0 + i) / 2] = __ffma2_rn(s2, sums_of<Q8>(d[i], d[i + 1]), acc[(c0 + i) / 2]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (e + 2 < steps * PER) {
            if (PER > 1) bar_arrive(kRead + (e & 1), 32 + team);
            else bar_arrive(kProducts + (e & 1), products);
          }
        }
      }
      const int row0 = item.column * BN + first, rows = min(CN, a.rows - row0);
      const int col = (item.tile + tile) * kW4Rows + (lane & 15);
      int width = a.chunk * kW4Rows;
      int64_t ldy = a.ldy;
      asm volatile("" : "+r"(width), "+l"(ldy));  // not known outside: or all their multiples are kept, in local memory
      if (c > 1) {
        if (tile < item.count) {
          float* to = part + first * width + tile * kW4Rows + (lane & 15);
#pragma unroll
          for (int i = 0; i < CN; ++i) {
            if (i < rows) *to = i & 1 ? acc[i / 2].y : acc[i / 2].x;
            to += width;
          }
        }
      } else if (tile < item.count && col < a.n) {
        __nv_bfloat16* y = a.y + row0 * a.ldy + col;
        const float* scales = a.a + row0;
#pragma unroll
        for (int i = 0; i < CN; ++i) {
          const float v = i & 1 ? acc[i / 2].y : acc[i / 2].x;
          if (i < rows) *y = __float2bfloat16_rn(v * (Q8 ? __ldg(scales + i) : kUnit));
          y += ldy;
        }
      }
    }
  }

  if (c > 1) {
    // A cluster has one item at most, so its blocks meet once: each adds up a share of the sums.
    __syncwarp();
    cluster_sync();
    if (mine > 0) {
      const Item item(a, unit);
      const int row0 = item.column * BN, rows = min(BN, a.rows - row0), fours = item.count * kW4Rows / 4;
      for (int i = rank * kThreads + static_cast<int>(threadIdx.x); i < rows * fours; i += c * kThreads) {
        const int m = i / fours, r = 4 * (i - m * fours), col = item.tile * kW4Rows + r;
        const float4 v = dsmem_sum4(part + m * (a.chunk * kW4Rows) + r, c);
        const float scale = Q8 ? __ldg(a.a + row0 + m) : kUnit;
        const float y4[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
        __nv_bfloat16* y = a.y + (row0 + m) * a.ldy + col;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col + k < a.n) y[k] = __float2bfloat16_rn(y4[k]);
      }
    }
    cluster_sync();  // everybody has read: a block may end
  }
  // Every product has ended before TMEM is given back, and every copy before the block ends.
  if (warp == 1 && elect_one()) {
    umma_commit(drain);
    mbar_wait(drain, 0, nullptr, a.err);
  }
  if (warp == 0 && lane == 0) {
    for (int i = it > S ? it - S : 0; i < it; ++i) mbar_wait(&full_at[i % S], i / S & 1, nullptr, a.err);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// What a call is made of: tiles of an item and blocks of a cluster, and what that is taken to cost, in us: a step takes the same
// whatever its tiles, an item 0.5 besides, a cluster's meeting 3.3.  Of what comes out alike the smallest items.
struct Plan {
  double cost;
  int cluster, chunk;
};

template <bool Q8, int GROUP, int BN, bool SPLIT>
int units_of(int c, int sms) {
  static PerDevice clusters[kMaxCluster + 1];
  return c == 1 ? sms : clusters_at_once(clusters[c], w4_gemm_kernel<Q8, GROUP, BN, SPLIT>, c, kThreads, kMostSmem);
}

template <bool Q8, int GROUP, int BN, bool SPLIT>
int prepare(const char* name) {
  static std::atomic<uint64_t> done{0};
  return set_smem_once(done, w4_gemm_kernel<Q8, GROUP, BN, SPLIT>, kMostSmem, name);
}

template <bool Q8, int GROUP, int BN, bool SPLIT>
Plan plan_of(const W4LinearCall& call, int sms) {
  using L = Layout<Q8, GROUP, BN, SPLIT>;
  const int tiles = (call.n + kW4Rows - 1) / kW4Rows, blocks = (call.k + kW4Cols - 1) / kW4Cols;
  const int columns = (call.rows + BN - 1) / BN;
  Plan best = {0, 0, 0};
  for (int c = 1; c <= kMaxCluster && c <= blocks; ++c) {
    const int units = units_of<Q8, GROUP, BN, SPLIT>(c, sms);
    for (int chunk = L::LEAST; chunk <= L::MOST && chunk <= tiles; ++chunk) {
      const int64_t items = static_cast<int64_t>((tiles + chunk - 1) / chunk) * columns;
      if (c > 1 && items > units) continue;  // a cluster meets once
      const double waves = static_cast<double>((items + units - 1) / units);
      const double cost = waves * ((blocks + c - 1) / c * L::step_us() + 0.5) + (c > 1 ? 3.3 : 0.0);
      if (best.chunk == 0 || cost < best.cost) best = {cost, c, chunk};
    }
  }
  return best;
}

template <bool Q8, int GROUP, int BN, bool SPLIT>
int run(const char* name, const W4LinearCall& call, const Plan& plan, int sms, cudaStream_t stream) {
  using L = Layout<Q8, GROUP, BN, SPLIT>;
  auto kernel = w4_gemm_kernel<Q8, GROUP, BN, SPLIT>;
  GemmW4Args a = {};
  a.y = call.y, a.ldy = call.ldy, a.a = call.row_scales, a.records = call.records, a.rows = call.rows, a.n = call.n;
  a.tiles = (call.n + kW4Rows - 1) / kW4Rows;
  a.blocks = (call.k + kW4Cols - 1) / kW4Cols;
  a.columns = (call.rows + BN - 1) / BN;
  a.err = device_status_ptr();
  a.cluster = plan.cluster;
  a.chunk = plan.chunk;
  a.chunks = (a.tiles + a.chunk - 1) / a.chunk;
  L at = {a.chunk, kMaxStages, a.cluster > 1};
  while (at.bytes() > kMostSmem) --at.stages;
  a.stages = at.stages;
  // One block an SM, whatever it needs, and none beside a block of the layer kernel (109 KB), whose blocks wait for one
  // another: a second would wait for the first one's TMEM, and where both are of one cluster the first for the second.
  const size_t smem = at.bytes() > 120 * 1024 ? at.bytes() : 120 * 1024;
  const int64_t items = static_cast<int64_t>(a.chunks) * a.columns;
  const int most = units_of<Q8, GROUP, BN, SPLIT>(a.cluster, sms), units = items < most ? static_cast<int>(items) : most;

  CUtensorMap tm;
  const uint64_t dims[2] = {static_cast<uint64_t>(call.k), static_cast<uint64_t>(call.rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(call.ldx) * (Q8 ? 1 : 2)};
  const uint32_t box[2] = {Q8 ? 128u : 64u, BN};
  MVB_TRY(encode_tiled(&tm, Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, call.x, dims, strides,
                       box, CU_TENSOR_MAP_SWIZZLE_128B));
  const dim3 grid(static_cast<unsigned>(units * a.cluster));
  if (a.cluster == 1) return launch(name, kernel, grid, dim3(kThreads), smem, stream, tm, a);
  return launch_cluster(name, kernel, grid, dim3(kThreads), static_cast<unsigned>(a.cluster), smem,
                        stream, tm, a);
}

template <bool Q8, int GROUP, int BN>
int run_either(const char* name, const W4LinearCall& call, int sms, cudaStream_t stream) {
  MVB_TRY((prepare<Q8, GROUP, BN, true>(name)));
  MVB_TRY((prepare<Q8, GROUP, BN, false>(name)));
  const Plan one = plan_of<Q8, GROUP, BN, true>(call, sms), two = plan_of<Q8, GROUP, BN, false>(call, sms);
  if (two.chunk == 0 || one.cost <= two.cost) return run<Q8, GROUP, BN, true>(name, call, one, sms, stream);
  return run<Q8, GROUP, BN, false>(name, call, two, sms, stream);
}

template <bool Q8, int GROUP>
int run_rows(const char* name, const W4LinearCall& call, cudaStream_t stream) {
  const int sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "%s: no device", name);
  // As few columns as hold all rows, with as many weight rows as come out cheaper: 64 by 24576 x 4096 takes 33.0 us with up to 16 tiles
  // and 36.5 with up to 8, 64 by 4096 x 4096 14.6 and 13.4.  Above 64 rows half the weight rows by twice the columns, so that
  // half is unpacked: 2048 by 24576 x 4096 361 us for 490 (8 bits: 426 for 512), 128 rows 37.7 for 49.1.
  if (call.rows <= 32) return run_either<Q8, GROUP, 32>(name, call, sms, stream);
  if (call.rows <= 64) return run_either<Q8, GROUP, 64>(name, call, sms, stream);
  MVB_TRY((prepare<Q8, GROUP, 128, true>(name)));
  return run<Q8, GROUP, 128, true>(name, call, plan_of<Q8, GROUP, 128, true>(call, sms), sms, stream);
}

template <bool Q8>
int run_group(const char* name, const W4LinearCall& call, cudaStream_t stream) {
  if (call.group == 32) return run_rows<Q8, 32>(name, call, stream);
  if (call.group == 64) return run_rows<Q8, 64>(name, call, stream);
  return run_rows<Q8, 128>(name, call, stream);
}

}  // namespace

int w4_gemm(const char* name, const W4LinearCall& call, cudaStream_t stream) {
  return call.row_scales != nullptr ? run_group<true>(name, call, stream) : run_group<false>(name, call, stream);
}

}  // namespace mvb
