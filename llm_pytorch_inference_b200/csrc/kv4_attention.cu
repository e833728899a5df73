// Attention of the newest T tokens of each sequence over the 4-bit paged pool (T = 1: a decode step).
//
//   out[b, i, h] = sum_t softmax_t(cap(q . k_t * scale)) v_t  over the keys t that query i sees,
//   k = m + s u,  v = m' + s' u'  per 64 channels (codes u in 0..15, pairs (s, m)).
//
// What it must read is 9/16 of a byte per cached value, once: the bound is memory.  That leaves an SM some 44
// values a clock, and its integer pipe takes 64 lane-operations a clock, so codes never become floating-point
// numbers one by one:
//   * fp16 holds u * 2^-24 and u * 2^-20 as bit patterns with the code in bits 0-3 or 4-7 (subnormal numbers, exact), so
//     one AND of a word yields two matrix operands.
//   * Scores: q . k = sum_g s_g (q_g . u_g) + m_g sum(q_g) over the groups of 64 channels, the pairs outside
//     the products.  The other operand is q times a power of two that puts its row's largest magnitude below 2^11:
//     exact in fp16 for what is above 2^-27 of that magnitude, and off by 2^-35 of it below.  So the scores are off by
//     what fp32 sums lose, whatever the number of rows.  (q as two signed bytes for the integer tensor cores, one
//     operation a word less, took 28.0 us where this takes 28.8 and 45.0 where this takes 47.1, but left q 16 bits of
//     its row's largest magnitude, which loses the small channels beside a large one.)
//   * Outputs: the weight of a token times s' is the other operand, and p m' is summed per group and query, on the
//     side.  That product p s' is rounded to 11 bits (8 times finer than the result's bf16).  It is scaled by a power of
//     two of its row and group, which follows the products themselves (choose_scale): a value scale however large does
//     not cost the others their bits unless its token has the weight to matter.  (One scaling for all groups and rows,
//     following the largest s', took 28.8 us where this takes 29.3 and 58.7 where this takes 63.5; it lost a group of
//     2^-14 of its neighbour's values 0.5 %, and all that came after a value of 2^20 30 %.  Value scales that vary by
//     2^4 either way cost another 8 to 17 %.)  Scores, statistics and sums are fp32.
// Both products run transposed on mma.sync, the query rows (query heads of the KV head times T) being the n = 8
// side: S^T = K Q^T (16 tokens x rows), O^T = V^T P^T.  The k index of the first product runs over the channels
// in the order in which a lane's words hold them (Q is stored in that order); the tokens of the second are
// permuted (tile_token) so that lanes reading the same word of different tokens fall into different banks.
// Up to 4 rows (RT = 0) take every other column of the first product, and all 8 of the second: the two halves of a
// masked word (two channels of one token) have one each, which halves its accumulators.
//
// Work split: the cache of an item (sequence, KV head, chunk of query rows) is a run of records of 16 tokens.
// The records of the whole batch are laid end to end and divided evenly over the resident warps, whatever the
// lengths: a warp is a worker of its own, without a barrier after the prologue.  It streams its records
// through a ring in shared memory (one bulk copy a record, several in flight) and keeps the running
// maximum, sum and output of an item in registers.  An item that spans workers leaves partial results, joined in
// worker order by a second small kernel: no atomics in global memory, nothing to clear, the same bits every time.
//
// Measured on a B200 (6.55 TB/s copy), device time with inputs turned over: 64 sequences of 1024-2048 tokens, 32 query
// and 8 KV heads of 128: 29.3 us for 115 MB, of which 3.5 us pass before the first copy, 18 until the median worker has
// seen its records, at the rate of memory, and 6 in the last workers and the join.  One sequence of 131072: 35.8 us
// (151 MB).  16 sequences of 4096-8192, 16 query and 8 KV heads of 256, capped: 48.0 us (226 MB, 4.7 TB/s).  5 query
// tokens of 4 sequences of 16K-32K: 63.5 us (115 MB), bound by what 8 warps of an SM can issue.  One short sequence:
// 6.4 us, latency.
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "host.h"
#include "kv4.cuh"
#include "mma_sync.cuh"

namespace mvb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kShortRecords = 8;  // items of at most this many records are never split
// What beginning an item costs a warp (its Q, its result), in bursts, for the division of the work: 64 sequences of
// 1024-2048 tokens and 8 query rows took 39.2 us at 1 and 37.6 at 3.
constexpr int kItemCost = 3;

// A weight is 2^(score - reference): the reference is a row's maximum when last raised, and is raised
// once a score passes it by more than kSlack (in powers of two), so that most records cost one vote instead
// of a reduction.  The weight times the scaled s' stays below 2^(kSlack + 9) = 2^15 in fp16.
constexpr float kSlack = 6.0f;
constexpr float kScaleMax = 512.0f;  // of s' times its scaling, where nothing else was chosen
constexpr int kFirstScale = 120;     // log2 of the scaling before any s', and its largest: times 2^kSlack in fp32's range
constexpr int kNothing = -10000;     // log2 of zero
constexpr float kFltMax = 3.40282347e38f;
constexpr float kNone = -kFltMax;     // reference of a row without a key: no special cases, any score passes it

// RT: 0 = up to 4 query rows per chunk, else up to 8 RT.
template <int RT>
struct Kv4Rows {
  static constexpr int NT = RT == 0 ? 1 : RT;       // n = 8 tiles
  static constexpr int NC = RT == 0 ? 1 : 2 * RT;   // rows per lane
  static constexpr int ROWS = RT == 0 ? 4 : 8 * RT;
  static constexpr bool HOLD_Q = RT < 2;            // the rows' factors and sums of q stay in registers
};

// BURST: records that a warp takes at once (one wait, one refill); STAGES of them are held, so that
// an SM has some 45 KB or more under way while it computes.  A wait and refill cost some 90 instructions, a record of
// 24 rows 510: 5 query tokens of 4 sequences of 16K-32K took 70.2 us with bursts of 1, 64.5 with 2, 61.9 with 4; one
// sequence of 500, which 4 spread over fewer workers, 17.3, 17.6 and 19.0.  WARPS of the one block per SM: 64 sequences
// of 1024-2048 tokens, 4 rows of 128, took 33.3 us with 8, 30.1 with 12, 31.0 with 16 (128 registers); 8 rows 40.9,
// 37.6, 44.1 (spills); 4 rows of 256, 16 x 4096-8192, 57, 47.1, 49.1.  16 rows and more of 128 or 256 need over 168
// registers.  One block, not two: the scheduler prefers the older one, whose warps then ended after 21 us of a
// call where the other's took 27.
template <int D, int RT>
struct Kv4Cfg {
  static constexpr int BURST = D == 256 ? 1 : D == 128 ? (RT > 1 ? 4 : 2) : RT == 0 ? 4 : 2;
  static constexpr int STAGES = D == 256 ? (RT > 1 ? 2 : 3) : D == 128 ? 2 : RT == 0 ? 2 : RT > 1 ? 3 : 4;
  static constexpr int MATH = RT > 1 ? 1 : BURST;  // records whose scores are in registers at once
  static constexpr int WARPS = (D == 256 && RT > 0) || (D == 128 && RT > 1) || RT > 2 ? 8 : 12;
};

struct Kv4AttnArgs {
  __nv_bfloat16* out;
  const __nv_bfloat16* q;
  int64_t out_stride, q_stride;  // elements between query tokens
  const uint8_t* pool;           // the layer's first record
  const int32_t* tables;
  int64_t table_stride;
  int max_blocks;
  const int32_t* ctx;
  int batch, T, group, hkv;
  int chunks;  // of ROWS query rows, per KV head
  int num_blocks, recs;
  float score_scale;  // scale * log2(e), or scale / softcap under a cap
  float cap_log2;     // softcap * log2(e); 0 = no cap
  int window;
  int chunk_rows;  // rows of the largest chunk
  bool split;     // items may be split: their rounds are bursts and kItemCost; else an item is one round
  // workspace
  struct Kv4Item* items;  // [batch * hkv * chunks]
  float2* part_ml;        // [2 workers][ROWS]
  float* part_o;          // [2 workers][ROWS][D]
  unsigned* err;
};

// The workers that an item spans.
struct Kv4Item {
  int first, last;
};

// The rounds of the batch among the workers: each `size`, the first `more` one more.
struct Kv4Split {
  int64_t size, more;
  __device__ __forceinline__ void set(int64_t total, int workers) {
    if (total >> 32) {
      size = total / workers;
    } else {
      size = static_cast<uint32_t>(total) / static_cast<uint32_t>(workers);
    }
    more = total - size * workers;
  }
  __device__ __forceinline__ int64_t start(int w) const { return w * size + (w < more ? w : more); }
  __device__ __forceinline__ int worker(int64_t x) const {
    const int64_t y = x - more * (size + 1);
    if (x >> 31) return static_cast<int>(y < 0 ? x / (size + 1) : more + y / size);
    return y < 0 ? static_cast<uint32_t>(x) / static_cast<uint32_t>(size + 1)
                 : static_cast<int>(more) + static_cast<uint32_t>(y) / static_cast<uint32_t>(size);
  }
};

// floor(log2 x) of x >= 0, at least -127 for numbers above zero.
__device__ __forceinline__ int log2_of(float x) {
  return x > 0.0f ? static_cast<int>(__float_as_uint(x) >> 23) - 127 : kNothing;
}
__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// log2 of the scaling of a row's products p s' in a group of channels, from logarithms: `old`, the present one;
// s, the largest s' of the records at hand; w, their largest product; o, what has been summed, as the sum of products
// that it stands for.  In fp16 a product below 2^-14 loses bits and is off by 2^-25 at most: the n products of a worker
// keep all but n 2^-25 of the largest one, or of their sum, where that is scaled to 2^0 or above.  The scaling stays
// while s' is within kScaleMax, and falls to where s' is within it, both while the products keep their bits; else it
// stays as long as the products themselves fit, and else follows them.
// What is not looked at again: where a row's heaviest tokens have no spread in a group (s' = 0), what weighs less than
// 2^-31 of them may count with its minimum alone, p m'.
__device__ __forceinline__ int choose_scale(int old, int s, int w, int o) {
  const int most = max(w, o);
  int e = s + old <= 8 ? old : 7 - s;
  if (most > kNothing && e + most < 0) e = old + most >= 0 && old + w <= 8 ? old : 7 - most;
  return min(max(e, -kFirstScale), kFirstScale);
}

// exp2 with results below 2^-126 flushed to zero.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh x = 1 - 2 / (e^2x + 1), with an absolute error of a few 2^-24: c times that in a score capped at c.
__device__ __forceinline__ float tanh_exp(float x) {
  return 1.0f - __fdividef(2.0f, ex2(x * (2.0f * kLog2e)) + 1.0f);
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // movmatrix_trans, free to be scheduled
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// N consecutive 32-bit words of shared memory, aligned to their size.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * k);
      w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
    }
  }
}
// A pair's scale (low half) and minimum (high half).
__device__ __forceinline__ float pair_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float pair_min(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned* err) {
  return mbar_wait(bar, parity, abort_flag, err);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Token of a record that is row r of the first product's tile and index r of the second's sum.  The four
// tokens of index 2c, 2c + 1, 8 + 2c and 9 + 2c are 4c .. 4c + 3, turned by c: in each of the four
// loads of V the lanes c = 0..3 then read rows of alternating parity, i.e. both halves of the banks.
__device__ __forceinline__ int tile_token(int r) {
  const int c = (r & 7) >> 1, i = (r & 1) | ((r >> 3) << 1);
  return 4 * c + ((i + c) & 3);
}

// What a sequence's cache has to offer: records [first, last), divided in rounds.
struct Kv4Seq {
  int ctx, first, last, rounds;
};
template <int BURST>
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs& a, int b, bool tell = false) {
  Kv4Seq s;
  const int most = a.max_blocks * a.recs * kKv4Tokens;
  const int raw = a.ctx[b];
  s.ctx = min(max(raw, 0), most);
  if (tell && s.ctx != raw) report(a.err, kDevBadPosition);
  s.first = 0;
  if (a.window > 0) s.first = max(s.ctx - a.T + 1 - a.window, 0) / kKv4Tokens;
  s.last = (s.ctx + kKv4Tokens - 1) / kKv4Tokens;
  s.rounds = a.split ? kItemCost + max(s.last - s.first + BURST - 1, 0) / BURST : 1;
  return s;
}
// Records [x, y) of rounds [r, r + n) of an item.
template <int BURST>
__device__ __forceinline__ int2 kv4_records(const Kv4AttnArgs& a, const Kv4Seq& s, int r, int n) {
  if (!a.split) return make_int2(s.first, s.last);
  return make_int2(s.first + max(r - kItemCost, 0) * BURST, min(s.first + max(r + n - kItemCost, 0) * BURST, s.last));
}

template <int D, int RT>
struct Kv4Smem {
  static constexpr int STAGES = Kv4Cfg<D, RT>::STAGES, ROWS = Kv4Rows<RT>::ROWS;
  // per warp: the ring, Q operands [D / 32][NT][32 lanes] x 16 bytes, per row the score factor, the
  // sums of q and the scalings per group and the number of keys it sees, room to choose scalings, the ring's barriers
  static constexpr int RING = STAGES * Kv4Cfg<D, RT>::BURST * Kv4<D>::RECORD;
  static constexpr int QF = RING;
  static constexpr int COL = QF + D / 32 * Kv4Rows<RT>::NT * 512;
  static constexpr int BAR = (COL + ROWS * (3 + 4 * Kv4<D>::NG) * 4 + 7) / 8 * 8;
  static constexpr int WARP = (BAR + STAGES * 8 + 127) / 128 * 128;
  static constexpr int BYTES = Kv4Cfg<D, RT>::WARPS * WARP;
  static_assert(BYTES + 1024 <= 227 * 1024, "shared memory of an SM");
};

template <int D, int RT, bool CAP>
__global__ void __launch_bounds__(Kv4Cfg<D, RT>::WARPS * 32, 1) kv4_attn_kernel(const Kv4AttnArgs a) {
  using P = Kv4<D>;
  using S = Kv4Smem<D, RT>;
  using R = Kv4Rows<RT>;
  constexpr int NG = P::NG, STAGES = S::STAGES, ROWS = R::ROWS, NT = R::NT, NC = R::NC;
  constexpr int BURST = Kv4Cfg<D, RT>::BURST, MATH = Kv4Cfg<D, RT>::MATH, WARPS = Kv4Cfg<D, RT>::WARPS;
  constexpr unsigned ALL = (1u << BURST) - 1, MATH_ALL = (1u << MATH) - 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ volatile int abort_flag;
  __shared__ Kv4Split split;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * S::WARP;
  uint4* qf = reinterpret_cast<uint4*>(ring + S::QF);
  float* col_f = reinterpret_cast<float*>(ring + S::COL);
  float* col_q = col_f + ROWS;  // [ROWS][NG]
  float* col_v = col_q + ROWS * NG;  // [ROWS][NG], where the rows' scalings differ
  int* col_see = reinterpret_cast<int*>(col_v + ROWS * NG);
  int* row_w = col_see + ROWS;    // [ROWS][NG]
  int* row_o = row_w + ROWS * NG;
  float* row_drop = reinterpret_cast<float*>(row_o + ROWS * NG);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + S::BAR);

  pdl_launch_dependents();
  if (lane < STAGES) mbar_init(bars + lane, 1);
  if constexpr (RT == 0)
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) qf[i * 32 + lane] = make_uint4(0u, 0u, 0u, 0u);  // the columns without a row
  fence_barrier_init();
  if (tid == 0) abort_flag = 0;
  __syncthreads();
  pdl_wait();

  // ---- this worker's rounds, [r0, r1) of the batch's total, and the sequence that r0 lies in: every warp scans the
  // lengths by itself, lane j a run of them
  const int subs = a.hkv * a.chunks;
  const int worker = warp * gridDim.x + blockIdx.x;  // few rounds: spread over the SMs
  const int run = (a.batch + 31) / 32, from = min(lane * run, a.batch), to = min(from + run, a.batch);
  int64_t end = 0;  // rounds up to and with the lane's sequences
  for (int b = from; b < to; ++b) end += static_cast<int64_t>(kv4_seq<BURST>(a, b, worker == 0).rounds) * subs;
  int64_t begin = end;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, end, o);
    if (lane >= o) end += y;
  }
  begin = end - begin;
  const int64_t total = __shfl_sync(0xffffffffu, end, 31);
  const int workers = static_cast<int>(min(static_cast<int64_t>(gridDim.x) * WARPS, total));
  if (worker >= workers) return;
  int64_t r0;
  int left;
  {
    Kv4Split mine;
    mine.set(total, workers);
    if (lane == 0) split = mine;  // the same from every warp
    r0 = mine.start(worker);
    left = static_cast<int>(mine.start(worker + 1) - r0);
  }
  int seq = 0;
  Kv4Seq sq = {};
  const bool mine = begin <= r0 && r0 < end;
  if (mine) {
    for (seq = from; seq < to; ++seq) {
      sq = kv4_seq<BURST>(a, seq);
      const int64_t n = static_cast<int64_t>(sq.rounds) * subs;
      if (r0 < begin + n) break;
      begin += n;
    }
  }
  const int owner = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
  seq = __shfl_sync(0xffffffffu, seq, owner);
  sq.ctx = __shfl_sync(0xffffffffu, sq.ctx, owner);
  sq.first = __shfl_sync(0xffffffffu, sq.first, owner);
  sq.last = __shfl_sync(0xffffffffu, sq.last, owner);
  sq.rounds = __shfl_sync(0xffffffffu, sq.rounds, owner);
  const int64_t in_seq = r0 - __shfl_sync(0xffffffffu, begin, owner);
  int sub = in_seq >> 31 ? static_cast<int>(in_seq / sq.rounds) : static_cast<int>(in_seq) / sq.rounds;
  int ra = static_cast<int>(in_seq - static_cast<int64_t>(sub) * sq.rounds);

  // ---- the worker's stream of records, STAGES bursts ahead of the arithmetic.  Up to 32 records of an item are
  // prepared at once, lane j seeing to record j: its block id is asked for a batch ahead, its copy is issued
  // by that lane when its turn comes.
  const int64_t block_bytes = static_cast<int64_t>(a.hkv) * a.recs * P::RECORD;
  int p_seq = seq, p_sub = sub, p_left = left - min(sq.rounds - ra, left);
  Kv4Seq p_sq = sq;
  const int2 p_first = kv4_records<BURST>(a, sq, ra, left - p_left);
  int p_t = p_first.x, p_end = p_first.y;
  int ask_n = 0, ask_id = 0, ask_rec = 0, ask_sub = 0;  // the next batch: records, the lane's block and record in it
  auto ask = [&]() {
    ask_n = 0;
    while (p_t >= p_end) {
      if (p_left <= 0) return;
      if (++p_sub == subs) {
        p_sub = 0;
        p_sq = kv4_seq<BURST>(a, ++p_seq);
      }
      const int n = min(p_sq.rounds, p_left);
      p_left -= n;
      const int2 recs = kv4_records<BURST>(a, p_sq, 0, n);
      p_t = recs.x;
      p_end = recs.y;
    }
    ask_n = min(p_end - p_t, 32);
    ask_sub = p_sub;
    if (lane < ask_n) {
      const int t = p_t + lane, blk = a.recs == 1 ? t : t / a.recs;
      ask_rec = t - blk * a.recs;
      ask_id = a.tables[p_seq * a.table_stride + blk];
    }
    p_t += ask_n;
  };
  int batch_left = 0, turn = 0;   // records of the current batch still to copy; the lane's own among them
  unsigned batch_ok = 0;          // those of them whose block is inside the pool
  const uint8_t* batch_src = a.pool;
  unsigned came = 0;              // the records in the ring whose block is, the current stage's lowest
  int pending = 0;                // stages still to be waited for
  auto issue = [&](int st, int place) {  // into stage st, `place` stages behind the current one
    const bool turned = batch_left <= 0;
    if (turned) {
      if (ask_n == 0) return;
      batch_left = ask_n;
      turn = lane;
      const bool mine = lane < ask_n, good = mine && static_cast<unsigned>(ask_id) < static_cast<unsigned>(a.num_blocks);
      batch_ok = __ballot_sync(0xffffffffu, good);
      if (mine && !good) report(a.err, kDevBadBlock);
      const int h = a.chunks == 1 ? ask_sub : ask_sub / a.chunks;
      if (good) batch_src = a.pool + ask_id * block_bytes + (static_cast<int64_t>(h) * a.recs + ask_rec) * P::RECORD;
    }
    const unsigned ok = batch_ok & ALL;
    batch_ok >>= BURST;
    came |= ok << (place * BURST);
    if constexpr (BURST == 1) {
      if (turn == 0) {
        mbar_arrive_expect_tx(bars + st, ok * P::RECORD);
        if (ok) bulk_load(ring + st * P::RECORD, batch_src, P::RECORD, bars + st);
      }
    } else {
      if (turn == 0) mbar_arrive_expect_tx(bars + st, __popc(ok) * P::RECORD);
      __syncwarp();
      if (static_cast<unsigned>(turn) < BURST && (ok >> turn & 1u))
        bulk_load(ring + (st * BURST + turn) * P::RECORD, batch_src, P::RECORD, bars + st);
    }
    turn -= BURST;
    batch_left -= BURST;
    ++pending;
    if (turned) ask();
  };
  // ---- Q, four rows at a time, eight lanes each; TAKE such passes under way at once, the first ones before any
  // copy, behind which they would wait
  constexpr int PASSES = ROWS / 4, TAKE = RT == 3 ? 3 : RT == 0 ? 1 : 2;
  uint4 raw_q[TAKE][NG];
  auto load_rows = [&](int pass) {
    const int h = a.chunks == 1 ? sub : sub / a.chunks, row0 = (sub - h * a.chunks) * ROWS;
#pragma unroll
    for (int x = 0; x < TAKE; ++x) {
      const int r = row0 + (pass + x) * 4 + (lane >> 3);
      const int i = r / a.group, hq = h * a.group + r - i * a.group;
      const __nv_bfloat16* src = a.q + (static_cast<int64_t>(seq) * a.T + i) * a.q_stride +
                                 static_cast<int64_t>(hq) * D + 8 * (lane & 7);
      const bool there = r < min(row0 + ROWS, a.group * a.T);
#pragma unroll
      for (int k = 0; k < NG; ++k)
        raw_q[x][k] = there ? *reinterpret_cast<const uint4*>(src + 64 * k) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  ask();
  load_rows(0);
#pragma unroll 1
  for (int st = 0; st < STAGES; ++st) issue(st, st);
  int cur = 0;
  uint32_t parity = 0;  // of the ring's current turn
  bool dead = false;

  const int tok0 = tile_token(g), tok1 = tile_token(g + 8);
  int vtok[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) vtok[i] = 4 * c + ((i + c) & 3);

  // ---- items
  auto row_of = [&](int q) { return RT == 0 ? c : (q >> 1) * 8 + 2 * c + (q & 1); };  // row of the lane's column q
  while (left > 0) {
    const int n_rounds = min(sq.rounds - ra, left);
    const int h = a.chunks == 1 ? sub : sub / a.chunks;
    const int row0 = (sub - h * a.chunks) * ROWS;
    const int rows = min(a.group * a.T - row0, ROWS);
    const int2 span = kv4_records<BURST>(a, sq, ra, n_rounds);

    // Q of the item in the order of the first product's operands
    __syncwarp();
#pragma unroll 1
    for (int pass0 = 0; pass0 < PASSES && span.x < span.y; pass0 += TAKE) {
      if (pass0 > 0) load_rows(pass0);
#pragma unroll
      for (int x = 0; x < TAKE; ++x) {
        const int r = (pass0 + x) * 4 + (lane >> 3), w = lane & 7;
        const uint4(&raw)[NG] = raw_q[x];
        if (w == 0) col_see[r] = r < rows ? sq.ctx - a.T + 1 + (row0 + r) / a.group : -(1 << 30);
        uint32_t big = 0;  // bits of the largest magnitude: ordered as integers, NaN and infinity on top
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const uint32_t x[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) big = max(big, max((x[j] << 16) & 0x7fffffffu, x[j] & 0x7fff0000u));
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
        const bool fine = big < 0x7f800000u;
        // times a power of two that puts the largest magnitude into [2^10, 2^11)
        const int e = big > 0 && fine ? min(max(137 - static_cast<int>(big >> 23), -126), 126) : 0;
        const float up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const uint32_t x[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
          float v[8], sum = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = fine ? __uint_as_float((j & 1) ? x[j >> 1] & 0xffff0000u : x[j >> 1] << 16) * up : 0.0f;
            sum += v[j];
          }
          // word w of the group is word w % 2 of lane w / 2; codes 2 h and 2 h + 4 are the first operand of half h,
          // 2 h + 1 and 2 h + 5 the second, which stands 4 bits higher
          const int col = RT == 0 ? 2 * r : r % 8;
          qf[((k * 2 + (w & 1)) * NT + (RT == 0 ? 0 : r / 8)) * 32 + col * 4 + (w >> 1)] =
              make_uint4(pack_f16(v[0] * 16.0f, v[4] * 16.0f), pack_f16(v[1], v[5]),
                         pack_f16(v[2] * 16.0f, v[6] * 16.0f), pack_f16(v[3], v[7]));
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          if (w == 0) col_q[r * NG + k] = sum;
        }
        if (w == 0) col_f[r] = !fine ? __int_as_float(0x7fc00000) : ldexpf(a.score_scale, -e);
      }
    }
    __syncwarp();

    auto load_f = [&](float (&f)[NC]) {
#pragma unroll
      for (int q = 0; q < NC; ++q) f[q] = col_f[row_of(q)];
    };
    auto load_qs = [&](float (&qs)[NC][NG]) {
#pragma unroll
      for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int k = 0; k < NG; ++k) qs[q][k] = col_q[row_of(q) * NG + k];
    };
    float f_item[NC], qs_item[NC][NG];
    if constexpr (R::HOLD_Q) load_f(f_item), load_qs(qs_item);
    const int see_least = col_see[0], see_most = col_see[rows - 1];  // keys that the first and the last row see

    // m tiles of 16 x 8 outputs.  RT > 0: (group, high half of the word, half of that), 16 channels x 8 rows each;
    // RT = 0: (group, half of a half word), 32 channels x 4 rows
    constexpr int OT = (RT == 0 ? 2 : 4) * NG;
    float o[OT][NT][4];
    float l[NC], mref[NC], mo[NC][NG];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < OT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][nt][e] = 0.0f;
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      l[q] = 0.0f;
      mref[q] = row_of(q) < rows ? kNone : kFltMax;  // a column without a row: no score passes it
#pragma unroll
      for (int k = 0; k < NG; ++k) mo[q][k] = 0.0f;
    }
    // Scaling of the products p s' per group: the lane's row's (RT = 0), or the largest of the rows', which is that of
    // all of them while `same`
    float vscale[NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) vscale[k] = power_of_2(kFirstScale);
    bool same = true;
    bool none = true;  // no reference chosen: nothing summed yet

    auto load_v = [&](float (&v)[NC][NG]) {
#pragma unroll
      for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int k = 0; k < NG; ++k) v[q][k] = vscale[k];
      if (RT > 0 && !same)
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
          for (int k = 0; k < NG; ++k) v[q][k] = col_v[row_of(q) * NG + k];
    };
    // MATH records from record t on, or with MASKED one: some row does not see some token, or the rows' scalings differ
    // or have to be chosen one by one; without it the records are left undone, false, where they have.
    auto burst = [&](auto masked_tag, int t, const uint8_t* recs) -> bool {
      constexpr bool MASKED = decltype(masked_tag)::value;
      constexpr int N = MASKED ? 1 : MATH;  // records
      asm volatile("" ::: "memory");  // Q is read from shared memory each time: held in registers it would spill
      float f_own[NC], qs_own[NC][NG];
      if constexpr (!R::HOLD_Q) load_f(f_own), load_qs(qs_own);
      const float(&f)[NC] = R::HOLD_Q ? f_item : f_own;
      const float(&qs)[NC][NG] = R::HOLD_Q ? qs_item : qs_own;
      // ---- scores
      float s[N][2][NC];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const uint8_t* rec = recs + u * P::RECORD;
        uint32_t kw[2][2 * NG], kp[2][NG];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          load_words(rec + (e ? tok1 : tok0) * P::ROW + c * (8 * NG), kw[e]);
          load_words(rec + P::K_PAIRS + (e ? tok1 : tok0) * P::PAIRS, kp[e]);
        }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          float acc[NT][4];
#pragma unroll
          for (int wi = 0; wi < 2; ++wi) {
            uint4 b[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) b[nt] = qf[((k * 2 + wi) * NT + nt) * 32 + lane];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint32_t x0 = kw[0][NG * wi + k] >> (8 * hh), x1 = kw[1][NG * wi + k] >> (8 * hh);
              const uint32_t a0 = x0 & 0x000F000Fu, a1 = x1 & 0x000F000Fu, a2 = x0 & 0x00F000F0u,
                             a3 = x1 & 0x00F000F0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t b0 = hh ? b[nt].z : b[nt].x, b1 = hh ? b[nt].w : b[nt].y;
                if (wi + hh == 0)
                  mma_f16_16816_zero(acc[nt], a0, a1, a2, a3, b0, b1);
                else
                  mma_f16_16816(acc[nt], a0, a1, a2, a3, b0, b1);
              }
            }
          }
          // The products are 2^-20 of what they stand for: made good on the scales, so that neither a row's factor nor
          // a small key's score leaves fp32's range.  Two scores at a time: of both tokens of the row (RT = 0), or of
          // two rows.
          const F2 scales = mul2({pair_scale(kp[0][k]), pair_scale(kp[1][k])}, {0x1p20f, 0x1p20f});
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const int e = RT == 0 ? 0 : i & 1, q = RT == 0 ? 0 : i & ~1;
            const int e1 = RT == 0 ? 1 : e, q1 = RT == 0 ? 0 : q + 1;
            const int nt = (q >> 1) % NT;
            const F2 dot = {acc[nt][2 * e], RT == 0 ? acc[nt][2] : acc[nt][2 * e + 1]};
            const F2 ps = {e ? scales.y : scales.x, e1 ? scales.y : scales.x};
            const F2 pm = {pair_min(kp[e][k]), pair_min(kp[e1][k])};
            const F2 part = k == 0 ? mul2(ps, dot) : fma2(ps, dot, {s[u][e][q], s[u][e1][q1]});
            const F2 sum = fma2(pm, {qs[q][k], qs[q1][k]}, part);
            s[u][e][q] = sum.x, s[u][e1][q1] = sum.y;
          }
        }
        if constexpr (CAP)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int q = 0; q < NC; ++q) s[u][e][q] = a.cap_log2 * tanh_exp(s[u][e][q] * f[q]);
      }
      // ---- distance of the scores to their references; the value scales as operands
      uint32_t vp[N][2][NG];
      unsigned in[N] = {};  // bit e * NC + q
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const uint8_t* rec = recs + u * P::RECORD;
#pragma unroll
        for (int e = 0; e < 2; ++e) load_words(rec + P::V_PAIRS + (e ? tok1 : tok0) * P::PAIRS, vp[u][e]);
        if constexpr (MASKED) {
          int see[NC];
#pragma unroll
          for (int q = 0; q < NC; ++q) see[q] = col_see[row_of(q)];
          const int low = a.window > 0 ? see_least - a.window : 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at = (t + u) * kKv4Tokens + (e ? tok1 : tok0);
                        if (!(at < see_most && at >= low))  // no row sees the token: its pairs hold anything
#pragma unroll
              for (int k = 0; k < NG; ++k) vp[u][e][k] = 0;
#pragma unroll
            for (int q = 0; q < NC; ++q)
              in[u] |= static_cast<unsigned>(at < see[q] && (a.window <= 0 || at >= see[q] - a.window))
                       << (e * NC + q);
          }
        }
      }
      auto distance = [&](int u, int e, int q) {
        const float x = CAP ? s[u][e][q] - mref[q] : fmaf(s[u][e][q], f[q], -mref[q]);
        return !MASKED || (in[u] >> (e * NC + q) & 1u) ? x : -INFINITY;
      };
      auto score = [&](int u, int e, int q) {
        const float x = CAP ? s[u][e][q] : s[u][e][q] * f[q];
        return !MASKED || (in[u] >> (e * NC + q) & 1u) ? x : -INFINITY;
      };
      float d[N][2][NC], vs[N][2][NG];
      float far = -INFINITY, top = 0.0f;
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if constexpr (!MASKED && RT > 0 && !CAP) {
#pragma unroll
            for (int q = 0; q < NC; q += 2) {
              const F2 x = fma2({s[u][e][q], s[u][e][q + 1]}, {f[q], f[q + 1]}, {-mref[q], -mref[q + 1]});
              d[u][e][q] = x.x, d[u][e][q + 1] = x.y;
            }
          } else {
#pragma unroll
            for (int q = 0; q < NC; ++q) d[u][e][q] = distance(u, e, q);
          }
#pragma unroll
          for (int q = 0; q < NC; ++q) far = fmaxf(far, d[u][e][q]);
#pragma unroll
          for (int k = 0; k < NG; k += 2) {
            const F2 x = mul2({pair_scale(vp[u][e][k]), pair_scale(vp[u][e][(k + 1) % NG])},
                              {vscale[k], vscale[(k + 1) % NG]});
            vs[u][e][k] = x.x;
            if (k + 1 < NG) vs[u][e][(k + 1) % NG] = x.y;
          }
#pragma unroll
          for (int k = 0; k < NG; ++k) top = fmaxf(top, vs[u][e][k]);
        }
      // ---- new references and scalings, where a score or a value scale outgrew them
      if (__any_sync(0xffffffffu, far > kSlack || top > kScaleMax)) {
        const bool empty = none;
        float m[NC];  // the references to be
#pragma unroll
        for (int q = 0; q < NC; ++q) {
          m[q] = -INFINITY;
#pragma unroll
          for (int u = 0; u < N; ++u) m[q] = fmaxf(m[q], fmaxf(score(u, 0, q), score(u, 1, q)));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) m[q] = fmaxf(m[q], __shfl_xor_sync(0xffffffffu, m[q], off));
          m[q] = fmaxf(m[q], mref[q]);
        }
        // Where s' is within kScaleMax and above 2^0 for the tokens that set new references, both as scaled now, nothing
        // but references changes.  The first scaling puts the largest s' into [2^7, 2^8).
        bool plain = RT == 0 || same;
        bool light[N][2] = {};  // tokens of a smaller s'
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          float hi = 0.0f;
#pragma unroll
          for (int u = 0; u < N; ++u) hi = fmaxf(hi, fmaxf(pair_scale(vp[u][0][k]), pair_scale(vp[u][1][k])));
          if (empty) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
            vscale[k] = power_of_2(choose_scale(kFirstScale, log2_of(hi), kNothing, kNothing));
          }
          plain = plain && hi * vscale[k] <= kScaleMax;
#pragma unroll
          for (int u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) light[u][e] = light[u][e] || !(pair_scale(vp[u][e][k]) * vscale[k] >= 1.0f);
        }
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
          for (int u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) plain = plain && !(light[u][e] && m[q] > mref[q] && score(u, e, q) == m[q]);
        plain = __all_sync(0xffffffffu, plain);
        if constexpr (!MASKED)
          if (__builtin_expect(!plain, 0)) return false;
        none = false;
        float fac[NC];
#pragma unroll
        for (int q = 0; q < NC; ++q) {
          fac[q] = ex2(mref[q] - m[q]);
          if (MASKED && !plain && g == 0) row_drop[row_of(q)] = fmaxf(mref[q] - m[q], -1000.0f);
          mref[q] = m[q];
          l[q] *= fac[q];
#pragma unroll
          for (int k = 0; k < NG; ++k) mo[q][k] *= fac[q];
#pragma unroll
          for (int u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) d[u][e][q] = distance(u, e, q);
        }
        if (__builtin_expect(plain, 1)) {
          if (!empty) {
#pragma unroll
            for (int k = 0; k < OT; ++k)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k][nt][e] *= fac[RT == 0 ? 0 : (nt * 2 + (e & 1)) % NC];
          } else if constexpr (!MASKED) {
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < NG; ++k) vs[u][e][k] = pair_scale(vp[u][e][k]) * vscale[k];
          }
        } else if constexpr (MASKED) {
          // Row by row and group by group, from the largest product and the largest sum of each, which a lane looks at:
          // code that hardly ever runs is to be small, as every kernel of 16 rows and more outgrows the instruction
          // cache (5 query tokens of 64 sequences of 2048: 94 us with all of it unrolled, 81 like this, 77 since records
          // that all rows see whole are not masked).
          for (int i = lane; i < ROWS * NG; i += 32) row_w[i] = row_o[i] = 0;
          if (RT == 0 || same)
#pragma unroll
            for (int q = 0; q < NC; ++q)
#pragma unroll
              for (int k = 0; k < NG; ++k)
                if (g == 0) col_v[row_of(q) * NG + k] = vscale[k];
          __syncwarp();
          float smax[NG];
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const float p0 = pair_scale(vp[0][0][k]), p1 = pair_scale(vp[0][1][k]);
            const float s0 = p0 <= kFltMax ? p0 : 0.0f, s1 = p1 <= kFltMax ? p1 : 0.0f;
            smax[k] = fmaxf(s0, s1);
#pragma unroll
            for (int q = 0; q < NC; ++q) {
              float sum = 0.0f;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float(&y)[4] = RT == 0 ? o[(k * 2 + x % 2) % OT][0] : o[(k * 4 + x) % OT][q >> 1];
                const int at = RT == 0 ? x / 2 : q & 1;
                sum = fmaxf(sum, fmaxf(y[at], y[at + 2] * 0x1p-4f));
              }
              const float w = fmaxf(fmaxf(ex2(d[0][0][q]) * s0, ex2(d[0][1][q]) * s1), 0.0f);
              atomicMax(row_w + row_of(q) * NG + k, __float_as_int(w));  // above zero bits are ordered as the numbers
              atomicMax(row_o + row_of(q) * NG + k, __float_as_int(sum));
            }
          }
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) smax[k] = fmaxf(smax[k], __shfl_xor_sync(0xffffffffu, smax[k], off));
          __syncwarp();
          int most = kNothing, least = -kNothing;  // of the lane's group, over the rows that anything weighs in
          float mine = smax[0];
#pragma unroll
          for (int k = 1; k < NG; ++k) mine = lane % NG == k ? smax[k] : mine;
          const int s_log = log2_of(mine);
#pragma unroll 1
          for (int i = lane; i < ROWS * NG; i += 32) {
            const float w = __int_as_float(row_w[i]), sum = __int_as_float(row_o[i]), drop = row_drop[i / NG];
            const int old = log2_of(col_v[i]);
            int chosen = kNothing;
            if (RT == 0 || w > 0.0f || sum > 0.0f) {
              // o holds code times product times 2^-24, at most 15 of the first
              chosen = choose_scale(old, s_log, log2_of(w),
                                    sum > 0.0f ? log2_of(sum) + 20 + __float2int_rd(drop) - old : kNothing);
              most = max(most, chosen);
              least = min(least, chosen);
              col_v[i] = power_of_2(chosen);
            }
            row_w[i] = chosen;
            row_o[i] = __float_as_int(sum > 0.0f ? ldexpf(ex2(drop), chosen - old) : 1.0f);  // what o is multiplied by
          }
          if constexpr (RT > 0) {
#pragma unroll
            for (int off = NG; off < 32; off <<= 1) {
              most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
              least = min(least, __shfl_xor_sync(0xffffffffu, least, off));
            }
            if (most == kNothing) {
              float v = vscale[0];
#pragma unroll
              for (int k = 1; k < NG; ++k) v = lane % NG == k ? vscale[k] : v;
              most = least = choose_scale(log2_of(v), s_log, kNothing, kNothing);
            }
#pragma unroll 1
            for (int i = lane; i < ROWS * NG; i += 32)
              if (row_w[i] == kNothing) col_v[i] = power_of_2(most);
            same = __all_sync(0xffffffffu, most == least);
#pragma unroll
            for (int k = 0; k < NG; ++k) vscale[k] = __shfl_sync(0xffffffffu, power_of_2(most), k);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            if constexpr (RT == 0) vscale[k] = col_v[row_of(0) * NG + k];
#pragma unroll
            for (int q = 0; q < NC; ++q) {
              const float f = __int_as_float(row_o[row_of(q) * NG + k]);
#pragma unroll
              for (int x = 0; x < (RT == 0 ? 2 : 4); ++x) {
                float(&y)[4] = RT == 0 ? o[(k * 2 + x) % OT][0] : o[(k * 4 + x) % OT][q >> 1];
#pragma unroll
                for (int j = 0; j < (RT == 0 ? 4 : 2); ++j) y[RT == 0 ? j : 2 * j + (q & 1)] *= f;
              }
            }
          }
          __syncwarp();
        }
      }
      // ---- weights, and outputs
      float v[NC][NG];
      if constexpr (MASKED) load_v(v);
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const uint8_t* rec = recs + u * P::RECORD;
        uint32_t vw[4][NG];
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words(rec + P::V_CODES + vtok[i] * P::ROW + 4 * NG * g, vw[i]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int q = 0; q < NC; ++q) {
            d[u][e][q] = ex2(d[u][e][q]);
            l[q] += d[u][e][q];
          }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          uint32_t b[NT][2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float w[NC];
            if constexpr (!MASKED && RT == 0 && NG > 1) {
              if (k % 2 == 0) {  // two groups at a time, the second one's weight kept for its turn
                const F2 p = {d[u][e][0], d[u][e][0]}, x = mul2(p, {vs[u][e][k], vs[u][e][(k + 1) % NG]});
                const F2 m = {pair_min(vp[u][e][k]), pair_min(vp[u][e][(k + 1) % NG])};
                const F2 y = fma2(p, m, {mo[0][k], mo[0][(k + 1) % NG]});
                vs[u][e][k] = x.x, vs[u][e][(k + 1) % NG] = x.y;
                mo[0][k] = y.x, mo[0][(k + 1) % NG] = y.y;
              }
              w[0] = vs[u][e][k];
            } else if constexpr (!MASKED && RT > 0) {
              const float pm = pair_min(vp[u][e][k]), ps = vs[u][e][k];
#pragma unroll
              for (int q = 0; q < NC; q += 2) {
                const F2 p = {d[u][e][q], d[u][e][q + 1]}, x = mul2(p, {ps, ps});
                const F2 y = fma2(p, {pm, pm}, {mo[q][k], mo[q + 1][k]});
                w[q] = x.x, w[q + 1] = x.y;
                mo[q][k] = y.x, mo[q + 1][k] = y.y;
              }
            } else if constexpr (MASKED) {
#pragma unroll
              for (int q = 0; q < NC; ++q) {
                const bool x = in[u] >> (e * NC + q) & 1u;  // a NaN pair that only later rows see
                w[q] = x ? d[u][e][q] * v[q][k] * pair_scale(vp[u][e][k]) : 0.0f;
                mo[q][k] += x ? d[u][e][q] * pair_min(vp[u][e][k]) : 0.0f;
              }
            } else {
              w[0] = d[u][e][0] * vs[u][e][k];
              mo[0][k] = fmaf(d[u][e][0], pair_min(vp[u][e][k]), mo[0][k]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              b[nt][e] = transposed(RT == 0 ? pack_f16(w[0], w[0]) : pack_f16(w[2 * nt % NC], w[(2 * nt + 1) % NC]));
          }
          if constexpr (RT == 0) {
            // Both halves of a masked word are operands of one token: channel j in its low half, j + 4 in its high one.
            // Column 2 r takes the weight of row r against the low halves, column 2 r + 1 against the high ones.
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // tokens vtok[2 e], vtok[2 e + 1]
              const uint32_t b0 = __byte_perm(b[0][e], 0, g & 1 ? 0x1044 : 0x4410);
              const uint32_t b1 = __byte_perm(b[0][e], 0, g & 1 ? 0x3244 : 0x4432);
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const uint32_t x0 = vw[2 * e][k] >> (8 * hh), x1 = vw[2 * e + 1][k] >> (8 * hh);
                mma_f16_16816(o[(k * 2 + hh) % OT][0], x0 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x000F000Fu,
                              x1 & 0x00F000F0u, b0, b1);
              }
            }
            continue;
          }
#pragma unroll
          for (int hv = 0; hv < 2; ++hv) {
            const uint32_t y0 = __byte_perm(vw[0][k], vw[1][k], hv ? 0x7632 : 0x5410);
            const uint32_t y1 = __byte_perm(vw[2][k], vw[3][k], hv ? 0x7632 : 0x5410);
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint32_t x0 = y0 >> (8 * hh), x1 = y1 >> (8 * hh);
              const uint32_t a0 = x0 & 0x000F000Fu, a1 = x0 & 0x00F000F0u, a2 = x1 & 0x000F000Fu,
                             a3 = x1 & 0x00F000F0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16_16816(o[((k * 2 + hv) * 2 + hh) % OT][nt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
            }
          }
        }
      }
      return true;
    };

    // MATH records from one in [t_low, t_high] on hold no token that some row does not see
    const int t_low = a.window > 0 ? max(see_most - a.window + kKv4Tokens - 1, 0) / kKv4Tokens : 0;
    const int t_high = max(see_least, 0) / kKv4Tokens - MATH;
    for (int t = dead ? span.y : span.x; t < span.y; t += BURST) {  // given up: the items still get an entry
      if (!__all_sync(0xffffffffu, mbar_try_wait(smem_u32(bars + cur), parity)) &&
          !__all_sync(0xffffffffu, wait_slow(bars + cur, parity, &abort_flag, a.err))) {
        dead = true;
        break;
      }
      const unsigned have = came & ALL;
      const uint8_t* recs = ring + cur * (BURST * P::RECORD);
#pragma unroll 1
      for (int x = 0; x < BURST; x += MATH) {
        const bool all_seen = (have >> x & MATH_ALL) == MATH_ALL && t + x >= t_low && t + x <= t_high;
        if (all_seen && same && burst(std::false_type{}, t + x, recs + x * P::RECORD)) continue;
#pragma unroll 1
        for (int y = x; y < x + MATH; ++y)  // a record without a block inside the pool: its tokens count as masked
          if (have >> y & 1u) burst(std::true_type{}, t + y, recs + y * P::RECORD);
      }
      __syncwarp();
      came >>= BURST;
      --pending;
      issue(cur, STAGES - 1);
      if (++cur == STAGES) cur = 0, parity ^= 1u;
    }
    // ---- the item's result, or this worker's part of it
#pragma unroll
    for (int q = 0; q < NC; ++q) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[q] += __shfl_xor_sync(0xffffffffu, l[q], off);
#pragma unroll
        for (int k = 0; k < NG; ++k) mo[q][k] += __shfl_xor_sync(0xffffffffu, mo[q][k], off);
      }
    }
    const bool whole = ra == 0 && n_rounds == sq.rounds;
    if (ra == 0 && lane == 0 && a.items != nullptr) {  // nullptr: items are not split
      Kv4Item it;
      it.first = worker;
      it.last = whole ? worker : split.worker(split.start(worker + 1) - left + sq.rounds - 1);
      a.items[static_cast<int64_t>(seq) * subs + sub] = it;
    }
    float v_item[NC][NG];
    load_v(v_item);
    const int64_t slot = 2 * static_cast<int64_t>(worker) + (ra == 0 ? 1 : 0);
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const int r = row_of(q), nt = q >> 1, j = q & 1;
      if (r >= rows) continue;
      const int i = (row0 + r) / a.group, hq = h * a.group + (row0 + r) - i * a.group;
      __nv_bfloat16* dst =
          a.out + (static_cast<int64_t>(seq) * a.T + i) * a.out_stride + static_cast<int64_t>(hq) * D + 8 * g;
      float* part = a.part_o + (slot * ROWS + r) * D + 8 * g;
      const float over = l[q] == 0.0f ? 0.0f : 1.0f / l[q];
      if (!whole && g == 0) a.part_ml[slot * ROWS + r] = make_float2(mref[q], l[q]);
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float inv = 1.0f / v_item[q][k];
        float v[8];  // channels 8 g + 4 hv + 2 hh (codes as u 2^-24) and the next one (u 2^-20)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float(&y)[4] = RT == 0 ? o[(k * 2 + x % 2) % OT][0] : o[(k * 4 + x) % OT][nt];
          const int at = RT == 0 ? x / 2 : j;
          v[2 * x] = fmaf(y[at] * 0x1p24f, inv, mo[q][k]);
          v[2 * x + 1] = fmaf(y[at + 2] * 0x1p20f, inv, mo[q][k]);
        }
        if (whole) {
          *reinterpret_cast<uint4*>(dst + 64 * k) =
              make_uint4(pack_bf16(v[0] * over, v[1] * over), pack_bf16(v[2] * over, v[3] * over),
                         pack_bf16(v[4] * over, v[5] * over), pack_bf16(v[6] * over, v[7] * over));
        } else {
          *reinterpret_cast<float4*>(part + 64 * k) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(part + 64 * k + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
      }
    }
    left -= n_rounds;
    if (left <= 0) break;
    ra = 0;
    if (++sub == subs) {
      sub = 0;
      sq = kv4_seq<BURST>(a, ++seq);
    }
    load_rows(0);
  }
  // a stream that was given up: its copies land before the block's shared memory goes
  if (dead)
    for (; pending > 0; --pending) {
      mbar_wait(bars + cur, parity, nullptr, a.err);
      if (++cur == STAGES) cur = 0, parity ^= 1u;
    }
}

// Adds parts p0, p0 + STEP, .. up to the last of row r of an item to (m, l, o), AHEAD of them under way at once.
template <int D, int RT, int STEP, int AHEAD>
__device__ __forceinline__ void kv4_join_parts(const Kv4AttnArgs& a, const Kv4Item& it, int p0, int r, int lane, float& m,
                                               float& l, float (&o)[D / 32]) {
  constexpr int ROWS = Kv4Rows<RT>::ROWS, N = D / 32;
  for (; p0 <= it.last; p0 += STEP * AHEAD) {
    float2 e[AHEAD];
    float y[AHEAD][N];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int p = p0 + i * STEP;
      const int64_t slot = (2 * static_cast<int64_t>(p) + (p == it.first ? 1 : 0)) * ROWS + r;
      e[i] = make_float2(kNone, 0.0f);
      if (p <= it.last) e[i] = a.part_ml[slot];
#pragma unroll
      for (int j = 0; j < N; ++j) y[i][j] = p <= it.last ? a.part_o[slot * D + 32 * j + lane] : 0.0f;
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, e[i].x);
    const float fm = ex2(m - top);
    l *= fm;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= fm;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float fe = ex2(e[i].x - top);
      l = fmaf(e[i].y, fe, l);
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = fmaf(y[i][j], fe, o[j]);
    }
    m = top;
  }
}

// Joins the parts of the items that span workers.  A block of WARPS warps takes PAIRS (item, row) pairs, one per
// warp: a pair of few parts is that warp's, in worker order; a pair of many is the whole block's, the warps
// taking turns.
constexpr int kFewParts = 16;
template <int D, int RT, int PAIRS, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) kv4_join_kernel(const Kv4AttnArgs a) {
  constexpr int ROWS = Kv4Rows<RT>::ROWS, N = D / 32;
  constexpr int FEW = kFewParts, AHEAD = WARPS == 32 ? 512 / D : D == 256 ? 4 : 8;
  __shared__ float acc[WARPS][D];
  __shared__ float2 ml[WARPS];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, subs = a.hkv * a.chunks;
  const int64_t work = static_cast<int64_t>(a.batch) * subs * a.chunk_rows;
  for (int64_t x0 = static_cast<int64_t>(blockIdx.x) * PAIRS; x0 < work; x0 += static_cast<int64_t>(gridDim.x) * PAIRS) {
    // lane j of every warp looks at pair x0 + j
    const int64_t x = x0 + lane;
    const bool mine = lane < PAIRS && x < work;
    const int64_t item = x >> 31 ? x / a.chunk_rows : static_cast<uint32_t>(x) / static_cast<uint32_t>(a.chunk_rows);
    const int row = static_cast<int>(x - item * a.chunk_rows);
    Kv4Item it = {0, 0};
    if (mine) it = a.items[item];
    const int seq = static_cast<int>(item / subs), sub = static_cast<int>(item - static_cast<int64_t>(seq) * subs);
    const int h = sub / a.chunks, at = (sub - h * a.chunks) * ROWS + row;  // row of the KV head
    const bool split = mine && it.first < it.last && at < a.group * a.T;
    const int64_t dst_at = (static_cast<int64_t>(seq) * a.T + at / a.group) * a.out_stride +
                           static_cast<int64_t>(h * a.group + at % a.group) * D;
    const bool shared = PAIRS == 1 || it.last - it.first >= FEW;
    const unsigned many = __ballot_sync(0xffffffffu, split && shared), few = __ballot_sync(0xffffffffu, split && !shared);
    float m = kNone, l = 0.0f, o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = 0.0f;
    if (PAIRS > 1 && (few >> warp & 1u)) {
      Kv4Item one;
      one.first = __shfl_sync(0xffffffffu, it.first, warp);
      one.last = __shfl_sync(0xffffffffu, it.last, warp);
      const int r = __shfl_sync(0xffffffffu, row, warp);
      __nv_bfloat16* dst = a.out + __shfl_sync(0xffffffffu, dst_at, warp);
      kv4_join_parts<D, RT, 1, AHEAD>(a, one, one.first, r, lane, m, l, o);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int j = 0; j < N; ++j) dst[32 * j + lane] = __float2bfloat16_rn(o[j] * inv);
    }
    for (unsigned left = many; left != 0; left &= left - 1) {
      const int k = __ffs(left) - 1;
      Kv4Item one;
      one.first = __shfl_sync(0xffffffffu, it.first, k);
      one.last = __shfl_sync(0xffffffffu, it.last, k);
      const int r = __shfl_sync(0xffffffffu, row, k);
      __nv_bfloat16* dst = a.out + __shfl_sync(0xffffffffu, dst_at, k);
      m = kNone, l = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = 0.0f;
      kv4_join_parts<D, RT, WARPS, AHEAD>(a, one, one.first + warp, r, lane, m, l, o);
      __syncthreads();  // the pair before has been read
      if (lane == 0) ml[warp] = make_float2(m, l);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[warp][32 * j + lane] = o[j];
      __syncthreads();
      float top = kNone;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[w].x);
      for (int ch = threadIdx.x; ch < D; ch += 32 * WARPS) {
        float sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float f = ex2(ml[w].x - top);
          sum += ml[w].y * f;
          v += acc[w][ch] * f;
        }
        dst[ch] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : v / sum);
      }
    }
  }
}

// How a call is cut: by its query rows per KV head and the head size.
struct Kv4Plan {
  int rt, rows, burst, warps;  // rows of a chunk at most
  int64_t chunks, grid;
  int64_t items_at, ml_at, o_at, bytes;  // workspace
};
template <int D, int RT>
void kv4_plan_rows(Kv4Plan& p, int64_t sms) {
  p.rt = RT;
  p.rows = Kv4Rows<RT>::ROWS;
  p.burst = Kv4Cfg<D, RT>::BURST;
  p.warps = Kv4Cfg<D, RT>::WARPS;
  p.grid = sms;
}
template <int D>
void kv4_plan_dim(Kv4Plan& p, int64_t rows, int64_t sms) {
  // The class of rows is the one of equal chunks; chunks are cut at its ROWS, so the last one may be smaller: 33 rows of
  // 128 are 24 and 9, 49 are 24, 24 and 1.  Every chunk reads the whole cache.
  const int64_t most = D == 256 ? 16 : 24, chunks = (rows + most - 1) / most, per = (rows + chunks - 1) / chunks;
  if (per <= 4) kv4_plan_rows<D, 0>(p, sms);
  else if (per <= 8) kv4_plan_rows<D, 1>(p, sms);
  else if (per <= 16 || D == 256) kv4_plan_rows<D, 2>(p, sms);
  else kv4_plan_rows<D, 3>(p, sms);
}
Kv4Plan kv4_plan(int64_t sms, int64_t head_dim, int64_t rows, int64_t batch, int64_t hkv) {
  Kv4Plan p = {};
  if (head_dim == 64) kv4_plan_dim<64>(p, rows, sms);
  else if (head_dim == 128) kv4_plan_dim<128>(p, rows, sms);
  else kv4_plan_dim<256>(p, rows, sms);
  p.chunks = (rows + p.rows - 1) / p.rows;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  p.items_at = 0;
  p.ml_at = p.items_at + up(batch * hkv * p.chunks * static_cast<int64_t>(sizeof(Kv4Item)));
  p.o_at = p.ml_at + up(2 * p.grid * p.warps * p.rows * 8);
  p.bytes = p.o_at + 2 * p.grid * p.warps * p.rows * head_dim * 4;
  return p;
}

template <int D, int RT, bool CAP>
int kv4_launch_cap(const Kv4AttnArgs& a, int64_t grid, int64_t join_grid, int pairs, cudaStream_t st) {
  constexpr size_t smem = Kv4Smem<D, RT>::BYTES;
  static std::atomic<uint64_t> done{0};
  MVB_TRY(set_smem_once(done, kv4_attn_kernel<D, RT, CAP>, smem, "kv4_attention"));
  MVB_TRY(launch("kv4_attention", kv4_attn_kernel<D, RT, CAP>, dim3(static_cast<unsigned>(grid)),
                 dim3(Kv4Cfg<D, RT>::WARPS * 32), smem,
                 st, a));
  if (join_grid == 0) return MVB_OK;
  const dim3 blocks(static_cast<unsigned>(join_grid));
  const char* what = "kv4_attention_join";  // pairs: 8; 1; 0 = 1 and a block of 32 warps
  if (pairs > 1) return launch_dependent(what, kv4_join_kernel<D, RT, 8, 8>, blocks, dim3(256), 0, st, a);
  if (pairs == 0) return launch_dependent(what, kv4_join_kernel<D, RT, 1, 32>, blocks, dim3(1024), 0, st, a);
  return launch_dependent(what, kv4_join_kernel<D, RT, 1, 8>, blocks, dim3(256), 0, st, a);
}

template <int D, int RT>
int kv4_launch_rows(const Kv4AttnArgs& a, int64_t grid, int64_t join_grid, int pairs, cudaStream_t st) {
  return a.cap_log2 > 0.0f ? kv4_launch_cap<D, RT, true>(a, grid, join_grid, pairs, st)
                           : kv4_launch_cap<D, RT, false>(a, grid, join_grid, pairs, st);
}

template <int D>
int kv4_launch(const Kv4AttnArgs& a, int rt, int64_t grid, int64_t join_grid, int pairs, cudaStream_t st) {
  switch (rt) {
    case 0: return kv4_launch_rows<D, 0>(a, grid, join_grid, pairs, st);
    case 1: return kv4_launch_rows<D, 1>(a, grid, join_grid, pairs, st);
    case 2: return kv4_launch_rows<D, 2>(a, grid, join_grid, pairs, st);
    default: break;
  }
  if constexpr (D < 256) return kv4_launch_rows<D, 3>(a, grid, join_grid, pairs, st);
  return fail(MVB_ERR_UNSUPPORTED, "kv4_attention: rows");
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int64_t mvb_paged_attention_decode_kv4_workspace_bytes(int64_t batch, int64_t query_len,
                                                                  int64_t num_q_heads, int64_t num_kv_heads,
                                                                  int64_t head_dim, int device) {
  if (batch <= 0 || num_kv_heads <= 0 || query_len <= 0) return 0;
  int sms = mvb_num_sms(device);
  if (sms <= 0) sms = 148;
  return kv4_plan(sms, head_dim, num_q_heads / num_kv_heads * query_len, batch, num_kv_heads).bytes;
}

extern "C" int mvb_paged_attention_decode_kv4(void* out, int64_t out_stride, const void* q, int64_t q_stride,
                                              const void* kv4, const int32_t* block_tables, int64_t table_stride,
                                              int64_t max_blocks, const int32_t* ctx_lens, int64_t batch,
                                              int64_t query_len, int64_t num_q_heads, int64_t num_kv_heads,
                                              int64_t head_dim, int64_t num_layers, int64_t layer,
                                              int64_t num_blocks, int64_t block_size, float scale, float softcap,
                                              int64_t window, void* workspace, int64_t workspace_bytes,
                                              mvb_stream_t stream) {
  const char* what = "mvb_paged_attention_decode_kv4";
  MVB_REQUIRE(batch >= 0 && batch <= 65536, "%s: batch %lld (at most 65536)", what, (long long)batch);
  MVB_REQUIRE(query_len >= 1 && query_len <= 1024, "%s: %lld query tokens (1 to 1024)", what, (long long)query_len);
  MVB_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0 && num_q_heads <= 4096,
              "%s: %lld query heads over %lld KV heads", what, (long long)num_q_heads, (long long)num_kv_heads);
  MVB_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: head_dim %lld (64, 128 or 256)", what,
              (long long)head_dim);
  MVB_REQUIRE(layer >= 0 && layer < num_layers, "%s: layer %lld of %lld", what, (long long)layer,
              (long long)num_layers);
  MVB_REQUIRE(block_size > 0 && block_size % 16 == 0 && block_size <= (1 << 20), "%s: block_size %lld", what,
              (long long)block_size);
  MVB_REQUIRE(num_blocks > 0 && num_blocks <= (int64_t(1) << 31) / (block_size / 16) && num_blocks <= INT_MAX,
              "%s: %lld blocks", what, (long long)num_blocks);
  MVB_REQUIRE(max_blocks > 0 && max_blocks <= (int64_t(1) << 30) / block_size, "%s: %lld blocks a sequence", what,
              (long long)max_blocks);
  MVB_REQUIRE(window >= 0 && softcap >= 0.0f && softcap <= kFltMax && fabsf(scale) <= kFltMax &&
                  (softcap == 0.0f || fabsf(scale / softcap) <= kFltMax),
              "%s: window, softcap or scale", what);
  if (batch == 0) return MVB_OK;
  MVB_REQUIRE(out && q && kv4 && block_tables && ctx_lens, "%s: null pointer", what);
  MVB_REQUIRE(table_stride >= max_blocks, "%s: table_stride %lld < max_blocks %lld", what, (long long)table_stride,
              (long long)max_blocks);
  MVB_REQUIRE(q_stride >= num_q_heads * head_dim && out_stride >= num_q_heads * head_dim && q_stride % 8 == 0 &&
                  out_stride % 8 == 0 && aligned(q, 16) && aligned(out, 16) && aligned(kv4, 16),
              "%s: q, out and the pool must be 16-byte aligned, rows at least a token apart", what);
  const int64_t recs = block_size / 16;
  Kv4AttnArgs a = {};
  a.out = static_cast<__nv_bfloat16*>(out);
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out_stride = out_stride;
  a.q_stride = q_stride;
  a.pool = static_cast<const uint8_t*>(kv4) + layer * num_blocks * num_kv_heads * recs * 18 * head_dim;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.max_blocks = static_cast<int>(max_blocks);
  a.ctx = ctx_lens;
  a.batch = static_cast<int>(batch);
  a.T = static_cast<int>(query_len);
  a.group = static_cast<int>(num_q_heads / num_kv_heads);
  a.hkv = static_cast<int>(num_kv_heads);
  a.num_blocks = static_cast<int>(num_blocks);
  a.recs = static_cast<int>(recs);
  a.score_scale = softcap > 0.0f ? scale / softcap : scale * kLog2e;
  a.cap_log2 = softcap * kLog2e;
  a.window = static_cast<int>(window < (1 << 30) ? window : (1 << 30));  // no context is longer
  a.err = device_status_ptr();

  const int sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "%s: no device", what);
  const int64_t rows = num_q_heads / num_kv_heads * query_len;
  const Kv4Plan p = kv4_plan(sms, head_dim, rows, batch, num_kv_heads);
  MVB_REQUIRE(num_kv_heads * p.chunks <= INT_MAX, "%s: heads", what);
  const int64_t items = batch * num_kv_heads * p.chunks, most = max_blocks * recs;  // records of an item
  // Short tables: an item goes to one worker and nothing is left to join.
  const bool split = most > kShortRecords;
  MVB_REQUIRE(!split || (workspace && aligned(workspace, 256) && workspace_bytes >= p.bytes),
              "%s: a workspace of %lld bytes, 256-byte aligned (got %lld)", what, (long long)p.bytes,
              (long long)workspace_bytes);
  a.split = split;
  int64_t grid = p.grid;
  const int64_t most_rounds = split ? kItemCost + (most + p.burst - 1) / p.burst : 1;
  if (items < grid && items * most_rounds < grid) grid = items * most_rounds;
  a.chunks = static_cast<int>(p.chunks);
  a.chunk_rows = static_cast<int>(rows < p.rows ? rows : p.rows);
  if (split) {
    char* ws = static_cast<char*>(workspace);
    a.items = reinterpret_cast<Kv4Item*>(ws + p.items_at);
    a.part_ml = reinterpret_cast<float2*>(ws + p.ml_at);
    a.part_o = reinterpret_cast<float*>(ws + p.o_at);
  }
  int64_t join_grid = 0;
  const int64_t all_pairs = items * a.chunk_rows;
  // a block per pair where there are few pairs, or where an item has many parts
  int pairs = all_pairs <= 2LL * sms || items * kFewParts < p.grid * p.warps ? 1 : 8;
  if (split) {
    join_grid = (all_pairs + pairs - 1) / pairs;
    if (pairs == 1 && all_pairs <= 2LL * sms && items * 32 < p.grid * p.warps) pairs = 0;  // and 32 warps for very many
    if (join_grid > 16LL * sms) join_grid = 16LL * sms;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (head_dim) {
    case 64: return kv4_launch<64>(a, p.rt, grid, join_grid, pairs, st);
    case 128: return kv4_launch<128>(a, p.rt, grid, join_grid, pairs, st);
    default: return kv4_launch<256>(a, p.rt, grid, join_grid, pairs, st);
  }
}
