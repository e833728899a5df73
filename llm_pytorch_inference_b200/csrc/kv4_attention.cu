// Attention of the newest T tokens of each sequence over the 4-bit paged pool (T = 1: a decode step).
//
//   out[b, i, h] = sum_t softmax_t(cap(q . k_t * scale)) v_t  over the keys t that query i sees,
//   k = m + s u,  v = m' + s' u'  per 64 channels (codes u in 0..15, pairs (s, m)).
//
// What it must read is 9/16 of a byte per cached value, once: the bound is memory.  That leaves an SM some
// 40 values a clock, so a value may cost about two instructions of a lane, and codes never become
// floating-point numbers one by one:
//   * fp16 holds u * 2^-24 and u * 2^-20 as bit patterns with the code in bits 0-3 or 4-7 (subnormal
//     numbers, exact).  One AND of a word thus yields two matrix operands, no conversion and no offset.
//   * The pairs stay outside the products.  Scores: q . k = sum_g s_g (q_g . u_g) + m_g sum(q_g), per group
//     of 64 channels.  Outputs: the weight of a token times s' is the operand against its codes, and
//     p m' is summed per group and query, on the side.
//   * q is scaled per row by a power of two into fp16's range and is exact there; scores and statistics
//     are fp32.  The weight p s' is the one rounding (11 bits, 8 times finer than the result's bf16); it is
//     scaled by a power of two that follows the largest s' seen.
// Both products run transposed on mma.sync m16n8k16, the query rows (query heads of the KV head times T)
// being the n = 8 side: S^T = K Q^T (16 tokens x 8 NT rows), O^T = V^T P^T.  The k index of the first product
// runs over the channels in the order in which a lane's words hold them (Q is stored in that order); the
// tokens of the second are permuted (tile_token) so that lanes reading the same word of different
// tokens fall into different banks.
//
// Work split: the cache of an item (sequence, KV head, chunk of 8 NT rows) is cut into rounds of W records
// (W warps, a record of 16 tokens each).  The rounds of the whole batch are laid end to end and divided
// evenly over the resident CTAs, whatever the lengths.  Each warp streams its own records through a ring in
// shared memory (one bulk copy a record, several in flight), and keeps its own running maximum, sum
// and output; they are joined in shared memory at the end of an item.  An item that spans CTAs
// leaves partial results, joined in CTA order by a second small kernel: no atomics, nothing to clear.
#include <climits>

#include "common.cuh"
#include "host.h"
#include "kv4.cuh"
#include "mma_sync.cuh"

namespace mvb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
// A weight is 2^(score - reference): the reference is a row's maximum when last raised, and is raised
// once a score passes it by more than kSlack (in powers of two), so that most records cost one vote instead
// of a reduction.  The weight times the scaled s' stays below 2^(kSlack + kScaleMax) = 2^15 in fp16.
constexpr float kSlack = 4.0f;
constexpr float kScaleMax = 2048.0f;  // 2^11; a new scaling puts the largest s' into [2^9, 2^10)
constexpr int kScaleTarget = 9;

// Records in flight per warp: an SM's share of the bandwidth needs some 45 KB.
template <int D, int NT>
constexpr int kv4_stages() {
  return D == 64 ? 6 : D == 256 && NT > 1 ? 2 : 4;
}
template <int D, int NT>
constexpr int kv4_ctas_per_sm() {
  return D == 256 || NT > 1 ? 1 : 2;
}

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
  int chunks;  // of 8 NT rows, per KV head
  int num_blocks, recs;
  float score_scale;  // scale * log2(e), or scale / softcap under a cap
  float cap_log2;     // softcap * log2(e); 0 = no cap
  int window;
  int slab_rows;  // rows of a chunk, at most 8 NT
  // workspace
  int64_t* head;       // [0]: CTAs that have work
  struct Kv4Start* starts;  // [grid]
  float2* part_ml;     // [2 grid][8 NT]
  float* part_o;       // [2 grid][8 NT][D]
  unsigned* err;
};

// Where a CTA's range of rounds begins.
struct Kv4Start {
  int64_t item_first;  // first round of the item, counted over the batch
  int rounds;          // of the item
  int seq;
  int sub;             // (KV head, chunk) within the sequence
  int pad[3];
};

__device__ __forceinline__ int64_t range_start(int c, int64_t total, int grid) {
  return static_cast<int64_t>(c) * total / grid;
}
__device__ __forceinline__ int cta_of(int64_t x, int64_t total, int grid) {
  return static_cast<int>(((x + 1) * grid + total - 1) / total - 1);
}

// exp2 with results below 2^-126 flushed to zero.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh x = 1 - 2 / (e^2x + 1): absolute error of a few 2^-24, where a score capped at c keeps c times that.
__device__ __forceinline__ float tanh_exp(float x) {
  return 1.0f - __fdividef(2.0f, ex2(x * (2.0f * kLog2e)) + 1.0f);
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// What a sequence's cache has to offer: tiles [first, last) of 16 tokens, cut into rounds.
struct Kv4Seq {
  int ctx, first, last, rounds;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs& a, int b, bool tell) {
  Kv4Seq s;
  const int most = a.max_blocks * a.recs * kKv4Tokens;
  const int raw = a.ctx[b];
  s.ctx = min(max(raw, 0), most);
  if (tell && s.ctx != raw) report(a.err, kDevBadPosition);
  s.first = 0;
  if (a.window > 0) s.first = max(s.ctx - a.T + 1 - a.window, 0) / kKv4Tokens;
  s.last = (s.ctx + kKv4Tokens - 1) / kKv4Tokens;
  s.rounds = max((s.last - s.first + kWarps - 1) / kWarps, 1);  // one for no keys too: it writes the zeros
  return s;
}

template <int D, int NT>
struct Kv4Smem {
  static constexpr int STAGES = kv4_stages<D, NT>();
  static constexpr int RING = kWarps * STAGES * Kv4<D>::RECORD;
  static constexpr int QF = RING;                              // Q operands [D / 16][NT][32] x 8 bytes
  static constexpr int COL = QF + D / 16 * NT * 256;           // per row: score factor, then sums of q per group
  static constexpr int ML = COL + 8 * NT * (1 + Kv4<D>::NG) * 4;  // [warps][8 NT] float2
  static constexpr int BAR = (ML + kWarps * 8 * NT * 8 + 15) / 16 * 16;
  static constexpr int SLAB = (BAR + kWarps * STAGES * 8 + 127) / 128 * 128;  // [warps][rows][D + 8] floats
  static constexpr int SLAB_ROW = D + 8;
  static constexpr size_t bytes(int rows) { return SLAB + static_cast<size_t>(kWarps) * rows * SLAB_ROW * 4; }
};

template <int D, int NT, bool CAP>
__global__ void __launch_bounds__(kThreads, kv4_ctas_per_sm<D, NT>()) kv4_attn_kernel(const Kv4AttnArgs a) {
  using P = Kv4<D>;
  using S = Kv4Smem<D, NT>;
  constexpr int NG = P::NG, STAGES = S::STAGES, KS = D / 16, ROWS = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ volatile int abort_flag;
  __shared__ int64_t scan_warp[kWarps];
  __shared__ int64_t found_first;
  __shared__ int found_seq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  uint2* qf = reinterpret_cast<uint2*>(smem + S::QF);
  float* col_f = reinterpret_cast<float*>(smem + S::COL);
  float* col_q = col_f + ROWS;  // [ROWS][NG]
  float2* ml = reinterpret_cast<float2*>(smem + S::ML);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR) + warp * STAGES;
  float* slab = reinterpret_cast<float*>(smem + S::SLAB);
  uint8_t* ring = smem + warp * STAGES * P::RECORD;

  pdl_launch_dependents();
  if (lane < STAGES) mbar_init(bars + lane, 1);
  fence_barrier_init();
  if (tid == 0) abort_flag = 0;
  pdl_wait();

  // ---- this CTA's rounds: [r0, r1) of the batch's total
  const int subs = a.hkv * a.chunks;
  int64_t carry = 0, incl = 0, own = 0;
  for (int base = 0; base < a.batch; base += kThreads) {
    const int b = base + tid;
    own = b < a.batch ? static_cast<int64_t>(kv4_seq(a, b, blockIdx.x == 0).rounds) * subs : 0;
    incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) scan_warp[warp] = incl;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) incl += scan_warp[w];
      all += scan_warp[w];
    }
    incl += carry;
    carry += all;
  }
  const int64_t total = carry;
  const int active = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));
  if (blockIdx.x == 0 && tid == 0) {
    a.head[0] = active;
    a.head[1] = total;
  }
  if (static_cast<int>(blockIdx.x) >= active) return;
  const int64_t r0 = range_start(blockIdx.x, total, active), r1 = range_start(blockIdx.x + 1, total, active);
  if (a.batch <= kThreads) {
    if (own > 0 && incl - own <= r0 && r0 < incl) {
      found_seq = tid;
      found_first = incl - own;
    }
  } else {
    carry = 0;
    for (int base = 0; base < a.batch && carry <= r0; base += kThreads) {
      const int b = base + tid;
      own = b < a.batch ? static_cast<int64_t>(kv4_seq(a, b, false).rounds) * subs : 0;
      incl = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      __syncthreads();
      if (lane == 31) scan_warp[warp] = incl;
      __syncthreads();
      int64_t all = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) incl += scan_warp[w];
        all += scan_warp[w];
      }
      incl += carry;
      carry += all;
      if (own > 0 && incl - own <= r0 && r0 < incl) {
        found_seq = b;
        found_first = incl - own;
      }
    }
  }
  __syncthreads();

  int seq = found_seq;
  Kv4Seq sq = kv4_seq(a, seq, false);
  int sub = static_cast<int>((r0 - found_first) / sq.rounds);
  int ra = static_cast<int>(r0 - found_first - static_cast<int64_t>(sub) * sq.rounds);
  int left = static_cast<int>(r1 - r0);
  if (tid == 0) {
    Kv4Start st = {};
    st.item_first = r0 - ra;
    st.rounds = sq.rounds;
    st.seq = seq;
    st.sub = sub;
    a.starts[blockIdx.x] = st;
  }

  // ---- the warp's stream of records, STAGES ahead of the arithmetic
  int p_seq = seq, p_sub = sub, p_left = left, p_n = min(sq.rounds - ra, left);
  Kv4Seq p_sq = sq;
  int p_t = sq.first + ra * kWarps + warp, p_end = min(sq.first + (ra + p_n) * kWarps, sq.last);
  int p_id = 0, p_rec = 0;
  bool p_ok = true;
  // Settles on the warp's next record at or after p_t, crossing into the next items, and asks for its block id
  // (one record ahead of the copy that needs it).
  auto settle = [&]() {
    while (p_t >= p_end) {
      p_left -= p_n;
      if (p_left <= 0) {
        p_ok = false;
        return;
      }
      if (++p_sub == subs) {
        p_sub = 0;
        p_sq = kv4_seq(a, ++p_seq, false);
      }
      p_n = min(p_sq.rounds, p_left);
      p_t = p_sq.first + warp;
      p_end = min(p_sq.first + p_n * kWarps, p_sq.last);
    }
    const int blk = a.recs == 1 ? p_t : p_t / a.recs;
    p_rec = p_t - blk * a.recs;
    p_id = a.tables[p_seq * a.table_stride + blk];
  };
  unsigned bad = 0, phase = 0;  // per stage: no record came (invalid block); parity of its barrier
  auto issue = [&](int st) {
    if (!p_ok) return;
    if (static_cast<unsigned>(p_id) < static_cast<unsigned>(a.num_blocks)) {
      bad &= ~(1u << st);
      if (lane == 0) {
        const int h = a.chunks == 1 ? p_sub : p_sub / a.chunks;
        const int64_t rec = (static_cast<int64_t>(p_id) * a.hkv + h) * a.recs + p_rec;
        mbar_arrive_expect_tx(bars + st, P::RECORD);
        bulk_load(ring + st * P::RECORD, a.pool + rec * P::RECORD, P::RECORD, bars + st);
      }
    } else {
      bad |= 1u << st;
      if (lane == 0) report(a.err, kDevBadBlock);
    }
    p_t += kWarps;
    settle();
  };
  settle();
  int pending = 0;  // stages whose copy is still to be waited for
#pragma unroll 1
  for (int st = 0; st < STAGES; ++st) {
    pending += p_ok;
    issue(st);
  }
  int cur = 0;
  bool dead = false;

  const int tok0 = tile_token(g), tok1 = tile_token(g + 8);
  int vtok[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) vtok[i] = 4 * c + ((i + c) & 3);

  // ---- items
  while (left > 0) {
    const int n_rounds = min(sq.rounds - ra, left);
    const int h = a.chunks == 1 ? sub : sub / a.chunks;
    const int row0 = (sub - h * a.chunks) * ROWS;
    const int rows = min(a.group * a.T - row0, ROWS);

    // Q of the item: row per warp, scaled by a power of two so that its largest magnitude lies in [2^10, 2^11)
    for (int r = warp; r < ROWS; r += kWarps) {
      constexpr int N = D / 32;
      float x[N];
      float big = 0.0f;
      const int i = (row0 + r) / a.group, hq = h * a.group + (row0 + r) - i * a.group;
      const __nv_bfloat16* src = a.q + (static_cast<int64_t>(seq) * a.T + i) * a.q_stride + static_cast<int64_t>(hq) * D;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[j] = r < rows ? __bfloat162float(src[lane * N + j]) : 0.0f;
        big = fmaxf(big, fabsf(x[j]));
      }
      big = warp_max(big);
      int e = 0;
      if (big > 0.0f && big <= 3.3895314e38f) e = 10 - ilogbf(big);
      e = min(max(e, -126), 126);
      const float up = ldexpf(1.0f, e);
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[j] *= up;
        part += x[j];
      }
      // lanes of a group of 64 channels: 64 / N of them
#pragma unroll
      for (int o = 1; o < 64 / N; o <<= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == 0) col_f[r] = ldexpf(a.score_scale, 20 - e);
      if (lane % (64 / N) == 0) col_q[r * NG + lane / (64 / N)] = part * 0x1p-20f;
      __half* dst = reinterpret_cast<__half*>(qf);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int ch = lane * N + j, grp = ch / 64, w = ch % 64 / 8, nib = ch % 8;
        // word w of the group belongs to lane c = w / 2; nibbles 2h', 2h' + 4 are the low k pair of half h', and
        // 2h' + 1, 2h' + 5 the high one, whose codes weigh 16 times as much
        const int ks = (grp * 2 + (w & 1)) * 2 + ((nib & 3) >> 1), hi = nib & 1, el = nib >> 2;
        dst[((ks * NT + r / 8) * 32 + (r % 8) * 4 + w / 2) * 4 + hi * 2 + el] = __float2half_rn(hi ? x[j] : x[j] * 16.0f);
      }
    }
    __syncthreads();

    float f[NT][2], qs[NT][2][NG];
    int see[NT][2];  // keys that the row sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = nt * 8 + 2 * c + j;
        f[nt][j] = col_f[r];
#pragma unroll
        for (int k = 0; k < NG; ++k) qs[nt][j][k] = col_q[r * NG + k];
        see[nt][j] = r < rows ? sq.ctx - a.T + 1 + (row0 + r) / a.group : -(1 << 30);
      }
    const int see_least = sq.ctx - a.T + 1 + row0 / a.group;
    const int see_most = sq.ctx - a.T + 1 + (row0 + rows - 1) / a.group;

    float o[KS][NT][4];  // m tiles: (group, high half of the word, half of that), 16 channels each
    float l[NT][2], mref[NT][2], mo[NT][2][NG];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][nt][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nt][j] = 0.0f;
        mref[nt][j] = -INFINITY;
#pragma unroll
        for (int k = 0; k < NG; ++k) mo[nt][j][k] = 0.0f;
      }
    }
    float vscale = 1.0f;  // power of two that the value scales are multiplied by
    bool fresh = true;

    const int t_end = min(sq.first + (ra + n_rounds) * kWarps, sq.last);
    for (int t = sq.first + ra * kWarps + warp; t < t_end; t += kWarps) {
      const bool came = !(bad >> cur & 1u);
      if (came && !dead) {
        const bool ok = mbar_wait(bars + cur, phase >> cur & 1u, &abort_flag, a.err);
        if (!__all_sync(0xffffffffu, ok)) dead = true;
      }
      if (!dead) {
        if (came) {
          phase ^= 1u << cur;
          const uint8_t* rec = ring + cur * P::RECORD;
          // ---- scores
          uint32_t kw[2][2 * NG];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t* at = rec + (r ? tok1 : tok0) * P::ROW + c * (8 * NG);
            if constexpr (NG == 1) {
              const uint2 v = *reinterpret_cast<const uint2*>(at);
              kw[r][0] = v.x, kw[r][1] = v.y;
            } else {
#pragma unroll
              for (int k = 0; k < NG / 2; ++k) {
                const uint4 v = *reinterpret_cast<const uint4*>(at + 16 * k);
                kw[r][4 * k] = v.x, kw[r][4 * k + 1] = v.y, kw[r][4 * k + 2] = v.z, kw[r][4 * k + 3] = v.w;
              }
            }
          }
          float s[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
#pragma unroll
            for (int wi = 0; wi < 2; ++wi)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const uint32_t x0 = kw[0][NG * wi + k] >> (8 * hh), x1 = kw[1][NG * wi + k] >> (8 * hh);
                const uint32_t a0 = x0 & 0x000F000Fu, a1 = x1 & 0x000F000Fu, a2 = x0 & 0x00F000F0u,
                               a3 = x1 & 0x00F000F0u;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  const uint2 b = qf[(((k * 2 + wi) * 2 + hh) * NT + nt) * 32 + lane];
                  mma_f16_16816(acc[nt], a0, a1, a2, a3, b.x, b.y);
                }
              }
            const float2 p0 = __bfloat1622float2(
                *reinterpret_cast<const __nv_bfloat162*>(rec + P::K_PAIRS + tok0 * P::PAIRS + 4 * k));
            const float2 p1 = __bfloat1622float2(
                *reinterpret_cast<const __nv_bfloat162*>(rec + P::K_PAIRS + tok1 * P::PAIRS + 4 * k));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 p = e < 2 ? p0 : p1;
                s[nt][e] = fmaf(p.x, acc[nt][e], fmaf(p.y, qs[nt][e & 1][k], s[nt][e]));
              }
          }
          float2 vp[2][NG];
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              vp[r][k] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(
                  rec + P::V_PAIRS + (r ? tok1 : tok0) * P::PAIRS + 4 * k));
          const int pos0 = t * kKv4Tokens + tok0, pos1 = t * kKv4Tokens + tok1;
          const bool masked = t * kKv4Tokens + kKv4Tokens > see_least ||
                              (a.window > 0 && t * kKv4Tokens < see_most - a.window);
          if (masked) {  // pairs of tokens that no row sees hold anything
            const int low = a.window > 0 ? see_least - a.window : 0;
            const bool in0 = pos0 < see_most && pos0 >= low, in1 = pos1 < see_most && pos1 >= low;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
              if (!in0) vp[0][k] = make_float2(0.0f, 0.0f);
              if (!in1) vp[1][k] = make_float2(0.0f, 0.0f);
            }
          }
          bool need = false;
          unsigned sees = 0;  // bit 4 nt + e: the key belongs to the row
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = s[nt][e] * f[nt][e & 1];
              if constexpr (CAP) v = a.cap_log2 * tanh_exp(v);
              if (masked) {
                const int pos = e < 2 ? pos0 : pos1, n = see[nt][e & 1];
                const bool in = pos < n && (a.window <= 0 || pos >= n - a.window);
                sees |= static_cast<unsigned>(in) << (4 * nt + e);
                v = in ? v : -INFINITY;
              }
              s[nt][e] = v;
              need |= v > mref[nt][e & 1] + kSlack;
            }
#pragma unroll
          for (int k = 0; k < NG; ++k) need |= vp[0][k].x * vscale > kScaleMax || vp[1][k].x * vscale > kScaleMax;
          // ---- new references and scaling, where a score or a scale outgrew them
          if (__any_sync(0xffffffffu, need)) {
            float smax = 0.0f;
#pragma unroll
            for (int k = 0; k < NG; ++k)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (vp[r][k].x <= 3.3895314e38f) smax = fmaxf(smax, vp[r][k].x);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, off));
            float fo = 1.0f;
            if (smax > 0.0f && (fresh || smax * vscale > kScaleMax)) {
              const float ns = ldexpf(1.0f, min(kScaleTarget - ilogbf(smax), 126));
              fo = ns / vscale;
              vscale = ns;
              if (fresh) fo = 1.0f;
              fresh = false;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float m = fmaxf(s[nt][j], s[nt][j + 2]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
                m = fmaxf(m, mref[nt][j]);
                const float fac = mref[nt][j] == -INFINITY ? 0.0f : ex2(mref[nt][j] - m);
                mref[nt][j] = m;
                l[nt][j] *= fac;
#pragma unroll
                for (int k = 0; k < NG; ++k) mo[nt][j][k] *= fac;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                  o[k][nt][j] *= fac * fo;
                  o[k][nt][j + 2] *= fac * fo;
                }
              }
          }
          // ---- weights
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float m = mref[nt][e & 1];
              s[nt][e] = ex2(s[nt][e] - (m == -INFINITY ? 0.0f : m));
              l[nt][e & 1] += s[nt][e];
            }
          // ---- outputs
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            uint32_t b[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 p = vp[e >> 1][k];
                w[e] = s[nt][e] * (p.x * vscale);
                float pm = s[nt][e] * p.y;
                if (masked && !(sees >> (4 * nt + e) & 1u)) w[e] = pm = 0.0f;  // a NaN that only later rows see
                mo[nt][e & 1][k] += pm;
              }
              movmatrix_trans(pack_f16(w[0], w[1]), b[nt][0]);
              movmatrix_trans(pack_f16(w[2], w[3]), b[nt][1]);
            }
            uint32_t vw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              vw[i] = *reinterpret_cast<const uint32_t*>(rec + P::V_CODES + vtok[i] * P::ROW + 4 * (NG * g + k));
#pragma unroll
            for (int hv = 0; hv < 2; ++hv) {
              const uint32_t y0 = __byte_perm(vw[0], vw[1], hv ? 0x7632 : 0x5410);
              const uint32_t y1 = __byte_perm(vw[2], vw[3], hv ? 0x7632 : 0x5410);
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const uint32_t x0 = y0 >> (8 * hh), x1 = y1 >> (8 * hh);
                const uint32_t a0 = x0 & 0x000F000Fu, a1 = x0 & 0x00F000F0u, a2 = x1 & 0x000F000Fu,
                               a3 = x1 & 0x00F000F0u;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[(k * 2 + hv) * 2 + hh][nt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
              }
            }
          }
        }
        --pending;
        __syncwarp();
        pending += p_ok;
        issue(cur);
        cur = cur + 1 == STAGES ? 0 : cur + 1;
      }
    }

    // ---- the warps' shares of the item joined
    const int busy = min(kWarps, max(t_end - (sq.first + ra * kWarps), 0));  // warps that had a record
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], off);
#pragma unroll
          for (int k = 0; k < NG; ++k) mo[nt][j][k] += __shfl_xor_sync(0xffffffffu, mo[nt][j][k], off);
        }
        if (g == 0) ml[warp * ROWS + nt * 8 + 2 * c + j] = make_float2(mref[nt][j], l[nt][j]);
      }
    __syncthreads();
    if (warp < busy) {
      const float inv = 1.0f / vscale;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = nt * 8 + 2 * c + j;
          if (r >= rows) continue;
          float top = -INFINITY;
          for (int w = 0; w < busy; ++w) top = fmaxf(top, ml[w * ROWS + r].x);
          const float fac = mref[nt][j] == -INFINITY ? 0.0f : ex2(mref[nt][j] - top);
          float* dst = slab + (warp * a.slab_rows + r) * S::SLAB_ROW + 8 * g;
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int hv = 0; hv < 2; ++hv) {
              // channels 8 g + 4 hv + 2 hh (codes as u 2^-24) and the next one (u 2^-20)
              const float(&x)[4] = o[(k * 2 + hv) * 2][nt];
              const float(&y)[4] = o[(k * 2 + hv) * 2 + 1][nt];
              const float mk = mo[nt][j][k];
              *reinterpret_cast<float4*>(dst + 64 * k + 4 * hv) = make_float4(
                  fac * fmaf(x[j] * 0x1p24f, inv, mk), fac * fmaf(x[j + 2] * 0x1p20f, inv, mk),
                  fac * fmaf(y[j] * 0x1p24f, inv, mk), fac * fmaf(y[j + 2] * 0x1p20f, inv, mk));
            }
        }
    }
    __syncthreads();
    const bool whole = ra == 0 && n_rounds == sq.rounds;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (ra == 0 ? 1 : 0);
    for (int x = tid; x < rows * (D / 4); x += kThreads) {
      const int r = x / (D / 4), ch = x % (D / 4) * 4;
      float top = -INFINITY, sum = 0.0f;
      for (int w = 0; w < busy; ++w) top = fmaxf(top, ml[w * ROWS + r].x);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int w = 0; w < busy; ++w) {
        const float2 e = ml[w * ROWS + r];
        sum += e.x == -INFINITY ? 0.0f : e.y * ex2(e.x - top);
        const float4 y = *reinterpret_cast<const float4*>(slab + (w * a.slab_rows + r) * S::SLAB_ROW + ch);
        v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
      }
      if (whole) {
        const int i = (row0 + r) / a.group, hq = h * a.group + (row0 + r) - i * a.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        __nv_bfloat16* dst = a.out + (static_cast<int64_t>(seq) * a.T + i) * a.out_stride + static_cast<int64_t>(hq) * D + ch;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
      } else {
        if (ch == 0) a.part_ml[slot * ROWS + r] = make_float2(top, sum);
        *reinterpret_cast<float4*>(a.part_o + (slot * ROWS + r) * D + ch) = v;
      }
    }
    left -= n_rounds;
    ra = 0;
    if (++sub == subs && left > 0) {
      sub = 0;
      sq = kv4_seq(a, ++seq, false);
    }
  }
  // a stream that was given up: its copies land before the block's shared memory goes
  if (dead)
    for (int st = cur; pending > 0; --pending, st = st + 1 == STAGES ? 0 : st + 1)
      if (!(bad >> st & 1u)) mbar_wait(bars + st, phase >> st & 1u, nullptr, a.err);
}

// Joins the parts of the items that span CTAs.  CTA (c - 1, r) looks at the boundary between CTAs c - 1 and c of
// the first kernel: if it is the first one inside its item, it joins row r of the item, parts in CTA order,
// eight warps taking every eighth part.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_join_kernel(const Kv4AttnArgs a) {
  constexpr int ROWS = 8 * NT, N = D / 32;
  __shared__ float acc[kWarps][D];
  __shared__ float2 ml[kWarps];
  pdl_wait();
  pdl_launch_dependents();
  const int cta = blockIdx.x + 1, r = blockIdx.y;
  const int active = static_cast<int>(a.head[0]);
  if (cta >= active) return;
  const int64_t total = a.head[1];
  const Kv4Start st = a.starts[cta];
  const int64_t here = range_start(cta, total, active), before = range_start(cta - 1, total, active);
  if (here == st.item_first || before > st.item_first) return;
  const int h = st.sub / a.chunks, row0 = (st.sub - h * a.chunks) * ROWS;
  if (r >= a.group * a.T - row0) return;
  const int last = cta_of(st.item_first + st.rounds - 1, total, active);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY, l = 0.0f, o[N];
#pragma unroll
  for (int j = 0; j < N; ++j) o[j] = 0.0f;
#pragma unroll 4
  for (int p = cta - 1 + warp; p <= last; p += kWarps) {
    const int64_t slot = (2 * static_cast<int64_t>(p) + (p == cta - 1 ? 1 : 0)) * ROWS + r;
    const float2 e = a.part_ml[slot];
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = a.part_o[slot * D + 32 * j + lane];
    const float top = fmaxf(m, e.x);
    const float fm = m == -INFINITY ? 0.0f : ex2(m - top), fe = e.x == -INFINITY ? 0.0f : ex2(e.x - top);
    l = l * fm + e.y * fe;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = o[j] * fm + x[j] * fe;
    m = top;
  }
  if (lane == 0) ml[warp] = make_float2(m, l);
#pragma unroll
  for (int j = 0; j < N; ++j) acc[warp][32 * j + lane] = o[j];
  __syncthreads();
  float top = -INFINITY;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w].x);
  const int i = (row0 + r) / a.group, hq = h * a.group + (row0 + r) - i * a.group;
  __nv_bfloat16* dst = a.out + (static_cast<int64_t>(st.seq) * a.T + i) * a.out_stride + static_cast<int64_t>(hq) * D;
  for (int ch = threadIdx.x; ch < D; ch += kThreads) {
    float sum = 0.0f, v = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
      const float f = ml[w].x == -INFINITY ? 0.0f : ex2(ml[w].x - top);
      sum += ml[w].y * f;
      v += acc[w][ch] * f;
    }
    dst[ch] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : v / sum);
  }
}

// Column tiles of 8 query rows that a CTA carries: up to 16 rows in one pass over the cache.
int64_t kv4_tiles(int64_t rows) { return rows <= 8 ? 1 : 2; }

int64_t kv4_grid(int64_t sms, int64_t head_dim, int64_t nt) { return sms * (head_dim == 256 || nt > 1 ? 1 : 2); }

struct Kv4Workspace {
  int64_t starts, ml, o, bytes;
};
Kv4Workspace kv4_workspace(int64_t grid, int64_t nt, int64_t head_dim) {
  Kv4Workspace w;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  w.starts = 256;
  w.ml = w.starts + up(grid * static_cast<int64_t>(sizeof(Kv4Start)));
  w.o = w.ml + up(2 * grid * 8 * nt * 8);
  w.bytes = w.o + 2 * grid * 8 * nt * head_dim * 4;
  return w;
}

template <int D, int NT, bool CAP>
int kv4_launch_cap(const Kv4AttnArgs& a, int64_t grid, int64_t most_rounds, cudaStream_t st) {
  const size_t smem = Kv4Smem<D, NT>::bytes(a.slab_rows);
  MVB_TRY(set_smem(kv4_attn_kernel<D, NT, CAP>, smem, "kv4_attention"));
  MVB_TRY(launch("kv4_attention", kv4_attn_kernel<D, NT, CAP>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem,
                 st, a));
  if (most_rounds <= 1 || grid <= 1) return MVB_OK;  // no item can span CTAs
  return launch_dependent("kv4_attention_join", kv4_join_kernel<D, NT>,
                          dim3(static_cast<unsigned>(grid - 1), static_cast<unsigned>(a.slab_rows)), dim3(kThreads), 0,
                          st, a);
}

template <int D>
int kv4_launch(const Kv4AttnArgs& a, int64_t nt, int64_t grid, int64_t most_rounds, cudaStream_t st) {
  const bool cap = a.cap_log2 > 0.0f;
  if (nt == 1)
    return cap ? kv4_launch_cap<D, 1, true>(a, grid, most_rounds, st)
               : kv4_launch_cap<D, 1, false>(a, grid, most_rounds, st);
  return cap ? kv4_launch_cap<D, 2, true>(a, grid, most_rounds, st)
             : kv4_launch_cap<D, 2, false>(a, grid, most_rounds, st);
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int64_t mvb_paged_attention_decode_kv4_workspace_bytes(int64_t batch, int64_t query_len,
                                                                  int64_t num_q_heads, int64_t num_kv_heads,
                                                                  int64_t head_dim, int device) {
  (void)batch;
  if (num_kv_heads <= 0 || query_len <= 0) return 0;
  int sms = mvb_num_sms(device);
  if (sms <= 0) sms = 148;
  const int64_t nt = kv4_tiles(num_q_heads / num_kv_heads * query_len);
  return kv4_workspace(kv4_grid(sms, head_dim, nt), nt, head_dim).bytes;
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
  MVB_REQUIRE(batch >= 0 && batch <= (1 << 20), "%s: batch %lld", what, (long long)batch);
  MVB_REQUIRE(query_len >= 1 && query_len <= 1024, "%s: %lld query tokens (1 to 1024)", what, (long long)query_len);
  MVB_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0 && num_q_heads <= 65536,
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
  MVB_REQUIRE(window >= 0 && softcap >= 0.0f && scale == scale, "%s: window, softcap or scale", what);
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
  const int64_t rows = num_q_heads / num_kv_heads * query_len, nt = kv4_tiles(rows);
  const int64_t chunks = (rows + 8 * nt - 1) / (8 * nt);
  const int64_t most_rounds = (max_blocks * recs + kWarps - 1) / kWarps;
  MVB_REQUIRE(num_kv_heads * chunks <= INT_MAX, "%s: heads", what);
  int64_t grid = kv4_grid(sms, head_dim, nt);
  const Kv4Workspace w = kv4_workspace(grid, nt, head_dim);
  MVB_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= w.bytes,
              "%s: a workspace of %lld bytes, 256-byte aligned (got %lld)", what, (long long)w.bytes,
              (long long)workspace_bytes);
  const int64_t bound = batch * num_kv_heads * chunks;  // items; times the rounds of the longest possible one
  if (bound < grid && bound * most_rounds < grid) grid = bound * most_rounds;
  a.chunks = static_cast<int>(chunks);
  a.slab_rows = static_cast<int>(rows < 8 * nt ? rows : 8 * nt);
  char* ws = static_cast<char*>(workspace);
  a.head = reinterpret_cast<int64_t*>(ws);
  a.starts = reinterpret_cast<Kv4Start*>(ws + w.starts);
  a.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  a.part_o = reinterpret_cast<float*>(ws + w.o);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (head_dim) {
    case 64: return kv4_launch<64>(a, nt, grid, most_rounds, st);
    case 128: return kv4_launch<128>(a, nt, grid, most_rounds, st);
    default: return kv4_launch<256>(a, nt, grid, most_rounds, st);
  }
}
