// Verification of drafted tokens against the target's probabilities.
//
// Draft i of a sequence (token d_i, drawn from the drafting distribution q_i) is accepted while
// u_i q_i(d_i) < p_i(d_i) with the given uniform u_i.  At the first rejection the token is drawn
// from max(p_i - q_i, 0) instead; when every draft passes, one more is drawn from the last row p_n.
// Drawing is the inverse CDF in vocabulary order: the smallest j with w_0 + .. + w_j > u * total.
// Without drafting probabilities q_i is one at d_i (a greedy or looked-up draft).
//
// Products and sums are held in 64 bits: the product of two fp32 numbers is exact there, and a sum
// of a vocabulary of fp32 probabilities is off by 1e-16 of the total, so the answer does not
// depend on how the sum is split unless u lies that close to a border.
//
// Only one row of p (and of q) is read per sequence: bound by those 4 (8) bytes an entry, and by latency for few
// sequences.  (64 sequences of 151,936 entries are 256 blocks on 296 places: an SM is busy for 72 % of the call.)
// A sequence is a cluster of up to 8 blocks: every lane looks at one draft, so that all of them cost one dependent load
// each; every warp sums a run of the vocabulary; the blocks exchange their sums through distributed shared memory; and
// the block in whose part the threshold falls reads one warp's run of it again (out of L2), all its warps together, to
// find the entry.  The order of all sums is fixed.
#include <climits>

#include "common.cuh"
#include "host.h"

namespace mvb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

struct VerifyArgs {
  int64_t* out;
  int32_t* accepted;
  const float* p;
  int64_t p_stride;  // elements between rows; a sequence has drafts + 1 of them
  const float* q;    // nullptr: one at the drafted token
  int64_t q_stride;
  const int64_t* tokens;
  const float* u;
  const int32_t* lens;  // nullptr: all `drafts`
  int drafts;
  int vocab;
  unsigned* err;
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What the entries of the row weigh in the draw.
struct Weights {
  const float* p;
  const float* q;   // the drafting row, or nullptr
  int token;        // the rejected one-hot draft, or -1
  __device__ __forceinline__ double of(int j, float pj, float qj) const {
    if (q != nullptr) return fmax(static_cast<double>(pj) - static_cast<double>(qj), 0.0);
    return j == token ? 0.0 : fmax(static_cast<double>(pj), 0.0);
  }
};

// Entries j .. j + 3 of a row, zeros from `end` on; VEC: j and the row are 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* row, int j, int end) {
  if (VEC && j + 4 <= end) return *reinterpret_cast<const float4*>(row + j);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (j < end) v.x = row[j];
  if (j + 1 < end) v.y = row[j + 1];
  if (j + 2 < end) v.z = row[j + 2];
  if (j + 3 < end) v.w = row[j + 3];
  return v;
}

// The lane's share of the sum over [begin, end), begin a multiple of 4.
template <bool VEC>
__device__ __forceinline__ double run_sum(const Weights& w, int begin, int end, int lane) {
  const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  double s = 0.0;
  float4 p[2], q[2];  // two steps under way while one is summed
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    p[i] = load4<VEC>(w.p, begin + 128 * i + 4 * lane, end);
    q[i] = w.q != nullptr ? load4<VEC>(w.q, begin + 128 * i + 4 * lane, end) : zero;
  }
#pragma unroll 1
  for (int j = begin + 4 * lane; j < end; j += 128) {
    const float4 pc = p[0], qc = q[0];
    p[0] = p[1];
    q[0] = q[1];
    p[1] = load4<VEC>(w.p, j + 256, end);
    q[1] = w.q != nullptr ? load4<VEC>(w.q, j + 256, end) : zero;
    s += (w.of(j, pc.x, qc.x) + w.of(j + 1, pc.y, qc.y)) + (w.of(j + 2, pc.z, qc.z) + w.of(j + 3, pc.w, qc.w));
  }
  return s;
}

// The first entry of [begin, end) at which `before` plus the weights so far exceed thr; the last one with any
// weight if rounding leaves none; -1 if nothing weighs.
template <bool VEC>
__device__ __forceinline__ int run_find(const Weights& w, int begin, int end, double before, double thr, int lane) {
  int last = -1;
  const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float4 p = load4<VEC>(w.p, begin + 4 * lane, end);
  float4 q = w.q != nullptr ? load4<VEC>(w.q, begin + 4 * lane, end) : zero;
  for (int j0 = begin; j0 < end; j0 += 128) {
    const int j = j0 + 4 * lane;
    const float4 pc = p, qc = q;
    p = load4<VEC>(w.p, j + 128, end);  // the next ones are under way meanwhile
    q = w.q != nullptr ? load4<VEC>(w.q, j + 128, end) : zero;
    const double x[4] = {w.of(j, pc.x, qc.x), w.of(j + 1, pc.y, qc.y), w.of(j + 2, pc.z, qc.z), w.of(j + 3, pc.w, qc.w)};
    const double own = (x[0] + x[1]) + (x[2] + x[3]);
    double c = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += y;
    }
    double at = before + (c - own);
    int hit = -1, some = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at += x[i];
      if (x[i] > 0.0) {
        some = j + i;
        if (hit < 0 && at > thr) hit = j + i;
      }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, some >= 0);
    if (hits) return __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
    if (any) last = __shfl_sync(0xffffffffu, some, 31 - __clz(any));
    before += __shfl_sync(0xffffffffu, c, 31);
  }
  return last;
}

// Of the n <= 32 sums of consecutive parts: the first one at which `before` plus the sums so far exceed thr (the
// last with any weight if rounding leaves none, -1 if nothing weighs), and what lies before it.  A whole warp's.
__device__ __forceinline__ int pick_part(const double* sums, int n, double before, double thr, int lane, double& start) {
  const double x = lane < n ? sums[lane] : 0.0;
  double c = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, c, o);
    if (lane >= o) c += y;
  }
  const unsigned hits = __ballot_sync(0xffffffffu, x > 0.0 && before + c > thr), any = __ballot_sync(0xffffffffu, x > 0.0);
  const int at = hits ? __ffs(hits) - 1 : any ? 31 - __clz(any) : -1;
  start = before + __shfl_sync(0xffffffffu, c - x, at < 0 ? 0 : at);
  return at;
}

__device__ __forceinline__ double dsmem_ld_f64(const double* p, uint32_t rank) {
  uint32_t remote;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(remote) : "memory");
  return v;
}

// A cluster of `blocks` blocks per sequence, warp x of it summing entries [x run, (x + 1) run).
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const VerifyArgs a, const int blocks, const int run) {
  __shared__ double warp_total[kWarps], part_total[kWarps];
  __shared__ double block_total, sums[kMaxCluster];
  // dependents start at this kernel's end only: they read its outputs as step metadata before they wait
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int b = blockIdx.x / blocks, rank = blockIdx.x - b * blocks;
  const int64_t* tok = a.tokens + static_cast<int64_t>(b) * a.drafts;
  const float* u = a.u + static_cast<int64_t>(b) * (a.drafts + 1);
  const int n_drafts = a.lens != nullptr ? min(max(a.lens[b], 0), a.drafts) : a.drafts;
  const float* p_rows = a.p + static_cast<int64_t>(b) * (a.drafts + 1) * a.p_stride;
  const float* q_rows = a.q + static_cast<int64_t>(b) * a.drafts * a.q_stride;  // used where a.q is given
  int n = n_drafts;  // the first draft that is not accepted
  for (int i0 = 0; i0 < a.drafts; i0 += 32) {
    // all given or not are looked at, so that no load waits for the number of drafts
    const int i = i0 + lane;
    bool ok = true, known = true;
    if (i < a.drafts) {
      const int64_t d = tok[i];
      const float ui = u[i];
      known = d >= 0 && d < a.vocab;
      if (known) {
        const double q = a.q != nullptr ? static_cast<double>(q_rows[i * a.q_stride + d]) : 1.0;
        ok = static_cast<double>(ui) * q < static_cast<double>(p_rows[i * a.p_stride + d]);
      }
    }
    if (i < n_drafts && !known && rank == 0 && wid == 0) report(a.err, kDevBadToken);
    const unsigned no = __ballot_sync(0xffffffffu, i < n_drafts && !(ok && known));
    if (no) {
      n = i0 + __ffs(no) - 1;
      break;
    }
  }
  const bool rejected = n < n_drafts;
  Weights w;
  w.p = p_rows + n * a.p_stride;
  w.q = rejected && a.q != nullptr ? q_rows + n * a.q_stride : nullptr;
  w.token = -1;
  if (rejected && a.q == nullptr && tok[n] >= 0 && tok[n] < a.vocab) w.token = static_cast<int>(tok[n]);
  const float draw = u[a.drafts];

  const int begin = (rank * kWarps + wid) * run, end = min(begin + run, a.vocab);
  double total = 0.0, before = 0.0;  // of the row, of the blocks before the owner
  int owner = -1;                    // the block that the threshold falls into
  bool vec = false;
  for (int pass = 0; pass < 2; ++pass) {
    vec = (reinterpret_cast<uintptr_t>(w.p) & 15) == 0 && (w.q == nullptr || (reinterpret_cast<uintptr_t>(w.q) & 15) == 0);
    const double s = warp_sum_f64(vec ? run_sum<true>(w, begin, end, lane) : run_sum<false>(w, begin, end, lane));
    if (lane == 0) warp_total[wid] = s;
    __syncthreads();
    if (wid == 0) {
      const double t = warp_sum_f64(lane < kWarps ? warp_total[lane] : 0.0);
      if (lane == 0) block_total = t;
    }
    cluster_sync();
    if (tid < blocks) sums[tid] = dsmem_ld_f64(&block_total, tid);
    cluster_sync();  // everybody has read: block_total may change, or its block end
    total = warp_sum_f64(lane < blocks ? sums[lane] : 0.0);
    owner = pick_part(sums, blocks, 0.0, static_cast<double>(draw) * total, lane, before);
    if (total > 0.0 || !rejected) break;
    __syncthreads();  // sums has been read
    // nothing is left of p - q (equal rows, or rounding): draw from p itself
    w.q = nullptr;
    w.token = -1;
  }

  int64_t* out = a.out + static_cast<int64_t>(b) * (a.drafts + 1);
  if (rank == 0) {
    for (int i = tid; i <= a.drafts; i += kThreads)
      if (i != n || owner < 0) out[i] = i < n ? tok[i] : -1;
    if (tid == 0) a.accepted[b] = n;
  }
  if (rank != owner) return;
  // Down to the entry: the warp's run that holds the threshold, summed again in kWarps parts where it is long,
  // and scanned.
  const double thr = static_cast<double>(draw) * total;
  double start;
  int first = (rank * kWarps + max(pick_part(warp_total, kWarps, before, thr, lane, start), 0)) * run;
  int last = min(first + run, a.vocab), by = 0;
  if (run > 512) {
    const int part = (run / kWarps + 3) / 4 * 4, at = first + wid * part, to = min(at + part, last);
    const double s = warp_sum_f64(vec ? run_sum<true>(w, at, to, lane) : run_sum<false>(w, at, to, lane));
    if (lane == 0) part_total[wid] = s;
    __syncthreads();
    by = max(pick_part(part_total, kWarps, start, thr, lane, start), 0);
    first += by * part;
    last = min(first + part, last);
  }
  if (wid != by) return;
  const int j = vec ? run_find<true>(w, first, last, start, thr, lane) : run_find<false>(w, first, last, start, thr, lane);
  if (lane == 0) out[n] = j;
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_verify_drafts(int64_t* out_tokens, int32_t* accepted, const float* target_probs,
                                 int64_t target_stride, const float* draft_probs, int64_t draft_stride,
                                 const int64_t* draft_tokens, const float* uniforms, const int32_t* draft_lens,
                                 int64_t batch, int64_t max_drafts, int64_t vocab, mvb_stream_t stream) {
  MVB_REQUIRE(batch >= 0 && batch <= INT_MAX, "mvb_verify_drafts: batch %lld", (long long)batch);
  MVB_REQUIRE(max_drafts >= 0 && max_drafts <= 4096, "mvb_verify_drafts: %lld drafts (at most 4096)",
              (long long)max_drafts);
  MVB_REQUIRE(vocab > 0 && vocab <= (1 << 24), "mvb_verify_drafts: vocab %lld", (long long)vocab);
  if (batch == 0) return MVB_OK;
  MVB_REQUIRE(out_tokens && accepted && target_probs && uniforms && (max_drafts == 0 || draft_tokens),
              "mvb_verify_drafts: null pointer");
  MVB_REQUIRE(target_stride >= vocab && (draft_probs == nullptr || draft_stride >= vocab),
              "mvb_verify_drafts: rows of %lld and %lld elements for %lld tokens", (long long)target_stride,
              (long long)draft_stride, (long long)vocab);
  VerifyArgs a = {out_tokens, accepted, target_probs, target_stride, draft_probs, draft_stride, draft_tokens, uniforms,
                  draft_lens, static_cast<int>(max_drafts), static_cast<int>(vocab), device_status_ptr()};
  // Blocks per sequence: as many as fill the GPU once (two blocks an SM), with some 2,048 entries each.  Rows of
  // 151,936 entries: at batch 1 one block took 33 us, 4 took 12.6 and 8 take 8.5; at batch 64, 4 take 23.1 us
  // (3.4 TB/s) and 8, in two waves, took 28.7.
  const int64_t sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "mvb_verify_drafts: no device");
  int blocks = kMaxCluster;
  while (blocks > 1 && (vocab < 2048LL * blocks || batch * blocks > 2 * sms)) blocks /= 2;
  const int64_t warps = static_cast<int64_t>(blocks) * kWarps;
  const int run = static_cast<int>(((vocab + warps - 1) / warps + 127) / 128 * 128);
  MVB_REQUIRE(batch * blocks <= INT_MAX, "mvb_verify_drafts: batch %lld", (long long)batch);
  return launch_cluster("verify_drafts", verify_kernel, dim3(static_cast<unsigned>(batch * blocks)), dim3(kThreads),
                        static_cast<unsigned>(blocks), 0, reinterpret_cast<cudaStream_t>(stream), a, blocks, run);
}
