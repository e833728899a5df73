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
// Only one row of p (and of q) is read per sequence: bound by those 4 (8) bytes an entry, and by
// latency for few sequences.
#include <climits>

#include "common.cuh"
#include "host.h"

namespace mvb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTiles = 2048;

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

// What entry j of the row weighs in the draw.
struct Weights {
  const float* p;
  const float* q;   // the drafting row, or nullptr
  int token;        // the rejected one-hot draft, or -1
  __device__ __forceinline__ double operator()(int j) const {
    const double a = p[j];
    if (q != nullptr) return fmax(a - static_cast<double>(q[j]), 0.0);
    return j == token ? 0.0 : fmax(a, 0.0);
  }
};

// One CTA per sequence.
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyArgs a) {
  __shared__ double tile_sum[kMaxTiles];
  __shared__ double total_s;
  __shared__ int found;
  // dependents start at this kernel's end only: they read its outputs as step metadata before they wait
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t* tok = a.tokens + static_cast<int64_t>(b) * a.drafts;
  const float* u = a.u + static_cast<int64_t>(b) * (a.drafts + 1);
  const int n_drafts = a.lens != nullptr ? min(max(a.lens[b], 0), a.drafts) : a.drafts;
  int n = 0;
  for (; n < n_drafts; ++n) {
    const int64_t d = tok[n];
    if (d < 0 || d >= a.vocab) {
      if (tid == 0) report(a.err, kDevBadToken);
      break;
    }
    const double pd = a.p[(static_cast<int64_t>(b) * (a.drafts + 1) + n) * a.p_stride + d];
    const double qd = a.q != nullptr ? a.q[(static_cast<int64_t>(b) * a.drafts + n) * a.q_stride + d] : 1.0;
    if (!(static_cast<double>(u[n]) * qd < pd)) break;
  }
  const bool rejected = n < n_drafts;
  Weights w;
  w.p = a.p + (static_cast<int64_t>(b) * (a.drafts + 1) + n) * a.p_stride;
  w.q = rejected && a.q != nullptr ? a.q + (static_cast<int64_t>(b) * a.drafts + n) * a.q_stride : nullptr;
  w.token = -1;
  if (rejected && a.q == nullptr && tok[n] >= 0 && tok[n] < a.vocab) w.token = static_cast<int>(tok[n]);

  const int tile = (((a.vocab + kMaxTiles - 1) / kMaxTiles + 127) / 128) * 128;
  const int tiles = (a.vocab + tile - 1) / tile;
  for (int pass = 0; pass < 2; ++pass) {
    for (int t = wid; t < tiles; t += kWarps) {
      double s = 0.0;
      const int end = min((t + 1) * tile, a.vocab);
      for (int j = t * tile + lane; j < end; j += 32) s += w(j);
      s = warp_sum_f64(s);
      if (lane == 0) tile_sum[t] = s;
    }
    __syncthreads();
    if (wid == 0) {
      double s = 0.0;
      for (int t = lane; t < tiles; t += 32) s += tile_sum[t];
      s = warp_sum_f64(s);
      if (lane == 0) total_s = s;
    }
    __syncthreads();
    if (total_s > 0.0 || !rejected) break;
    // nothing is left of p - q (equal rows, or rounding): draw from p itself
    __syncthreads();
    w.q = nullptr;
    w.token = -1;
  }
  if (wid == 0) {
    // `total_s > 0` false: no entry weighs anything (or a NaN): no token
    int pick = -1;
    const double total = total_s;
    if (total > 0.0) {
      const double thr = static_cast<double>(u[a.drafts]) * total;
      double before = 0.0;
      int t = 0;
      for (; t < tiles - 1 && !(before + tile_sum[t] > thr); ++t) before += tile_sum[t];
      const int end = min((t + 1) * tile, a.vocab);
      int last = -1;
      for (int j0 = t * tile; j0 < end && pick < 0; j0 += 32) {
        const int j = j0 + lane;
        const double x = j < end ? w(j) : 0.0;
        double c = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) c += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + c > thr && x > 0.0);
        const unsigned any = __ballot_sync(0xffffffffu, x > 0.0);
        if (hit) pick = j0 + __ffs(hit) - 1;
        if (any) last = j0 + 31 - __clz(any);
        before += __shfl_sync(0xffffffffu, c, 31);
      }
      if (pick < 0) pick = last;
    }
    if (lane == 0) found = pick;
  }
  __syncthreads();
  int64_t* out = a.out + static_cast<int64_t>(b) * (a.drafts + 1);
  for (int i = tid; i <= a.drafts; i += kThreads) out[i] = i < n ? tok[i] : i == n ? found : -1;
  if (tid == 0) a.accepted[b] = n;
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
  return launch("verify_drafts", verify_kernel, dim3(static_cast<unsigned>(batch)), dim3(kThreads), 0,
                reinterpret_cast<cudaStream_t>(stream), a);
}
