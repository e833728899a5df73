// Attention of the newest tokens of each sequence over a 4-bit paged KV pool.
#include <climits>

#include "common.cuh"
#include "host.h"
#include "kv4.cuh"

namespace mvb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct Kv4AttnArgs {
  __nv_bfloat16* out;
  const __nv_bfloat16* q;
  int64_t out_stride, q_stride;  // elements between query tokens
  const uint8_t* pool;           // the layer's first record
  const int32_t* tables;
  int64_t table_stride;
  int max_blocks;
  const int32_t* ctx;
  int batch, T, hq, hkv;
  int num_blocks, recs;
  float scale_log2, cap_scale, cap_log2;
  int window;
  unsigned* err;
};

// One warp per (query token, query head): lane l owns channels l, l + 32, ...
template <int D>
__global__ void __launch_bounds__(128) kv4_attn_simple(Kv4AttnArgs a) {
  using P = Kv4<D>;
  constexpr int N = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (id >= static_cast<int64_t>(a.batch) * a.T * a.hq) return;
  const int h = static_cast<int>(id % a.hq);
  const int64_t bt = id / a.hq;
  const int t = static_cast<int>(bt % a.T), b = static_cast<int>(bt / a.T);
  const int kvh = h / (a.hq / a.hkv);
  const int bs = a.recs * 16;
  int ctx = a.ctx[b];
  if (ctx < 0 || ctx > a.max_blocks * bs) {
    if (lane == 0) report(a.err, kDevBadPosition);
    ctx = min(max(ctx, 0), a.max_blocks * bs);
  }
  const int end = ctx - a.T + 1 + t;
  const int lo = a.window > 0 ? max(end - a.window, 0) : 0;
  float q[N], o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = __bfloat162float(a.q[bt * a.q_stride + h * D + lane + 32 * i]);
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int pos = lo; pos < end; ++pos) {
    const int blk = a.tables[b * a.table_stride + pos / bs];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) report(a.err, kDevBadBlock);
      continue;
    }
    const uint8_t* r = a.pool + ((static_cast<int64_t>(blk) * a.hkv + kvh) * a.recs + pos % bs / 16) * P::RECORD;
    const int row = pos % 16;
    float k[N], v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = lane + 32 * i, g = c / 64, w = c % 64 / 8, nib = c % 8;
      const int at = row * P::ROW + 4 * (P::NG * w + g) + nib / 2;
      const __nv_bfloat162 kp = *reinterpret_cast<const __nv_bfloat162*>(r + P::K_PAIRS + row * P::PAIRS + 4 * g);
      const __nv_bfloat162 vp = *reinterpret_cast<const __nv_bfloat162*>(r + P::V_PAIRS + row * P::PAIRS + 4 * g);
      const int ku = (r[at] >> (4 * (nib & 1))) & 15, vu = (r[P::V_CODES + at] >> (4 * (nib & 1))) & 15;
      k[i] = fmaf(__bfloat162float(kp.x), static_cast<float>(ku), __bfloat162float(kp.y));
      v[i] = fmaf(__bfloat162float(vp.x), static_cast<float>(vu), __bfloat162float(vp.y));
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], k[i], s);
    s = warp_sum(s);
    s = a.cap_log2 > 0.0f ? a.cap_log2 * tanhf(s * a.cap_scale) : s * a.scale_log2;
    const float mn = fmaxf(m, s);
    const float c0 = exp2f(m - mn), p = exp2f(s - mn);
    l = l * c0 + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * c0 + p * v[i];
    m = mn;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) a.out[bt * a.out_stride + h * D + lane + 32 * i] = __float2bfloat16_rn(o[i] * inv);
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int64_t mvb_paged_attention_decode_kv4_workspace_bytes(int64_t batch, int64_t query_len,
                                                                  int64_t num_q_heads, int64_t num_kv_heads,
                                                                  int64_t head_dim, int device) {
  (void)batch, (void)query_len, (void)num_q_heads, (void)num_kv_heads, (void)head_dim, (void)device;
  return 0;
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
  a.hq = static_cast<int>(num_q_heads);
  a.hkv = static_cast<int>(num_kv_heads);
  a.num_blocks = static_cast<int>(num_blocks);
  a.recs = static_cast<int>(recs);
  a.scale_log2 = scale * kLog2e;
  a.cap_scale = softcap > 0.0f ? scale / softcap : 0.0f;
  a.cap_log2 = softcap * kLog2e;
  a.window = static_cast<int>(window < INT_MAX ? window : INT_MAX);
  a.err = device_status_ptr();
  (void)workspace, (void)workspace_bytes;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t warps = batch * query_len * num_q_heads;
  MVB_REQUIRE((warps + 3) / 4 <= INT_MAX, "%s: batch", what);
  dim3 grid(static_cast<unsigned>((warps + 3) / 4)), block(128);
  switch (head_dim) {
    case 64: return launch("kv4_attention", kv4_attn_simple<64>, grid, block, 0, st, a);
    case 128: return launch("kv4_attention", kv4_attn_simple<128>, grid, block, 0, st, a);
    default: return launch("kv4_attention", kv4_attn_simple<256>, grid, block, 0, st, a);
  }
}
