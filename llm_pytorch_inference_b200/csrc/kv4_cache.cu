// Writing K and V into the 4-bit paged pool, and reading them back.
//
// Per (token, K|V, head, group of 64 channels), with x the bf16 inputs:
//   m = min x,   s = bf16((max x - m) / 15),   u = round((x - m) / s) in 0..15  (0 where s = 0),
// and back: bf16(m + s u).  The division is the IEEE one and the rounding is to even, so codes do
// not depend on how a reciprocal rounds: (x - m) / s of bf16 values lands on .5 exactly quite often.
// A group that holds a NaN or an infinity (or spans more than fp32 holds) gets a NaN pair and reads
// back as NaN.
//
// Both are bound by memory: 2 bytes a value on the bf16 side, 9/16 on the other.  A lane owns
// 8 channels: a 16-byte load (or store) of bf16 and one 32-bit word of codes; eight lanes share a
// group and find its minimum and maximum with three exchanges.
#include "common.cuh"
#include "host.h"
#include "kv4.cuh"

namespace mvb {
namespace {

constexpr int kThreads = 256;

struct Kv4Args {
  uint8_t* pool;          // the layer's first record
  const int64_t* slots;
  int64_t tokens;
  int64_t k_stride, k_head_stride, v_stride, v_head_stride;  // elements
  uint32_t slot_limit16;  // num_blocks * block_size / 16
  uint32_t recs;          // records of a (block, head): block_size / 16
  int heads;
  unsigned* err;
};

// Record and row of a slot; false for a slot outside the pool (negative slots are padding).
__device__ __forceinline__ bool slot_record(const Kv4Args& a, int64_t slot, int head, int64_t& rec, int& row) {
  if (slot < 0) return false;
  const int64_t t16 = slot >> 4;
  if (t16 >= a.slot_limit16) {
    report(a.err, kDevBadBlock);
    return false;
  }
  const uint32_t t = static_cast<uint32_t>(t16);
  const uint32_t block = t / a.recs;
  rec = (static_cast<int64_t>(block) * a.heads + head) * a.recs + (t - block * a.recs);
  row = static_cast<int>(slot & 15);
  return true;
}

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) {
  return *reinterpret_cast<__nv_bfloat162*>(&v);
}
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }

// One lane per (token, K|V, head, 8 channels).
template <int D>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(Kv4Args a, const __nv_bfloat16* __restrict__ k,
                                                             const __nv_bfloat16* __restrict__ v) {
  using P = Kv4<D>;
  constexpr int LANES = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t gt = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t unit = gt / LANES;
  const int cb = static_cast<int>(gt % LANES);
  const int64_t token = unit / (2 * a.heads);
  const int rest = static_cast<int>(unit - token * 2 * a.heads);
  const bool is_v = rest >= a.heads;
  const int head = is_v ? rest - a.heads : rest;
  // all lanes of an 8-lane group share the unit, so they stay or leave together; the exchanges below
  // name the whole warp, so no lane returns before them
  bool live = token < a.tokens;
  int64_t rec = 0;
  int row = 0;
  live = live && slot_record(a, live ? a.slots[token] : -1, head, rec, row);
  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  if (live) {
    const __nv_bfloat16* src = is_v ? v + token * a.v_stride + head * a.v_head_stride
                                    : k + token * a.k_stride + head * a.k_head_stride;
    raw = *reinterpret_cast<const uint4*>(src + 8 * cb);
  }
  const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
  __nv_bfloat162 lo2 = as_bf162(x[0]), hi2 = lo2;
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    lo2 = __hmin2_nan(lo2, as_bf162(x[i]));
    hi2 = __hmax2_nan(hi2, as_bf162(x[i]));
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo2 = __hmin2_nan(lo2, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(lo2), o)));
    hi2 = __hmax2_nan(hi2, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(hi2), o)));
  }
  if (!live) return;
  const float low = __bfloat162float(__hmin_nan(lo2.x, lo2.y));
  const float high = __bfloat162float(__hmax_nan(hi2.x, hi2.y));
  float scale = bf16_round(__fdiv_rn(high - low, 15.0f));
  float base = low;
  if (!(fabsf(scale) <= 3.3895314e38f) || !(fabsf(low) <= 3.3895314e38f))
    scale = base = __int_as_float(0x7fc00000);
  uint32_t word = 0;
  if (scale > 0.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float xv = __uint_as_float((i & 1) ? (x[i >> 1] & 0xffff0000u) : (x[i >> 1] << 16));
      const int u = __float2int_rn(__fdiv_rn(xv - base, scale));
      word |= static_cast<uint32_t>(min(max(u, 0), 15)) << (4 * i);
    }
  }
  const int g = cb >> 3, w = cb & 7;
  uint8_t* r = a.pool + rec * P::RECORD;
  *reinterpret_cast<uint32_t*>(r + (is_v ? P::V_CODES : 0) + row * P::ROW + 4 * (P::NG * w + g)) = word;
  if (w == 0)
    *reinterpret_cast<__nv_bfloat162*>(r + (is_v ? P::V_PAIRS : P::K_PAIRS) + row * P::PAIRS + 4 * g) =
        __floats2bfloat162_rn(scale, base);
}

// One lane per (token, K|V, head, 8 channels).  A token without a slot in the pool reads as zeros.
template <int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Kv4Args a, __nv_bfloat16* __restrict__ k,
                                                            __nv_bfloat16* __restrict__ v) {
  using P = Kv4<D>;
  constexpr int LANES = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t gt = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t unit = gt / LANES;
  const int cb = static_cast<int>(gt % LANES);
  const int64_t token = unit / (2 * a.heads);
  if (token >= a.tokens) return;
  const int rest = static_cast<int>(unit - token * 2 * a.heads);
  const bool is_v = rest >= a.heads;
  const int head = is_v ? rest - a.heads : rest;
  int64_t rec;
  int row;
  uint4 o = make_uint4(0u, 0u, 0u, 0u);
  if (slot_record(a, a.slots[token], head, rec, row)) {
    const uint8_t* r = a.pool + rec * P::RECORD;
    const int g = cb >> 3, w = cb & 7;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(r + (is_v ? P::V_CODES : 0) + row * P::ROW +
                                                             4 * (P::NG * w + g));
    const __nv_bfloat162 pair = *reinterpret_cast<const __nv_bfloat162*>(r + (is_v ? P::V_PAIRS : P::K_PAIRS) +
                                                                         row * P::PAIRS + 4 * g);
    const float scale = __bfloat162float(pair.x), base = __bfloat162float(pair.y);
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // scale * u is exact in fp32 (8 + 4 bits): one rounding in the fma, one to bf16
      q[i] = as_u32(__floats2bfloat162_rn(fmaf(scale, static_cast<float>((word >> (8 * i)) & 15u), base),
                                          fmaf(scale, static_cast<float>((word >> (8 * i + 4)) & 15u), base)));
    o = make_uint4(q[0], q[1], q[2], q[3]);
  }
  __nv_bfloat16* dst = is_v ? v + token * a.v_stride + head * a.v_head_stride
                            : k + token * a.k_stride + head * a.k_head_stride;
  *reinterpret_cast<uint4*>(dst + 8 * cb) = o;
}

int kv4_args(Kv4Args& a, const char* what, const void* pool, const int64_t* slots, int64_t tokens, int64_t heads,
             int64_t head_dim, int64_t num_layers, int64_t layer, int64_t num_blocks, int64_t block_size) {
  MVB_REQUIRE(pool && slots, "%s: null pointer", what);
  MVB_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: head_dim %lld (64, 128 or 256)", what,
              (long long)head_dim);
  MVB_REQUIRE(heads > 0 && heads <= 65536, "%s: %lld KV heads", what, (long long)heads);
  MVB_REQUIRE(layer >= 0 && layer < num_layers, "%s: layer %lld of %lld", what, (long long)layer,
              (long long)num_layers);
  MVB_REQUIRE(block_size > 0 && block_size % kKv4Tokens == 0 && block_size <= (1 << 20),
              "%s: block_size %lld (a multiple of 16)", what, (long long)block_size);
  MVB_REQUIRE(num_blocks > 0 && num_blocks <= (int64_t(1) << 31) / (block_size / 16), "%s: %lld blocks", what,
              (long long)num_blocks);
  MVB_REQUIRE(aligned(pool, 16), "%s: the pool must be 16-byte aligned", what);
  MVB_REQUIRE(tokens >= 0 && tokens <= (int64_t(1) << 31) * 8 / (heads * head_dim), "%s: %lld tokens", what,
              (long long)tokens);
  a.recs = static_cast<uint32_t>(block_size / 16);
  a.slot_limit16 = static_cast<uint32_t>(num_blocks * a.recs);
  a.pool = static_cast<uint8_t*>(const_cast<void*>(pool)) + layer * num_blocks * heads * a.recs * 18 * head_dim;
  a.slots = slots;
  a.tokens = tokens;
  a.heads = static_cast<int>(heads);
  return MVB_OK;
}

int stride_ok(const char* what, const void* p, int64_t stride, int64_t head_stride, int64_t head_dim) {
  MVB_REQUIRE(p, "%s: null pointer", what);
  MVB_REQUIRE(aligned(p, 16) && stride % 8 == 0 && head_stride % 8 == 0 && stride >= 0 && head_stride >= 0,
              "%s: rows of K and V must be 16-byte aligned (strides %lld, %lld)", what, (long long)stride,
              (long long)head_stride);
  (void)head_dim;
  return MVB_OK;
}

}  // namespace
}  // namespace mvb

using namespace mvb;

#define MVB_KV4_LAUNCH(NAME, KERNEL, ...)                                                                \
  do {                                                                                                   \
    const int64_t lanes = tokens * 2 * num_kv_heads * (head_dim / 8);                                    \
    dim3 grid(static_cast<unsigned>((lanes + kThreads - 1) / kThreads)), block(kThreads);                \
    switch (head_dim) {                                                                                  \
      case 64: return launch(NAME, KERNEL<64>, grid, block, 0, st, a, __VA_ARGS__);                      \
      case 128: return launch(NAME, KERNEL<128>, grid, block, 0, st, a, __VA_ARGS__);                    \
      default: return launch(NAME, KERNEL<256>, grid, block, 0, st, a, __VA_ARGS__);                     \
    }                                                                                                    \
  } while (0)

extern "C" int mvb_kv4_write(void* kv4, const void* k, int64_t k_stride, int64_t k_head_stride, const void* v,
                             int64_t v_stride, int64_t v_head_stride, const int64_t* slots, int64_t tokens,
                             int64_t num_kv_heads, int64_t head_dim, int64_t num_layers, int64_t layer,
                             int64_t num_blocks, int64_t block_size, mvb_stream_t stream) {
  Kv4Args a = {};
  MVB_TRY(kv4_args(a, "mvb_kv4_write", kv4, slots, tokens, num_kv_heads, head_dim, num_layers, layer, num_blocks,
                   block_size));
  MVB_TRY(stride_ok("mvb_kv4_write", k, k_stride, k_head_stride, head_dim));
  MVB_TRY(stride_ok("mvb_kv4_write", v, v_stride, v_head_stride, head_dim));
  if (tokens == 0) return MVB_OK;
  a.k_stride = k_stride;
  a.k_head_stride = k_head_stride;
  a.v_stride = v_stride;
  a.v_head_stride = v_head_stride;
  a.err = device_status_ptr();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  MVB_KV4_LAUNCH("kv4_write", kv4_write_kernel, static_cast<const __nv_bfloat16*>(k),
                 static_cast<const __nv_bfloat16*>(v));
}

extern "C" int mvb_kv4_read(void* k, void* v, const void* kv4, const int64_t* slots, int64_t tokens,
                            int64_t num_kv_heads, int64_t head_dim, int64_t num_layers, int64_t layer,
                            int64_t num_blocks, int64_t block_size, mvb_stream_t stream) {
  Kv4Args a = {};
  MVB_TRY(kv4_args(a, "mvb_kv4_read", kv4, slots, tokens, num_kv_heads, head_dim, num_layers, layer, num_blocks,
                   block_size));
  MVB_TRY(stride_ok("mvb_kv4_read", k, num_kv_heads * head_dim, head_dim, head_dim));
  MVB_TRY(stride_ok("mvb_kv4_read", v, num_kv_heads * head_dim, head_dim, head_dim));
  if (tokens == 0) return MVB_OK;
  a.k_stride = a.v_stride = num_kv_heads * head_dim;
  a.k_head_stride = a.v_head_stride = head_dim;
  a.err = device_status_ptr();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  MVB_KV4_LAUNCH("kv4_read", kv4_read_kernel, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v));
}
