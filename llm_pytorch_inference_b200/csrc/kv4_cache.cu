// Writing K and V into the 4-bit paged pool, and reading them back.
//
// Per (token, K|V, head, group of 64 channels), with x the bf16 inputs:
//   m = min x,   s = bf16((max x - m) / 15),   u = round((x - m) / s) in 0..15  (0 where s = 0),
// and back: bf16(m + s u).  The division is the IEEE one and the rounding is to even, so codes do
// not depend on how a reciprocal rounds: (x - m) / s of bf16 values lands on .5 exactly quite often.
// A group that holds a NaN or an infinity (or spans more than fp32 holds) gets a NaN pair and reads
// back as NaN.
//
// Both should be bound by memory: 2 bytes a value on the bf16 side, 9/16 on the other.  A lane owns 8 channels of
// K and of V of a token, for one head or two (HEADS): a 16-byte load (or store) of bf16 and one 32-bit word of
// codes each, all under way together and with one look at the token's slot.  Eight lanes share a group.  Its minimum
// and maximum, on packed bf16, are exchanged so that each lane ends up with one of the 2 to 8 groups, works out that
// group's pair alone and hands it round.  Writing still takes 63 % of the issue slots, beside two loads in a row that it
// waits for (the slot, then the rows of K and V; 57 registers leave half of the warps to cover them), so a quotient is a
// product and its correction, two values to an instruction, added to 1.5 * 2^23, which rounds it to even and leaves the
// code in the low bits, and a multiply-add puts it into the word.
// Measured on a B200, K and V of 8 heads of 128: writing 16,384 tokens takes 18.0 us for 86 MB (4.8 TB/s); with every
// lane working out all pairs, values one by one, it took 25, with IEEE divisions 57.  64 tokens: 1.9 us.
// Reading 16,384 tokens: 13.7 us (6.3 TB/s, copying reaches 6.55); 32,768: 29.7 us.
#include <type_traits>

#include "common.cuh"
#include "host.h"
#include "kv4.cuh"

namespace mvb {
namespace {

constexpr int kThreads = 128;  // 64 and 256 took 37.4 and 34.2 us where 128 took 31.6 (the calls at MVB_KV4_LAUNCH)

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

// Record (of head 0) and row of a slot; false for a slot outside the pool (negative slots are padding).
__device__ __forceinline__ bool slot_record(const Kv4Args& a, int64_t slot, int64_t& rec, int& row) {
  if (slot < 0) return false;
  const int64_t t16 = slot >> 4;
  if (t16 >= a.slot_limit16) {
    report(a.err, kDevBadBlock);
    return false;
  }
  const uint32_t t = static_cast<uint32_t>(t16);
  const uint32_t block = a.recs == 1 ? t : t / a.recs;
  rec = static_cast<int64_t>(block) * a.heads * a.recs + (t - block * a.recs);
  row = static_cast<int>(slot & 15);
  return true;
}

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) { return *reinterpret_cast<__nv_bfloat162*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }

constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: a sum's low bits are the rounded addend
constexpr float kFltMax = 3.40282347e38f;
constexpr uint32_t kPackBias = 0x4B400000u * 0x11111111u;  // the magic numbers' bits in the packed word, mod 2^32

// x / d correctly rounded, with y = RN(1 / d): q = RN(x y) is near the quotient, and q + (x - d q) y rounds to it
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  The remainder is
// exact away from underflow.
__device__ __forceinline__ float divided(float x, float d, float y) {
  const float q = x * y;
  return fmaf(fmaf(-d, q, x), y, q);
}

constexpr float kTiny = 0x1p-90f;  // magnitudes from here on are away from underflow

__device__ __forceinline__ float bf16_low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// Codes of 8 values of a group with minimum `low` and scale `scale`, lowest nibble first; inv = RN(1 / scale) where
// scale >= kTiny, which PLAIN says of every group of the warp.
template <bool PLAIN>
__device__ __forceinline__ uint32_t quantise8(const uint32_t (&x)[4], float low, float scale, float inv) {
  uint32_t word = 0;
  if (PLAIN || scale >= kTiny) {
    const F2 low2 = {-low, -low}, scale2 = {-scale, -scale}, inv2 = {inv, inv}, magic2 = {kMagic, kMagic};
#pragma unroll
    for (int j = 3; j >= 0; --j) {  // `divided`, two at a time
      const F2 v = add2({bf16_low(x[j]), bf16_high(x[j])}, low2), q = mul2(v, inv2);
      const F2 u = add2(fma2(fma2(scale2, q, v), inv2, q), magic2);  // at most 15: scale is within 2^-9
      word = (word * 16u + __float_as_uint(u.y)) * 16u + __float_as_uint(u.x);
    }
    return word - kPackBias;
  }
  if (!(scale > 0.0f)) return 0u;  // one value throughout, or none that is a number
#pragma unroll 1
  for (int j = 7; j >= 0; --j) {  // a subnormal scale may leave the largest code above 15
    const uint32_t h = j >= 6 ? x[3] : j >= 4 ? x[2] : j >= 2 ? x[1] : x[0];
    const float v = ((j & 1) ? bf16_high(h) : bf16_low(h)) - low;
    word = word * 16u + static_cast<uint32_t>(fminf(rintf(__fdiv_rn(v, scale)), 15.0f));
  }
  return word;
}

// A lane per (token, HEADS heads, 8 channels).
template <int D, int HEADS>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(const Kv4Args a, const __nv_bfloat16* __restrict__ k,
                                                             const __nv_bfloat16* __restrict__ v) {
  using P = Kv4<D>;
  constexpr int LANES = D / 8, N = 2 * HEADS;  // N groups: K and V of each head
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t x0 = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t per = static_cast<uint32_t>(a.heads / HEADS) * LANES;  // lanes of a token
  const uint32_t token = x0 / per, rest = x0 - token * per;
  const int head = static_cast<int>(rest / LANES) * HEADS, cb = static_cast<int>(rest % LANES);
  const int g = cb >> 3, w = cb & 7;
  // the eight lanes of a group stay or leave together, but the exchanges below name the whole warp: no lane
  // returns before them
  int64_t rec = 0;
  int row = 0;
  const bool live = token < a.tokens && slot_record(a, a.slots[token], rec, row);
  uint4 raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
  if (live) {
    const __nv_bfloat16* ks = k + token * a.k_stride + head * a.k_head_stride + 8 * cb;
    const __nv_bfloat16* vs = v + token * a.v_stride + head * a.v_head_stride + 8 * cb;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      raw[i] = *reinterpret_cast<const uint4*>(ks);
      raw[i + 1] = *reinterpret_cast<const uint4*>(vs);
      ks += a.k_head_stride;
      vs += a.v_head_stride;
    }
  }
  // (minimum, -maximum) of the lane's values of each group, in one word
  uint32_t ext[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    __nv_bfloat162 lo2 = as_bf162(x[0]), hi2 = lo2;
#pragma unroll
    for (int j = 1; j < 4; ++j) {
      lo2 = __hmin2_nan(lo2, as_bf162(x[j]));
      hi2 = __hmax2_nan(hi2, as_bf162(x[j]));
    }
    ext[i] = as_u32(__halves2bfloat162(__hmin_nan(lo2.x, lo2.y), __hneg(__hmax_nan(hi2.x, hi2.y))));
  }
  // Exchanged among the eight lanes so that lane w ends up with group w % N: half of the groups are handed over at a
  // time.  That group's pair is this lane's work; all read it afterwards.
  auto least = [](uint32_t x, uint32_t y) { return as_u32(__hmin2_nan(as_bf162(x), as_bf162(y))); };
#pragma unroll
  for (int o = 1; o < N; o <<= 1) {
    const bool odd = w & o;
#pragma unroll
    for (int i = 0; i < N / 2 / o; ++i) {  // those left: numbers i and i + 1 differ in bit o of the group
      const uint32_t keep = odd ? ext[2 * i + 1] : ext[2 * i], give = odd ? ext[2 * i] : ext[2 * i + 1];
      ext[i] = least(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
#pragma unroll
  for (int o = N; o < 8; o <<= 1) ext[0] = least(ext[0], __shfl_xor_sync(0xffffffffu, ext[0], o));
  float low = bf16_low(ext[0]);
  const float span = -bf16_high(ext[0]) - low;
  float scale = bf16_round(span < kTiny ? __fdiv_rn(span, 15.0f) : divided(span, 15.0f, 1.0f / 15.0f));
  if (!(scale <= kFltMax) || !(fabsf(low) <= kFltMax)) scale = low = __int_as_float(0x7fc00000);
  const float inv = __frcp_rn(scale);
  const uint32_t pair = as_u32(__floats2bfloat162_rn(scale, low));

  uint8_t* at = a.pool + (rec + static_cast<int64_t>(head) * a.recs) * P::RECORD;
  if (live && w < N)
    *reinterpret_cast<uint32_t*>(at + (w >> 1) * a.recs * P::RECORD + ((w & 1) ? P::V_PAIRS : P::K_PAIRS) +
                                 row * P::PAIRS + 4 * g) = pair;
  at += row * P::ROW + 4 * (P::NG * w + g);
  auto store = [&](auto plain_tag) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int from = (threadIdx.x & 24) | i;
      const uint32_t pi = __shfl_sync(0xffffffffu, pair, from);
      const float inv_i = __shfl_sync(0xffffffffu, inv, from);
      const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      const uint32_t word = quantise8<decltype(plain_tag)::value>(x, bf16_high(pi), bf16_low(pi), inv_i);
      if (live) *reinterpret_cast<uint32_t*>(at + (i >> 1) * a.recs * P::RECORD + ((i & 1) ? P::V_CODES : 0)) = word;
    }
  };
  if (__all_sync(0xffffffffu, scale >= kTiny))  // no branch a group: 33.4 -> 32.5 us at head size 256
    store(std::true_type{});
  else
    store(std::false_type{});
}

// A lane per (token, HEADS heads, 8 channels).  A token without a slot in the pool reads as zeros.  A code is
// the bf16 number 128 + u by its bits; scale * u + min is one bf16 fma, rounded once.
template <int D, int HEADS>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const Kv4Args a, __nv_bfloat16* __restrict__ k,
                                                            __nv_bfloat16* __restrict__ v) {
  using P = Kv4<D>;
  constexpr int LANES = D / 8, N = 2 * HEADS;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t x0 = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t per = static_cast<uint32_t>(a.heads / HEADS) * LANES;
  const uint32_t token = x0 / per, rest = x0 - token * per;
  if (token >= a.tokens) return;
  const int head = static_cast<int>(rest / LANES) * HEADS, cb = static_cast<int>(rest % LANES);
  const int g = cb >> 3, w = cb & 7;
  int64_t rec = 0;
  int row = 0;
  const bool live = slot_record(a, a.slots[token], rec, row);
  const uint8_t* r = a.pool + (rec + static_cast<int64_t>(head) * a.recs) * P::RECORD;
  uint32_t word[N], pair[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    word[i] = pair[i] = 0;
    if (live) {
      const uint8_t* at = r + (i >> 1) * a.recs * P::RECORD;
      word[i] = *reinterpret_cast<const uint32_t*>(at + ((i & 1) ? P::V_CODES : 0) + row * P::ROW + 4 * (P::NG * w + g));
      pair[i] = *reinterpret_cast<const uint32_t*>(at + ((i & 1) ? P::V_PAIRS : P::K_PAIRS) + row * P::PAIRS + 4 * g);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const __nv_bfloat162 scale = as_bf162(__byte_perm(pair[i], 0, 0x1010)), low = as_bf162(__byte_perm(pair[i], 0, 0x3232));
    const __nv_bfloat162 bias = as_bf162(0x43004300u);  // 128, 128
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // codes j and j + 4
      const uint32_t u = ((word[i] >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
      y[j] = as_u32(__hfma2(scale, __hsub2(as_bf162(u), bias), low));
    }
    const uint4 o = make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410),
                               __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632));
    const int h = head + (i >> 1);
    __nv_bfloat16* dst = (i & 1) ? v + token * a.v_stride + h * a.v_head_stride
                                 : k + token * a.k_stride + h * a.k_head_stride;
    *reinterpret_cast<uint4*>(dst + 8 * cb) = o;
  }
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

// Two or four heads a lane where they come in such numbers and there are lanes enough to fill the GPU all the same.
// Writing and reading 16,384 tokens, K and V of 8 heads of 128: 34.0 us with two, 31.6 with four.
#define MVB_KV4_LAUNCH(NAME, KERNEL, ...)                                                                 \
  do {                                                                                                    \
    const int64_t lanes = tokens * num_kv_heads * (head_dim / 8);                                         \
    const int each = lanes < (1 << 18) || num_kv_heads % 2 ? 1 : lanes < (1 << 19) || num_kv_heads % 4 ? 2 : 4; \
    const dim3 grid(static_cast<unsigned>((lanes / each + kThreads - 1) / kThreads)), block(kThreads);    \
    switch (head_dim + each) {                                                                            \
      case 65: return launch(NAME, KERNEL<64, 1>, grid, block, 0, st, a, __VA_ARGS__);                    \
      case 66: return launch(NAME, KERNEL<64, 2>, grid, block, 0, st, a, __VA_ARGS__);                    \
      case 68: return launch(NAME, KERNEL<64, 4>, grid, block, 0, st, a, __VA_ARGS__);                    \
      case 129: return launch(NAME, KERNEL<128, 1>, grid, block, 0, st, a, __VA_ARGS__);                  \
      case 130: return launch(NAME, KERNEL<128, 2>, grid, block, 0, st, a, __VA_ARGS__);                  \
      case 132: return launch(NAME, KERNEL<128, 4>, grid, block, 0, st, a, __VA_ARGS__);                  \
      case 257: return launch(NAME, KERNEL<256, 1>, grid, block, 0, st, a, __VA_ARGS__);                  \
      case 258: return launch(NAME, KERNEL<256, 2>, grid, block, 0, st, a, __VA_ARGS__);                  \
      default: return launch(NAME, KERNEL<256, 4>, grid, block, 0, st, a, __VA_ARGS__);                   \
    }                                                                                                     \
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
