// Weights in 4 bits with group scales (w4.cuh): quantised from a bf16 matrix, packed from a checkpoint's codes, read back.
//
// Quantised, per row and group: lo = min(0, min w), hi = max(0, max w), scale = bf16((hi - lo) / 15),
// zero = rint(-lo / scale), code = rint(w / scale) + zero, both cut to 0 .. 15.  The codes are chosen against the rounded
// scale, so that its rounding adds nothing to their half step.  A group with a NaN or an infinity, or whose hi - lo leaves
// fp32's range, gets the scale NaN and reads back as NaN.
//
// Bound by memory: 2 bytes in and 0.53 out per weight (and back).  Half a warp takes 128 columns of a row, 8 a lane:
// one 16-byte load, and one word of codes; a warp takes a record, 8 pairs of rows, whose loads are all under way first.
// A group's extremes cross 16, 8 or 4 lanes as one packed pair (max of -w and of w), 4, 3 or 2 exchanges.
// Measured, 24576 x 4096 in groups of 64 (255 MB either way, 39 us at the rate of a copy): quantising 59 us, bound by
// what it computes (81 % of the issue slots before its last step, which took two sums a code out); reading back 42.6 us,
// bound by memory.
//
// The makers let no kernel start before they end, and what they wrote is at the GPU's scope before they do: products read
// records before they wait for the kernel before them.
#include <climits>

#include "common.cuh"
#include "host.h"
#include "w4.cuh"

namespace mvb {
namespace {

constexpr int kThreads = 256;

struct W4Shape {
  int n, k, tiles, blocks;
  int64_t records;
};

// The record that a warp works on.
struct Place {
  int tile, block;
  __device__ __forceinline__ Place(int64_t r, const W4Shape& s) {
    const int64_t whole = static_cast<int64_t>(s.tiles & ~7) * s.blocks;
    if (r < whole) {
      const int64_t q = r >> 3;
      const int big = static_cast<int>(q / s.blocks);
      block = static_cast<int>(q - static_cast<int64_t>(big) * s.blocks);
      tile = big * 8 + static_cast<int>(r & 7);
    } else {
      const int left = s.tiles & 7, at = static_cast<int>(r - whole);
      block = at / left;
      tile = (s.tiles & ~7) + (at - block * left);
    }
  }
};

__device__ __forceinline__ uint32_t word_of(const uint32_t (&u)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= u[e] << (4 * w4_nibble(e));
  return w;
}

// Larger and smaller numbers of two pairs of bf16, NaN where either is.
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ float low_bf16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_bf16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// x / 15, rounded once: the product with 1/15 and what it leaves over.  NaN for an infinity.
__device__ __forceinline__ float fifteenth(float x) {
  const float q = x * (1.0f / 15.0f);
  return fmaf(fmaf(-15.0f, q, x), 1.0f / 15.0f, q);
}

template <int GROUP>
__global__ void __launch_bounds__(kThreads) quantise_w4_kernel(uint8_t* __restrict__ records,
                                                               const __nv_bfloat16* __restrict__ w, int64_t w_stride,
                                                               const W4Shape s) {
  constexpr int PER = kW4Cols / GROUP, LANES = GROUP / 8;
  pdl_wait();
  const int lane = threadIdx.x & 31, part = lane & 15, half = lane >> 4;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= s.records) return;
  const Place at(r, s);
  uint8_t* rec = records + r * w4_record_bytes(GROUP);
  const int col = at.block * kW4Cols + 8 * part;
  uint4 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = at.tile * kW4Rows + 2 * i + half;
    x[i] = make_uint4(0, 0, 0, 0);
    if (row < s.n && col < s.k) x[i] = *reinterpret_cast<const uint4*>(w + row * w_stride + col);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 2 * i + half;
    const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    // high: the largest, low: the largest of the negated
    const uint32_t up = max2(max2(v[0], v[1]), max2(v[2], v[3]));
    const uint32_t down = min2(min2(v[0], v[1]), min2(v[2], v[3])) ^ 0x80008000u;
    uint32_t both = max2(__byte_perm(down, up, 0x5410), __byte_perm(down, up, 0x7632));
    both = max2(both, 0u);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) both = max2(both, __shfl_xor_sync(0xffffffffu, both, o));
    const float low = low_bf16(both), high = high_bf16(both);  // -lo and hi
    const __nv_bfloat16 sb = __float2bfloat16_rn(fifteenth(high + low));
    const float scale = __bfloat162float(sb);
    uint32_t word = 0, zero = 0;
    if (scale > 0.0f && scale < __uint_as_float(0x7f800000u)) {
      // Quotients of two bf16 numbers below 16 either fall on a border between codes or are 1e-3 away from it, and
      // the product with the reciprocal is off by 4e-6: rounded to a multiple of 2^-13 (the sum with 1536), it falls on the
      // right side, or on the border.  The next sum, 1.5 * 2^23 and 16 above the quotient, has the whole number and
      // 16 for its low bits.  It is never below -zero, since rounding is monotonic and odd; the most is cut.
      constexpr float kMagic = 12582928.0f;
      float y[8], least = low, by = scale;
#pragma unroll
      for (int e = 0; e < 8; e += 2) y[e] = low_bf16(v[e >> 1]), y[e + 1] = high_bf16(v[e >> 1]);
      if (scale < 1.1754944e-38f) {
        // Its reciprocal would overflow: all times 2^64.  And it may have been rounded down by so much that -lo is more than
        // 15.5 of it (normal scales: 15.06 at most): cut to 15 there, and with it what is below -15.
        constexpr float kUp = 1.8446744e19f;
        by *= kUp;
        least = fminf(least * kUp, 15.0f * by);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaxf(y[e] * kUp, -15.0f * by);
      }
      float inv;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(by));
      const float z = (least * inv + 1536.0f) + (kMagic - 1536.0f);
      zero = __float_as_uint(z) - __float_as_uint(kMagic);
      const float most = (kMagic + 15.0f) - (z - kMagic);
      uint32_t u[8];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float2 t = __fmul2_rn(make_float2(y[e], y[e + 1]), make_float2(inv, inv));
        t = __fadd2_rn(__fadd2_rn(t, make_float2(1536.0f, 1536.0f)), make_float2(kMagic - 1536.0f, kMagic - 1536.0f));
        u[e] = __float_as_uint(fminf(t.x, most));
        u[e + 1] = __float_as_uint(fminf(t.y, most));
      }
      // The low bytes of columns 0 4 1 5 make the low nibbles, those of 2 6 3 7 the high ones; all less 16 plus zero.
      const uint32_t more = zero * 0x01010101u - 0x10101010u;
      const uint32_t below = __byte_perm(__byte_perm(u[0], u[4], 0x0040), __byte_perm(u[1], u[5], 0x0040), 0x5410) + more;
      const uint32_t above = __byte_perm(__byte_perm(u[2], u[6], 0x0040), __byte_perm(u[3], u[7], 0x0040), 0x5410) + more;
      word = below | above << 4;
    }
    const bool some = at.tile * kW4Rows + row < s.n && col < s.k;  // else it stays zero
    *reinterpret_cast<uint32_t*>(rec + row * 64 + w4_place(part & 3, row) * 16 + (part >> 2) * 4) = some ? word : 0u;
    if (part % LANES == 0) {
      const uint32_t pair = __bfloat16_as_ushort(sb) | (0x4300u | zero) << 16;
      *reinterpret_cast<uint32_t*>(rec + kW4CodeBytes + (row * PER + part / LANES) * 4) = some ? pair : 0u;
    }
  }
  fence_acq_rel_gpu();
}

template <int GROUP>
__global__ void __launch_bounds__(kThreads) pack_w4_kernel(uint8_t* __restrict__ records,
                                                           const uint8_t* __restrict__ codes,
                                                           const uint16_t* __restrict__ scales,
                                                           const uint8_t* __restrict__ zeros, const W4Shape s) {
  constexpr int PER = kW4Cols / GROUP, LANES = GROUP / 8;
  pdl_wait();
  const int lane = threadIdx.x & 31, part = lane & 15, half = lane >> 4;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= s.records) return;
  const Place at(r, s);
  uint8_t* rec = records + r * w4_record_bytes(GROUP);
  const int col = at.block * kW4Cols + 8 * part;
  const int64_t groups = (s.k + GROUP - 1) / GROUP;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 2 * i + half;
    const int64_t n = at.tile * kW4Rows + row;
    const bool some = n < s.n && col < s.k;
    uint32_t u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (some) {
      const uint2 c = *reinterpret_cast<const uint2*>(codes + n * s.k + col);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = (e < 4 ? c.x >> (8 * e) : c.y >> (8 * (e - 4))) & 15u;
    }
    *reinterpret_cast<uint32_t*>(rec + row * 64 + w4_place(part & 3, row) * 16 + (part >> 2) * 4) = word_of(u);
    if (part % LANES == 0) {
      uint32_t pair = 0;
      if (some) {
        const int64_t g = n * groups + col / GROUP;
        pair = scales[g] | (0x4300u | (zeros != nullptr ? zeros[g] & 15u : 8u)) << 16;
      }
      *reinterpret_cast<uint32_t*>(rec + kW4CodeBytes + (row * PER + part / LANES) * 4) = pair;
    }
  }
  fence_acq_rel_gpu();
}

template <int GROUP, typename T>
__global__ void __launch_bounds__(kThreads) dequantise_w4_kernel(T* __restrict__ out, const uint8_t* __restrict__ records,
                                                                 const W4Shape s) {
  constexpr int PER = kW4Cols / GROUP, LANES = GROUP / 8;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, part = lane & 15, half = lane >> 4;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= s.records) return;
  const Place at(r, s);
  const uint8_t* rec = records + r * w4_record_bytes(GROUP);
  const int col = at.block * kW4Cols + 8 * part;
  uint32_t word[8], pair[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 2 * i + half;
    word[i] = *reinterpret_cast<const uint32_t*>(rec + row * 64 + w4_place(part & 3, row) * 16 + (part >> 2) * 4);
    pair[i] = *reinterpret_cast<const uint32_t*>(rec + kW4CodeBytes + (row * PER + part / LANES) * 4);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = at.tile * kW4Rows + 2 * i + half;
    if (n >= s.n || col >= s.k) continue;
    const float scale = low_bf16(pair[i]), zero = static_cast<float>(pair[i] >> 16 & 15u);
    T* o = out + n * s.k + col;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = scale * (static_cast<float>(word[i] >> (4 * w4_nibble(e)) & 15u) - zero);
    if (sizeof(T) == 4) {
      reinterpret_cast<float4*>(o)[0] = make_float4(y[0], y[1], y[2], y[3]);
      reinterpret_cast<float4*>(o)[1] = make_float4(y[4], y[5], y[6], y[7]);
    } else {
      uint4 v;
      T* p = reinterpret_cast<T*>(&v);
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = from_f<T>(y[e]);
      *reinterpret_cast<uint4*>(o) = v;
    }
  }
}

int shape_of(const char* name, int64_t n, int64_t k, int64_t group, W4Shape& s) {
  MVB_REQUIRE(n >= 0 && n <= (1 << 24), "%s: %lld rows", name, (long long)n);
  MVB_REQUIRE(k > 0 && k <= (1 << 24) && k % 32 == 0, "%s: %lld columns (a multiple of 32)", name, (long long)k);
  MVB_REQUIRE(group == 32 || group == 64 || group == 128, "%s: groups of %lld columns (32, 64 or 128)", name,
              (long long)group);
  s.n = static_cast<int>(n);
  s.k = static_cast<int>(k);
  s.tiles = (s.n + kW4Rows - 1) / kW4Rows;
  s.blocks = (s.k + kW4Cols - 1) / kW4Cols;
  s.records = static_cast<int64_t>(s.tiles) * s.blocks;
  MVB_REQUIRE(s.records <= 8LL * INT_MAX, "%s: %lld by %lld", name, (long long)n, (long long)k);
  return MVB_OK;
}

template <typename... KArgs, typename... Args>
int run_records(const char* name, void (*kernel)(KArgs...), const W4Shape& s, cudaStream_t stream, Args&&... args) {
  const int64_t blocks = (s.records + kThreads / 32 - 1) / (kThreads / 32);
  return launch(name, kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, args..., s);
}

template <int GROUP>
int run_dequantise(const char* name, void* out, const uint8_t* records, const W4Shape& s, int dtype, cudaStream_t st) {
  if (dtype == MVB_F32) return run_records(name, dequantise_w4_kernel<GROUP, float>, s, st, static_cast<float*>(out), records);
  return run_records(name, dequantise_w4_kernel<GROUP, __nv_bfloat16>, s, st, static_cast<__nv_bfloat16*>(out), records);
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int64_t mvb_w4_bytes(int64_t n, int64_t k, int64_t group) {
  W4Shape s;
  if (shape_of("mvb_w4_bytes", n, k, group, s) != MVB_OK) return -1;
  return s.records * w4_record_bytes(static_cast<int>(group));
}

extern "C" int mvb_quantise_w4(void* records, const void* weight, int64_t weight_stride, int64_t n, int64_t k,
                               int64_t group, mvb_stream_t stream) {
  const char* name = "mvb_quantise_w4";
  W4Shape s;
  MVB_TRY(shape_of(name, n, k, group, s));
  if (n == 0) return MVB_OK;
  MVB_REQUIRE(records && weight, "%s: null pointer", name);
  MVB_REQUIRE(aligned(records, 16) && aligned(weight, 16) && weight_stride % 8 == 0 && (n == 1 || weight_stride >= k),
              "%s: records and rows of weight on 16 bytes, rows %lld apart", name, (long long)weight_stride);
  auto* r = static_cast<uint8_t*>(records);
  auto* w = static_cast<const __nv_bfloat16*>(weight);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (group == 32) return run_records(name, quantise_w4_kernel<32>, s, st, r, w, weight_stride);
  if (group == 64) return run_records(name, quantise_w4_kernel<64>, s, st, r, w, weight_stride);
  return run_records(name, quantise_w4_kernel<128>, s, st, r, w, weight_stride);
}

extern "C" int mvb_pack_w4(void* records, const uint8_t* codes, const void* scales, const uint8_t* zeros, int64_t n,
                           int64_t k, int64_t group, mvb_stream_t stream) {
  const char* name = "mvb_pack_w4";
  W4Shape s;
  MVB_TRY(shape_of(name, n, k, group, s));
  if (n == 0) return MVB_OK;
  MVB_REQUIRE(records && codes && scales, "%s: null pointer", name);
  MVB_REQUIRE(aligned(records, 16) && aligned(codes, 8), "%s: records on 16 and codes on 8 bytes", name);
  auto* r = static_cast<uint8_t*>(records);
  auto* sc = static_cast<const uint16_t*>(scales);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (group == 32) return run_records(name, pack_w4_kernel<32>, s, st, r, codes, sc, zeros);
  if (group == 64) return run_records(name, pack_w4_kernel<64>, s, st, r, codes, sc, zeros);
  return run_records(name, pack_w4_kernel<128>, s, st, r, codes, sc, zeros);
}

extern "C" int mvb_dequantise_w4(void* out, const void* records, int64_t n, int64_t k, int64_t group, int dtype,
                                 mvb_stream_t stream) {
  const char* name = "mvb_dequantise_w4";
  W4Shape s;
  MVB_TRY(shape_of(name, n, k, group, s));
  MVB_REQUIRE(dtype == MVB_BF16 || dtype == MVB_F32, "%s: dtype code %d", name, dtype);
  if (n == 0) return MVB_OK;
  MVB_REQUIRE(out && records, "%s: null pointer", name);
  MVB_REQUIRE(aligned(records, 16) && aligned(out, 16), "%s: records and out on 16 bytes", name);
  auto* r = static_cast<const uint8_t*>(records);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (group == 32) return run_dequantise<32>(name, out, r, s, dtype, st);
  if (group == 64) return run_dequantise<64>(name, out, r, s, dtype, st);
  return run_dequantise<128>(name, out, r, s, dtype, st);
}
