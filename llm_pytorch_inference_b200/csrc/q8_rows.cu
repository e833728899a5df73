// Rows in 8 bits with one scale each, made where the values are made: RMSNorm (with the residual's addition), the
// gated activations, plain rows; and read back.
//
// A row y stands as codes q = rint(127 y / amax) in -127 .. 127 and the scale amax / 127, amax = max |y|.
//   plain     y = x
//   norm      y = h w r, r = 1 / sqrt(mean(h^2) + eps); h = x, or T(residual + x), which is written too
//   gated     y = act(gate) up
// all in 32 bits, without the roundings to T that the unquantised forms have in between.  In the norm r cancels out of
// 127 y / amax, so the codes are those of p = h w, and the mean goes into the scale alone: one pass, in which the sum
// of squares and the maximum are reduced together.  For bf16 p is exact in 32 bits, and so is 127 p: the codes
// are then the correctly rounded ones.
//
// Bound by memory for many rows (2 bytes in and 1 out an element, 4 and 3 with the addition, 4 and 1 gated), by the way
// through a row for few.  What an SM can do in that time is some 20 instructions an element, so pairs of 16-bit
// numbers are taken apart and made two at a time, and so are products and sums.
//
// Measured: addition and norm of 16384 x 4096 82 us (87 % of the rate of a copy), SwiGLU of 8192 x 14336 138
// (65 %); both issue in two thirds of the slots.  64 x 4096, norm and reading back, 3.8: two launches.
//
// A row with an infinity or a NaN (in y, before r) gets the scale NaN: it reads back as NaN, and so does a product with it.
// A row of zeros gets the scale 0.
#include <climits>

#include "common.cuh"
#include "host.h"

namespace mvb {
namespace {

enum Kind { kPlain, kNorm, kAddNorm, kSilu, kGelu };

struct RowArgs {
  int8_t* q;        // [rows, width]
  float* scale;     // [rows]
  const void* a;    // x; the residual; gate
  int64_t a_stride;
  const void* b;    // x of the addition; up
  int64_t b_stride;
  void* sum;        // residual + x
  int64_t sum_stride;
  const void* w;
  int64_t rows;
  int width;
  float eps;
  float one;        // 1 for the (1 + w) norm, else 0
};

// The activations by the logistic function: silu(g) = g / (1 + e^-z) with z = g, and gelu's 0.5 g (1 + tanh(z / 2)) the same
// with its z.  With e = e^-|z| it is g / (1 + e) or g e / (1 + e), so that nothing leaves fp32's range before the result
// does.  The quotient and the exponential are the hardware's: (6 + 1.2 |z|) 2^-24 relative, for gelu 3 |z| 2^-24 more by
// the rounding of z; half a code is 4e-3 of the row's largest.
template <int KIND>
__device__ __forceinline__ float act_of(float g) {
  const float z = KIND == kSilu ? g : 1.5957691216057308f * g * fmaf(0.044715f * g, g, 1.0f);  // 2 sqrt(2 / pi)
  const float e = __expf(-fabsf(z));
  return __fdividef(z < 0.0f ? g * e : g, 1.0f + e);
}

template <int KIND, typename T>
__device__ __forceinline__ float value_of(float a, float b, float w, float one, float& h, float& ss) {
  if (KIND == kNorm || KIND == kAddNorm) {
    h = KIND == kAddNorm ? rnd<T>(a + b) : a;
    ss = fmaf(h, h, ss);
    return h * (w + one);
  }
  if (KIND == kSilu || KIND == kGelu) return act_of<KIND>(a) * b;
  return a;
}

// The codes of one row, eight at a time, each in the low byte of its result.  The product with 127 / amax is off by less
// than 2e-5 of a code.  Where one of the eight comes so near a border between two (or lies on it, which 8-bit numbers
// often do), 127 y - code amax, exact in one multiply-add for bf16, tells on which side each is.  In rows below 2^-80 or
// above 2^100, where 127 / amax or 127 y would leave fp32's range, the quotients are worked out, from numbers taken
// times a power of two.
struct Coder {
  float amax, inv;
  bool edge;
  __device__ __forceinline__ explicit Coder(float top) : amax(top), edge(top > 1.2676506e30f || top < 8.2718061e-25f) {
    inv = edge ? 0.0f : 127.0f / top;
  }
  // not inlined: it is hardly ever called
  static __device__ __noinline__ uint32_t quotient(float y, float amax, bool edge) {
    const float f = !edge ? 1.0f : amax > 1.0f ? 5.4210109e-20f : 1.8446744e19f;  // 2^-64, 2^64
    return __float_as_uint(amax > 0.0f ? __fdiv_rn(127.0f * (y * f), amax * f) + 12582912.0f : 0.0f);
  }
  __device__ __forceinline__ void of(const float (&y)[8], uint32_t (&c)[8]) const {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are the nearest whole number
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 t = __fmul2_rn(make_float2(y[i], y[i + 1]), make_float2(inv, inv));
      const float2 m = __fadd2_rn(t, make_float2(kMagic, kMagic));
      const float2 n = __fadd2_rn(m, make_float2(-kMagic, -kMagic));
      const float2 d = __ffma2_rn(n, make_float2(-1.0f, -1.0f), t);
      far = fmaxf(fmaxf(far, fabsf(d.x)), fabsf(d.y));
      c[i] = __float_as_uint(m.x);
      c[i + 1] = __float_as_uint(m.y);
    }
    if (far > 0.49998f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float left = fmaf(kMagic - __uint_as_float(c[i]), amax, 127.0f * y[i]), twice = 2.0f * fabsf(left);
        if (twice > amax || (twice == amax && (c[i] & 1u))) c[i] += left > 0.0f ? 1u : ~0u;
      }
    }
    if (edge) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = quotient(y[i], amax, true);
    }
  }
};
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

__device__ __forceinline__ float abs_max(float m, float y) {  // the larger size; NaN where either is
  float d;
  asm("{\n\t.reg .f32 a;\n\tabs.f32 a, %2;\n\tmax.NaN.f32 %0, %1, a;\n\t}" : "=f"(d) : "f"(m), "f"(y));
  return d;
}
__device__ __forceinline__ bool is_fine(float top) { return top <= 3.4028235e38f; }  // neither infinite nor NaN

// The row's sum and its largest size, in every thread of its blockDim.x.
__device__ __forceinline__ void row_both(float& ss, float& top, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    top = abs_max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return;
  if (lane == 0) red[threadIdx.x >> 5] = make_float2(ss, top);
  __syncthreads();
  const float2 v = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);
  ss = v.x;
  top = v.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    top = abs_max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
}

template <int KIND>
__device__ __forceinline__ float row_scale(const RowArgs& a, float ss, float top) {
  if (!is_fine(top)) return __uint_as_float(0x7fc00000u);
  if (KIND == kNorm || KIND == kAddNorm) return top * (1.0f / sqrtf(ss / static_cast<float>(a.width) + a.eps)) / 127.0f;
  return top / 127.0f;
}

// Eight elements, taken apart and rounded in pairs.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
  v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
}
__device__ __forceinline__ void apart(const uint4& x, float (&v)[8], __nv_bfloat16) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void apart(const uint4& x, float (&v)[8], __half) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  apart(*reinterpret_cast<const uint4*>(p), v, T());
}
__device__ __forceinline__ uint32_t round2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t round2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Stores v rounded to T, and leaves in v what was stored.
__device__ __forceinline__ void store8(float* p, float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, float (&v)[8]) {
  const uint4 x = make_uint4(round2(v[0], v[1], T()), round2(v[2], v[3], T()), round2(v[4], v[5], T()), round2(v[6], v[7], T()));
  *reinterpret_cast<uint4*>(p) = x;
  apart(x, v, T());
}

// A row stays in registers: vector j of a thread holds elements 8 (j blockDim.x + thread) .. + 7.  A block has one row,
// or (32 threads a row) several.  Four vectors a thread with 40 registers: more rows in an SM are worth a few spills
// (SwiGLU of 8192 x 14336: 156 us with 56 registers, 138 with 40).
template <int KIND, typename T, int VPT>
__global__ void __maxnreg__(VPT == 4 ? 40 : 64) q8_rows_kernel(const RowArgs a) {
  constexpr bool NORM = KIND == kNorm || KIND == kAddNorm;
  __shared__ float2 red[32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;  // a warp has a row, or the block one
  const T* pa = static_cast<const T*>(a.a) + row * a.a_stride;
  const T* pb = static_cast<const T*>(a.b) + row * a.b_stride;
  const int vectors = a.width >> 3;
  float y[VPT][8];
  float2 squares = make_float2(0.0f, 0.0f);
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int v = j * blockDim.x + threadIdx.x;
    if (v < vectors) {
      float x[8], z[8], w[8];
      load8(pa + 8 * v, x);
      if (KIND >= kAddNorm) load8(pb + 8 * v, z);
      if (NORM) load8(static_cast<const T*>(a.w) + 8 * v, w);
      if (KIND == kAddNorm) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 h = __fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(z[i], z[i + 1]));
          x[i] = h.x, x[i + 1] = h.y;
        }
        store8(static_cast<T*>(a.sum) + row * a.sum_stride + 8 * v, x);
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float2 u = make_float2(x[i], x[i + 1]);
        if (NORM) {
          squares = __ffma2_rn(u, u, squares);
          u = __fmul2_rn(u, __fadd2_rn(make_float2(w[i], w[i + 1]), make_float2(a.one, a.one)));
        }
        if (KIND == kSilu || KIND == kGelu)
          u = __fmul2_rn(make_float2(act_of<KIND>(u.x), act_of<KIND>(u.y)), make_float2(z[i], z[i + 1]));
        top = abs_max(abs_max(top, u.x), u.y);
        y[j][i] = u.x, y[j][i + 1] = u.y;
      }
    }
  }
  float ss = squares.x + squares.y;
  row_both(ss, top, red);
  const float scale = row_scale<KIND>(a, ss, top);
  if (threadIdx.x == 0) a.scale[row] = scale;
  const bool fine = is_fine(top);
  const Coder code(top);
  uint2* q = reinterpret_cast<uint2*>(a.q + row * a.width);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int v = j * blockDim.x + threadIdx.x;
    if (v < vectors) {
      uint32_t c[8];
      code.of(y[j], c);
      uint2 bytes = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
      if (!fine) bytes = make_uint2(0, 0);
      q[v] = bytes;
    }
  }
}

// Any width and alignment: as above with single elements, j blockDim.x + thread, EPT of them a thread.  2.0 TB/s of bf16 at
// best, by instructions an element: norm of 16001 x 3583 with its addition 193 us, SwiGLU 140.  8 elements a thread where 1024
// threads hold a row so, since blocks of fewer threads do not hide what loads take (16: 268 and 272 us).
template <int KIND, typename T, int EPT>
__global__ void __launch_bounds__(1024, 1) q8_ragged_kernel(const RowArgs a) {
  __shared__ float2 red[32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const T* pa = static_cast<const T*>(a.a) + row * a.a_stride;
  const T* pb = static_cast<const T*>(a.b) + row * a.b_stride;
  const T* pw = static_cast<const T*>(a.w);
  T* sum = static_cast<T*>(a.sum) + row * a.sum_stride;
  constexpr bool NORM = KIND == kNorm || KIND == kAddNorm;
  float y[EPT], ss = 0.0f, top = 0.0f, h = 0.0f;
  T u[EPT], v[EPT];  // everything is asked for before anything is used
#pragma unroll
  for (int j = 0; j < EPT; ++j) {
    const int i = j * blockDim.x + threadIdx.x;
    u[j] = i < a.width ? pa[i] : from_f<T>(0.0f);
    if (KIND >= kAddNorm) v[j] = i < a.width ? pb[i] : from_f<T>(0.0f);
  }
#pragma unroll
  for (int j = 0; j < EPT; ++j) {
    y[j] = to_f<T>(u[j]);
    if (KIND == kAddNorm) y[j] = rnd<T>(y[j] + to_f<T>(v[j]));
    if (KIND > kAddNorm) y[j] = value_of<KIND, T>(y[j], to_f<T>(v[j]), 0.0f, a.one, h, ss);
  }
  if (NORM) {  // sums are stored when all is read: no load then waits behind a store
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
      const int i = j * blockDim.x + threadIdx.x;
      if (i < a.width) {
        if (KIND == kAddNorm) sum[i] = from_f<T>(y[j]);
        ss = fmaf(y[j], y[j], ss);
        y[j] *= to_f<T>(__ldg(pw + i)) + a.one;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < EPT; ++j) top = abs_max(top, y[j]);
  row_both(ss, top, red);
  if (threadIdx.x == 0) a.scale[row] = row_scale<KIND>(a, ss, top);
  const bool fine = is_fine(top);
  const Coder code(top);
  int8_t* q = a.q + row * a.width;
#pragma unroll
  for (int j0 = 0; j0 < EPT; j0 += 8) {
    float eight[8];
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) eight[j] = y[j0 + j];
    code.of(eight, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = (j0 + j) * blockDim.x + threadIdx.x;
      if (i < a.width) q[i] = static_cast<int8_t>(fine ? c[j] & 0xffu : 0u);
    }
  }
}

// Rows that no block's registers hold: element by element, worked out again for the codes.
template <int KIND, typename T>
__global__ void __launch_bounds__(1024) q8_any_kernel(const RowArgs a) {
  __shared__ float2 red[32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const T* pa = static_cast<const T*>(a.a) + row * a.a_stride;
  const T* pb = static_cast<const T*>(a.b) + row * a.b_stride;
  const T* pw = static_cast<const T*>(a.w);
  T* sum = static_cast<T*>(a.sum) + row * a.sum_stride;
  float ss = 0.0f, top = 0.0f, h = 0.0f;
  for (int i = threadIdx.x; i < a.width; i += blockDim.x) {
    const float w = KIND == kNorm || KIND == kAddNorm ? to_f<T>(pw[i]) : 0.0f;
    const float y = value_of<KIND, T>(to_f<T>(pa[i]), KIND >= kAddNorm ? to_f<T>(pb[i]) : 0.0f, w, a.one, h, ss);
    if (KIND == kAddNorm) sum[i] = from_f<T>(h);
    top = abs_max(top, y);
  }
  row_both(ss, top, red);
  if (threadIdx.x == 0) a.scale[row] = row_scale<KIND>(a, ss, top);
  const bool fine = is_fine(top);
  const Coder code(top);
  for (int i = threadIdx.x; i < a.width; i += blockDim.x) {
    float y;
    if (KIND == kAddNorm)
      y = to_f<T>(sum[i]) * (to_f<T>(pw[i]) + a.one);  // what this thread has written: the residual may be gone
    else
      y = value_of<KIND, T>(to_f<T>(pa[i]), KIND >= kAddNorm ? to_f<T>(pb[i]) : 0.0f,
                            KIND == kNorm ? to_f<T>(pw[i]) : 0.0f, a.one, h, ss);
    a.q[row * a.width + i] = fine ? static_cast<int8_t>(Coder::quotient(y, code.amax, code.edge) & 0xffu) : int8_t(0);
  }
}

// Codes times scales: 8 codes a thread and step, four steps under way; `per` of them make a row.
template <typename T>
__global__ void __launch_bounds__(256) dequantise_q8_kernel(T* __restrict__ out, const int8_t* __restrict__ q,
                                                            int64_t q_stride, const float* __restrict__ scale,
                                                            int64_t rows, int width) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int N = 8, STEPS = 4;
  const uint32_t per = width / N;
  const int64_t n = rows * per, all = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i0 < n; i0 += STEPS * all) {
    int64_t row[STEPS];
    int col[STEPS];
    float s[STEPS];
    uint2 c[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int64_t i = i0 + j * all;
      if (i >= n) continue;
      // whole numbers of 32 bits divide at a third of the cost of 64
      row[j] = i < (int64_t{1} << 32) ? static_cast<uint32_t>(i) / per : i / per;
      col[j] = static_cast<int>(i - row[j] * per) * N;
      s[j] = scale[row[j]];
      c[j] = *reinterpret_cast<const uint2*>(q + row[j] * q_stride + col[j]);
    }
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      if (i0 + j * all >= n) continue;
      const int8_t* e = reinterpret_cast<const int8_t*>(&c[j]);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = static_cast<float>(e[k]) * s[j];
      store8(out + row[j] * width + col[j], v);
    }
  }
}

// Any width and alignment: a block has kRagged elements of a row.
constexpr int kRagged = 2048;
template <typename T>
__global__ void __launch_bounds__(256) dequantise_q8_ragged_kernel(T* __restrict__ out, const int8_t* __restrict__ q,
                                                                   int64_t q_stride, const float* __restrict__ scale,
                                                                   int width) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int first = blockIdx.y * kRagged + threadIdx.x;
  const float s = scale[row];
  int8_t c[kRagged / 256];
#pragma unroll
  for (int j = 0; j < kRagged / 256; ++j) {
    const int i = first + 256 * j;
    c[j] = i < width ? q[row * q_stride + i] : int8_t(0);
  }
#pragma unroll
  for (int j = 0; j < kRagged / 256; ++j) {
    const int i = first + 256 * j;
    if (i < width) out[row * width + i] = from_f<T>(static_cast<float>(c[j]) * s);
  }
}

template <int KIND, typename T>
int run_rows(const char* name, const RowArgs& a, int64_t rows, cudaStream_t stream) {
  const size_t e = sizeof(T);
  auto whole = [&](const void* p, int64_t stride) { return aligned(p, 16) && stride * e % 16 == 0; };
  const bool vec = a.width % 8 == 0 && aligned(a.q, 8) && whole(a.a, a.a_stride) && whole(a.w, 0) &&
                   (KIND < kAddNorm || whole(a.b, a.b_stride)) && (KIND != kAddNorm || whole(a.sum, a.sum_stride));
  const int vectors = a.width / 8;
  if (a.width > 32 * 1024)
    return launch(name, q8_any_kernel<KIND, T>, dim3(static_cast<unsigned>(rows)), dim3(1024), 0, stream, a);
  if (!vec) {
    // The fewest elements a thread (8, 16 or 32) with which 1024 threads hold a row, whatever the number of rows.
    const int ept = a.width > 16 * 1024 ? 32 : a.width > 8 * 1024 ? 16 : 8;
    const dim3 grid(static_cast<unsigned>(rows)), block(static_cast<unsigned>(((a.width + ept - 1) / ept + 31) / 32 * 32));
    if (ept == 8) return launch(name, q8_ragged_kernel<KIND, T, 8>, grid, block, 0, stream, a);
    if (ept == 16) return launch(name, q8_ragged_kernel<KIND, T, 16>, grid, block, 0, stream, a);
    return launch(name, q8_ragged_kernel<KIND, T, 32>, grid, block, 0, stream, a);
  }
  // Few rows: a vector a thread, the shortest way through a row.  Many: four, and rows of up to 1024 elements a warp each.
  const int most = rows <= 2 * current_sm_count() ? 1 : 4;
  int threads = (vectors + most - 1) / most;
  threads = threads > 1024 ? 1024 : (threads + 31) / 32 * 32;
  const int per = (vectors + threads - 1) / threads, together = threads == 32 ? 8 : 1;
  const dim3 block(static_cast<unsigned>(threads), static_cast<unsigned>(together));
  const dim3 grid(static_cast<unsigned>((rows + together - 1) / together));
  if (per <= 1) return launch(name, q8_rows_kernel<KIND, T, 1>, grid, block, 0, stream, a);
  if (per <= 2) return launch(name, q8_rows_kernel<KIND, T, 2>, grid, block, 0, stream, a);
  return launch(name, q8_rows_kernel<KIND, T, 4>, grid, block, 0, stream, a);
}

template <int KIND>
int run_kind(const char* name, const RowArgs& a, int64_t rows, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case MVB_F32: return run_rows<KIND, float>(name, a, rows, stream);
    case MVB_F16: return run_rows<KIND, __half>(name, a, rows, stream);
    case MVB_BF16: return run_rows<KIND, __nv_bfloat16>(name, a, rows, stream);
  }
  return fail(MVB_ERR_INVALID_ARG, "%s: dtype code %d", name, dtype);
}

int check_rows(const char* name, int64_t rows, int64_t width, int dtype) {
  MVB_REQUIRE(rows >= 0 && rows <= INT_MAX, "%s: %lld rows", name, (long long)rows);
  MVB_REQUIRE(width > 0 && width <= (1 << 24), "%s: rows of %lld elements", name, (long long)width);
  MVB_REQUIRE(dtype == MVB_F32 || dtype == MVB_F16 || dtype == MVB_BF16, "%s: dtype code %d", name, dtype);
  return MVB_OK;
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_quantise_q8(int8_t* values, float* scales, const void* in, int64_t in_stride, int64_t rows,
                               int64_t width, int dtype, mvb_stream_t stream) {
  const char* name = "mvb_quantise_q8";
  MVB_TRY(check_rows(name, rows, width, dtype));
  if (rows == 0) return MVB_OK;
  MVB_REQUIRE(values && scales && in, "%s: null pointer", name);
  MVB_REQUIRE(rows == 1 || in_stride >= width, "%s: rows %lld apart", name, (long long)in_stride);
  RowArgs a = {};
  a.rows = rows;
  a.q = values, a.scale = scales, a.a = in, a.a_stride = in_stride, a.width = static_cast<int>(width);
  return run_kind<kPlain>(name, a, rows, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int mvb_rmsnorm_q8(int8_t* values, float* scales, const void* in, int64_t in_stride, const void* weight,
                              int64_t rows, int64_t hidden, float eps, int plus_one, int dtype, mvb_stream_t stream) {
  const char* name = "mvb_rmsnorm_q8";
  MVB_TRY(check_rows(name, rows, hidden, dtype));
  if (rows == 0) return MVB_OK;
  MVB_REQUIRE(values && scales && in && weight, "%s: null pointer", name);
  MVB_REQUIRE(rows == 1 || in_stride >= hidden, "%s: rows %lld apart", name, (long long)in_stride);
  RowArgs a = {};
  a.rows = rows;
  a.q = values, a.scale = scales, a.a = in, a.a_stride = in_stride, a.w = weight;
  a.width = static_cast<int>(hidden), a.eps = eps, a.one = plus_one ? 1.0f : 0.0f;
  return run_kind<kNorm>(name, a, rows, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int mvb_fused_add_rmsnorm_q8(int8_t* values, float* scales, void* residual_out, int64_t out_stride,
                                        const void* residual, int64_t residual_stride, const void* in,
                                        int64_t in_stride, const void* weight, int64_t rows, int64_t hidden, float eps,
                                        int plus_one, int dtype, mvb_stream_t stream) {
  const char* name = "mvb_fused_add_rmsnorm_q8";
  MVB_TRY(check_rows(name, rows, hidden, dtype));
  if (rows == 0) return MVB_OK;
  MVB_REQUIRE(values && scales && residual_out && residual && in && weight, "%s: null pointer", name);
  MVB_REQUIRE(rows == 1 || (in_stride >= hidden && residual_stride >= hidden && out_stride >= hidden),
              "%s: rows %lld, %lld and %lld apart", name, (long long)in_stride, (long long)residual_stride,
              (long long)out_stride);
  RowArgs a = {};
  a.rows = rows;
  a.q = values, a.scale = scales, a.a = residual, a.a_stride = residual_stride, a.b = in, a.b_stride = in_stride;
  a.sum = residual_out, a.sum_stride = out_stride, a.w = weight;
  a.width = static_cast<int>(hidden), a.eps = eps, a.one = plus_one ? 1.0f : 0.0f;
  return run_kind<kAddNorm>(name, a, rows, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int mvb_gated_q8(int8_t* values, float* scales, const void* gate, int64_t gate_stride, const void* up,
                            int64_t up_stride, int64_t rows, int64_t width, int act, int dtype, mvb_stream_t stream) {
  const char* name = "mvb_gated_q8";
  MVB_TRY(check_rows(name, rows, width, dtype));
  MVB_REQUIRE(act == MVB_ACT_SILU || act == MVB_ACT_GELU_TANH, "%s: activation %d", name, act);
  if (rows == 0) return MVB_OK;
  MVB_REQUIRE(values && scales && gate && up, "%s: null pointer", name);
  MVB_REQUIRE(rows == 1 || (gate_stride >= width && up_stride >= width), "%s: rows %lld and %lld apart", name,
              (long long)gate_stride, (long long)up_stride);
  RowArgs a = {};
  a.rows = rows;
  a.q = values, a.scale = scales, a.a = gate, a.a_stride = gate_stride, a.b = up, a.b_stride = up_stride;
  a.width = static_cast<int>(width);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return act == MVB_ACT_SILU ? run_kind<kSilu>(name, a, rows, dtype, st) : run_kind<kGelu>(name, a, rows, dtype, st);
}

extern "C" int mvb_dequantise_q8(void* out, const int8_t* values, int64_t values_stride, const float* scales,
                                 int64_t rows, int64_t width, int dtype, mvb_stream_t stream) {
  const char* name = "mvb_dequantise_q8";
  MVB_TRY(check_rows(name, rows, width, dtype));
  if (rows == 0) return MVB_OK;
  MVB_REQUIRE(out && values && scales, "%s: null pointer", name);
  MVB_REQUIRE(rows == 1 || values_stride >= width, "%s: rows %lld apart", name, (long long)values_stride);
  const bool vec = width % 8 == 0 && aligned(values, 8) && values_stride % 8 == 0 && aligned(out, 16);
  const int64_t sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "%s: no device", name);
  const int64_t blocks = (rows * (width / 8) + 255) / 256;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int w = static_cast<int>(width);
  auto run = [&](auto* o) {
    using T = std::remove_pointer_t<decltype(o)>;
    if (vec)
      return launch(name, dequantise_q8_kernel<T>, dim3(static_cast<unsigned>(blocks < 8 * sms ? blocks : 8 * sms)), dim3(256),
                    0, st, o, values, values_stride, scales, rows, w);
    const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>((w + kRagged - 1) / kRagged));
    return launch(name, dequantise_q8_ragged_kernel<T>, grid, dim3(256), 0, st, o, values, values_stride, scales, w);
  };
  if (dtype == MVB_F32) return run(static_cast<float*>(out));
  if (dtype == MVB_F16) return run(static_cast<__half*>(out));
  return run(static_cast<__nv_bfloat16*>(out));
}
