// 8-bit floating-point values with one scale per 128 values of a row (activations) or per 128 x 128 block (weights), and products of such matrices.
//
//   quantise   A = max(max |x|, 2^-96) over a block, scale = A / 448, q = e4m3(x * (448 / A)); scale, fraction and product are rounded to fp32 each
//   product    y[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k]
#pragma once

#include "common.cuh"

namespace mtx {

constexpr int kScaleBlock = 128;
constexpr uint32_t kLeastLargest = 0x0F800000u;  // 2^-96: a block of zeros has a scale like any other, and 448 / A stays finite

// |x| of finite values, infinities and NaN in the order of their bits: a maximum over them keeps a NaN, as the definition's does
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// two e4m3 bytes, `lo` in the low one; a product that its rounding put behind 448 becomes 448, NaN stays NaN
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// eight consecutive values of a row, as many as there are (the rest 0)
template <bool VEC>
__device__ __forceinline__ void load8(const bf16* p, int n, float (&v)[8]) {
  if (VEC && n >= 8) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.0f;
}
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int n, float (&v)[8]) {
  if (VEC && n >= 8) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
}

__device__ __forceinline__ void store8_e4m3(uint8_t* p, int n, const float (&v)[8], float by) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = e4m3_pair(v[2 * i] * by, v[2 * i + 1] * by);
  if (n >= 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = uint8_t(w[i / 2] >> (i % 2 * 8));
}

// ---- quantisation ----------------------------------------------------------------------------------------------------------------

constexpr int kQuantThreads = 256;

struct QuantParams {
  const void* x;
  long long ldx;
  int rows, k, blocks;  // blocks of 128 columns
  uint8_t* q;
  long long ldq;
  float* scale;         // [.., blocks]
  long long scale_row, scale_block;  // strides of a row (of a row of blocks) and of a block of columns
};

// 1 x 128: half a warp per block, eight values per thread.
template <class T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const QuantParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 15;
  const uint32_t block = blockIdx.x * (kQuantThreads / 16) + (threadIdx.x >> 4), all = uint32_t(p.rows) * uint32_t(p.blocks);
  const uint32_t row = block / uint32_t(p.blocks), b = block - row * uint32_t(p.blocks);
  const bool there = block < all;
  const int c = int(b) * kScaleBlock + lane * 8, n = there ? p.k - c : 0;
  float v[8];
  load8<VEC>(static_cast<const T*>(p.x) + (n > 0 ? row * p.ldx + c : 0), n, v);
  uint32_t top = kLeastLargest;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude_bits(v[i]));
#pragma unroll
  for (int i = 8; i > 0; i >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, i));
  if (n > 0) store8_e4m3(p.q + row * p.ldq + c, n, v, __fdiv_rn(448.0f, __uint_as_float(top)));
  if (lane == 0 && there) p.scale[row * p.scale_row + b * p.scale_block] = __fdiv_rn(__uint_as_float(top), 448.0f);
}

// 128 x 128: a CTA per block, eight rows of eight values per thread.
template <class T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_blocks_kernel(const QuantParams p) {
  __shared__ uint32_t part[kQuantThreads / 32];
  griddep_launch_dependents();
  griddep_wait();
  const int up = blockIdx.x / p.blocks, b = blockIdx.x - up * p.blocks;
  const int row0 = up * kScaleBlock + (threadIdx.x >> 4), c = b * kScaleBlock + (threadIdx.x & 15) * 8;
  float v[8][8];
  uint32_t top = kLeastLargest;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + 16 * i, n = row < p.rows ? p.k - c : 0;
    load8<VEC>(static_cast<const T*>(p.x) + (n > 0 ? row * p.ldx + c : 0), n, v[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(v[i][j]));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; ++i) top = max(top, part[i]);
  const float by = __fdiv_rn(448.0f, __uint_as_float(top));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + 16 * i, n = row < p.rows ? p.k - c : 0;
    if (n > 0) store8_e4m3(p.q + row * p.ldq + c, n, v[i], by);
  }
  if (threadIdx.x == 0) p.scale[up * p.scale_row + b * p.scale_block] = __fdiv_rn(__uint_as_float(top), 448.0f);
}

// ---- products ----------------------------------------------------------------------------------------------------------------------

struct Fp8LinearParams {
  const uint8_t* x;
  long long ldx;
  const float* x_scale;
  long long x_scale_row, x_scale_block;
  const uint8_t* w;
  long long ldw;
  const float* w_scale;  // [ceil(n / 128), blocks]
  void* out;
  long long ldo;
  int out_f32;
  int rows, n, k, blocks;
};

__device__ __forceinline__ float e4m3_value(uint8_t b) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)b));
  float f;
  asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"((unsigned short)(h & 0xffff)));
  return f;
}

// a CTA per 16 x 16 outputs
__global__ void __launch_bounds__(256) fp8_linear_kernel(const Fp8LinearParams p) {
  __shared__ float xs[16][kScaleBlock + 1], ws[16][kScaleBlock + 1];
  griddep_launch_dependents();
  griddep_wait();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const int m = m0 + ty, n = n0 + tx;
  float acc = 0.0f;
  for (int b = 0; b < p.blocks; ++b) {
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * kScaleBlock; i += 256) {
      const int r = i / kScaleBlock, c = i % kScaleBlock, k = b * kScaleBlock + c;
      xs[r][c] = m0 + r < p.rows && k < p.k ? e4m3_value(p.x[(m0 + r) * p.ldx + k]) : 0.0f;
      ws[r][c] = n0 + r < p.n && k < p.k ? e4m3_value(p.w[(n0 + r) * p.ldw + k]) : 0.0f;
    }
    __syncthreads();
    float part = 0.0f;
    for (int c = 0; c < kScaleBlock; ++c) part += xs[ty][c] * ws[tx][c];
    if (m < p.rows && n < p.n) acc += part * (p.x_scale[m * p.x_scale_row + b * p.x_scale_block] * p.w_scale[(n / kScaleBlock) * (long long)p.blocks + b]);
  }
  if (m < p.rows && n < p.n) {
    if (p.out_f32) static_cast<float*>(p.out)[m * p.ldo + n] = acc;
    else static_cast<bf16*>(p.out)[m * p.ldo + n] = __float2bfloat16_rn(acc);
  }
}

}  // namespace mtx
