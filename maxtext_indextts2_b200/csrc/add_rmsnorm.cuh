// Residual sum, RMS norm and the next product's operand in one pass over a row.
//
//   h = x + residual, rounded to the residual's type       (kept as the new residual)
//   y = h (offset + weight) / sqrt(mean(h^2) + eps)
//   out = y, or blocks of 128 values as 8 bits: A = max(max |y|, 2^-96), scale = A / 448, e4m3(y (448 / A))
//
// A row lives in the registers of its threads, eight neighbouring values of every 8 T (T threads), so that the sixteen lanes of half a warp hold a block of 128.
#pragma once

#include "fp8_linear.cuh"
#include "row_pieces.cuh"

namespace mtx {

struct AddNormParams {
  const void* x;
  long long ldx;
  const void* residual;
  long long ldr;
  void* sum;
  long long lds;
  const void* weight;
  int weight_f32;
  float weight_offset, eps;
  void* out;
  int out_type;  // MTX_BF16, MTX_F32 or MTX_E4M3
  long long ldo;
  float* scale;  // [rows, blocks]
  int rows, width, blocks;
};

constexpr int kNormWarpRows = 8;  // rows of a CTA whose rows have a warp each

struct NoResidual {};

template <class TX, class TR>
struct AddNormRow {
  typedef typename std::conditional<std::is_same<TR, NoResidual>::value, TX, TR>::type TH;  // h's type
  static constexpr bool kAdd = !std::is_same<TR, NoResidual>::value;

  const TX* x;
  const TH* r;
  TH* s;
  uintptr_t xb, xe, rb, re;

  __device__ __forceinline__ AddNormRow(const AddNormParams& p, int row) {
    const TX* x0 = static_cast<const TX*>(p.x);
    x = x0 + row * p.ldx;
    xb = reinterpret_cast<uintptr_t>(x0), xe = reinterpret_cast<uintptr_t>(x0 + (p.rows - 1) * p.ldx + p.width);
    if (kAdd) {
      const TH* r0 = static_cast<const TH*>(p.residual);
      r = r0 + row * p.ldr;
      rb = reinterpret_cast<uintptr_t>(r0), re = reinterpret_cast<uintptr_t>(r0 + (p.rows - 1) * p.ldr + p.width);
      s = p.sum != nullptr ? static_cast<TH*>(p.sum) + row * p.lds : nullptr;
    }
  }
};

template <class TX, class TR, int J>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const AddNormParams p) {
  typedef AddNormRow<TX, TR> Row;
  typedef typename Row::TH TH;
  __shared__ float part[32];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, threads = blockDim.x;  // of a row; rows of a warp each lie along threadIdx.y
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;  // (whole warps; the block waits for one another only where it has one row)
  const Row at(p, row);
  uint32_t rx[J][kPieceWords<TX>], rr[J][kPieceWords<TH>];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (threadIdx.x + j * threads) * 8;
    load_piece<TX>(at.x + c, p.width - c, at.xb, at.xe, rx[j]);
    if (Row::kAdd) load_piece<TH>(at.r + c, p.width - c, at.rb, at.re, rr[j]);
  }
  float h[J][8], sum = 0.0f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (threadIdx.x + j * threads) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[j][i] = piece_value<TX>(rx[j], i) + (Row::kAdd ? piece_value<TH>(rr[j], i) : 0.0f);
    if (Row::kAdd) {
      pack_piece<TH>(h[j], rr[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] = piece_value<TH>(rr[j], i);
      if (at.s != nullptr) store_piece<TH>(at.s + c, p.width - c, rr[j]);
    }
    float local = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) local = fmaf(h[j][i], h[j][i], local);
    sum += local;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threads > 32) {
    if (lane == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = lane < threads / 32 ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  const float inv = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum, float(p.width)), p.eps));
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (threadIdx.x + j * threads) * 8, n = p.width - c;
    if (p.weight != nullptr) {
      float w[8];
      if (p.weight_f32) {
        const float* w0 = static_cast<const float*>(p.weight);
        uint32_t u[8];
        load_piece<float>(w0 + c, n, reinterpret_cast<uintptr_t>(w0), reinterpret_cast<uintptr_t>(w0 + p.width), u);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = piece_value<float>(u, i);
      } else {
        const bf16* w0 = static_cast<const bf16*>(p.weight);
        uint32_t u[4];
        load_piece<bf16>(w0 + c, n, reinterpret_cast<uintptr_t>(w0), reinterpret_cast<uintptr_t>(w0 + p.width), u);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = piece_value<bf16>(u, i);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] *= p.weight_offset + w[i];
    }
    if (p.out_type == MTX_E4M3) {
      // the block's largest |y| by its bits, so that a NaN stays
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) top = max(top, __float_as_uint(h[j][i] * inv) & 0x7fffffffu);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float largest = __uint_as_float(max(top, kLeastLargest)), up = __fdiv_rn(448.0f, largest);
      const bool apart = !(inv * up < INFINITY);                          // (rows next to zero with an eps next to it)
      const float by = apart ? up : inv * up, first = apart ? inv : 1.0f;  // one factor for both steps: one rounding less per value
      if (n > 0) {
        if ((lane & 15) == 0) p.scale[(long long)row * p.blocks + c / kScaleBlock] = __fdiv_rn(largest, 448.0f);
        uint32_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = e4m3_pair(h[j][2 * i] * first * by, h[j][2 * i + 1] * first * by);
        uint8_t* to = static_cast<uint8_t*>(p.out) + row * p.ldo + c;
        if (n >= 8) {
          *reinterpret_cast<uint2*>(to) = make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < n) to[i] = uint8_t(e[i / 2] >> (i % 2 * 8));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] *= inv;
      if (p.out_type == MTX_F32) {
        uint32_t w[8];
        pack_piece<float>(h[j], w);
        store_piece<float>(static_cast<float*>(p.out) + row * p.ldo + c, n, w);
      } else {
        uint32_t w[4];
        pack_piece<bf16>(h[j], w);
        store_piece<bf16>(static_cast<bf16*>(p.out) + row * p.ldo + c, n, w);
      }
    }
  }
}

}  // namespace mtx
