// Residual sum, RMS norm and the next product's operand in one pass over a row.
//
//   h = x + residual, rounded to the residual's type       (kept as the new residual)
//   y = h (offset + weight) / sqrt(mean(h^2) + eps)
//   out = y, or blocks of 128 values as 8 bits: A = max(max |y|, 2^-96), scale = A / 448, e4m3(y (448 / A))
//
// A row lives in the registers of its threads, eight neighbouring values of every 8 T (T threads), so that the sixteen lanes of half a warp hold a block of 128.
// Bound: bytes, each value read and written once; where rows wait for SMs to 8 bits the instructions, some 170 for eight values.  4096 rows of 5376: to bf16 33.8 us (176 MB, 5.2 TB/s), to 8 bits
// 40.9 (155 MB, 3.8 TB/s).
//
// The mean, of 32-bit sums of eight squares (off by 5 * 2^-24 at most), the norm's factor and the scales' fractions are 64-bit, so that scales and 8-bit values are those of the definition with
// that mean; what 64 bits cost is spent once per row and block, by one warp.  Eight values are formed twice in 32 bits, by factors 2^-21 below and above theirs, which is more than 32 bits' three
// roundings: where both are the same 8-bit values so is the definition's, otherwise (of eight one in 10,000) they are formed again in 64.  Other results have two roundings in 32 bits and
// their type's own.  A row whose squares 32 bits do not hold is formed in 64 bits throughout.
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
  double by_width;  // 1 / width
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
};

// x + r as it is stored
template <class TX, class TR>
__device__ __forceinline__ float norm_sum(TX x, float r) {
  const float h = static_cast<float>(x) + r;
  return std::is_same<TR, bf16>::value ? bf16r(h) : h;
}

// whole 16 bytes
template <class T, int N>
__device__ __forceinline__ void norm_words(const T* from, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint4 u = reinterpret_cast<const uint4*>(from)[i];
    w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
  }
}

// offset + weight of a thread's eight values
template <bool VEC>
__device__ __forceinline__ void norm_weights(const AddNormParams& p, int c, float (&w)[8]) {
  const int n = p.width - c;
  if (p.weight == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.0f;
    return;
  }
  if (p.weight_f32) {
    const float* w0 = static_cast<const float*>(p.weight);
    uint32_t u[8] = {};
    if (!VEC) load_piece<float>(w0 + c, n, reinterpret_cast<uintptr_t>(w0), reinterpret_cast<uintptr_t>(w0 + p.width), u);
    else if (n > 0) norm_words(w0 + c, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = piece_value<float>(u, i);
  } else {
    const bf16* w0 = static_cast<const bf16*>(p.weight);
    uint32_t u[4] = {};
    if (!VEC) load_piece<bf16>(w0 + c, n, reinterpret_cast<uintptr_t>(w0), reinterpret_cast<uintptr_t>(w0 + p.width), u);
    else if (n > 0) norm_words(w0 + c, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = piece_value<bf16>(u, i);
  }
  if (p.weight_offset != 0.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] += p.weight_offset;
  }
}

// a product in 64 bits as the fp32 number that rounds to any shorter format as the product would: towards zero, and odd where something was cut
__device__ __forceinline__ float norm_odd(double v) {
  const float t = __double2float_rz(v);
  return double(t) == v || !(fabsf(t) < INFINITY) ? t : __uint_as_float(__float_as_uint(t) | 1u);
}

// h as it was stored, from memory (behind a barrier of the threads that store the row's sum)
template <class TX, class TR>
__device__ __forceinline__ float norm_value(const AddNormParams& p, int row, int c) {
  typedef AddNormRow<TX, TR> Row;
  typedef typename Row::TH TH;
  if (Row::kAdd && p.sum != nullptr) return static_cast<float>(static_cast<const TH*>(p.sum)[row * p.lds + c]);
  return norm_sum<TX, TR>(static_cast<const TX*>(p.x)[row * p.ldx + c], Row::kAdd ? static_cast<float>(static_cast<const TH*>(p.residual)[row * p.ldr + c]) : 0.0f);
}

__device__ __forceinline__ float norm_weight(const AddNormParams& p, int c) {
  return p.weight == nullptr ? 1.0f : (p.weight_f32 ? static_cast<const float*>(p.weight)[c] : static_cast<float>(static_cast<const bf16*>(p.weight)[c])) + p.weight_offset;
}

// NaN where one is
__device__ __forceinline__ double norm_larger(double a, double b) { return a != a || b <= a ? a : b; }

// A row whose squares 32 bits do not hold (values from some 2^60 on; mean and eps below 2^-100), or one with values that are no numbers: all of it in 64 bits and from memory, by the threads
// that have the row, every warp its own sum.  Not inlined: the registers of such a row are no other row's.
template <class TX, class TR, bool E4M3>
__device__ __noinline__ void norm_row_in_64_bits(const AddNormParams& p, int row) {
  const int lane = threadIdx.x & 31, threads = blockDim.x;
  double sum = 0.0;
  for (int c = lane; c < p.width; c += 32) {
    const double h = norm_value<TX, TR>(p, row, c);
    sum = fma(h, h, sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const double inv = rsqrt(sum * p.by_width + double(p.eps));
  if (threads > 32) __syncthreads();  // (results in an input's place)
  else __syncwarp();
  if (!E4M3) {
    for (int c = threadIdx.x; c < p.width; c += threads) {
      const double y = double(norm_value<TX, TR>(p, row, c)) * double(norm_weight(p, c)) * inv;
      if (p.out_type == MTX_F32) static_cast<float*>(p.out)[row * p.ldo + c] = float(y);
      else static_cast<bf16*>(p.out)[row * p.ldo + c] = __float2bfloat16_rn(norm_odd(y));
    }
    return;
  }
  for (int b = threadIdx.x >> 5; b < p.blocks; b += threads >> 5) {
    double y[4], largest = 0x1p-96;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = b * kScaleBlock + i * 32 + lane;
      y[i] = c < p.width ? double(norm_value<TX, TR>(p, row, c)) * double(norm_weight(p, c)) * inv : 0.0;
      largest = norm_larger(largest, fabs(y[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = norm_larger(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    const double by = 448.0 / largest;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = b * kScaleBlock + i * 32 + lane;
      if (c < p.width) static_cast<uint8_t*>(p.out)[row * p.ldo + c] = uint8_t(e4m3_pair(norm_odd(y[i] * double(float(by))), 0.0f));
    }
    if (lane == 0) p.scale[(long long)row * p.blocks + b] = float(largest * (1.0 / 448.0));
  }
}

// CTA = a row, or eight rows of a warp each.  VEC: all rows and the weights lie on 16 bytes and end with whole eight values.
template <class TX, class TR, bool E4M3, bool VEC, int J, int T>
__global__ void __launch_bounds__(T, J == 1 ? 1536 / T : J == 2 && T <= 768 ? 1536 / T : J == 3 ? 2 : 1) add_rmsnorm_kernel(const __grid_constant__ AddNormParams p) {
  typedef AddNormRow<TX, TR> Row;
  typedef typename Row::TH TH;
  __shared__ double part[32], inv_of_row;
  __shared__ float2 block_f[256];
  __shared__ float block_top[256], block_low[256], block_by[256];  // of a row; of the warps' rows four blocks each
  // (what comes next starts when this ends: with an early start 333 rows of 2560 took 3.6 us, not 3.1)
  griddep_wait();
  const int lane = threadIdx.x & 31, threads = blockDim.x;  // of a row; rows of a warp each lie along threadIdx.y
  const int row = blockIdx.x * blockDim.y + threadIdx.y, block0 = threadIdx.y * 4;
  const bool single = threads == 32;
  if (row >= p.rows) return;  // (whole warps; the CTA's threads wait for one another only where it has one row)
  const TX* x0 = static_cast<const TX*>(p.x);
  const TH* r0 = static_cast<const TH*>(p.residual);
  auto load = [&](auto* base, long long ld, int c, auto& w) {
    typedef typename std::remove_const<typename std::remove_pointer<decltype(base)>::type>::type V;
    if (VEC) {
#pragma unroll
      for (int i = 0; i < kPieceWords<V> / 4; ++i) {
        const uint4 u = c < p.width ? reinterpret_cast<const uint4*>(base + row * ld + c)[i] : make_uint4(0, 0, 0, 0);
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
      }
    } else {
      load_piece<V>(base + row * ld + c, p.width - c, reinterpret_cast<uintptr_t>(base), reinterpret_cast<uintptr_t>(base + (p.rows - 1) * ld + p.width), w);
    }
  };
  auto store = [&](auto* base, long long ld, int c, const auto& w) {
    typedef typename std::remove_pointer<decltype(base)>::type V;
    if (VEC) {
      if (c < p.width) {
#pragma unroll
        for (int i = 0; i < kPieceWords<V> / 4; ++i) reinterpret_cast<uint4*>(base + row * ld + c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
    } else {
      store_piece<V>(base + row * ld + c, p.width - c, w);
    }
  };
  uint32_t x[J][kPieceWords<TX>], r[J][kPieceWords<TH>];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (threadIdx.x + j * threads) * 8;
    load(x0, p.ldx, c, x[j]);
    if (Row::kAdd) load(r0, p.ldr, c, r[j]);
  }
  double sum = 0.0;
  float v[J][8];  // h times the weight
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (threadIdx.x + j * threads) * 8;
    float h[8], w[8], local[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = piece_value<TX>(x[j], i) + (Row::kAdd ? piece_value<TH>(r[j], i) : 0.0f);
    if (Row::kAdd) {
      pack_piece<TH>(h, r[j]);
      if (p.sum != nullptr) store(static_cast<TH*>(p.sum), p.lds, c, r[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = piece_value<TH>(r[j], i);
    }
    norm_weights<VEC>(p, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      local[i & 1] = fmaf(h[i], h[i], local[i & 1]);
      v[j][i] = h[i] * w[i];
    }
    sum += double(local[0] + local[1]);
    if (E4M3) {  // 16 lanes have a block: its largest product, and what that product's rounding took off
      float mine = 0.0f, low = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine = fmaxf(mine, fabsf(v[j][i]));
#pragma unroll
      for (int i = 0; i < 8; ++i) low = fmaxf(low, fmaf(fabsf(h[i]), fabsf(w[i]), -mine));  // (of products that were rounded to less it is less)
      float top = mine;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (mine != top) low = -INFINITY;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) low = fmaxf(low, __shfl_xor_sync(0xffffffffu, low, o));
      if ((lane & 15) == 0 && c < p.width) block_top[block0 + c / kScaleBlock] = top, block_low[block0 + c / kScaleBlock] = low;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  double inv;
  auto whole = [&]() {
    if (!single) {
      sum = lane < threads / 32 ? part[lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    return sum * p.by_width + double(p.eps);
  };
  if (!single) {
    if (lane == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
  } else {
    __syncwarp();
  }
  auto held = [](double mean) { return mean >= 0x1p-100 && mean < double(INFINITY); };  // by 32-bit squares
  if (!E4M3) {
    const double mean = whole();
    if (!held(mean)) {
      norm_row_in_64_bits<TX, TR, false>(p, row);
      return;
    }
    const float f = __frsqrt_rn(float(mean));
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = (threadIdx.x + j * threads) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] *= f;
      if (p.out_type == MTX_F32) {
        uint32_t o[8];
        pack_piece<float>(v[j], o);
        store(static_cast<float*>(p.out), p.ldo, c, o);
      } else {
        uint32_t o[4];
        pack_piece<bf16>(v[j], o);
        store(static_cast<bf16*>(p.out), p.ldo, c, o);
      }
    }
    return;
  }
  // one warp has the row's factor and the blocks' fractions, a lane a block
  if (threadIdx.x < 32) {
    const double mean = whole();
    inv = held(mean) ? rsqrt(mean) : -1.0;
    for (int b = lane; b < p.blocks; b += 32) {
      const float top = block_top[block0 + b], low = block_low[block0 + b];
      double largest = (double(top) + double(fabsf(low) < INFINITY ? low : 0.0f)) * inv;
      if (largest < 0x1p-96) largest = 0x1p-96;
      const double rough = double(__frcp_rn(float(largest))), off = fma(-largest, rough, 1.0), recip = fma(rough, fma(off, off, off), rough);
      const float by = float(448.0 * recip);
      block_by[block0 + b] = by;
      const float f = float(inv * double(by));
      block_f[block0 + b] = f < INFINITY ? make_float2(f * (1.0f - 0x1p-21f), f * (1.0f + 0x1p-21f)) : make_float2(0.0f, INFINITY);  // (no factor of 32 bits: no two values alike)
      p.scale[(long long)row * p.blocks + b] = float(largest * (1.0 / 448.0));
    }
    if (!single && lane == 0) inv_of_row = inv;
  }
  if (!single) __syncthreads();
  else __syncwarp();
  int again = 0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (threadIdx.x + j * threads) * 8, n = p.width - c;
    if (n <= 0) continue;
    const float2 f = block_f[block0 + c / kScaleBlock];
    uint32_t e[4], other = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = e4m3_pair(v[j][2 * i] * f.x, v[j][2 * i + 1] * f.x);
      other |= e[i] ^ e4m3_pair(v[j][2 * i] * f.y, v[j][2 * i + 1] * f.y);
    }
    if (other != 0) again |= 1 << j;
    uint8_t* to = static_cast<uint8_t*>(p.out) + row * p.ldo + c;
    if (VEC || n >= 8) {
      *reinterpret_cast<uint2*>(to) = make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) to[i] = uint8_t(e[i / 2] >> (i % 2 * 8));
    }
  }
  // values next to a border once more, with their neighbours and from memory (registers for this would be every row's)
  __syncwarp();  // (a sum may have been stored by the next lane)
  const double row_inv = single ? inv : inv_of_row;
  if (row_inv < 0.0) {  // (here nothing of the row is in registers; what is stored so far is stored again)
    norm_row_in_64_bits<TX, TR, true>(p, row);
    return;
  }
  if (again == 0) return;
#pragma unroll 1
  for (int j = 0; j < J; ++j) {
    if (!(again >> j & 1)) continue;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const int c = (threadIdx.x + j * threads) * 8 + i;
      if (c >= p.width) break;
      const float h = norm_value<TX, TR>(p, row, c), w = norm_weight(p, c);
      const int b = block0 + c / kScaleBlock;
      static_cast<uint8_t*>(p.out)[row * p.ldo + c] = uint8_t(e4m3_pair(norm_odd(double(h) * double(w) * (row_inv * double(block_by[b]))), 0.0f));
    }
  }
}

}  // namespace mtx
