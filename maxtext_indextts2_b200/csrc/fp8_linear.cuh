// 8-bit floating-point values with one scale per 128 values of a row (activations) or per 128 x 128 block (weights), and products of such matrices.
//
//   quantise   A = max(max |x|, 2^-96) over a block, scale = A / 448, q = e4m3(x * (448 / A)); scale, fraction and product are rounded to fp32 each
//   product    y[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k]
#pragma once

#include "gemm_wide.cuh"

namespace mtx {

constexpr int kScaleBlock = 128;
constexpr uint32_t kLeastLargest = 0x0F800000u;  // 2^-96: a block of zeros has a scale like any other, and 448 / A stays finite

// two e4m3 bytes, `lo` in the low one; a product that its rounding put behind 448 becomes 448, NaN stays NaN
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight consecutive values of a row as they lie in memory: the registers of the values that a thread holds until it knows their scale.
template <class T>
struct Raw8 {
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t w[kWords];

  // the values from n on become 0
  __device__ __forceinline__ void cut(int n) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if (sizeof(T) == 4) w[i] = i < n ? w[i] : 0u;
      else w[i] &= (2 * i < n ? 0xffffu : 0u) | (2 * i + 1 < n ? 0xffff0000u : 0u);
    }
  }
  // the bits of the largest magnitude as fp32: those of finite values, infinities and NaN have the order of their bits, so that a NaN stays (as the definition's does)
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t top = 0;
    if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) top = max(top, w[i] & 0x7fffffffu);
      return top;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
    return max(top & 0xffff0000u, top << 16);
  }
  // the words, and behind them the first M of the next lane's; for the last of 16 lanes those of `far` in lane i
  template <int M>
  __device__ __forceinline__ void with_next(uint32_t (&out)[kWords + 4], const uint32_t (&far)[4], int i, uint32_t lanes) const {
#pragma unroll
    for (int j = 0; j < kWords; ++j) out[j] = w[j];
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const uint32_t next = __shfl_down_sync(lanes, w[j], 1, 16), last = __shfl_sync(lanes, far[j], i, 16);
      out[kWords + j] = (threadIdx.x & 15) == 15 ? last : next;
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if (sizeof(T) == 4) return __uint_as_float(w[i % kWords]);
    return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
  }
  __device__ __forceinline__ void store_e4m3(uint8_t* p, int n, float by) const {
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = e4m3_pair(value(2 * i) * by, value(2 * i + 1) * by);
    if (n >= 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = uint8_t(e[i / 2] >> (i % 2 * 8));
  }
};

struct QuantParams {
  const void* x;
  long long ldx;
  int rows, k, blocks;  // blocks of 128 columns
  uint8_t* q;
  long long ldq;
  float* scale;         // [.., blocks]
  long long scale_row, scale_block;  // strides of a row (of a row of blocks) and of a block of columns
};

// N times eight values per thread, 16 lanes side by side: the i-th are the values from `from` + i * step on, of which left(i) are there (eight or more: all; none or less: all are 0).
// left(i) + 8 lane is the same in all 16 lanes, or not above 0 in any: nothing is read for it then.  VEC: they lie on 16 bytes.  Otherwise a lane loads the aligned 16
// bytes in which its values begin, takes the following ones from the next lane and shifts, unless that would reach over the matrix's ends.  ALIKE: all N lie alike (step is whole
// 16 bytes), so that they shift by one choice.  (4001 x 10239, at odd places: 24.3 us; 27.2 with an address and a choice for every eight values, 32 with two pieces of its own
// for every lane.)
template <class T, bool VEC, bool ALIKE, int N, class Left>
__device__ __forceinline__ void load_all(const QuantParams& p, const T* from, long long step, Left&& left, Raw8<T> (&v)[N]) {
  constexpr int W = Raw8<T>::kWords, kPieces = W / 4;
  if (!VEC) {
    const int lane = threadIdx.x & 15;
    const T* x = static_cast<const T*>(p.x);
    const uintptr_t begin = reinterpret_cast<uintptr_t>(x), end = reinterpret_cast<uintptr_t>(x + (p.rows - 1) * p.ldx + p.k);
    bool inside = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uintptr_t first = reinterpret_cast<uintptr_t>(from - lane * 8 + i * step) & ~uintptr_t(15);  // of lane 0
      inside = inside && (left(i) + lane * 8 <= 0 || (first >= begin && first + 16 * (16 * kPieces + 1) <= end));
    }
    if (inside) {
      const uint32_t half = 0xffffu << (threadIdx.x & 16);
      auto piece_of = [&](int i) { return reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(from + i * step) & ~uintptr_t(15)); };
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool any = left(i) + lane * 8 > 0;  // (the half warp's)
        const uint4* piece = piece_of(i);
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
          const uint4 u = any ? __ldcs(piece + j) : make_uint4(0, 0, 0, 0);
          v[i].w[4 * j] = u.x, v[i].w[4 * j + 1] = u.y, v[i].w[4 * j + 2] = u.z, v[i].w[4 * j + 3] = u.w;
        }
      }
      uint4 far = make_uint4(0, 0, 0, 0);  // lane i: what follows lane 15's pieces of the i-th
      if (lane < N && left(lane) + lane * 8 > 0) far = *(piece_of(lane) + (15 - lane) * kPieces + kPieces);
      const uint32_t f[4] = {far.x, far.y, far.z, far.w};
      if (ALIKE) {
        const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(from) & 15);
        auto shift = [&](auto words) {
          constexpr int O = decltype(words)::value;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            uint32_t w[W + 4];
            v[i].template with_next<O + 1>(w, f, i, half);
#pragma unroll
            for (int j = 0; j < W; ++j) v[i].w[j] = __funnelshift_r(w[j + O], w[j + O + 1], (off & 3) * 8);
          }
        };
        if (off >> 2 == 0) shift(std::integral_constant<int, 0>());
        else if (off >> 2 == 1) shift(std::integral_constant<int, 1>());
        else if (off >> 2 == 2) shift(std::integral_constant<int, 2>());
        else shift(std::integral_constant<int, 3>());
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(from + i * step) & 15);
          uint32_t w[W + 4];
          v[i].template with_next<4>(w, f, i, half);
#pragma unroll
          for (int j = 0; j < W + 2; ++j) w[j] = off & 8 ? w[j + 2] : w[j];
#pragma unroll
          for (int j = 0; j < W + 1; ++j) w[j] = off & 4 ? w[j + 1] : w[j];
#pragma unroll
          for (int j = 0; j < W; ++j) v[i].w[j] = __funnelshift_r(w[j], w[j + 1], (off & 3) * 8);
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (left(i) < 8) v[i].cut(left(i));
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const T* at = from + i * step;
    const int n = left(i);
#pragma unroll
    for (int j = 0; j < W; ++j) v[i].w[j] = 0;
    if (VEC && n >= 8) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(at) + j);
        v[i].w[4 * j] = u.x, v[i].w[4 * j + 1] = u.y, v[i].w[4 * j + 2] = u.z, v[i].w[4 * j + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) {
          if (sizeof(T) == 4) v[i].w[j % W] = reinterpret_cast<const uint32_t*>(at)[j];
          else v[i].w[j / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(at)[j]) << (j % 2 * 16);
        }
    }
  }
}

// ---- quantisation ----------------------------------------------------------------------------------------------------------------
//
// One pass: a thread keeps its values until the block's maximum is known.  Bound: bytes (2 or 4 in, 1 out per value).  4001 x 10240 bfloat16 by rows 19.8 us (6.2 TB/s; 29.3 with one
// load per thread and two divisions per eight values), 264192 x 1280 by blocks 149 us (6.8 TB/s; 455 with the values held as fp32, two CTAs per SM instead
// of four).  Rows at odd places: 24.3 and 219 us, the shifts (issue slots three quarters full).

constexpr int kQuantThreads = 256;
constexpr int kQuantGroup = 4;  // blocks of a row that half a warp works on at a time

// 1 x 128: eight values per thread and block, half a warp per four blocks of a row, whose loads are on their way together; the four maxima are halved over the lanes
// so that a lane divides for one block alone.
template <class T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const QuantParams p) {
  griddep_wait();
  griddep_launch_dependents();  // (behind the wait: a product that starts now may read weights that an earlier kernel wrote)
  const int lane = threadIdx.x & 15;
  const uint32_t groups = uint32_t(p.blocks + kQuantGroup - 1) / kQuantGroup, unit = blockIdx.x * (kQuantThreads / 16) + (threadIdx.x >> 4), row = unit / groups;
  const bool there = row < uint32_t(p.rows);
  const int b0 = int(unit - row * groups) * kQuantGroup, c = b0 * kScaleBlock + lane * 8, left = there ? p.k - c : -kScaleBlock;
  Raw8<T> v[kQuantGroup];
  uint32_t top[kQuantGroup];
  load_all<T, VEC, true>(p, static_cast<const T*>(p.x) + (there ? row * p.ldx : 0) + c, kScaleBlock, [&](int i) { return left - i * kScaleBlock; }, v);
#pragma unroll
  for (int i = 0; i < kQuantGroup; ++i) top[i] = max(v[i].largest(), kLeastLargest);
  const bool up8 = lane & 8, up4 = lane & 4;
  uint32_t a = max(up8 ? top[2] : top[0], __shfl_xor_sync(0xffffffffu, up8 ? top[0] : top[2], 8));
  uint32_t b = max(up8 ? top[3] : top[1], __shfl_xor_sync(0xffffffffu, up8 ? top[1] : top[3], 8));
  uint32_t mine = max(up4 ? b : a, __shfl_xor_sync(0xffffffffu, up4 ? a : b, 4));  // of block lane / 4
  mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
  mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
  const float by = __fdiv_rn(448.0f, __uint_as_float(mine));
  if ((lane & 3) == 0 && there && b0 + (lane >> 2) < p.blocks) p.scale[row * p.scale_row + (b0 + (lane >> 2)) * p.scale_block] = __fdiv_rn(__uint_as_float(mine), 448.0f);
#pragma unroll
  for (int i = 0; i < kQuantGroup; ++i) {
    const float f = __shfl_sync(0xffffffffu, by, i * 4, 16);
    if (left - i * kScaleBlock > 0) v[i].store_e4m3(p.q + row * p.ldq + c + i * kScaleBlock, left - i * kScaleBlock, f);
  }
}

// 128 x 128: a CTA per block, eight rows of eight values per thread.
template <class T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 4 ? 2 : 4) quantize_blocks_kernel(const QuantParams p) {
  __shared__ uint32_t part[kQuantThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const int up = blockIdx.x / p.blocks, b = blockIdx.x - up * p.blocks;
  const int row0 = up * kScaleBlock + (threadIdx.x >> 4), c = b * kScaleBlock + (threadIdx.x & 15) * 8;
  Raw8<T> v[8];
  uint32_t top = kLeastLargest;
  load_all<T, VEC, false>(p, static_cast<const T*>(p.x) + row0 * p.ldx + c, 16 * p.ldx, [&](int i) { return row0 + 16 * i < p.rows ? p.k - c : -kScaleBlock; }, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, v[i].largest());
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; ++i) top = max(top, part[i]);
  const float by = __fdiv_rn(448.0f, __uint_as_float(top));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + 16 * i;
    if (row < p.rows && c < p.k) v[i].store_e4m3(p.q + row * p.ldq + c, p.k - c, by);
  }
  if (threadIdx.x == 0) p.scale[up * p.scale_row + b * p.scale_block] = __fdiv_rn(__uint_as_float(top), 448.0f);
}

// ---- products ----------------------------------------------------------------------------------------------------------------------
//
// The kernels multiply one block of 128 columns at a time on the tensor cores (kind::f8f6f4, four instructions of 32), each into an accumulator of its
// own in TMEM, and add acc += d * (xs ws) in registers, so that the scales are applied once per block and sums are fp32 throughout.  (The block-scaled
// MMAs take powers of two alone as scales.)  The way of an accumulator from the MMAs' barrier through registers and back to the next MMAs is what many rows are bound by.
// Scales come by ordinary loads: the kernels begin while the one in front still writes them, and the read-only path (__ldg) is for what nobody writes in a kernel's
// life; a compiler may also move such loads in front of the wait for that kernel.  (4096 x 5376 by 21504: 407 us, by the read-only path 405; 5310 x 4000 by 13887 291
// and 288; the other kernels are as fast.)

struct Fp8LinearParams {
  const float* x_scale;
  long long x_scale_row, x_scale_block;  // strides of a row and of a block of columns
  const float* w_scale;  // [ceil(n / 128), blocks]
  void* out;
  long long ldo;
  int out_f32;
  int rows, n, blocks;
  int splits;       // stream and tile: CTAs of a cluster that share a tile's blocks
  int stages;       // of operands in shared memory
  int early;        // stream and tile: the weights may be read before the kernel in front is done (it waited for everything before itself)
  int tma_cols;     // pair and tile: results leave by TMA in boxes that end by this column (0: none)
};

// Waits that run out (some 2 s: a protocol error) end the kernel instead of the GPU: the CTA's roles go through their loops without waiting and without
// issuing anything, its copies get time to land, TMEM is freed, and this counter (mtx_linear_fp8_stalls) says that results are wrong.  (Everything inline and no way
// out of the loops: with a call and breaks behind the waits 4096 x 5376 by 21504 took 833 us, so 451.)
__device__ unsigned int d_fp8_waits_failed = 0;

__device__ __forceinline__ bool fp8_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  do {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (clock64() - t0 > 4000000000LL) {
      atomicAdd(&d_fp8_waits_failed, 1u);
      *failed = 1;
    }
  } while (*failed == 0);
  return false;
}
// after a wait that ran out: copies and MMAs in flight have a millisecond to end before the CTA's shared memory and TMEM go
__device__ __forceinline__ void fp8_let_copies_land() {
  const long long t0 = clock64();
  while (clock64() - t0 < 2000000) __nanosleep(1000);
}

// Instruction descriptor, kind::f8f6f4: A = B = e4m3 (format 0), D = fp32, both operands K-major.
__host__ __device__ inline uint32_t umma_idesc_e4m3(int M, int N) { return 1u << 4 | uint32_t(N >> 3) << 17 | uint32_t(M >> 4) << 24; }

__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void fma_pair(unsigned long long& acc, unsigned long long d, unsigned long long s) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(d), "l"(s));
}
__device__ __forceinline__ unsigned long long pair_of(uint32_t lo, uint32_t hi) { return (unsigned long long)hi << 32 | lo; }
__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float pair_lo(unsigned long long v) { return __uint_as_float(uint32_t(v)); }
__device__ __forceinline__ float pair_hi(unsigned long long v) { return __uint_as_float(uint32_t(v >> 32)); }

// Hands an accumulator back to the thread that issues MMAs.  The loads from TMEM are complete (wait::ld) and ordered (tcgen05.fence), nothing else is published:
// a releasing arrive would wait for the next block's scales, which are on their way from L2 at that moment (4096 x 5376 by 21504: 1106 us, 833 without).
__device__ __forceinline__ void fp8_release(uint64_t* bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fp8_release_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(smem_u32(bar) & kPairLeaderMask) : "memory");
}

// f(c, v) for 16 accumulator columns c .. at a time; the next ones are on their way meanwhile.  done() behind the last load.
template <int COLS, class F, class D>
__device__ __forceinline__ void fp8_columns(uint32_t taddr, F&& f, D&& done) {
  uint32_t v[2][16];
  tmem_ld_x16_issue(taddr, v[0]);
#pragma unroll
  for (int c = 0; c < COLS; c += 16) {
    tmem_ld_wait();
    if (c + 16 < COLS) tmem_ld_x16_issue(taddr + uint32_t(c + 16), v[(c / 16 + 1) & 1]);
    else done();
    f(c, v[(c / 16) & 1]);
  }
}

constexpr int kFp8OperandBytes = 128 * kScaleBlock;  // 128 rows of one block
constexpr int kFp8MaxStages = 16;
constexpr int kFp8MaxSplits = 8;  // CTAs of a cluster

struct Fp8SmemTail {
  uint64_t full[kFp8MaxStages];  // a stage's operands are there
  uint64_t done[kFp8MaxStages];  // its MMAs are done: the stage may be filled again, and the block's accumulator is complete (one commit for both)
  uint64_t tmem_empty[4];        // the epilogue has taken an accumulator in
  uint32_t tmem_base;
  int failed;
};

// ---- few rows: the weights as they stream by ------------------------------------------------------------------------------------------
//
// The 128 rows of a weight tile are the MMA's M, the activation rows, up to BN, its N: nothing is padded but the last few rows, and a CTA takes in 16 KB of weights
// with BN * 128 bytes of activations per block.  An epilogue thread owns a weight row and BN sums.  Bound: the weights' bytes.
// Few tiles are shared by the CTAs of a cluster, each with a part of the blocks, and the parts are added over distributed shared memory in
// the order of the blocks (so that a result never depends on timing).  1 x 1280 by 264192 columns 52.1 us (the weights at 6.5 TB/s), 64 rows 67.4 (the
// logits, 68 MB, beside them); 64 x 5120 by 1280, ten tiles in eight parts each, 7.6: launch, fill and exchange, the weights are 1.0 of it.

template <int BN>
__host__ __device__ constexpr int fp8_stream_warps() { return BN <= 32 ? 4 : 8; }  // epilogue warps: 16 or 32 activation rows each
template <int BN>
__host__ __device__ constexpr int fp8_stream_buffers() { return BN == 32 ? 2 : 4; }  // accumulators in TMEM (two or three CTAs share an SM's 512 columns), at most as many as stages
template <int BN>
__host__ __device__ constexpr int fp8_stream_stage_bytes() { return kFp8OperandBytes + BN * kScaleBlock; }
template <int BN>
__host__ __device__ constexpr int fp8_stream_tail_at(int stages) { return stages * fp8_stream_stage_bytes<BN>() + 4 * 2 * BN * int(sizeof(float)); }
template <int BN>
constexpr size_t fp8_stream_smem_bytes(int stages) { return 1024 + fp8_stream_tail_at<BN>(stages) + sizeof(Fp8SmemTail); }

template <int BN>
__global__ void __launch_bounds__(64 + 32 * fp8_stream_warps<BN>()) fp8_stream_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                                                                                      const Fp8LinearParams p) {
  constexpr int NB = fp8_stream_buffers<BN>(), kStage = fp8_stream_stage_bytes<BN>(), kTmemCols = NB * BN, kWarps = fp8_stream_warps<BN>(), kCols = BN * 4 / kWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* factors = reinterpret_cast<float*>(smem + size_t(p.stages) * kStage);  // [warps][2][kCols]
  static_assert(kWarps * 2 * kCols == 4 * 2 * BN, "the factors lie between the stages and the tail");
  Fp8SmemTail* tail = reinterpret_cast<Fp8SmemTail*>(smem + fp8_stream_tail_at<BN>(p.stages));
  volatile int* failed = &tail->failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = blockIdx.y;
  const int b0 = int((long long)part * p.blocks / p.splits), b1 = int((long long)(part + 1) * p.blocks / p.splits), per = b1 - b0;
  const int tiles = (p.n + 127) / 128;
  const int mine = int(blockIdx.x) < tiles ? (tiles - 1 - int(blockIdx.x)) / int(gridDim.x) + 1 : 0, F = mine * per;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->done[s], 1);
    }
    for (int b = 0; b < NB; ++b) mbar_init(&tail->tmem_empty[b], kWarps);
    tail->failed = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tail->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = tail->tmem_base;

  if (warp == 0) {
    const bool issuer = elect_one();
    auto load_w = [&](int s, int n0, int b) {
      mbar_expect_tx(&tail->full[s], kStage);
      tma_load_2d(smem + s * kStage, &tm_w, b * kScaleBlock, n0, &tail->full[s], kEvictFirst);
    };
    auto load_x = [&](int s, int b) { tma_load_2d(smem + s * kStage + kFp8OperandBytes, &tm_x, b * kScaleBlock, 0, &tail->full[s], kEvictLast); };
    const int pre = p.early ? min(F, p.stages) : 0;
    int s = 0, b = b0, t = blockIdx.x;
    if (issuer)
      for (int f = 0; f < pre; ++f) {
        load_w(f, t * 128, b);
        if (++b == b1) b = b0, t += gridDim.x;
      }
    griddep_wait();
    b = b0;
    t = blockIdx.x;
    uint32_t phase = 1;
    bool good = true;
    for (int f = 0; f < F; ++f) {
      if (f >= p.stages) good &= fp8_wait(&tail->done[s], phase, failed);
      if (issuer && good) {
        if (f >= pre) load_w(s, t * 128, b);
        load_x(s, b);
      }
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++b == b1) b = b0, t += gridDim.x;
    }
    __syncwarp();
  } else if (warp == 1) {
    griddep_wait();  // (no stage is full before; what the kernel in front takes is not counted in the waits' limit)
    const bool issuer = elect_one();
    const uint32_t idesc = umma_idesc_e4m3(128, BN);
    int s = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 1;
    bool good = true;
    for (int f = 0; f < F; ++f) {
      good &= fp8_wait(&tail->full[s], phase, failed);
      good &= fp8_wait(&tail->tmem_empty[buf], acc_phase, failed);
      tcgen05_fence_after();
      if (issuer && good) {
        const uint64_t dw = umma_desc_sw128(smem + s * kStage), dx = umma_desc_sw128(smem + s * kStage + kFp8OperandBytes);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) umma_e4m3(tmem_base + uint32_t(buf * BN), dw + 2 * kk, dx + 2 * kk, idesc, kk != 0);
        umma_commit(&tail->done[s]);
      }
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++buf == NB) buf = 0, acc_phase ^= 1;
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, local = quarter * 32 + lane, c0 = (warp - 2) / 4 * kCols;  // this thread's weight row, and the first of its activation rows
    float* factor = factors + (warp - 2) * 2 * kCols;
    const uint32_t lanes = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(c0);
    static_assert(kCols <= 32, "a lane brings the scale of one activation row");
    griddep_wait();  // (scales and activations of the kernel in front)
    int t = blockIdx.x, s = 0, buf = 0;
    uint32_t phase = 0;
    // The tile's weight rows share a scale; a lane brings that and the one of an activation row, two blocks ahead (a round through L2 takes as long as several
    // blocks); behind the last row they are not stored: any scale will do.
    const float *next_x = p.x_scale, *next_w = p.w_scale;
    float xs[2], ws[2];
    auto fetch = [&](int i) {
      xs[i] = *next_x;
      ws[i] = *next_w;
      next_x += p.x_scale_block;
      ++next_w;
    };
    auto begin = [&](int tt) {
      next_x = p.x_scale + min(c0 + (lane & (kCols - 1)), p.rows - 1) * p.x_scale_row + b0 * p.x_scale_block;
      next_w = p.w_scale + tt * (long long)p.blocks + b0;
      fetch(0);
      if (per > 1) fetch(1);
    };
    if (mine > 0) begin(t);
    unsigned long long acc[kCols / 2];
    auto step = [&](int b, int i) {
      float* now = factor + i * kCols;
      now[lane & (kCols - 1)] = xs[i] * ws[i];
      if (b + 2 < per) fetch(i);
      __syncwarp();
      fp8_wait(&tail->done[s], phase, failed);
      tcgen05_fence_after();
      fp8_columns<kCols>(
          lanes + uint32_t(buf * BN),
          [&](int c, const uint32_t(&v)[16]) {
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
              const float4 by = *reinterpret_cast<const float4*>(now + c + x);
              fma_pair(acc[(c + x) / 2], pair_of(v[x], v[x + 1]), pair_of(by.x, by.y));
              fma_pair(acc[(c + x) / 2 + 1], pair_of(v[x + 2], v[x + 3]), pair_of(by.z, by.w));
            }
          },
          [&]() {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) fp8_release(&tail->tmem_empty[buf]);
          });
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++buf == NB) buf = 0;
    };
    for (int j = 0; j < mine; ++j, t += gridDim.x) {
#pragma unroll
      for (int c = 0; c < kCols / 2; ++c) acc[c] = 0;
      for (int b = 0; b < per; b += 2) {
        step(b, 0);
        if (b + 1 < per) step(b + 1, 1);
      }
      __syncwarp();  // (an odd number of blocks: the next tile's first factors go where the last ones were)
      if (j + 1 < mine) begin(t + int(gridDim.x));
      if (p.splits == 1) {
        const int n = t * 128 + local, left = p.rows - c0;
        if (n < p.n) {
          if (p.out_f32) {
            float* o = static_cast<float*>(p.out) + c0 * p.ldo + n;
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              if (c < left) __stcs(o, c & 1 ? pair_hi(acc[c / 2]) : pair_lo(acc[c / 2]));
              o += p.ldo;
            }
          } else {
            bf16* o = static_cast<bf16*>(p.out) + c0 * p.ldo + n;
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              if (c < left) *o = __float2bfloat16_rn(c & 1 ? pair_hi(acc[c / 2]) : pair_lo(acc[c / 2]));
              o += p.ldo;
            }
          }
        }
      }
    }
    if (p.splits > 1 && mine > 0) {  // (one tile per CTA) the parts lie where the operands were: the last MMA has read them
      float* parts = reinterpret_cast<float*>(smem) + c0 * 128 + local;
#pragma unroll
      for (int c = 0; c < kCols; ++c) parts[c * 128] = c & 1 ? pair_hi(acc[c / 2]) : pair_lo(acc[c / 2]);
    }
    __syncwarp();
  }
  if (*failed) fp8_let_copies_land();
  if (p.splits > 1) {
    cluster_sync_all();
    if (warp >= 2) {  // a thread adds four neighbouring columns of the result, all parts on their way at once
      const int n0 = blockIdx.x * 128 + lane * 4, count = min(4, p.n - n0);
      const uint32_t own = smem_u32(smem) + lane * 16;
      for (int c = part + (warp - 2) * p.splits; c < p.rows; c += kWarps * p.splits) {
        float4 v[kFp8MaxSplits];
#pragma unroll
        for (int q = 0; q < kFp8MaxSplits; ++q)
          if (q < p.splits) v[q] = ld_dsmem_f32x4(dsmem_addr(own + c * 512, q));
        float4 sum = v[0];
#pragma unroll
        for (int q = 1; q < kFp8MaxSplits; ++q)
          if (q < p.splits) sum.x += v[q].x, sum.y += v[q].y, sum.z += v[q].z, sum.w += v[q].w;
        const float o[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < count) {
            const long long at = c * p.ldo + n0 + i;
            if (p.out_f32) static_cast<float*>(p.out)[at] = o[i];
            else static_cast<bf16*>(p.out)[at] = __float2bfloat16_rn(o[i]);
          }
      }
      __syncwarp();
    }
    cluster_sync_all();  // the parts are read from the other CTAs until here
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, kTmemCols);
}

// ---- many rows: pairs of CTAs ------------------------------------------------------------------------------------------------------------
//
// Two CTAs of a cluster (a TPC's two SMs) work on one tile of 256 rows x 256 columns with cta_group::2 MMAs: CTA c of the pair holds rows 128 c .. of the
// activations and half of the weight tile, so an SM takes in 32 KB per block for 2^22 multiply-adds.  A thread of the
// epilogue warps owns one row and half of the columns: its scale of a block is ONE number, which the sums take in with packed fused
// multiply-adds while the next block's MMAs run into another accumulator.
// 4096 x 5376 by 21504: 407 us, 2.3 PFLOP/s.  A block of a tile takes 0.42 us where its MMAs take 0.28: TMEM holds two such accumulators, and one is
// on its way (MMAs, barrier, 128 columns through registers in some 450 cycles, barriers of both CTAs) for two blocks.  (Without the sums in between: 342 us of 421.)

constexpr int kFp8PairRows = 256, kFp8PairCols = 256;

// Epilogue warps: 32 rows x half of the columns each.  (Sixteen with a quarter of the columns take longer, 532 us for 421 at 4096 x 5376 by 21504: every
// arrival at the leader's barrier is on the way from one block's sums to the next MMAs into their accumulator.  So do registers moved from the
// first warps to these, 482 us, and MMAs and barriers for each half of the columns, 402 for 390.)
constexpr int kFp8PairWarps = 8;
constexpr int kFp8PairThreads = 64 + 32 * kFp8PairWarps;  // warp 0: copies, warp 1: MMAs, then the sums
constexpr int kFp8PairStage = kFp8OperandBytes + kFp8PairCols / 2 * kScaleBlock;
constexpr int kFp8PairStages = 5;
constexpr int kFp8PairBuffers = 2;  // of 32 rows x 128 bytes per epilogue warp, for results on their way
__host__ __device__ constexpr int fp8_pair_tail_at(int stages) { return stages * kFp8PairStage + kFp8PairWarps * kFp8PairBuffers * 4096; }
constexpr size_t kFp8PairSmem = 1024 + fp8_pair_tail_at(kFp8PairStages) + sizeof(Fp8SmemTail);
static_assert(kFp8PairSmem <= 227 * 1024, "what an SM has");

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* tm, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}

// A warp's 32 rows from row0 on, COLS columns from col0 on, from registers (a thread has a row) to memory: 32 rows x 128 bytes at a time through shared memory
// (chunk j of row r at j ^ (r & 7): the 128-byte swizzle of the tensor map).  stage: BUFFERS times 4096 bytes.
template <int COLS, int BUFFERS, class OUT>
__device__ __forceinline__ void fp8_store(const unsigned long long (&acc)[COLS / 2], uint8_t* stage, const CUtensorMap& tm_out, const Fp8LinearParams& p, int row0, int col0) {
  constexpr int kBox = 128 / int(sizeof(OUT));
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < COLS; c += kBox) {
    if (col0 + c < p.n && row0 < p.rows) {
      uint8_t* to = stage + c / kBox % BUFFERS * 4096;
      if (p.tma_cols > 0) {  // the buffer's last store has been read: one of the tile before, or of this one's box but BUFFERS
        if (lane == 0 && c == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        if (lane == 0 && c >= BUFFERS * kBox) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BUFFERS - 1) : "memory");
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint4 u;
        if (sizeof(OUT) == 2) {
          const unsigned long long* a = acc + (c + 8 * j) / 2;
          u = make_uint4(pack_bf16x2(pair_lo(a[0]), pair_hi(a[0])), pack_bf16x2(pair_lo(a[1]), pair_hi(a[1])), pack_bf16x2(pair_lo(a[2]), pair_hi(a[2])),
                         pack_bf16x2(pair_lo(a[3]), pair_hi(a[3])));
        } else {
          const unsigned long long* a = acc + (c + 4 * j) / 2;
          u = make_uint4(uint32_t(a[0]), uint32_t(a[0] >> 32), uint32_t(a[1]), uint32_t(a[1] >> 32));
        }
        *reinterpret_cast<uint4*>(to + lane * 128 + ((j ^ (lane & 7)) << 4)) = u;
      }
      if (col0 + c + kBox <= p.tma_cols) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tm_out, to, col0 + c, row0);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else {  // results at odd places, or a last box: a row's values by neighbouring lanes, sixteen rows on their way at a time (5310 x 4000 by 13887: 418 us row by row, 291 so)
        __syncwarp();
        const int rows = min(32, p.rows - row0), cols = min(kBox, p.n - col0 - c);
        OUT* o = static_cast<OUT*>(p.out) + row0 * p.ldo + col0 + c + lane;
        auto value = [&](int r, int k) {
          const int i = lane + 32 * k;
          return *reinterpret_cast<const OUT*>(to + r * 128 + (((i / (kBox / 8)) ^ (r & 7)) << 4) + i % (kBox / 8) * sizeof(OUT));
        };
        if (rows == 32 && cols == kBox) {
#pragma unroll 1
          for (int r0 = 0; r0 < 32; r0 += 16) {
            OUT x[16][kBox / 32];
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
              for (int k = 0; k < kBox / 32; ++k) x[r][k] = value(r0 + r, k);
#pragma unroll
            for (int r = 0; r < 16; ++r, o += p.ldo)
#pragma unroll
              for (int k = 0; k < kBox / 32; ++k) o[32 * k] = x[r][k];
          }
        } else {
          for (int r = 0; r < rows; ++r, o += p.ldo)
#pragma unroll
            for (int k = 0; k < kBox / 32; ++k)
              if (lane + 32 * k < cols) o[32 * k] = value(r, k);
        }
        __syncwarp();
      }
    }
  }
}

template <class OUT>
__global__ void __launch_bounds__(kFp8PairThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_out, const Fp8LinearParams p) {
  constexpr int BN = kFp8PairCols, kStage = kFp8PairStage, NB = 512 / BN, kHalf = BN / 2, kWarps = kFp8PairWarps, kCols = BN * 4 / kWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // (the number of stages comes with the call: as a constant it leaves the sums' threads too few registers, 408 us for 400 at 4096 x 5376 by 21504)
  uint8_t* staged = smem + p.stages * kStage;
  Fp8SmemTail* tail = reinterpret_cast<Fp8SmemTail*>(smem + fp8_pair_tail_at(p.stages));
  volatile int* failed = &tail->failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(blockIdx.x) & 1, pair = int(blockIdx.x) >> 1, pairs = int(gridDim.x) >> 1;
  const int m_tiles = (p.rows + kFp8PairRows - 1) / kFp8PairRows, tiles = m_tiles * ((p.n + BN - 1) / BN);
  const int mine = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0, F = mine * p.blocks;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_out);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->done[s], 1);
    }
    for (int b = 0; b < NB; ++b) mbar_init(&tail->tmem_empty[b], 2 * kWarps);  // the epilogue warps of both CTAs
    tail->failed = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&tail->tmem_base, 512);
    tmem_relinquish_pair();
  }
  tcgen05_fence_before();
  cluster_sync_all();
  tcgen05_fence_after();
  const uint32_t tmem_base = tail->tmem_base;
  griddep_wait();

  if (warp >= 2) {
    const int c0 = (warp - 2) / 4 * kCols, quarter = warp & 3;
    uint8_t* stage = staged + (warp - 2) * kFp8PairBuffers * 4096;
    const uint32_t lanes = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(c0);
    int t = pair, s = 0, buf = 0;
    uint32_t phase = 0;
    // This thread's scales, of its row and of its columns, come two blocks ahead (a round through L2 takes as long as the MMAs of two); rows and columns behind
    // the last are not stored: any scale will do.
    const float *next_x = p.x_scale, *next_w = p.w_scale;
    float xs[2], ws[2];
    auto fetch = [&](int i) {
      xs[i] = *next_x;
      ws[i] = *next_w;
      next_x += p.x_scale_block;
      ++next_w;
    };
    auto begin = [&](int tt) {
      const int nt = tt / m_tiles, r = (tt - nt * m_tiles) * kFp8PairRows + rank * 128 + quarter * 32 + lane, c = nt * BN + c0;
      next_x = p.x_scale + min(r, p.rows - 1) * p.x_scale_row;
      next_w = p.w_scale + min(c, p.n - 1) / kScaleBlock * (long long)p.blocks;
      fetch(0);
      if (p.blocks > 1) fetch(1);
    };
    if (mine > 0) begin(t);
    unsigned long long acc[kCols / 2];
    auto step = [&](int b, int i) {
      fp8_wait(&tail->done[s], phase, failed);
      tcgen05_fence_after();
      float scale;  // (volatile: multiplied here, not right behind the loads)
      asm volatile("mul.rn.f32 %0, %1, %2;" : "=f"(scale) : "f"(xs[i]), "f"(ws[i]));
      const unsigned long long by = pair_of(scale, scale);
      fp8_columns<kCols>(
          lanes + uint32_t(buf * BN),
          [&](int c, const uint32_t(&v)[16]) {
#pragma unroll
            for (int x = 0; x < 16; x += 2) fma_pair(acc[(c + x) / 2], pair_of(v[x], v[x + 1]), by);
            // (beside the last columns' way from TMEM: 5310 x 4000 by 13887 291 us, behind them 295)
            if (c == kCols - 32 && b + 2 < p.blocks) fetch(i);
          },
          [&]() {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) fp8_release_leader(&tail->tmem_empty[buf]);
          });
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++buf == NB) buf = 0;
    };
    for (int j = 0; j < mine; ++j, t += pairs) {
#pragma unroll
      for (int c = 0; c < kCols / 2; ++c) acc[c] = 0;
      for (int b = 0; b < p.blocks; b += 2) {
        step(b, 0);
        if (b + 1 < p.blocks) step(b + 1, 1);
      }
      if (j + 1 < mine) begin(t + pairs);
      fp8_store<kCols, kFp8PairBuffers, OUT>(acc, stage, tm_out, p, t % m_tiles * kFp8PairRows + rank * 128 + quarter * 32, t / m_tiles * BN + c0);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  } else if (warp == 0) {
    const bool issuer = elect_one();
    int s = 0, b = 0, t = pair;
    uint32_t phase = 1;
    bool good = true;
    for (int f = 0; f < F; ++f) {
      if (f >= p.stages) good &= fp8_wait(&tail->done[s], phase, failed);
      if (issuer && good) {
        if (rank == 0) mbar_expect_tx(&tail->full[s], 2 * kStage);
        tma_load_2d_pair(smem + s * kStage, &tm_x, b * kScaleBlock, t % m_tiles * kFp8PairRows + rank * 128, &tail->full[s], kEvictLast);
        tma_load_2d_pair(smem + s * kStage + kFp8OperandBytes, &tm_w, b * kScaleBlock, t / m_tiles * BN + rank * kHalf, &tail->full[s], kEvictNormal);
      }
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++b == p.blocks) b = 0, t += pairs;
    }
    // the commits of the last stages arrive on this CTA's barriers too: they have to be there before it may leave
    const int last = min(F, p.stages);
    for (int f = 0; f < last; ++f) {
      if (s == 0) s = p.stages, phase ^= 1;
      --s;
      fp8_wait(&tail->done[s], phase ^ 1, failed);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const bool issuer = elect_one();
      const uint32_t idesc = umma_idesc_e4m3(kFp8PairRows, BN);
      const uint64_t d0 = umma_desc_sw128(smem);
      const uint32_t desc_hi = uint32_t(d0 >> 32), desc_lo = uint32_t(d0);  // (the low words alone count on)
      int s = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 1;
      bool good = true;
      for (int f = 0; f < F; ++f) {
        good &= fp8_wait(&tail->full[s], phase, failed);
        good &= fp8_wait(&tail->tmem_empty[buf], acc_phase, failed);
        tcgen05_fence_after();
        if (issuer && good) {
          const uint32_t at = desc_lo + uint32_t(s) * (kStage >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_e4m3_pair(tmem_base + uint32_t(buf * BN), umma_desc_of(at + kk * 2, desc_hi), umma_desc_of(at + (kFp8OperandBytes >> 4) + kk * 2, desc_hi), idesc, kk != 0);
          umma_commit_pair(&tail->done[s]);
        }
        if (++s == p.stages) s = 0, phase ^= 1;
        if (++buf == NB) buf = 0, acc_phase ^= 1;
      }
    }
    __syncwarp();
  }
  if (*failed) fp8_let_copies_land();
  tcgen05_fence_before();
  cluster_sync_all();  // the pair's shared memory and TMEM are in use until both CTAs are done
  tcgen05_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// ---- some rows: a tile per CTA -------------------------------------------------------------------------------------------------------------
//
// 128 rows x BN columns of a CTA's own, rows as the MMA's M like the pairs' (one scale per thread and block).  BN = 128: the sum may be shared by a cluster's CTAs
// like the streamed weights', and TMEM holds four accumulators.  No barrier of another CTA is on an accumulator's way, and the bound is what an SM takes in from L2:
// 32 KB of operands in 0.30 us, some 60 bytes a clock.  BN = 256: 48 KB in 0.36 to 0.45 us for twice the work, but half as many tiles.
// 333 x 2560 by 10240: 240 tiles of 128 columns (two waves) 18.1 us, 120 of 256 (one) 14.9; 128 x 2560 by 10240 11.3 and 14.2; 333 x 5120 by 1280, 30 tiles in four
// parts each, 10.1.  (Pairs of CTAs with tiles of 128 columns take 26.1, 18.9 and 17.8, and 128 activation rows as the N of streamed weights 23.9, 13.7
// and 12.1: the pairs for their barriers, the others for a scale per column.)

constexpr int kFp8TileWarps = 8;  // epilogue warps: 32 rows x half of the columns each
constexpr int kFp8TileThreads = 64 + 32 * kFp8TileWarps;
template <int BN>
__host__ __device__ constexpr int fp8_tile_stage() { return kFp8OperandBytes + BN * kScaleBlock; }
template <int BN>
constexpr int fp8_tile_stages() { return BN == 128 ? 6 : 4; }  // (what shared memory holds; in the kernel from the call, like the pairs')
template <int BN>
__host__ __device__ constexpr int fp8_tile_tail_at(int stages) { return stages * fp8_tile_stage<BN>() + kFp8TileWarps * 4096; }
template <int BN>
constexpr size_t fp8_tile_smem() { return 1024 + fp8_tile_tail_at<BN>(fp8_tile_stages<BN>()) + sizeof(Fp8SmemTail); }
static_assert(fp8_tile_smem<128>() <= 227 * 1024 && fp8_tile_smem<256>() <= 227 * 1024, "what an SM has");
static_assert(128 * 128 * sizeof(float) <= fp8_tile_stages<128>() * fp8_tile_stage<128>(), "a CTA's part of a tile lies where the operands were");

template <int BN, class OUT>
__global__ void __launch_bounds__(kFp8TileThreads, 1)
fp8_tile_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_out, const Fp8LinearParams p) {
  constexpr int NB = 512 / BN, kCols = BN / 2, kStage = fp8_tile_stage<BN>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* staged = smem + p.stages * kStage;
  Fp8SmemTail* tail = reinterpret_cast<Fp8SmemTail*>(smem + fp8_tile_tail_at<BN>(p.stages));
  volatile int* failed = &tail->failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = blockIdx.y;
  // (256 columns with shared sums gain 2 us of 28 at best, and the code for it leaves the sums' threads too few registers: 2048 x 10240 by 2560 97 us for 72)
  const bool shared = BN == 128 && p.splits > 1;
  const int b0 = int((long long)part * p.blocks / p.splits), b1 = int((long long)(part + 1) * p.blocks / p.splits), per = b1 - b0;
  const int m_tiles = (p.rows + 127) / 128, tiles = m_tiles * ((p.n + BN - 1) / BN);
  const int mine = int(blockIdx.x) < tiles ? (tiles - 1 - int(blockIdx.x)) / int(gridDim.x) + 1 : 0, F = mine * per;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_out);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->done[s], 1);
    }
    for (int b = 0; b < NB; ++b) mbar_init(&tail->tmem_empty[b], kFp8TileWarps);
    tail->failed = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tail->tmem_base, 512);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = tail->tmem_base;

  if (warp >= 2) {
    const int c0 = (warp - 2) / 4 * kCols, quarter = warp & 3;
    const uint32_t lanes = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(c0);
    griddep_wait();  // (scales and activations of the kernel in front)
    int t = blockIdx.x, s = 0, buf = 0;
    uint32_t phase = 0;
    // this thread's scales, of its row and of its columns, two blocks ahead; behind the last row any scale will do
    const float *next_x = p.x_scale, *next_w = p.w_scale;
    float xs[2], ws[2];
    auto fetch = [&](int i) {
      xs[i] = *next_x;
      ws[i] = *next_w;
      next_x += p.x_scale_block;
      ++next_w;
    };
    auto begin = [&](int tt) {
      const int nt = tt / m_tiles, r = (tt - nt * m_tiles) * 128 + quarter * 32 + lane;
      next_x = p.x_scale + min(r, p.rows - 1) * p.x_scale_row + b0 * p.x_scale_block;
      next_w = p.w_scale + min(nt * BN + c0, p.n - 1) / kScaleBlock * (long long)p.blocks + b0;
      fetch(0);
      if (per > 1) fetch(1);
    };
    if (mine > 0) begin(t);
    unsigned long long acc[kCols / 2];
    auto step = [&](int b, int i) {
      fp8_wait(&tail->done[s], phase, failed);
      tcgen05_fence_after();
      float scale;  // (volatile: multiplied here, not right behind the loads)
      asm volatile("mul.rn.f32 %0, %1, %2;" : "=f"(scale) : "f"(xs[i]), "f"(ws[i]));
      const unsigned long long by = pair_of(scale, scale);
      fp8_columns<kCols>(
          lanes + uint32_t(buf * BN),
          [&](int c, const uint32_t(&v)[16]) {
#pragma unroll
            for (int x = 0; x < 16; x += 2) fma_pair(acc[(c + x) / 2], pair_of(v[x], v[x + 1]), by);
          },
          [&]() {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) fp8_release(&tail->tmem_empty[buf]);
          });
      if (b + 2 < per) fetch(i);
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++buf == NB) buf = 0;
    };
    for (int j = 0; j < mine; ++j, t += gridDim.x) {
#pragma unroll
      for (int c = 0; c < kCols / 2; ++c) acc[c] = 0;
      for (int b = 0; b < per; b += 2) {
        step(b, 0);
        if (b + 1 < per) step(b + 1, 1);
      }
      if (j + 1 < mine) begin(t + int(gridDim.x));
      if (!shared) fp8_store<kCols, 1, OUT>(acc, staged + (warp - 2) * 4096, tm_out, p, t % m_tiles * 128 + quarter * 32, t / m_tiles * BN + c0);
    }
    if (shared) {  // (one tile per CTA) this CTA's part, where the operands were: row r's chunk j of four columns at j ^ (r & 31)
      const int r = quarter * 32 + lane;
#pragma unroll
      for (int j = 0; j < kCols / 4; ++j)
        *reinterpret_cast<uint4*>(smem + r * 512 + (((c0 / 4 + j) ^ lane) << 4)) = make_uint4(uint32_t(acc[2 * j]), uint32_t(acc[2 * j] >> 32), uint32_t(acc[2 * j + 1]), uint32_t(acc[2 * j + 1] >> 32));
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  } else if (warp == 0) {
    const bool issuer = elect_one();
    auto load_w = [&](int s, int n0, int b) {
      mbar_expect_tx(&tail->full[s], kStage);
      tma_load_2d(smem + s * kStage + kFp8OperandBytes, &tm_w, b * kScaleBlock, n0, &tail->full[s], kEvictNormal);
    };
    const int pre = p.early ? min(F, p.stages) : 0;
    int s = 0, b = b0, t = blockIdx.x;
    if (issuer)
      for (int f = 0; f < pre; ++f) {
        load_w(f, t / m_tiles * BN, b);
        if (++b == b1) b = b0, t += gridDim.x;
      }
    griddep_wait();
    b = b0;
    t = blockIdx.x;
    int n0 = t / m_tiles * BN, r0 = t % m_tiles * 128;
    uint32_t phase = 1;
    bool good = true;
    for (int f = 0; f < F; ++f) {
      if (f >= p.stages) good &= fp8_wait(&tail->done[s], phase, failed);
      if (issuer && good) {
        if (f >= pre) load_w(s, n0, b);
        tma_load_2d(smem + s * kStage, &tm_x, b * kScaleBlock, r0, &tail->full[s], kEvictLast);
      }
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++b == b1) {
        b = b0;
        t += gridDim.x;
        n0 = t / m_tiles * BN;
        r0 = t % m_tiles * 128;
      }
    }
    __syncwarp();
  } else {
    griddep_wait();  // (no stage is full before; what the kernel in front takes is not counted in the waits' limit)
    const bool issuer = elect_one();
    const uint32_t idesc = umma_idesc_e4m3(128, BN);
    const uint64_t d0 = umma_desc_sw128(smem);
    const uint32_t desc_hi = uint32_t(d0 >> 32), desc_lo = uint32_t(d0);  // (the low words alone count on)
    int s = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 1;
    bool good = true;
    for (int f = 0; f < F; ++f) {
      good &= fp8_wait(&tail->full[s], phase, failed);
      good &= fp8_wait(&tail->tmem_empty[buf], acc_phase, failed);
      tcgen05_fence_after();
      if (issuer && good) {
        const uint32_t at = desc_lo + uint32_t(s) * (kStage >> 4);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_e4m3(tmem_base + uint32_t(buf * BN), umma_desc_of(at + kk * 2, desc_hi), umma_desc_of(at + (kFp8OperandBytes >> 4) + kk * 2, desc_hi), idesc, kk != 0);
        umma_commit(&tail->done[s]);
      }
      if (++s == p.stages) s = 0, phase ^= 1;
      if (++buf == NB) buf = 0, acc_phase ^= 1;
    }
    __syncwarp();
  }
  if (*failed) fp8_let_copies_land();
  if (shared) {
    cluster_sync_all();
    if (warp >= 2) {  // a warp adds a row, a lane four columns of it, all parts on their way at once
      const int nt = blockIdx.x / m_tiles, row0 = (blockIdx.x - nt * m_tiles) * 128, n0 = nt * 128 + lane * 4, left = min(128, p.rows - row0), count = min(4, p.n - n0);
      const uint32_t own = smem_u32(smem);
      for (int r = part + (warp - 2) * p.splits; r < left; r += kFp8TileWarps * p.splits) {
        float4 v[kFp8MaxSplits];
#pragma unroll
        for (int q = 0; q < kFp8MaxSplits; ++q)
          if (q < p.splits) v[q] = ld_dsmem_f32x4(dsmem_addr(own + r * 512 + ((lane ^ (r & 31)) << 4), q));
        float4 sum = v[0];
#pragma unroll
        for (int q = 1; q < kFp8MaxSplits; ++q)
          if (q < p.splits) sum.x += v[q].x, sum.y += v[q].y, sum.z += v[q].z, sum.w += v[q].w;
        const float o[4] = {sum.x, sum.y, sum.z, sum.w};
        OUT* to = static_cast<OUT*>(p.out) + (row0 + r) * p.ldo + n0;
        if (count == 4 && p.tma_cols > 0) {  // (whole 16 bytes of a base and a pitch)
          if (sizeof(OUT) == 4) *reinterpret_cast<float4*>(to) = sum;
          else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < count) to[i] = OUT(o[i]);
        }
      }
      __syncwarp();
    }
    cluster_sync_all();  // the parts are read from the other CTAs until here
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

}  // namespace mtx
