// Eight consecutive values of a row per thread, wherever the row begins: loads and stores of whole aligned 16 bytes.
//
// Lane l of a warp has the values from `at` + 8 l on.  Where they do not lie on 16 bytes, a load takes the aligned pieces that hold them (the next lane's first piece again,
// from L1) and shifts; a store takes its neighbour's first values for the last piece.  (Sums and norms of 4001 x 5377 in bf16: 50.7 us; with eight single loads
// and stores per thread 62.9.)
#pragma once

#include "common.cuh"

namespace mtx {

template <class T>
constexpr int kPieceWords = 2 * sizeof(T);  // 32-bit words of eight values

// w[i + o], shifted by `bits`; o is the same in all threads of a warp
template <int N, int M>
__device__ __forceinline__ void shift_words(uint32_t (&out)[N], const uint32_t (&w)[M], int o, int bits) {
  static_assert(M >= N + 4, "up to three words and a half");
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (o == c) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(w[i + c], w[i + c + 1], bits);
    }
}

// the words of eight values; those from n on are 0.  [begin, end): the memory that pieces may be taken from.
template <class T>
__device__ __forceinline__ void load_piece(const T* at, int n, uintptr_t begin, uintptr_t end, uint32_t (&w)[kPieceWords<T>]) {
  constexpr int W = kPieceWords<T>;
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = 0;
  if (n <= 0) return;
  const uintptr_t a = reinterpret_cast<uintptr_t>(at);
  const int off = int(a & 15);
  if (n >= 8 && off == 0) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(at)[i];
      w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
    }
    return;
  }
  const uintptr_t first = a - off;
  if (n >= 8 && first >= begin && first + W * 4 + 16 <= end) {
    uint32_t raw[W + 4];
#pragma unroll
    for (int i = 0; i < W / 4 + 1; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(first)[i];
      raw[4 * i] = u.x, raw[4 * i + 1] = u.y, raw[4 * i + 2] = u.z, raw[4 * i + 3] = u.w;
    }
    shift_words(w, raw, off >> 2, (off & 3) * 8);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) {
      if (sizeof(T) == 4) w[i % W] = __float_as_uint(static_cast<float>(at[i]));
      else w[i / 2 % W] |= uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(static_cast<float>(at[i])))) << (i & 1) * 16;
    }
}

template <class T>
__device__ __forceinline__ float piece_value(const uint32_t (&w)[kPieceWords<T>], int i) {
  if (sizeof(T) == 4) return __uint_as_float(w[i % kPieceWords<T>]);
  return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
}

template <class T>
__device__ __forceinline__ void pack_piece(const float (&v)[8], uint32_t (&w)[kPieceWords<T>]) {
#pragma unroll
  for (int i = 0; i < kPieceWords<T>; ++i) {
    if (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
    else w[i] = pack_bf16x2(v[2 * i % 8], v[(2 * i + 1) % 8]);
  }
}

template <class T>
__device__ __forceinline__ void store_single(T* at, const uint32_t (&w)[kPieceWords<T>], int from, int to) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i >= from && i < to) {
      if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(at)[i] = w[i % kPieceWords<T>];
      else reinterpret_cast<uint16_t*>(at)[i] = uint16_t(w[i / 2 % kPieceWords<T>] >> (i & 1) * 16);
    }
}

// Stores the first n of eight values (n <= 0: none).  All 32 lanes call it together, lane l with at = lane 0's + 8 l.
template <class T>
__device__ __forceinline__ void store_piece(T* at, int n, const uint32_t (&w)[kPieceWords<T>]) {
  constexpr int W = kPieceWords<T>;
  const int lane = threadIdx.x & 31;
  const int off = int(reinterpret_cast<uintptr_t>(at) & 15);  // (the same in all lanes)
  if (off == 0) {
    if (n >= 8) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) reinterpret_cast<uint4*>(at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
      store_single(at, w, 0, n);
    }
    return;
  }
  const int head = (16 - off) / int(sizeof(T));  // values in front of the first whole piece
  uint32_t raw[W + 4];
#pragma unroll
  for (int i = 0; i < W; ++i) raw[i] = w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[W + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
  const int next = __shfl_down_sync(0xffffffffu, n, 1);
  const bool whole = n >= 8 && lane < 31 && next >= head;  // this lane's values behind `head` and the next lane's in front of it
  if (whole) {
    uint32_t out[W];
    const int bytes = head * int(sizeof(T));
    shift_words(out, raw, bytes >> 2, (bytes & 3) * 8);
    uint4* to = reinterpret_cast<uint4*>(at + head);
#pragma unroll
    for (int i = 0; i < W / 4; ++i) to[i] = make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
  } else {
    store_single(at, w, head, n);
  }
  const int stored = __shfl_up_sync(0xffffffffu, int(whole), 1);  // whether the lane in front has stored this one's first values
  if (lane == 0 || stored == 0) store_single(at, w, 0, n < head ? n : head);
}

}  // namespace mtx
