// Rotary positions: the pair (a, b) of channels i becomes amplitude (a cos t - b sin t, a sin t + b cos t), t = pos freq[i]; channels behind the rotated ones pass.
// Keys and values go to rows of their own or to the pages of their sequences.
//
// The angle is formed and brought into a turn in 64 bits (positions of some 100,000 lose the last digits of a 32-bit angle), cosine and sine are 32-bit.
// CTA = one to sixteen tokens: a thread computes the cosines and sines of a pair, then all turn the heads with them.  Bound: bytes; a token's projected heads are read once and written once
// (4001 tokens of 24 heads of 128 channels, 49 MB: 14.3 us, 3.4 TB/s).
#pragma once

#include <type_traits>

#include "common.cuh"

namespace mtx {

constexpr int kRotaryThreads = 320;
constexpr int kRotaryMostDims = 1024;

struct RotaryParams {
  int rows, heads, kv_heads, dim, pairs, half;  // pairs: of rotated channels
  float amplitude;
  const double* freq;
  const int* pos;
  const void *q, *k, *v;
  long long ldq, ldk, ldv;
  void *q_out, *k_out;
  long long ldq_out, ldk_out;
  bf16 *k_pages, *v_pages;
  int groups, num_pages, tokens_per_page, max_pages;
  const int *group, *page_map;
};

__device__ __forceinline__ void rotary_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void rotary_store(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

// eight values as they lie in memory, or one
template <class T, bool VEC>
struct RotaryRaw {
  static constexpr int N = VEC ? sizeof(T) / 2 : 1;
  typedef typename std::conditional<VEC, uint4, T>::type Word;
  Word w[N];

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const Word*>(p)[i];
  }
  // the same values as another type; of their own as they are
  template <class TO>
  __device__ __forceinline__ void pass(TO* p) const;
  __device__ __forceinline__ void values(float (&v)[VEC ? 8 : 1]) const {
    if constexpr (!VEC) {
      v[0] = static_cast<float>(w[0]);
    } else {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = sizeof(T) == 4 ? __uint_as_float(u[i % (4 * N)]) : i & 1 ? bf16_hi(u[i / 2]) : bf16_lo(u[i / 2]);
    }
  }
};

__device__ __forceinline__ void rotary_store8(bf16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void rotary_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// cosine and sine of pos * freq
__device__ __forceinline__ float2 rotary_turn(int pos, double freq, float amplitude) {
  const double turns = double(pos) * freq * 0.15915494309189533577;  // 1 / 2 pi
  float s, c;
  sincospif(2.0f * float(turns - rint(turns)), &s, &c);
  return make_float2(amplitude * c, amplitude * s);
}

__device__ __forceinline__ void rotary_store_unit(bf16* p, const float (&v)[8]) { rotary_store8(p, v); }
__device__ __forceinline__ void rotary_store_unit(float* p, const float (&v)[8]) { rotary_store8(p, v); }
template <class T>
__device__ __forceinline__ void rotary_store_unit(T* p, const float (&v)[1]) { rotary_store(p, v[0]); }

template <class T, bool VEC>
template <class TO>
__device__ __forceinline__ void RotaryRaw<T, VEC>::pass(TO* p) const {
  if constexpr (std::is_same<T, TO>::value) {
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<Word*>(p)[i] = w[i];
  } else {
    float v[VEC ? 8 : 1];
    values(v);
    rotary_store_unit(p, v);
  }
}

constexpr int kRotaryTokens = 16;  // of a CTA, at most

// VEC: heads, rotated channels and everything's place are whole eight values, so that a thread turns eight pairs (or passes eight channels) at a time.
// Every value is read and written by one thread alone: results may lie where the inputs are.  A thread has the same channels of all of its CTA's tokens (where they are is worked out
// once), and a token's values are on their way before the positions are, or while the token before is turned.
template <class TI, class TO, bool VEC>
__global__ void __launch_bounds__(kRotaryThreads, 3) rotary_kernel(const RotaryParams p, int tokens) {
  constexpr int S = VEC ? 8 : 1;  // pairs or channels of a unit
  extern __shared__ __align__(16) float2 turn[];  // [tokens][pairs]
  __shared__ long long place[kRotaryTokens];  // of a token in the pages of key head 0; -1: its keys and values have none; -2: it belongs to nobody
  // (what comes next starts when this ends: with an early start 4001 tokens of 24 heads of 128 channels took 18.6 us, not 16.4)
  griddep_wait();
  const int row0 = blockIdx.x * tokens, rows = min(tokens, p.rows - row0), dim = p.dim, pairs = p.pairs;
  // units: all heads' turned pairs, then their channels that pass, then the values (so that the lanes of most warps do the same)
  const int turning = pairs / S, passing = (dim - 2 * pairs) / S, each = dim / S, heads = p.heads + p.kv_heads;
  const int turned = heads * turning, passed = turned + heads * passing, total = passed + (p.k_pages != nullptr ? p.kv_heads * each : 0);
  const int angles = rows * pairs;
  const double freq = int(threadIdx.x) < angles ? p.freq[threadIdx.x % pairs] : 0.0;
  const int first_pos = int(threadIdx.x) < angles ? p.pos[row0 + threadIdx.x / pairs] : 0;
  const long long head_step = (long long)p.num_pages * p.tokens_per_page * dim;
  bool begun = false;
  for (int u = threadIdx.x; u < total || !begun; u += blockDim.x) {
    // the unit: its head, where its channels begin; second < 0: they pass
    const bool there = u < total, turns = u < turned, value = u >= passed;
    const int w = turns ? u : value ? u - passed : u - turned, per = turns ? turning : value ? each : passing, h0 = there ? w / per : 0, i = w - h0 * per;
    const bool query = !value && h0 < p.heads;
    const int h = value || query ? h0 : h0 - p.heads;
    const int first = turns ? (p.half ? i * S : 2 * i * S) : value ? i * S : 2 * pairs + i * S, second = turns ? (p.half ? pairs + i * S : (2 * i + 1) * S) : -1;
    const long long ld = value ? p.ldv : query ? p.ldq : p.ldk;
    const TI* from = static_cast<const TI*>(value ? p.v : query ? p.q : p.k) + row0 * ld + h * dim;
    TO* to = nullptr;
    const long long ld_to = query ? p.ldq_out : p.ldk_out;
    if (!value && (query ? p.q_out : p.k_out) != nullptr) to = static_cast<TO*>(query ? p.q_out : p.k_out) + row0 * ld_to + h * dim;
    bf16* page = nullptr;
    if (!query && p.k_pages != nullptr) page = (value ? p.v_pages : p.k_pages) + h * head_step;
    RotaryRaw<TI, VEC> a_next, b_next;
    if (there) {
      a_next.load(from + first);
      if (second >= 0) b_next.load(from + second);
    }
    if (!begun) {
      begun = true;
      if (int(threadIdx.x) < rows) {
        long long at = -1;
        if (p.k_pages != nullptr) {
          const int row = row0 + threadIdx.x, pos = p.pos[row], group = p.group != nullptr ? p.group[row] : row;
          if (group < 0 || group >= p.groups || pos < 0) {
            at = -2;
          } else {
            const int index = pos / p.tokens_per_page;
            const int number = index < p.max_pages ? p.page_map[(long long)group * p.max_pages + index] : -1;
            if (number >= 0 && number < p.num_pages) at = ((long long)number * p.tokens_per_page + pos % p.tokens_per_page) * dim;
          }
        }
        place[threadIdx.x] = at;
      }
      for (int j = threadIdx.x; j < angles; j += blockDim.x)
        turn[j] = j == int(threadIdx.x) ? rotary_turn(first_pos, freq, p.amplitude) : rotary_turn(p.pos[row0 + j / pairs], p.freq[j % pairs], p.amplitude);
      __syncthreads();
    }
    if (!there) break;
    const float2* angle = turn + (p.half ? first : first / 2);
    for (int token = 0; token < rows; ++token, angle += pairs) {
      const RotaryRaw<TI, VEC> a_now = a_next, b_now = b_next;
      if (token + 1 < rows) {
        from += ld;
        a_next.load(from + first);
        if (second >= 0) b_next.load(from + second);
      }
      const long long at = place[token];
      if (at != -2 && turns) {
        float a[S], b[S];
        a_now.values(a);
        b_now.values(b);
        if (VEC && !p.half) {
#pragma unroll
          for (int e = 0; e < S; e += 2) {
            const float2 t0 = angle[e / 2], t1 = angle[S / 2 + e / 2];
            const float x0 = a[e], y0 = a[(e + 1) % S], x1 = b[e], y1 = b[(e + 1) % S];
            a[e] = x0 * t0.x - y0 * t0.y;
            a[(e + 1) % S] = x0 * t0.y + y0 * t0.x;
            b[e] = x1 * t1.x - y1 * t1.y;
            b[(e + 1) % S] = x1 * t1.y + y1 * t1.x;
          }
        } else {
#pragma unroll
          for (int e = 0; e < S; ++e) {
            const float2 t = angle[e];
            const float x0 = a[e], y0 = b[e];
            a[e] = x0 * t.x - y0 * t.y;
            b[e] = x0 * t.y + y0 * t.x;
          }
        }
        if (to != nullptr) rotary_store_unit(to + first, a), rotary_store_unit(to + second, b);
        if (page != nullptr && at >= 0) rotary_store_unit(page + at + first, a), rotary_store_unit(page + at + second, b);
      } else if (at != -2) {
        if (to != nullptr) a_now.pass(to + first);
        if (page != nullptr && at >= 0) a_now.pass(page + at + first);
      }
      if (to != nullptr) to += ld_to;
    }
  }
}

}  // namespace mtx
