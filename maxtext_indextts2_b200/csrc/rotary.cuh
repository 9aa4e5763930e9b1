// Rotary positions: the pair (a, b) of channels i becomes amplitude (a cos t - b sin t, a sin t + b cos t), t = pos freq[i]; channels behind the rotated ones pass.
// Keys and values go to rows of their own or to the pages of their sequences.
//
// The angle is formed and brought into a turn in 64 bits (positions of some 100,000 lose the last digits of a 32-bit angle), cosine and sine are 32-bit.
// CTA = one token: its threads compute a pair's cosine and sine each, then turn all heads with them.  Bound: bytes; a token's projected heads are read once and written once.
#pragma once

#include "common.cuh"

namespace mtx {

constexpr int kRotaryThreads = 256;
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

template <class T>
__device__ __forceinline__ float rotary_load(const T* p) { return static_cast<float>(*p); }
__device__ __forceinline__ void rotary_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void rotary_store(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ void rotary_load8(const bf16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
}
__device__ __forceinline__ void rotary_load8(const float* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 u = reinterpret_cast<const float4*>(p)[i];
    v[4 * i] = u.x, v[4 * i + 1] = u.y, v[4 * i + 2] = u.z, v[4 * i + 3] = u.w;
  }
}
__device__ __forceinline__ void rotary_store8(bf16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void rotary_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// cosine and sine of pos * freq
__device__ __forceinline__ float2 rotary_turn(int pos, double freq, float amplitude) {
  const double t = double(pos) * freq, turns = rint(t * 0.15915494309189533577);
  const double r = fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586232, t));  // t - 2 pi turns, 2 pi in two parts
  float s, c;
  sincosf(float(r), &s, &c);
  return make_float2(amplitude * c, amplitude * s);
}

// VEC: heads, rotated channels and everything's place are whole eight values, so that a thread turns eight pairs (or passes eight channels) at a time.
// Every value is read and written by one thread alone: results may lie where the inputs are.
template <class TI, class TO, bool VEC>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
  __shared__ float2 turn[kRotaryMostDims / 2];
  griddep_launch_dependents();
  griddep_wait();
  const int row = blockIdx.x, dim = p.dim, pairs = p.pairs;
  const int pos = p.pos[row];
  bf16 *kp = nullptr, *vp = nullptr;  // the token's place in the pages of key head 0
  const long long head_step = (long long)p.num_pages * p.tokens_per_page * dim;
  if (p.k_pages != nullptr) {
    const int group = p.group != nullptr ? p.group[row] : row;
    if (group < 0 || group >= p.groups || pos < 0) return;  // a row that belongs to nobody
    const int index = pos / p.tokens_per_page;
    const int page = index < p.max_pages ? p.page_map[(long long)group * p.max_pages + index] : -1;
    if (page >= 0 && page < p.num_pages) {
      const long long at = ((long long)page * p.tokens_per_page + pos % p.tokens_per_page) * dim;
      kp = p.k_pages + at;
      vp = p.v_pages + at;
    }
  }
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) turn[i] = rotary_turn(pos, p.freq[i], p.amplitude);
  __syncthreads();
  const TI* q = static_cast<const TI*>(p.q) + row * p.ldq;
  const TI* k = static_cast<const TI*>(p.k) + row * p.ldk;
  const TI* v = static_cast<const TI*>(p.v) + row * p.ldv;
  TO* qo = static_cast<TO*>(p.q_out) + row * p.ldq_out;
  TO* ko = p.k_out != nullptr ? static_cast<TO*>(p.k_out) + row * p.ldk_out : nullptr;
  const int heads = p.heads + p.kv_heads;  // that are turned
  constexpr int S = VEC ? 8 : 1;           // pairs or channels of a unit
  const int turning = pairs / S, passing = (dim - 2 * pairs) / S, units = turning + passing;
  for (int u = threadIdx.x; u < heads * units; u += blockDim.x) {
    const int head = u / units, i = u - head * units;
    const bool query = head < p.heads;
    const int h = query ? head : head - p.heads;
    const TI* from = (query ? q : k) + h * dim;
    TO* to = query ? qo + h * dim : ko != nullptr ? ko + h * dim : nullptr;
    bf16* page = query || kp == nullptr ? nullptr : kp + h * head_step;
    if (VEC) {
      float a[8], b[8];
      if (i < turning) {
        const int first = p.half ? i * 8 : i * 16, second = p.half ? pairs + i * 8 : i * 16 + 8;
        rotary_load8(from + first, a);
        rotary_load8(from + second, b);
        const float2* t = turn + i * 8;
        if (p.half) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = a[e], y = b[e];
            a[e] = x * t[e].x - y * t[e].y;
            b[e] = x * t[e].y + y * t[e].x;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float2 t0 = t[e / 2], t1 = t[4 + e / 2];
            const float x0 = a[e], y0 = a[e + 1], x1 = b[e], y1 = b[e + 1];
            a[e] = x0 * t0.x - y0 * t0.y;
            a[e + 1] = x0 * t0.y + y0 * t0.x;
            b[e] = x1 * t1.x - y1 * t1.y;
            b[e + 1] = x1 * t1.y + y1 * t1.x;
          }
        }
        if (to != nullptr) {
          rotary_store8(to + first, a);
          rotary_store8(to + second, b);
        }
        if (page != nullptr) {
          rotary_store8(page + first, a);
          rotary_store8(page + second, b);
        }
      } else {
        const int c = 2 * pairs + (i - turning) * 8;
        rotary_load8(from + c, a);
        if (to != nullptr) rotary_store8(to + c, a);
        if (page != nullptr) rotary_store8(page + c, a);
      }
    } else if (i < turning) {
      const int first = p.half ? i : 2 * i, second = p.half ? pairs + i : 2 * i + 1;
      const float x = rotary_load(from + first), y = rotary_load(from + second);
      const float2 t = turn[i];
      const float a = x * t.x - y * t.y, b = x * t.y + y * t.x;
      if (to != nullptr) {
        rotary_store(to + first, a);
        rotary_store(to + second, b);
      }
      if (page != nullptr) {
        rotary_store(page + first, a);
        rotary_store(page + second, b);
      }
    } else {
      const int c = 2 * pairs + i - turning;
      const float x = rotary_load(from + c);
      if (to != nullptr) rotary_store(to + c, x);
      if (page != nullptr) rotary_store(page + c, x);
    }
  }
  if (vp == nullptr) return;
  const int each = dim / S;
  for (int u = threadIdx.x; u < p.kv_heads * each; u += blockDim.x) {
    const int h = u / each, c = (u - h * each) * S;
    bf16* to = vp + h * head_step + c;
    if (VEC) {
      float a[8];
      rotary_load8(v + h * dim + c, a);
      rotary_store8(to, a);
    } else {
      rotary_store(to, rotary_load(v + h * dim + c));
    }
  }
}

}  // namespace mtx
