// Controls of a batch's logits between the projection and the sampler: penalties for seen tokens, biases, masks; and the record of seen tokens.
//
// The record of a slot is a 16-bit word per token: bit 15 says that the prompt held it, the other 15 count how often it was generated (they stay at
// 32767).  Beside it a bit per EIGHT tokens says whether any of their words is not zero: a history of some thousand tokens leaves nearly
// all of a vocabulary's groups untouched, so that the penalties read 1/64 byte per logit instead of 2.
#pragma once

#include "common.cuh"

namespace mtx {

constexpr int kControlThreads = 256;
constexpr int kControlWords = 4;  // runs of 256 tokens that a warp takes one after the other
constexpr int kControlSpan = kControlThreads / 32 * kControlWords * 256;

struct ControlParams {
  const float* logits;
  long long ld;
  float* out;
  long long ldo;
  int rows, vocab, spans;
  int slots;
  const int32_t* slot;
  const uint16_t* seen;
  long long ld_seen;
  const uint32_t* touched;
  long long ld_touched;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const int32_t* bias_off;
  const int32_t* bias_token;
  const float* bias_value;
  int allowed_rows;
  const int32_t* allowed_row;
  const uint32_t* allowed;
  long long ld_allowed;
};

// l with the penalties of a token whose word is `word`, each operation rounded on its own
__device__ __forceinline__ float penalised(float l, uint32_t word, float repetition, float presence, float frequency) {
  if (word == 0) return l;
  l = l > 0.0f ? __fdiv_rn(l, repetition) : __fmul_rn(l, repetition);
  const uint32_t count = word & 0x7fffu;
  l = __fsub_rn(l, __fmul_rn(frequency, float(count)));
  return count ? __fsub_rn(l, presence) : l;
}

// index of the first of the n ascending tokens that is at least t: each round 32 probes
__device__ __forceinline__ int first_at_least(const int32_t* token, int n, int t, int lane) {
  int lo = 0, hi = n;  // it lies in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const bool below = at < hi && token[at] < t;
    const int c = __popc(__ballot_sync(0xffffffffu, below));  // probes 0 .. c - 1 are below t
    if (c == 0) return lo;
    hi = min(hi, lo + c * step);
    lo = lo + (c - 1) * step + 1;
  }
  return lo;
}

// VEC: rows of logits and results lie on 16 bytes: lane l has the tokens 8 l .. 8 l + 7 of a run; otherwise the tokens l, l + 32, ..
template <bool VEC>
__global__ void __launch_bounds__(kControlThreads) control_logits_kernel(const ControlParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x / p.spans, span = blockIdx.x - row * p.spans;
  const int first = span * kControlSpan + (threadIdx.x >> 5) * (kControlWords * 256), last = min(p.vocab, first + kControlWords * 256);
  if (first >= p.vocab) return;
  const float* in = p.logits + row * p.ld;
  float* out = p.out + row * p.ldo;
  const bool in_place = in == out;

  const uint16_t* seen = nullptr;
  const uint32_t* touched = nullptr;
  float repetition = 1.0f, presence = 0.0f, frequency = 0.0f;
  if (p.seen != nullptr) {
    const int slot = p.slot != nullptr ? p.slot[row] : row;
    if (slot >= 0 && slot < p.slots) {
      if (p.repetition != nullptr) repetition = p.repetition[slot];
      if (p.presence != nullptr) presence = p.presence[slot];
      if (p.frequency != nullptr) frequency = p.frequency[slot];
      if (repetition != 1.0f || presence != 0.0f || frequency != 0.0f) {
        seen = p.seen + slot * p.ld_seen;
        if (p.touched != nullptr) touched = p.touched + slot * p.ld_touched;
      }
    }
  }
  const uint32_t* allowed = nullptr;
  if (p.allowed != nullptr) {
    const int a = p.allowed_row != nullptr ? p.allowed_row[row] : row;
    if (a >= 0 && a < p.allowed_rows) allowed = p.allowed + a * p.ld_allowed;
  }

  for (int t0 = first; t0 < last; t0 += 256) {
    const uint32_t hit = seen == nullptr ? 0u : touched != nullptr ? touched[t0 >> 8] : 0xffffffffu;
    if (VEC) {
      const int t = t0 + lane * 8, n = min(p.vocab - t, 8);
      if (n <= 0) continue;
      uint32_t may = 0xffu;
      if (allowed != nullptr) may = allowed[t >> 5] >> (t & 31) & 0xffu;
      const bool marked = hit >> lane & 1;
      if (in_place && may == 0xffu && !marked) continue;
      uint4 s = make_uint4(0, 0, 0, 0);
      if (marked) s = *reinterpret_cast<const uint4*>(seen + t);
      const uint32_t w[4] = {s.x, s.y, s.z, s.w};
      float v[8];
      if (n == 8) {
        if (may != 0) {
          const float4 a = *reinterpret_cast<const float4*>(in + t), b = *reinterpret_cast<const float4*>(in + t + 4);
          v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? in[t + i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = may >> i & 1 ? penalised(v[i], w[i / 2] >> (i % 2 * 16) & 0xffffu, repetition, presence, frequency) : -INFINITY;
      if (n == 8) {
        *reinterpret_cast<float4*>(out + t) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(out + t + 4) = make_float4(v[4], v[5], v[6], v[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) out[t + i] = v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + i * 32 + lane;
        if (t >= p.vocab) break;
        const bool may = allowed == nullptr || (allowed[t >> 5] >> lane & 1), marked = hit >> (t >> 3 & 31) & 1;
        if (in_place && may && !marked) continue;
        out[t] = may ? penalised(in[t], marked ? seen[t] : 0u, repetition, presence, frequency) : -INFINITY;
      }
    }
  }

  if (p.bias_off != nullptr) {
    const int b0 = p.bias_off[row], n = p.bias_off[row + 1] - b0;
    const int32_t* token = p.bias_token + b0;
    __syncwarp();  // (the warp's stores are there for its other lanes)
    for (int i = first_at_least(token, n, first, lane) + lane; i < n; i += 32) {
      const int t = token[i];
      if (t >= last) break;
      if (t < first) continue;  // (tokens that are not ascending: none is written twice or outside the warp's)
      if (i > 0 && token[i - 1] == t) continue;
      if (allowed == nullptr || (allowed[t >> 5] >> (t & 31) & 1)) out[t] = __fadd_rn(out[t], p.bias_value[b0 + i]);
    }
  }
}

// ---- the record -------------------------------------------------------------------------------------------------------------------

struct NoteParams {
  uint16_t* seen;
  long long ld_seen;
  uint32_t* touched;
  long long ld_touched;
  int slots, vocab;
  const int32_t* token;
  const int32_t* slot;
  int n, prompt;
};

// a thread per token; lanes with the same token of the same slot add once
__global__ void __launch_bounds__(kControlThreads) note_tokens_kernel(const NoteParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int i = blockIdx.x * kControlThreads + threadIdx.x, lane = threadIdx.x & 31;
  const int token = i < p.n ? p.token[i] : -1, slot = i < p.n ? (p.slot != nullptr ? p.slot[i] : i) : -1;
  const bool there = token >= 0 && token < p.vocab && slot >= 0 && slot < p.slots;
  const long long at = there ? slot * p.ld_seen + token : -1 - lane;
  const uint32_t same = __match_any_sync(0xffffffffu, at);
  if (!there || (same & ((1u << lane) - 1)) != 0) return;
  uint32_t* word = reinterpret_cast<uint32_t*>(p.seen) + (at >> 1);
  const int shift = int(at & 1) * 16;
  if (p.prompt) {
    atomicOr(word, 0x8000u << shift);
  } else {
    uint32_t old = *word, want;
    do {
      want = old;
      const uint32_t count = min((old >> shift & 0x7fffu) + uint32_t(__popc(same)), 0x7fffu);
      const uint32_t next = (old & ~(0x7fffu << shift)) | count << shift;
      if (next == old) break;
      old = atomicCAS(word, want, next);
    } while (old != want);
  }
  if (p.touched != nullptr) {
    uint32_t* bits = p.touched + slot * p.ld_touched + (token >> 8);
    const uint32_t bit = 1u << (token >> 3 & 31);
    if ((*bits & bit) == 0) atomicOr(bits, bit);
  }
}

}  // namespace mtx
