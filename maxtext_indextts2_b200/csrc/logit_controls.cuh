// Controls of a batch's logits between the projection and the sampler: penalties for seen tokens, biases, masks; and the record of seen tokens.
//
// The record of a slot is a 16-bit word per token: bit 15 says that the prompt held it, the other 15 count how often it was generated (they stay at
// 32767).  Beside it a bit per EIGHT tokens says whether any of their words is not zero: a history of some thousand tokens leaves nearly
// all of a vocabulary's groups untouched, so that the penalties read 1/64 byte per logit instead of 2.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace mtx {

constexpr int kControlThreads = 256;
constexpr int kControlRun = 256;  // tokens that a warp works on at a time: twice four per lane
constexpr int kControlWarps = 148 * 192;  // warps of a large call: four times as many as run at once (40 registers per thread), for an even end

struct ControlParams {
  const float* logits;
  long long ld;
  float* out;
  long long ldo;
  int rows, vocab;
  int runs, spans;  // runs of a warp, CTAs of a row
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
  return count ? __fsub_rn(__fsub_rn(l, __fmul_rn(frequency, float(count))), presence) : l;  // (a count of 0 takes nothing off, an infinite penalty's product neither)
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

// How a lane's four tokens of a run lie.  Logits and results of a token t lie on 16 bytes where t is ...
enum ControlForm {
  kControlAligned,  // ... a multiple of 4, in every row: a lane's tokens lie in one word of the mask, under one bit of `touched` and in 8 bytes of `seen`
  kControlShifted,  // ... s + a multiple of 4, s = -3 .. 0 by row (vocabularies of odd sizes): they may share two of each
  kControlSingle,   // ... something else in the results than in the logits: lane l has the tokens l, l + 32, .., one by one
};

// Bound: bytes, 4 read and 4 written per logit where all is allowed.  Four tokens of which none is allowed are written without being read, and in place four that nothing changes are
// neither.  64 x 264192 logits: unmasked 26.2 us (5.2 TB/s), behind masks that leave a few 23.0, where the stores alone take 19.5; at an odd size of the vocabulary 33.
// A warp takes up to three or so neighbouring runs (one each: 29.1 and 30.1, eight each: 28.5 and 23.7); runs fetched ahead in more registers by fewer warps took 30 to 39.
template <int FORM>
__global__ void __launch_bounds__(kControlThreads, 6) control_logits_kernel(const ControlParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x / p.spans, span = blockIdx.x - row * p.spans;
  const float* in = p.logits + row * p.ld;
  float* out = p.out + row * p.ldo;
  const bool in_place = in == out;
  const int shift = FORM == kControlShifted ? -int(reinterpret_cast<uintptr_t>(in) >> 2 & 3) : 0;  // in[shift] lies on 16 bytes
  const int begin = (span * (kControlThreads / 32) + (threadIdx.x >> 5)) * p.runs * kControlRun + shift;  // the warp's tokens
  const int first = max(begin, 0), last = min(p.vocab, begin + p.runs * kControlRun);
  if (first >= last) return;

  const int slot = p.seen == nullptr ? -1 : p.slot != nullptr ? p.slot[row] : row;
  const int mask_row = p.allowed == nullptr ? -1 : p.allowed_row != nullptr ? p.allowed_row[row] : row;
  const uint16_t* seen = nullptr;
  const uint32_t *touched = nullptr, *allowed = nullptr;
  float repetition = 1.0f, presence = 0.0f, frequency = 0.0f;
  if (mask_row >= 0 && mask_row < p.allowed_rows) allowed = p.allowed + mask_row * p.ld_allowed;
  if (slot >= 0 && slot < p.slots) {
    if (p.repetition != nullptr) repetition = p.repetition[slot];
    if (p.presence != nullptr) presence = p.presence[slot];
    if (p.frequency != nullptr) frequency = p.frequency[slot];
    if (p.repetition != nullptr || p.presence != nullptr || p.frequency != nullptr) {
      seen = p.seen + slot * p.ld_seen;
      if (p.touched != nullptr) touched = p.touched + slot * p.ld_touched;
    }
  }
  auto may_one = [&](int t) { return allowed == nullptr || (allowed[t >> 5] >> (t & 31) & 1); };
  auto touched_one = [&](int t) { return seen != nullptr && (touched == nullptr || (touched[t >> 8] >> (t >> 3 & 31) & 1)); };

  auto one = [&](int t) {
    const bool may = may_one(t), marked = touched_one(t);
    if (in_place && may && !marked) return;
    out[t] = may ? penalised(in[t], marked ? seen[t] : 0u, repetition, presence, frequency) : -INFINITY;
  };

  if (FORM == kControlSingle) {
    for (int t = first + lane; t < last; t += 32) one(t);
  } else {
    auto runs = [&](auto masked) {
      constexpr bool MASKED = decltype(masked)::value;
      for (int t0 = begin; t0 < last; t0 += kControlRun) {
        if (t0 < 0 || t0 + kControlRun > p.vocab) {  // the row's ends
          for (int t = max(t0, 0) + lane; t < min(t0 + kControlRun, p.vocab); t += 32) one(t);
          continue;
        }
        const int t = t0 + lane * 4;  // and 128 further on
        float* to = out + t;
        uint32_t may[2] = {0xfu, 0xfu};
        if (MASKED) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t* word = allowed + ((t + j * 128) >> 5);
            const uint32_t hi = FORM == kControlShifted && (t & 31) > 28 ? word[1] : 0u;
            may[j] = __funnelshift_r(word[0], hi, t & 31) & 0xfu;
          }
          if (!__any_sync(0xffffffffu, (may[0] | may[1]) != 0)) {  // (most runs of a mask that leaves one part of the vocabulary)
            *reinterpret_cast<float4*>(to) = *reinterpret_cast<float4*>(to + 128) = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            continue;
          }
        }
        // of `touched`: one word where runs begin at multiples of 256, else the end of one and nearly all of the next
        uint32_t hit = 0;
        if (seen != nullptr) {
          hit = 0xffffffffu;
          if (touched != nullptr) {
            hit = touched[t0 >> 8];
            if (FORM == kControlShifted) hit |= touched[(t0 + kControlRun - 1) >> 8];
          }
        }
        bool marked[2] = {false, false};
        if (hit != 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (FORM == kControlAligned) marked[j] = hit >> (t + j * 128 >> 3 & 31) & 1;
            else marked[j] = touched_one(t + j * 128) || touched_one(t + j * 128 + 3);
            marked[j] = marked[j] && may[j] != 0;
          }
        }
        float4 v[2];
        uint2 w[2];  // words of `seen`
        bool write[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          write[j] = !in_place || may[j] != 0xfu || marked[j];
          v[j] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          w[j] = make_uint2(0, 0);
          if ((!MASKED || may[j] != 0) && write[j]) v[j] = *reinterpret_cast<const float4*>(in + t + j * 128);
          if (marked[j]) {
            const uint16_t* word = seen + t + j * 128;
            if (FORM == kControlAligned) w[j] = *reinterpret_cast<const uint2*>(word);
            else w[j] = make_uint2(word[0] | uint32_t(word[1]) << 16, word[2] | uint32_t(word[3]) << 16);
          }
        }
        if (hit != 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (w[j].x != 0) {
              v[j].x = penalised(v[j].x, w[j].x & 0xffffu, repetition, presence, frequency);
              v[j].y = penalised(v[j].y, w[j].x >> 16, repetition, presence, frequency);
            }
            if (w[j].y != 0) {
              v[j].z = penalised(v[j].z, w[j].y & 0xffffu, repetition, presence, frequency);
              v[j].w = penalised(v[j].w, w[j].y >> 16, repetition, presence, frequency);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (MASKED) {
            if (!(may[j] & 1)) v[j].x = -INFINITY;
            if (!(may[j] & 2)) v[j].y = -INFINITY;
            if (!(may[j] & 4)) v[j].z = -INFINITY;
            if (!(may[j] & 8)) v[j].w = -INFINITY;
          }
          if (write[j]) *reinterpret_cast<float4*>(to + j * 128) = v[j];
        }
      }
    };
    if (allowed != nullptr) runs(std::true_type());
    else runs(std::false_type());
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
      if (may_one(t)) out[t] = __fadd_rn(out[t], p.bias_value[b0 + i]);
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
