// Drafted tokens against the target's probabilities.
//
//   row r, drafted token x = token[r + 1]:  x stays when u q(x) < p(x);  p = softmax(target / T), q = softmax(draft / T'), or q(x) = 1
//   the first row whose draft does not stay draws from max(p - q, 0), the row behind the last draft from p: the first token at which the weights' sum in the tokens' order
//   exceeds pick_u times their whole sum
//
// Three kernels.  The first goes through all rows in chunks, a warp each, and leaves every chunk's largest logit and its sum of 2^((l - largest) / T log2 e).  The second, a CTA per
// sequence, joins the chunks, settles which drafts stay and draws where the target's own weights are drawn from: the chunks' sums say which chunk, which is then read once more.  The
// third goes through the rows that draw from a difference; the last CTA of a sequence draws.  Bound: bytes, every row once and those of the third kernel twice.
//
// Weights are 32-bit powers of two (the results are tokens and comparisons: 64-bit weights would cost the first kernel's pace) of an exponent that is rounded twice, relative to itself; sums of a
// thread's tokens are 32-bit, all others 64-bit.  A border between two tokens lies within 2^-19.5 of the whole sum of where it belongs where p is drawn from.  Where max(p - q, 0) is, it lies within
// 2^-18.5 of p's whole sum, however little of that the difference leaves: both sums' errors come to q's part beside its weights' own.  (A draft is turned down as seldom as
// that difference is small.)  The same call always draws the same token.
//
// The first two kernels let the next one start when they end: started as soon as it fits, it made 32 sequences of 4 rows over 32768 tokens (in chunks of 4096) 17.2 us, not 15.2.
// 64 sequences of 5 rows over 264192 tokens take 127 us: 539 MB in 91 us, 5.9 TB/s, the decisions 12, the rows that differ, 76 MB of them, some 28.
#pragma once

#include "common.cuh"

namespace mtx {

constexpr int kVerifyThreads = 256;

// A chunk of a row, or a row: the largest logit, and the weights relative to it
struct VerifySum {
  double sum;
  float top;   // -infinity: nothing, and the sum is 0
  int best;    // the first token with that logit (greedy sequences)
};

// What the third kernel goes through: rows that draw from max(p - q, 0)
struct VerifyTask {
  int row;  // -1: nothing to do
  VerifySum target, draft;
};

struct VerifyParams {
  int rows, sequences, vocab, chunks;
  int left_chunks;  // of the differences
  const int *row0, *token;
  const float* target;
  long long ld_target;
  const float* draft;
  long long ld_draft;
  const float *temperature, *draft_temperature, *accept_u, *pick_u;
  int *accepted, *emitted;
  VerifySum *target_sum, *draft_sum;  // [rows, chunks]
  double* left;                       // [sequences, left_chunks]: sums of max(p - q, 0), in p's weights
  VerifyTask* task;                   // [sequences]
  int* done;                          // [sequences]: chunks that are through
};

// A logit as it counts: NaN as -infinity, infinity as the largest number
__device__ __forceinline__ float verify_logit(float l) { return fminf(fmaxf(l, -INFINITY), 3.402823466e38f); }

// 2^(l c - base) with c = log2 e / T in two parts: both products are exact in their sums, so that the exponent has two roundings of its own size and none of the logit's
struct VerifyScale {
  float hi, lo;

  __device__ __forceinline__ explicit VerifyScale(float heat) {
    const double c = 1.4426950408889634074 / double(fmaxf(heat, 9.5367431640625e-07f));  // (2^-20: products with any logit's lower part stay finite)
    hi = float(c);
    lo = float(c - double(hi));
  }
  __device__ __forceinline__ double exact() const { return double(hi) + double(lo); }
  __device__ __forceinline__ float base(float top) const { return float(double(top) * exact()); }
};

// From an exponent of 2^30 on the largest logit alone weighs anything: the next smaller one is 2^-24 of it below, a weight of 2^-64 at most, and all of 2^28 tokens 2^-36.  There the rounding of `base`
// (half of its last bit: up to 32 below 2^30, so that the largest weight lies within 2^-32 and 2^32) would reach the exponents that 32-bit numbers have.
constexpr float kVerifyFar = 1073741824.0f;

struct VerifyWeight {
  VerifyScale scale;
  float top, base;
  bool far;  // only the largest logits weigh, 1 each

  __device__ __forceinline__ VerifyWeight(const VerifyScale& s, float t) : scale(s), top(t), base(t == -INFINITY ? 0.0f : s.base(t)), far(!(fabsf(base) < kVerifyFar)) {}
  __device__ __forceinline__ float operator()(float l) const {
    if (far) return l == top ? 1.0f : 0.0f;
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(l, scale.lo, fmaf(l, scale.hi, -base))));
    return l == -INFINITY ? 0.0f : y;  // (its two products may be infinite to either side)
  }
};

__device__ __forceinline__ float verify_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// how much of b's unit a's is, for sums relative to the logits a <= b
__device__ __forceinline__ float verify_rescale(const VerifyScale& s, float a, float b) {
  if (a == b) return 1.0f;
  if (a == -INFINITY) return 0.0f;
  const VerifyWeight x(s, a), y(s, b);
  return x.far || y.far ? 0.0f : verify_ex2(x.base - y.base);
}

template <class T, class F>
__device__ __forceinline__ T verify_warp(T v, F&& join) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// over the CTA; `shared`: a value per warp
template <class T, class F>
__device__ __forceinline__ T verify_block(T v, F&& join, T* shared) {
  v = verify_warp(v, join);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
#pragma unroll
  for (int w = 1; w < kVerifyThreads / 32; ++w) v = join(v, shared[w]);
  return v;
}

struct VerifyMax {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
};
struct VerifyMin {
  __device__ __forceinline__ int operator()(int a, int b) const { return min(a, b); }
};
struct VerifyAdd {
  __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// the first token of a row's chunk: rows lie anywhere, chunks begin on 16 bytes (the first up to three tokens in front of the row)
template <int E>
__device__ __forceinline__ int verify_begin(const float* row, int chunk) { return chunk * (E * kVerifyThreads) - int(reinterpret_cast<uintptr_t>(row) >> 2 & 3); }

// A thread's E tokens of a chunk, four neighbours of every 4 x 256; -infinity outside the row.
template <int E>
__device__ __forceinline__ void verify_load(const float* row, int begin, int vocab, float (&l)[E]) {
  const bool aligned = (reinterpret_cast<uintptr_t>(row + begin) & 15) == 0;
#pragma unroll
  for (int j = 0; j < E / 4; ++j) {
    const int t = begin + (j * kVerifyThreads + int(threadIdx.x)) * 4;
    if (aligned && t >= 0 && t + 4 <= vocab) {
      const float4 u = *reinterpret_cast<const float4*>(row + t);
      l[4 * j] = u.x, l[4 * j + 1] = u.y, l[4 * j + 2] = u.z, l[4 * j + 3] = u.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) l[4 * j + i] = t + i >= 0 && t + i < vocab ? row[t + i] : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) l[i] = verify_logit(l[i]);
}

__device__ __forceinline__ float verify_heat(const VerifyParams& p, int s) { return p.temperature != nullptr ? p.temperature[s] : 1.0f; }
__device__ __forceinline__ float verify_draft_heat(const VerifyParams& p, int s) { return p.draft_temperature != nullptr ? p.draft_temperature[s] : verify_heat(p, s); }

constexpr int kVerifyStep = 512;  // tokens of a warp at a time: four times four per lane

// A lane's 16 tokens from `begin` on, four neighbours of every 128; -infinity outside the row.
__device__ __forceinline__ void verify_load16(const float* row, int begin, int vocab, float (&l)[16]) {
  const int lane = threadIdx.x & 31;
  const float* at = row + begin + lane * 4;
  if ((reinterpret_cast<uintptr_t>(at) & 15) == 0 && begin >= 0 && begin + kVerifyStep <= vocab) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 u = *reinterpret_cast<const float4*>(at + j * 128);
      l[4 * j] = u.x, l[4 * j + 1] = u.y, l[4 * j + 2] = u.z, l[4 * j + 3] = u.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int t = begin + i / 4 * 128 + lane * 4 + i % 4;
    l[i] = t >= 0 && t < vocab ? row[t] : -INFINITY;
  }
}

// A row's chunk of `steps` times 512 tokens by a warp: its largest logit and its sum; every lane relative to its own largest so far
__device__ __forceinline__ void verify_chunk(const float* row, int begin, int steps, int vocab, float heat, VerifySum* out) {
  const int lane = threadIdx.x & 31;
  const bool greedy = !(heat > 0.0f);
  const VerifyScale scale(greedy ? 1.0f : heat);
  VerifyWeight weight(scale, -INFINITY);
  float sums[2] = {0.0f, 0.0f}, next[16];
  int best = 0x7fffffff;
  verify_load16(row, begin, vocab, next);
#pragma unroll 1
  for (int it = 0; it < steps; ++it) {
    float l[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) l[i] = verify_logit(next[i]);
    if (it + 1 < steps) verify_load16(row, begin + (it + 1) * kVerifyStep, vocab, next);
    float top = l[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, l[i]);
    if (top > weight.top) {
      if (greedy) {
        weight.top = top;
#pragma unroll
        for (int i = 15; i >= 0; --i)
          if (l[i] == top) best = begin + it * kVerifyStep + i / 4 * 128 + lane * 4 + i % 4;
      } else {
        const VerifyWeight grown(scale, top);
        const float by = weight.far || weight.top == -INFINITY ? 0.0f : verify_ex2(weight.base - grown.base);
        sums[0] *= by;
        sums[1] *= by;
        weight = grown;
      }
    }
    if (!greedy && !weight.far) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[i & 1] += weight(l[i]);
    }
  }
  VerifySum r;
  r.top = verify_warp(weight.top, VerifyMax());
  r.sum = 0.0;
  r.best = 0x7fffffff;
  if (greedy) {
    r.best = verify_warp(weight.top == r.top ? best : 0x7fffffff, VerifyMin());
  } else if (r.top != -INFINITY) {
    if (VerifyWeight(scale, r.top).far) {  // only the largest logits weigh anything: counted
      int n = 0;
      for (int it = 0; it < steps; ++it) {
        verify_load16(row, begin + it * kVerifyStep, vocab, next);
#pragma unroll
        for (int i = 0; i < 16; ++i) n += verify_logit(next[i]) == r.top;
      }
      r.sum = verify_warp(double(n), VerifyAdd());
    } else {
      r.sum = verify_warp(double(sums[0] + sums[1]) * double(verify_rescale(scale, weight.top, r.top)), VerifyAdd());
    }
  }
  if (lane == 0) *out = r;
}

constexpr int kVerifyKnown = 1024;  // sequences whose rows a CTA keeps

// A warp has every (grid's warps)-th chunk of either side of every row
template <int E>
__global__ void __launch_bounds__(kVerifyThreads, 4) verify_sums_kernel(const VerifyParams p) {
  __shared__ int known[kVerifyKnown + 1];
  griddep_wait();
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kVerifyThreads / 32);
  if (blockIdx.x == 0)
    for (int s = threadIdx.x; s < p.sequences; s += kVerifyThreads) p.done[s] = 0;
  const int* row0 = p.row0;
  if (p.sequences <= kVerifyKnown) {
    for (int s = threadIdx.x; s <= p.sequences; s += kVerifyThreads) known[s] = p.row0[s];
    row0 = known;
    __syncthreads();
  }
  const int sides = p.draft != nullptr ? 2 : 1;
  const long long items = (long long)p.rows * p.chunks * sides;
  for (long long item = blockIdx.x * (kVerifyThreads / 32) + (threadIdx.x >> 5); item < items; item += warps) {
    const int row = int(item / (p.chunks * sides)), in = int(item - (long long)row * (p.chunks * sides)), side = in >= p.chunks, chunk = in - side * p.chunks;
    // the last sequence that begins at the row or in front of it: 32 probes at a time
    int lo = 0, hi = p.sequences;
    while (lo < hi) {
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const int c = __popc(__ballot_sync(0xffffffffu, at < hi && row0[at] <= row));
      if (c == 0) break;
      hi = min(hi, lo + c * step);
      lo = lo + (c - 1) * step + 1;
    }
    const int s = lo - 1;
    if (s < 0 || row >= row0[s + 1]) continue;  // nobody's
    const float heat = verify_heat(p, s);
    if (side == 0) {
      const float* target = p.target + row * p.ld_target;
      verify_chunk(target, verify_begin<E>(target, chunk), E * kVerifyThreads / kVerifyStep, p.vocab, heat, p.target_sum + (long long)row * p.chunks + chunk);
    } else {
      const float draft_heat = verify_draft_heat(p, s);
      if (!(heat > 0.0f) || !(draft_heat > 0.0f) || row + 1 >= row0[s + 1]) continue;
      const float* draft = p.draft + row * p.ld_draft;
      verify_chunk(draft, verify_begin<E>(draft, chunk), E * kVerifyThreads / kVerifyStep, p.vocab, draft_heat, p.draft_sum + (long long)row * p.chunks + chunk);
    }
  }
}

// a row's chunks joined, by a warp; 128 of them are read once
__device__ __forceinline__ VerifySum verify_join(const VerifySum* part, int chunks, float heat) {
  const int lane = threadIdx.x & 31;
  const VerifyScale scale(heat > 0.0f ? heat : 1.0f);
  VerifySum r;
  r.top = -INFINITY;
  r.sum = 0.0;
  r.best = 0x7fffffff;
  for (int c0 = 0; c0 < chunks; c0 += 128) {
    VerifySum x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + i * 32 + lane;
      x[i].top = -INFINITY;
      x[i].sum = 0.0;
      x[i].best = 0x7fffffff;
      if (c < chunks) x[i] = part[c];
    }
    float top = r.top;
    int best = r.best;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (x[i].top > top) top = x[i].top, best = x[i].best;  // (of equal ones the first chunk's)
    const float all = verify_warp(top, VerifyMax());
    r.best = verify_warp(top == all ? best : 0x7fffffff, VerifyMin());
    double sum = 0.0;
    if (all != -INFINITY && heat > 0.0f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += x[i].sum * double(verify_rescale(scale, x[i].top, all));
      sum = verify_warp(sum, VerifyAdd()) + r.sum * double(verify_rescale(scale, r.top, all));
    }
    r.sum = sum;
    r.top = all;
  }
  return r;
}

// The first of `chunks` at which sums exceed `want` (in the order of the chunks; else the last one whose sum is not 0) and what is left of want in it; by a warp.  of(c): its sum.
template <class Of>
__device__ __forceinline__ int verify_find_chunk(Of&& of, int chunks, double& want) {
  const int lane = threadIdx.x & 31;
  double before = 0.0, left = 0.0;
  int found = -1;
  for (int c0 = 0; c0 < chunks; c0 += 32) {
    const double x = c0 + lane < chunks ? of(c0 + lane) : 0.0;
    double up = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += t;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, x > 0.0 && before + up > want), some = __ballot_sync(0xffffffffu, x > 0.0);
    const int at = over != 0 ? __ffs(over) - 1 : some != 0 ? 31 - __clz(some) : -1;
    const double front = __shfl_sync(0xffffffffu, before + (up - x), at < 0 ? 0 : at);
    if (at >= 0) {
      found = c0 + at;
      left = over != 0 ? want - front : INFINITY;
    }
    if (over != 0) break;
    before += __shfl_sync(0xffffffffu, up, 31);
  }
  want = left;
  return found;
}

// The first token of [begin, begin + E * 256) at which the weights' sum exceeds `want`, else the last one with a weight; by the CTA.  weight(t): of token t, 0 outside the row.
template <int E, class Weight>
__device__ __forceinline__ int verify_find_token(Weight&& weight, int begin, double want, double* doubles, int* ints) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t0 = begin + int(threadIdx.x) * E;
  float w[E];
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    w[i] = weight(t0 + i);
    sum += double(w[i]);
  }
  double up = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += t;
  }
  __syncthreads();
  if (lane == 31) doubles[warp] = up;
  __syncthreads();
  double before = up - sum;
  for (int v = 0; v < warp; ++v) before += doubles[v];
  int found = 0x7fffffff, last = -1;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    before += double(w[i]);
    if (w[i] > 0.0f) {
      last = t0 + i;
      if (before > want && found == 0x7fffffff) found = t0 + i;
    }
  }
  found = verify_block(found, VerifyMin(), ints);
  last = verify_block(last, VerifyMax(), ints);
  return found != 0x7fffffff ? found : last;
}

// A token drawn from the target's own weights of a row, whose sum is `all`; `without`: a token that is not drawn (-1: none).  By the CTA.  -1: nothing to draw.
template <int E>
__device__ int verify_draw_target(const VerifyParams& p, int row, const VerifySum& all, float heat, float pick, int without, double* doubles, int* ints) {
  __shared__ double want_in;
  __shared__ int chunk_in;
  __syncthreads();
  const float* target = p.target + row * p.ld_target;
  const VerifySum* part = p.target_sum + (long long)row * p.chunks;
  const VerifyScale scale(heat);
  if (all.top == -INFINITY) return -1;
  // the chunk without its token: anew, for a difference would leave the rounding of what may be nearly all of it
  int chunk_of = -1;
  double rest = 0.0;
  if (without >= 0) {
    chunk_of = (without - verify_begin<E>(target, 0)) / (E * kVerifyThreads);
    const int begin = verify_begin<E>(target, chunk_of);
    float l[E];
    verify_load<E>(target, begin, p.vocab, l);
    const VerifyWeight weight(scale, part[chunk_of].top);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (part[chunk_of].top != -INFINITY) {
#pragma unroll
      for (int j = 0; j < E / 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (begin + (j * kVerifyThreads + int(threadIdx.x)) * 4 + i != without) sum[i] += weight(l[4 * j + i]);
    }
    rest = verify_block(double((sum[0] + sum[1]) + (sum[2] + sum[3])), VerifyAdd(), doubles);
  }
  auto of = [&](int c) { return (c == chunk_of ? rest : part[c].sum) * double(verify_rescale(scale, part[c].top, all.top)); };
  if (threadIdx.x < 32) {
    double total = 0.0;
    for (int c = threadIdx.x; c < p.chunks; c += 32) total += of(c);
    total = verify_warp(total, VerifyAdd());
    double want = double(pick) * total;
    int chunk = verify_find_chunk(of, p.chunks, want);
    if (chunk >= 0) want /= double(verify_rescale(scale, part[chunk].top, all.top));
    if (threadIdx.x == 0) want_in = want, chunk_in = chunk;
  }
  __syncthreads();
  const int chunk = chunk_in;
  if (chunk < 0) return -1;
  const VerifyWeight weight(scale, part[chunk].top);
  return verify_find_token<E>([&](int t) { return t >= 0 && t < p.vocab && t != without ? weight(verify_logit(target[t])) : 0.0f; }, verify_begin<E>(target, chunk), want_in, doubles, ints);
}

// CTA = sequence
template <int E>
__global__ void __launch_bounds__(kVerifyThreads) verify_settle_kernel(const VerifyParams p) {
  __shared__ double doubles[8];
  __shared__ int ints[8], first_stop;
  __shared__ VerifySum stop_sum;
  const int s = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) first_stop = 0x7fffffff;
  griddep_wait();
  const int first = max(p.row0[s], 0), end = min(p.row0[s + 1], p.rows);
  if (threadIdx.x == 0 && p.task != nullptr) p.task[s].row = -1;
  if (end <= first) {
    if (threadIdx.x == 0) p.accepted[s] = 0;
    return;
  }
  const float heat = verify_heat(p, s), draft_heat = verify_draft_heat(p, s);
  const bool greedy = !(heat > 0.0f), sure = p.draft == nullptr || !(draft_heat > 0.0f);
  __syncthreads();
  VerifySum a, b;  // of this warp's first row whose draft does not stay
  int mine = -1;
  a.top = b.top = -INFINITY;
  a.sum = b.sum = 0.0;
  a.best = b.best = 0x7fffffff;
  for (int row = first + warp; row < end; row += kVerifyThreads / 32) {
    const bool final = row == end - 1;
    const int x = final ? -1 : p.token[row + 1];
    const bool known = x >= 0 && x < p.vocab;
    const float logit = known ? verify_logit(p.target[row * p.ld_target + x]) : 0.0f, drafted = known && !greedy && !sure ? verify_logit(p.draft[row * p.ld_draft + x]) : 0.0f;
    a = verify_join(p.target_sum + (long long)row * p.chunks, p.chunks, heat);
    if (!final && !greedy && !sure) b = verify_join(p.draft_sum + (long long)row * p.chunks, p.chunks, draft_heat);
    bool stays = known && a.top != -INFINITY;
    if (stays && greedy) {
      stays = a.best == x;
    } else if (stays) {
      const double here = double(VerifyWeight(VerifyScale(heat), a.top)(logit)) / a.sum;
      const double there = sure ? 1.0 : b.top == -INFINITY ? 0.0 : double(VerifyWeight(VerifyScale(draft_heat), b.top)(drafted)) / b.sum;
      stays = double(p.accept_u[row]) * there < here;
    }
    if (!stays) {
      mine = row;
      if (lane == 0) atomicMin(&first_stop, row);
      break;
    }
  }
  __syncthreads();
  const int stop = first_stop;
  for (int row = first + threadIdx.x; row < end; row += kVerifyThreads)
    if (row != stop) p.emitted[row] = row < stop ? p.token[row + 1] : -1;
  if (threadIdx.x == 0) p.accepted[s] = stop - first;
  const bool final = stop == end - 1;
  if (!greedy && (final || sure)) {
    if (mine == stop && lane == 0) stop_sum = a;
    __syncthreads();
    const int x = final ? -1 : p.token[stop + 1];
    int drawn = -1;
#pragma unroll 1
    for (int without = x >= 0 && x < p.vocab ? x : -1;; without = -1) {
      drawn = verify_draw_target<E>(p, stop, stop_sum, heat, p.pick_u[s], without, doubles, ints);
      if (drawn >= 0 || without < 0) break;  // (otherwise the draft is all that the target may say)
    }
    if (threadIdx.x == 0) p.emitted[stop] = drawn;
  } else if (mine == stop && lane == 0) {
    p.emitted[stop] = greedy && a.top != -INFINITY ? a.best : -1;
    if (!greedy && a.top != -INFINITY) {
      VerifyTask task;
      task.row = stop;
      task.target = a;
      task.draft = b;
      p.task[s] = task;
    }
  }
}

// max(p - q, 0) of a row's tokens, in p's weights: t - d (sum of p's weights / sum of q's), that factor in two parts, so that what both weigh alike cancels to the last bit (as products with 1 / sum
// of either side, each rounded, a difference of 10^-4 of p drew its tokens by up to 2^-15 of it beside)
struct VerifyDifference {
  VerifyWeight target, draft;
  float hi, lo;

  __device__ __forceinline__ VerifyDifference(const VerifyTask& t, float heat, float draft_heat) : target(VerifyScale(heat), t.target.top), draft(VerifyScale(draft_heat), t.draft.top) {
    const double by = t.draft.top == -INFINITY ? 0.0 : t.target.sum / t.draft.sum;
    hi = float(by);
    lo = float(by - double(hi));
  }
  __device__ __forceinline__ float operator()(float l, float d) const {
    const float w = draft(d);
    return fmaxf(fmaf(-w, lo, fmaf(-w, hi, target(l))), 0.0f);
  }
};

// CTA = (eight chunks of D * 256 tokens, a warp each; sequence), the last sequences first: their rows are what the first kernel has left in L2
template <int E, int D>
__global__ void __launch_bounds__(kVerifyThreads, 3) verify_difference_kernel(const VerifyParams p) {
  __shared__ double doubles[8], want_in;
  __shared__ int ints[8], is_last, chunk_in;
  griddep_launch_dependents();
  griddep_wait();
  const int s = p.sequences - 1 - int(blockIdx.y), chunk = blockIdx.x * (kVerifyThreads / 32) + int(threadIdx.x >> 5);
  const VerifyTask task = p.task[s];
  if (task.row < 0) return;
  const float heat = verify_heat(p, s), draft_heat = verify_draft_heat(p, s);
  const float *target = p.target + task.row * p.ld_target, *draft = p.draft + task.row * p.ld_draft;
  const VerifyDifference weight(task, heat, draft_heat);
  if (chunk < p.left_chunks) {
    constexpr int kSteps = D * kVerifyThreads / kVerifyStep;
    const int begin = verify_begin<D>(target, chunk);
    float l[16], d[16];
    double sum = 0.0;
    verify_load16(target, begin, p.vocab, l);
    verify_load16(draft, begin, p.vocab, d);
#pragma unroll 1
    for (int it = 0; it < kSteps; ++it) {
      float part[2] = {0.0f, 0.0f};
      float x[16], y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = l[i], y[i] = d[i];
      if (it + 1 < kSteps) {
        verify_load16(target, begin + (it + 1) * kVerifyStep, p.vocab, l);
        verify_load16(draft, begin + (it + 1) * kVerifyStep, p.vocab, d);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) part[i & 1] += weight(verify_logit(x[i]), verify_logit(y[i]));
      sum += double(part[0] + part[1]);
    }
    sum = verify_warp(sum, VerifyAdd());
    if ((threadIdx.x & 31) == 0) {
      p.left[(long long)s * p.left_chunks + chunk] = sum;
      __threadfence();
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    is_last = atomicAdd(&p.done[s], 1) == int(gridDim.x) - 1;
    __threadfence();
  }
  __syncthreads();
  if (!is_last) return;
  const double* left = p.left + (long long)s * p.left_chunks;
  if (threadIdx.x < 32) {
    double total = 0.0;
    for (int c = threadIdx.x; c < p.left_chunks; c += 32) total += __ldcg(left + c);
    total = verify_warp(total, VerifyAdd());
    double want = double(p.pick_u[s]) * total;
    const int found = verify_find_chunk([&](int c) { return __ldcg(left + c); }, p.left_chunks, want);
    if (threadIdx.x == 0) want_in = want, chunk_in = found;
  }
  __syncthreads();
  int drawn;
  if (chunk_in >= 0)
    drawn = verify_find_token<D>([&](int t) { return t >= 0 && t < p.vocab ? weight(verify_logit(target[t]), verify_logit(draft[t])) : 0.0f; }, verify_begin<D>(target, chunk_in), want_in,
                                 doubles, ints);
  else  // (no difference that 32 bits show: the target's own)
    drawn = verify_draw_target<E>(p, task.row, task.target, heat, p.pick_u[s], -1, doubles, ints);
  if (threadIdx.x == 0) p.emitted[task.row] = drawn;
}

}  // namespace mtx
