// Drafted tokens against the target's probabilities (simple form).
#pragma once

#include "common.cuh"

namespace mtx {

struct VerifyParams {
  int rows, sequences, vocab;
  const int *row0, *token;
  const float* target;
  long long ld_target;
  const float* draft;
  long long ld_draft;
  const float *temperature, *draft_temperature, *accept_u, *pick_u;
  int *accepted, *emitted;
};

constexpr int kVerifyThreads = 1024;

// a logit as it counts: NaN as -infinity, infinity as the largest number
__device__ __forceinline__ float verify_logit(float l) { return l != l ? -INFINITY : fminf(l, 3.402823466e38f); }

template <class T, class F>
__device__ __forceinline__ T verify_reduce(T v, F&& join, T* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// CTA = sequence
__global__ void __launch_bounds__(kVerifyThreads) verify_simple_kernel(const VerifyParams p) {
  __shared__ double sums[32];
  __shared__ int ints[32];
  griddep_launch_dependents();
  griddep_wait();
  const int s = blockIdx.x, tid = threadIdx.x, V = p.vocab;
  const int first = max(p.row0[s], 0), end = min(p.row0[s + 1], p.rows);
  if (end <= first) {
    if (tid == 0) p.accepted[s] = 0;
    return;
  }
  const float heat = p.temperature != nullptr ? p.temperature[s] : 1.0f, draft_heat = p.draft_temperature != nullptr ? p.draft_temperature[s] : heat;
  const bool greedy = !(heat > 0.0f), sure = p.draft == nullptr || !(draft_heat > 0.0f);
  auto add = [](double a, double b) { return a + b; };
  auto more = [](double a, double b) { return a > b ? a : b; };
  auto less = [](int a, int b) { return a < b ? a : b; };
  auto later = [](int a, int b) { return a > b ? a : b; };
  struct Stat { double top, sum; };
  auto stat = [&](const float* l, float t) {
    double top = -INFINITY, sum = 0.0;
    for (int i = tid; i < V; i += kVerifyThreads) top = more(top, double(verify_logit(l[i])));
    top = verify_reduce(top, more, sums);
    if (top == -INFINITY || !(t > 0.0f)) return Stat{top, 0.0};
    for (int i = tid; i < V; i += kVerifyThreads) sum += exp((double(verify_logit(l[i])) - top) / t);
    return Stat{top, verify_reduce(sum, add, sums)};
  };
  int row = first;
  for (;; ++row) {
    const float *l = p.target + row * p.ld_target, *d = sure ? nullptr : p.draft + row * p.ld_draft;
    const bool final = row == end - 1;
    const int x = final ? -1 : p.token[row + 1];
    const Stat a = stat(l, heat);
    const bool known = x >= 0 && x < V;
    if (greedy) {
      int best = V;
      if (a.top != -INFINITY)
        for (int i = tid; i < V; i += kVerifyThreads)
          if (double(verify_logit(l[i])) == a.top) best = min(best, i);
      best = verify_reduce(best, less, ints);
      if (!final && known && best == x) {
        if (tid == 0) p.emitted[row] = x;
        continue;
      }
      if (tid == 0) p.emitted[row] = best < V ? best : -1;
      break;
    }
    const Stat b = final || sure ? Stat{0.0, 0.0} : stat(d, draft_heat);
    auto prob = [&](int i) { return a.top == -INFINITY ? 0.0 : exp((double(verify_logit(l[i])) - a.top) / heat) / a.sum; };
    auto drafted = [&](int i) { return b.top == -INFINITY ? 0.0 : exp((double(verify_logit(d[i])) - b.top) / draft_heat) / b.sum; };
    if (!final && known && double(p.accept_u[row]) * (sure ? 1.0 : drafted(x)) < prob(x)) {
      if (tid == 0) p.emitted[row] = x;
      continue;
    }
    int out = -1;
    for (int plain = 0; plain < 2 && out < 0; ++plain) {  // (what is left may be nothing: then the target's own)
      auto weight = [&](int i) {
        const double w = prob(i);
        if (plain || final) return w;
        if (sure) return i == x ? 0.0 : w;
        return w > drafted(i) ? w - drafted(i) : 0.0;
      };
      // a thread has neighbouring tokens
      const int each = (V + kVerifyThreads - 1) / kVerifyThreads, i0 = min(tid * each, V), i1 = min(i0 + each, V);
      double sum = 0.0;
      for (int i = i0; i < i1; ++i) sum += weight(i);
      double before = sum;  // inclusive sums over the threads
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, before, o);
        if ((tid & 31) >= o) before += t;
      }
      __syncthreads();
      if ((tid & 31) == 31) sums[tid >> 5] = before;
      __syncthreads();
      double base = 0.0, total = 0.0;
      for (int w = 0; w < 32; ++w) {
        if (w < tid >> 5) base += sums[w];
        total += sums[w];
      }
      before = base + before - sum;
      const double want = double(p.pick_u[s]) * total;
      int found = V, last = -1;
      for (int i = i0; i < i1; ++i) {
        const double w = weight(i);
        before += w;
        if (w > 0.0) {
          last = i;
          if (before > want) found = min(found, i);
        }
      }
      found = verify_reduce(found, less, ints);
      last = verify_reduce(last, later, ints);
      out = found < V ? found : last;
    }
    if (tid == 0) p.emitted[row] = out;
    break;
  }
  if (tid == 0) p.accepted[s] = row - first;
  for (int r = row + 1 + tid; r < end; r += kVerifyThreads) p.emitted[r] = -1;
}

}  // namespace mtx
