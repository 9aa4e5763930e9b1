// Attention of a batch's last rows over the paged cache, where neighbouring sequences share the first tokens of their contexts (simple form).
#pragma once

#include "common.cuh"

namespace mtx {

struct PrefixAttnParams {
  const bf16* q;
  long long ldq;
  const bf16 *k, *v;
  bf16* out;
  long long ldo;
  int rows, sequences, prefixes;
  const int *row0, *lengths, *page_map, *prefix_seq0, *prefix_len;
  int heads, kv_heads, num_pages, tokens_per_page, max_pages;
  float scale, softcap;
};

// CTA = (row, query head); warps take every fourth key, lanes D / 32 channels each
template <int D>
__global__ void __launch_bounds__(128) prefix_simple_kernel(const PrefixAttnParams p) {
  constexpr int E = D / 32;
  __shared__ float sm[4], sl[4], so[4][D];
  griddep_launch_dependents();
  griddep_wait();
  const int row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = head / (p.heads / p.kv_heads);
  int s = -1;
  for (int i = 0; i < p.sequences; ++i)
    if (p.row0[i] <= row && row < p.row0[i + 1]) s = i;
  if (s < 0) return;
  const int most = p.max_pages * p.tokens_per_page;
  int seen = p.lengths[s] - (p.row0[s + 1] - row) + 1;
  if (seen > most) seen = most;
  if (seen <= 0) return;
  float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
  for (int e = 0; e < E; ++e) q[e] = __bfloat162float(p.q[row * p.ldq + head * D + lane * E + e]) * p.scale;
  for (int j = warp; j < seen; j += 4) {
    const unsigned page = p.page_map[(long long)s * p.max_pages + j / p.tokens_per_page];
    const long long at = (((long long)kvh * p.num_pages + (page < unsigned(p.num_pages) ? page : 0)) * p.tokens_per_page + j % p.tokens_per_page) * D + lane * E;
    float x = 0.0f;
    for (int e = 0; e < E; ++e) x = fmaf(q[e], __bfloat162float(p.k[at + e]), x);
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    if (p.softcap > 0.0f) x = tanhf(x / p.softcap) * p.softcap;
    const float top = fmaxf(m, x), fix = __expf(m - top), w = __expf(x - top);
    l = l * fix + w;
    m = top;
    for (int e = 0; e < E; ++e) o[e] = o[e] * fix + w * __bfloat162float(p.v[at + e]);
  }
  sm[warp] = m;
  sl[warp] = l;
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], sum = 0.0f;
  for (int w = 0; w < 4; ++w) f[w] = sm[w] == -INFINITY ? 0.0f : __expf(sm[w] - top), sum += f[w] * sl[w];
  for (int c = threadIdx.x; c < D; c += 128) {
    float x = 0.0f;
    for (int w = 0; w < 4; ++w) x += f[w] == 0.0f ? 0.0f : f[w] * so[w][c];
    p.out[row * p.ldo + head * D + c] = __float2bfloat16_rn(x / sum);
  }
}

}  // namespace mtx
