// Attention of a batch's last rows over the paged cache, where neighbouring sequences share the first tokens of their contexts.
//
//   row i of the n rows of sequence s:  out = sum_j softmax_j(cap(scale <q, k_j>)) v_j,  j < lengths[s] - n + i + 1
//
// The keys of a prefix are the same for all rows of its sequences, so that one pass over them serves all: work is cut into ENTRIES, a prefix (all rows of its sequences; its
// tokens) or the tail of a sequence (its own rows; the tokens behind its prefix).  An entry's (row, query head of the key head) pairs lie side by side, an ITEM is a block
// of them over the entry's tokens, a UNIT one tile of tokens of an item.  The CTAs share all units evenly, in order: a CTA goes through a contiguous run, leaves the partial results
// of each item in it (running maximum, sum, weighted values), and a second kernel joins a row's parts in the order of the tokens.  So a batch of one long sequence
// fills the GPU like one of many short ones, and the same call always adds in the same order.
#pragma once

#include "flash_tmem.cuh"

namespace mtx {

struct PrefixAttnParams {
  const bf16* q;
  long long ldq;
  const bf16 *k, *v;
  bf16* out;
  long long ldo;
  int rows, sequences, prefixes;
  const int *row0, *lengths, *page_map, *prefix_seq0, *prefix_len;
  int heads, kv_heads, group, num_pages, tokens_per_page, max_pages;
  float scale, softcap;
  int box;  // tokens of a copy: a page, or a part of one, at most a tile
};

// Entries that one kernel goes through, and where its results are.
struct PrefixWork {
  int first, count;  // the entries: prefixes, then sequences
  int kt, pairs;     // tokens of a tile, pairs of an item
  int workers;       // CTAs that share the units, at most
  int tabled;        // the table is there already (more entries than a CTA keeps)
  float* part;       // [place][D]: weighted values
  float2* stat;      // [place]: maximum (of the scores times log2 e) and sum
  struct PrefixEntry* table;  // [count + 1], for the join
};

// What a CTA needs of an entry.  The one behind the last holds the sums.
struct PrefixEntry {
  int row, rows;        // the first, and how many
  int key0, key1;       // its tokens
  int first_seen;       // tokens that the first row sees (the next row one more, at most key1)
  int map;              // the page map's row
  int pairs;            // pairs of one key head in the entries before
  int prefix;           // a tail's prefix where it begins behind one, else -1
  long long units;      // units of one key head in the entries before
};

constexpr float kPrefixLog2e = 1.4426950408889634f;
constexpr int kPrefixPairs = 32;      // pairs of an item: two MMA tiles
constexpr int kPrefixCached = 128;    // entries that a CTA keeps in shared memory
constexpr int kPrefixWarps = 4;       // that compute; one more copies
constexpr int kPrefixThreads = 32 * (kPrefixWarps + 1);
constexpr int kPrefixPieces = 5;      // K or V tiles in flight, 16 KB each
constexpr int kPrefixPieceBytes = 16384;

template <int D>
struct PrefixShape {
  static constexpr int KT = 8192 / D;               // tokens of a tile
  static constexpr int CH = D / 64;                 // 64-channel chunks of a row
  static constexpr int kKeys = KT / kPrefixWarps;   // a warp's tokens of a tile (its part of S)
  static constexpr int kCols = D / kPrefixWarps;    // a warp's channels (its part of P V)
  static constexpr int kPRow = KT * 2 + 16;         // bytes of a row of P: 16 more than its values, so that eight rows lie in different banks
};

struct PrefixTail {
  PrefixEntry entry[kPrefixCached + 1];
  uint64_t full[kPrefixPieces], empty[kPrefixPieces];
  alignas(16) float top[2][kPrefixPairs][kPrefixWarps];
  alignas(16) float sum[kPrefixPairs][kPrefixWarps];
  int not_finite[2];
  int failed;
};

template <int D>
constexpr size_t prefix_smem_bytes() {
  return 1024 + size_t(kPrefixPieces) * kPrefixPieceBytes + kPrefixPairs * D * 2 + kPrefixPairs * PrefixShape<D>::kPRow + sizeof(PrefixTail) + 16;
}

// ---- waits -----------------------------------------------------------------------------------------------------------------------
// A wait that lasts some two seconds is a protocol error: it gives up, then so does every other wait of the CTA, and the counter (mtx_prefix_attention_stalls) says that results are wrong.
__device__ unsigned int d_prefix_waits_failed = 0;

__device__ __forceinline__ bool prefix_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  do {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (clock64() - t0 > 4000000000LL) {
      atomicAdd(&d_prefix_waits_failed, 1u);
      *failed = 1;
    }
  } while (*failed == 0);
  return false;
}

// ---- the entries -----------------------------------------------------------------------------------------------------------------

// entry e without its sums; `kt` tokens a tile
__device__ __forceinline__ PrefixEntry prefix_entry(const PrefixAttnParams& p, int e) {
  const int most = p.max_pages * p.tokens_per_page;
  auto row_of = [&](int s) { return min(max(p.row0[s], 0), p.rows); };
  auto seq_of = [&](int i) { return min(max(p.prefix_seq0[i], 0), p.sequences); };
  PrefixEntry x;
  x.pairs = 0;
  x.units = 0;
  x.prefix = -1;
  if (e < p.prefixes) {
    const int s0 = seq_of(e), s1 = max(seq_of(e + 1), s0);
    x.row = row_of(s0);
    x.rows = s1 > s0 ? max(row_of(s1) - x.row, 0) : 0;
    x.key0 = 0;
    x.key1 = min(max(p.prefix_len[e], 0), most);
    x.first_seen = x.key1;
    x.map = s0 < p.sequences ? s0 : 0;
  } else {
    const int s = e - p.prefixes;
    x.row = row_of(s);
    x.rows = max(row_of(s + 1) - x.row, 0);
    const int length = p.lengths[s];
    x.key1 = min(max(length, 0), most);
    x.first_seen = length - x.rows + 1;  // (lengths and rows are far from 2^31 together: a length below -2^30 counts as none)
    if (length < 0) x.first_seen = -(1 << 30);
    x.map = s;
    x.key0 = 0;
    // the prefix: the last one that begins at s or in front of it
    int lo = 0, hi = p.prefixes;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (seq_of(mid) <= s) lo = mid + 1;
      else hi = mid;
    }
    if (lo > 0 && s < seq_of(lo)) {
      const int shared = min(max(p.prefix_len[lo - 1], 0), most);
      if (shared > 0 && x.first_seen > shared) x.key0 = shared, x.prefix = lo - 1;  // every row lies behind the prefix; otherwise the sequence reads its own pages throughout
    }
  }
  
  return x;
}

// a tile begins where a copy may: at key0 rounded down to one
__device__ __forceinline__ int prefix_first(const PrefixEntry& x, int box) { return x.key0 & ~(box - 1); }
__device__ __forceinline__ int prefix_tiles(const PrefixEntry& x, int kt, int box) { return x.rows > 0 && x.key1 > x.key0 ? (x.key1 - prefix_first(x, box) + kt - 1) / kt : 0; }

// All of a work's entries with their sums, by `threads` threads (whole warps, at most 1024) of a CTA; carry: two words of shared memory per warp.
__device__ __forceinline__ void prefix_build_table(const PrefixAttnParams& p, const PrefixWork& k, PrefixEntry* table, long long* carry, int tid, int threads) {
  const int lane = tid & 31, warp = tid >> 5, total = k.count;
  long long units = 0;
  int pairs = 0;
  for (int e0 = 0; e0 <= total; e0 += threads) {
    const int e = e0 + tid;
    PrefixEntry x;
    long long u = 0;
    int b = 0;
    if (e < total) {
      x = prefix_entry(p, k.first + e);
      const int tiles = prefix_tiles(x, k.kt, p.box);
      b = tiles > 0 ? x.rows * p.group : 0;
      u = (long long)tiles * ((b + k.pairs - 1) / k.pairs);
    } else {
      x.row = x.rows = x.key0 = x.key1 = x.first_seen = x.map = 0;
      x.prefix = -1;
    }
    long long us = u;
    int bs = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, us, o);
      const int w = __shfl_up_sync(0xffffffffu, bs, o);
      if (lane >= o) us += t, bs += w;
    }
    __syncthreads();
    if (lane == 31) carry[2 * warp] = us, carry[2 * warp + 1] = bs;
    __syncthreads();
    long long before = units, sum_u = 0;
    int before_b = pairs, sum_b = 0;
    for (int w = 0; w < threads / 32; ++w) {
      if (w < warp) before += carry[2 * w], before_b += int(carry[2 * w + 1]);
      sum_u += carry[2 * w], sum_b += int(carry[2 * w + 1]);
    }
    if (e <= total) {
      x.units = before + us - u;
      x.pairs = before_b + bs - b;
      table[e] = x;
    }
    units += sum_u;
    pairs += sum_b;
  }
  __syncthreads();
}

// for batches of more entries than a CTA keeps: one CTA in front of the others
__global__ void __launch_bounds__(1024) prefix_plan_kernel(const PrefixAttnParams p, const PrefixWork a, const PrefixWork b) {
  __shared__ long long carry[64];
  griddep_wait();
  griddep_launch_dependents();
  if (a.tabled) prefix_build_table(p, a, a.table, carry, threadIdx.x, 1024);
  if (b.tabled) prefix_build_table(p, b, b.table, carry, threadIdx.x, 1024);
}

// A CTA's run of units: worker c of W has those from begin(c) on.
struct PrefixShare {
  long long units;  // of all key heads
  int workers;

  __device__ __forceinline__ PrefixShare(long long u, int most) : units(u), workers(u < most ? int(u) : most) {}
  __device__ __forceinline__ long long begin(int c) const { return units / workers * c + units % workers * c / workers; }
  __device__ __forceinline__ int of(long long u) const {  // the worker that has unit u
    int c = int(double(u) * workers / double(units));
    c = min(max(c, 0), workers - 1);
    while (c > 0 && begin(c) > u) --c;
    while (c + 1 < workers && begin(c + 1) <= u) ++c;
    return c;
  }
};

// One item of a CTA's run: its tiles [tile0, tile1).
struct PrefixSegment {
  PrefixEntry x;
  int e, kvh, block, tiles, tile0, tile1;
  int first;        // the first tile's first token
  long long place;  // of its first pair's results
};

// Goes through a CTA's run item by item; all threads of a warp alike.
struct PrefixWalk {
  const PrefixEntry* table;
  int total, kt, box, most, worker;
  long long per_head, at, end;
  int e, kvh;

  __device__ __forceinline__ PrefixWalk(const PrefixAttnParams& p, const PrefixWork& k, const PrefixEntry* t, const PrefixShare& share, int c)
      : table(t), total(k.count), kt(k.kt), box(p.box), most(k.pairs), worker(c) {
    per_head = t[total].units;
    at = share.begin(c);
    end = share.begin(c + 1);
    kvh = int(at / per_head);
    const long long rest = at - kvh * per_head;
    int lo = 0, hi = total;  // the last entry whose units begin at `rest` or before (entries without units are in front of it)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (t[mid].units <= rest) lo = mid;
      else hi = mid;
    }
    e = lo;
  }
  __device__ __forceinline__ bool next(PrefixSegment& s) {
    if (at >= end) return false;
    long long rest = at - kvh * per_head;
    if (rest >= per_head) ++kvh, rest = 0, e = 0;
    while (table[e + 1].units <= rest) ++e;
    s.x = table[e];
    s.e = e;
    s.kvh = kvh;
    s.tiles = prefix_tiles(s.x, kt, box);
    s.first = prefix_first(s.x, box);
    const long long in = rest - s.x.units;
    s.block = int(in / s.tiles);
    s.tile0 = int(in - (long long)s.block * s.tiles);
    s.tile1 = int(min((long long)s.tiles, s.tile0 + (end - at)));
    s.place = (long long)kvh * table[total].pairs + s.x.pairs + (long long)(s.block + worker) * most;  // (every step to the next one goes to another item, another CTA or both)
    at += s.tile1 - s.tile0;
    return true;
  }
};

__device__ __forceinline__ bool prefix_whole(const PrefixSegment& s) { return s.x.key0 == 0 && s.tile0 == 0 && s.tile1 == s.tiles; }

// ---- units on the warps' MMAs ------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void prefix_bar() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kPrefixWarps) : "memory"); }

// Warp 4 copies K and V tiles, warps 0 to 3 compute: of every tile each has a quarter of the tokens for S = Q K^T and a quarter of the channels for P V, so that no accumulators
// have to be joined; maxima and P pass through shared memory, two barriers a tile.
template <int D>
__global__ void __launch_bounds__(kPrefixThreads, 2)
prefix_units_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PrefixAttnParams p, const PrefixWork k) {
  typedef PrefixShape<D> F;
  constexpr int KT = F::KT, CH = F::CH, NS = F::kKeys / 8, NO = F::kCols / 8, MT = kPrefixPairs / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // piece: [CH][KT tokens][128 B], swizzled
  uint8_t* sq = ring + kPrefixPieces * kPrefixPieceBytes;                        // [CH][pairs][128 B], swizzled alike
  uint8_t* sp = sq + kPrefixPairs * D * 2;                                       // [pairs][kPRow]
  PrefixTail* tail = reinterpret_cast<PrefixTail*>(sp + kPrefixPairs * F::kPRow);
  volatile int* failed = &tail->failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int i = 0; i < kPrefixPieces; ++i) {
      mbar_init(&tail->full[i], 1);
      mbar_init(&tail->empty[i], kPrefixWarps);
    }
    tail->failed = 0;
    tail->not_finite[0] = tail->not_finite[1] = 0;
    fence_barrier_init();
  }
  // (behind the prefixes' kernel: that one has waited for what is in front of it, and the join waits for this one, which waits for that one before it ends)
  if (k.first == 0 || k.tabled) griddep_wait();
  griddep_launch_dependents();
  const PrefixEntry* table = k.table;
  if (!k.tabled) {
    prefix_build_table(p, k, tail->entry, reinterpret_cast<long long*>(sp), threadIdx.x, kPrefixThreads);
    table = tail->entry;
    if (blockIdx.x == 0)  // for the join
      for (int e = threadIdx.x; e <= k.count; e += kPrefixThreads) k.table[e] = table[e];
  } else {
    __syncthreads();
  }
  const PrefixShare share(table[k.count].units * p.kv_heads, k.workers);
  if (int(blockIdx.x) >= share.workers) {
    griddep_wait();
    return;
  }
  PrefixWalk walk(p, k, table, share, blockIdx.x);
  PrefixSegment s;

  if (warp == kPrefixWarps) {
    const bool issuer = elect_one();
    const int boxes = KT / p.box, tpp = p.tokens_per_page;
    int piece = 0;
    uint32_t phase = 1;
    bool good = true;
    while (walk.next(s)) {
      const int* pages = p.page_map + (long long)s.x.map * p.max_pages;
      const long long head_row = (long long)s.kvh * p.num_pages * tpp;
      // lane i: the pool's row where box i of the tile begins; boxes behind the last token: that token's page
      auto row_of = [&](int tile) {
        const int key = min(s.first + tile * KT + (lane < boxes ? lane : 0) * p.box, s.x.key1 - 1);
        const int page = pages[key / tpp];
        return int(head_row + (long long)(page >= 0 && page < p.num_pages ? page : 0) * tpp + key % tpp / p.box * p.box);
      };
      int row = row_of(s.tile0);
      for (int t = s.tile0; t < s.tile1; ++t) {
        const int next = t + 1 < s.tile1 ? row_of(t + 1) : 0;
        for (int kv = 0; kv < 2; ++kv) {
          good = good && prefix_wait(&tail->empty[piece], phase, failed);
          uint8_t* to = ring + piece * kPrefixPieceBytes;
          if (issuer && good) mbar_expect_tx(&tail->full[piece], kPrefixPieceBytes);
          for (int b = 0; b < boxes; ++b) {
            const int from = __shfl_sync(0xffffffffu, row, b);
            if (issuer && good)
              for (int c = 0; c < CH; ++c) tma_load_2d(to + c * KT * 128 + b * p.box * 128, kv == 0 ? &tm_k : &tm_v, c * 64, from, &tail->full[piece], kEvictNormal);
          }
          if (++piece == kPrefixPieces) piece = 0, phase ^= 1;
        }
        row = next;
      }
    }
    if (!good) {  // copies in flight have a millisecond to end
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000) __nanosleep(1000);
    }
    griddep_wait();
    return;
  }

  const float mul = p.softcap > 0.0f ? p.scale / p.softcap : p.scale * kPrefixLog2e, cap = p.softcap * kPrefixLog2e;
  const int r = lane >> 2;  // this lane's pairs of an MMA tile: r and r + 8
  const uint32_t sq_addr = smem_u32(sq), sp_addr = smem_u32(sp), ring_addr = smem_u32(ring);
  int piece = 0;
  uint32_t phase = 0;
  int turn = 0;  // which buffer of maxima
  while (walk.next(s)) {
    const int pair0 = s.block * kPrefixPairs, pairs = min(kPrefixPairs, s.x.rows * p.group - pair0), mts = (pairs + 15) / 16;
    prefix_bar();  // (the item before has left Q and the sums)
    for (int i = threadIdx.x; i < mts * 16 * (D / 8); i += 32 * kPrefixWarps) {
      const int pair = i / (D / 8), c = i - pair * (D / 8), at = pair0 + pair;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (pair < pairs) v = *reinterpret_cast<const uint4*>(p.q + (s.x.row + at / p.group) * p.ldq + (s.kvh * p.group + at % p.group) * D + c * 8);
      *reinterpret_cast<uint4*>(sq + (c >> 3) * kPrefixPairs * 128 + pair * 128 + (((c & 7) ^ (pair & 7)) << 4)) = v;
    }
    int seen[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) seen[mt][h] = k.first + s.e < p.prefixes ? s.x.key1 : min(s.x.first_seen + (pair0 + mt * 16 + r + 8 * h) / p.group, s.x.key1);
    float m[MT][2], l[MT][2], o[MT][NO][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) m[mt][h] = -INFINITY, l[mt][h] = 0.0f;
#pragma unroll
      for (int n = 0; n < NO; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.0f;
    }
    prefix_bar();
    for (int t = s.tile0; t < s.tile1; ++t) {
      const int key = s.first + t * KT;  // the tile's first token
      const bool masked = key < s.x.key0 || key + KT > min(s.x.first_seen, s.x.key1);
      // S of this warp's tokens
      prefix_wait(&tail->full[piece], phase, failed);
      float x[MT][NS][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[mt][n][i] = 0.0f;
      const uint32_t k_addr = ring_addr + piece * kPrefixPieceBytes;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t a[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          if (mt < mts) {
            const int pair = mt * 16 + (lane & 15), c = kk % 4 * 2 + (lane >> 4);
            ldmatrix_x4(sq_addr + kk / 4 * kPrefixPairs * 128 + pair * 128 + ((c ^ (pair & 7)) << 4), a[mt][0], a[mt][1], a[mt][2], a[mt][3]);
          }
#pragma unroll
        for (int n = 0; n < NS; n += 2) {
          uint32_t b[4];
          if (NS == 1) {  // eight tokens: the two halves of 16 channels
            const int token = warp * F::kKeys + (lane & 7), c = kk % 4 * 2 + (lane >> 3 & 1);
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(b[0]), "=r"(b[1]) : "r"(k_addr + kk / 4 * KT * 128 + token * 128 + ((c ^ (token & 7)) << 4)) : "memory");
            b[2] = b[3] = 0;
          } else {
            const int token = warp * F::kKeys + n * 8 + (lane & 7) + (lane >> 4) * 8, c = kk % 4 * 2 + (lane >> 3 & 1);
            ldmatrix_x4(k_addr + kk / 4 * KT * 128 + token * 128 + ((c ^ (token & 7)) << 4), b[0], b[1], b[2], b[3]);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            if (mt < mts) {
              mma_m16n8k16_bf16(x[mt][n], a[mt], b[0], b[1]);
              if (NS > 1) mma_m16n8k16_bf16(x[mt][n + (NS > 1)], a[mt], b[2], b[3]);
            }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&tail->empty[piece]);
      if (++piece == kPrefixPieces) piece = 0, phase ^= 1;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        if (mt < mts) {
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float& v = x[mt][n][i];
              v *= mul;
              if (p.softcap > 0.0f) v = cap * tanhf(v);
              if (masked) {
                const int j = key + warp * F::kKeys + n * 8 + (lane & 3) * 2 + (i & 1);
                if (j < s.x.key0 || j >= seen[mt][i >> 1]) v = -INFINITY;
              }
              top[i >> 1] = fmaxf(top[i >> 1], v);
            }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            if ((lane & 3) == 0) tail->top[turn][mt * 16 + r + 8 * h][warp] = top[h];
          }
        }
      // V: tokens outside the entry's count 0 whatever they hold.  So do numbers that are none, in tokens that some rows see and others do not (0 times them is none either); the rows that see them
      // add them behind the products
      prefix_wait(&tail->full[piece], phase, failed);
      uint8_t* v = ring + piece * kPrefixPieceBytes;
      const int some = max(s.x.first_seen - key, 0), hi = s.x.key1 - key;  // of the tile, tokens that not all rows see
      if (masked) {
        const int lo = s.x.key0 - key;
        bool odd = false;
        for (int i = threadIdx.x; i < KT * (D / 8); i += 32 * kPrefixWarps) {
          const int token = i / (D / 8), c = i - token * (D / 8);
          uint4* at = reinterpret_cast<uint4*>(v + (c >> 3) * KT * 128 + token * 128 + ((c & 7) << 4));  // (any order of a row's pieces)
          if (token < lo || token >= hi) {
            *at = make_uint4(0, 0, 0, 0);
          } else if (token >= some) {
            const uint4 u = *at;
            uint32_t w[4] = {u.x, u.y, u.z, u.w}, gone = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const uint32_t none = ((w[b] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w[b] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
              w[b] &= ~none;
              gone |= none;
            }
            if (gone != 0) {
              *at = make_uint4(w[0], w[1], w[2], w[3]);
              odd = true;
            }
          }
        }
        if (odd) tail->not_finite[turn] = 1;
      }
      prefix_bar();
      const bool odd_tile = masked && *reinterpret_cast<volatile int*>(&tail->not_finite[turn]) != 0;
      if (threadIdx.x == 0) tail->not_finite[turn ^ 1] = 0;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        if (mt < mts) {
          float base[2], fix[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 u = *reinterpret_cast<const float4*>(tail->top[turn][mt * 16 + r + 8 * h]);
            const float now = fmaxf(m[mt][h], fmaxf(fmaxf(u.x, u.y), fmaxf(u.z, u.w)));
            base[h] = now == -INFINITY ? 0.0f : now;
            fix[h] = exp2f(m[mt][h] - base[h]);
            m[mt][h] = now;
            l[mt][h] *= fix[h];
          }
#pragma unroll
          for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float p0 = exp2f(x[mt][n][2 * h] - base[h]), p1 = exp2f(x[mt][n][2 * h + 1] - base[h]);
              l[mt][h] += p0 + p1;
              *reinterpret_cast<uint32_t*>(sp + (mt * 16 + r + 8 * h) * F::kPRow + (warp * F::kKeys + n * 8 + (lane & 3) * 2) * 2) = pack_bf16x2(p0, p1);
            }
          }
#pragma unroll
          for (int n = 0; n < NO; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[mt][n][i] *= fix[i >> 1];
        }
      prefix_bar();
      // P V: this warp's channels
      const uint32_t v_addr = ring_addr + piece * kPrefixPieceBytes;
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk) {
        uint32_t a[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          if (mt < mts) ldmatrix_x4(sp_addr + (mt * 16 + (lane & 15)) * F::kPRow + kk * 32 + (lane >> 4) * 16, a[mt][0], a[mt][1], a[mt][2], a[mt][3]);
#pragma unroll
        for (int n = 0; n < NO; n += 2) {
          const int token = kk * 16 + (lane & 15), c = warp * (F::kCols / 8) + n + (lane >> 4);
          uint32_t b[4];
          ldmatrix_x4_trans(v_addr + (c >> 3) * KT * 128 + token * 128 + (((c & 7) ^ (token & 7)) << 4), b[0], b[1], b[2], b[3]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            if (mt < mts) {
              mma_m16n8k16_bf16(o[mt][n], a[mt], b[0], b[1]);
              mma_m16n8k16_bf16(o[mt][n + 1], a[mt], b[2], b[3]);
            }
        }
      }
      if (odd_tile) {  // the sum is none either, whatever the token's weight
#pragma unroll 1
        for (int i = some; i < min(hi, KT); ++i) {
          const int page = p.page_map[(long long)s.x.map * p.max_pages + (key + i) / p.tokens_per_page];
          const bf16* y = p.v + (((long long)s.kvh * p.num_pages + (page >= 0 && page < p.num_pages ? page : 0)) * p.tokens_per_page + (key + i) % p.tokens_per_page) * D +
                          warp * F::kCols + (lane & 3) * 2;
#pragma unroll
          for (int n = 0; n < NO; ++n)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const float value = __bfloat162float(y[n * 8 + f]);
              if (!(fabsf(value) < INFINITY))
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                  for (int h = 0; h < 2; ++h)
                    if (key + i < seen[mt][h]) o[mt][n][2 * h + f] += value;
            }
        }
      }
      if (masked) fence_proxy_async();  // (zeros in a piece that the next copy overwrites)
      __syncwarp();
      if (lane == 0) mbar_arrive(&tail->empty[piece]);
      if (++piece == kPrefixPieces) piece = 0, phase ^= 1;
      turn ^= 1;
    }
    // the item's results: as they are where no other part joins them
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 1);
        l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 2);
        if (mt < mts && (lane & 3) == 0) tail->sum[mt * 16 + r + 8 * h][warp] = l[mt][h];
      }
    prefix_bar();
    const bool whole = prefix_whole(s) && k.first + s.e >= p.prefixes;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pair = mt * 16 + r + 8 * h, at = pair0 + pair;
        if (pair >= pairs) continue;
        const float4 u = *reinterpret_cast<const float4*>(tail->sum[pair]);
        const float sum = (u.x + u.y) + (u.z + u.w);
        const int col0 = warp * F::kCols + (lane & 3) * 2;
        if (whole) {
          if (seen[mt][h] <= 0) continue;  // a row that sees nothing
          const float inv = 1.0f / sum;
          bf16* out = p.out + (s.x.row + at / p.group) * p.ldo + (s.kvh * p.group + at % p.group) * D + col0;
#pragma unroll
          for (int n = 0; n < NO; ++n) *reinterpret_cast<uint32_t*>(out + n * 8) = pack_bf16x2(o[mt][n][2 * h] * inv, o[mt][n][2 * h + 1] * inv);
        } else {
          const long long place = s.place + pair;
          float* out = k.part + place * D + col0;
#pragma unroll
          for (int n = 0; n < NO; ++n) *reinterpret_cast<float2*>(out + n * 8) = make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
          if (warp == 0 && (lane & 3) == 0) k.stat[place] = make_float2(m[mt][h], sum);
        }
      }
  }
  griddep_wait();
}

// ---- units of many rows on the tensor cores ------------------------------------------------------------------------------------------
//
// Prefixes whose sequences bring some hundred pairs.  Warp 0 copies K and V tiles, warp 1 issues the MMAs, four softmax warps have each 128 pairs of the item:
//   S = Q K^T    tcgen05.mma, M = 128, N = KT, fp32 in TMEM
//   P = exp2(..) a thread owns a pair: it reads its row of S, keeps maximum and sum in registers and writes P as bf16 over S
//   O += P V     tcgen05.mma with P as the TMEM operand and V as an MN-major one, fp32 in TMEM
// With two times 128 pairs the MMAs of one half run under the softmax of the other.  The accumulator is brought to a new maximum only when a pair's grew by more than 2^8.

template <int D>
struct PrefixTcShape {
  static constexpr int NQ = D == 256 ? 1 : 2, KT = D == 256 ? 64 : 128, CH = D / 64;
  static constexpr int kPairs = NQ * 128;
  static constexpr int kPieceBytes = KT * D * 2, kPieces = 131072 / kPieceBytes;
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kThreads = 64 + NQ * 128;
  static constexpr int kOCol = NQ * KT;
};

struct PrefixTcTail {
  PrefixEntry entry[kPrefixCached + 1];
  uint64_t full[8], empty[8];
  uint64_t q_ready, s_full[2], p_ready[2], o_done[2];
  long long carry[20];
  uint32_t tmem_base;
  int failed;
};

template <int D>
constexpr size_t prefix_tc_smem_bytes() {
  typedef PrefixTcShape<D> F;
  return 1024 + size_t(F::NQ) * F::kQBytes + size_t(F::kPieces) * F::kPieceBytes + sizeof(PrefixTcTail) + 16;
}

__device__ __forceinline__ float prefix_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D>
__global__ void __launch_bounds__(PrefixTcShape<D>::kThreads, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PrefixAttnParams p, const PrefixWork k) {
  typedef PrefixTcShape<D> F;
  constexpr int NQ = F::NQ, KT = F::KT, CH = F::CH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sq = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // [NQ][CH][128 pairs][128 B], swizzled
  uint8_t* ring = sq + NQ * F::kQBytes;                                         // piece: [CH][KT tokens][128 B]
  PrefixTcTail* tail = reinterpret_cast<PrefixTcTail*>(ring + F::kPieces * F::kPieceBytes);
  volatile int* failed = &tail->failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int i = 0; i < F::kPieces; ++i) {
      mbar_init(&tail->full[i], 1);
      mbar_init(&tail->empty[i], 1);
    }
    mbar_init(&tail->q_ready, NQ * 4);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&tail->s_full[t], 1);
      mbar_init(&tail->p_ready[t], 4);  // one arrival per softmax warp
      mbar_init(&tail->o_done[t], 1);
    }
    tail->failed = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tail->tmem_base, 512);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch_dependents();
  const PrefixEntry* table = k.table;
  tcgen05_fence_before();
  if (!k.tabled) {
    prefix_build_table(p, k, tail->entry, tail->carry, threadIdx.x, F::kThreads);
    table = tail->entry;
    if (blockIdx.x == 0)  // for the join
      for (int e = threadIdx.x; e <= k.count; e += F::kThreads) k.table[e] = table[e];
  } else {
    __syncthreads();
  }
  tcgen05_fence_after();
  const uint32_t tmem = tail->tmem_base;
  const PrefixShare share(table[k.count].units * p.kv_heads, k.workers);
  const bool mine = int(blockIdx.x) < share.workers;
  PrefixSegment s;

  if (!mine) {
  } else if (warp == 0) {
    PrefixWalk walk(p, k, table, share, blockIdx.x);
    const bool issuer = elect_one();
    const int boxes = KT / p.box, tpp = p.tokens_per_page;
    int piece = 0;
    uint32_t phase = 1;
    bool good = true;
    while (walk.next(s)) {
      const int* pages = p.page_map + (long long)s.x.map * p.max_pages;
      const long long head_row = (long long)s.kvh * p.num_pages * tpp;
      auto row_of = [&](int tile) {  // as in prefix_units_kernel
        const int key = min(s.first + tile * KT + (lane < boxes ? lane : 0) * p.box, s.x.key1 - 1);
        const int page = pages[key / tpp];
        return int(head_row + (long long)(page >= 0 && page < p.num_pages ? page : 0) * tpp + key % tpp / p.box * p.box);
      };
      int row = row_of(s.tile0);
      for (int t = s.tile0; t < s.tile1; ++t) {
        const int next = t + 1 < s.tile1 ? row_of(t + 1) : 0;
        for (int kv = 0; kv < 2; ++kv) {
          good = good && prefix_wait(&tail->empty[piece], phase, failed);
          uint8_t* to = ring + piece * F::kPieceBytes;
          if (issuer && good) mbar_expect_tx(&tail->full[piece], F::kPieceBytes);
          for (int b = 0; b < boxes; ++b) {
            const int from = __shfl_sync(0xffffffffu, row, b);
            if (issuer && good)
              for (int c = 0; c < CH; ++c) tma_load_2d(to + c * KT * 128 + b * p.box * 128, kv == 0 ? &tm_k : &tm_v, c * 64, from, &tail->full[piece], kEvictNormal);
          }
          if (++piece == F::kPieces) piece = 0, phase ^= 1;
        }
        row = next;
      }
    }
    for (int i = 0; i < F::kPieces; ++i) {  // the MMAs' arrivals have to be in before the CTA may leave
      good = good && prefix_wait(&tail->empty[piece], phase, failed);
      if (++piece == F::kPieces) piece = 0, phase ^= 1;
    }
    if (!good) {  // copies and MMAs in flight have a millisecond to end
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000) __nanosleep(1000);
    }
  } else if (warp == 1) {
    PrefixWalk walk(p, k, table, share, blockIdx.x);
    const bool issuer = elect_one();
    const uint32_t idesc_s = umma_idesc_bf16(128, KT), idesc_o = umma_idesc_bf16(128, D) | kIdescBMajorMN;
    const uint64_t dq = umma_desc_sw128(sq), dk = umma_desc_sw128(ring);
    const uint32_t ring_addr = smem_u32(ring);
    bool good = true;
    auto issue_s = [&](int t, int piece) {
      if (!issuer || !good) return;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_bf16(tmem + t * KT, dq + uint64_t((t * F::kQBytes + c * 16384 + kk * 32) >> 4), dk + uint64_t((piece * F::kPieceBytes + c * KT * 128 + kk * 32) >> 4), idesc_s,
                    uint32_t((c | kk) != 0));
      umma_commit(&tail->s_full[t]);
    };
    auto issue_o = [&](int t, int piece, bool start) {
      if (!issuer || !good) return;
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk)
        umma_bf16_ts(tmem + F::kOCol + t * D, tmem + t * KT + kk * 8, umma_desc_sw128_mn(ring_addr + piece * F::kPieceBytes + kk * 2048, KT * 128), idesc_o, uint32_t(!start || kk != 0));
    };
    int piece = 0, segment = 0;  // pieces: K, V, K, V ..
    uint32_t phase = 0, turn[2] = {0, 0};
    auto advance = [&]() {
      const int at = piece;
      if (++piece == F::kPieces) piece = 0, phase ^= 1;
      return at;
    };
    while (walk.next(s)) {
      const int halves = NQ == 2 && s.x.rows * p.group - s.block * F::kPairs > 128 ? 2 : 1;
      good = good && prefix_wait(&tail->q_ready, segment & 1, failed);
      ++segment;
      good = good && prefix_wait(&tail->full[piece], phase, failed);
      tcgen05_fence_after();
      int at = advance();
      for (int t = 0; t < halves; ++t) issue_s(t, at);
      if (issuer && good) umma_commit(&tail->empty[at]);
      for (int j = s.tile0; j < s.tile1; ++j) {
        const bool more = j + 1 < s.tile1;
        good = good && prefix_wait(&tail->full[piece], phase, failed);
        const int v_at = advance();
        const int beyond = s.x.key1 - (s.first + j * KT);  // the tile's first token that the prefix does not have
        if (beyond < KT) {                                 // it may hold anything, and 0 * NaN is not 0
          uint8_t* v = ring + v_at * F::kPieceBytes;
          for (int c = 0; c < CH; ++c)
            for (int b = beyond * 128 + lane * 16; b < KT * 128; b += 512) *reinterpret_cast<uint4*>(v + c * KT * 128 + b) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
          __syncwarp();
        }
        int k_at = 0;
        if (more) {
          good = good && prefix_wait(&tail->full[piece], phase, failed);
          k_at = advance();
        }
        for (int t = 0; t < halves; ++t) {
          good = good && prefix_wait(&tail->p_ready[t], turn[t], failed);
          turn[t] ^= 1;
          tcgen05_fence_after();
          issue_o(t, v_at, j == s.tile0);
          if (more) issue_s(t, k_at);
          else if (issuer && good) umma_commit(&tail->o_done[t]);
        }
        if (issuer && good) {
          umma_commit(&tail->empty[v_at]);
          if (more) umma_commit(&tail->empty[k_at]);
        }
      }
    }
    __syncwarp();
  } else {
    PrefixWalk walk(p, k, table, share, blockIdx.x);
    const int t = (warp - 2) >> 2, quarter = warp & 3, own = quarter * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16), acc = lanes + F::kOCol + t * D, scores = lanes + t * KT;
    const float mul = p.softcap > 0.0f ? 1.0f : p.scale * kPrefixLog2e, cap = p.softcap * kPrefixLog2e, by_cap = p.softcap > 0.0f ? p.scale / p.softcap : 0.0f;
    uint32_t turn = 0, done = 0;
    int segment = 0;
    while (walk.next(s)) {
      const int pair0 = s.block * F::kPairs + t * 128, pairs = s.x.rows * p.group - pair0;
      // Q: a thread brings its pair's row
      {
        uint4 v[D / 8];
        const int at = pair0 + own;
        const bf16* from = p.q + (s.x.row + at / p.group) * p.ldq + (s.kvh * p.group + at % p.group) * D;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) v[c] = own < pairs ? reinterpret_cast<const uint4*>(from)[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(sq + t * F::kQBytes + (c >> 3) * 16384 + own * 128 + (((c & 7) ^ (own & 7)) << 4)) = v[c];
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->q_ready);
      }
      const int now_segment = segment++;
      if (pairs <= 0) {  // (not two arrivals for one item)
        prefix_wait(&tail->q_ready, now_segment & 1, failed);
        continue;
      }
      float m = -INFINITY, l = 0.0f;  // the maximum that the accumulator stands at (times log2 e), the sum
      for (int j = s.tile0; j < s.tile1; ++j) {
        prefix_wait(&tail->s_full[t], turn, failed);
        turn ^= 1;
        tcgen05_fence_after();
        float x[KT];
        {
          uint32_t raw[KT / 32][32];
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) tmem_ld_x32(scores + c * 32, raw[c]);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < KT; ++c) x[c] = __uint_as_float(raw[c / 32][c % 32]);
        }
        if (p.softcap > 0.0f) {
#pragma unroll
          for (int c = 0; c < KT; ++c) x[c] = cap * tanhf(x[c] * by_cap);
        }
        const int beyond = s.x.key1 - (s.first + j * KT);
        if (beyond < KT) {
#pragma unroll
          for (int c = 0; c < KT; ++c)
            if (c >= beyond) x[c] = -INFINITY;
        }
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < KT; ++c) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
        const float now = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mul);
        if (__any_sync(0xffffffffu, now > m + 8.0f)) {  // (m = -inf: the first tile)
          const float fix = now == -INFINITY ? 1.0f : prefix_ex2(m - now);
          l *= fix;
          m = now;
          if (j > s.tile0) {  // the accumulator holds the tiles before: they are complete (s_full came behind them)
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_x32(acc + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
              tmem_st_x32(acc + c, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
        for (int c = 0; c < KT; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p0 = prefix_ex2(fmaf(x[c + 2 * e], mul, -base)), p1 = prefix_ex2(fmaf(x[c + 2 * e + 1], mul, -base));
            l0 += p0;
            l1 += p1;
            pk[e] = pack_bf16x2(p0, p1);
          }
          tmem_st_x16(scores + c / 2, pk);
        }
        l += l0 + l1;
        tmem_wait_st();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->p_ready[t]);
      }
      prefix_wait(&tail->o_done[t], done, failed);
      done ^= 1;
      tcgen05_fence_after();
      const long long place = s.place + t * 128 + own;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld_x32(acc + c, o);
        tmem_wait_ld();
        if (own < pairs) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(k.part + place * D + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
      if (own < pairs) k.stat[place] = make_float2(m, l);
      tcgen05_fence_before();
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---- the join ----------------------------------------------------------------------------------------------------------------------

// CTA = row; a thread has four channels of a head.  A row's parts: its prefix's (of `a`), then its tail's (of `b`), in the tokens' order.
template <int D>
__global__ void __launch_bounds__(512) prefix_join_kernel(const PrefixAttnParams p, const PrefixWork a, const PrefixWork b) {
  griddep_launch_dependents();
  griddep_wait();
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const PrefixEntry* sequences = b.table + (p.prefixes - b.first);
  // the last sequence that begins at the row or in front of it: 32 probes at a time
  int lo = 0, hi = p.sequences;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const bool below = at < hi && sequences[at].row <= row;
    const int c = __popc(__ballot_sync(0xffffffffu, below));
    if (c == 0) break;
    hi = min(hi, lo + c * step);
    lo = lo + (c - 1) * step + 1;
  }
  if (lo == 0) return;
  const PrefixEntry tail = sequences[lo - 1];
  if (row >= tail.row + tail.rows) return;
  if (min(tail.first_seen + row - tail.row, tail.key1) <= 0) return;
  const PrefixEntry front = a.table[max(tail.prefix, 0)];
  const PrefixEntry last[2] = {a.table[a.count], b.table[b.count]};
  for (int i = threadIdx.x; i < p.heads * (D / 4); i += blockDim.x) {
    const int head = i / (D / 4), c = (i - head * (D / 4)) * 4, kvh = head / p.group, g = head - kvh * p.group;
    long long place[2];
    int parts[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      place[k] = parts[k] = 0;
      const PrefixWork& w = k == 0 ? a : b;
      const PrefixEntry& x = k == 0 ? front : tail;
      const int tiles = prefix_tiles(x, w.kt, p.box);
      if ((k == 0 && tail.prefix < 0) || tiles == 0) continue;
      const long long at = (long long)(row - x.row) * p.group + g;
      const int block = int(at / w.pairs);
      const long long first = kvh * last[k].units + x.units + (long long)block * tiles;
      const PrefixShare share(last[k].units * p.kv_heads, w.workers);
      const int c0 = share.of(first), c1 = share.of(first + tiles - 1);
      place[k] = (long long)kvh * last[k].pairs + x.pairs + at + (long long)c0 * w.pairs;
      parts[k] = c1 - c0 + 1;
    }
    if (tail.key0 == 0 && parts[1] == 1) continue;  // written already
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const PrefixWork& w = k == 0 ? a : b;
      for (int j = 0; j < parts[k]; ++j) top = fmaxf(top, w.stat[place[k] + (long long)j * w.pairs].x);
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const PrefixWork& w = k == 0 ? a : b;
      for (int j = 0; j < parts[k]; ++j) {
        const long long at = place[k] + (long long)j * w.pairs;
        const float2 st = w.stat[at];
        const float4 v = *reinterpret_cast<const float4*>(w.part + at * D + c);
        const float f = exp2f(st.x - base);
        if (st.x == -INFINITY) continue;  // (a part of which the row sees nothing)
        sum = fmaf(st.y, f, sum);
        o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
      }
    }
    const float inv = 1.0f / sum;
    *reinterpret_cast<uint2*>(p.out + row * p.ldo + head * D + c) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
}

}  // namespace mtx
