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
  int heads, kv_heads, group, num_pages, tokens_per_page, page_bits, max_pages;
  float scale, softcap;
  int box;  // tokens of a copy of the tails' kernel: a page, or a part of one, at most a tile (tiles begin at its multiples)
};

// Entries that one kernel goes through, and where its results are.
struct PrefixWork {
  int first, count;  // the entries: prefixes, then sequences
  int kt, pairs;     // tokens of a tile, pairs of an item
  int box_bits;      // log2 of the tokens of a copy
  int round_bits;    // log2 of the tiles whose copies 32 lanes look up
  int workers;       // CTAs that share the units, at most
  int tabled;        // the table is there already (more entries than a CTA keeps)
  int mixed;         // an item's weighted values lie as [D / 4][pairs][4], not [pairs][D]
  float* part;       // [place][D]: weighted values
  float2* stat;      // [place]: maximum (of the scores times log2 e) and sum
  struct PrefixEntry* table;  // [count + 1], for the join
};

// What a CTA needs of an entry.  The one behind the last holds the sums.
struct alignas(16) PrefixEntry {
  int row, rows;     // the first, and how many
  int key0, key1;    // its tokens
  int first_seen;    // tokens that the first row sees (the next row one more, at most key1)
  int map;           // the page map's row
  int prefix;        // a tail's prefix where it begins behind one, else -1
  int first, tiles;  // the first tile's first token: key0 rounded down to where a copy may begin; tiles of an item
  int pairs, units;  // of one key head in the entries before
  int bad;           // row0 or prefix_seq0 descends; of the sums: somewhere, and nothing is done (places in the scratch are counted for entries side by side)
};

constexpr float kPrefixLog2e = 1.4426950408889634f;
constexpr int kPrefixCached = 128;  // entries that a CTA keeps in shared memory

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

// entry e without its sums; bounds, lens: the batch's prefix_seq0 and prefix_len, or copies of them
__device__ __forceinline__ PrefixEntry prefix_entry(const PrefixAttnParams& p, int kt, int e, const int* bounds, const int* lens) {
  const int most = p.max_pages * p.tokens_per_page;
  auto row_of = [&](int s) { return min(max(p.row0[s], 0), p.rows); };
  auto seq_of = [&](int i) { return min(max(bounds[i], 0), p.sequences); };
  PrefixEntry x;
  x.pairs = x.units = x.bad = 0;
  x.prefix = -1;
  if (e < p.prefixes) {
    const int s0 = seq_of(e), s1 = seq_of(e + 1);
    x.row = row_of(s0);
    x.rows = row_of(s1) - x.row;
    x.bad = bounds[e + 1] < bounds[e] || x.rows < 0;
    x.key0 = 0;
    x.key1 = min(max(lens[e], 0), most);
    x.first_seen = x.key1;
    x.map = s0 < p.sequences ? s0 : 0;
  } else {
    const int s = e - p.prefixes;
    const int r0 = row_of(s), r1 = row_of(s + 1), length = p.lengths[s];
    x.row = r0;
    x.rows = r1 - r0;
    x.bad = p.row0[s + 1] < p.row0[s];
    x.key1 = min(max(length, 0), most);
    x.first_seen = length < 0 ? -(1 << 30) : length - x.rows + 1;
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
      const int shared = min(max(lens[lo - 1], 0), most);
      if (shared > 0 && x.first_seen > shared) x.key0 = shared, x.prefix = lo - 1;  // every row lies behind the prefix; otherwise the sequence reads its own pages throughout
    }
  }
  x.first = x.key0 & ~(p.box - 1);
  x.tiles = x.rows > 0 && x.key1 > x.key0 ? (x.key1 - x.first + kt - 1) / kt : 0;
  return x;
}

constexpr int kPrefixKnown = 64;  // prefixes whose bounds and lengths a CTA copies

struct PrefixBuild {
  int carry[64];
  int bounds[kPrefixKnown + 1], lens[kPrefixKnown];
};

// All of a work's entries with their sums, by `threads` threads (whole warps, at most 1024) of a CTA.
__device__ __forceinline__ void prefix_build_table(const PrefixAttnParams& p, const PrefixWork& k, PrefixEntry* table, PrefixBuild* build, int tid, int threads) {
  const int lane = tid & 31, warp = tid >> 5, total = k.count;
  const int *bounds = p.prefix_seq0, *lens = p.prefix_len;
  if (p.prefixes <= kPrefixKnown) {
    for (int i = tid; i <= p.prefixes && p.prefixes > 0; i += threads) {
      build->bounds[i] = bounds[i];
      if (i < p.prefixes) build->lens[i] = lens[i];
    }
    bounds = build->bounds;
    lens = build->lens;
    __syncthreads();
  }
  int units = 0, pairs = 0, bad = 0;
  if (k.first > 0)  // (the prefixes have a table of their own; tails that no other part joins are stored without a look at it)
    for (int i = tid; i < p.prefixes; i += threads) bad |= bounds[i + 1] < bounds[i];
  for (int e0 = 0; e0 <= total; e0 += threads) {
    const int e = e0 + tid;
    PrefixEntry x;
    int u = 0, b = 0;
    if (e < total) {
      x = prefix_entry(p, k.kt, k.first + e, bounds, lens);
      bad |= x.bad;
      b = x.tiles > 0 ? x.rows * p.group : 0;
      u = x.tiles * ((b + k.pairs - 1) / k.pairs);
    } else {
      memset(&x, 0, sizeof(x));
      x.prefix = -1;
    }
    int us = u, bs = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, us, o), w = __shfl_up_sync(0xffffffffu, bs, o);
      if (lane >= o) us += t, bs += w;
    }
    __syncthreads();
    if (lane == 31) build->carry[2 * warp] = us, build->carry[2 * warp + 1] = bs;
    __syncthreads();
    int before = units, before_b = pairs;
    for (int w = 0; w < threads / 32; ++w) {
      const int cu = build->carry[2 * w], cb = build->carry[2 * w + 1];
      if (w < warp) before += cu, before_b += cb;
      units += cu, pairs += cb;
    }
    if (e <= total) {
      x.units = before + us - u;
      x.pairs = before_b + bs - b;
      table[e] = x;
    }
  }
  if (__syncthreads_or(bad) && tid == 0) table[total].units = 0, table[total].bad = 1;
  __syncthreads();
}

// for batches of more entries than a CTA keeps: one CTA in front of the others
__global__ void __launch_bounds__(1024) prefix_plan_kernel(const PrefixAttnParams p, const PrefixWork a, const PrefixWork b) {
  __shared__ PrefixBuild build;
  griddep_wait();
  griddep_launch_dependents();
  if (a.tabled) prefix_build_table(p, a, a.table, &build, threadIdx.x, 1024);
  if (b.tabled) prefix_build_table(p, b, b.table, &build, threadIdx.x, 1024);
}

// A CTA's run of units: worker c has those from begin(c) on, the first workers one more than the others.  (All numbers of units stay below 2^31: the call's sizes say so.)
struct PrefixShare {
  int workers, each, more;

  __device__ __forceinline__ PrefixShare(int units, int most) {
    workers = min(units, most);
    each = workers > 0 ? units / workers : 0;
    more = units - each * workers;
  }
  __device__ __forceinline__ int begin(int c) const { return each * c + min(c, more); }
  __device__ __forceinline__ int of(int u) const {  // the worker that has unit u
    const int longer = more * (each + 1);
    return u < longer ? u / (each + 1) : more + (u - longer) / each;
  }
};

// One item of a CTA's run: its tiles [tile0, tile1).
struct PrefixSegment {
  PrefixEntry x;
  int e, kvh, block, tile0, tile1;
  long long place;  // of its first pair's results
};

// Goes through a CTA's run item by item; all threads of a warp alike.
struct PrefixWalk {
  const PrefixEntry* table;
  int total, most, worker, per_head, at, end, e, kvh;

  __device__ __forceinline__ PrefixWalk(const PrefixWork& k, const PrefixEntry* t, const PrefixShare& share, int c) : table(t), total(k.count), most(k.pairs), worker(c) {
    per_head = t[total].units;
    at = share.begin(c);
    end = share.begin(c + 1);
    kvh = at / per_head;
    const int rest = at - kvh * per_head;
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
    int rest = at - kvh * per_head;
    if (rest >= per_head) ++kvh, rest = 0, e = 0;
    while (table[e + 1].units <= rest) ++e;
    s.x = table[e];
    s.e = e;
    s.kvh = kvh;
    const int in = rest - s.x.units;
    s.block = in / s.x.tiles;
    s.tile0 = in - s.block * s.x.tiles;
    s.tile1 = min(s.x.tiles, s.tile0 + (end - at));
    s.place = (long long)kvh * table[total].pairs + s.x.pairs + (long long)(s.block + worker) * most;  // (every step to the next one goes to another item, another CTA or both)
    at += s.tile1 - s.tile0;
    return true;
  }
};

__device__ __forceinline__ bool prefix_whole(const PrefixSegment& s) { return s.x.key0 == 0 && s.tile0 == 0 && s.tile1 == s.x.tiles; }

// ---- copies of tiles ---------------------------------------------------------------------------------------------------------------

// Where the boxes of an item's tiles lie in the pool: the 32 lanes look up as many boxes at a time.
struct PrefixRows {
  const int* pages;
  int head_row, num_pages, page_bits, box_bits, boxes, per, first, last, lane;  // (pages, boxes, boxes of a tile and tiles of a round are powers of two: a division in a tile's way takes 100 cycles)

  __device__ __forceinline__ PrefixRows(const PrefixAttnParams& p, const PrefixWork& k, const PrefixSegment& s, int kt)
      : pages(p.page_map + (long long)s.x.map * p.max_pages), head_row(s.kvh * p.num_pages * p.tokens_per_page), num_pages(p.num_pages), page_bits(p.page_bits),
        box_bits(k.box_bits), boxes(kt >> k.box_bits), per(k.round_bits), first(s.x.first + s.tile0 * kt), last(s.x.key1 - 1), lane(threadIdx.x & 31) {}
  __device__ __forceinline__ int round_of(int t) const { return t >> per; }
  __device__ __forceinline__ bool begins_round(int t) const { return (t & ((1 << per) - 1)) == 0; }
  // round r: lane i has box i of the round's tiles; boxes behind the last token: that token's page
  __device__ __forceinline__ int look_up(int r) const {
    const int key = min(first + ((r * 32 + lane) << box_bits), last), page = pages[key >> page_bits], in = key & ((1 << page_bits) - 1);
    return head_row + ((page >= 0 && page < num_pages ? page : 0) << page_bits) + (in >> box_bits << box_bits);
  }
  // of a round: the row of tile t's box b, the same in all lanes as the compiler sees it
  __device__ __forceinline__ int row(int round, int t, int b) const { return __reduce_max_sync(0xffffffffu, lane == (t & ((1 << per) - 1)) * boxes + b ? round : int(0x80000000)); }
};

// A box [CH][box tokens][128 B], or one chunk of channels of it
__device__ __forceinline__ void prefix_load_box(void* dst, const CUtensorMap* tm, int row, int c, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;"
      :
      : "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(c), "l"(kEvictNormal)
      : "memory");
}

// Tile t of K or V into a piece [CH][kt tokens][128 B]: one copy where a box is a whole tile, else one for each box and chunk.
template <int CH>
__device__ __forceinline__ void prefix_load_tile(const PrefixRows& rows, int round, int t, int kt, uint8_t* to, const CUtensorMap* tm, uint64_t* bar, bool issue) {
  for (int b = 0; b < rows.boxes; ++b) {
    const int from = rows.row(round, t, b);
    if (!issue) continue;
    if (rows.boxes == 1) {
      prefix_load_box(to, tm, from, 0, bar);
    } else {
      for (int c = 0; c < CH; ++c) prefix_load_box(to + c * kt * 128 + (b << rows.box_bits) * 128, tm, from, c, bar);
    }
  }
}

// ---- units on the warps' MMAs ------------------------------------------------------------------------------------------------------
//
// Tails, and prefixes whose sequences bring few pairs.  Warp 4 copies K and V tiles of 8 KB each.  Warps 0 to 3 compute, each a tile of its own for 16 of the item's pairs, with S, P and O
// in its registers: an item of up to 16 pairs has every fourth tile in a warp, one of up to 32 every second, one of up to 64 all.  Where several warps have parts of the
// same pairs, they are joined in shared memory at the item's end.
// Bound: the tails' bytes, each read once.  64 sequences of 8 rows of 32 heads of 128 channels over up to 3000 tokens: 107 us, 255 MB at 2.4 TB/s.  A warp's tile of 32 tokens takes 2500 to 3000
// cycles, most of them waits of its own chain (copy, 32 MMAs of scores, maximum, weights, 32 MMAs of values) with two or three warps on a scheduler, and an item some 5000 to begin, join
// and store: short tails are bound by that.  (Queries in shared memory, and so three CTAs of an SM, were slower: 64 sequences of one row 39.2 us, not 35.5.)

constexpr int kPrefixPairs = 64;    // pairs of an item: four MMA tiles
constexpr int kPrefixWarps = 4;     // that compute; one more copies
constexpr int kPrefixThreads = 32 * (kPrefixWarps + 1);
constexpr int kPrefixPieceBytes = 8192;

template <int D>
struct PrefixShape {
  static constexpr int KT = kPrefixPieceBytes / 2 / D;  // tokens of a tile
  static constexpr int CH = D / 64;                     // 64-channel chunks of a row
  static constexpr int kCtas = D == 256 ? 1 : 2;        // per SM (registers: Q and O of 16 pairs are 3/8 D per thread)
  static constexpr int kPieces = D == 64 ? 12 : D == 128 ? 10 : 16;
};

struct PrefixTail {
  PrefixEntry entry[kPrefixCached + 1];
  uint64_t full[16], empty[16];
  int armed[16];  // the tile that a piece is for
  PrefixBuild build;
  float2 stat[2][16];
  int failed;
};

template <int D>
constexpr size_t prefix_smem_bytes() {
  return 1024 + size_t(PrefixShape<D>::kPieces) * kPrefixPieceBytes + 2 * 16 * (D + 4) * 4 + sizeof(PrefixTail) + 16;
}

__device__ __forceinline__ void prefix_bar() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kPrefixWarps) : "memory"); }
// Waits for a piece of tile n.  A warp does not see every tile of a piece, and copies end in any order: by its parity alone a barrier that still waits for the tile before (another warp's)
// looks as if tile n were there.  So the copying warp says which tile a piece is for, once the one before is used up.
__device__ __forceinline__ void prefix_wait_tile(volatile int* armed, int n, uint64_t* full, uint32_t phase, volatile int* failed) {
  if (*armed != n) {
    const long long t0 = clock64();
    while (*armed != n && *failed == 0)
      if (clock64() - t0 > 4000000000LL) {
        atomicAdd(&d_prefix_waits_failed, 1u);
        *failed = 1;
      }
  }
  prefix_wait(full, phase, failed);
}
// `count` of a barrier's four arrivals
__device__ __forceinline__ void prefix_arrive(uint64_t* bar, int count) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory"); }

__device__ __forceinline__ float prefix_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D, bool CAP>
__global__ void __launch_bounds__(kPrefixThreads, PrefixShape<D>::kCtas)
prefix_units_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PrefixAttnParams p, const PrefixWork k) {
  typedef PrefixShape<D> F;
  constexpr int KT = F::KT, CH = F::CH, NS = KT / 8, NO = D / 8, P = F::kPieces;
  extern __shared__ uint8_t smem_raw[];
  static_assert(P % 2 == 0 && P <= 16 && P >= 2 * kPrefixWarps, "the warps' next tiles lie at most a ring further on");
  uint8_t* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // piece: [CH][KT tokens][128 B], swizzled
  float* joint = reinterpret_cast<float*>(ring + P * kPrefixPieceBytes);         // [2][16 pairs][D + 4]
  PrefixTail* tail = reinterpret_cast<PrefixTail*>(joint + 2 * 16 * (D + 4));
  volatile int* failed = &tail->failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int i = 0; i < P; ++i) {
      mbar_init(&tail->full[i], 1);
      mbar_init(&tail->empty[i], kPrefixWarps);
      tail->armed[i] = -1;
    }
    tail->failed = 0;
    fence_barrier_init();
  }
  // (behind the prefixes' kernel: that one has waited for what is in front of it, and the join waits for this one, which waits for that one before it ends)
  if (k.first == 0 || k.tabled) griddep_wait();
  const PrefixEntry* table = k.table;
  if (!k.tabled) {
    prefix_build_table(p, k, tail->entry, &tail->build, threadIdx.x, kPrefixThreads);
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
  PrefixWalk walk(k, table, share, blockIdx.x);
  PrefixSegment s;

  if (warp == kPrefixWarps) {
    const bool issuer = elect_one();
    int piece = 0, tile = 0;  // (of all that the CTA goes through)
    uint32_t phase = 1;
    bool good = true;
    while (walk.next(s)) {
      const PrefixRows rows(p, k, s, KT);
      const int n = s.tile1 - s.tile0;
      int round = rows.look_up(0), ahead = rows.look_up(1);
      for (int i = 0; i < n; ++i, ++tile) {
        if (i > 0 && rows.begins_round(i)) round = ahead, ahead = rows.look_up(rows.round_of(i) + 1);
        for (int kv = 0; kv < 2; ++kv) {
          good = __all_sync(0xffffffffu, good && prefix_wait(&tail->empty[piece], phase, failed));
          if (issuer && good) {
            mbar_expect_tx(&tail->full[piece], kPrefixPieceBytes);
            *const_cast<volatile int*>(&tail->armed[piece]) = tile;
          }
          prefix_load_tile<CH>(rows, round, i, KT, ring + piece * kPrefixPieceBytes, kv == 0 ? &tm_k : &tm_v, &tail->full[piece], issuer && good);
          if (++piece == P) piece = 0, phase ^= 1;
        }
      }
    }
    griddep_launch_dependents();
    if (!good) {  // copies in flight have a millisecond to end
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000) __nanosleep(1000);
    }
    griddep_wait();
    return;
  }

  const float mul = CAP ? p.scale / p.softcap : p.scale * kPrefixLog2e, cap = p.softcap * kPrefixLog2e;
  const int r = lane >> 2, q2 = (lane & 3) * 2;  // this lane's pairs of an MMA tile: r and r + 8; its columns
  const uint32_t ring_addr = smem_u32(ring);
  int piece0 = 0, tile0 = 0;  // the item's first tile: its piece, its number
  uint32_t phase0 = 0;
  uint32_t q[D / 16][4];
  int wm, mt;  // MMA tiles of the item, this warp's
  auto load_q = [&]() {
    const int left = s.x.rows * p.group - s.block * kPrefixPairs;
    wm = left > 32 ? 4 : left > 16 ? 2 : 1;
    mt = warp & (wm - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int pair = mt * 16 + r + 8 * h, at = s.block * kPrefixPairs + pair;
      const bf16* from = p.q + (s.x.row + at / p.group) * p.ldq + (s.kvh * p.group + at % p.group) * D + q2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        q[kk][h] = pair < left ? *reinterpret_cast<const uint32_t*>(from + kk * 16) : 0u;
        q[kk][2 + h] = pair < left ? *reinterpret_cast<const uint32_t*>(from + kk * 16 + 8) : 0u;
      }
    }
  };
  bool more = walk.next(s);
  if (more) load_q();
  while (more) {
    const int pair0 = s.block * kPrefixPairs + mt * 16, left = s.x.rows * p.group - pair0;  // (pairs from this warp's first on)
    const int groups = kPrefixWarps / wm;  // of warps, with a tile each; a barrier has as many arrivals of each of a tile's warps
    const bool prefix = k.first + s.e < p.prefixes;
    int seen[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) seen[h] = prefix ? s.x.key1 : min(s.x.first_seen + (pair0 + r + 8 * h) / p.group, s.x.key1);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[NO][4];
#pragma unroll
    for (int n = 0; n < NO; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    const int mine = warp / wm;  // of the groups
    int piece = piece0 + 2 * mine;
    uint32_t phase = phase0;
    if (piece >= P) piece -= P, phase ^= 1;
    for (int t = s.tile0 + mine, number = tile0 + mine; t < s.tile1; t += groups, number += groups) {
      const int key = s.x.first + t * KT;  // the tile's first token
      const bool masked = key < s.x.key0 || key + KT > min(s.x.first_seen, s.x.key1);
      int v_piece = piece + 1;
      uint32_t v_phase = phase;
      if (v_piece == P) v_piece = 0, v_phase ^= 1;
      float x[NS][4];
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = 0.0f;
      prefix_wait_tile(&tail->armed[piece], number, &tail->full[piece], phase, failed);
      {
        // ldmatrix: lanes 0-7 and 8-15 the two halves of 16 channels of eight tokens, lanes 16-31 of the next eight
        const int token = (lane & 7) + (lane >> 4) * 8;
        const uint32_t k_addr = ring_addr + piece * kPrefixPieceBytes + token * 128;
        const int half = lane >> 3 & 1, turn = lane & 7;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int n = 0; n < NS; n += 2) {
            uint32_t b[4];
            ldmatrix_x4(k_addr + kk / 4 * KT * 128 + n * 1024 + (((kk % 4 * 2 + half) ^ turn) << 4), b[0], b[1], b[2], b[3]);
            mma_m16n8k16_bf16(x[n], q[kk], b[0], b[1]);
            mma_m16n8k16_bf16(x[n + 1], q[kk], b[2], b[3]);
          }
      }
      __syncwarp();
      if (lane == 0) prefix_arrive(&tail->empty[piece], groups);
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[n][i] *= mul;
          if (CAP) x[n][i] = cap * tanhf(x[n][i]);
        }
      if (masked) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = key + n * 8 + q2 + (i & 1);
            if (j < s.x.key0 || j >= seen[i >> 1]) x[n][i] = -INFINITY;
          }
      }
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i >> 1] = fmaxf(top[i >> 1], x[n][i]);
      float base[2];
      bool grown = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        top[h] = fmaxf(top[h], m[h]);
        grown = grown || top[h] > m[h];
        base[h] = top[h] == -INFINITY ? 0.0f : top[h];
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float fix = prefix_ex2(m[h] - base[h]);
          m[h] = top[h];
          l[h] *= fix;
#pragma unroll
          for (int n = 0; n < NO; ++n) o[n][2 * h] *= fix, o[n][2 * h + 1] *= fix;
        }
      }
      uint32_t a[KT / 16][4];  // weights as bf16, half a step of 2^-8 each: the MMAs take both factors in the values' type
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = pack_bf16x2(prefix_ex2(x[n][2 * h] - base[h]), prefix_ex2(x[n][2 * h + 1] - base[h]));
          l[h] += bf16_lo(w) + bf16_hi(w);  // (of the rounded weights: where one key has nearly all, its rounding cancels)
          a[n / 2][n % 2 * 2 + h] = w;
        }
      prefix_wait_tile(&tail->armed[v_piece], number, &tail->full[v_piece], v_phase, failed);
      bool odd = false;
      int some = 0, hi = 0;
      if (masked) {
        // V: tokens outside the entry's count 0 whatever they hold.  So do numbers that are none, in tokens that some rows see and others do not (0 times them is none either); the rows
        // that see them add them behind the products
        uint8_t* v = ring + v_piece * kPrefixPieceBytes;
        const int lo = min(max(s.x.key0 - key, 0), KT);
        hi = min(s.x.key1 - key, KT);
        some = min(max(s.x.first_seen - key, lo), hi);
        auto piece_of = [&](int token, int i) { return reinterpret_cast<uint4*>(v + (i >> 3) * KT * 128 + token * 128 + ((i & 7) << 4)); };  // (any order of a row's pieces)
        uint32_t gone = 0;
        for (int i = some * (D / 8) + lane; i < hi * (D / 8); i += 32) {
          const uint4 u = *piece_of(i / (D / 8), i % (D / 8));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int b = 0; b < 4; ++b) gone |= (w[b] & 0x7f80u) == 0x7f80u || (w[b] & 0x7f800000u) == 0x7f800000u;
        }
        odd = __any_sync(0xffffffffu, gone != 0);
        if (wm > 1) asm volatile("bar.sync %0, %1;" ::"r"(2 + mine), "r"(32 * wm) : "memory");  // (the tile's other warps have looked too)
        for (int i = lane; i < lo * (D / 8); i += 32) *piece_of(i / (D / 8), i % (D / 8)) = make_uint4(0, 0, 0, 0);
        for (int i = hi * (D / 8) + lane; i < KT * (D / 8); i += 32) *piece_of(i / (D / 8), i % (D / 8)) = make_uint4(0, 0, 0, 0);
        if (odd) {
          for (int i = some * (D / 8) + lane; i < hi * (D / 8); i += 32) {
            uint4 u = *piece_of(i / (D / 8), i % (D / 8));
            uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
            for (int b = 0; b < 4; ++b) w[b] &= ~(((w[b] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w[b] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u));
            *piece_of(i / (D / 8), i % (D / 8)) = u;
          }
        }
        __syncwarp();
      }
      {
        const uint32_t v_addr = ring_addr + v_piece * kPrefixPieceBytes + (lane & 15) * 128;
        const int half = lane >> 4, turn = lane & 7;
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
          for (int n = 0; n < NO; n += 2) {
            uint32_t b[4];
            ldmatrix_x4_trans(v_addr + n / 8 * KT * 128 + kk * 2048 + (((n % 8 + half) ^ turn) << 4), b[0], b[1], b[2], b[3]);
            mma_m16n8k16_bf16(o[n], a[kk], b[0], b[1]);
            mma_m16n8k16_bf16(o[n + 1], a[kk], b[2], b[3]);
          }
      }
      if (masked) {
        if (odd) {  // the sum is none either, whatever the token's weight
#pragma unroll 1
          for (int i = some; i < hi; ++i) {
            const int page = p.page_map[(long long)s.x.map * p.max_pages + (key + i) / p.tokens_per_page];
            const bf16* y = p.v + (((long long)s.kvh * p.num_pages + (page >= 0 && page < p.num_pages ? page : 0)) * p.tokens_per_page + (key + i) % p.tokens_per_page) * D + q2;
#pragma unroll
            for (int n = 0; n < NO; ++n)
#pragma unroll
              for (int f = 0; f < 2; ++f) {
                const float value = __bfloat162float(y[n * 8 + f]);
                if (!(fabsf(value) < INFINITY)) {
#pragma unroll
                  for (int h = 0; h < 2; ++h)
                    if (key + i < seen[h]) o[n][2 * h + f] += value;
                }
              }
          }
        }
        fence_proxy_async();  // (zeros in a piece that the next copy overwrites)
      }
      __syncwarp();
      if (lane == 0) prefix_arrive(&tail->empty[v_piece], groups);
      piece += 2 * groups;
      if (piece >= P) piece -= P, phase ^= 1;
    }
    // the next item's queries are on their way while this one's warps are joined
    const PrefixSegment done = s;
    const int pieces = 2 * (s.tile1 - s.tile0), here = mt;
    tile0 += s.tile1 - s.tile0;
    piece0 += pieces % P;
    phase0 ^= pieces / P & 1;
    if (piece0 >= P) piece0 -= P, phase0 ^= 1;
    more = walk.next(s);
    const int was = wm;
    if (more) load_q();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    // warps w and w + n have the same pairs: the upper ones leave their part, the lower ones add it, n = 2, 1 (for 32 pairs 2 alone, for 64 none)
    for (int n = 2; n >= was; n >>= 1) {
      prefix_bar();  // (the buffers are free)
      if (warp >= n && warp < 2 * n) {
        float* to = joint + (warp - n) * 16 * (D + 4);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if ((lane & 3) == 0) tail->stat[warp - n][r + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
          for (int c = 0; c < NO; ++c) *reinterpret_cast<float2*>(to + (r + 8 * h) * (D + 4) + c * 8 + q2) = make_float2(o[c][2 * h], o[c][2 * h + 1]);
        }
      }
      prefix_bar();
      if (warp < n) {
        const float* from = joint + warp * 16 * (D + 4);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 st = tail->stat[warp][r + 8 * h];
          const float now = fmaxf(m[h], st.x), base = now == -INFINITY ? 0.0f : now, f0 = prefix_ex2(m[h] - base), f1 = prefix_ex2(st.x - base);
          m[h] = now;
          l[h] = l[h] * f0 + st.y * f1;
#pragma unroll
          for (int c = 0; c < NO; ++c) {
            const float2 u = *reinterpret_cast<const float2*>(from + (r + 8 * h) * (D + 4) + c * 8 + q2);
            o[c][2 * h] = o[c][2 * h] * f0 + u.x * f1;
            o[c][2 * h + 1] = o[c][2 * h + 1] * f0 + u.y * f1;
          }
        }
      }
    }
    if (warp >= was) continue;
    // the item's results: as they are where no other part joins them
    const bool whole = prefix_whole(done) && !prefix;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = pair0 + r + 8 * h;
      if (r + 8 * h >= left) continue;
      if (whole) {
        if (seen[h] <= 0) continue;  // a row that sees nothing
        const float inv = 1.0f / l[h];
        bf16* out = p.out + (done.x.row + at / p.group) * p.ldo + (done.kvh * p.group + at % p.group) * D + q2;
#pragma unroll
        for (int n = 0; n < NO; ++n) *reinterpret_cast<uint32_t*>(out + n * 8) = pack_bf16x2(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
      } else {
        const long long place = done.place + here * 16 + r + 8 * h;
        float* out = k.part + place * D + q2;
#pragma unroll
        for (int n = 0; n < NO; ++n) *reinterpret_cast<float2*>(out + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if ((lane & 3) == 0) k.stat[place] = make_float2(m[h], l[h]);
      }
    }
  }
  // (now: a join that waits beside the units for their whole run made 48 sequences of 5 rows over 4096 shared tokens 59.8 us, not 53.6)
  griddep_launch_dependents();
  griddep_wait();
}

// ---- units of many rows on the tensor cores ------------------------------------------------------------------------------------------
//
// Prefixes whose sequences bring some hundred pairs.  Warp 0 copies queries and tiles of 64 tokens, warp 1 issues the MMAs, four softmax warps have each half of the item:
//   S = Q K^T    tcgen05.mma, M = 128, N = 64, fp32 in TMEM
//   P = exp2(..) a thread owns a pair: it reads its row of S, keeps maximum and sum in registers and writes P as bf16 over S
//   O += P V     tcgen05.mma with P as the TMEM operand and V as an MN-major one, fp32 in TMEM
// Each half has two places for S: the next tile's is there before a softmax ends, so that neither waits for the other in turn (with one place of 128 tokens an item's tile of
// 128 tokens took 3450 cycles: 2000 of softmax, 1000 of MMAs, the rest signals).  The accumulator is brought to a new maximum only when a pair's grew by more than 2^8.
// Bound: MMAs, whose operands come from shared memory at 128 bytes a clock (of 256 pairs, 64 tokens and 128 channels 1280 cycles), and the special-function units (1024).  A tile takes some
// 1700 cycles: 575 rows of 16 heads over 16384 shared tokens, 77 GFLOP, in some 75 us.

template <int D>
struct PrefixTcShape {
  static constexpr int NQ = D == 256 ? 1 : 2, KT = 64, CH = D / 64;
  static constexpr int kTileBytes = KT * D * 2, kStages = 65536 / kTileBytes;  // a stage: V of a tile and K of the next but one (an item's first: K of two tiles)
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kThreads = 32 * (1 + NQ + 4 * NQ);  // a warp that copies, one that issues MMAs for each half, four of the softmax for each
  static constexpr int kOCol = NQ * 2 * KT;
  // Every second pair of weights by a polynomial, not the special-function units, whose weights are rounded to bf16 (2^-8) all the same.  With heads of 128 channels the units and the
  // MMAs are both near their limits (575 rows of 16 heads over 16384 shared tokens: 122.7 us without, 116.2 so); with 64 the softmax's instructions bound (105.9 us without,
  // 116.2 so), with 256 the MMAs (66.3 and 66.7)
  static constexpr bool kByPolynomial = D == 128;
};

struct PrefixTcTail {
  PrefixEntry entry[kPrefixCached + 1];
  uint64_t full[8], empty[8];
  uint64_t q_full, q_empty, s_full[2][2], p_ready[2][2], o_done[2][2];
  PrefixBuild build;
  uint32_t tmem_base;
  int failed;
};

template <int D>
constexpr size_t prefix_tc_smem_bytes() {
  typedef PrefixTcShape<D> F;
  return 1024 + size_t(F::NQ) * F::kQBytes + size_t(F::kStages) * 2 * F::kTileBytes + sizeof(PrefixTcTail) + 16;
}

// two fp32 operations at a time
__device__ __forceinline__ float2 prefix_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 prefix_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// the largest; NaN where one is
__device__ __forceinline__ float prefix_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of two numbers of at most 2^6 by 32-bit operations alone: n = x to the nearest integer is what x + 1.5 * 2^23 ends in, 2^(x - n) a polynomial that is 1 at 0 and off by at most 2^-13.2
// on [-1/2, 1/2] (least squares, reweighted until the largest relative errors were alike).  What is less than 2^-126 (of -infinity too) becomes 2^-126, below a sum's last bit, and so does that of NaN.
__device__ __forceinline__ float2 prefix_ex2_poly(float2 x) {
  x.x = fmaxf(x.x, -126.0f);
  x.y = fmaxf(x.y, -126.0f);
  const float2 n = prefix_add2(x, make_float2(12582912.0f, 12582912.0f)), f = prefix_fma2(prefix_add2(n, make_float2(-12582912.0f, -12582912.0f)), make_float2(-1.0f, -1.0f), x);
  float2 y = prefix_fma2(f, make_float2(0.05500895f, 0.05500895f), make_float2(0.24221101f, 0.24221101f));
  y = prefix_fma2(y, f, make_float2(0.69328293f, 0.69328293f));
  y = prefix_fma2(y, f, make_float2(1.0f, 1.0f));
  return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(n.x) << 23)), __int_as_float(__float_as_int(y.y) + (__float_as_int(n.y) << 23)));
}

__device__ __forceinline__ void prefix_load_heads(void* dst, const CUtensorMap* tm, int c, int head, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;"
      :
      : "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(c), "r"(head), "r"(row), "l"(kEvictNormal)
      : "memory");
}

// umma_desc_sw128 of a shared address
__device__ __forceinline__ uint64_t prefix_desc(uint32_t addr) { return uint64_t((addr & 0x3FFFFu) >> 4) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61; }

// pairs of a half of an item: as many whole rows as fit
__device__ __forceinline__ int prefix_half(int group) { return 128 / group * group; }

template <int D, bool CAP>
__global__ void __launch_bounds__(PrefixTcShape<D>::kThreads, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PrefixAttnParams p, const PrefixWork k) {
  typedef PrefixTcShape<D> F;
  constexpr int NQ = F::NQ, KT = F::KT, CH = F::CH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sq = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // [NQ][CH][128 pairs][128 B], swizzled
  uint8_t* ring = sq + NQ * F::kQBytes;                                         // stage: two tiles [CH][KT tokens][128 B]
  PrefixTcTail* tail = reinterpret_cast<PrefixTcTail*>(ring + F::kStages * 2 * F::kTileBytes);
  volatile int* failed = &tail->failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = prefix_half(p.group);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int i = 0; i < F::kStages; ++i) {
      mbar_init(&tail->full[i], 1);
      mbar_init(&tail->empty[i], NQ);
    }
    mbar_init(&tail->q_full, 1);
    mbar_init(&tail->q_empty, NQ);
    for (int t = 0; t < 2; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&tail->s_full[t][b], 1);
        mbar_init(&tail->p_ready[t][b], 4);  // one arrival per softmax warp
        mbar_init(&tail->o_done[t][b], 1);   // (two: a wait for a tile's products may come while those of the tile before are not done)
      }
    }
    tail->failed = 0;
    fence_barrier_init();
  }
  // Tensor memory behind the wait: a kernel in front that lets this one start before it has its own columns (the products do) would wait for these, and this CTA for that kernel.  What comes next
  // starts when this CTA has its columns, for the same reason.
  griddep_wait();
  if (warp == 1) {
    tmem_alloc(&tail->tmem_base, 512);
    tmem_relinquish();
    griddep_launch_dependents();
  }
  const PrefixEntry* table = k.table;
  tcgen05_fence_before();
  if (!k.tabled) {
    prefix_build_table(p, k, tail->entry, &tail->build, threadIdx.x, F::kThreads);
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
    PrefixWalk walk(k, table, share, blockIdx.x);
    const bool issuer = elect_one();
    int stage = 0;
    uint32_t phase = 1, q_phase = 1;
    bool good = true;
    auto wait = [&](uint64_t* bar, uint32_t par) { good = __all_sync(0xffffffffu, good && prefix_wait(bar, par, failed)); };
    while (walk.next(s)) {
      const PrefixRows rows(p, k, s, KT);
      const int n = s.tile1 - s.tile0, halves = NQ == 2 && s.x.rows * p.group - s.block * k.pairs > half ? 2 : 1;
      int round[3] = {rows.look_up(0), rows.look_up(1), rows.look_up(2)};  // of V's tile, and the next two
      wait(&tail->q_empty, q_phase);
      q_phase ^= 1;
      if (issuer && good) {
        mbar_expect_tx(&tail->q_full, uint32_t(halves * CH * half * 128));
        for (int t = 0; t < halves; ++t)
          for (int c = 0; c < CH; ++c)
            prefix_load_heads(sq + t * F::kQBytes + c * 16384, &tm_q, c * 64, s.kvh * p.group, s.x.row + (s.block * k.pairs + t * half) / p.group, &tail->q_full);
      }
      for (int i = -1; i < n; ++i) {  // as the MMAs take them
        if (i > 0 && rows.begins_round(i)) round[0] = round[1], round[1] = round[2], round[2] = rows.look_up(rows.round_of(i) + 2);
        const int first = i < 0 ? 0 : i, second = i + 2;  // V of `first` (K where i < 0), K of `second`
        const bool more = second < n;
        wait(&tail->empty[stage], phase);
        uint8_t* to = ring + stage * 2 * F::kTileBytes;
        if (issuer && good) mbar_expect_tx(&tail->full[stage], (more ? 2 : 1) * F::kTileBytes);
        prefix_load_tile<CH>(rows, round[0], first, KT, to, i < 0 ? &tm_k : &tm_v, &tail->full[stage], issuer && good);
        if (more) prefix_load_tile<CH>(rows, rows.round_of(second) == rows.round_of(first) ? round[0] : round[1], second, KT, to + F::kTileBytes, &tm_k, &tail->full[stage], issuer && good);
        if (++stage == F::kStages) stage = 0, phase ^= 1;
      }
    }
    for (int i = 0; i < F::kStages; ++i) {  // the MMAs' arrivals have to be in before the CTA may leave
      wait(&tail->empty[stage], phase);
      if (++stage == F::kStages) stage = 0, phase ^= 1;
    }
    good = good && prefix_wait(&tail->q_empty, q_phase, failed);
    if (!good) {  // copies and MMAs in flight have a millisecond to end
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000) __nanosleep(1000);
    }
  } else if (warp <= NQ) {
    PrefixWalk walk(k, table, share, blockIdx.x);
    const bool issuer = elect_one();
    // numbers that the compiler takes for the same in all lanes: otherwise it brings every operand of every MMA to where the MMA reads it by itself (16 MMAs 1550 cycles, 950 so)
    auto same = [](int x) { return __reduce_max_sync(0xffffffffu, x); };
    const int t = same(warp - 1);
    const uint32_t tmem_at = uint32_t(same(int(tmem))), ring_addr = uint32_t(same(int(smem_u32(ring)))), s_at = tmem_at + t * 2 * KT, o_at = tmem_at + F::kOCol + t * D;
    const uint32_t idesc_s = umma_idesc_bf16(128, KT), idesc_o = umma_idesc_bf16(128, D) | kIdescBMajorMN;
    const uint64_t dq = prefix_desc(uint32_t(same(int(smem_u32(sq)))) + t * F::kQBytes), dk = prefix_desc(ring_addr);
    bool good = true;
    int stage = 0;
    uint32_t phase = 0, q_phase = 0, p_phase = 0;  // p_phase: bit b
    // by the issuing lane
    auto issue_s = [&](int b, uint32_t from) {
      const uint64_t d = dk + (from >> 4);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_bf16(s_at + b * KT, dq + uint64_t((c * 16384 + kk * 32) >> 4), d + uint64_t((c * KT * 128 + kk * 32) >> 4), idesc_s, uint32_t((c | kk) != 0));
      umma_commit(&tail->s_full[t][b]);
    };
    auto issue_o = [&](int b, uint32_t from, bool start) {
      const uint64_t d = umma_desc_sw128_mn(ring_addr, KT * 128) + (from >> 4);
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk) umma_bf16_ts(o_at, s_at + b * KT + kk * 8, d + uint64_t(kk * 2048 >> 4), idesc_o, uint32_t(!start || kk != 0));
      umma_commit(&tail->o_done[t][b]);
    };
    auto wait = [&](uint64_t* bar, uint32_t par) {
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, par))) return;
      good = __all_sync(0xffffffffu, good && prefix_wait(bar, par, failed));
    };
    auto used = [&]() {  // a stage
      if (++stage == F::kStages) stage = 0, phase ^= 1;
    };
    while (walk.next(s)) {
      const int halves = same(NQ == 2 && s.x.rows * p.group - s.block * k.pairs > half ? 2 : 1), n = same(s.tile1 - s.tile0), beyond = same(s.x.key1 - s.x.first - s.tile0 * KT);
      wait(&tail->q_full, q_phase);
      q_phase ^= 1;
      if (t >= halves) {  // nothing of this half: the stages go back as they come
        if (issuer && good) mbar_arrive(&tail->q_empty);
        for (int i = -1; i < n; ++i, used()) {
          wait(&tail->full[stage], phase);
          if (issuer && good) mbar_arrive(&tail->empty[stage]);
        }
        continue;
      }
      wait(&tail->full[stage], phase);
      tcgen05_fence_after();
      if (issuer && good) {
        const uint32_t from = stage * 2 * F::kTileBytes;
        issue_s(0, from);
        if (n > 1) issue_s(1, from + F::kTileBytes);
        umma_commit(&tail->empty[stage]);
        if (n <= 2) umma_commit(&tail->q_empty);
      }
      used();
      for (int i = 0; i < n; ++i, used()) {
        const int b = i & 1;
        const uint32_t from = stage * 2 * F::kTileBytes;
        wait(&tail->full[stage], phase);
        if (beyond - i * KT < KT) {  // tokens that the prefix does not have: V may hold anything, and 0 * NaN is not 0
          uint8_t* v = ring + from;
          for (int c = 0; c < CH; ++c)
            for (int at = (beyond - i * KT) * 128 + lane * 16; at < KT * 128; at += 512) *reinterpret_cast<uint4*>(v + c * KT * 128 + at) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
          __syncwarp();
        }
        wait(&tail->p_ready[t][b], p_phase >> b & 1);
        p_phase ^= 1u << b;
        tcgen05_fence_after();
        if (issuer && good) {
          issue_o(b, from, i == 0);
          if (i + 2 < n) issue_s(b, from + F::kTileBytes);
          umma_commit(&tail->empty[stage]);
          if (i + 3 == n) umma_commit(&tail->q_empty);
        }
      }
    }
    __syncwarp();
  } else {
    PrefixWalk walk(k, table, share, blockIdx.x);
    const int t = (warp - 1 - NQ) >> 2, quarter = warp & 3, own = quarter * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16), acc = lanes + F::kOCol + t * D;
    const float mul = CAP ? 1.0f : p.scale * kPrefixLog2e, cap = p.softcap * kPrefixLog2e, by_cap = CAP ? p.scale / p.softcap : 0.0f;
    const float2 mul2 = make_float2(mul, mul);
    uint32_t s_phase = 0;  // bit b
    uint32_t o_phase = 0;  // the same of the products
    while (walk.next(s)) {
      const int all = min(k.pairs, s.x.rows * p.group - s.block * k.pairs), pairs = min(half, all - t * half);  // of the item, of this half
      if (pairs <= 0) continue;
      const bool valid = own < pairs;
      float m = -INFINITY, l = 0.0f;  // the maximum that the accumulator stands at (times log2 e), the sum
      const int n = s.tile1 - s.tile0;
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int b = i & 1;
        const uint32_t scores = lanes + (t * 2 + b) * KT;
        prefix_wait(&tail->s_full[t][b], s_phase >> b & 1, failed);
        s_phase ^= 1u << b;
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
        if (CAP) {
#pragma unroll
          for (int c = 0; c < KT; ++c) x[c] = cap * tanhf(x[c] * by_cap);
        }
        const int beyond = s.x.key1 - s.x.first - (s.tile0 + i) * KT;
        if (beyond < KT) {
#pragma unroll
          for (int c = 0; c < KT; ++c)
            if (c >= beyond) x[c] = -INFINITY;
        }
        auto max3 = [](float a, float b, float c) { return F::kByPolynomial ? prefix_max3(a, b, c) : fmaxf(fmaxf(a, b), c); };
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c + 8 <= KT; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[c + e], x[c + 4 + e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], mx[e], x[KT - 4 + e]);
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]), now = fmaxf(m, top * mul);
        if (F::kByPolynomial && !(top < INFINITY)) m = 0.0f, l = top - top;  // a score is none or infinite: the row is none (weights by the polynomial are numbers all the same)
        if (__any_sync(0xffffffffu, valid && now > m + 8.0f)) {  // (m = -inf: the first tile)
          const float fix = now == -INFINITY ? 1.0f : prefix_ex2(m - now);
          l *= fix;
          m = now;
          if (i > 0) {  // the accumulator holds the tiles before
            prefix_wait(&tail->o_done[t][b ^ 1], ~o_phase >> (b ^ 1) & 1, failed);
            tcgen05_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_x32(acc + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix);
              tmem_st_x32(acc + c, o);
            }
          }
        }
        o_phase ^= 1u << b;
        const float base = m == -INFINITY ? 0.0f : m;
        const float2 base2 = make_float2(-base, -base);
        float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int c = 0; c < KT; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 w = prefix_fma2(make_float2(x[c + 2 * e], x[c + 2 * e + 1]), mul2, base2);
            if (F::kByPolynomial && e % 2 == 1) {
              w = prefix_ex2_poly(w);
            } else {
              w.x = prefix_ex2(w.x);
              w.y = prefix_ex2(w.y);
            }
            // the sum is of the weights before they are rounded to the values' type for the MMA: unpacking them again is two instructions more for each pair, in the half of the kernel that bounds heads
            // of 64 channels.  Where one key has nearly all of a row it is off by that rounding, half a step of 2^-8, as its result is anyway
            sums[e & 1] = prefix_add2(sums[e & 1], w);
            pk[e] = pack_bf16x2(w.x, w.y);
          }
          tmem_st_x16(scores + c / 2, pk);
        }
        l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
        tmem_wait_st();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->p_ready[t][b]);
      }
      prefix_wait(&tail->o_done[t][(n - 1) & 1], ~o_phase >> ((n - 1) & 1) & 1, failed);
      tcgen05_fence_after();
      // the item's results [D / 4][pairs][4]: neighbouring lanes store side by side (a row of each lane of its own took 7200 cycles, most of them the stores' 128-byte lines)
      float* out = k.part + s.place * D + (t * half + own) * 4;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld_x32(acc + c, o);
        tmem_wait_ld();
        if (valid) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(out + (long long)(c + e) * all) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      if (valid) k.stat[s.place + t * half + own] = make_float2(m, l);
      tcgen05_fence_before();
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---- the join ----------------------------------------------------------------------------------------------------------------------

// CTA = (row, key head); a thread has eight channels of a head, and every blockDim.y-th part of the row's: its prefix's (of `a`), then its tail's (of `b`), in the tokens' order, N of them
// in flight.
constexpr int kPrefixJoinMost = 256;  // threads

template <int D, int N>
__global__ void __launch_bounds__(kPrefixJoinMost) prefix_join_kernel(const PrefixAttnParams p, const PrefixWork a, const PrefixWork b) {
  __shared__ PrefixEntry found[4];  // the row's prefix and tail, the sums of both works
  __shared__ int is;
  __shared__ float joint[kPrefixJoinMost][10];
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  if (tid == 0) is = 0;
  __syncthreads();
  griddep_launch_dependents();
  griddep_wait();
  const int row = blockIdx.x, kvh = blockIdx.y;
  const PrefixEntry* sequences = b.table + (p.prefixes - b.first);
  if (tid == 0) found[2] = a.table[a.count];
  if (tid == 1) found[3] = b.table[b.count];
  for (int s = tid; s < p.sequences; s += threads) {
    const PrefixEntry x = sequences[s];
    if (x.row <= row && row < x.row + x.rows) {
      found[1] = x;
      if (x.prefix >= 0) found[0] = a.table[x.prefix];
      is = 1;
    }
  }
  __syncthreads();
  if (is == 0 || found[2].bad || found[3].bad) return;
  const PrefixEntry &front = found[0], &tail = found[1];
  if (min(tail.first_seen + row - tail.row, tail.key1) <= 0) return;
  const int lanes = D / 8, most = p.group * lanes;
  for (int i0 = 0; i0 < most; i0 += blockDim.x) {  // (one round where blockDim.x threads have all heads)
    const int i = i0 + threadIdx.x, g = min(i / lanes, p.group - 1), c = i % lanes * 8;
    const bool mine = i < most;
    long long place[2], value[2];  // of the first part's statistics, and of its values from channel c on
    int parts[2], step[2];         // between those and the next four channels
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      place[k] = value[k] = parts[k] = 0, step[k] = 4;
      const PrefixWork& w = k == 0 ? a : b;
      const PrefixEntry &x = k == 0 ? front : tail, &last = found[2 + k];
      if ((k == 0 && tail.prefix < 0) || x.tiles == 0) continue;
      const int at = (row - x.row) * p.group + g, first = kvh * last.units + x.units + at / w.pairs * x.tiles;
      const PrefixShare share(last.units * p.kv_heads, w.workers);
      const int c0 = share.of(first), c1 = share.of(first + x.tiles - 1);
      place[k] = (long long)kvh * last.pairs + x.pairs + at + (long long)c0 * w.pairs;
      value[k] = place[k] * D + c;
      if (w.mixed) {
        const int pair = at % w.pairs, all = min(w.pairs, x.rows * p.group - (at - pair));
        value[k] = (place[k] - pair) * D + pair * 4 + (long long)c * all;
        step[k] = 4 * all;
      }
      parts[k] = c1 - c0 + 1;
    }
    const bool written = tail.key0 == 0 && parts[1] == 1;  // already
    float top = -INFINITY, sum = 0.0f, o[8] = {};
    const int all = mine && !written ? parts[0] + parts[1] : 0;
    for (int j0 = threadIdx.y; j0 < all; j0 += N * blockDim.y) {
      float2 st[N];
      float4 v[N][2];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int j = min(j0 + n * int(blockDim.y), all - 1);
        const bool of_tail = j >= parts[0];
        const long long off = of_tail ? (long long)(j - parts[0]) * b.pairs : (long long)j * a.pairs;
        const float* from = of_tail ? b.part + value[1] + off * D : a.part + value[0] + off * D;
        st[n] = of_tail ? b.stat[place[1] + off] : a.stat[place[0] + off];
        v[n][0] = *reinterpret_cast<const float4*>(from);
        v[n][1] = *reinterpret_cast<const float4*>(from + (of_tail ? step[1] : step[0]));
      }
      float now = top;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (j0 + n * int(blockDim.y) < all) now = fmaxf(now, st[n].x);
      const float base = now == -INFINITY ? 0.0f : now, fix = exp2f(top - base);
      top = now;
      sum *= fix;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= fix;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (j0 + n * int(blockDim.y) >= all || st[n].y == 0.0f) continue;  // (0: a part of which the row sees nothing; of one whose scores are none the sum is none)
        const float f = exp2f(st[n].x - base);
        sum = fmaf(st[n].y, f, sum);
        o[0] = fmaf(v[n][0].x, f, o[0]), o[1] = fmaf(v[n][0].y, f, o[1]), o[2] = fmaf(v[n][0].z, f, o[2]), o[3] = fmaf(v[n][0].w, f, o[3]);
        o[4] = fmaf(v[n][1].x, f, o[4]), o[5] = fmaf(v[n][1].y, f, o[5]), o[6] = fmaf(v[n][1].z, f, o[6]), o[7] = fmaf(v[n][1].w, f, o[7]);
      }
    }
    if (blockDim.y > 1) {  // the threads of one place, in order
      __syncthreads();
      joint[tid][8] = top;
      joint[tid][9] = sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) joint[tid][e] = o[e];
      __syncthreads();
      if (threadIdx.y > 0) continue;
      float now = top;
      for (int y = 1; y < int(blockDim.y); ++y) now = fmaxf(now, joint[y * blockDim.x + threadIdx.x][8]);
      const float base = now == -INFINITY ? 0.0f : now, fix = exp2f(top - base);
      sum *= fix;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= fix;
      for (int y = 1; y < int(blockDim.y); ++y) {
        const float* other = joint[y * blockDim.x + threadIdx.x];
        if (other[9] == 0.0f) continue;
        const float f = exp2f(other[8] - base);
        sum = fmaf(other[9], f, sum);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(other[e], f, o[e]);
      }
    }
    if (all == 0) continue;
    const float inv = 1.0f / sum;
    *reinterpret_cast<uint4*>(p.out + row * p.ldo + (kvh * p.group + g) * D + c) =
        make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv), pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
  }
}

}  // namespace mtx
