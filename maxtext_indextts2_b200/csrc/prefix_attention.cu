// C entry points of the attention over shared prefixes (prefix_attention.cuh).
#include <cmath>

#include "host_util.cuh"
#include "operator_args.cuh"
#include "prefix_attention.cuh"

namespace {

constexpr int kPrefixSms = 148;
constexpr int kPrefixWorkers = 2 * kPrefixSms;  // most CTAs of prefix_units_kernel
constexpr int kPrefixTcPairs = 256;             // most pairs of an item of prefix_tc_kernel

int bits_of(int power_of_two) { return __builtin_ctz(unsigned(power_of_two)); }

// Prefixes may go to the tensor cores' kernel when their sequences bring at least 64 pairs on the average (its tiles have 128).
bool prefix_may_tc(int rows, int prefixes, int group) { return prefixes > 0 && (long long)rows * group >= 64ll * prefixes; }

// They do where that kernel, a fifth of the other's time for full tiles of 128 pairs, makes up for what it costs by itself (its launch, and some 20 MB of parts that the join reads): by pairs x
// channels x tokens, as many as the page map has room for.  In us, tensor cores' kernel and tails' kernel, for pairs x tokens of 4 key heads and prefixes that fill the map:
//   64 channels: 320 x 2048 25.1, 21.1;  640 x 2048 24.3, 23.5;  2560 x 512 27.5, 24.8;  320 x 8192 27.9, 33.6;  1280 x 2048 28.0, 32.3
//   128: 512 x 2048 36.6, 32.1;  128 x 8192 35.3, 34.6;  2048 x 512 43.5, 38.1;  256 x 8192 43.1, 50.5;  1024 x 2048 40.5, 49.3;  2048 x 8192 64.7, 260.9
//   256: 256 x 2048 48.0, 41.4;  1024 x 512 54.2, 49.3;  64 x 8192 43.5, 42.0;  128 x 8192 56.0, 65.9;  512 x 2048 49.9, 61.3
bool prefix_on_tc(int rows, int prefixes, int group, int kv_heads, int dim, long long tokens) {
  if (!prefix_may_tc(rows, prefixes, group)) return false;
  const double pairs = double(rows) * group, tiles = ceil(pairs / prefixes / 128.0) * prefixes;
  return (pairs - 128.0 / 5.0 * tiles) * kv_heads * dim * double(tokens) >= (dim == 64 ? 340e6 : 550e6);
}

// the scratch: the entries, a maximum, a sum and weighted values per place; where prefixes have a kernel of their own, the same for them
struct PrefixLayout {
  size_t table[2], stat[2], part[2], bytes;

  PrefixLayout(int rows, int sequences, int prefixes, int heads, int kv_heads, int dim, bool tc) {
    const size_t group = size_t(heads / kv_heads), all = size_t(rows) * group;
    bytes = 0;
    for (int k = 0; k < 2; ++k) {  // prefixes, tails
      // every pair has a place in one tail and at most one prefix, and another in every CTA that shares its item with the CTA before
      const size_t entries = k == 0 ? size_t(prefixes) : size_t(sequences) + size_t(prefixes);
      const size_t extra = k == 0 ? size_t(dim == 256 ? 128 : kPrefixTcPairs) * kPrefixSms : size_t(kPrefixPairs) * kPrefixWorkers;
      const size_t places = k == 0 && !tc ? 0 : all * size_t(kv_heads) * (k == 0 || tc ? 1 : 2) + extra;
      table[k] = bytes;
      stat[k] = table[k] + align_up((entries + 1) * sizeof(PrefixEntry), 256);
      part[k] = stat[k] + align_up(places * sizeof(float2), 256);
      bytes = part[k] + align_up(places * size_t(dim) * sizeof(float), 256);
    }
  }
};

// bf16 rows [rows, ld] that hold `heads` vectors of `dim` side by side, box [64, box_heads, box_rows] with the 128-byte swizzle; what is behind the last row reads as zeros
int make_map_heads(CUtensorMap* m, const void* base, int dim, int heads, int rows, long long ld, int box_heads, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled is not available (no CUDA driver?)");
  const cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(rows)}, strides[2] = {cuuint64_t(dim) * 2, cuuint64_t(ld) * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(box_heads), cuuint32_t(box_rows)}, estr[3] = {1, 1, 1};
  CUresult rc = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled (heads) failed with CUresult %d", int(rc));
  return MTX_OK;
}

// a pool [rows, dim] in chunks of 64 channels, box [64, box_rows, chunks] with the 128-byte swizzle
int make_map_pool(CUtensorMap* m, const void* base, int dim, uint64_t rows, int box_rows, int chunks) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled is not available (no CUDA driver?)");
  const cuuint64_t dims[3] = {64, rows, cuuint64_t(dim / 64)}, strides[2] = {cuuint64_t(dim) * 2, 128};
  const cuuint32_t box[3] = {64, cuuint32_t(box_rows), cuuint32_t(chunks)}, estr[3] = {1, 1, 1};
  CUresult rc = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled (pool) failed with CUresult %d", int(rc));
  return MTX_OK;
}

template <int D>
int launch_prefix(PrefixAttnParams p, uint8_t* scratch, cudaStream_t st) {
  static std::atomic<uint64_t> done{0}, cap_done{0}, tc_done{0}, tc_cap_done{0};
  constexpr int KT = PrefixShape<D>::KT;
  typedef PrefixTcShape<D> Tc;
  const bool tc = prefix_on_tc(p.rows, p.prefixes, p.group, p.kv_heads, D, (long long)p.max_pages * p.tokens_per_page);
  const PrefixLayout at(p.rows, p.sequences, p.prefixes, p.heads, p.kv_heads, D, tc);
  p.box = p.tokens_per_page < KT ? p.tokens_per_page : KT;
  PrefixWork w[2];
  memset(w, 0, sizeof(w));
  for (int k = 0; k < 2; ++k) {
    w[k].first = k == 1 && tc ? p.prefixes : 0;
    w[k].count = k == 0 ? p.prefixes : p.sequences + (tc ? 0 : p.prefixes);
    w[k].kt = k == 0 ? Tc::KT : KT;
    w[k].pairs = k == 0 ? Tc::NQ * (128 / p.group * p.group) : kPrefixPairs;
    w[k].mixed = k == 0;
    const int box = p.tokens_per_page < w[k].kt ? p.tokens_per_page : w[k].kt;
    w[k].box_bits = bits_of(box);
    w[k].round_bits = bits_of(32 * box / w[k].kt);
    w[k].workers = k == 0 ? kPrefixSms : PrefixShape<D>::kCtas * kPrefixSms;
    w[k].tabled = (k == 1 || tc) && w[k].count > kPrefixCached;
    w[k].table = reinterpret_cast<PrefixEntry*>(scratch + at.table[k]);
    w[k].stat = reinterpret_cast<float2*>(scratch + at.stat[k]);
    w[k].part = reinterpret_cast<float*>(scratch + at.part[k]);
  }
  CUtensorMap tk[2], tv[2];
  const uint64_t pool = uint64_t(p.kv_heads) * p.num_pages * p.tokens_per_page;
  for (int k = tc ? 0 : 1; k < 2; ++k) {
    const int box = 1 << w[k].box_bits, chunks = box == w[k].kt ? D / 64 : 1;
    MTX_TRY(make_map_pool(&tk[k], p.k, D, pool, box, chunks));
    MTX_TRY(make_map_pool(&tv[k], p.v, D, pool, box, chunks));
  }
  if (w[0].tabled || w[1].tabled) MTX_TRY(launch(prefix_plan_kernel, dim3(1), dim3(1024), 0, st, p, w[0], w[1]));
  if (tc) {
    CUtensorMap tq;
    MTX_TRY(make_map_heads(&tq, p.q, D, p.heads, p.rows, p.ldq, p.group, 128 / p.group));
    auto kernel = p.softcap > 0.0f ? prefix_tc_kernel<D, true> : prefix_tc_kernel<D, false>;
    MTX_TRY(allow_smem(kernel, prefix_tc_smem_bytes<D>(), p.softcap > 0.0f ? tc_cap_done : tc_done));
    MTX_TRY(launch(kernel, dim3(w[0].workers), dim3(Tc::kThreads), prefix_tc_smem_bytes<D>(), st, tq, tk[0], tv[0], p, w[0]));
  }
  auto units = p.softcap > 0.0f ? prefix_units_kernel<D, true> : prefix_units_kernel<D, false>;
  MTX_TRY(allow_smem(units, prefix_smem_bytes<D>(), p.softcap > 0.0f ? cap_done : done));
  MTX_TRY(launch(units, dim3(w[1].workers), dim3(kPrefixThreads), prefix_smem_bytes<D>(), st, tk[1], tv[1], p, w[1]));
  // the join: some 800 threads of an SM, several of them for each place where rows and key heads are few (64 of 860 CTAs: drafts of 48 sequences 54.0 us, twice as many 53.4, four times 56.0);
  // where they are fewer than two per SM, six parts in flight and not four (64 rows of 4 key heads 33.6 us, not 35.0; the 860 CTAs 55.4, not 53.4)
  const int lanes = p.group * (D / 8) < 128 ? (p.group * (D / 8) + 31) / 32 * 32 : 128;
  const long long ctas = (long long)p.rows * p.kv_heads, room = 800ll * kPrefixSms / (ctas * lanes);
  const int shares = room < 1 ? 1 : room < kPrefixJoinMost / lanes ? int(room) : kPrefixJoinMost / lanes;
  return launch(ctas < 2 * kPrefixSms ? prefix_join_kernel<D, 6> : prefix_join_kernel<D, 4>, dim3(p.rows, p.kv_heads), dim3(lanes, shares), 0, st, p, tc ? w[0] : w[1], w[1]);
}

}  // namespace

extern "C" {

size_t mtx_prefix_attention_scratch_bytes(int rows, int sequences, int prefixes, int num_q_heads, int num_kv_heads, int head_dim) {
  if (rows < 1 || sequences < 1 || prefixes < 0 || num_kv_heads < 1 || num_q_heads < num_kv_heads || head_dim < 1) return 0;
  // with a kernel of their own for the prefixes there are more places, and as many entries: enough for every smaller call, whichever kernel its prefixes have
  return PrefixLayout(rows, sequences, prefixes, num_q_heads, num_kv_heads, head_dim, prefixes > 0).bytes;
}

int mtx_prefix_attention(const void* q, long long ldq, const void* k_pages, const void* v_pages, const mtx_prefix_batch* b, void* out, long long ldo, int num_q_heads,
                         int num_kv_heads, int head_dim, int num_pages, int tokens_per_page, int max_pages_per_group, float scale, float softcap, void* scratch,
                         size_t scratch_bytes, mtx_stream stream) {
  if (!b) return fail(MTX_ERR_ARG, "null batch");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(MTX_ERR_UNSUPPORTED, "head_dim %d: only 64, 128 and 256", head_dim);
  if (num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 16 || num_q_heads > 1024)
    return fail(MTX_ERR_UNSUPPORTED, "a key head has 1 to 16 query heads");
  if (tokens_per_page < 8 || (tokens_per_page & (tokens_per_page - 1)) != 0) return fail(MTX_ERR_UNSUPPORTED, "tokens_per_page must be a power of two >= 8");
  if (num_pages < 1 || max_pages_per_group < 1 || (long long)max_pages_per_group * tokens_per_page >= 1ll << 30) return fail(MTX_ERR_ARG, "bad page counts");
  if ((long long)num_kv_heads * num_pages * tokens_per_page >= 1ll << 31) return fail(MTX_ERR_UNSUPPORTED, "the page pool has too many rows for one tensor map");
  if (b->rows < 0 || b->rows > 1 << 20 || b->sequences < 0 || b->sequences > 1 << 16 || b->prefixes < 0 || b->prefixes > b->sequences) return fail(MTX_ERR_ARG, "bad rows / sequences / prefixes");
  const long long wide = (long long)num_q_heads * head_dim;
  const double blocks = 2.0 * b->rows * (num_q_heads / num_kv_heads) / kPrefixPairs + b->sequences + b->prefixes, tiles = double(max_pages_per_group) * tokens_per_page * head_dim / 4096 + 1;
  if (blocks * num_kv_heads * tiles >= double(1ll << 31)) return fail(MTX_ERR_ARG, "rows * tokens is too large for one call");
  if (ldq < wide || ldo < wide) return fail(MTX_ERR_ARG, "bad pitches");
  if (!(scale > 0.0f && scale < INFINITY) || !(softcap >= 0.0f && softcap < INFINITY)) return fail(MTX_ERR_ARG, "scale is positive, softcap not negative");
  if (b->rows == 0 || b->sequences == 0) return MTX_OK;
  if (!q || !k_pages || !v_pages || !out || !b->row0 || !b->lengths || !b->page_map || (b->prefixes && (!b->prefix_seq0 || !b->prefix_len))) return fail(MTX_ERR_ARG, "null argument");
  if (!lie_on(16, {q, k_pages, v_pages, out}) || ldq % 8 != 0 || ldo % 8 != 0) return fail(MTX_ERR_ARG, "q, out and the pages lie on 16 bytes, with pitches of whole 16 bytes");
  if (!lie_on(4, {b->row0, b->lengths, b->page_map, b->prefixes ? b->prefix_seq0 : nullptr, b->prefixes ? b->prefix_len : nullptr})) return fail(MTX_ERR_ARG, "a batch's arrays lie on 4 bytes");
  if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255) != 0 || scratch_bytes < mtx_prefix_attention_scratch_bytes(b->rows, b->sequences, b->prefixes, num_q_heads, num_kv_heads, head_dim))
    return fail(MTX_ERR_ARG, "a scratch of mtx_prefix_attention_scratch_bytes() bytes that lies on 256");
  MTX_TRY(on_this_device({q, k_pages, v_pages, out, b->row0, b->lengths, b->page_map, b->prefixes ? b->prefix_seq0 : nullptr, b->prefixes ? b->prefix_len : nullptr, scratch}));
  PrefixAttnParams p;
  memset(&p, 0, sizeof(p));
  p.q = static_cast<const bf16*>(q);
  p.ldq = ldq;
  p.k = static_cast<const bf16*>(k_pages);
  p.v = static_cast<const bf16*>(v_pages);
  p.out = static_cast<bf16*>(out);
  p.ldo = ldo;
  p.rows = b->rows;
  p.sequences = b->sequences;
  p.prefixes = b->prefixes;
  p.row0 = b->row0;
  p.lengths = b->lengths;
  p.page_map = b->page_map;
  p.prefix_seq0 = b->prefix_seq0;
  p.prefix_len = b->prefix_len;
  p.heads = num_q_heads;
  p.kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.num_pages = num_pages;
  p.tokens_per_page = tokens_per_page;
  p.page_bits = bits_of(tokens_per_page);
  p.max_pages = max_pages_per_group;
  p.scale = scale;
  p.softcap = softcap;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* at = static_cast<uint8_t*>(scratch);
  return head_dim == 64 ? launch_prefix<64>(p, at, st) : head_dim == 128 ? launch_prefix<128>(p, at, st) : launch_prefix<256>(p, at, st);
}

int mtx_prefix_attention_stalls(uint32_t* count) {
  if (!count) return fail(MTX_ERR_ARG, "null argument");
  MTX_CUDA(cudaDeviceSynchronize());  // (the copy below does not wait for streams that do not block)
  MTX_CUDA(cudaMemcpyFromSymbol(count, d_prefix_waits_failed, sizeof(uint32_t)));
  return MTX_OK;
}

}  // extern "C"
