// C entry points of the attention over shared prefixes (prefix_attention.cuh).
#include "host_util.cuh"
#include "operator_args.cuh"
#include "prefix_attention.cuh"

extern "C" {

size_t mtx_prefix_attention_scratch_bytes(int rows, int sequences, int prefixes, int num_q_heads, int num_kv_heads, int head_dim) {
  if (rows < 1 || sequences < 1 || prefixes < 0 || num_kv_heads < 1 || num_q_heads < num_kv_heads || head_dim < 1) return 0;
  return 1024;
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
  p.num_pages = num_pages;
  p.tokens_per_page = tokens_per_page;
  p.max_pages = max_pages_per_group;
  p.scale = scale;
  p.softcap = softcap;
  return launch(head_dim == 64 ? prefix_simple_kernel<64> : head_dim == 128 ? prefix_simple_kernel<128> : prefix_simple_kernel<256>, dim3(p.rows, p.heads), dim3(128), 0,
                static_cast<cudaStream_t>(stream), p);
}

}  // extern "C"
