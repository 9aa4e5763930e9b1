// C entry points of the operators that go through a batch row by row: residual sums with norms (add_rmsnorm.cuh) and rotary positions (rotary.cuh).
#include <cmath>

#include "host_util.cuh"
#include "add_rmsnorm.cuh"
#include "operator_args.cuh"
#include "rotary.cuh"

namespace {

constexpr int kMostRows = 1 << 30;
constexpr int kMostWidth = 32768;  // four times eight values in each of 1024 threads

int value_bytes(int type) { return type == MTX_F32 ? 4 : type == MTX_BF16 ? 2 : 1; }

// Threads of a row, each with J times eight of its values: a warp up to 512 values (no barrier, eight rows in a CTA), then as many warps as have eight values for each lane, from 4096
// values on twice eight, from 16384 on four times.  Where rows wait for SMs (more than 148) and a row's registers would leave room for one CTA, it has fewer, for two: to 8 bits 2000 rows of
// 10000 took 59.9 us with one, 43.8 so, 1600 of 14336 with three times eight 51.4, not 64.0 (with x of 32 bits 82.0, not 70.9: not there).  100 rows of 10000 or 14336 took 5.8 and 8.2 us with
// one, 6.3 and 9.2 so.
template <class TX, class TR, bool E4M3, bool VEC>
int launch_norm_rows(const AddNormParams& p, cudaStream_t st) {
  const int lanes = (p.width + 7) / 8;
  if (lanes <= 64) {
    const dim3 grid((p.rows + kNormWarpRows - 1) / kNormWarpRows), block(32, kNormWarpRows);
    return launch(lanes <= 32 ? add_rmsnorm_kernel<TX, TR, E4M3, VEC, 1, 256> : add_rmsnorm_kernel<TX, TR, E4M3, VEC, 2, 256>, grid, block, 0, st, p);
  }
  const bool two = p.rows > 148;
  const int each = lanes <= 512 ? 1 : lanes > 1536 && lanes <= 1920 && two && sizeof(TX) == 2 ? 3 : lanes <= 2048 ? 2 : 4, threads = ((lanes + each - 1) / each + 31) / 32 * 32;
  return launch(each == 1 ? (threads <= 256 ? add_rmsnorm_kernel<TX, TR, E4M3, VEC, 1, 256> : add_rmsnorm_kernel<TX, TR, E4M3, VEC, 1, 512>)
                : each == 2 ? (threads <= 512          ? add_rmsnorm_kernel<TX, TR, E4M3, VEC, 2, 512>
                               : threads <= 768 && two ? add_rmsnorm_kernel<TX, TR, E4M3, VEC, 2, 768>
                                                       : add_rmsnorm_kernel<TX, TR, E4M3, VEC, 2, 1024>)
                : each == 3 ? add_rmsnorm_kernel<TX, TR, E4M3, VEC, 3, 640>
                            : (threads <= 768 ? add_rmsnorm_kernel<TX, TR, E4M3, VEC, 4, 768> : add_rmsnorm_kernel<TX, TR, E4M3, VEC, 4, 1024>),
                dim3(p.rows), dim3(threads), 0, st, p);
}

template <class TX, class TR>
int launch_add_rmsnorm(const AddNormParams& p, bool vec, cudaStream_t st) {
  if (p.out_type == MTX_E4M3) return vec ? launch_norm_rows<TX, TR, true, true>(p, st) : launch_norm_rows<TX, TR, true, false>(p, st);
  return vec ? launch_norm_rows<TX, TR, false, true>(p, st) : launch_norm_rows<TX, TR, false, false>(p, st);
}

// whether rows lie on 16 bytes
bool rows_on_16(const void* base, long long pitch, int size) { return ((reinterpret_cast<uintptr_t>(base) | uintptr_t(pitch * size)) & 15) == 0; }

template <class TI, class TO>
int launch_rotary(const RotaryParams& p, bool vec, cudaStream_t st) {
  const int step = vec ? 8 : 1;
  const long long units = (long long)(p.heads + p.kv_heads) * (p.dim - p.pairs) / step + (p.k_pages != nullptr ? (long long)p.kv_heads * p.dim / step : 0);
  const int threads = units < kRotaryThreads ? int(units + 31) / 32 * 32 : kRotaryThreads;
  // as many tokens per CTA as bring the grid to whole waves of the 1024 threads that an SM has room for, in as few as the most tokens allow: 1000 tokens of 24 heads of 128 channels 5.3 us, 7.2 with
  // one token in each of 1000 CTAs; 4001 14.3 us in one wave of CTAs of ten, 16.0 with six in one and a half
  const int most = p.pairs <= 256 ? kRotaryTokens : 4096 / p.pairs;  // (cosines and sines of up to 32 KB)
  const int room = 148 * (1024 / threads), waves = (p.rows + room * most - 1) / (room * most), tokens = (p.rows + waves * room - 1) / (waves * room);
  return launch(vec ? rotary_kernel<TI, TO, true> : rotary_kernel<TI, TO, false>, dim3((p.rows + tokens - 1) / tokens), dim3(threads), size_t(tokens) * p.pairs * sizeof(float2), st,
                p, tokens);
}

// a result in an input's place, but not value by value
bool misplaced(const void* in, long long ld_in, int type_in, const void* out, long long ld_out, int type_out) { return in == out && (ld_in != ld_out || type_in != type_out); }

}  // namespace

extern "C" {

int mtx_add_rmsnorm(const void* x, int x_type, long long ldx, const void* residual, int residual_type, long long ld_residual, void* sum, long long ld_sum, const void* weight,
                    int weight_type, float weight_offset, float eps, void* out, int out_type, long long ldo, float* out_scale, int rows, int width, mtx_stream stream) {
  if (x_type != MTX_BF16 && x_type != MTX_F32) return fail(MTX_ERR_ARG, "x_type %d is neither MTX_BF16 nor MTX_F32", x_type);
  if (residual && residual_type != MTX_BF16 && residual_type != MTX_F32) return fail(MTX_ERR_ARG, "residual_type %d is neither MTX_BF16 nor MTX_F32", residual_type);
  if (weight && weight_type != MTX_BF16 && weight_type != MTX_F32) return fail(MTX_ERR_ARG, "weight_type %d is neither MTX_BF16 nor MTX_F32", weight_type);
  if (out_type != MTX_BF16 && out_type != MTX_F32 && out_type != MTX_E4M3) return fail(MTX_ERR_ARG, "out_type %d is none of MTX_BF16, MTX_F32 and MTX_E4M3", out_type);
  if (rows < 0 || rows > kMostRows || width < 1 || width > kMostWidth || ldx < width || ldo < width || (residual && ld_residual < width) || (sum && ld_sum < width))
    return fail(MTX_ERR_ARG, "bad rows / width / pitches (rows of up to %d values)", kMostWidth);
  if (!(eps >= 0.0f)) return fail(MTX_ERR_ARG, "eps is not negative");
  if (sum && !residual) return fail(MTX_ERR_ARG, "a sum needs a residual");
  if (rows == 0) return MTX_OK;
  if (!x || !out || (out_type == MTX_E4M3 && !out_scale)) return fail(MTX_ERR_ARG, "null argument");
  if (out_type == MTX_E4M3 && ((reinterpret_cast<uintptr_t>(out) & 15) != 0 || ldo % 16 != 0))
    return fail(MTX_ERR_ARG, "8-bit values lie at a 16-byte aligned base and a pitch of whole 16 bytes");
  if (!lie_on(value_bytes(x_type), {x}) || (residual && !lie_on(value_bytes(residual_type), {residual, sum})) || (weight && !lie_on(value_bytes(weight_type), {weight})) ||
      !lie_on(value_bytes(out_type), {out}) || !lie_on(4, {out_type == MTX_E4M3 ? out_scale : nullptr}))
    return fail(MTX_ERR_ARG, "values lie on multiples of their types' sizes");
  if (misplaced(x, ldx, x_type, out, ldo, out_type) || (residual && (misplaced(residual, ld_residual, residual_type, out, ldo, out_type) || misplaced(residual, ld_residual, 0, sum, ld_sum, 0) ||
                                                                     (sum && misplaced(x, ldx, x_type, sum, ld_sum, residual_type)))))
    return fail(MTX_ERR_ARG, "results in an input's place have its type and pitch");
  if (sum && sum == out) return fail(MTX_ERR_ARG, "sum and out are two results");
  MTX_TRY(on_this_device({x, residual, sum, weight, out, out_type == MTX_E4M3 ? out_scale : nullptr}));
  AddNormParams p;
  memset(&p, 0, sizeof(p));
  p.x = x;
  p.ldx = ldx;
  p.residual = residual;
  p.ldr = ld_residual;
  p.sum = sum;
  p.lds = ld_sum;
  p.weight = weight;
  p.weight_f32 = weight_type == MTX_F32;
  p.weight_offset = weight_offset;
  p.eps = eps;
  p.out = out;
  p.out_type = out_type;
  p.ldo = ldo;
  p.scale = out_scale;
  p.rows = rows;
  p.width = width;
  p.by_width = 1.0 / width;
  p.blocks = (width + kScaleBlock - 1) / kScaleBlock;
  const bool vec = width % 8 == 0 && rows_on_16(x, ldx, value_bytes(x_type)) && (!residual || rows_on_16(residual, ld_residual, value_bytes(residual_type))) &&
                   (!sum || rows_on_16(sum, ld_sum, value_bytes(residual_type))) && rows_on_16(out, ldo, value_bytes(out_type)) && lie_on(16, {weight});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!residual) return x_type == MTX_F32 ? launch_add_rmsnorm<float, NoResidual>(p, vec, st) : launch_add_rmsnorm<bf16, NoResidual>(p, vec, st);
  if (residual_type == MTX_F32) return x_type == MTX_F32 ? launch_add_rmsnorm<float, float>(p, vec, st) : launch_add_rmsnorm<bf16, float>(p, vec, st);
  return x_type == MTX_F32 ? launch_add_rmsnorm<float, bf16>(p, vec, st) : launch_add_rmsnorm<bf16, bf16>(p, vec, st);
}

int mtx_rotary_frequencies(int rot_dims, double base, int scaling, double factor, double original_len, double low, double high, double* freq, float* amplitude) {
  if (rot_dims < 2 || rot_dims % 2 != 0 || !(base > 1.0) || !std::isfinite(base)) return fail(MTX_ERR_ARG, "bad rot_dims / base");
  if (!freq || !amplitude) return fail(MTX_ERR_ARG, "null argument");
  if (scaling < MTX_ROTARY_PLAIN || scaling > MTX_ROTARY_YARN) return fail(MTX_ERR_ARG, "scaling %d is none of MTX_ROTARY_*", scaling);
  if (scaling != MTX_ROTARY_PLAIN && !(factor >= 1.0 && std::isfinite(factor))) return fail(MTX_ERR_ARG, "a factor of at least 1");
  if (scaling >= MTX_ROTARY_BANDS && !(original_len > 0.0 && low > 0.0 && high > low)) return fail(MTX_ERR_ARG, "original_len and the bands' borders are positive, low < high");
  constexpr double kTurn = 6.283185307179586477;
  const double slower = scaling == MTX_ROTARY_PLAIN ? 1.0 : factor;
  *amplitude = scaling == MTX_ROTARY_YARN && factor > 1.0 ? float(0.1 * std::log(factor) + 1.0) : 1.0f;
  const int pairs = rot_dims / 2;
  // YARN: the pairs that turn `high` and `low` times over the original length, as places in the row of pairs
  double first = std::floor(rot_dims * std::log(original_len / (high * kTurn)) / (2.0 * std::log(base))), last = std::ceil(rot_dims * std::log(original_len / (low * kTurn)) / (2.0 * std::log(base)));
  if (!(first > 0.0)) first = 0.0;
  if (!(last < rot_dims - 1.0)) last = rot_dims - 1.0;
  if (!(last > first)) last = first + 0.001;
  for (int i = 0; i < pairs; ++i) {
    const double f = std::pow(base, -2.0 * i / rot_dims);
    double stretched = 0.0;  // the part of the frequency that is divided by the factor
    if (scaling == MTX_ROTARY_LINEAR) stretched = 1.0;
    if (scaling == MTX_ROTARY_BANDS) stretched = 1.0 - (original_len * f / kTurn - low) / (high - low);
    if (scaling == MTX_ROTARY_YARN) stretched = (i - first) / (last - first);
    stretched = stretched < 0.0 ? 0.0 : stretched > 1.0 ? 1.0 : stretched;
    freq[i] = f * (1.0 - stretched) + f / slower * stretched;
  }
  return MTX_OK;
}

int mtx_rotary(const mtx_rotary_batch* b, mtx_stream stream) {
  if (!b) return fail(MTX_ERR_ARG, "null batch");
  if (b->rows < 0 || b->rows > kMostRows || b->heads < 0 || b->kv_heads < 0 || b->heads + (long long)b->kv_heads < 1 || b->heads > 65536 || b->kv_heads > 65536 || b->dim < 1 || b->dim > kRotaryMostDims ||
      b->rot_dims < 0 || b->rot_dims > b->dim || b->rot_dims % 2 != 0)
    return fail(MTX_ERR_ARG, "bad rows / heads / dim / rot_dims (heads of up to %d channels, an even number of them rotated)", kRotaryMostDims);
  if ((b->type != MTX_BF16 && b->type != MTX_F32) || (b->out_type != MTX_BF16 && b->out_type != MTX_F32)) return fail(MTX_ERR_ARG, "type and out_type are MTX_BF16 or MTX_F32");
  const bool paged = b->k_pages || b->v_pages;
  const long long q_wide = (long long)b->heads * b->dim, k_wide = (long long)b->kv_heads * b->dim;
  if (paged && (!b->k_pages || !b->v_pages || !b->page_map)) return fail(MTX_ERR_ARG, "k_pages, v_pages and page_map together");
  if (paged && (b->kv_heads < 1 || b->groups < 1 || b->num_pages < 1 || b->tokens_per_page < 1 || b->max_pages_per_group < 1)) return fail(MTX_ERR_ARG, "bad groups / pages");
  if (paged && !b->group && b->rows > b->groups) return fail(MTX_ERR_ARG, "without group, row r belongs to group r: %d rows for %d groups", b->rows, b->groups);
  if ((b->heads && (b->ldq < q_wide || b->ldq_out < q_wide)) || (b->kv_heads && b->ldk < k_wide) || (b->k_out && b->ldk_out < k_wide) || (paged && b->ldv < k_wide))
    return fail(MTX_ERR_ARG, "bad pitches");
  if (b->rows == 0) return MTX_OK;
  if (!b->pos || (b->rot_dims && !b->freq) || (b->heads && (!b->q || !b->q_out)) || (b->kv_heads && (!b->k || (!b->k_out && !paged))) || (paged && !b->v)) return fail(MTX_ERR_ARG, "null argument");
  const int in = value_bytes(b->type), out = value_bytes(b->out_type);
  if (!lie_on(in, {b->q, b->k, b->v}) || !lie_on(out, {b->q_out, b->k_out}) || !lie_on(2, {b->k_pages, b->v_pages}) || !lie_on(4, {b->pos, b->group, b->page_map}) || !lie_on(8, {b->freq}))
    return fail(MTX_ERR_ARG, "values lie on multiples of their types' sizes");
  if ((b->heads && misplaced(b->q, b->ldq, b->type, b->q_out, b->ldq_out, b->out_type)) || (b->k_out && misplaced(b->k, b->ldk, b->type, b->k_out, b->ldk_out, b->out_type)))
    return fail(MTX_ERR_ARG, "results in an input's place have its type and pitch");
  RotaryParams p;
  memset(&p, 0, sizeof(p));
  p.rows = b->rows;
  p.heads = b->heads;
  p.kv_heads = b->kv_heads;
  p.dim = b->dim;
  p.pairs = b->rot_dims / 2;
  p.half = b->rot_half != 0;
  p.amplitude = b->amplitude == 0.0f ? 1.0f : b->amplitude;
  p.freq = b->rot_dims ? b->freq : nullptr;
  p.pos = b->pos;
  if (b->heads) p.q = b->q, p.ldq = b->ldq, p.q_out = b->q_out, p.ldq_out = b->ldq_out;
  if (b->kv_heads) p.k = b->k, p.ldk = b->ldk, p.k_out = b->k_out, p.ldk_out = b->k_out ? b->ldk_out : 0;
  if (paged) {
    p.v = b->v;
    p.ldv = b->ldv;
    p.k_pages = static_cast<bf16*>(b->k_pages);
    p.v_pages = static_cast<bf16*>(b->v_pages);
    p.groups = b->groups;
    p.num_pages = b->num_pages;
    p.tokens_per_page = b->tokens_per_page;
    p.max_pages = b->max_pages_per_group;
    p.group = b->group;
    p.page_map = b->page_map;
  }
  MTX_TRY(on_this_device({p.freq, p.pos, p.q, p.k, p.v, p.q_out, p.k_out, p.k_pages, p.v_pages, p.group, p.page_map}));
  const bool vec = p.dim % 8 == 0 && p.pairs % 8 == 0 && rows_on_16(p.q, p.ldq, in) && rows_on_16(p.k, p.ldk, in) && rows_on_16(p.v, p.ldv, in) && rows_on_16(p.q_out, p.ldq_out, out) &&
                   rows_on_16(p.k_out, p.ldk_out, out) && rows_on_16(p.k_pages, 0, 2) && rows_on_16(p.v_pages, 0, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (b->type == MTX_F32) return b->out_type == MTX_F32 ? launch_rotary<float, float>(p, vec, st) : launch_rotary<float, bf16>(p, vec, st);
  return b->out_type == MTX_F32 ? launch_rotary<bf16, float>(p, vec, st) : launch_rotary<bf16, bf16>(p, vec, st);
}

}  // extern "C"
