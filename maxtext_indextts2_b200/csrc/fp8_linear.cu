// C entry points of the 8-bit products (fp8_linear.cuh).
#include "host_util.cuh"
#include "fp8_linear.cuh"
#include "operator_args.cuh"

namespace {

constexpr int kMaxK = 1 << 30;  // (column numbers, rounded up to a block, stay 32-bit)

bool fits16(const void* p, long long pitch_bytes) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch_bytes % 16 == 0; }

int blocks_of(int k) { return (k + kScaleBlock - 1) / kScaleBlock; }

template <class T>
int launch_quantize(const QuantParams& p, int block_rows, cudaStream_t st) {
  const bool vec = fits16(p.x, p.ldx * (long long)sizeof(T));
  if (block_rows == 1) {
    const dim3 grid(unsigned(((long long)p.rows * p.blocks + kQuantThreads / 16 - 1) / (kQuantThreads / 16)));
    return launch(vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, grid, dim3(kQuantThreads), 0, st, p);
  }
  const dim3 grid(unsigned((p.rows + kScaleBlock - 1) / kScaleBlock) * unsigned(p.blocks));
  return launch(vec ? quantize_blocks_kernel<T, true> : quantize_blocks_kernel<T, false>, grid, dim3(kQuantThreads), 0, st, p);
}

int quantize(const void* x, int x_type, long long ldx, int rows, int k, int block_rows, void* q, long long ldq, float* scale, long long scale_row, long long scale_block,
             cudaStream_t st) {
  QuantParams p;
  p.x = x;
  p.ldx = ldx;
  p.rows = rows;
  p.k = k;
  p.blocks = blocks_of(k);
  p.q = static_cast<uint8_t*>(q);
  p.ldq = ldq;
  p.scale = scale;
  p.scale_row = scale_row;
  p.scale_block = scale_block;
  return x_type == MTX_BF16 ? launch_quantize<bf16>(p, block_rows, st) : launch_quantize<float>(p, block_rows, st);
}

// what a linear keeps of its quantised activations in the caller's scratch: the values at a pitch of whole 16 bytes, then a row's scales side by side
size_t scratch_pitch(int k) { return align_up(size_t(k), 16); }
size_t scratch_scales_at(int rows, int k) { return align_up(size_t(rows) * scratch_pitch(k), 256); }

}  // namespace

extern "C" {

int mtx_quantize_fp8(const void* x, int x_type, long long ldx, int rows, int k, int block_rows, void* q, long long ldq, float* scale, mtx_stream stream) {
  if (x_type != MTX_BF16 && x_type != MTX_F32) return fail(MTX_ERR_ARG, "x_type %d: values of type MTX_BF16 or MTX_F32 are quantised", x_type);
  if (block_rows != 1 && block_rows != kScaleBlock) return fail(MTX_ERR_ARG, "block_rows is 1 (activations) or 128 (weights), not %d", block_rows);
  if (rows < 0 || k < 1 || k > kMaxK || ldx < k || ldq < k) return fail(MTX_ERR_ARG, "bad rows / k / ldx / ldq");
  if (rows == 0) return MTX_OK;
  if (!x || !q || !scale) return fail(MTX_ERR_ARG, "null argument");
  if (!fits16(q, ldq)) return fail(MTX_ERR_ARG, "8-bit values lie at a 16-byte aligned base and a pitch of whole 16 bytes");
  if ((long long)rows * blocks_of(k) >= 1ll << 31) return fail(MTX_ERR_ARG, "more than 2^31 blocks");
  MTX_TRY(on_this_device({x, q, scale}));
  return quantize(x, x_type, ldx, rows, k, block_rows, q, ldq, scale, blocks_of(k), 1, static_cast<cudaStream_t>(stream));
}

size_t mtx_linear_fp8_scratch_bytes(int rows, int k) {
  if (rows < 1 || k < 1) return 0;
  return scratch_scales_at(rows, k) + size_t(rows) * blocks_of(k) * sizeof(float);
}

int mtx_linear_fp8(const void* x, int x_type, long long ldx, const float* x_scale, const void* wq, long long ldw, const float* w_scale, void* out, int out_type, long long ldo,
                   int rows, int n, int k, void* scratch, size_t scratch_bytes, mtx_stream stream) {
  if (x_type != MTX_BF16 && x_type != MTX_F32 && x_type != MTX_E4M3) return fail(MTX_ERR_ARG, "x_type %d is none of MTX_BF16, MTX_F32 and MTX_E4M3", x_type);
  if (out_type != MTX_BF16 && out_type != MTX_F32) return fail(MTX_ERR_ARG, "out_type %d: a product is stored as MTX_BF16 or MTX_F32", out_type);
  if (rows < 0 || n < 1 || k < 1 || k > kMaxK || ldx < k || ldw < k || ldo < n) return fail(MTX_ERR_ARG, "bad rows / n / k / ldx / ldw / ldo");
  if (rows == 0) return MTX_OK;
  const bool quantised = x_type == MTX_E4M3;
  if (!x || !wq || !w_scale || !out || (quantised && !x_scale)) return fail(MTX_ERR_ARG, "null argument");
  if (!fits16(wq, ldw) || (quantised && !fits16(x, ldx))) return fail(MTX_ERR_ARG, "8-bit values lie at a 16-byte aligned base and a pitch of whole 16 bytes");
  if ((long long)rows * blocks_of(k) >= 1ll << 31) return fail(MTX_ERR_ARG, "more than 2^31 blocks");
  if (!quantised && (!scratch || scratch_bytes < mtx_linear_fp8_scratch_bytes(rows, k) || (reinterpret_cast<uintptr_t>(scratch) & 15) != 0))
    return fail(MTX_ERR_ARG, "values that are quantised here need a 16-byte aligned scratch of mtx_linear_fp8_scratch_bytes(rows, k) bytes");
  MTX_TRY(on_this_device({x, quantised ? x_scale : static_cast<const void*>(scratch), wq, w_scale, out}));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Fp8LinearParams p;
  p.x = static_cast<const uint8_t*>(x);
  p.ldx = ldx;
  p.x_scale = x_scale;
  p.blocks = blocks_of(k);
  p.x_scale_row = p.blocks;
  p.x_scale_block = 1;
  if (!quantised) {
    uint8_t* q = static_cast<uint8_t*>(scratch);
    float* scales = reinterpret_cast<float*>(q + scratch_scales_at(rows, k));
    MTX_TRY(quantize(x, x_type, ldx, rows, k, 1, q, (long long)scratch_pitch(k), scales, p.x_scale_row, p.x_scale_block, st));
    p.x = q;
    p.ldx = (long long)scratch_pitch(k);
    p.x_scale = scales;
  }
  p.w = static_cast<const uint8_t*>(wq);
  p.ldw = ldw;
  p.w_scale = w_scale;
  p.out = out;
  p.ldo = ldo;
  p.out_f32 = out_type == MTX_F32;
  p.rows = rows;
  p.n = n;
  p.k = k;
  return launch(fp8_linear_kernel, dim3((n + 15) / 16, (rows + 15) / 16), dim3(256), 0, st, p);
}

}  // extern "C"
