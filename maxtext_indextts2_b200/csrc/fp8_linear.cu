// C entry points of the 8-bit products (fp8_linear.cuh).
#include <climits>

#include "host_util.cuh"
#include "fp8_linear.cuh"
#include "operator_args.cuh"

namespace {

constexpr int kMost = 1 << 30;  // rows and columns: their numbers, rounded up to a tile, stay 32-bit

bool fits16(const void* p, long long pitch_bytes) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch_bytes % 16 == 0; }

int blocks_of(int k) { return (k + kScaleBlock - 1) / kScaleBlock; }

template <class T>
int launch_quantize(const QuantParams& p, int block_rows, cudaStream_t st) {
  const bool vec = fits16(p.x, p.ldx * (long long)sizeof(T));
  if (block_rows == 1) {
    const long long units = (long long)p.rows * ((p.blocks + kQuantGroup - 1) / kQuantGroup);
    const dim3 grid(unsigned((units + kQuantThreads / 16 - 1) / (kQuantThreads / 16)));
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

// what a linear keeps of its quantised activations in the caller's scratch: the values at a pitch of whole 16 bytes, then a block's scales side by side
size_t scratch_pitch(int k) { return align_up(size_t(k), 16); }
size_t scratch_scales_at(int rows, int k) { return align_up(size_t(rows) * scratch_pitch(k), 256); }

// 8-bit rows [rows, k] in boxes of `box_rows` rows x 128 columns with the 128-byte swizzle; columns behind k and rows behind the last read as zeros
int make_map_e4m3(CUtensorMap* m, const void* base, long long k, long long rows, long long ld, uint32_t box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled is not available (no CUDA driver?)");
  const cuuint64_t dims[2] = {cuuint64_t(k), cuuint64_t(rows)}, strides[1] = {cuuint64_t(ld)};
  const cuuint32_t box[2] = {kScaleBlock, box_rows}, estr[2] = {1, 1};
  CUresult rc = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled (e4m3) failed with CUresult %d", int(rc));
  return MTX_OK;
}

// a result [rows, n] in boxes of 32 rows x 128 bytes
int make_map_result(CUtensorMap* m, void* base, bool f32, long long n, long long rows, long long ld) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled is not available (no CUDA driver?)");
  const cuuint64_t dims[2] = {cuuint64_t(n), cuuint64_t(rows)}, strides[1] = {cuuint64_t(ld) * (f32 ? 4 : 2)};
  const cuuint32_t box[2] = {f32 ? 32u : 64u, 32}, estr[2] = {1, 1};
  CUresult rc = fn(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(MTX_ERR_CUDA, "cuTensorMapEncodeTiled (result) failed with CUresult %d", int(rc));
  return MTX_OK;
}

constexpr int kSms = 148;

struct Fp8Call {
  Fp8LinearParams p;
  const void* x;
  long long ldx;
  const void* w;
  long long ldw;
  int k;
};

template <int BN>
constexpr int fp8_stream_most_stages() {
  constexpr int n = 200 * 1024 / fp8_stream_stage_bytes<BN>();
  return n < kFp8MaxStages ? n : kFp8MaxStages;
}

// Parts of the sum that CTAs of a cluster share: as many as leave every CTA an SM to itself, all clusters at once (a cluster lies in one GPC, so that fewer
// large ones fit than SMs).  64 rows of 5120 by 1280 columns: 16.9 us in one part, 8.8 in four, 7.6 in eight; with a CTA of 128 rows of 10240 by 2560 columns
// (20 tiles) 14.6 in six, 24.0 in eight, whose clusters take turns.  More than half as many tiles as SMs: one part (64 x 2560 by 10240, 80 tiles: 11.3 us, 12.6 in two).
// Joining the parts takes as long as `worth` blocks; a sum that sharing shortens by less stays in one part (32 x 1280 by 1280 columns, 10 blocks, in one part 6.3 us,
// in eight 5.7; 32 x 512 by 1280 4.3 and 5.1; 128 x 1280 by 1280 7.2 and 8.1, 128 x 2560 by 1280 10.0 and 8.6).
template <class Kernel>
int cluster_splits(Kernel kernel, int threads, size_t smem, std::atomic<int>* fit, long long tiles, int blocks, int worth) {  // fit[s]: clusters of s CTAs that run at once; 0: not asked yet
  for (int s = kFp8MaxSplits; s > 1; --s) {
    if (s > blocks || tiles * s > kSms) continue;
    int n = fit[s].load(std::memory_order_relaxed);
    if (n == 0) {
      cudaLaunchConfig_t cfg;
      memset(&cfg, 0, sizeof(cfg));
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 1;
      attr.val.clusterDim.y = unsigned(s);
      attr.val.clusterDim.z = 1;
      cfg.gridDim = dim3(kSms / s, s);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = 1;
      }
      fit[s].store(n, std::memory_order_relaxed);
    }
    if (tiles <= n) return blocks - (blocks + s - 1) / s >= worth ? s : 1;
  }
  return 1;
}

template <int BN>
int stream_splits(long long tiles, int blocks, int* splits) {
  static std::atomic<int> fit[kFp8MaxSplits + 1];
  static std::atomic<uint64_t> done{0};
  const size_t smem = fp8_stream_smem_bytes<BN>(fp8_stream_most_stages<BN>());
  MTX_TRY(allow_smem(fp8_stream_kernel<BN>, smem, done));
  *splits = cluster_splits(fp8_stream_kernel<BN>, 64 + 32 * fp8_stream_warps<BN>(), smem, fit, tiles, blocks, BN == 16 ? 5 : BN == 32 ? 7 : 6);
  return MTX_OK;
}

template <class OUT>
int tile_splits(long long tiles, int blocks, int* splits) {
  static std::atomic<int> fit[kFp8MaxSplits + 1];
  static std::atomic<uint64_t> done{0};
  MTX_TRY(allow_smem(fp8_tile_kernel<128, OUT>, fp8_tile_smem<128>(), done));
  *splits = cluster_splits(fp8_tile_kernel<128, OUT>, kFp8TileThreads, fp8_tile_smem<128>(), fit, tiles, blocks, 12);
  return MTX_OK;
}

template <int BN>
int launch_stream(const Fp8Call& c, cudaStream_t st) {
  constexpr int kPerSm = BN <= 32 ? 3 : 2;  // CTAs that may share an SM
  constexpr int kLeast = BN == 32 ? 3 : 4;
  static_assert(kLeast >= fp8_stream_buffers<BN>(), "a stage's barrier would turn twice before the sums have seen it");
  Fp8LinearParams p = c.p;
  const long long tiles = (p.n + 127) / 128;
  if (tiles * p.blocks >= 1ll << 31) return fail(MTX_ERR_ARG, "too many tiles for one call");
  MTX_TRY(stream_splits<BN>(tiles, p.blocks, &p.splits));
  // an SM's shared memory in stages, whether one CTA has it or several: 64 KB in flight are too few for a CTA alone (16 x 2560 by 10240, 80 CTAs: 11.1 us, 8.8 with all)
  const long long per_sm = (tiles * p.splits + kSms - 1) / kSms;
  p.stages = per_sm >= kPerSm ? kLeast : kLeast * kPerSm / int(per_sm);
  if (p.stages > fp8_stream_most_stages<BN>()) p.stages = fp8_stream_most_stages<BN>();
  const size_t smem = fp8_stream_smem_bytes<BN>(p.stages);
  CUtensorMap tw, tx;
  MTX_TRY(make_map_e4m3(&tw, c.w, c.k, p.n, c.ldw, 128));
  MTX_TRY(make_map_e4m3(&tx, c.x, c.k, p.rows, c.ldx, BN));
  const dim3 grid(unsigned(p.splits > 1 || tiles < kSms * kPerSm ? tiles : kSms * kPerSm), unsigned(p.splits));
  g_cluster_y = p.splits;
  const int rc = launch(fp8_stream_kernel<BN>, grid, dim3(64 + 32 * fp8_stream_warps<BN>()), smem, st, tw, tx, p);
  g_cluster_y = 1;
  return rc;
}

// A TMA store writes whole 16 bytes: of a box across the end of a row it would fill the values behind the last column, up to seven, with zeros.
template <class OUT>
int tma_columns(const Fp8LinearParams& p) {
  if (!fits16(p.out, p.ldo * (long long)sizeof(OUT))) return 0;
  return p.n % int(16 / sizeof(OUT)) == 0 ? INT_MAX : p.n;
}

template <class OUT>
int launch_pair(const Fp8Call& c, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  static_assert(kFp8PairStages >= 512 / kFp8PairCols, "a stage's barrier would turn twice before the sums have seen it");
  Fp8LinearParams p = c.p;
  const long long tiles = (long long)((p.rows + kFp8PairRows - 1) / kFp8PairRows) * ((p.n + kFp8PairCols - 1) / kFp8PairCols);
  if (tiles * p.blocks >= 1ll << 31) return fail(MTX_ERR_ARG, "too many tiles for one call");
  p.stages = kFp8PairStages;
  p.tma_cols = tma_columns<OUT>(p);
  MTX_TRY(allow_smem(fp8_pair_kernel<OUT>, kFp8PairSmem, done));
  CUtensorMap tw, tx, to;
  MTX_TRY(make_map_e4m3(&tw, c.w, c.k, p.n, c.ldw, kFp8PairCols / 2));
  MTX_TRY(make_map_e4m3(&tx, c.x, c.k, p.rows, c.ldx, 128));
  if (p.tma_cols > 0) MTX_TRY(make_map_result(&to, p.out, p.out_f32, p.n, p.rows, p.ldo));
  else to = tx;  // (not read)
  const unsigned pairs = unsigned(tiles < kSms / 2 ? tiles : kSms / 2);
  g_cluster_x = 2;
  const int rc = launch(fp8_pair_kernel<OUT>, dim3(2 * pairs), dim3(kFp8PairThreads), kFp8PairSmem, st, tw, tx, to, p);
  g_cluster_x = 1;
  return rc;
}

template <int BN, class OUT>
int launch_tile(const Fp8Call& c, int splits, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  static_assert(fp8_tile_stages<BN>() >= 512 / BN, "a stage's barrier would turn twice before the sums have seen it");
  Fp8LinearParams p = c.p;
  const long long tiles = (long long)((p.rows + 127) / 128) * ((p.n + BN - 1) / BN);
  if (tiles * p.blocks >= 1ll << 31) return fail(MTX_ERR_ARG, "too many tiles for one call");
  p.stages = fp8_tile_stages<BN>();
  p.splits = splits;
  p.tma_cols = tma_columns<OUT>(p);
  MTX_TRY(allow_smem(fp8_tile_kernel<BN, OUT>, fp8_tile_smem<BN>(), done));
  CUtensorMap tw, tx, to;
  MTX_TRY(make_map_e4m3(&tw, c.w, c.k, p.n, c.ldw, BN));
  MTX_TRY(make_map_e4m3(&tx, c.x, c.k, p.rows, c.ldx, 128));
  if (p.tma_cols > 0) MTX_TRY(make_map_result(&to, p.out, p.out_f32, p.n, p.rows, p.ldo));
  else to = tx;  // (not read)
  g_cluster_y = splits;
  const int rc = launch(fp8_tile_kernel<BN, OUT>, dim3(unsigned(tiles < kSms ? tiles : kSms), unsigned(splits)), dim3(kFp8TileThreads), fp8_tile_smem<BN>(), st, tw, tx, to, p);
  g_cluster_y = 1;
  return rc;
}

// Which kernel: up to 64 rows the streamed weights.  Above, each form's time as it was measured, in ns: what a call takes besides its blocks, and in every wave of
// tiles the blocks (which take longer where rows of weights do not begin with a line of L2, and in CTAs of 256 columns with the SMs that take in as much) and the
// tile's end, which goes by the results' type and place.  Measured, us:
//                                    128 columns   256 columns   pairs
//   333 x 5120 by 1280                      10.1          21.2    22.6
//   128 x 2560 by 10240                     11.3          14.2    15.3
//   333 x 2560 by 10240                     18.1          14.9    25.5
//   128 x 5376 by 21504                     34.6          27.1    44.9
//   333 x 5376 by 21504                     60.7          44.8    63.7
//   1000 x 2560 by 10240                    39.9          35.5    35.9
//   2048 x 5376 by 21504                   271.6         213.9   210.4
//   4096 x 5376 by 21504                   533.4         416.1   404.9
//   153 x 7306 by 10997, fp32               53.3          41.9    35.6
int launch_linear(const Fp8Call& c, cudaStream_t st) {
  const int rows = c.p.rows;
  if (rows <= 16) return launch_stream<16>(c, st);
  if (rows <= 32) return launch_stream<32>(c, st);
  if (rows <= 64) return launch_stream<64>(c, st);
  const bool f32 = c.p.out_f32, aligned = fits16(c.p.out, c.p.ldo * (f32 ? 4 : 2)), lines = c.ldw % 128 == 0;
  const int end = (f32 ? 2 : 0) + (aligned ? 0 : 1);
  const long long blocks = c.p.blocks, m = (rows + 127) / 128, tiles = m * ((c.p.n + 127) / 128), wide = m * ((c.p.n + 255) / 256), pairs = (m + 1) / 2 * ((c.p.n + 255) / 256);
  int splits;
  if (f32) MTX_TRY(tile_splits<float>(tiles, c.p.blocks, &splits));
  else MTX_TRY(tile_splits<bf16>(tiles, c.p.blocks, &splits));
  constexpr int kTileEnd[4] = {500, 1100, 1400, 2400}, kWideEnd[4] = {1800, 4900, 4100, 6000}, kPairEnd[4] = {1800, 3700, 3850, 5800};  // bf16 in place, at odd places, fp32 both
  const long long waves = (wide + kSms - 1) / kSms;
  const long long tile = 4700 + (splits > 1 ? 2600 : 0) + (tiles * splits + kSms - 1) / kSms * ((blocks + splits - 1) / splits * (lines ? 300 : 370) + kTileEnd[end]);
  const long long wide_ns = 4300 + waves * (blocks * ((lines ? 360 : 450) + 90 * wide / (waves * kSms)) + kWideEnd[end]);
  const long long pair = 4300 + (pairs + kSms / 2 - 1) / (kSms / 2) * (blocks * (lines ? 430 : 460) + kPairEnd[end]);
  if (tile <= wide_ns && tile <= pair) return f32 ? launch_tile<128, float>(c, splits, st) : launch_tile<128, bf16>(c, splits, st);
  if (wide_ns <= pair) return f32 ? launch_tile<256, float>(c, 1, st) : launch_tile<256, bf16>(c, 1, st);
  return f32 ? launch_pair<float>(c, st) : launch_pair<bf16>(c, st);
}

}  // namespace

extern "C" {

int mtx_quantize_fp8(const void* x, int x_type, long long ldx, int rows, int k, int block_rows, void* q, long long ldq, float* scale, mtx_stream stream) {
  if (x_type != MTX_BF16 && x_type != MTX_F32) return fail(MTX_ERR_ARG, "x_type %d: values of type MTX_BF16 or MTX_F32 are quantised", x_type);
  if (block_rows != 1 && block_rows != kScaleBlock) return fail(MTX_ERR_ARG, "block_rows is 1 (activations) or 128 (weights), not %d", block_rows);
  if (rows < 0 || rows > kMost || k < 1 || k > kMost || ldx < k || ldq < k) return fail(MTX_ERR_ARG, "bad rows / k / ldx / ldq");
  if (rows == 0) return MTX_OK;
  if (!x || !q || !scale) return fail(MTX_ERR_ARG, "null argument");
  if (!fits16(q, ldq)) return fail(MTX_ERR_ARG, "8-bit values lie at a 16-byte aligned base and a pitch of whole 16 bytes");
  if (!lie_on(x_type == MTX_BF16 ? 2 : 4, {x}) || !lie_on(4, {scale})) return fail(MTX_ERR_ARG, "x and scale lie on multiples of their types' sizes");
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
  if (rows < 0 || rows > kMost || n < 1 || n > kMost || k < 1 || k > kMost || ldx < k || ldw < k || ldo < n) return fail(MTX_ERR_ARG, "bad rows / n / k / ldx / ldw / ldo");
  if (rows == 0) return MTX_OK;
  const bool quantised = x_type == MTX_E4M3;
  if (!x || !wq || !w_scale || !out || (quantised && !x_scale)) return fail(MTX_ERR_ARG, "null argument");
  if (!fits16(wq, ldw) || (quantised && !fits16(x, ldx))) return fail(MTX_ERR_ARG, "8-bit values lie at a 16-byte aligned base and a pitch of whole 16 bytes");
  if ((long long)rows * blocks_of(k) >= 1ll << 31) return fail(MTX_ERR_ARG, "more than 2^31 blocks");
  if (!quantised && (!scratch || scratch_bytes < mtx_linear_fp8_scratch_bytes(rows, k) || (reinterpret_cast<uintptr_t>(scratch) & 15) != 0))
    return fail(MTX_ERR_ARG, "values that are quantised here need a 16-byte aligned scratch of mtx_linear_fp8_scratch_bytes(rows, k) bytes");
  if (!lie_on(x_type == MTX_BF16 ? 2 : 4, {x}) || !lie_on(out_type == MTX_BF16 ? 2 : 4, {out}) || !lie_on(4, {w_scale, quantised ? x_scale : nullptr}))
    return fail(MTX_ERR_ARG, "x, out and the scales lie on multiples of their types' sizes");
  MTX_TRY(on_this_device({x, quantised ? x_scale : static_cast<const void*>(scratch), wq, w_scale, out}));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Fp8Call c;
  memset(&c, 0, sizeof(c));
  c.x = x;
  c.ldx = ldx;
  c.w = wq;
  c.ldw = ldw;
  c.k = k;
  c.p.x_scale = x_scale;
  c.p.blocks = blocks_of(k);
  c.p.x_scale_row = c.p.blocks;
  c.p.x_scale_block = 1;
  if (!quantised) {
    uint8_t* q = static_cast<uint8_t*>(scratch);
    float* scales = reinterpret_cast<float*>(q + scratch_scales_at(rows, k));
    c.p.x_scale_row = 1;  // (a block's scales side by side: neighbouring threads have neighbouring rows)
    c.p.x_scale_block = rows;
    MTX_TRY(quantize(x, x_type, ldx, rows, k, 1, q, (long long)scratch_pitch(k), scales, c.p.x_scale_row, c.p.x_scale_block, st));
    c.x = q;
    c.ldx = (long long)scratch_pitch(k);
    c.p.x_scale = scales;
    c.p.early = 1;
  }
  c.p.w_scale = w_scale;
  c.p.out = out;
  c.p.ldo = ldo;
  c.p.out_f32 = out_type == MTX_F32;
  c.p.rows = rows;
  c.p.n = n;
  return launch_linear(c, st);
}

int mtx_linear_fp8_stalls(uint32_t* count) {
  if (!count) return fail(MTX_ERR_ARG, "null argument");
  MTX_CUDA(cudaDeviceSynchronize());  // (the copy below does not wait for streams that do not block)
  MTX_CUDA(cudaMemcpyFromSymbol(count, d_fp8_waits_failed, sizeof(uint32_t)));
  return MTX_OK;
}

}  // extern "C"
