// C entry points of the verification of drafted tokens (verify_drafts.cuh).
#include "host_util.cuh"
#include "operator_args.cuh"
#include "verify_drafts.cuh"

namespace {

constexpr int kMaxVocab = 1 << 28;
constexpr int kMostSequences = 65535;  // (a grid's second dimension)

// Tokens per thread of a chunk: 4 where there is little to read (chunks of 1024 are drawn from in less time, and they fill the SMs), 16 where there is much, and sooner in long rows (where a row's
// sums are many).  With drafts, in us, 4 and 16:  1024 rows of 32768 71, 83;  2048 of 32768 123, 121;  500 of 65536 76.5, 79.2;  1250 of 50000 126, 118;  80 of 128000 38.2, 39.9;  160 of 128000
// 54.5, 52.6;  20 of 264192 35.0, 38.1;  40 of 264192 43.9, 42.4;  320 of 264192 160, 132
constexpr double kVerifyLittle = 36e6;
int verify_each(int rows, int vocab) { return double(rows) * vocab * (vocab > 65536 ? vocab / 65536.0 : 1.0) < kVerifyLittle ? 4 : 16; }
int verify_chunks(int each, int vocab) { return (vocab + 3 - 1) / (each * kVerifyThreads) + 1; }  // (rows begin up to three tokens behind a chunk's)

// Of the differences: chunks of 1024 tokens, or of 2048 beside those of 4096 (64 sequences of 264192 tokens 129.5 us with 4096, 127.0 with 2048, 128.0 with 1024)
constexpr int verify_left_each(int each) { return each == 4 ? 4 : 8; }

// the scratch: sums of chunks of either side, of the differences, tasks, counters
struct VerifyLayout {
  size_t draft, left, task, done, bytes;

  VerifyLayout(int rows, int sequences, int vocab) {
    const int each = verify_each(rows, vocab);
    const size_t chunks = size_t(verify_chunks(each, vocab));
    draft = size_t(rows) * chunks * sizeof(VerifySum);
    left = 2 * draft;
    task = left + size_t(sequences) * verify_chunks(verify_left_each(each), vocab) * sizeof(double);
    done = task + size_t(sequences) * sizeof(VerifyTask);
    bytes = done + size_t(sequences) * sizeof(int);
  }
};

// What every call of at most so many rows, sequences and tokens finds room in: chunks of 1024 tokens of as many rows as may have them (kVerifyLittle / 1024 and a part of one for each row), or larger ones of all
size_t verify_scratch(int rows, int sequences, int vocab) {
  const size_t small = size_t(rows) * verify_chunks(4, vocab), large = size_t(rows) * verify_chunks(16, vocab), little = size_t(kVerifyLittle / 1024) + 1 + size_t(rows) + size_t(rows) / 512 + 1;
  const size_t chunks = large > (small < little ? small : little) ? large : small < little ? small : little;
  return align_up(2 * chunks * sizeof(VerifySum) + size_t(sequences) * (verify_chunks(4, vocab) * sizeof(double) + sizeof(VerifyTask) + sizeof(int)), 256);
}

template <int E>
int launch_verify(const VerifyParams& p, cudaStream_t st) {
  constexpr int kWarps = kVerifyThreads / 32;
  const long long ctas = ((long long)p.rows * p.chunks * (p.draft != nullptr ? 2 : 1) + kWarps - 1) / kWarps;
  if (p.rows > 0) MTX_TRY(launch(verify_sums_kernel<E>, dim3(unsigned(ctas < 4 * 148 ? ctas : 4 * 148)), dim3(kVerifyThreads), 0, st, p));
  MTX_TRY(launch(verify_settle_kernel<E>, dim3(p.sequences), dim3(kVerifyThreads), 0, st, p));
  return p.task != nullptr ? launch(verify_difference_kernel<E, verify_left_each(E)>, dim3((p.left_chunks + kWarps - 1) / kWarps, p.sequences), dim3(kVerifyThreads), 0, st, p) : MTX_OK;
}

}  // namespace

extern "C" {

size_t mtx_verify_drafts_scratch_bytes(int rows, int sequences, int vocab) {
  if (rows < 1 || sequences < 1 || vocab < 1) return 0;
  return verify_scratch(rows, sequences, vocab);
}

int mtx_verify_drafts(const mtx_draft_batch* b, int32_t* accepted, int32_t* emitted, void* scratch, size_t scratch_bytes, mtx_stream stream) {
  if (!b) return fail(MTX_ERR_ARG, "null batch");
  if (b->rows < 0 || b->rows > 1 << 20 || b->sequences < 0 || b->sequences > kMostSequences || b->vocab < 1 || b->vocab > kMaxVocab || b->ld_target < b->vocab || (b->draft && b->ld_draft < b->vocab))
    return fail(MTX_ERR_ARG, "bad rows / sequences / vocab / pitches");
  const int each = verify_each(b->rows, b->vocab), chunks = verify_chunks(each, b->vocab);
  if ((long long)b->rows * chunks >= 1ll << 31) return fail(MTX_ERR_ARG, "rows * vocab is too large for one call");
  if (b->sequences == 0) return MTX_OK;
  if (!accepted || !b->row0 || (b->rows && (!emitted || !b->token || !b->target || !b->accept_u)) || !b->pick_u) return fail(MTX_ERR_ARG, "null argument");
  if (!lie_on(4, {accepted, emitted, b->row0, b->token, b->target, b->draft, b->temperature, b->draft_temperature, b->accept_u, b->pick_u})) return fail(MTX_ERR_ARG, "a batch's arrays lie on 4 bytes");
  if (b->rows && (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) != 0 || scratch_bytes < mtx_verify_drafts_scratch_bytes(b->rows, b->sequences, b->vocab)))
    return fail(MTX_ERR_ARG, "a scratch of mtx_verify_drafts_scratch_bytes() bytes that lies on 16");
  MTX_TRY(on_this_device({accepted, emitted, b->row0, b->token, b->target, b->draft, b->temperature, b->draft_temperature, b->accept_u, b->pick_u, scratch}));
  VerifyParams p;
  memset(&p, 0, sizeof(p));
  p.rows = b->rows;
  p.sequences = b->sequences;
  p.vocab = b->vocab;
  p.row0 = b->row0;
  p.token = b->token;
  p.target = b->target;
  p.ld_target = b->ld_target;
  p.draft = b->draft;
  p.ld_draft = b->ld_draft;
  p.temperature = b->temperature;
  p.draft_temperature = b->draft_temperature;
  p.accept_u = b->accept_u;
  p.pick_u = b->pick_u;
  p.accepted = accepted;
  p.emitted = emitted;
  p.chunks = chunks;
  p.left_chunks = verify_chunks(verify_left_each(each), b->vocab);
  if (b->rows > 0) {
    const VerifyLayout at(b->rows, b->sequences, b->vocab);
    uint8_t* base = static_cast<uint8_t*>(scratch);
    p.target_sum = reinterpret_cast<VerifySum*>(base);
    p.draft_sum = reinterpret_cast<VerifySum*>(base + at.draft);
    p.left = reinterpret_cast<double*>(base + at.left);
    if (b->draft) p.task = reinterpret_cast<VerifyTask*>(base + at.task);
    p.done = reinterpret_cast<int*>(base + at.done);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return each == 4 ? launch_verify<4>(p, st) : launch_verify<16>(p, st);
}

}  // extern "C"
