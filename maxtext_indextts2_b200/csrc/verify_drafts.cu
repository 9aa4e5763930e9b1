// C entry points of the verification of drafted tokens (verify_drafts.cuh).
#include "host_util.cuh"
#include "operator_args.cuh"
#include "verify_drafts.cuh"

namespace {

constexpr int kMaxVocab = 1 << 28;

}  // namespace

extern "C" {

size_t mtx_verify_drafts_scratch_bytes(int rows, int sequences, int vocab) {
  if (rows < 1 || sequences < 1 || vocab < 1) return 0;
  return 1024;
}

int mtx_verify_drafts(const mtx_draft_batch* b, int32_t* accepted, int32_t* emitted, void* scratch, size_t scratch_bytes, mtx_stream stream) {
  if (!b) return fail(MTX_ERR_ARG, "null batch");
  if (b->rows < 0 || b->rows > 1 << 20 || b->sequences < 0 || b->sequences > 1 << 16 || b->vocab < 1 || b->vocab > kMaxVocab || b->ld_target < b->vocab || (b->draft && b->ld_draft < b->vocab))
    return fail(MTX_ERR_ARG, "bad rows / sequences / vocab / pitches");
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
  return launch(verify_simple_kernel, dim3(p.sequences), dim3(kVerifyThreads), 0, static_cast<cudaStream_t>(stream), p);
}

}  // extern "C"
