// C entry points of the controls of a batch's logits (logit_controls.cuh).
#include "host_util.cuh"
#include "logit_controls.cuh"
#include "operator_args.cuh"

namespace {

constexpr int kMaxVocab = 1 << 28;  // (token numbers, rounded up to what a warp goes through, stay 32-bit)

int check_record(const void* seen, long long ld_seen, const void* touched, long long ld_touched, int slots, int vocab) {
  if (slots < 1 || ld_seen < vocab || ld_seen % 8 != 0 || (reinterpret_cast<uintptr_t>(seen) & 15) != 0)
    return fail(MTX_ERR_ARG, "the record of seen tokens has at least one slot, a 16-byte aligned base and a pitch of whole eight tokens");
  if (touched != nullptr && ((long long)ld_touched * 256 < vocab || (reinterpret_cast<uintptr_t>(touched) & 3) != 0))
    return fail(MTX_ERR_ARG, "touched has a word per 256 tokens");
  return MTX_OK;
}

}  // namespace

extern "C" {

int mtx_control_logits(const float* logits, long long ld, float* out, long long ldo, int rows, int vocab, const mtx_logit_controls* c, mtx_stream stream) {
  if (rows < 0 || vocab < 1 || vocab > kMaxVocab || ld < vocab || ldo < vocab) return fail(MTX_ERR_ARG, "bad rows / vocab / ld / ldo");
  if (!c) return fail(MTX_ERR_ARG, "null controls");
  if (rows == 0) return MTX_OK;
  if (!logits || !out) return fail(MTX_ERR_ARG, "null argument");
  if (!lie_on(4, {logits, out, c->slot, c->repetition, c->presence, c->frequency, c->bias_off, c->bias_token, c->bias_value, c->allowed, c->allowed_row}))
    return fail(MTX_ERR_ARG, "logits and their controls lie on 4 bytes");
  if (logits == out && ld != ldo) return fail(MTX_ERR_ARG, "logits that are controlled in place have one pitch");
  if ((c->repetition || c->presence || c->frequency) && !c->seen) return fail(MTX_ERR_ARG, "penalties need the record of seen tokens");
  ControlParams p;
  memset(&p, 0, sizeof(p));
  if (c->seen) {
    MTX_TRY(check_record(c->seen, c->ld_seen, c->touched, c->ld_touched, c->slots, vocab));
    p.slots = c->slots;
    p.slot = c->slot;
    p.seen = c->seen;
    p.ld_seen = c->ld_seen;
    p.touched = c->touched;
    p.ld_touched = c->ld_touched;
    p.repetition = c->repetition;
    p.presence = c->presence;
    p.frequency = c->frequency;
  }
  if (c->bias_off || c->bias_token || c->bias_value) {
    if (!c->bias_off || !c->bias_token || !c->bias_value) return fail(MTX_ERR_ARG, "biases are bias_off, bias_token and bias_value together");
    p.bias_off = c->bias_off;
    p.bias_token = c->bias_token;
    p.bias_value = c->bias_value;
  }
  if (c->allowed) {
    if (c->allowed_rows < 1 || c->ld_allowed * 32 < vocab) return fail(MTX_ERR_ARG, "allowed has at least one row, and a word per 32 tokens");
    p.allowed_rows = c->allowed_rows;
    p.allowed_row = c->allowed_row;
    p.allowed = c->allowed;
    p.ld_allowed = c->ld_allowed;
  }
  p.logits = logits;
  p.ld = ld;
  p.out = out;
  p.ldo = ldo;
  p.rows = rows;
  p.vocab = vocab;
  const long long runs = (vocab + 2) / kControlRun + 1;  // of a row (three tokens more: rows that begin up to three in front of 16 bytes)
  p.runs = int((rows * runs + kControlWarps - 1) / kControlWarps);
  if (p.runs > runs) p.runs = int(runs);
  p.spans = int((runs - 1) / ((long long)p.runs * (kControlThreads / 32)) + 1);
  if ((long long)rows * p.spans >= 1ll << 31) return fail(MTX_ERR_ARG, "rows * vocab is too large for one call");
  MTX_TRY(on_this_device({logits, out, p.seen, p.slot, p.touched, p.repetition, p.presence, p.frequency, p.bias_off, p.bias_token, p.bias_value, p.allowed, p.allowed_row}, true));
  const uintptr_t a = reinterpret_cast<uintptr_t>(logits), o = reinterpret_cast<uintptr_t>(out);
  const bool aligned = ((a | o) & 15) == 0 && ld % 4 == 0 && ldo % 4 == 0, alike = ((a ^ o) & 15) == 0 && (ld - ldo) % 4 == 0;
  return launch(aligned ? control_logits_kernel<kControlAligned> : alike ? control_logits_kernel<kControlShifted> : control_logits_kernel<kControlSingle>,
                dim3(unsigned(rows) * unsigned(p.spans)), dim3(kControlThreads), 0, static_cast<cudaStream_t>(stream), p);
}

int mtx_note_tokens(uint16_t* seen, long long ld_seen, uint32_t* touched, long long ld_touched, int slots, int vocab, const int32_t* token, const int32_t* slot, int n, int prompt,
                    mtx_stream stream) {
  if (n < 0 || vocab < 1 || vocab > kMaxVocab) return fail(MTX_ERR_ARG, "bad n / vocab");
  if (n == 0) return MTX_OK;
  if (!seen || !token) return fail(MTX_ERR_ARG, "null argument");
  if (!slot && n > slots) return fail(MTX_ERR_ARG, "without slot, token i belongs to slot i: %d tokens for %d slots", n, slots);
  MTX_TRY(check_record(seen, ld_seen, touched, ld_touched, slots, vocab));
  if (!lie_on(4, {token, slot})) return fail(MTX_ERR_ARG, "token and slot lie on 4 bytes");
  MTX_TRY(on_this_device({seen, touched, token, slot}, true));
  NoteParams p;
  p.seen = seen;
  p.ld_seen = ld_seen;
  p.touched = touched;
  p.ld_touched = ld_touched;
  p.slots = slots;
  p.vocab = vocab;
  p.token = token;
  p.slot = slot;
  p.n = n;
  p.prompt = prompt;
  return launch(note_tokens_kernel, dim3((n - 1) / kControlThreads + 1), dim3(kControlThreads), 0, static_cast<cudaStream_t>(stream), p);
}

}  // extern "C"
