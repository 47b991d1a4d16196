// The policy loss's gradient, made in its forward pass for a loss gradient of one, taken to another
// loss gradient (muon_policy_loss_rescale; the formulas are those of logprob.hip).
//
// Bound by memory like the pass it repeats: 6144 rows of 128000 bf16 values, a quarter of them left
// out, take 458 us, 5.2 TB/s of what is read and written. Scaling the gradient in place moves as much
// (630 us over all its rows), and would round each value twice.
#include "logits.h"

extern "C" {

int muon_policy_loss_rescale(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                             int64_t vocab, const int64_t* tokens, float temperature,
                             const float* stats, const float* coef, const float* scale,
                             void* dlogits, void* stream) {
  const int rc = check("policy_loss_rescale", dtype, rows, vocab, row_stride, temperature);
  if (rc || rows == 0) return rc;
  if (!logits || !tokens || !stats || !coef || !scale || !dlogits) {
    muon_set_error("policy_loss_rescale: null tensor");
    return MUON_ERR_ARG;
  }
  if (!muon_policy_loss_one_pass(dtype, vocab)) {
    muon_set_error("policy_loss_rescale: no forward pass makes a gradient for dtype %d, vocabulary %lld",
                   dtype, (long long)vocab);
    return MUON_ERR_ARG;
  }
  const double inv = 1.0 / (double)temperature;
  const Back a = {logits, row_stride, rows, vocab, tokens, stats, coef, scale,
                  (float)(LOG2E_D * inv), (float)inv, dlogits, 0};
  return launch_backward<true>("policy_loss_rescale", a, dtype, (hipStream_t)stream);
}

}  // extern "C"
