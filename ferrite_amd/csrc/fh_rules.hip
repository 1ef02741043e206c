// Each request's rules on its row of logits: y = pen(x) - frequency n - presence [n > 0] + bias, and -inf where the row's
// mask bit is 0. pen(x) is x / repetition for x > 0 and x repetition otherwise, for the columns among the row's tokens;
// n is a column's count among the tokens after the prompt.
//
// A workgroup a part of a row's columns: the row's tokens that fall into the part are counted in LDS (integers: their
// order does not show), the biases' sums formed there, and then the part is read and written once. Bound by that read and
// write and, for long histories, by each part's read of the row's tokens.
#include <math.h>
#include "fh_common.h"

namespace fh {

constexpr int RT = 256;            // threads a workgroup
constexpr int RPART = 4096;        // columns a part
constexpr uint32_t SEEN = 1u << 31;  // a column's word: SEEN if among the tokens, the count of those after the prompt below

struct RuleArgs {
  const float* x; int64_t ldx; int64_t vocab;
  const int32_t* tokens; int64_t ldt, max_tokens; const int32_t* lengths; const int32_t* prompts;
  const float* repetition; const float* presence; const float* frequency;
  const int32_t* bias_ids; const float* bias; int64_t ldb; int nbias;
  const uint32_t* allowed; int64_t ldm;
  float* out; int64_t ldo;
};

__global__ __launch_bounds__(RT) void rules_kernel(RuleArgs a) {
  __shared__ uint32_t count[RPART];
  __shared__ float add[RPART];
  const int64_t row = blockIdx.y, c0 = (int64_t)blockIdx.x * RPART;
  const int tid = threadIdx.x, n = (int)min((int64_t)RPART, a.vocab - c0);
  for (int i = tid; i < n; i += RT) { count[i] = 0; add[i] = 0.f; }
  __syncthreads();
  if (a.tokens) {
    const int64_t len = a.lengths ? min((int64_t)a.lengths[row], a.max_tokens) : a.max_tokens;
    const int64_t prompt = a.prompts ? a.prompts[row] : 0;
    for (int64_t i = tid; i < len; i += RT) {
      const int64_t c = a.tokens[row * a.ldt + i] - c0;
      if (c < 0 || c >= n) continue;
      atomicOr(&count[c], SEEN);
      if (i >= prompt) atomicAdd(&count[c], 1u);
    }
  }
  // each column's biases, in the list's order: the thread of a column's first entry adds them
  for (int i = tid; i < a.nbias; i += RT) {
    const int32_t* ids = a.bias_ids + row * a.ldb;
    const int64_t c = ids[i] - c0;
    if (c < 0 || c >= n) continue;
    bool first = true;
    for (int j = 0; j < i; ++j) first = first && ids[j] != ids[i];
    if (!first) continue;
    float s = 0.f;
    for (int j = i; j < a.nbias; ++j)
      if (ids[j] == ids[i]) s += a.bias[row * a.ldb + j];
    add[c] = s;
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[row] : 1.f, pre = a.presence ? a.presence[row] : 0.f, fre = a.frequency ? a.frequency[row] : 0.f;
  for (int i = tid; i < n; i += RT) {
    const int64_t c = c0 + i;
    float y = a.x[row * a.ldx + c];
    const uint32_t w = count[i], k = w & ~SEEN;
    if (w & SEEN) y = y > 0.f ? y / rep : y * rep;
    if (k) y = y - fre * (float)k - pre;
    y += add[i];
    if (a.allowed && !(a.allowed[row * a.ldm + (c >> 5)] >> (c & 31) & 1u)) y = -INFINITY;
    a.out[row * a.ldo + c] = y;
  }
}

}  // namespace fh

using namespace fh;

extern "C" int fh_logit_rules(const float* logits, int64_t ldl, int64_t rows, int64_t vocab, const int32_t* tokens,
                              int64_t ldt, int64_t max_tokens, const int32_t* lengths, const int32_t* prompt_lengths,
                              const float* repetition, const float* presence, const float* frequency,
                              const int32_t* bias_ids, const float* bias, int64_t ldb, int64_t biases,
                              const int32_t* allowed, int64_t ldm, float* out, int64_t ldo, void* stream) {
  if (!logits || !out) return fail(FH_EINVAL, "fh_logit_rules: null pointer");
  if (rows < 1 || vocab < 1 || ldl < vocab || ldo < vocab) return fail(FH_EINVAL, "fh_logit_rules: need rows, vocab >= 1, ldl and ldo >= vocab");
  if (rows > 65535 || vocab > (1LL << 31) - 1) return fail(FH_EUNSUP, "fh_logit_rules: at most 65535 rows and 2^31 - 1 columns");
  if (out == logits && ldo != ldl) return fail(FH_EINVAL, "fh_logit_rules: in place, ldo is ldl");
  if (tokens ? max_tokens < 0 || ldt < max_tokens || max_tokens > (1LL << 31) - 1 : lengths || prompt_lengths)
    return fail(FH_EINVAL, "fh_logit_rules: tokens' rows at least max_tokens apart, lengths only with tokens");
  if ((bias_ids == nullptr) != (bias == nullptr) || (bias_ids && (biases < 0 || ldb < biases)))
    return fail(FH_EINVAL, "fh_logit_rules: bias_ids and bias go together, rows at least biases apart");
  if (bias_ids && biases > 1024) return fail(FH_EUNSUP, "fh_logit_rules: at most 1024 biases a row");
  if (allowed && ldm < (vocab + 31) / 32) return fail(FH_EINVAL, "fh_logit_rules: a mask's row holds a bit a column");
  RuleArgs a = {};
  a.x = logits; a.ldx = ldl; a.vocab = vocab; a.tokens = max_tokens ? tokens : nullptr; a.ldt = ldt; a.max_tokens = max_tokens;
  a.lengths = lengths; a.prompts = prompt_lengths; a.repetition = repetition; a.presence = presence; a.frequency = frequency;
  a.bias_ids = bias_ids; a.bias = bias; a.ldb = ldb; a.nbias = bias_ids ? (int)biases : 0;
  a.allowed = (const uint32_t*)allowed; a.ldm = ldm; a.out = out; a.ldo = ldo;
  hipLaunchKernelGGL(rules_kernel, dim3((unsigned)((vocab + RPART - 1) / RPART), (unsigned)rows), dim3(RT), 0, as_stream(stream), a);
  return check_launch("fh_logit_rules");
}
