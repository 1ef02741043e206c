// Each request's rules on its row of logits: y = pen(x) - frequency n - presence [n > 0] + bias, and -inf where the row's
// mask bit is 0. pen(x) is x / repetition for x > 0 and x repetition otherwise, for the columns among the row's tokens;
// n is a column's count among the tokens after the prompt.
//
// A workgroup a part of a row's columns: the loads of its tokens and logits go out together, the tokens that fall into the part
// are counted in LDS (integers: their order does not show), the logits changed in registers and written. A column with a bias
// is the thread's of the first entry that names it, which adds the column's entries in the list's order and writes the column
// once more, behind the others. Bound by the
// logits' read and write; each part reads the row's tokens again, so parts are as wide as fill the GPU: two workgroups a CU
// of up to 32768 columns, a count of 16 bits a column (32 where a row may hold 32768 tokens or more: half the columns).
#include <math.h>
#include <algorithm>
#include "fh_common.h"

namespace fh {

constexpr int RU = 8;              // loads of logits a thread has in flight
constexpr int RBIAS = 1024;        // biases a row, at most

struct RuleArgs {
  const float* x; int64_t ldx; int64_t vocab;
  const int32_t* tokens; int64_t ldt; int max_tokens; const int32_t* lengths; const int32_t* prompts;
  const float* repetition; const float* presence; const float* frequency;
  const int32_t* bias_ids; const float* bias; int64_t ldb; int nbias;
  const uint32_t* allowed; int64_t ldm;
  float* out; int64_t ldo;
  int part;                        // columns a workgroup, a multiple of 1024
};

// A column's cell of CB bits: the count after the prompt, and above it a bit for a token of the prompt
template <int CB>
__device__ inline float ruled(float x, uint32_t cell, float rep, float pre, float fre) {
  constexpr uint32_t PROMPT = 1u << (CB - 1);
  if (!cell) return x;
  const uint32_t n = cell & (PROMPT - 1);
  float y = x > 0.f ? x / rep : x * rep;
  if (n) y = y - fre * (float)n - pre;
  return y;
}

// VEC: rows aligned to 16 bytes, 4 columns a load
template <int CB, bool VEC>
__global__ __launch_bounds__(1024) void rules_kernel(RuleArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t cells[];  // [part] of CB bits, then the biases' columns
  constexpr int W = VEC ? 4 : 1;
  const int64_t row = blockIdx.y, c0 = (int64_t)blockIdx.x * a.part;
  const int tid = threadIdx.x, nt = blockDim.x, n = (int)min((int64_t)a.part, a.vocab - c0);
  const float* x = a.x + row * a.ldx + c0;
  float* out = a.out + row * a.ldo + c0;
  const uint32_t* allowed = a.allowed ? a.allowed + row * a.ldm + (c0 >> 5) : nullptr;
  const int words = a.part * CB / 32;
  int* at = (int*)(cells + words);                                  // [nbias in fours] a bias's column in the part (-1: not in it)
  float* add = (float*)(at + (a.nbias + 3) / 4 * 4);                // the biases

  // the first tokens, the biases' columns and the first logits on their way together
  const int len = !a.tokens ? 0 : a.lengths ? min(a.lengths[row], a.max_tokens) : a.max_tokens, prompt = a.prompts ? a.prompts[row] : 0;
  const int32_t* tok = a.tokens + row * a.ldt;
  int t[RU];
  auto load_tokens = [&](int i0) {
#pragma unroll
    for (int u = 0; u < RU; ++u) { const int i = i0 + u * nt + tid; t[u] = i < len ? tok[i] : -1; }
  };
  float v[RU][W];
  auto load = [&](int j0) {
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int c = W * (j0 + u * nt + tid);
      if constexpr (VEC) {
        if (c + 4 <= n) { const float4 f = *(const float4*)(x + c); v[u][0] = f.x; v[u][1] = f.y; v[u][2] = f.z; v[u][3] = f.w; }
        else
#pragma unroll
          for (int i = 0; i < 4; ++i) v[u][i] = c + i < n ? x[c + i] : 0.f;
      } else v[u][0] = c < n ? x[c] : 0.f;
    }
  };
  load_tokens(0);
  const int nb4 = (a.nbias + 3) / 4 * 4;
  for (int i = tid; i < nb4; i += nt) {
    const int64_t c = i < a.nbias ? a.bias_ids[row * a.ldb + i] - c0 : -1;
    at[i] = c < 0 || c >= n ? -1 : (int)c;
    add[i] = i < a.nbias ? a.bias[row * a.ldb + i] : 0.f;
  }
  const float rep = a.repetition ? a.repetition[row] : 1.f, pre = a.presence ? a.presence[row] : 0.f, fre = a.frequency ? a.frequency[row] : 0.f;
  load(0);
  if (a.tokens)
    for (int i = tid; i < words / 4; i += nt) ((uint4*)cells)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  for (int i0 = 0; i0 < len; i0 += RU * nt) {
    if (i0) load_tokens(i0);
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int64_t c = t[u] - c0;
      if (c < 0 || c >= n) continue;
      const int sh = CB == 16 ? 16 * (int)(c & 1) : 0;
      uint32_t* cell = cells + (CB == 16 ? c >> 1 : c);
      if (i0 + u * nt + tid < prompt) atomicOr(cell, 1u << (sh + CB - 1));
      else atomicAdd(cell, 1u << sh);
    }
  }
  // this thread's columns with a bias: the logit (read before any is written), the biases' sum
  constexpr int RB = RBIAS / 256;
  int bc[RB];
  float bx[RB], bs[RB];
#pragma unroll
  for (int e = 0; e < RB; ++e) {
    const int i = e * nt + tid;
    bc[e] = -1;
    if (i >= a.nbias) continue;
    const int c = at[i];
    if (c < 0 || (allowed && !(allowed[c >> 5] >> (c & 31) & 1u))) continue;
    bx[e] = x[c];
    bool first = true;
    float sum = 0.f;
#pragma unroll 4
    for (int j = 0; j < nb4; j += 4) {
      const int4 k = *(const int4*)(at + j);
      if (k.x != c && k.y != c && k.z != c && k.w != c) continue;
      if (k.x == c) { first = first && j >= i; sum += add[j]; }
      if (k.y == c) { first = first && j + 1 >= i; sum += add[j + 1]; }
      if (k.z == c) { first = first && j + 2 >= i; sum += add[j + 2]; }
      if (k.w == c) { first = first && j + 3 >= i; sum += add[j + 3]; }
    }
    if (first) { bc[e] = c; bs[e] = sum; }
  }
  __syncthreads();
  for (int j0 = 0; W * j0 < n; j0 += RU * nt) {
    if (j0) load(j0);
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int c = W * (j0 + u * nt + tid);
      if (c >= n) continue;
      if (a.tokens) {
        uint32_t cell[W];
        if constexpr (CB == 16 && VEC) {
          const uint2 w = *(const uint2*)(cells + (c >> 1));
          cell[0] = w.x & 0xFFFFu; cell[1] = w.x >> 16; cell[2] = w.y & 0xFFFFu; cell[3] = w.y >> 16;
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) cell[i] = CB == 16 ? ((const uint16_t*)cells)[c + i] : cells[c + i];
        }
#pragma unroll
        for (int i = 0; i < W; ++i) v[u][i] = ruled<CB>(v[u][i], cell[i], rep, pre, fre);
      }
      if (allowed) {
        const uint32_t m = allowed[c >> 5] >> (c & 31);  // (4 columns lie in one word)
#pragma unroll
        for (int i = 0; i < W; ++i) v[u][i] = m >> i & 1u ? v[u][i] : -INFINITY;
      }
      if constexpr (VEC) {
        if (c + 4 <= n) { *(float4*)(out + c) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]); continue; }
      }
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (c + i < n) out[c + i] = v[u][i];
    }
  }
  if (!a.nbias) return;
  __syncthreads();  // (the part is written)
#pragma unroll
  for (int e = 0; e < RB; ++e)
    if (bc[e] >= 0) {
      const uint32_t cell = !a.tokens ? 0u : CB == 16 ? ((const uint16_t*)cells)[bc[e]] : cells[bc[e]];
      out[bc[e]] = ruled<CB>(bx[e], cell, rep, pre, fre) + bs[e];
    }
}

template <int CB, bool VEC>
static void launch_rules(dim3 g, int threads, size_t lds, hipStream_t s, const RuleArgs& a) {
  static const hipError_t allowed = hipFuncSetAttribute((const void*)rules_kernel<CB, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);
  (void)allowed;  // (a refusal shows as the launch's error)
  hipLaunchKernelGGL((rules_kernel<CB, VEC>), g, dim3(threads), lds, s, a);
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
  if (bias_ids && biases > RBIAS) return fail(FH_EUNSUP, "fh_logit_rules: at most 1024 biases a row");
  if (allowed && ldm < (vocab + 31) / 32) return fail(FH_EINVAL, "fh_logit_rules: a mask's row holds a bit a column");
  RuleArgs a = {};
  a.x = logits; a.ldx = ldl; a.vocab = vocab; a.tokens = max_tokens ? tokens : nullptr; a.ldt = ldt; a.max_tokens = (int)max_tokens;
  a.lengths = lengths; a.prompts = prompt_lengths; a.repetition = repetition; a.presence = presence; a.frequency = frequency;
  a.bias_ids = bias_ids; a.bias = bias; a.ldb = ldb; a.nbias = bias_ids ? (int)biases : 0;
  a.allowed = (const uint32_t*)allowed; a.ldm = ldm; a.out = out; a.ldo = ldo;
  // parts: two workgroups a CU of 256, at least 1024 columns, at most 64 KB of cells; 8 columns a thread up to 1024 threads
  const bool wide = a.tokens && max_tokens >= 32768;
  const int64_t most = wide ? 16384 : 32768, even = (vocab * rows / 512 + 1023) / 1024 * 1024;
  a.part = (int)std::min(most, std::max<int64_t>(1024, even));
  const int threads = std::min(1024, std::max(256, a.part / 8));
  const size_t lds = (size_t)a.part * (wide ? 4 : 2) + (size_t)(a.nbias + 3) / 4 * 32;
  const bool vec = ldl % 4 == 0 && ldo % 4 == 0 && !((uintptr_t)logits & 15) && !((uintptr_t)out & 15);
  const dim3 g((unsigned)((vocab + a.part - 1) / a.part), (unsigned)rows);
  if (wide) {
    if (vec) launch_rules<32, true>(g, threads, lds, as_stream(stream), a);
    else launch_rules<32, false>(g, threads, lds, as_stream(stream), a);
  } else {
    if (vec) launch_rules<16, true>(g, threads, lds, as_stream(stream), a);
    else launch_rules<16, false>(g, threads, lds, as_stream(stream), a);
  }
  return check_launch("fh_logit_rules");
}
