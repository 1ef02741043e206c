// Each request's rules on its row of logits: y = pen(x) - frequency n - presence [n > 0] + bias, and -inf where the row's
// mask bit is 0. pen(x) is x / repetition for x > 0 and x repetition otherwise, for the columns among the row's tokens;
// n is a column's count among the tokens after the prompt.
//
// A workgroup a part of a row's columns: the loads of its biases, tokens and logits go out together, the tokens that fall
// into the part are counted in LDS (integers: their order does not show) and the columns with a bias marked there, the
// logits changed in registers and written once. Bound by the logits' read and write; each part reads the row's tokens again, so
// parts are as wide as fill the GPU: two workgroups a CU of up to 32768 columns, a cell of 16 bits a column (32 where a row
// may hold 16384 tokens or more: half the columns). A marked column finds its biases by a hash of the column, a chain of
// them in LDS; more than one of a column are added in the list's order. 128 rows of 128256 columns with 8000 tokens, 300
// biases and a mask: 40 us (33 from the Infinity Cache), 3.4 TB/s of what has to move (a copy of the logits alone takes 23.5 us).
#include <math.h>
#include <algorithm>
#include "fh_common.h"

namespace fh {

constexpr int RU = 8;              // loads of logits a thread has in flight
constexpr int RBIAS = 1024;        // biases a row, at most
constexpr int RHASH = 256;         // chains of them

struct RuleArgs {
  const float* x; int64_t ldx; int64_t vocab;
  const int32_t* tokens; int64_t ldt; int max_tokens; const int32_t* lengths; const int32_t* prompts;
  const float* repetition; const float* presence; const float* frequency;
  const int32_t* bias_ids; const float* bias; int64_t ldb; int nbias;
  const uint32_t* allowed; int64_t ldm;
  float* out; int64_t ldo;
  int part;                        // columns a workgroup, a multiple of 1024
};

// A column's cell of CB bits: the count after the prompt, above it a bit for a token of the prompt and one for a bias
template <int CB>
struct RuleCell { static constexpr uint32_t PROMPT = 1u << (CB - 2), BIAS = 1u << (CB - 1); };

template <int CB>
__device__ inline float ruled(float x, uint32_t cell, float rep, float pre, float fre) {
  constexpr uint32_t PROMPT = RuleCell<CB>::PROMPT;
  const uint32_t n = cell & (PROMPT - 1);
  if (!(cell & (2 * PROMPT - 1))) return x;
  float y = x > 0.f ? x / rep : x * rep;
  if (n) y = y - fre * (float)n - pre;
  return y;
}

// VEC: rows aligned to 16 bytes and a multiple of 4 columns, 4 a load
template <int CB, bool VEC>
__global__ __launch_bounds__(512) void rules_kernel(RuleArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t cells[];  // [part] of CB bits, then the biases'
  constexpr int W = VEC ? 4 : 1;
  const int64_t row = blockIdx.y, c0 = (int64_t)blockIdx.x * a.part;
  const int tid = threadIdx.x, nt = blockDim.x, n = (int)min((int64_t)a.part, a.vocab - c0);
  const float* x = a.x + row * a.ldx + c0;
  float* out = a.out + row * a.ldo + c0;
  const uint32_t* allowed = a.allowed ? a.allowed + row * a.ldm + (c0 >> 5) : nullptr;
  const int words = a.part * CB / 32;  // (of the cells: there with tokens or biases)
  int* head = (int*)(cells + words);                                // [RHASH] a chain's first bias, or -1
  const int nb4 = (a.nbias + 3) / 4 * 4;
  int* at = head + RHASH;                                           // [nb4] a bias's column in the part (-1: not in it)
  int* next = at + nb4;                                             // [nb4] the chain's next
  float* add = (float*)(next + nb4);                                // [nb4]

  // the biases, the first tokens and the first logits on their way together (every address inside its row: no branches)
  constexpr int RB = RBIAS / 256;
  int bc[RB];
  float bv[RB];
  if (a.nbias) {
#pragma unroll
    for (int e = 0; e < RB; ++e) {
      const int64_t i = row * a.ldb + min(e * nt + tid, a.nbias - 1);
      bc[e] = a.bias_ids[i];
      bv[e] = a.bias[i];
    }
  }
  const int len = !a.tokens ? 0 : a.lengths ? min(a.lengths[row], a.max_tokens) : a.max_tokens, prompt = a.prompts ? a.prompts[row] : 0;
  const int32_t* tok = a.tokens + row * a.ldt;
  int t[RU];
  auto load_tokens = [&](int i0) {
#pragma unroll
    for (int u = 0; u < RU; ++u) t[u] = tok[min(i0 + u * nt + tid, len - 1)];
  };
  if (len > 0) load_tokens(0);
  float v[RU][W];
  uint32_t m[RU];
  auto load = [&](int j0) {
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int c = min(W * (j0 + u * nt + tid), n - W);
      if constexpr (VEC) { const float4 f = *(const float4*)(x + c); v[u][0] = f.x; v[u][1] = f.y; v[u][2] = f.z; v[u][3] = f.w; }
      else v[u][0] = x[c];
    }
    if (allowed)
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        const int c = min(W * (j0 + u * nt + tid), n - W);
        m[u] = allowed[c >> 5] >> (c & 31);  // (4 columns lie in one word)
      }
  };
  const float rep = a.repetition ? a.repetition[row] : 1.f, pre = a.presence ? a.presence[row] : 0.f, fre = a.frequency ? a.frequency[row] : 0.f;
  load(0);
  if (a.tokens || a.nbias)
    for (int i = tid; i < words / 4; i += nt) ((uint4*)cells)[i] = make_uint4(0, 0, 0, 0);
  if (a.nbias)
    for (int i = tid; i < RHASH; i += nt) head[i] = -1;
  __syncthreads();
  for (int i0 = 0; i0 < len; i0 += RU * nt) {
    if (i0) load_tokens(i0);
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int64_t c = t[u] - c0;
      if (c < 0 || c >= n || i0 + u * nt + tid >= len) continue;
      const int sh = CB == 16 ? 16 * (int)(c & 1) : 0;
      uint32_t* cell = cells + (CB == 16 ? c >> 1 : c);
      if (i0 + u * nt + tid < prompt) atomicOr(cell, RuleCell<CB>::PROMPT << sh);
      else atomicAdd(cell, 1u << sh);
    }
  }
  if (a.nbias) {
#pragma unroll
    for (int e = 0; e < RB; ++e) {
      const int i = e * nt + tid;
      if (i >= nb4) continue;
      const int64_t at_c = bc[e] - c0;
      const int c = at_c < 0 || at_c >= n || i >= a.nbias ? -1 : (int)at_c;
      at[i] = c;
      add[i] = bv[e];
      if (c < 0) continue;
      atomicOr(cells + (CB == 16 ? c >> 1 : c), RuleCell<CB>::BIAS << (CB == 16 ? 16 * (c & 1) : 0));
      next[i] = atomicExch(head + c % RHASH, i);
    }
  }
  __syncthreads();
  for (int j0 = 0; W * j0 < n; j0 += RU * nt) {
    if (j0) load(j0);
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int c = W * (j0 + u * nt + tid);
      if (c >= n) continue;
      if (a.tokens || a.nbias) {
        uint32_t cell[W];
        if constexpr (CB == 16 && VEC) {
          const uint2 w = *(const uint2*)(cells + (c >> 1));
          cell[0] = w.x & 0xFFFFu; cell[1] = w.x >> 16; cell[2] = w.y & 0xFFFFu; cell[3] = w.y >> 16;
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) cell[i] = CB == 16 ? ((const uint16_t*)cells)[c + i] : cells[c + i];
        }
        uint32_t marks = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          v[u][i] = ruled<CB>(v[u][i], cell[i], rep, pre, fre);
          if (cell[i] & RuleCell<CB>::BIAS) marks |= 1u << i;
        }
        while (marks) {
          const int i = __builtin_ctz(marks), col = c + i;
          marks &= marks - 1;
          int found = 0;
          float sum = 0.f;
          for (int j = head[col % RHASH]; j >= 0; j = next[j])
            if (at[j] == col) { ++found; sum += add[j]; }
          if (found > 2) {  // (two have one sum in either order)
            sum = 0.f;
#pragma unroll 4
            for (int j = 0; j < nb4; j += 4) {
              const int4 k = *(const int4*)(at + j);
              if (k.x == col) sum += add[j];
              if (k.y == col) sum += add[j + 1];
              if (k.z == col) sum += add[j + 2];
              if (k.w == col) sum += add[j + 3];
            }
          }
#pragma unroll
          for (int k = 0; k < W; ++k) v[u][k] = k == i ? v[u][k] + sum : v[u][k];
        }
      }
      if (allowed) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[u][i] = m[u] >> i & 1u ? v[u][i] : -INFINITY;
      }
    }
    // (the writes apart: a marked column's chain of LDS reads would wait for those before it)
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int c = W * (j0 + u * nt + tid);
      if (c >= n) continue;
      if constexpr (VEC) *(float4*)(out + c) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
      else out[c] = v[u][0];
    }
  }
}

template <int CB, bool VEC>
static void launch_rules(dim3 g, int threads, size_t lds, hipStream_t s, const RuleArgs& a) {
  if (lds > 65536)  // (on the current device, whichever it is; a refusal shows as the launch's error)
    (void)hipFuncSetAttribute((const void*)rules_kernel<CB, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);
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
  if (tokens && max_tokens >= (1LL << 30)) return fail(FH_EUNSUP, "fh_logit_rules: fewer than 2^30 tokens a row");
  if (tokens ? max_tokens < 0 || ldt < max_tokens : lengths || prompt_lengths)
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
  // Parts: two workgroups a CU of 256 share the columns in whole 1024s, at most 64 KB of cells (with the biases more than a
  // launch may have unasked: launch_rules asks). Threads by the part: 64 columns each, 256 to 512 (128 rows of 128256 with
  // tokens, 300 biases and a mask, in parts of 32768: 40 us; 256 threads 47, 1024 46; parts of 16384 42 to 50, of 26624 50).
  const bool wide = a.tokens && max_tokens >= 16384;
  const int64_t most = wide ? 16384 : 32768, even = (vocab * rows / 512 + 1023) / 1024 * 1024;
  a.part = (int)std::min(most, std::max<int64_t>(1024, even));
  const int threads = std::min(512, std::max(256, (a.part / 64 + 63) / 64 * 64));
  const size_t lds = (a.tokens || a.nbias ? (size_t)a.part * (wide ? 4 : 2) : 0) + (a.nbias ? (size_t)(a.nbias + 3) / 4 * 48 + RHASH * 4 : 0);
  const bool vec = vocab % 4 == 0 && ldl % 4 == 0 && ldo % 4 == 0 && !((uintptr_t)logits & 15) && !((uintptr_t)out & 15);
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
