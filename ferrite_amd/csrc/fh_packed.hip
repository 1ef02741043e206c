// Attention of many sequences at once over a KV cache of slots: the packed prompts of a batch (causal, each its own
// length) and the decode step of a batch whose rows share a prefix. In both a sequence's place p lies at cache row
// prefix_row + p where p < shared (rows that other sequences read too) and at first_row + p - shared behind them, and a
// query at place p sees places 0 .. p: o = sum_k softmax_k(q k / sqrt(hd)) v. A query that sees no place gives zeros.
//
// A wave a query row and head: 64 keys a round, a lane a key's score, the running max and sum of the softmax (each
// round rescales what is there), then a lane HD / 64 dimensions of p v.
#include <math.h>
#include "fh_common.h"

namespace fh {

struct SeqArgs {
  const void* q; int q_bf16; int64_t ldq;
  const void* cache; int64_t cache_len; const uint8_t* cache_exps;
  int heads, kv_heads; float scale;
  int64_t rows; int n;          // query rows; sequences
  const int32_t* starts;        // [n + 1] each sequence's first row (NULL: row b is sequence b)
  const int32_t* places;        // [n] the place of a sequence's first row
  const int32_t* first_row; const int32_t* prefix_row; const int32_t* shared;
  int64_t max_prefix, max_own;  // bounds of shared, and of the places behind it
  void* o; int o_bf16, o_tiles; int64_t ldo;
};

__device__ inline void put_out(const SeqArgs& a, int64_t row, int64_t col, float v) {
  const int64_t at = a.o_tiles ? tile16_at(row, col, a.ldo) : row * a.ldo + col;
  if (a.o_bf16) ((uint16_t*)a.o)[at] = (uint16_t)bf16_rne_f(v);
  else ((float*)a.o)[at] = v;
}

// a cache row's value, whatever the cache holds
template <int HD, int CF>
__device__ inline float cache_value(const SeqArgs& a, int64_t row, int c) {
  if constexpr (CF == FH_F32) return ((const float*)a.cache)[row * HD + c];
  else if constexpr (CF == FH_BF16) return bf16_to_f(((const uint16_t*)a.cache)[row * HD + c]);
  else {
    const uint32_t e = a.cache_exps[row * (HD / 16) + c / 16];
    int q;
    if constexpr (CF == FH_BFP8) q = ((const int8_t*)a.cache)[row * HD + c];
    else q = (int)(int8_t)(((const uint8_t*)a.cache)[row * (HD / 2) + c / 2] << ((c & 1) ? 0 : 4)) >> 4;
    return bf16_to_f(bfp_value_bf16(CF == FH_BFP4 ? 16 * q : q, e));
  }
}

// the sequence of row r: the last whose start is at most r, if r lies before its end (-1: none)
__device__ inline int sequence_of(const SeqArgs& a, int64_t r) {
  if (!a.starts) return (int)r;
  for (int s = 0; s < a.n; ++s)
    if (a.starts[s] <= r && r < a.starts[s + 1]) return s;
  return -1;
}

template <int HD, int CF>
__global__ __launch_bounds__(64) void seq_attention_kernel(SeqArgs a) {
  __shared__ float qs[HD];
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y, lane = threadIdx.x;
  const int s = sequence_of(a, row);
  if (s < 0) return;
  const int64_t shared = a.shared ? min(max((int64_t)a.shared[s], (int64_t)0), a.max_prefix) : 0;
  const int64_t place = a.places[s] + (a.starts ? row - a.starts[s] : 0);
  const int64_t keys = min(place + 1, shared + a.max_own);
  const int64_t first = (int64_t)a.first_row[s] - shared, prefix = a.prefix_row ? *a.prefix_row : 0;
  const int kvh = h / (a.heads / a.kv_heads);
  for (int i = lane; i < HD; i += 64) {
    const int64_t at = row * a.ldq + (int64_t)h * HD + i;
    qs[i] = a.q_bf16 ? bf16_to_f(((const uint16_t*)a.q)[at]) : ((const float*)a.q)[at];
  }
  __syncthreads();
  auto cache_row = [&](int64_t k) {
    const int64_t r = k < shared ? prefix + k : first + k;
    return min(max(r, (int64_t)0), a.cache_len - 1);
  };
  float m = -INFINITY, l = 0.f, o[HD / 64];
  for (int i = 0; i < HD / 64; ++i) o[i] = 0.f;
  for (int64_t k0 = 0; k0 < keys; k0 += 64) {
    const bool in = k0 + lane < keys;
    float sc = -INFINITY;
    if (in) {
      const int64_t r = (int64_t)kvh * a.cache_len + cache_row(k0 + lane);
      sc = 0.f;
      for (int c = 0; c < HD; ++c) sc = fmaf(qs[c], cache_value<HD, CF>(a, r, c), sc);
      sc *= a.scale;
    }
    const float mn = fmaxf(m, wave_max(sc));
    const float p = in ? expf(sc - mn) : 0.f, f = m == -INFINITY ? 0.f : expf(m - mn);
    l = l * f + wave_sum(p);
    m = mn;
    for (int i = 0; i < HD / 64; ++i) o[i] *= f;
    const int n = (int)min((int64_t)64, keys - k0);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl(p, j, 64);
      const int64_t r = (int64_t)(a.kv_heads + kvh) * a.cache_len + cache_row(k0 + j);
      for (int i = 0; i < HD / 64; ++i) o[i] = fmaf(pj, cache_value<HD, CF>(a, r, lane + 64 * i), o[i]);
    }
  }
  for (int i = 0; i < HD / 64; ++i) put_out(a, row, (int64_t)h * HD + lane + 64 * i, keys > 0 ? o[i] / l : 0.f);
}

template <int HD>
static void launch_seq(int cf, hipStream_t s, const SeqArgs& a) {
  const dim3 g((unsigned)a.rows, a.heads), b(64);
  switch (cf) {
    case FH_F32: hipLaunchKernelGGL((seq_attention_kernel<HD, FH_F32>), g, b, 0, s, a); break;
    case FH_BF16: hipLaunchKernelGGL((seq_attention_kernel<HD, FH_BF16>), g, b, 0, s, a); break;
    case FH_BFP8: hipLaunchKernelGGL((seq_attention_kernel<HD, FH_BFP8>), g, b, 0, s, a); break;
    default: hipLaunchKernelGGL((seq_attention_kernel<HD, FH_BFP4>), g, b, 0, s, a); break;
  }
}

// what both entry points ask of their operands (fn: the name in the message)
static int seq_check(const char* fn, const SeqArgs& a, int q_dtype, int cache_dtype, int head_dim, int o_dtype) {
  auto no = [&](int code, const char* what) { set_error("%s: %s", fn, what); return code; };
  if (!a.q || !a.cache || !a.o || !a.places || !a.first_row) return no(FH_EINVAL, "null pointer");
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads) return no(FH_EINVAL, "heads must be a multiple of kv_heads");
  if (a.heads > 65535) return no(FH_EUNSUP, "at most 65535 heads");
  if (head_dim != 64 && head_dim != 128) return no(FH_EUNSUP, "head_dim 64 or 128");
  if (q_dtype != FH_F32 && q_dtype != FH_BF16) return no(FH_EINVAL, "q is FH_F32 or FH_BF16");
  if (cache_dtype < FH_F32 || cache_dtype > FH_BFP4) return no(FH_EUNSUP, "cache is FH_F32, FH_BF16, FH_BFP8 or FH_BFP4");
  if (a.cache_len < 1) return no(FH_EINVAL, "cache_len at least 1");
  if ((a.shared == nullptr) != (a.prefix_row == nullptr)) return no(FH_EINVAL, "prefix_row and shared go together");
  const int64_t cols = (int64_t)a.heads * head_dim;
  if (a.ldq < cols || a.ldo < cols || a.ldq % (q_dtype == FH_F32 ? 4 : 8) || (o_dtype != FH_BF16_T16 && a.ldo % 4) ||
      ((uintptr_t)a.q & 15) || ((uintptr_t)a.cache & 15) || ((uintptr_t)a.o & (o_dtype == FH_F32 ? 15 : 7)))
    return no(FH_EINVAL, "rows at least heads * head_dim, q's and the cache's 16-byte aligned, o's 4 values");
  return FH_OK;
}

}  // namespace fh

using namespace fh;

extern "C" size_t fh_attention_packed_workspace_bytes(int64_t rows, int sequences, int heads, int kv_heads, int head_dim,
                                                      int64_t max_context) {
  return 0;
}

extern "C" int fh_attention_prefill_packed(const void* q, int q_dtype, int64_t ldq, const void* cache, int cache_dtype,
                                           int64_t cache_len, int64_t rows, int sequences, int heads, int kv_heads,
                                           int head_dim, const int32_t* starts, const int32_t* p0,
                                           const int32_t* first_row, const int32_t* prefix_row, const int32_t* shared,
                                           int64_t max_context, void* o, int o_dtype, int64_t ldo, void* workspace,
                                           size_t ws_bytes, void* stream) {
  const char* fn = "fh_attention_prefill_packed";
  SeqArgs a = {};
  a.q = q; a.q_bf16 = q_dtype == FH_BF16; a.ldq = ldq; a.cache = cache; a.cache_len = cache_len;
  a.heads = heads; a.kv_heads = kv_heads; a.rows = rows; a.n = sequences;
  a.starts = starts; a.places = p0; a.first_row = first_row; a.prefix_row = prefix_row; a.shared = shared;
  a.max_prefix = max_context; a.max_own = max_context; a.o = o; a.o_bf16 = o_dtype == FH_BF16; a.ldo = ldo;
  if (!starts) return fail(FH_EINVAL, "fh_attention_prefill_packed: null pointer");
  if (rows < 1 || rows >= (1LL << 31) || sequences < 1 || max_context < 1)
    return fail(FH_EINVAL, "fh_attention_prefill_packed: need 1 <= rows < 2^31, sequences >= 1 and max_context >= 1");
  if (o_dtype != FH_F32 && o_dtype != FH_BF16) return fail(FH_EINVAL, "fh_attention_prefill_packed: o is FH_F32 or FH_BF16");
  if (int rc = seq_check(fn, a, q_dtype, cache_dtype, head_dim, o_dtype)) return rc;
  a.cache_exps = (const uint8_t*)cache + kv_exps_at(cache_dtype, kv_heads, cache_len, head_dim);
  a.scale = 1.0f / sqrtf((float)head_dim);
  if (head_dim == 128) launch_seq<128>(cache_dtype, as_stream(stream), a);
  else launch_seq<64>(cache_dtype, as_stream(stream), a);
  return check_launch(fn);
}

extern "C" size_t fh_attention_shared_workspace_bytes(int batch, int heads, int kv_heads, int head_dim, int64_t max_prefix,
                                                      int64_t max_own) {
  return 0;
}

extern "C" int fh_attention_decode_shared(const void* q, int q_dtype, const void* cache, int cache_dtype, int64_t cache_len,
                                          int batch, int heads, int kv_heads, int head_dim, const int32_t* places,
                                          const int32_t* first_row, const int32_t* prefix_row, const int32_t* shared,
                                          int64_t max_prefix, int64_t max_own, void* o, int o_dtype, void* workspace,
                                          size_t ws_bytes, void* stream) {
  const char* fn = "fh_attention_decode_shared";
  SeqArgs a = {};
  a.q = q; a.q_bf16 = q_dtype == FH_BF16; a.ldq = (int64_t)heads * head_dim; a.cache = cache; a.cache_len = cache_len;
  a.heads = heads; a.kv_heads = kv_heads; a.rows = batch; a.n = batch;
  a.places = places; a.first_row = first_row; a.prefix_row = prefix_row; a.shared = shared;
  a.max_prefix = max_prefix; a.max_own = max_own;
  a.o = o; a.o_bf16 = o_dtype != FH_F32; a.o_tiles = o_dtype == FH_BF16_T16; a.ldo = a.ldq;
  if (!prefix_row || !shared) return fail(FH_EINVAL, "fh_attention_decode_shared: null pointer");
  if (batch < 1 || max_prefix < 0 || max_own < 0)
    return fail(FH_EINVAL, "fh_attention_decode_shared: need batch >= 1, max_prefix and max_own at least 0");
  if (o_dtype != FH_F32 && o_dtype != FH_BF16 && o_dtype != FH_BF16_T16)
    return fail(FH_EINVAL, "fh_attention_decode_shared: o is FH_F32, FH_BF16 or FH_BF16_T16");
  if (int rc = seq_check(fn, a, q_dtype, cache_dtype, head_dim, o_dtype)) return rc;
  a.cache_exps = (const uint8_t*)cache + kv_exps_at(cache_dtype, kv_heads, cache_len, head_dim);
  a.scale = 1.0f / sqrtf((float)head_dim);
  if (head_dim == 128) launch_seq<128>(cache_dtype, as_stream(stream), a);
  else launch_seq<64>(cache_dtype, as_stream(stream), a);
  return check_launch(fn);
}
