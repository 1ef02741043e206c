// Attention of many sequences at once over a KV cache of slots: the packed prompts of a batch (causal, each its own
// length) and the decode step of a batch whose rows share a prefix. In both a sequence's place p lies at cache row
// prefix_row + p where p < shared (rows that other sequences read too) and at first_row + p - shared behind them, and a
// query at place p sees places 0 .. p: o = sum_k softmax_k(q k / sqrt(hd)) v. A query that sees no place gives zeros.
//
// The query heads of a key head read the same keys, so a workgroup of 4 waves takes pairs (query row, head of the group) of one
// key head, 32 a wave: a prompt of 20 rows of 4 heads a key head is one tile of 80 pairs, and 8 rows of a decode step behind one
// prefix are 32. 128 pairs a workgroup, or 64 with the tile's keys shared by two groups of waves (a decode step, prompts of few
// rows: what those wait for is a wave's chain of products). It walks the keys its pairs see in tiles of 64 staged in LDS, the
// next tile's loads in flight meanwhile. Scores transposed, S^T = K Q^T, keys down and pairs across: a lane holds one pair's
// scores, so the softmax's statistics need one exchange between the wave's halves; and P^T is the next product's operand as it
// lies, O^T += V^T P^T. The running max moves only when a tile's lies more than 2^8 above it: weights up to 256 lose nothing in
// fp32 sums or bf16 products, and the output is rescaled a few times a row rather than every tile.
//
// The arithmetic goes by the types. A bf16 or block-float cache (whose values are bf16) takes v_mfma_f32_32x32x16_bf16: for bf16
// output an fp32 q and the softmax's weights go in as two bf16 terms each, off by 2^-16 of themselves at most, as the decode
// attention over whole slots keeps them (a bf16 q is exact in one; the weights' sum is taken before their rounding). Weights in
// one term, 2^-8, are 1-24% faster (4 prompts of up to 4096 334 us, two terms 441; 16 of up to 400 46 and 51; 64 rows behind
// 16384 54 and 62), but take the output's error from its own rounding's 1.6e-3 to 2.3e-3. For fp32 output q and the weights go
// in as three terms, off by 2^-24 at most. An fp32 cache takes v_mfma_f32_32x32x2_f32, nothing rounded.
//
// Where tiles are few, the keys are split among workgroups (splits_for), each leaving its weighted sum, max and sum of weights
// in the workspace, and a second kernel joins them; a shared prefix's keys and a row's own are always parts of their own. Joining
// in the last workgroup instead would need a release at device scope, which costs more here than the second launch.
//
// A key that a pair does not see has the weight 0, but 0 times an infinite or NaN value is NaN: a wave whose result is not
// finite takes its pairs again one at a time over the keys each sees alone (attend_again).
//
// What bounds it (32 heads of 128, 8 key heads, MI355X; ranges over cards and runs): four prompts of up to 4096 tokens 441-481 us
// with a bf16 q, 537-567 with an fp32 one: the products, counted with their terms, at 950-1030 and 1070-1130 TFLOP/s where the
// library's 8192^3 product reaches 1200; the matrix cores are busy 52% of the cycles at the 1.76 GHz the chip holds under this
// load. 16 prompts of up to 400 tokens, fp32 q: 51-56 us for 122 MB; a workgroup's few tiles do not hide its start and end. 64 rows
// behind a prefix of 16384, each with up to 700 rows of its own: 62-73 us, 5 of them the join; 16 rows behind 4096: 18-19, a
// chain of two launches and their latencies.
#include "fh_seq.h"

using namespace fh;

extern "C" size_t fh_attention_packed_workspace_bytes(int64_t rows, int sequences, int heads, int kv_heads, int head_dim,
                                                      int64_t max_context) {
  if (rows < 1 || sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_context < 1) return 0;
  const int s = most_splits(max_context);
  return s == 1 ? 0 : parts_bytes(std::min(rows * heads * s, SQ_PACKED_PARTS), head_dim);
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
  a.max_prefix = cache_len; a.max_own = std::min(max_context, 2 * cache_len);  // (no more than a prefix and a slot hold)
  a.o = o; a.o_bf16 = o_dtype == FH_BF16; a.ldo = ldo;
  if (!starts) return fail(FH_EINVAL, "fh_attention_prefill_packed: null pointer");
  if (rows < 1 || rows >= (1LL << 31) || sequences < 1 || max_context < 1)
    return fail(FH_EINVAL, "fh_attention_prefill_packed: need 1 <= rows < 2^31, sequences >= 1 and max_context >= 1");
  if (o_dtype != FH_F32 && o_dtype != FH_BF16) return fail(FH_EINVAL, "fh_attention_prefill_packed: o is FH_F32 or FH_BF16");
  if (int rc = seq_check(fn, a, q_dtype, cache_dtype, head_dim, o_dtype)) return rc;
  a.rep = heads / kv_heads;
  a.cache_exps = (const uint8_t*)cache + kv_exps_at(cache_dtype, kv_heads, cache_len, head_dim);
  a.scale = 1.0f / sqrtf((float)head_dim);
  a.splits = a.parts = packed_splits(rows, sequences, heads, kv_heads, head_dim, cache_dtype, max_context);
  a.part = (float*)workspace;
  if (a.parts > 1 && (!workspace || ws_bytes < parts_bytes(rows * heads * a.parts, head_dim) || ((uintptr_t)workspace & 15)))
    return fail(FH_EINVAL, "fh_attention_prefill_packed: a 16-byte aligned workspace of fh_attention_packed_workspace_bytes");
  const int pairs = packed_pairs(rows, sequences, a.rep, cache_dtype);
  return launch_seq<false>(fn, head_dim, cache_dtype, pairs, packed_tiles(rows, sequences, a.rep, pairs) * a.splits * kv_heads, as_stream(stream), a);
}

extern "C" size_t fh_attention_shared_workspace_bytes(int batch, int heads, int kv_heads, int head_dim, int64_t max_prefix,
                                                      int64_t max_own) {
  if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_prefix < 0 || max_own < 0) return 0;
  const int64_t pairs = (int64_t)batch * heads;
  return parts_bytes(std::max(2 * pairs, std::min(pairs * (most_splits(max_prefix) + most_splits(max_own)), SQ_SHARED_PARTS)), head_dim);
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
  a.max_prefix = std::min(max_prefix, cache_len); a.max_own = std::min(max_own, cache_len);
  a.o = o; a.o_bf16 = o_dtype != FH_F32; a.o_tiles = o_dtype == FH_BF16_T16; a.ldo = a.ldq;
  if (!prefix_row || !shared) return fail(FH_EINVAL, "fh_attention_decode_shared: null pointer");
  if (batch < 1 || max_prefix < 0 || max_own < 0)
    return fail(FH_EINVAL, "fh_attention_decode_shared: need batch >= 1, max_prefix and max_own at least 0");
  if (o_dtype != FH_F32 && o_dtype != FH_BF16 && o_dtype != FH_BF16_T16)
    return fail(FH_EINVAL, "fh_attention_decode_shared: o is FH_F32, FH_BF16 or FH_BF16_T16");
  if (int rc = seq_check(fn, a, q_dtype, cache_dtype, head_dim, o_dtype)) return rc;
  a.rep = heads / kv_heads;
  a.cache_exps = (const uint8_t*)cache + kv_exps_at(cache_dtype, kv_heads, cache_len, head_dim);
  a.scale = 1.0f / sqrtf((float)head_dim);
  shared_splits(batch, heads, kv_heads, head_dim, cache_dtype, max_prefix, max_own, a.tiles, a.splits, a.own_splits);
  a.parts = a.splits + a.own_splits;
  a.part = (float*)workspace;
  if (!workspace || ws_bytes < parts_bytes((int64_t)batch * heads * a.parts, head_dim) || ((uintptr_t)workspace & 15))
    return fail(FH_EINVAL, "fh_attention_decode_shared: a 16-byte aligned workspace of fh_attention_shared_workspace_bytes");
  const int pairs = shared_pairs(cache_dtype), row_tiles = (a.rep + pairs - 1) / pairs;
  return launch_seq<false>(fn, head_dim, cache_dtype, 64, ((int64_t)a.tiles * a.splits + (int64_t)batch * row_tiles * a.own_splits) * kv_heads, as_stream(stream), a);
}
