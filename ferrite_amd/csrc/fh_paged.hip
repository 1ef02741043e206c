// Attention of ragged rows over a KV cache in pages: prompts, chunks of them and single tokens in one call. A sequence's place p
// lies at row table[p / page] page + p % page of the cache, and a query at place p sees places 0 .. p:
// o = sum_k softmax_k(q k / sqrt(hd)) v.
#include "fh_seq.h"

using namespace fh;

extern "C" size_t fh_attention_paged_workspace_bytes(int64_t rows, int sequences, int heads, int kv_heads, int head_dim,
                                                     int64_t max_context) {
  if (rows < 1 || sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_context < 1) return 0;
  const int s = most_splits(max_context);
  return s == 1 ? 0 : parts_bytes(std::min(rows * heads * s, SQ_PACKED_PARTS), head_dim);
}

extern "C" int fh_attention_paged(const void* q, int q_dtype, int64_t ldq, const void* cache, int cache_dtype, int64_t cache_len,
                                  int64_t rows, int sequences, int heads, int kv_heads, int head_dim, const int32_t* starts,
                                  const int32_t* p0, const int32_t* tables, int64_t ldt, int64_t table_cols, int page,
                                  int64_t max_context, void* o, int o_dtype, int64_t ldo, void* workspace, size_t ws_bytes,
                                  void* stream) {
  const char* fn = "fh_attention_paged";
  SeqArgs a = {};
  a.q = q; a.q_bf16 = q_dtype == FH_BF16; a.ldq = ldq; a.cache = cache; a.cache_len = cache_len;
  a.heads = heads; a.kv_heads = kv_heads; a.rows = rows; a.n = sequences;
  a.starts = starts; a.places = p0; a.tables = tables; a.ldt = ldt;
  a.o = o; a.o_bf16 = o_dtype == FH_BF16; a.ldo = ldo;
  if (!starts || !tables) return fail(FH_EINVAL, "fh_attention_paged: null pointer");
  if (rows < 1 || rows >= (1LL << 31) || sequences < 1 || max_context < 1)
    return fail(FH_EINVAL, "fh_attention_paged: need 1 <= rows < 2^31, sequences >= 1 and max_context >= 1");
  if (page < 16 || (page & (page - 1))) return fail(FH_EUNSUP, "fh_attention_paged: pages of 16, 32, 64, ... rows (a power of 2)");
  if (cache_len < page || cache_len % page) return fail(FH_EINVAL, "fh_attention_paged: cache_len is whole pages");
  if (table_cols < 1 || ldt < table_cols) return fail(FH_EINVAL, "fh_attention_paged: tables of at least one page a sequence, rows at least as far apart");
  if (o_dtype != FH_F32 && o_dtype != FH_BF16) return fail(FH_EINVAL, "fh_attention_paged: o is FH_F32 or FH_BF16");
  if (int rc = seq_check(fn, a, q_dtype, cache_dtype, head_dim, o_dtype)) return rc;
  a.page_shift = __builtin_ctz((unsigned)page);
  a.pages = (int)(cache_len >> a.page_shift);
  a.table_cols = (int)std::min<int64_t>(table_cols, 1 << 30);
  max_context = std::min(max_context, (int64_t)a.table_cols << a.page_shift);
  a.max_own = max_context;
  a.rep = heads / kv_heads;
  a.cache_exps = (const uint8_t*)cache + kv_exps_at(cache_dtype, kv_heads, cache_len, head_dim);
  a.scale = 1.0f / sqrtf((float)head_dim);
  a.splits = a.parts = packed_splits(rows, sequences, heads, kv_heads, head_dim, cache_dtype, max_context);
  a.part = (float*)workspace;
  if (a.parts > 1 && (!workspace || ws_bytes < parts_bytes(rows * heads * a.parts, head_dim) || ((uintptr_t)workspace & 15)))
    return fail(FH_EINVAL, "fh_attention_paged: a 16-byte aligned workspace of fh_attention_paged_workspace_bytes");
  const int pairs = packed_pairs(rows, sequences, a.rep, cache_dtype);
  return launch_seq<true>(fn, head_dim, cache_dtype, pairs, packed_tiles(rows, sequences, a.rep, pairs) * a.splits * kv_heads, as_stream(stream), a);
}
