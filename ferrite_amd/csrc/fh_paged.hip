// Attention of ragged rows over a KV cache in pages: prompts, chunks of them and single tokens in one call. A sequence's place p
// lies at row table[p / page] page + p % page of the cache, and a query at place p sees places 0 .. p:
// o = sum_k softmax_k(q k / sqrt(hd)) v.
#include "fh_seq.h"

using namespace fh;

// Workgroups that the GPU holds at a time: two a CU, three of the smaller dimensions' where their registers leave room. They share
// the keys (SeqWalk); a call of no more rows than sequences with at most PG_WHOLE places takes a workgroup a sequence and key head instead
// and needs no second launch. The rest is what was measured best:
// the least share of a workgroup, and the cost from which a tile of 128 pairs of 128 dimensions is cut (its parts are 66 KB each, written and read).
constexpr int PG_WHOLE = 448, PG_LEAST_TOKENS = 128, PG_LEAST = 256, PG_UNCUT = 512;
static int paged_slots(int head_dim) { return SQ_CUS * (head_dim == 64 ? 3 : 2); }

extern "C" size_t fh_attention_paged_workspace_bytes(int64_t rows, int sequences, int heads, int kv_heads, int head_dim,
                                                     int64_t max_context) {
  if (rows < 1 || sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_context < 1) return 0;
  // (two parts a workgroup, at most 128 pairs each and no more than there are: the bound of any call of no more)
  const int64_t pairs = std::min<int64_t>(128, rows * (heads / kv_heads));
  return parts_bytes(2 * std::max<int64_t>(paged_slots(head_dim), (int64_t)kv_heads * ((heads / kv_heads + 63) / 64)) * pairs, head_dim);
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
  const int pairs = packed_pairs(rows, sequences, a.rep, cache_dtype);
  const bool tokens = pairs == 64, small = tokens || cache_dtype == FH_F32;
  a.tile_rows = std::max(1, pairs / a.rep);
  a.head_tiles = (a.rep + pairs - 1) / pairs;
  a.slot_pairs = (int)std::min<int64_t>(pairs, rows * a.rep);
  a.whole = tokens && rows <= sequences && max_context <= PG_WHOLE;
  a.walkers = a.whole ? sequences : std::max(1, paged_slots(head_dim) / (kv_heads * a.head_tiles));
  // (the costs' unit: their sum stays below 2^30)
  const int64_t tiles = rows / a.tile_rows + std::min<int64_t>(sequences, rows), cost = max_context + SEQ_START + a.tile_rows;
  while ((double)tiles * (double)((cost + rows) >> a.unit) >= (double)(1 << 30) && a.unit < 30) ++a.unit;
  a.least = std::max(1, (small ? PG_LEAST_TOKENS : PG_LEAST) >> a.unit);
  a.uncut = small ? 0 : PG_UNCUT * head_dim / 128 >> a.unit;
  a.parts = a.walkers > 1 && !a.whole && cost >> a.unit >= a.uncut ? 2 : 1;
  if (a.parts == 1) a.uncut = 0x7FFFFFFF;
  a.part = (float*)workspace;
  const int64_t blocks = (int64_t)a.walkers * kv_heads * a.head_tiles;
  if (a.parts > 1 && (!workspace || ws_bytes < parts_bytes(2 * blocks * a.slot_pairs, head_dim) || ((uintptr_t)workspace & 15)))
    return fail(FH_EINVAL, "fh_attention_paged: a 16-byte aligned workspace of fh_attention_paged_workspace_bytes");
  return launch_seq<true>(fn, head_dim, cache_dtype, pairs, blocks, as_stream(stream), a);
}
